"""Serving over a paged KV cache on the GPU (yllm_amd/paged.py) against plain 64-bit forms.

Tolerances count roundings: at most half a step each (f16 2^-11, bf16 2^-8, fp32 2^-24 of the value)."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- paged_plan ----------------------------------------------------------------------------------

def plan_oracle(table, ctx, new, free, n_free, block, n_tok):
    """The plan in plain Python; table (a list of rows) is updated.  What passes 31 bits is reported as 2^31 - 1."""
    top = 0x7fffffff
    width, n = len(table[0]) if table else 1, len(ctx)
    cu, lens, slots, pos = [0], [], [-1] * n_tok, [0] * n_tok
    taken = used = missed = 0
    nf = min(max(n_free, 0), len(free))
    for i in range(n):
        rows, ok = max(new[i], 0), ctx[i] >= 0 and new[i] >= 0
        c = max(ctx[i], 0)
        held = -(-c // block)
        ok = ok and -(-(c + rows) // block) <= width  # (of those that can never be served no blocks are counted)
        need = -(-(c + rows) // block) - held if ok else 0
        ok = ok and (need == 0 or taken + need <= nf) and cu[-1] + rows <= n_tok
        if ok:
            for t in range(need):
                table[i][held + t] = free[nf - 1 - taken - t]
            used += need
        else:
            missed += 1
        for r in range(min(rows, max(0, n_tok - cu[-1]))):
            at = cu[-1] + r
            pos[at] = c + r
            page = table[i][(c + r) // block] if ok else -1
            slots[at] = page * block + (c + r) % block if page >= 0 else -1
        lens.append(c + rows if ok else 0)
        taken += need
        cu.append(cu[-1] + rows)
    cut = [[min(x, top) for x in v] for v in (cu, lens, slots, pos)]
    return *cut, [nf - used, min(cu[-1], top), missed, max(0, taken - nf)]


def _plan_case(ctx, new, block, width, n_free, pad=0, seed=0, cap=None):
    g = torch.Generator().manual_seed(seed)
    n = len(ctx)
    held = [min(width, -(-max(c, 0) // block)) for c in ctx]
    total = sum(held) + n_free + 3
    ids = torch.randperm(total, generator=g).tolist()
    table, k = [], 0
    for h in held:
        row = ids[k:k + h]
        k += h
        table.append((row + [-7] * width)[:width])
    free = ids[k:k + (n_free if cap is None else cap)]
    return table, free, sum(max(x, 0) for x in new) + pad


def _check_plan(ctx, new, block, width, n_free, pad=0, seed=0, cap=None, n_tok=None):
    from yllm_amd.paged import paged_plan

    table, free, T = _plan_case(ctx, new, block, width, n_free, pad, seed, cap)
    T = T if n_tok is None else n_tok
    dev = _i32(table) if table else torch.zeros((0, width), dtype=torch.int32, device="cuda")
    step = paged_plan(dev, _i32(ctx), _i32(new), _i32(free), _i32([n_free]), block, T)
    want = plan_oracle(table, ctx, new, free, n_free, block, T)
    got = [t.tolist() for t in (step.cu_new, step.kv_lens, step.slots, step.positions, step.counts)]
    for name, a, b in zip(("cu_new", "kv_lens", "slots", "positions", "counts"), got, want):
        assert a == b, name
    assert dev.tolist() == table
    return step


@pytest.mark.parametrize("block", [64, 256])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 256, 257, 700])
def test_plan(cuda, n, block):
    g = torch.Generator().manual_seed(n * 7 + block)
    ctx = torch.randint(0, 3 * block, (n,), generator=g).tolist()
    new = [(1, 0, 1, block, 5, 2 * block + 1)[int(x)] for x in torch.randint(0, 6, (n,), generator=g)]
    _check_plan(ctx, new, block, 8, 4 * n + 3, pad=5, seed=n)


def test_plan_block_edges(cuda):
    """New tokens that begin or end exactly at, one before and one behind a block's border."""
    ctx = [0, 63, 64, 65, 127, 128, 0, 0, 0, 64, 1]
    new = [0, 1, 1, 1, 2, 0, 64, 65, 63, 128, 191]
    _check_plan(ctx, new, 64, 5, 30)


def test_plan_runs_out_of_blocks(cuda):
    """Sequences are served in order while their blocks last; one that needs none is served all the same."""
    _check_plan([64, 10, 128, 64, 0, 70], [64, 3, 100, 1, 65, 2], 64, 6, 3)
    _check_plan([0, 0], [1, 1], 64, 6, 0)
    _check_plan([0, 5], [1, 1], 64, 6, -4, cap=2)


def test_plan_narrow_table_bad_lengths_and_few_rows(cuda):
    _check_plan([100, 128, 0], [29, 1, 3], 64, 2, 9)           # 129 positions pass a row of two blocks
    _check_plan([-1, 5, 3, 0], [4, -2, 2, 1], 64, 2, 9)        # negative lengths
    _check_plan([0, 0, 0], [5, 6, 7], 64, 2, 9, n_tok=11)      # the third one's rows pass n_tok
    _check_plan([0, 0, 0], [5, 6, 7], 64, 2, 9, n_tok=8)
    _check_plan([7, 9], [0, 0], 64, 2, 9, n_tok=0)
    _check_plan([0x7fffffff, 3], [0x7fffffff, 2], 64, 2, 9, n_tok=4)
    _check_plan([], [], 64, 2, 2, n_tok=3)


@pytest.mark.parametrize("width", [2, 3, 5])
@pytest.mark.parametrize("n_free", [0, 5, 40, 90])
def test_plan_hands_out_no_block_twice(cuda, width, n_free):
    """What is left on the free list is no one's, whichever sequences were refused: a step's blocks are its last."""
    g = torch.Generator().manual_seed(width * 100 + n_free)
    n = 70
    ctx = [int(x) for x in torch.randint(-20, 200, (n,), generator=g)]
    new = [int(x) for x in torch.randint(-2, 260, (n,), generator=g)]
    ctx = [min(c, width * 64) for c in ctx]
    table, free, T = _plan_case(ctx, new, 64, width, n_free, seed=n_free)
    for n_tok in (T, T // 2):
        from yllm_amd.paged import paged_plan

        dev = _i32(table)
        step = paged_plan(dev, _i32(ctx), _i32(new), _i32(free), _i32([n_free]), 64, n_tok)
        left = set(free[:int(step.counts[0])])
        held = [e for r, L in zip(dev.tolist(), step.kv_lens.tolist()) for e in r[:-(-L // 64)]]
        assert len(held) == len(set(held)) and not left & set(held)
        new_ones = sum(a != b for r, s in zip(dev.tolist(), table) for a, b in zip(r, s))
        assert len(left) + new_ones == n_free


def test_plan_many_sequences(cuda):
    g = torch.Generator().manual_seed(3)
    n = 8192
    ctx = torch.randint(0, 300, (n,), generator=g).tolist()
    new = torch.randint(0, 3, (n,), generator=g).tolist()
    _check_plan(ctx, new, 64, 6, 3000, pad=1)


def test_plan_table_rows_of_a_wider_table_and_reused_outputs(cuda):
    from yllm_amd.paged import paged_plan

    wide = torch.full((3, 12), -7, dtype=torch.int32, device="cuda")
    free, nf = _i32(list(range(20, 60))), _i32([40])
    ctx, new = _i32([0, 0, 0]), _i32([70, 1, 130])
    step = paged_plan(wide[:, 2:6], ctx, new, free, nf, 64, 201)
    table = [[-7] * 4 for _ in range(3)]
    want = plan_oracle(table, [0, 0, 0], [70, 1, 130], list(range(20, 60)), 40, 64, 201)
    assert step.slots.tolist() == want[2] and wide[:, 2:6].tolist() == table
    assert (wide[:, :2] == -7).all() and (wide[:, 6:] == -7).all()
    nf = step.counts[:1].clone()
    again = paged_plan(wide[:, 2:6], step.kv_lens.clone(), _i32([58, 67, 0]), free, nf, 64, 201, out=step)
    want = plan_oracle(table, [70, 1, 130], [58, 67, 0], list(range(20, 60)), want[4][0], 64, 201)
    assert again is step and step.slots.tolist() == want[2] and step.counts.tolist() == want[4]
    assert wide[:, 2:6].tolist() == table


# ---- qk_norm_rope_kv_store -------------------------------------------------------------------------

KINDS = {"none": 0, "pairs": 1, "half": 2, "mrope": 3}


def rope_oracle(x, pos, w, eps, kind, n_rot, theta):
    """x [T, H, d] in 64 bits: norm and rotation, and a bound of the fp32 arithmetic's error."""
    d = x.shape[-1]
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    y, size = x.clone(), x.abs()
    if kind != "none":
        span = n_rot if kind == "mrope" else d
        ang = pos.double()[:, None, None] * theta ** (-2.0 * torch.arange(span // 2, dtype=torch.float64, device=x.device) / span)
        i = torch.arange(span // 2, device=x.device)
        a, b = (2 * i, 2 * i + 1) if kind == "pairs" else (i, i + span // 2)
        cs, sn = ang.cos(), ang.sin()
        y[..., a], y[..., b] = x[..., a] * cs - x[..., b] * sn, x[..., a] * sn + x[..., b] * cs
        both = x[..., a].abs() + x[..., b].abs()
        size[..., a], size[..., b] = both, both
    # the sum of squares (at most d roundings of positive terms, halved by the root), root, two products; the angle
    # (rounded once, below half a turn: 2^-25 * 2 pi), sine and cosine (4 ulp), two products and a sum
    return y, size * 2.0 ** -24 * (d / 2 + 16)


def _slots(T, block, n_blocks, seed, start=5):
    """Runs of rows in different pages: a run starts and ends anywhere in a page."""
    g = torch.Generator().manual_seed(seed)
    pages = torch.randperm(n_blocks, generator=g).tolist()
    slots, off, k = [], start % block, 0
    for r in range(T):
        slots.append(pages[k] * block + off)
        off += 1
        if off == block or (r % 37 == 36):
            off, k = (0 if off == block else (off * 7) % block), k + 1
    return slots


def _check_rope(T, nh, nkv, d, kind, dtype, out_dtype, norm=True, block=64, n_rot=0, wide=0, skip=(), seed=0,
                norm_dtype=F32, far=0, theta=1e6, in_place=False, with_q=True):
    from yllm_amd.paged import PagedKV, qk_norm_rope_kv_store

    g = _gen(seed + T)
    width = (nh + 2 * nkv) * d
    rows = (torch.randn(T, width + wide, generator=g, device="cuda") * 1.5).to(dtype)
    x = rows[:, :width]
    q, k, v = x[:, :nh * d], x[:, nh * d:(nh + nkv) * d], x[:, (nh + nkv) * d:]
    n_blocks = T // 37 + T // block + 3
    cache = PagedKV.empty(n_blocks, nkv, d, block, zero=False)
    cache.k.fill_(-3.0)
    cache.v.fill_(-3.0)
    slots = _slots(T, block, n_blocks, seed)
    for i, s in skip:
        slots[i] = s
    pos = (torch.arange(T) * 3 + far).tolist()
    qw = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(norm_dtype) if norm else None
    kw = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(norm_dtype) if norm else None
    given = rows.clone()
    q_out = None
    if with_q:
        q_out = q if in_place else torch.full((T, nh * d), 9.0, dtype=out_dtype, device="cuda")
    got = qk_norm_rope_kv_store(cache, q if with_q else None, k, v, nh, KINDS[kind], theta, n_rot,
                                positions=_i32(pos), slots=_i32(slots), q_norm=qw, k_norm=kw, eps=1e-5, q_out=q_out)
    x = given[:, :width].double().view(T, nh + 2 * nkv, d)
    ok = [i for i, s in enumerate(slots) if 0 <= s < n_blocks * block]
    p = _i32(pos)
    wq, wk = (None, None) if not norm else (qw.double(), kw.double())
    if with_q:
        want, tol = rope_oracle(x[:, :nh], p, wq, 1e-5, kind, n_rot, theta)
        err = (got.double().view(T, nh, d)[ok] - want[ok]).abs()
        # (a subnormal f16 result is off by half of 2^-24)
        assert (err <= tol[ok] + U[out_dtype] * want[ok].abs() + 2.0 ** -25).all(), float(err.max())
        rest = [i for i in range(T) if i not in set(ok)]
        if rest:
            before = given[:, :nh * d].to(out_dtype) if in_place else torch.full_like(got, 9.0)
            assert torch.equal(got[rest], before[rest])
    else:
        assert got is None
    if not in_place:
        assert torch.equal(rows, given)
    want, tol = rope_oracle(x[:, nh:nh + nkv], p, wk, 1e-5, kind, n_rot, theta)
    K = torch.full((n_blocks * block, nkv, d), -3.0, dtype=torch.float64, device="cuda")
    V, KT = K.clone(), torch.zeros_like(K)
    at = torch.tensor([slots[i] for i in ok], device="cuda")
    if ok:
        K[at], V[at], KT[at] = want[ok], x[ok][:, nh + nkv:], tol[ok] + U[F16] * want[ok].abs() + 2.0 ** -25
    gk = cache.k.double().transpose(1, 2).reshape(-1, nkv, d)
    gv = cache.v.double().permute(0, 2, 4, 1, 3).reshape(-1, nkv, d)
    assert ((gk - K).abs() <= KT).all(), float((gk - K).abs().max())
    assert ((gv - V).abs() <= U[F16] * V.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (16, 2, 256), (5, 5, 64), (3, 2, 128)])
@pytest.mark.parametrize("T", [1, 7, 129])
def test_qk_norm_rope(cuda, kind, nh, nkv, d, T):
    dt, out = [(F32, F32), (BF16, F16), (F16, BF16)][(T + nh) % 3]
    _check_rope(T, nh, nkv, d, kind, dt, out, n_rot=64 if kind == "mrope" else 0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("out", [F32, F16, BF16])
def test_qk_norm_rope_types(cuda, dtype, out):
    _check_rope(200, 8, 2, 128, "half", dtype, out, wide=24)
    _check_rope(30, 8, 2, 128, "pairs", dtype, out, wide=4, norm=False)


@pytest.mark.parametrize("T", [64, 127, 128, 130, 191, 200, 519])
def test_qk_norm_rope_row_counts(cuda, T):
    """Both forms of the V store, groups of eight that begin and end in any window."""
    _check_rope(T, 4, 2, 64, "half", F32, F16, seed=T)
    _check_rope(T, 2, 1, 256, "mrope", BF16, BF16, block=128, n_rot=64, seed=T + 1)


@pytest.mark.parametrize("n_rot", [8, 24, 64, 128])
def test_qk_norm_rope_partial_rotation(cuda, n_rot):
    _check_rope(40, 4, 2, 128, "mrope", F32, F32, n_rot=n_rot)


def test_qk_norm_rope_far_positions(cuda):
    _check_rope(140, 4, 2, 128, "pairs", F32, F32, far=131071 * 8)
    _check_rope(9, 4, 2, 64, "half", F32, F32, far=(1 << 31) - 100, theta=1e4)


def test_qk_norm_rope_rows_without_a_slot(cuda):
    big = 0x7fffffff
    for T in (12, 200):
        _check_rope(T, 4, 2, 128, "half", BF16, BF16, skip=[(0, -1), (3, -5), (T - 1, big), (T - 2, -big)])
        _check_rope(T, 4, 2, 128, "half", F32, F32, skip=[(i, -1) for i in range(T)])


def test_qk_norm_rope_in_place_f16_weights_and_keys_only(cuda):
    _check_rope(150, 6, 2, 128, "half", F32, F32, in_place=True, norm_dtype=F16)
    _check_rope(3, 6, 2, 128, "pairs", BF16, BF16, in_place=True)
    _check_rope(150, 6, 2, 128, "half", F16, F16, with_q=False)


def test_qk_norm_rope_into_a_contiguous_cache(cuda):
    """A LayerKV is a pool of one page; without a norm the stored bits are those of rope_kv_store but for its fp32
    angles, so at positions where both angles are exact (position 0, and no rotation) they are equal."""
    from yllm_amd.attention import ROPE_HALF, ROPE_NONE, LayerKV, rope_kv_store
    from yllm_amd.paged import qk_norm_rope_kv_store

    nh, nkv, d, T, cap = 8, 2, 128, 150, 320
    g = _gen(5)
    x = torch.randn(T, (nh + 2 * nkv) * d, generator=g, device="cuda")
    q, k, v = x[:, :nh * d], x[:, nh * d:(nh + nkv) * d], x[:, (nh + nkv) * d:]
    for rope, n, start in ((ROPE_NONE, T, 33), (ROPE_HALF, 1, 0)):
        a, b = LayerKV.empty(nkv, d, cap), LayerKV.empty(nkv, d, cap)
        qa = rope_kv_store(a, q[:n], k[:n], v[:n], start, nh, rope, 1e6)
        qb = qk_norm_rope_kv_store(b, q[:n], k[:n], v[:n], nh, rope, 1e6, pos_start=start)
        assert torch.equal(qa, qb) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


@pytest.mark.parametrize("T", [4, 160])
def test_qk_norm_rope_stores_the_bits_that_kv_store_stores(cuda, T):
    """Ties, f16 subnormals, results at the ends of the range, inf and NaN, of every type that can hold them."""
    from yllm_amd.attention import ROPE_NONE, LayerKV, kv_store
    from yllm_amd.paged import qk_norm_rope_kv_store

    g = _gen(3)
    e = torch.randint(-30, 18, (T, 2 * 64), generator=g, device="cuda").float()
    m = 1.0 + torch.randint(0, 2048, e.shape, generator=g, device="cuda") / 2048.0  # ties at 11 bits
    x = m * torch.exp2(e) * torch.where(torch.rand(e.shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    x[:, ::5] = torch.nextafter(x[:, ::5], torch.zeros_like(x[:, ::5]))
    x[:, 1::7] = torch.nextafter(x[:, 1::7], torch.full_like(x[:, 1::7], math.inf))
    special = [0.0, -0.0, math.inf, -math.inf, math.nan, 65504.0, 65519.99, 65520.0, -65520.0, 65536.0, 3e38, 1e-45, -1e-40,
               2.0 ** -14, 2.0 ** -14 - 2.0 ** -38, 2.0 ** -14 - 2.0 ** -25, 2.0 ** -24, 2.0 ** -25, 2.0 ** -25 - 2.0 ** -49,
               3 * 2.0 ** -25, 1.5 * 2.0 ** -15]
    x[0, :len(special)] = torch.tensor(special, device="cuda")
    for dtype in (F32, BF16, F16):
        y = x.to(dtype)
        a, b = LayerKV.empty(2, 64, 192), LayerKV.empty(2, 64, 192)
        kv_store(a, y, y.flip(0).contiguous(), 3)
        qk_norm_rope_kv_store(b, None, y, y.flip(0).contiguous(), 2, ROPE_NONE, 1.0, pos_start=3)
        for s, t in ((a.k, b.k), (a.v, b.v)):
            nan = s.isnan()
            assert torch.equal(nan, t.isnan())
            s, t = s.view(torch.int16).masked_fill(nan, 0), t.view(torch.int16).masked_fill(nan, 0)
            assert torch.equal(s, t), (dtype, int((s != t).sum()))


# ---- paged_attn --------------------------------------------------------------------------------------

class Batch:
    """Sequences (length, new tokens) over a pool whose unused positions hold NaN."""

    def __init__(self, seqs, nh, nkv, d, block=64, dtype=F16, seed=0, behind=0, gated=False, qscale=1.0, more=2):
        from yllm_amd.paged import PagedKV

        g = _gen(seed + 11)
        self.seqs, self.nh, self.nkv, self.d, self.block, self.dtype = seqs, nh, nkv, d, block, dtype
        blocks = [-(-max(L, 0) // block) for L, _ in seqs]
        nb = sum(blocks) + more
        self.cache = PagedKV.empty(nb, nkv, d, block, zero=False)
        self.cache.k.fill_(math.nan)
        self.cache.v.fill_(math.nan)
        order = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).tolist()
        width = max(blocks + [1]) + 1
        self.table = torch.full((len(seqs), width), -1, dtype=torch.int32)
        self.K, self.V = [], []
        at = 0
        for i, (L, _) in enumerate(seqs):
            L = max(L, 0)
            K = torch.randn(nkv, L, d, generator=g, device="cuda").half()
            V = torch.randn(nkv, L, d, generator=g, device="cuda").half()
            for j in range(blocks[i]):
                page, n = order[at], min(block, L - j * block)
                at += 1
                self.table[i, j] = page
                self.cache.k[page, :, :n] = K[:, j * block:j * block + n]
                vt = self.cache.v[page].permute(0, 1, 3, 2).reshape(nkv, block, d)
                vt[:, :n] = V[:, j * block:j * block + n]
                self.cache.v[page] = vt.view(nkv, block // 32, 32, d).permute(0, 1, 3, 2)
            self.K.append(K)
            self.V.append(V)
        self.table = self.table.cuda()
        new = [n for _, n in seqs]
        self.cu = [sum(new[:i]) for i in range(len(new) + 1)]
        self.T = self.cu[-1] + behind
        self.q = (torch.randn(self.T, nh * d, generator=g, device="cuda") * qscale).to(dtype)
        self.gate = torch.randn(self.T, nh * d, generator=g, device="cuda") * 3 if gated else None
        self.max_new, self.max_len = max(new + [1]), max([L for L, _ in seqs] + [1])

    def run(self, **kw):
        from yllm_amd.paged import paged_attn

        kw = {"max_new": self.max_new, "max_len": self.max_len, "gate": self.gate, **kw}
        mn, ml = kw.pop("max_new"), kw.pop("max_len")
        return paged_attn(self.q, self.cache, self.table, _i32([max(L, 0) for L, _ in self.seqs]), _i32(self.cu),
                          self.nh, mn, ml, **kw)

    def exact(self):
        """(output, error bound before the output's own rounding) in 64 bits."""
        d, out = self.d, torch.zeros(self.T, self.nh, self.d, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)
        u_p = 2.0 ** -22 if self.dtype == F32 else 2.0 ** -11  # rounding of a probability
        for i, (L, n) in enumerate(self.seqs):
            L = max(L, 0)
            if L == 0 or n == 0:
                continue
            q = self.q[self.cu[i]:self.cu[i] + n].double().view(n, self.nh, d)
            pos = torch.arange(L - n, L, device="cuda")
            hide = torch.arange(L, device="cuda")[None, :] > pos[:, None]
            for h in range(self.nh):
                K, V = self.K[i][h * self.nkv // self.nh].double(), self.V[i][h * self.nkv // self.nh].double()
                s = (q[:, h] @ K.t() / math.sqrt(d)).masked_fill(hide, -math.inf)
                top = s.amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(top.isinf(), 0.0, top)).masked_fill(hide, 0.0)
                z = p.sum(-1, keepdim=True)
                p = p / torch.where(z == 0, 1.0, z)
                # the fp32 sum of a score's d products, twice (numerator and denominator), exp and sums
                e = 2 * d * 2.0 ** -24 * (q[:, h].abs() @ K.abs().t() / math.sqrt(d)).amax(-1, keepdim=True)
                e = e + u_p + 2.0 ** -20
                w = torch.where(p > 0, p, 0.0)
                seen = V.masked_fill(~torch.isfinite(V), 0.0)
                out[self.cu[i]:self.cu[i] + n, h] = w @ seen
                tol[self.cu[i]:self.cu[i] + n, h] = (w @ seen.abs()) * e
        out, tol = out.view(self.T, -1), tol.view(self.T, -1)
        if self.gate is not None:
            s = self.gate.double().sigmoid()
            out, tol = out * s, tol * s + out.abs() * s * 2.0 ** -20
        return out, tol

    def check(self, **kw):
        got = self.run(**kw)
        want, tol = self.exact()
        n = self.cu[-1]
        err = (got.double() - want).abs()[:n]
        # (2^-24: half a step of a subnormal f16)
        ok = err <= tol[:n] + U[got.dtype] * want[:n].abs() + 2.0 ** -24
        assert ok.all(), (float(err.max()), torch.nonzero(~ok)[:4].tolist(), int((~ok).sum()))
        return got


HEADS = [(14, 2, 64), (28, 4, 128), (32, 8, 128), (16, 2, 256), (3, 2, 64), (4, 4, 128), (16, 1, 128)]


@pytest.mark.parametrize("nh,nkv,d", HEADS)
@pytest.mark.parametrize("L", [1, 2, 31, 64, 65, 511, 1500])
def test_attn_one_token(cuda, nh, nkv, d, L):
    Batch([(L, 1)], nh, nkv, d, dtype=(F16, BF16, F32)[L % 3], seed=L).check()


@pytest.mark.parametrize("nh,nkv,d", HEADS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_attn_decode_batch(cuda, nh, nkv, d, dtype):
    seqs = [(1, 1), (700, 1), (64, 1), (0, 1), (129, 1), (2000, 1), (63, 1), (333, 1)]
    Batch(seqs, nh, nkv, d, dtype=dtype, block=128, seed=2).check()


@pytest.mark.parametrize("nh,nkv,d", HEADS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_attn_mixed_batch(cuda, nh, nkv, d, dtype):
    """Decode tokens, drafts, chunks, a whole prompt, a sequence without keys or without new tokens."""
    seqs = [(300, 1), (200, 200), (77, 3), (0, 0), (900, 130), (50, 0), (0, 2), (513, 64), (65, 17), (128, 128)]
    Batch(seqs, nh, nkv, d, dtype=dtype, seed=3, gated=d == 256, behind=3).check()


@pytest.mark.parametrize("new", [1, 2, 5, 16, 31, 33, 63, 64, 65, 127, 128, 129, 200, 257, 515])
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (16, 2, 256)])
def test_attn_chunk_lengths(cuda, nh, nkv, d, new):
    for k, ctx in enumerate((0, 1, 100, 704)):
        Batch([(ctx + new, new)], nh, nkv, d, dtype=(F16, BF16, F32)[(new + k) % 3], block=(64, 256)[k % 2],
              seed=new).check()


@pytest.mark.parametrize("block", [64, 128, 256, 1024])
def test_attn_blocks(cuda, block):
    Batch([(1000, 300), (70, 1), (513, 9)], 8, 2, 128, block=block, seed=block).check()


def test_attn_more_tokens_than_positions(cuda):
    """Tokens at negative positions see nothing: zero rows."""
    b = Batch([(3, 7), (0, 5), (1, 140), (130, 200)], 8, 2, 128, seed=1)
    out = b.check()
    assert (out[:4] == 0).all() and (out[7:12] == 0).all() and (out[12:12 + 139] == 0).all()


@pytest.mark.parametrize("out_dtype", [F16, BF16, F32])
def test_attn_output_types_strides_and_rows_behind(cuda, out_dtype):
    b = Batch([(100, 3), (333, 90), (64, 1)], 8, 2, 128, seed=4, behind=6, gated=True)
    width = 8 * 128
    wide = torch.full((b.T, width + 24), 7.0, dtype=out_dtype, device="cuda")
    qw = torch.zeros((b.T, width + 8), dtype=b.dtype, device="cuda")
    gw = torch.zeros((b.T, width + 5), device="cuda")
    qw[:, 8:], gw[:, 3:3 + width] = b.q, b.gate
    b.q, b.gate = qw[:, 8:], gw[:, 3:3 + width]
    got = b.check(out=wide[:, 16:16 + width])
    assert (wide[:, :16] == 7).all() and (wide[:, 16 + width:] == 7).all() and (got[b.cu[-1]:] == 7).all()


@pytest.mark.parametrize("seqs", [[(200, 1)] * 3, [(200, 5), (90, 1)], [(400, 150), (64, 64)]])
def test_attn_table_entries_outside_the_pool(cuda, seqs):
    """They read as zeros: keys that score 0 with a value of 0."""
    for block, nkv, d in ((64, 2, 128), (128, 2, 256), (256, 4, 64)):
        b = Batch(seqs, 8, nkv, d, block=block, seed=9)
        b.table[0, 0], b.table[1, 0] = 1 << 30, -9
        for i in (0, 1):
            b.K[i][:, :block], b.V[i][:, :block] = 0, 0
        b.check()


@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("L,new", [(70, 1), (70, 6), (400, 40), (400, 300), (64, 64)])
def test_attn_values_that_a_query_does_not_see(cuda, nh, nkv, d, dtype, L, new):
    """inf and NaN in the keys and values of the last token reach the rows of that token and no other."""
    b = Batch([(L, new), (129, 2)], nh, nkv, d, dtype=dtype, seed=5)
    page, off = int(b.table[0, (L - 1) // 64]), (L - 1) % 64
    bad = torch.tensor([math.inf, -math.inf, math.nan, 1.0], device="cuda").half().repeat(d // 4)
    b.cache.v[page, :, off // 32, :, off % 32] = bad
    b.V[0][:, L - 1] = 0  # what rows that do not see it are held to
    got = b.run()
    want, tol = b.exact()
    rows = [r for r in range(b.T) if r != new - 1]
    err = (got.double() - want).abs()[rows]
    assert (err <= tol[rows] + U[got.dtype] * want[rows].abs() + 2.0 ** -24).all(), float(err.nan_to_num(9.0).max())
    last = got[new - 1].view(nh, d).float()
    assert (last[:, 0::4] == math.inf).all() and (last[:, 1::4] == -math.inf).all() and last[:, 2::4].isnan().all()
    assert last[:, 3::4].isfinite().all()
    # a key of NaN: every score of the last row, no other row's
    b.cache.k[page, :, off] = math.nan
    got = b.run()
    err = (got.double() - want).abs()[rows]
    assert (err <= tol[rows] + U[got.dtype] * want[rows].abs() + 2.0 ** -24).all()
    assert got[new - 1].isnan().all()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attn_large_scores(cuda, dtype):
    """Softmax maxima far apart from tile to tile, up and down."""
    b = Batch([(1000, 1), (600, 70), (900, 4)], 8, 2, 128, dtype=dtype, seed=6, qscale=6.0)
    b.check()


def test_attn_long_context(cuda):
    """Many splits of one sequence, and pages past 32 bits of byte offset from the first one."""
    b = Batch([(40000, 1), (17, 1)], 32, 8, 128, dtype=BF16, block=256, seed=7)
    b.check()
    b = Batch([(9000, 1), (9100, 33)], 16, 2, 256, dtype=F16, block=64, seed=8)
    b.check()


def test_attn_pool_past_4_gib(cuda):
    from yllm_amd.paged import PagedKV

    nkv, d, block = 8, 128, 1024
    nb = (5 << 30) // (nkv * d * block * 2)  # 5 GiB of K
    b = Batch([(2000, 1), (1500, 140)], 32, nkv, d, block=block, seed=10)
    big = PagedKV(torch.empty((nb, nkv, block, d), dtype=F16, device="cuda"),
                  torch.empty((nb, nkv, block // 32, d, 32), dtype=F16, device="cuda"))
    for i in range(2):
        for j in range(2):
            old, page = int(b.table[i, j]), nb - 1 - 2 * j - i
            big.k[page], big.v[page] = b.cache.k[old], b.cache.v[old]
            b.table[i, j] = page
    b.cache = big
    b.check()


def test_attn_many_sequences(cuda):
    """More sequences than threads of a workgroup."""
    g = torch.Generator().manual_seed(1)
    seqs = [(int(L), 1) for L in torch.randint(0, 90, (1100,), generator=g)]
    Batch(seqs, 4, 2, 64, seed=12).check()
    seqs = [(L, min(L, 1 + i % 3)) for i, (L, _) in enumerate(seqs)]
    Batch(seqs, 4, 2, 64, seed=13).check()


def test_attn_loose_bounds_and_a_larger_workspace(cuda):
    """Bounds larger than the batch give the same rows; so does a workspace for more."""
    from yllm_amd.paged import paged_attn_workspace

    for seqs in ([(300, 1), (2000, 1)], [(300, 20), (2000, 190), (70, 1)]):
        b = Batch(seqs, 28, 4, 128, seed=14)
        ws = paged_attn_workspace(4096, 64, 512, 32768, 28, 4, 128)
        b.check(max_len=None)
        b.check(workspace=ws)
        b.check(max_new=b.T, workspace=torch.empty(256, dtype=torch.uint8, device="cuda"))


def test_attn_same_result_twice(cuda):
    """No order of arrival in the sums: the same bits every time."""
    b = Batch([(3000, 1), (700, 200), (5000, 7)], 28, 4, 128, seed=15)
    first = b.run()
    for _ in range(3):
        assert torch.equal(b.run(), first)
    b = Batch([(30000, 1), (700, 1)], 28, 4, 128, seed=16)
    first = b.run()
    for _ in range(3):
        assert torch.equal(b.run(), first)


def test_attn_on_another_stream(cuda):
    b = Batch([(3000, 1), (700, 200)], 28, 4, 128, seed=17)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        b.check()
    torch.cuda.current_stream().wait_stream(st)


def test_attn_more_new_tokens_than_the_bound(cuda):
    """A sequence with more than max_new new tokens: the first max_new rows are computed, the rest left as they were."""
    for seqs, cut in (([(90, 5), (200, 2)], 2), ([(300, 200), (64, 3)], 150), ([(300, 200), (64, 3)], 60)):
        b = Batch(seqs, 8, 2, 128, seed=21)
        whole, out = b.check(), torch.full((b.T, 8 * 128), 5.0, dtype=F16, device="cuda")
        b.run(max_new=cut, out=out)
        want, tol = b.exact()
        for i, (_, n) in enumerate(seqs):
            at = slice(b.cu[i], b.cu[i] + min(n, cut))
            assert ((out[at].double() - want[at]).abs() <= tol[at] + U[F16] * want[at].abs() + 2.0 ** -24).all()
            assert (out[b.cu[i] + min(n, cut):b.cu[i + 1]] == 5).all()
        assert torch.equal(b.run(), whole)


def test_attn_captured_chunks_replay_with_new_lengths(cuda):
    """A captured call with prompt chunks follows the lengths, offsets and tables that it finds when it runs."""
    from yllm_amd.paged import paged_attn, paged_attn_workspace

    steps = [Batch(s, 28, 4, 128, seed=30 + i) for i, s in enumerate(
        ([(700, 200), (90, 1), (3000, 33)], [(1, 1), (0, 0), (233, 233)], [(5000, 1), (64, 64), (129, 128)],
         [(2, 2), (1, 1), (1, 1)], [(400, 100), (2000, 130), (77, 4)]))]
    T, w, nb = max(b.T for b in steps), max(b.table.shape[1] for b in steps), max(b.cache.n_blocks for b in steps)
    k, v = (torch.zeros((nb, *x.shape[1:]), dtype=F16, device="cuda") for x in (steps[0].cache.k, steps[0].cache.v))
    pool = type(steps[0].cache)(k, v)
    q, out = torch.zeros((T, 28 * 128), dtype=F16, device="cuda"), torch.empty((T, 28 * 128), dtype=F16, device="cuda")
    table, lens, cu = torch.zeros((3, w), dtype=torch.int32, device="cuda"), _i32([1, 1, 1]), _i32([0, 1, 2, 3])
    ws = paged_attn_workspace(T, 3, 233, 5000, 28, 4, 128)
    paged_attn(q, pool, table, lens, cu, 28, 233, 5000, out=out, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_attn(q, pool, table, lens, cu, 28, 233, 5000, out=out, workspace=ws)
    for b in steps * 2:
        q[:b.T], out[:] = b.q, 5.0
        pool.k[:b.cache.n_blocks], pool.v[:b.cache.n_blocks] = b.cache.k, b.cache.v
        table[:, :b.table.shape[1]] = b.table
        lens.copy_(_i32([L for L, _ in b.seqs])), cu.copy_(_i32(b.cu))
        graph.replay()
        want, tol = b.exact()
        err = (out[:b.T].double() - want).abs()
        assert (err <= tol + U[F16] * want.abs() + 2.0 ** -24).all() and (out[b.T:] == 5).all()


@pytest.mark.parametrize("nh,nkv,d", [(3, 2, 64), (28, 4, 128), (5, 3, 128), (16, 2, 256)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("L,new", [(0, 0), (50, 10), (300, 1), (130, 130), (129, 129), (700, 127), (640, 200), (90, 150)])
def test_attn_one_sequence_below_its_bounds(cuda, nh, nkv, d, dtype, L, new):
    """A launch sized for 200 tokens and 700 keys, as a captured one is, with fewer of either."""
    b = Batch([(L, new)], nh, nkv, d, dtype=dtype, seed=60, behind=200 - new)
    out = torch.full((200, nh * d), 5.0, dtype=dtype, device="cuda")
    if b.table.shape[1] * 64 < 700:
        b.table = torch.cat([b.table, torch.full((1, 11 - b.table.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    b.check(max_new=200, max_len=700, out=out)
    assert (out[new:] == 5).all()


def test_attn_calls_on_two_streams_at_once(cuda):
    """Each with its own workspace."""
    from yllm_amd.paged import paged_attn_workspace

    batches = [Batch([(3000, 1), (700, 200)], 28, 4, 128, seed=40), Batch([(9000, 1), (50, 1)], 16, 2, 256, seed=41)]
    want = [b.check() for b in batches]
    spaces = [paged_attn_workspace(b.T, 2, b.max_new, b.max_len, b.nh, b.nkv, b.d) for b in batches]
    streams, got = [torch.cuda.Stream() for _ in batches], [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for st, b, ws, o in zip(streams, batches, spaces, got):
            with torch.cuda.stream(st):
                o.append(b.run(workspace=ws))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w) for o in outs)


def test_store_into_a_pool_past_4_gib(cuda):
    from yllm_amd.attention import ROPE_NONE
    from yllm_amd.paged import PagedKV, qk_norm_rope_kv_store

    nkv, d, block = 8, 128, 256
    nb = (5 << 30) // (nkv * d * block * 2)  # 5 GiB of K
    big = PagedKV(torch.empty((nb, nkv, block, d), dtype=F16, device="cuda"),
                  torch.empty((nb, nkv, block // 32, d, 32), dtype=F16, device="cuda"))
    for T in (3, 200):  # single rows, and groups of rows
        first = (nb - 2) * block + 17
        big.k[-2:], big.v[-2:] = 3.0, 3.0
        kv = torch.randn((2, T, nkv * d), generator=_gen(T), device="cuda").half()
        qk_norm_rope_kv_store(big, None, kv[0], kv[1], nkv, ROPE_NONE, 1.0, positions=_i32(list(range(T))),
                              slots=_i32(list(range(first, first + T))))
        K = big.k[-2:].transpose(1, 2).reshape(-1, nkv * d)
        V = big.v[-2:].permute(0, 2, 4, 1, 3).reshape(-1, nkv * d)
        for got, want in ((K, kv[0]), (V, kv[1])):
            assert torch.equal(got[17:17 + T], want) and (got[:17] == 3).all() and (got[17 + T:] == 3).all()


def test_calls_without_rows_and_single_rows_of_odd_strides(cuda):
    from yllm_amd.paged import paged_attn, qk_norm_rope_kv_store

    b = Batch([(70, 1)], 8, 2, 128, seed=50)
    none = torch.empty((0, 256), dtype=F16, device="cuda")
    empty = _i32([])
    assert qk_norm_rope_kv_store(b.cache, torch.empty((0, 1024), dtype=F16, device="cuda"), none, none, 8, 2, 1e6,
                                 positions=empty, slots=empty).shape == (0, 1024)
    q = torch.empty((0, 1024), dtype=F16, device="cuda")
    assert paged_attn(q, b.cache, b.table, _i32([70]), _i32([0, 0]), 8, 1, 70).shape == (0, 1024)
    assert paged_attn(q, b.cache, b.table[:0], empty, _i32([0]), 8, 1, 70).shape == (0, 1024)
    wide = torch.zeros((1, 1024 + 13), dtype=F16, device="cuda")  # the next row would not be aligned
    wide[:, :1024] = b.q
    want = b.check()
    b.q = wide[:, :1024]
    assert torch.equal(b.run(), want)


# ---- a step, and steps in a row ------------------------------------------------------------------------

class Serve:
    """Two layers of paged serving, step by step, and the same in 64 bits from the rows themselves."""

    def __init__(self, n_seq, nh, nkv, d, block, kind, dtype, n_blocks, width, seed=0):
        from yllm_amd.paged import PagedKV

        self.__dict__.update(nh=nh, nkv=nkv, d=d, block=block, kind=kind, dtype=dtype, n=n_seq)
        self.layers = [PagedKV.empty(n_blocks, nkv, d, block) for _ in range(2)]
        g = self.g = _gen(seed)
        self.w = [(1 + 0.1 * torch.randn(d, generator=g, device="cuda"), 1 + 0.1 * torch.randn(d, generator=g, device="cuda"))
                  for _ in range(2)]
        self.table = torch.full((n_seq, width), -1, dtype=torch.int32, device="cuda")
        self.ctx = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        self.free, self.n_free = torch.arange(n_blocks, dtype=torch.int32, device="cuda").flip(0).contiguous(), _i32([n_blocks])
        self.hist = [[[] for _ in range(n_seq)] for _ in range(2)]  # rows of k | v after norm and rotation

    def rows(self, T):
        return [torch.randn(T, (self.nh + 2 * self.nkv) * self.d, generator=self.g, device="cuda").to(self.dtype) for _ in range(2)]

    def step(self, new, rows, n_tok, max_new, max_len):
        from yllm_amd import paged as P

        p = P.paged_plan(self.table, self.ctx, new, self.free, self.n_free, self.block, n_tok)
        out, qd, kd = [], self.nh * self.d, self.nkv * self.d
        for layer, x, (wq, wk) in zip(self.layers, rows, self.w):
            q = torch.zeros(n_tok, qd, dtype=self.dtype, device="cuda")
            P.qk_norm_rope_kv_store(layer, x[:, :qd], x[:, qd:qd + kd], x[:, qd + kd:], self.nh, KINDS[self.kind], 1e6, 64,
                                    positions=p.positions, slots=p.slots, q_norm=wq, k_norm=wk, q_out=q)
            o = torch.zeros(n_tok, qd, dtype=self.dtype, device="cuda")
            out.append(P.paged_attn(q, layer, p.block_table, p.kv_lens, p.cu_new, self.nh, max_new, max_len, out=o))
        self.ctx.copy_(torch.where(p.kv_lens > 0, p.kv_lens, self.ctx))
        self.n_free.copy_(p.counts[:1])
        return out

    def exact(self, new, rows):
        """The step's outputs in 64 bits from unrounded keys and values, with their bounds."""
        outs = []
        for li, (x, (wq, wk)) in enumerate(zip(rows, self.w)):
            got, tols, at = [], [], 0
            for i, n in enumerate(new):
                if n == 0:
                    continue
                y = x[at:at + n].double().view(n, -1, self.d)
                at += n
                h = self.hist[li][i]
                pos = torch.arange(len(h), len(h) + n, device="cuda")
                q, _ = rope_oracle(y[:, :self.nh], pos, wq.double(), 1e-6, self.kind, 64, 1e6)
                k, _ = rope_oracle(y[:, self.nh:self.nh + self.nkv], pos, wk.double(), 1e-6, self.kind, 64, 1e6)
                h += list(torch.stack([k, y[:, self.nh + self.nkv:]], 1))
                kv = torch.stack(h)  # [L, 2, n_kv, d]
                hide = torch.arange(len(h), device="cuda")[None, :] > pos[:, None]
                o = torch.empty_like(q)
                t = torch.empty_like(q)
                for hd in range(self.nh):
                    K, V = kv[:, 0, hd * self.nkv // self.nh], kv[:, 1, hd * self.nkv // self.nh]
                    s = (q[:, hd] @ K.t() / math.sqrt(self.d)).masked_fill(hide, -math.inf)
                    p = s.softmax(-1)
                    o[:, hd] = p @ V
                    # q and k are rounded (u of each product's size): twice that in the softmax; V and P at f16
                    size = (q[:, hd].abs() @ K.abs().t() / math.sqrt(self.d)).masked_fill(hide, 0).amax(-1, keepdim=True)
                    t[:, hd] = (p @ V.abs()) * (2 * size * (U[self.dtype] + U[F16]) + 2 * U[F16] + 2.0 ** -16)
                got.append(o.reshape(n, -1))
                tols.append(t.reshape(n, -1))
            outs.append((torch.cat(got), torch.cat(tols)))
        return outs


def _hold(got, want, tol):
    err = (got.double()[:want.shape[0]] - want).abs()
    assert (err <= tol * 1.01 + U[got.dtype] * (want.abs() + tol) + 2.0 ** -24).all(), float((err / (tol + 1e-9)).max())


@pytest.mark.parametrize("nh,nkv,d,kind,dtype", [(14, 2, 64, "half", BF16), (8, 2, 128, "pairs", F16), (16, 2, 256, "mrope", F32)])
def test_serving_steps(cuda, nh, nkv, d, kind, dtype):
    """Prompts in chunks, then decode tokens, with sequences that join and pause: every step's attention rows."""
    s = Serve(4, nh, nkv, d, 64, kind, dtype, n_blocks=40, width=8)
    for new in ([70, 0, 33, 1], [130, 64, 1, 1], [1, 1, 1, 1], [1, 200, 0, 1], [5, 1, 1, 3], [1, 1, 1, 1]):
        T = sum(new)
        rows = s.rows(T + 3)
        got = s.step(_i32(new), rows, T + 3, max(new), 500)
        for o, (want, tol) in zip(got, s.exact(new, [r[:T] for r in rows])):
            _hold(o, want, tol)
            assert (o[T:] == 0).all()
    assert int(s.n_free) == 40 - sum(-(-int(c) // 64) for c in s.ctx)


def test_serving_when_blocks_run_out(cuda):
    """A sequence that gets no block keeps its pages and its rows are zero; the others go on."""
    s = Serve(3, 8, 2, 128, 64, "half", F16, n_blocks=4, width=4)
    for new, served in (([64, 64, 60], [1, 1, 1]), ([1, 1, 4], [1, 0, 1]), ([1, 0, 0], [1, 1, 1])):
        T = sum(new)
        rows = s.rows(T)
        got = s.step(_i32(new), rows, T, max(new), 256)
        at, keep = 0, []
        for n, ok in zip(new, served):
            keep += list(range(at, at + n)) if ok else []
            if not ok:
                assert (got[0][at:at + n] == 0).all() and (got[1][at:at + n] == 0).all()
            at += n
        eff = [n if ok else 0 for n, ok in zip(new, served)]
        for o, (want, tol) in zip(got, s.exact(eff, [r[keep] for r in rows])):
            _hold(o[keep], want, tol)


def test_serving_step_captured_and_replayed(cuda):
    """One captured decode step replays with the lengths, tables and free blocks that the replays themselves change,
    between eager work of the same kind; two captured graphs share nothing but the pool."""
    s = Serve(3, 8, 2, 128, 64, "half", BF16, n_blocks=24, width=6)
    prompt = [100, 63, 20]
    rows = s.rows(sum(prompt))
    for o, (want, tol) in zip(s.step(_i32(prompt), rows, 183, 100, 384), s.exact(prompt, rows)):
        _hold(o, want, tol)
    new, static = _i32([1, 1, 1]), s.rows(3)
    keep = (s.ctx.clone(), s.n_free.clone(), s.table.clone(), [(l.k.clone(), l.v.clone()) for l in s.layers])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a first pass outside the capture
        s.step(new, static, 3, 1, 384)
    torch.cuda.current_stream().wait_stream(side)
    s.ctx.copy_(keep[0]), s.n_free.copy_(keep[1]), s.table.copy_(keep[2])
    for l, (k, v) in zip(s.layers, keep[3]):
        l.k.copy_(k), l.v.copy_(v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.step(new, static, 3, 1, 384)
    for i in range(5):
        fresh = s.rows(3)
        for a, b in zip(static, fresh):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for o, (want, tol) in zip(out, s.exact([1, 1, 1], fresh)):
            _hold(o, want, tol)
        if i == 2:  # an eager step in between
            rows = s.rows(40)
            for o, (want, tol) in zip(s.step(_i32([0, 39, 1]), rows, 40, 39, 384), s.exact([0, 39, 1], rows)):
                _hold(o, want, tol)


# ---- calls that the documentation allows at the ends of its ranges ---------------------------------------

@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (32, 8, 128), (16, 2, 256)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("seqs", [[(0, 600), (0, 600)], [(100, 600), (0, 700), (256, 1)], [(0, 3000)], [(256, 900), (5, 400)]])
def test_attn_many_more_tokens_than_positions(cuda, nh, nkv, d, dtype, seqs):
    """Bounds of at most 256 keys, and prompts of more tokens than that, as the plan leaves a prompt that its table row
    cannot hold: every row is written."""
    b = Batch(seqs, nh, nkv, d, dtype=dtype, seed=70)
    out = torch.full((b.T, nh * d), math.nan, dtype=dtype, device="cuda")
    b.check(max_len=256 if b.table.shape[1] >= 4 else b.max_len, out=out)
    for (L, n), at in zip(seqs, b.cu):
        assert (out[at:at + max(0, n - L)] == 0).all()


def test_serving_prompts_that_their_table_rows_cannot_hold(cuda):
    """Refused by the plan, their attention rows are zero, whatever the output held."""
    from yllm_amd import paged as P

    new, width, (nh, nkv, d) = [600, 1, 500, 300], 4, (32, 8, 128)
    table = torch.full((4, width), -1, dtype=torch.int32, device="cuda")
    pool, T = P.PagedKV.empty(20, nkv, d), sum(new)
    step = P.paged_plan(table, _i32([0, 0, 0, 0]), _i32(new), _i32(list(range(20))), _i32([20]), 64, T)
    assert step.kv_lens.tolist() == [0, 1, 0, 0] and step.counts.tolist() == [19, T, 3, 0]
    x = torch.randn(T, (nh + 2 * nkv) * d, generator=_gen(71), device="cuda").half()
    q, k, v = x[:, :nh * d], x[:, nh * d:(nh + nkv) * d], x[:, (nh + nkv) * d:]
    P.qk_norm_rope_kv_store(pool, q, k, v, nh, KINDS["half"], 1e6, positions=step.positions, slots=step.slots)
    out = torch.full((T, nh * d), math.nan, dtype=F16, device="cuda")
    P.paged_attn(q, pool, step.block_table, step.kv_lens, step.cu_new, nh, max(new), width * 64, out=out)
    want = torch.zeros_like(out)
    want[600] = v[600].view(nkv, 1, d).expand(nkv, nh // nkv, d).reshape(-1)  # its only key
    assert torch.equal(out, want)


@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("L,new", [(70, 1), (70, 6), (900, 2), (400, 40), (400, 300)])
def test_attn_nan_of_any_bits_stays_nan(cuda, nh, nkv, d, dtype, out_dtype, L, new):
    """Values of all ones, as a page filled with 0xff bytes holds, are NaN in every output type, of the rows that see them."""
    for at in (L - 1, 0):  # seen by the last row alone, by all
        b = Batch([(L, new), (129, 2)], nh, nkv, d, dtype=dtype, seed=72)
        page, off = int(b.table[0, at // 64]), at % 64
        bits = torch.tensor([0x7fff, -1, 0x7c01, -0x3ff], dtype=torch.int16, device="cuda").repeat(d // 4)
        b.cache.v.view(torch.int16)[page, :, off // 32, :, off % 32] = bits
        got = b.run(out_dtype=out_dtype)
        assert got[new - 1].isnan().all()
        rest = got[new:] if at == 0 else torch.cat([got[:new - 1], got[new:]])
        assert rest.isfinite().all()
        if at == 0:
            assert got[:new].isnan().all()


@pytest.mark.parametrize("nh,nkv,d", [(32, 8, 64), (16, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n_seq,L,new", [(1, 131072, 2048), (72, 32768, 1)])
def test_attn_many_small_probabilities(cuda, nh, nkv, d, dtype, n_seq, L, new):
    """One key far above all others, which are so many that they count all the same: with a score of s the first key, of
    value 0, and of 0 the others, of value 1, the row at position p is p e^-s / (1 + p e^-s)."""
    from yllm_amd.paged import PagedKV, paged_attn

    c = 19.0 / math.sqrt(d)  # e^-19 = 2^-27.4
    c = float(torch.tensor(c).half())
    s = c * math.sqrt(d)
    pages = L // 1024
    pool = PagedKV(torch.zeros((pages, nkv, 1024, d), dtype=F16, device="cuda"),
                   torch.ones((pages, nkv, 32, d, 32), dtype=F16, device="cuda"))
    pool.k[0, :, 0], pool.v[0, :, 0, :, 0] = c, 0.0
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(n_seq, pages).contiguous()
    q = torch.ones((n_seq * new, nh * d), dtype=dtype, device="cuda")
    got = paged_attn(q, pool, table, _i32([L] * n_seq), _i32([i * new for i in range(n_seq + 1)]), nh, new, L, out_dtype=F32)
    p = torch.arange(L - new, L, device="cuda").double().repeat(n_seq)
    w = p * math.exp(-s)
    want = (w / (1 + w))[:, None]
    # a probability: half a step of f16 (of a hi and lo pair, 2^-22), or, below the f16 normals, half of 2^-24 times the
    # 2^-7 by which the largest is scaled up; the score's sum and exp2: 2^-24 of s = 19 three times, its sums 2^-20
    u = 2.0 ** -22 if dtype == F32 else 2.0 ** -11
    tol = want * (u + 2.0 ** -20 + 3 * 19 * 2.0 ** -24) + p[:, None] * 2.0 ** -32 + want * 2.0 ** -24
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (float(err.max()), float((err / tol).max()), float(want.max()))


@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("n_seq", [1, 9])
@pytest.mark.parametrize("new", [1, 2])
def test_attn_contexts_about_the_longest_that_is_not_cut(cuda, nh, nkv, d, n_seq, new):
    for L in (65536 // d - 128, 65536 // d - 1, 65536 // d, 65536 // d + 1, 65536 // d + 129):
        b = Batch([(max(new, L - 37 * i), new) for i in range(n_seq)], nh, nkv, d, dtype=(F16, F32)[L % 2], seed=L)
        b.check()
        # under another bound, on either side of that length, the same rows
        b.check(max_len=b.table.shape[1] * 64)
