"""Serving over a paged KV cache held in 8 bits on the GPU (PagedKV8 of yllm_amd/paged.py) against plain 64-bit forms.

Tolerances count roundings: at most half a step each (e4m3 2^-4 of the value, or 2^-10 scales where that is more; f16 2^-11,
bf16 2^-8, fp32 2^-24).  What is quantised from the rows themselves, without arithmetic before it, has to match byte for byte."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_paged import BF16, F16, F32, HEADS, KINDS, U, Batch, _gen, _i32, _slots, rope_oracle

pytestmark = pytest.mark.gpu

U8 = torch.uint8
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def quantise(x):
    """(codes, scales) of rows in 64 bits, as numbers: the smallest scale whose 448 reaches the largest finite magnitude, codes
    to the nearest multiple of their step, ties to even; NaN where x is not finite."""
    x = x.double()
    fin = torch.isfinite(x)
    top = torch.where(fin, x.abs(), 0.0).amax(-1)
    scale = torch.full_like(top, 2.0 ** 7)
    for k in range(6, -15, -1):
        scale = torch.where(top <= 448.0 * 2.0 ** k, 2.0 ** k, scale)
    y = (x / scale[..., None]).nan_to_num(0.0, 0.0, 0.0).clamp(-448.0, 448.0)
    step = torch.full_like(y, 2.0 ** -9)
    for e in range(-5, 9):
        step = torch.where(y.abs() >= 2.0 ** e, 2.0 ** (e - 3), step)
    return torch.where(fin, (y / step).round() * step, math.nan), scale


def as_codes(y):
    """Numbers that e4m3 holds, as it holds them (NaN as 0x7f)."""
    return y.float().to(E4M3).view(U8).masked_fill(y.isnan(), 0x7f)


def pool8(n_blocks, nkv, d, block, fill=0xff):
    """A pool whose every byte is `fill` (0xff: NaN codes and NaN scales)."""
    from yllm_amd.paged import PagedKV8

    p = PagedKV8.empty(n_blocks, nkv, d, block, zero=False)
    for t in (p.k, p.v, p.k_scale, p.v_scale):
        t.view(U8).fill_(fill)
    return p


def rows_of_pool(p):
    """Codes and scales of K and V by slot: [slots, n_kv, d] bytes and [slots, n_kv] bytes."""
    nkv, d = p.n_kv, p.head_dim
    return (p.k.view(U8).transpose(1, 2).reshape(-1, nkv, d), p.v.view(U8).permute(0, 2, 4, 1, 3).reshape(-1, nkv, d),
            p.k_scale.view(U8).transpose(1, 2).reshape(-1, nkv), p.v_scale.view(U8).transpose(1, 2).reshape(-1, nkv))


def values(codes, scales):
    return codes.contiguous().view(E4M3).double() * scales.contiguous().view(E5M2).double()[..., None]


# ---- qk_norm_rope_kv8_store ------------------------------------------------------------------------

def _check_store(T, nh, nkv, d, kind, dtype, out_dtype, norm=True, block=64, n_rot=0, wide=0, skip=(), seed=0,
                 norm_dtype=F32, far=0, theta=1e6, in_place=False, with_q=True, spread=0.0):
    from yllm_amd.paged import qk_norm_rope_kv8_store

    g = _gen(seed + T)
    width = (nh + 2 * nkv) * d
    rows = torch.randn(T, width + wide, generator=g, device="cuda") * 1.5
    if spread:
        rows *= torch.exp2(torch.rand(T, 1, generator=g, device="cuda") * spread - spread / 2)
    rows = rows.to(dtype)
    x = rows[:, :width]
    q, k, v = x[:, :nh * d], x[:, nh * d:(nh + nkv) * d], x[:, (nh + nkv) * d:]
    n_blocks = T // 37 + T // block + 3
    cache = pool8(n_blocks, nkv, d, block, fill=0x2a)
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
    got = qk_norm_rope_kv8_store(cache, q if with_q else None, k, v, nh, KINDS[kind], theta, n_rot,
                                 positions=_i32(pos), slots=_i32(slots), q_norm=qw, k_norm=kw, eps=1e-5, q_out=q_out)
    x = given[:, :width].double().view(T, nh + 2 * nkv, d)
    ok = [i for i, s in enumerate(slots) if 0 <= s < n_blocks * block]
    p = _i32(pos)
    wq, wk = (None, None) if not norm else (qw.double(), kw.double())
    if with_q:
        want, tol = rope_oracle(x[:, :nh], p, wq, 1e-5, kind, n_rot, theta)
        err = (got.double().view(T, nh, d)[ok] - want[ok]).abs()
        assert (err <= tol[ok] + U[out_dtype] * want[ok].abs() + 2.0 ** -25).all(), float(err.max())
        rest = [i for i in range(T) if i not in set(ok)]
        if rest:
            before = given[:, :nh * d].to(out_dtype) if in_place else torch.full_like(got, 9.0)
            assert torch.equal(got[rest], before[rest])
    else:
        assert got is None
    if not in_place:
        assert torch.equal(rows, given)
    K, V, KS, VS = rows_of_pool(cache)
    at = torch.tensor([slots[i] for i in ok], device="cuda", dtype=torch.long)
    free = torch.ones(len(K), dtype=torch.bool, device="cuda")
    free[at] = False
    for t in (K, V, KS, VS):  # nothing else is written
        assert (t[free] == 0x2a).all()
    if not ok:
        return
    code, scale = quantise(x[ok][:, nh + nkv:])
    assert torch.equal(V[at], as_codes(code)) and torch.equal(VS[at], scale.to(E5M2).view(U8))
    want, tol = rope_oracle(x[:, nh:nh + nkv], p, wk, 1e-5, kind, n_rot, theta)
    want, tol = want[ok], tol[ok]
    s = KS[at].view(E5M2).double()
    # a scale is that of an amax within its error of the exact one
    lo, hi = (quantise(want.abs().amax(-1, keepdim=True) + e * tol.amax(-1, keepdim=True))[1] for e in (-1, 1))
    assert ((s == lo) | (s == hi)).all()
    half = torch.maximum((want.abs() + tol) * 2.0 ** -4, 2.0 ** -10 * s[..., None])
    err = (values(K[at], KS[at]) - want).abs()
    over = (want.abs() - 57344.0).clamp(min=0.0)
    assert (err <= half + tol + over).all(), float((err / half).max())


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (16, 2, 256), (5, 5, 64), (3, 2, 128)])
@pytest.mark.parametrize("T", [1, 7, 129, 401])
def test_store(cuda, kind, nh, nkv, d, T):
    dt, out = [(F32, F32), (BF16, F16), (F16, BF16)][(T + nh) % 3]
    _check_store(T, nh, nkv, d, kind, dt, out, n_rot=64 if kind == "mrope" else 0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("out", [F32, F16, BF16])
def test_store_types(cuda, dtype, out):
    _check_store(500, 8, 2, 128, "half", dtype, out, wide=24, spread=12.0)
    _check_store(30, 8, 2, 128, "pairs", dtype, out, wide=4, norm=False, spread=12.0)


@pytest.mark.parametrize("T", [64, 127, 128, 130, 191, 200, 383, 384, 385, 386, 400, 447, 463, 519, 700])
def test_store_row_counts(cuda, T):
    """Both forms of the V store, groups of sixteen that begin and end in any window."""
    _check_store(T, 4, 2, 64, "half", F32, F16, seed=T)
    _check_store(T, 2, 1, 256, "mrope", BF16, BF16, block=128, n_rot=64, seed=T + 1)
    _check_store(T, 4, 3, 128, "pairs", F16, BF16, block=256, seed=T + 2)


@pytest.mark.parametrize("n_rot", [8, 24, 64, 128])
def test_store_partial_rotation(cuda, n_rot):
    _check_store(40, 4, 2, 128, "mrope", F32, F32, n_rot=n_rot)


def test_store_far_positions(cuda):
    for T in (140, 450):
        _check_store(T, 4, 2, 128, "pairs", F32, F32, far=131071 * 8)
    _check_store(9, 4, 2, 64, "half", F32, F32, far=(1 << 31) - 100, theta=1e4)


def test_store_rows_without_a_slot(cuda):
    big = 0x7fffffff
    for T in (12, 200, 500):
        _check_store(T, 4, 2, 128, "half", BF16, BF16, skip=[(0, -1), (3, -5), (T - 1, big), (T - 2, -big)])
        _check_store(T, 4, 2, 128, "half", F32, F32, skip=[(i, -1) for i in range(T)])


def test_store_in_place_f16_weights_and_keys_only(cuda):
    _check_store(450, 6, 2, 128, "half", F32, F32, in_place=True, norm_dtype=F16)
    _check_store(3, 6, 2, 128, "pairs", BF16, BF16, in_place=True)
    _check_store(150, 6, 2, 128, "half", F16, F16, with_q=False)
    _check_store(450, 6, 2, 64, "half", F16, F16, with_q=False)


def _edges(T, d, dtype, seed):
    """Rows about every border of the format: ties and their neighbours, largest magnitudes at and beside 448 * 2^k, tiny and
    large rows, zeros, inf and NaN."""
    g = _gen(seed)
    e = torch.randint(-12, 4, (T, d), generator=g, device="cuda").float()
    m = 1.0 + torch.randint(0, 16, e.shape, generator=g, device="cuda") / 16.0  # ties at 4 bits
    x = m * torch.exp2(e) * torch.where(torch.rand(e.shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    x[:, ::5] = torch.nextafter(x[:, ::5], torch.zeros_like(x[:, ::5]))
    x[:, 1::7] = torch.nextafter(x[:, 1::7], torch.full_like(x[:, 1::7], math.inf))
    k = torch.arange(T, device="cuda") % 26 - 17  # a row's exponent, past both ends of the range
    x = x * torch.exp2(k.float())[:, None]
    top = 448.0 * torch.exp2(k.float())
    up, down = (torch.nextafter(top, torch.full_like(top, v)) for v in (math.inf, 0.0))
    x[:, 3] = torch.stack([top, up, down, top * 0.99, top * 1.03], 1)[torch.arange(T, device="cuda"), torch.arange(T, device="cuda") // 26 % 5]
    x[0], x[1], x[2, 4:] = 0.0, -0.0, 0.0
    x[5, 9], x[6, 9], x[7, 9], x[8] = math.inf, -math.inf, math.nan, math.nan
    x[9, 1], x[10, 1] = 1e-45, 3e38
    return x.to(dtype)


@pytest.mark.parametrize("T", [60, 460])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_store_of_every_border_is_the_format_byte_for_byte(cuda, T, d, dtype):
    from yllm_amd.attention import ROPE_NONE
    from yllm_amd.paged import qk_norm_rope_kv8_store

    k = _edges(T, 2 * d, dtype, d)
    v = k.flip(0).contiguous()
    p = pool8(4, 2, d, 128)
    qk_norm_rope_kv8_store(p, None, k, v, 2, ROPE_NONE, 1.0, pos_start=5)
    K, V, KS, VS = (t[5:5 + T] for t in rows_of_pool(p))  # (without slots: the positions from 5 on, in pages one behind the other)
    for x, c, s in ((k, K, KS), (v, V, VS)):
        code, scale = quantise(x.view(T, 2, d))
        assert torch.equal(s, scale.to(E5M2).view(U8))
        want = as_codes(code)
        nan = want == 0x7f
        assert torch.equal(c & 0x7f, want & 0x7f), int(((c ^ want) & 0x7f != 0).sum())
        assert torch.equal(c[~nan], want[~nan])  # signs, of zeros too


@pytest.mark.parametrize("d", [64, 128, 256])
def test_store_gives_the_same_bytes_in_any_chunks(cuda, d):
    from yllm_amd.paged import qk_norm_rope_kv8_store

    T, nkv, g = 700, 2, _gen(8)
    k, v = (torch.randn(T, nkv * d, generator=g, device="cuda") for _ in range(2))
    w = 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    pools = []
    for cuts in ([0, T], [0, 1, 2, 60, 61, 190, 299, T], [0, 400, T], list(range(0, T, 7)) + [T]):
        p = pool8(6, nkv, d, 128, fill=0)
        for a, e in zip(cuts, cuts[1:]):
            qk_norm_rope_kv8_store(p, None, k[a:e], v[a:e], nkv, KINDS["half"], 1e6, positions=pos[a:e], slots=pos[a:e],
                                   q_norm=w, k_norm=w)
        pools.append(rows_of_pool(p))
    order = torch.randperm(T, generator=torch.Generator().manual_seed(1)).cuda()
    p = pool8(6, nkv, d, 128, fill=0)
    qk_norm_rope_kv8_store(p, None, k[order], v[order], nkv, KINDS["half"], 1e6, positions=pos[order], slots=pos[order],
                           q_norm=w, k_norm=w)
    pools.append(rows_of_pool(p))
    for other in pools[1:]:
        assert all(torch.equal(a, b) for a, b in zip(pools[0], other))


def test_store_queries_are_those_of_the_f16_store(cuda):
    from yllm_amd.paged import PagedKV, qk_norm_rope_kv8_store, qk_norm_rope_kv_store

    for T in (3, 140, 400):
        x = torch.randn(T, 12 * 128, generator=_gen(T), device="cuda").to(BF16)
        q, k, v = x[:, :1024], x[:, 1024:1280], x[:, 1280:]
        pos = torch.arange(T, dtype=torch.int32, device="cuda")
        a = qk_norm_rope_kv_store(PagedKV.empty(7, 2, 128), q, k, v, 8, KINDS["pairs"], 5e5, positions=pos, slots=pos)
        b = qk_norm_rope_kv8_store(pool8(7, 2, 128, 64), q, k, v, 8, KINDS["pairs"], 5e5, positions=pos, slots=pos)
        assert torch.equal(a, b)


def test_store_into_a_pool_past_4_gib(cuda):
    from yllm_amd.attention import ROPE_NONE
    from yllm_amd.paged import PagedKV8, qk_norm_rope_kv8_store

    nkv, d, block = 8, 128, 256
    nb = (5 << 30) // (nkv * d * block)  # 5 GiB of K
    big = PagedKV8.empty(nb, nkv, d, block, zero=False)
    for T in (3, 200, 480):
        first = (nb - 2) * block + 17
        for t in (big.k, big.v, big.k_scale, big.v_scale):
            t.view(U8)[-2:] = 3
        kv = torch.randn((2, T, nkv * d), generator=_gen(T), device="cuda").half()
        qk_norm_rope_kv8_store(big, None, kv[0], kv[1], nkv, ROPE_NONE, 1.0, positions=_i32(list(range(T))),
                               slots=_i32(list(range(first, first + T))))
        K, V, KS, VS = rows_of_pool(PagedKV8(big.k[-2:], big.v[-2:], big.k_scale[-2:], big.v_scale[-2:]))
        for x, c, s in ((kv[0], K, KS), (kv[1], V, VS)):
            code, scale = quantise(x.view(T, nkv, d))
            assert torch.equal(c[17:17 + T], as_codes(code)) and torch.equal(s[17:17 + T], scale.to(E5M2).view(U8))
            assert (c[:17] == 3).all() and (c[17 + T:] == 3).all() and (s[:17] == 3).all() and (s[17 + T:] == 3).all()


# ---- pages ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("nkv,d", [(2, 64), (3, 128), (1, 256)])
@pytest.mark.parametrize("block", [64, 256])
def test_pages_both_ways(cuda, nkv, d, block):
    from yllm_amd.paged import PagedKV, kv8_from_pages, kv8_to_pages

    half = PagedKV.empty(7, nkv, d, block)
    x = _edges(7 * nkv * block, 2 * d, F16, block)  # rows of K and V
    rows = [t.reshape(7, nkv, block, d) for t in (x[:, :d], x[:, d:])]
    half.k.copy_(rows[0])
    half.v.copy_(rows[1].reshape(7, nkv, block // 32, 32, d).transpose(-1, -2))
    p = pool8(9, nkv, d, block, fill=0x2a)
    dst, src = _i32([8, 0, -1, 3, 9, 2]), _i32([1, 6, 2, 3, 0, 1])  # (the third and the fifth are outside)
    kv8_from_pages(p, half, dst, src)
    pairs = [(8, 1), (0, 6), (3, 3), (2, 1)]
    V8 = p.v.view(U8).permute(0, 1, 2, 4, 3).reshape(9, nkv, block, d)
    for d8, s16 in pairs:
        for x, c, s in ((rows[0], p.k.view(U8), p.k_scale), (rows[1], V8, p.v_scale)):
            code, scale = quantise(x[s16])
            assert torch.equal(s.view(U8)[d8], scale.to(E5M2).view(U8))
            want = as_codes(code)
            nan = want == 0x7f
            assert torch.equal(c[d8] & 0x7f, want & 0x7f) and torch.equal(c[d8][~nan], want[~nan])
    for other in (1, 4, 5, 6, 7):
        for t in (p.k, p.v, p.k_scale, p.v_scale):
            assert (t.view(U8)[other] == 0x2a).all()
    back = PagedKV.empty(4, nkv, d, block)
    back.k.fill_(7.0), back.v.fill_(7.0)
    kv8_to_pages(back, p, _i32([2, 0, 4, 1]), _i32([8, 3, 0, 9]))
    bv = back.v.transpose(-1, -2).reshape(4, nkv, block, d)
    for d16, s8 in ((2, 8), (0, 3)):
        for got, c, s in ((back.k, p.k.view(U8), p.k_scale), (bv, V8, p.v_scale)):
            want = values(c[s8], s.view(U8)[s8])  # (exactly: f16 holds every value)
            nan = want.isnan()
            assert torch.equal(got[d16].isnan(), nan) and torch.equal(got[d16].double()[~nan], want[~nan])
    for other in (1, 3):
        assert (back.k[other] == 7).all() and (back.v[other] == 7).all()
    # quantised again, the same values: a code's scale is the smallest only where 448 is reached, the values stay
    again = pool8(9, nkv, d, block)
    kv8_from_pages(again, back, _i32([0, 1]), _i32([2, 0]))
    for a, s8 in ((0, 8), (1, 3)):
        x, y = values(again.k.view(U8)[a], again.k_scale.view(U8)[a]), values(p.k.view(U8)[s8], p.k_scale.view(U8)[s8])
        assert torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0))


def test_pages_hold_what_the_store_holds(cuda):
    """Rows stored in f16 pages and converted, or stored in 8 bits from f16 rows: the same bytes."""
    from yllm_amd.attention import ROPE_NONE
    from yllm_amd.paged import PagedKV, kv8_from_pages, qk_norm_rope_kv8_store, qk_norm_rope_kv_store

    kv = torch.randn((2, 192, 256), generator=_gen(3), device="cuda").half()
    pos = torch.arange(192, dtype=torch.int32, device="cuda")
    half, a, b = PagedKV.empty(3, 2, 128), pool8(3, 2, 128, 64), pool8(3, 2, 128, 64)
    qk_norm_rope_kv_store(half, None, kv[0], kv[1], 2, ROPE_NONE, 1.0, positions=pos, slots=pos)
    kv8_from_pages(a, half, _i32([0, 1, 2]), _i32([0, 1, 2]))
    qk_norm_rope_kv8_store(b, None, kv[0], kv[1], 2, ROPE_NONE, 1.0, positions=pos, slots=pos)
    assert all(torch.equal(x, y) for x, y in zip(rows_of_pool(a), rows_of_pool(b)))


# ---- paged_attn8 ----------------------------------------------------------------------------------------

class Batch8(Batch):
    """The same over 8-bit pages, whose unused positions hold NaN codes and NaN scales; K and V become what is held."""

    def __init__(self, seqs, nh, nkv, d, block=64, spread=0.0, **kw):
        super().__init__(seqs, nh, nkv, d, block=block, **kw)
        self.cache = pool8(self.cache.n_blocks, nkv, d, block)
        g = _gen(77)
        for i, (L, _) in enumerate(seqs):
            L = max(L, 0)
            for name in ("K", "V"):
                x = getattr(self, name)[i].double()
                if spread:  # rows of different magnitude
                    x = x * torch.exp2((torch.rand(nkv, L, 1, generator=g, device="cuda") - 0.5) * spread).double()
                code, scale = quantise(x)
                getattr(self, name)[i] = (code * scale[..., None]).half()
                for j in range(-(-L // block)):
                    self.put(name, int(self.table[i, j]), slice(0, min(block, L - j * block)),
                             as_codes(code[:, j * block:(j + 1) * block]), scale[:, j * block:(j + 1) * block].to(E5M2).view(U8))

    def put(self, name, page, at, codes, scales):
        """codes [n_kv, n, d] and scales [n_kv, n] (bytes) at positions `at` of a page."""
        nkv, d, block = self.nkv, self.d, self.block
        c = self.cache
        if name == "K":
            c.k.view(U8)[page][:, at], c.k_scale.view(U8)[page][:, at] = codes, scales
        else:
            rows = c.v.view(U8)[page].transpose(-1, -2).reshape(nkv, block, d).clone()
            rows[:, at] = codes
            c.v.view(U8)[page] = rows.view(nkv, block // 64, 64, d).transpose(-1, -2)
            c.v_scale.view(U8)[page][:, at] = scales

    def run(self, **kw):
        from yllm_amd.paged import paged_attn8

        kw = {"max_new": self.max_new, "max_len": self.max_len, "gate": self.gate, **kw}
        mn, ml = kw.pop("max_new"), kw.pop("max_len")
        return paged_attn8(self.q, self.cache, self.table, _i32([max(L, 0) for L, _ in self.seqs]), _i32(self.cu),
                           self.nh, mn, ml, **kw)


@pytest.mark.parametrize("nh,nkv,d", HEADS)
@pytest.mark.parametrize("L", [1, 2, 31, 64, 65, 511, 1500])
def test_attn_one_token(cuda, nh, nkv, d, L):
    Batch8([(L, 1)], nh, nkv, d, dtype=(F16, BF16, F32)[L % 3], seed=L, spread=6.0).check()


@pytest.mark.parametrize("nh,nkv,d", HEADS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_attn_decode_batch(cuda, nh, nkv, d, dtype):
    seqs = [(1, 1), (700, 1), (64, 1), (0, 1), (129, 1), (2000, 1), (63, 1), (333, 1)]
    Batch8(seqs, nh, nkv, d, dtype=dtype, block=128, seed=2).check()


@pytest.mark.parametrize("nh,nkv,d", HEADS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_attn_mixed_batch(cuda, nh, nkv, d, dtype):
    """Decode tokens, drafts, chunks, a whole prompt, a sequence without keys or without new tokens."""
    seqs = [(300, 1), (200, 200), (77, 3), (0, 0), (900, 130), (50, 0), (0, 2), (513, 64), (65, 17), (128, 128)]
    Batch8(seqs, nh, nkv, d, dtype=dtype, seed=3, gated=d == 256, behind=3, spread=6.0).check()


@pytest.mark.parametrize("new", [1, 2, 5, 16, 31, 33, 63, 64, 65, 127, 128, 129, 200, 257, 515])
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (16, 2, 256)])
def test_attn_chunk_lengths(cuda, nh, nkv, d, new):
    for k, ctx in enumerate((0, 1, 100, 704)):
        Batch8([(ctx + new, new)], nh, nkv, d, dtype=(F16, BF16, F32)[(new + k) % 3], block=(64, 256)[k % 2],
               seed=new).check()


@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("new", [1, 2, 3, 4, 5, 8, 16])
def test_attn_drafted_tokens(cuda, nh, nkv, d, new):
    """A few tokens of each of many sequences: one block of rows, and two."""
    for dt in (F16, F32):
        Batch8([(max(new, 90 * i), new) for i in range(1, 12)], nh, nkv, d, dtype=dt, seed=new).check()


@pytest.mark.parametrize("block", [64, 128, 256, 1024])
def test_attn_blocks(cuda, block):
    Batch8([(1000, 300), (70, 1), (513, 9)], 8, 2, 128, block=block, seed=block).check()


def test_attn_more_tokens_than_positions(cuda):
    """Tokens at negative positions see nothing: zero rows."""
    b = Batch8([(3, 7), (0, 5), (1, 140), (130, 200)], 8, 2, 128, seed=1)
    out = b.check()
    assert (out[:4] == 0).all() and (out[7:12] == 0).all() and (out[12:12 + 139] == 0).all()


@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (32, 8, 128), (16, 2, 256)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("seqs", [[(0, 600), (0, 600)], [(100, 600), (0, 700), (256, 1)], [(0, 3000)], [(256, 900), (5, 400)]])
def test_attn_many_more_tokens_than_positions(cuda, nh, nkv, d, dtype, seqs):
    b = Batch8(seqs, nh, nkv, d, dtype=dtype, seed=70)
    out = torch.full((b.T, nh * d), math.nan, dtype=dtype, device="cuda")
    b.check(max_len=256 if b.table.shape[1] >= 4 else b.max_len, out=out)
    for (L, n), at in zip(seqs, b.cu):
        assert (out[at:at + max(0, n - L)] == 0).all()


@pytest.mark.parametrize("out_dtype", [F16, BF16, F32])
def test_attn_output_types_strides_and_rows_behind(cuda, out_dtype):
    b = Batch8([(100, 3), (333, 90), (64, 1)], 8, 2, 128, seed=4, behind=6, gated=True)
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
        b = Batch8(seqs, 8, nkv, d, block=block, seed=9)
        b.table[0, 0], b.table[1, 0] = 1 << 30, -9
        for i in (0, 1):
            b.K[i][:, :block], b.V[i][:, :block] = 0, 0
        b.check()


@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("L,new", [(70, 1), (70, 6), (400, 40), (400, 300), (64, 64), (514, 2), (515, 9)])
def test_attn_values_that_a_query_does_not_see(cuda, nh, nkv, d, dtype, L, new):
    """NaN in the keys and values of the last token reaches the rows of that token and no other."""
    b = Batch8([(L, new), (129, 2)], nh, nkv, d, dtype=dtype, seed=5)
    page, off = int(b.table[0, (L - 1) // 64]), (L - 1) % 64
    bad = torch.tensor([0x7f, 0xff, 0x38, 0xb8], dtype=U8, device="cuda").repeat(d // 4)  # NaN, NaN, 1, -1
    b.put("V", page, slice(off, off + 1), bad.expand(nkv, 1, d), torch.full((nkv, 1), 0x3c, dtype=U8, device="cuda"))
    b.V[0][:, L - 1] = 0  # what rows that do not see it are held to
    got = b.run()
    want, tol = b.exact()
    rows = [r for r in range(b.T) if r != new - 1]
    err = (got.double() - want).abs()[rows]
    assert (err <= tol[rows] + U[got.dtype] * want[rows].abs() + 2.0 ** -24).all(), float(err.nan_to_num(9.0).max())
    last = got[new - 1].view(nh, d).float()
    assert last[:, 0::4].isnan().all() and last[:, 1::4].isnan().all() and last[:, 2::4].isfinite().all()
    assert last[:, 3::4].isfinite().all()
    # a key of NaN: every score of the last row, no other row's
    b.put("K", page, slice(off, off + 1), torch.full((nkv, 1, d), 0x7f, dtype=U8, device="cuda"),
          torch.full((nkv, 1), 0x3c, dtype=U8, device="cuda"))
    got = b.run()
    err = (got.double() - want).abs()[rows]
    assert (err <= tol[rows] + U[got.dtype] * want[rows].abs() + 2.0 ** -24).all()
    assert got[new - 1].isnan().all()
    # a value of NaN that all rows see
    b = Batch8([(L, new), (129, 2)], nh, nkv, d, dtype=dtype, seed=5)
    b.put("V", int(b.table[0, 0]), slice(0, 1), bad.expand(nkv, 1, d), torch.full((nkv, 1), 0x3c, dtype=U8, device="cuda"))
    seen = b.run()[:new].view(new, nh, d).float() if L > new else b.run()[:new].view(new, nh, d).float()
    assert seen[:, :, 0::4].isnan().all() and seen[:, :, 2::4].isfinite().all() and b.run()[new:].isfinite().all()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attn_large_scores_and_scales(cuda, dtype):
    """Softmax maxima far apart from tile to tile, up and down; rows of every scale."""
    Batch8([(1000, 1), (600, 70), (900, 4)], 8, 2, 128, dtype=dtype, seed=6, qscale=6.0).check()
    Batch8([(1000, 1), (600, 70), (900, 4)], 8, 2, 128, dtype=dtype, seed=6, spread=16.0).check()


@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (16, 2, 256)])
def test_attn_codes_and_scales_at_the_ends_of_their_ranges(cuda, nh, nkv, d):
    """Subnormal codes, 448, the smallest and the largest scale: what is held is what enters the sums."""
    g = _gen(4)
    for seqs in ([(200, 1), (130, 2)], [(200, 150), (64, 40)]):
        b = Batch8(seqs, nh, nkv, d, dtype=F32, seed=8)
        for i, (L, _) in enumerate(seqs):
            for name, scales in (("K", [0x04, 0x3c]), ("V", [0x04, 0x58])):
                codes = torch.randint(0, 0x7f, (nkv, L, d), generator=g, device="cuda").to(U8)
                codes |= torch.randint(0, 2, codes.shape, generator=g, device="cuda").to(U8) << 7
                if name == "K":
                    codes &= 0x8f  # subnormals (keys of 448 would leave one key per row)
                s = torch.tensor(scales, dtype=U8, device="cuda")[torch.randint(0, 2, (nkv, L), generator=g, device="cuda")]
                getattr(b, name)[i] = values(codes, s).half()
                assert torch.equal(getattr(b, name)[i].double(), values(codes, s))
                for j in range(-(-L // 64)):
                    at = slice(64 * j, min(L, 64 * j + 64))
                    b.put(name, int(b.table[i, j]), slice(0, at.stop - at.start), codes[:, at], s[:, at])
        b.check()


def test_attn_long_context(cuda):
    """Many splits of one sequence."""
    Batch8([(40000, 1), (17, 1)], 32, 8, 128, dtype=BF16, block=256, seed=7).check()
    Batch8([(9000, 1), (9100, 33)], 16, 2, 256, dtype=F16, block=64, seed=8).check()


def test_attn_pool_past_4_gib(cuda):
    from yllm_amd.paged import PagedKV8

    nkv, d, block = 8, 128, 1024
    nb = (5 << 30) // (nkv * d * block)  # 5 GiB of K
    b = Batch8([(2000, 1), (1500, 140)], 32, nkv, d, block=block, seed=10)
    big = PagedKV8.empty(nb, nkv, d, block, zero=False)
    for i in range(2):
        for j in range(2):
            old, page = int(b.table[i, j]), nb - 1 - 2 * j - i
            for x, y in ((big.k, b.cache.k), (big.v, b.cache.v), (big.k_scale, b.cache.k_scale), (big.v_scale, b.cache.v_scale)):
                x.view(U8)[page] = y.view(U8)[old]
            b.table[i, j] = page
    b.cache = big
    b.check()


def test_attn_many_sequences(cuda):
    """More sequences than threads of a workgroup."""
    g = torch.Generator().manual_seed(1)
    seqs = [(int(L), 1) for L in torch.randint(0, 90, (1100,), generator=g)]
    Batch8(seqs, 4, 2, 64, seed=12).check()
    seqs = [(L, min(L, 1 + i % 3)) for i, (L, _) in enumerate(seqs)]
    Batch8(seqs, 4, 2, 64, seed=13).check()
    seqs = [(L, min(L, 1 + (i % 5) * 17)) for i, (L, _) in enumerate(seqs[:300])]
    Batch8(seqs, 4, 2, 64, seed=14).check()


def test_attn_loose_bounds_and_a_larger_workspace(cuda):
    """Bounds larger than the batch give the same rows; so does a workspace for more."""
    from yllm_amd.paged import paged_attn8_workspace

    for seqs in ([(300, 1), (2000, 1)], [(300, 20), (2000, 190), (70, 1)]):
        b = Batch8(seqs, 28, 4, 128, seed=14)
        ws = paged_attn8_workspace(4096, 64, 512, 32768, 28, 4, 128)
        b.check(max_len=None)
        b.check(workspace=ws)
        b.check(max_new=b.T, workspace=torch.empty(256, dtype=U8, device="cuda"))


def test_attn_same_result_twice(cuda):
    """No order of arrival in the sums: the same bits every time."""
    for seqs in ([(3000, 1), (700, 200), (5000, 7)], [(30000, 1), (700, 1)]):
        b = Batch8(seqs, 28, 4, 128, seed=15)
        first = b.run()
        for _ in range(3):
            assert torch.equal(b.run(), first)


def test_attn_on_another_stream_and_two_at_once(cuda):
    """Each with its own workspace."""
    from yllm_amd.paged import paged_attn8_workspace

    batches = [Batch8([(3000, 1), (700, 200)], 28, 4, 128, seed=40), Batch8([(9000, 1), (50, 1)], 16, 2, 256, seed=41)]
    want = [b.check() for b in batches]
    spaces = [paged_attn8_workspace(b.T, 2, b.max_new, b.max_len, b.nh, b.nkv, b.d) for b in batches]
    streams, got = [torch.cuda.Stream() for _ in batches], [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for st, b, ws, o in zip(streams, batches, spaces, got):
            with torch.cuda.stream(st):
                o.append(b.run(workspace=ws))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w) for o in outs)


def test_attn_more_new_tokens_than_the_bound(cuda):
    """A sequence with more than max_new new tokens: the first max_new rows are computed, the rest left as they were."""
    for seqs, cut in (([(90, 5), (200, 2)], 2), ([(300, 200), (64, 3)], 150), ([(300, 200), (64, 3)], 60)):
        b = Batch8(seqs, 8, 2, 128, seed=21)
        whole, out = b.check(), torch.full((b.T, 8 * 128), 5.0, dtype=F16, device="cuda")
        b.run(max_new=cut, out=out)
        want, tol = b.exact()
        for i, (_, n) in enumerate(seqs):
            at = slice(b.cu[i], b.cu[i] + min(n, cut))
            assert ((out[at].double() - want[at]).abs() <= tol[at] + U[F16] * want[at].abs() + 2.0 ** -24).all()
            assert (out[b.cu[i] + min(n, cut):b.cu[i + 1]] == 5).all()
        assert torch.equal(b.run(), whole)


def test_attn_captured_chunks_replay_with_new_lengths(cuda):
    """A captured call with prompt chunks follows the lengths, offsets and tables that it finds when it runs; eager calls of
    the same kind run between the replays."""
    from yllm_amd.paged import paged_attn8, paged_attn8_workspace

    steps = [Batch8(s, 28, 4, 128, seed=30 + i) for i, s in enumerate(
        ([(700, 200), (90, 1), (3000, 33)], [(1, 1), (0, 0), (233, 233)], [(5000, 1), (64, 64), (129, 128)],
         [(2, 2), (1, 1), (1, 1)], [(400, 100), (2000, 130), (77, 4)]))]
    T, w, nb = max(b.T for b in steps), max(b.table.shape[1] for b in steps), max(b.cache.n_blocks for b in steps)
    pool = pool8(nb, 4, 128, 64)
    q, out = torch.zeros((T, 28 * 128), dtype=F16, device="cuda"), torch.empty((T, 28 * 128), dtype=F16, device="cuda")
    table, lens, cu = torch.zeros((3, w), dtype=torch.int32, device="cuda"), _i32([1, 1, 1]), _i32([0, 1, 2, 3])
    ws = paged_attn8_workspace(T, 3, 233, 5000, 28, 4, 128)
    paged_attn8(q, pool, table, lens, cu, 28, 233, 5000, out=out, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_attn8(q, pool, table, lens, cu, 28, 233, 5000, out=out, workspace=ws)
    for b in steps * 2:
        q[:b.T], out[:] = b.q, 5.0
        for x, y in ((pool.k, b.cache.k), (pool.v, b.cache.v), (pool.k_scale, b.cache.k_scale), (pool.v_scale, b.cache.v_scale)):
            x.view(U8)[:b.cache.n_blocks] = y.view(U8)
        table[:, :b.table.shape[1]] = b.table
        lens.copy_(_i32([L for L, _ in b.seqs])), cu.copy_(_i32(b.cu))
        graph.replay()
        want, tol = b.exact()
        err = (out[:b.T].double() - want).abs()
        assert (err <= tol + U[F16] * want.abs() + 2.0 ** -24).all() and (out[b.T:] == 5).all()
        b.check()


@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (32, 8, 128), (16, 2, 256)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("few,chunks", [(40, 0), (0, 5), (1, 9), (90, 1), (64, 1), (200, 6), (7, 2)])
def test_attn_few_rows_beside_chunks(cuda, nh, nkv, d, dtype, few, chunks):
    """One launch for both kinds of sequences, from all of one to all of the other, under bounds that let every one be a
    chunk; a workspace with anything in it; a gate; empty sequences between."""
    from yllm_amd.paged import paged_attn8_workspace

    seqs = [(1 + 37 * i * i % 2900, 1 + i % 2) for i in range(few)]
    seqs = [(max(L, n), n) for L, n in seqs]
    for i in range(chunks):
        seqs.insert(i * len(seqs) // chunks, (300 + 411 * i, (300, 40, 129)[i % 3]))
    seqs.insert(len(seqs) // 2, (0, 0))
    seqs.insert(0, (50, 0))
    b = Batch8(seqs, nh, nkv, d, dtype=dtype, seed=few + chunks, gated=few % 2 == 1, behind=2, spread=4.0)
    bound = min(512, b.T)
    ws = paged_attn8_workspace(b.T, len(seqs), bound, b.max_len, nh, nkv, d)
    n = b.cu[-1]  # (rows behind the last sequence are not written)
    out = b.check(max_new=bound, workspace=ws)[:n]
    for fill in (0, 0xff, 0x01):
        ws.fill_(fill)
        assert torch.equal(b.run(max_new=bound, workspace=ws)[:n], out)


@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128)])
def test_attn_long_contexts_beside_chunks(cuda, nh, nkv, d):
    """Pieces of both lines joined; twice the same bits."""
    for seqs in ([(60000, 1), (40000, 300), (9, 3)], [(9000, 200)] + [(30000 + 77 * i, 2) for i in range(9)]):
        b = Batch8(seqs, nh, nkv, d, dtype=BF16, seed=51)
        assert torch.equal(b.check(), b.run())


@pytest.mark.parametrize("nh,nkv,d", [(3, 2, 64), (28, 4, 128), (5, 3, 128), (16, 2, 256)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("L,new", [(0, 0), (50, 10), (300, 1), (130, 130), (129, 129), (700, 127), (640, 200), (90, 150)])
def test_attn_one_sequence_below_its_bounds(cuda, nh, nkv, d, dtype, L, new):
    """A launch sized for 200 tokens and 700 keys, as a captured one is, with fewer of either."""
    b = Batch8([(L, new)], nh, nkv, d, dtype=dtype, seed=60, behind=200 - new)
    out = torch.full((200, nh * d), 5.0, dtype=dtype, device="cuda")
    if b.table.shape[1] * 64 < 700:
        b.table = torch.cat([b.table, torch.full((1, 11 - b.table.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    b.check(max_new=200, max_len=700, out=out)
    assert (out[new:] == 5).all()


@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (28, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("n_seq", [1, 9])
@pytest.mark.parametrize("new", [1, 2])
def test_attn_contexts_about_the_longest_that_is_not_cut(cuda, nh, nkv, d, n_seq, new):
    for whole in (65536 // d, 131072 // d):
        for L in (whole - 256, whole - 1, whole, whole + 1, whole + 257):
            b = Batch8([(max(new, L - 37 * i), new) for i in range(n_seq)], nh, nkv, d, dtype=(F16, F32)[L % 2], seed=L)
            b.check()
            b.check(max_len=b.table.shape[1] * 64)  # under another bound, on either side of that length, the same rows


@pytest.mark.parametrize("nh,nkv,d", [(32, 8, 64), (16, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n_seq,L,new", [(1, 131072, 2048), (72, 32768, 1)])
def test_attn_many_small_probabilities(cuda, nh, nkv, d, dtype, n_seq, L, new):
    """One key far above all others, which are so many that they count all the same (as the f16 pool's test)."""
    from yllm_amd.paged import paged_attn8

    c = {64: 2.25, 128: 1.625, 256: 1.25}[d]  # e4m3 numbers near 19 / sqrt(d)
    s = c * math.sqrt(d)
    pages = L // 1024
    pool = pool8(pages, nkv, d, 1024, fill=0)
    pool.k_scale.view(U8).fill_(0x3c), pool.v_scale.view(U8).fill_(0x3c)
    pool.v.view(U8).fill_(0x38)
    pool.k.view(U8)[0, :, 0] = int(torch.tensor(c).to(E4M3).view(U8))
    pool.v.view(U8)[0, :, 0, :, 0] = 0
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(n_seq, pages).contiguous()
    q = torch.ones((n_seq * new, nh * d), dtype=dtype, device="cuda")
    got = paged_attn8(q, pool, table, _i32([L] * n_seq), _i32([i * new for i in range(n_seq + 1)]), nh, new, L, out_dtype=F32)
    p = torch.arange(L - new, L, device="cuda").double().repeat(n_seq)
    w = p * math.exp(-s)
    want = (w / (1 + w))[:, None]
    # a probability: half a step of f16 (of a hi and lo pair, 2^-22), or, below the f16 normals, half of 2^-24 times the
    # 2^-7 by which the largest is scaled up; the score's sum and exp2: 2^-24 of s <= 20 three times, its sums 2^-20
    u = 2.0 ** -22 if dtype == F32 else 2.0 ** -11
    tol = want * (u + 2.0 ** -20 + 3 * 20 * 2.0 ** -24) + p[:, None] * 2.0 ** -32 + want * 2.0 ** -24
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (float(err.max()), float((err / tol).max()), float(want.max()))


# ---- a step, and steps in a row ---------------------------------------------------------------------------

class Serve8:
    """Two layers of serving over 8-bit pages, step by step; the oracle attends in 64 bits to its own quantised rows."""

    def __init__(self, n_seq, nh, nkv, d, block, kind, dtype, n_blocks, width, seed=0):
        self.__dict__.update(nh=nh, nkv=nkv, d=d, block=block, kind=kind, dtype=dtype, n=n_seq)
        self.layers = [pool8(n_blocks, nkv, d, block) for _ in range(2)]
        g = self.g = _gen(seed)
        self.w = [(1 + 0.1 * torch.randn(d, generator=g, device="cuda"), 1 + 0.1 * torch.randn(d, generator=g, device="cuda"))
                  for _ in range(2)]
        self.table = torch.full((n_seq, width), -1, dtype=torch.int32, device="cuda")
        self.ctx = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        self.free, self.n_free = torch.arange(n_blocks, dtype=torch.int32, device="cuda").flip(0).contiguous(), _i32([n_blocks])

    def rows(self, T):
        return [torch.randn(T, (self.nh + 2 * self.nkv) * self.d, generator=self.g, device="cuda").to(self.dtype) for _ in range(2)]

    def step(self, new, rows, n_tok, max_new, max_len):
        from yllm_amd import paged as P

        p = P.paged_plan(self.table, self.ctx, new, self.free, self.n_free, self.block, n_tok)
        out, qs, qd, kd = [], [], self.nh * self.d, self.nkv * self.d
        for layer, x, (wq, wk) in zip(self.layers, rows, self.w):
            q = torch.zeros(n_tok, qd, dtype=self.dtype, device="cuda")
            P.qk_norm_rope_kv8_store(layer, x[:, :qd], x[:, qd:qd + kd], x[:, qd + kd:], self.nh, KINDS[self.kind], 1e6, 64,
                                     positions=p.positions, slots=p.slots, q_norm=wq, k_norm=wk, q_out=q)
            o = torch.zeros(n_tok, qd, dtype=self.dtype, device="cuda")
            out.append(P.paged_attn8(q, layer, p.block_table, p.kv_lens, p.cu_new, self.nh, max_new, max_len, out=o))
            qs.append(q)
        self.ctx.copy_(torch.where(p.kv_lens > 0, p.kv_lens, self.ctx))
        self.n_free.copy_(p.counts[:1])
        return out, qs

    def hold(self, new, rows, out, qs):
        """The step's stored rows against the rows themselves, its outputs against attention over what is held."""
        ctx, table = self.ctx.tolist(), self.table.tolist()
        for layer, x, (wq, wk), o, q in zip(self.layers, rows, self.w, out, qs):
            K, V, KS, VS = rows_of_pool(layer)
            at = 0
            for i, n in enumerate(new):
                if n == 0:
                    continue
                L = ctx[i]
                slot = torch.tensor([table[i][p // self.block] * self.block + p % self.block for p in range(L)], device="cuda")
                k, v = values(K[slot], KS[slot]), values(V[slot], VS[slot])
                y = x[at:at + n].double().view(n, -1, self.d)
                pos = torch.arange(L - n, L, device="cuda")
                want, tol = rope_oracle(y[:, self.nh:self.nh + self.nkv], pos, wk.double(), 1e-6, self.kind, 64, 1e6)
                half = torch.maximum((want.abs() + tol) * 2.0 ** -4, 2.0 ** -10 * KS[slot[L - n:]].view(E5M2).double()[..., None])
                assert ((k[L - n:] - want).abs() <= half + tol).all()
                code, scale = quantise(y[:, self.nh + self.nkv:])
                assert torch.equal(v[L - n:], code * scale[..., None])
                qq = q[at:at + n].double().view(n, self.nh, self.d)
                hide = torch.arange(L, device="cuda")[None, :] > pos[:, None]
                got = o[at:at + n].double().view(n, self.nh, self.d)
                for h in range(self.nh):
                    kk, vv = k[:, h * self.nkv // self.nh], v[:, h * self.nkv // self.nh]
                    p = (qq[:, h] @ kk.t() / math.sqrt(self.d)).masked_fill(hide, -math.inf).softmax(-1)
                    ref = p @ vv
                    size = (qq[:, h].abs() @ kk.abs().t() / math.sqrt(self.d)).amax(-1, keepdim=True)
                    u_p = 2.0 ** -22 if self.dtype == F32 else 2.0 ** -11
                    t = (p @ vv.abs()) * (2 * self.d * 2.0 ** -24 * size + u_p + 2.0 ** -20)
                    assert ((got[:, h] - ref).abs() <= t + U[self.dtype] * ref.abs() + 2.0 ** -24).all()
                at += n


@pytest.mark.parametrize("nh,nkv,d,kind,dtype", [(14, 2, 64, "half", BF16), (8, 2, 128, "pairs", F16), (16, 2, 256, "mrope", F32)])
def test_serving_steps(cuda, nh, nkv, d, kind, dtype):
    """Prompts in chunks, then decode tokens, with sequences that join and pause: every step's rows and attention."""
    s = Serve8(4, nh, nkv, d, 64, kind, dtype, n_blocks=40, width=8)
    for new in ([70, 0, 33, 1], [130, 64, 1, 1], [1, 1, 1, 1], [1, 200, 0, 1], [5, 1, 1, 3], [1, 1, 1, 1]):
        T = sum(new)
        rows = s.rows(T + 3)
        out, qs = s.step(_i32(new), rows, T + 3, max(new), 500)
        s.hold(new, rows, out, qs)
        assert all((o[T:] == 0).all() for o in out)
    assert int(s.n_free) == 40 - sum(-(-int(c) // 64) for c in s.ctx)


def test_serving_step_captured_and_replayed(cuda):
    """One captured decode step replays with the lengths, tables and free blocks that the replays themselves change,
    between eager work of the same kind."""
    s = Serve8(3, 8, 2, 128, 64, "half", BF16, n_blocks=24, width=6)
    prompt = [100, 63, 20]
    rows = s.rows(sum(prompt))
    s.hold(prompt, rows, *s.step(_i32(prompt), rows, 183, 100, 384))
    new, static = _i32([1, 1, 1]), s.rows(3)
    pools = [t.view(U8) for l in s.layers for t in (l.k, l.v, l.k_scale, l.v_scale)]
    keep = (s.ctx.clone(), s.n_free.clone(), s.table.clone(), [t.clone() for t in pools])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a first pass outside the capture
        s.step(new, static, 3, 1, 384)
    torch.cuda.current_stream().wait_stream(side)
    s.ctx.copy_(keep[0]), s.n_free.copy_(keep[1]), s.table.copy_(keep[2])
    for t, k in zip(pools, keep[3]):
        t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, qs = s.step(new, static, 3, 1, 384)
    for i in range(5):
        fresh = s.rows(3)
        for a, b in zip(static, fresh):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        s.hold([1, 1, 1], fresh, out, qs)
        if i == 2:  # an eager step in between
            rows = s.rows(40)
            s.hold([0, 39, 1], rows, *s.step(_i32([0, 39, 1]), rows, 40, 39, 384))


def test_a_prompt_on_f16_pages_goes_on_in_8_bits(cuda):
    """A prompt through the f16 operators, its pages converted, decode steps over the 8-bit pool."""
    from yllm_amd import paged as P

    nh, nkv, d, T = 8, 2, 128, 200
    half, g = P.PagedKV.empty(8, nkv, d), _gen(5)
    s = Serve8(1, nh, nkv, d, 64, "half", F16, n_blocks=8, width=6)
    plan = P.paged_plan(s.table, s.ctx, _i32([T]), s.free, s.n_free, 64, T)
    wq, wk = s.w[0]
    x = torch.randn(T, (nh + 2 * nkv) * d, generator=g, device="cuda").half()
    q, k, v = x[:, :nh * d], x[:, nh * d:(nh + nkv) * d], x[:, (nh + nkv) * d:]
    P.qk_norm_rope_kv_store(half, q, k, v, nh, KINDS["half"], 1e6, positions=plan.positions, slots=plan.slots, q_norm=wq, k_norm=wk)
    used = s.table[0, :4].contiguous()
    for layer in s.layers:
        P.kv8_from_pages(layer, half, used, used)
    s.ctx.copy_(plan.kv_lens)
    s.n_free.copy_(plan.counts[:1])
    for _ in range(3):
        rows = s.rows(1)
        s.hold([1], rows, *s.step(_i32([1]), rows, 1, 1, 384))
