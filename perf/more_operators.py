"""The operators of serving over a paged KV cache held in 8 bits: codes in e4m3, and a scale, a power of two in e5m2, for
each position and kv head of K and of V.

Kinds:

  store  RMSNorm of every query and key head, the position rotation, and the quantised store of K and V into
         the pages, in one pass over the projected rows (qk_norm_rope_kv8_store)
  attn   attention of each sequence's new tokens over its pages (paged_attn8): decode tokens, drafted tokens
         being checked, chunks of a prompt, whole prompts, and batches of all of them
  pages  pages of an f16 pool into the 8-bit pool (kv8_from_pages) and back (kv8_to_pages)

A pool holds pages of `block` positions: codes K [n_blocks, n_kv, block, d] and V [n_blocks, n_kv, block/64, d, 64],
scales [n_blocks, n_kv, block]; the f16 pool is that of perf/operators.py.  With amax the largest magnitude of a
position's head, k = ceil(log2(amax / 448)) within -14..7, the scale is 2^k and a code is x / 2^k in e4m3, to nearest
even.  A case's lengths follow from its numbers alone; its values, and which pages a sequence has, from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3, E5M2, U8 = torch.float8_e4m3fn, torch.float8_e5m2, torch.uint8
# (query heads, kv heads, head_dim, rope, theta): the head layouts of the benchmark's configurations
HEADS = [(14, 2, 64, "half", 1e6), (28, 4, 128, "half", 1e6), (32, 8, 128, "pairs", 5e5), (16, 2, 256, "mrope", 1e7)]
N_ROT = 64  # rotated dimensions of a qwen35 head
EPS = 1e-6


def _h(i: int) -> dict:
    nh, nkv, d, rope, theta = HEADS[i]
    return {"nh": nh, "nkv": nkv, "d": d, "rope": rope, "theta": theta}


def listed() -> list[dict]:
    return [
        # one decode token of a qwen35 attention layer: the smallest store
        {"name": "store_token", "kind": "store", **_h(3), "n_seq": 1, "lo": 2501, "hi": 2501, "chunks": 0, "new": 1, "block": 64, "dtype": "f32", "out": "f32"},
        # the decode tokens of 64 sequences
        {"name": "store_decode_64", "kind": "store", **_h(2), "n_seq": 64, "lo": 1024, "hi": 32768, "chunks": 0, "new": 1, "block": 64, "dtype": "bf16", "out": "bf16"},
        # four chunks of a prompt and decode tokens, fp32 rows as the engine holds them
        {"name": "store_mixed_f32", "kind": "store", **_h(1), "n_seq": 32, "lo": 300, "hi": 8192, "chunks": 4, "new": 512, "block": 128, "dtype": "f32", "out": "f16"},
        # whole prompts of about 8192 tokens in all
        {"name": "store_prompts_8k", "kind": "store", **_h(3), "n_seq": 3, "lo": 2700, "hi": 2760, "chunks": 3, "new": 2731, "block": 64, "dtype": "bf16", "out": "bf16"},
        # one decode token of the smallest model over a short context: latency
        {"name": "attn_token_500", "kind": "attn", **_h(0), "n_seq": 1, "lo": 500, "hi": 500, "chunks": 0, "new": 1, "block": 64, "dtype": "f32", "gated": False},
        # decode deep into one long context
        {"name": "attn_token_128k", "kind": "attn", **_h(2), "n_seq": 1, "lo": 131072, "hi": 131072, "chunks": 0, "new": 1, "block": 256, "dtype": "f16", "gated": False},
        # serving: one token each of 64 sequences between 1k and 32k
        {"name": "attn_decode_64", "kind": "attn", **_h(2), "n_seq": 64, "lo": 1024, "hi": 32768, "chunks": 0, "new": 1, "block": 64, "dtype": "bf16", "gated": False},
        # a mixed step: four chunks of a prompt among decode tokens
        {"name": "attn_mixed_32", "kind": "attn", **_h(1), "n_seq": 32, "lo": 300, "hi": 8192, "chunks": 4, "new": 512, "block": 128, "dtype": "bf16", "gated": False},
        # the second half of a 4096-token prompt through the qwen35 gated attention
        {"name": "attn_gated_chunk", "kind": "attn", **_h(3), "n_seq": 1, "lo": 4096, "hi": 4096, "chunks": 1, "new": 2048, "block": 64, "dtype": "bf16", "gated": True},
        # a whole long prompt
        {"name": "attn_prompt_8k", "kind": "attn", **_h(2), "n_seq": 1, "lo": 8192, "hi": 8192, "chunks": 1, "new": 8192, "block": 64, "dtype": "f16", "gated": False},
        # a prompt of 8192 tokens, computed on f16 pages, kept in 8 bits
        {"name": "pages_in_8k", "kind": "pages", **_h(2), "pages": 128, "block": 64, "to": "e4m3"},
        # a short sequence handed out in f16: latency
        {"name": "pages_out_3", "kind": "pages", **_h(3), "pages": 3, "block": 64, "to": "f16"},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["store", "store", "attn", "attn", "attn", "pages"])
    block = rng.choice([64, 64, 128, 256])
    h = _h(rng.randrange(len(HEADS)))
    if kind == "pages":
        return {"kind": kind, **h, "pages": _log(rng, 1, 16384 // block), "block": block, "to": rng.choice(["e4m3", "f16"])}
    if kind == "store":
        n = _log(rng, 1, 64)
        chunks = rng.choice([0, 1, _log(rng, 1, 8)])
        hi = _log(rng, 64, 32768)
        return {"kind": kind, **h, "n_seq": n, "lo": max(1, hi // 32), "hi": hi, "chunks": min(n, chunks),
                "new": 1 if chunks == 0 else _log(rng, 2, 1024), "block": block,
                "dtype": rng.choice(["f32", "f16", "bf16"]), "out": rng.choice(["f32", "f16", "bf16"])}
    dtype = rng.choice(["f32", "f16", "bf16"])
    form = rng.choice(["one", "batch", "chunk", "mixed"])
    gated = h["d"] == 256
    if form == "one":
        hi = _log(rng, 1, 131072)
        n, lo, chunks, new = 1, hi, 0, 1
    elif form == "batch":  # one to four tokens of each sequence (several: drafted tokens being checked)
        n, hi, new = _log(rng, 2, 48), _log(rng, 64, 32768), rng.choice([1, 1, 2, 4])
        lo, chunks = max(1, hi // 32), n if new > 1 else 0
    elif form == "chunk":
        new = _log(rng, 2, 4096)
        n, hi, chunks = 1, new + rng.choice([0, _log(rng, 1, 4096)]), 1
        lo = hi
    else:
        n, hi, new = _log(rng, 2, 24), _log(rng, 256, 6144), _log(rng, 2, 512)
        lo, chunks = max(1, hi // 32), min(n, _log(rng, 1, 6))
    return {"kind": kind, **h, "n_seq": n, "lo": lo, "hi": hi, "chunks": chunks, "new": new, "block": block,
            "dtype": dtype, "gated": gated}


# ---- inputs ------------------------------------------------------------------------------------

def _lengths(c: dict) -> list[tuple[int, int]]:
    """(tokens after the step, new tokens) of every sequence: lengths spread evenly over their logarithm
    between lo and hi, and `chunks` sequences, spread over the batch, with up to `new` tokens, no two alike
    (a whole prompt where the sequence is no longer than that)."""
    n, chunks, got = c["n_seq"], c["chunks"], []
    for i in range(n):
        u = (0.5 + i * 0.6180339887498949) % 1.0
        L = min(c["hi"], max(c["lo"], round(c["lo"] * (c["hi"] / c["lo"]) ** u)))
        chunk = chunks and i * chunks // n != (i - 1) * chunks // n
        got.append((L, min(L, max(1, c["new"] - (i * chunks // n if c["new"] > 8 else 0)) if chunk else 1)))
    return got


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, scale: float = 1.0) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _i32(v) -> torch.Tensor:
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _empty(nb: int, nkv: int, B: int, d: int) -> dict:
    z = lambda *shape: torch.zeros(shape, dtype=U8, device="cuda")  # noqa: E731
    return {"k": z(nb, nkv, B, d).view(E4M3), "v": z(nb, nkv, B // 64, d, 64).view(E4M3),
            "ks": z(nb, nkv, B).view(E5M2), "vs": z(nb, nkv, B).view(E5M2)}


def _held(g, nb: int, nkv: int, B: int, d: int) -> dict:
    """A pool in use: normal values of scale 1 with a few strong key channels, as a store leaves them."""
    k = torch.randn((nb, nkv, B, d), generator=g, device="cuda", dtype=torch.float16)
    k[..., 5::29] *= 4.0
    v = torch.randn((nb, nkv, B // 64, 64, d), generator=g, device="cuda", dtype=torch.float16)
    s = _empty(nb, nkv, B, d)
    step = max(1, (1 << 28) // (nkv * B * d))  # pages at a time
    for a in range(0, nb, step):
        e = slice(a, a + step)
        code, scale = _quantise(k[e].float())
        s["k"].view(U8)[e], s["ks"].view(U8)[e] = code.view(U8), scale.view(U8)
        code, scale = _quantise(v[e].float())
        s["v"].view(U8)[e] = code.view(U8).transpose(-1, -2)
        s["vs"].view(U8)[e] = scale.view(U8).flatten(-2)
    return s


def prepare(case: dict, seed: int) -> dict:
    c, g, B = case, _gen(seed), case["block"]
    nh, nkv, d = c["nh"], c["nkv"], c["d"]
    if c["kind"] == "pages":
        n = c["pages"]
        src, dst = (torch.randperm(n + 5, generator=g, device="cuda")[:n].int() for _ in range(2))
        s = {"c": c, "src": src, "dst": dst}
        if c["to"] == "f16":
            s.update(_held(g, n + 5, nkv, B, d))
            s["k16"] = torch.zeros((n + 5, nkv, B, d), dtype=torch.float16, device="cuda")
            s["v16"] = torch.zeros((n + 5, nkv, B // 32, d, 32), dtype=torch.float16, device="cuda")
        else:
            s.update(_empty(n + 5, nkv, B, d))
            s["k16"] = torch.randn((n + 5, nkv, B, d), generator=g, device="cuda", dtype=torch.float16)
            s["k16"][..., 5::29] *= 4.0
            s["v16"] = torch.randn((n + 5, nkv, B // 32, d, 32), generator=g, device="cuda", dtype=torch.float16)
        return s
    lens = _lengths(c)
    n, T = len(lens), sum(m for _, m in lens)
    most = max(-(-L // B) for L, _ in lens)
    s = {"c": c, "T": T, "max_len": max(L for L, _ in lens), "max_new": max(m for _, m in lens)}
    total = _i32([L for L, _ in lens])
    new = _i32([m for _, m in lens])
    # the pages of every sequence, anywhere in the pool
    free = sum(-(-L // B) for L, _ in lens) + 8
    order = torch.randperm(free, generator=g, device="cuda").int()
    held = (total + B - 1).div(B, rounding_mode="floor")
    if c["kind"] == "store":
        seq = torch.repeat_interleave(torch.arange(n, device="cuda"), new.long(), output_size=T)
        cu = new.cumsum(0) - new
        pos = ((total - new)[seq] + torch.arange(T, device="cuda") - cu[seq]).int()
        # the pool of the pages that this step writes: each sequence's last ones
        lo = (total - new).div(B, rounding_mode="floor")
        used = held - lo
        page = torch.randperm(int(used.sum()), generator=g, device="cuda").int()
        slot = page[(used.cumsum(0) - used)[seq] + pos // B - lo[seq]] * B + pos % B
        s["n_blocks"] = page.numel()
        s.update(pos=pos, slot=slot.int(), qkv=_normal(g, T, (nh + 2 * nkv) * d).to(DTYPES[c["dtype"]]),
                 q_norm=1.0 + _normal(g, d, scale=0.1), k_norm=1.0 + _normal(g, d, scale=0.1),
                 q=torch.empty((T, nh * d), dtype=DTYPES[c["out"]], device="cuda"), **_empty(page.numel(), nkv, B, d))
        return s
    first = held.cumsum(0) - held
    at = torch.arange(most, device="cuda")[None, :]
    table = torch.where(at < held[:, None], order[(first[:, None] + at).clamp(max=free - 1)], -1).int()
    dt = DTYPES[c["dtype"]]
    s.update(table=table, lens=total, cu=torch.cat([_i32([0]), new.cumsum(0).int()]), **_held(g, free, nkv, B, d),
             q=_normal(g, T, nh * d).to(dt), gate=_normal(g, T, nh * d) if c["gated"] else None,
             out=torch.empty((T, nh * d), dtype=dt, device="cuda"))
    return s


# ---- one pass ----------------------------------------------------------------------------------

def _own(s: dict):
    from yllm_amd import attention as A
    from yllm_amd import paged as P

    c = s["c"]
    cache = P.PagedKV8(s["k"], s["v"], s["ks"], s["vs"])
    if c["kind"] == "pages":
        half = P.PagedKV(s["k16"], s["v16"])
        if c["to"] == "f16":
            P.kv8_to_pages(half, cache, s["dst"], s["src"])
            return {"k": s["k16"], "v": s["v16"]}
        P.kv8_from_pages(cache, half, s["dst"], s["src"])
        return {"k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}
    if c["kind"] == "store":
        rope = {"half": A.ROPE_HALF, "pairs": A.ROPE_PAIRS, "mrope": A.ROPE_MROPE}[c["rope"]]
        kd, qd = c["nkv"] * c["d"], c["nh"] * c["d"]
        q, k, v = s["qkv"][:, :qd], s["qkv"][:, qd:qd + kd], s["qkv"][:, qd + kd:]
        P.qk_norm_rope_kv8_store(cache, q, k, v, c["nh"], rope, c["theta"], N_ROT if c["rope"] == "mrope" else 0,
                                 positions=s["pos"], slots=s["slot"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                                 eps=EPS, q_out=s["q"])
        return {"q": s["q"], "k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}
    if "ws" not in s:  # a program keeps one workspace for all its layers
        s["ws"] = P.paged_attn8_workspace(s["T"], c["n_seq"], s["max_new"], s["max_len"], c["nh"], c["nkv"], c["d"])
    return P.paged_attn8(s["q"], cache, s["table"], s["lens"], s["cu"], c["nh"], s["max_new"], s["max_len"],
                         gate=s["gate"], out=s["out"], workspace=s["ws"])


def run(s: dict):
    if own:
        return _own(s)
    return {"store": _store, "attn": _attn, "pages": _pages}[s["c"]["kind"]](s)


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of rows of fp32 values (the last dimension is a head)."""
    top = x.abs().amax(-1)
    m, e = torch.frexp(top.double() / 448.0)  # amax / 448 = m 2^e, m in [1/2, 1)
    k = torch.where(top > 0, torch.where(m > 0.5, e, e - 1), -14).clamp(-14, 7)
    scale = torch.ldexp(torch.ones_like(top), k)
    return (x / scale[..., None]).clamp(-448.0, 448.0).to(E4M3), scale.to(E5M2)


def _turn(x: torch.Tensor, cs: torch.Tensor, sn: torch.Tensor, rope: str, span: int) -> torch.Tensor:
    if rope == "pairs":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cs - b * sn, a * sn + b * cs], -1).flatten(-2)
    a, b = x[..., :span // 2], x[..., span // 2:span]
    return torch.cat([a * cs - b * sn, a * sn + b * cs, x[..., span:]], -1)


def _store(s: dict) -> dict:
    c, T, B = s["c"], s["T"], s["c"]["block"]
    nh, nkv, d = c["nh"], c["nkv"], c["d"]
    span = N_ROT if c["rope"] == "mrope" else d
    x = s["qkv"].float().view(T, nh + 2 * nkv, d)
    q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
    q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"]
    k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"]
    freq = c["theta"] ** (-2.0 * torch.arange(span // 2, dtype=torch.float64, device=x.device) / span)
    ang = s["pos"].double()[:, None] * freq
    cs, sn = ang.cos().float()[:, None, :], ang.sin().float()[:, None, :]
    s["q"].copy_(_turn(q, cs, sn, c["rope"], span).reshape(T, nh * d))
    page, off = torch.div(s["slot"], B, rounding_mode="floor").long(), (s["slot"] % B).long()
    code, scale = _quantise(_turn(k, cs, sn, c["rope"], span))
    s["k"].view(U8)[page, :, off], s["ks"].view(U8)[page, :, off] = code.view(U8), scale.view(U8)
    code, scale = _quantise(v)
    s["v"].view(U8)[page, :, off // 64, :, off % 64] = code.view(U8)
    s["vs"].view(U8)[page, :, off] = scale.view(U8)
    return {"q": s["q"], "k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}


def _attn(s: dict) -> torch.Tensor:
    """Every sequence padded to the longest context and the largest chunk."""
    c, T, M, L = s["c"], s["T"], s["max_new"], s["max_len"]
    nh, nkv, d, B = c["nh"], c["nkv"], c["d"], c["block"]
    G, n, dev = nh // nkv, s["table"].shape[0], s["q"].device
    at = torch.arange(L, device=dev)
    page, off = s["table"][:, at // B].clamp(min=0).long(), (at % B)[None, :]
    k = s["k"].view(U8)[page, :, off].view(E4M3).float()                                      # [n, L, n_kv, d]
    k *= s["ks"].view(U8)[page, :, off].view(E5M2).float()[..., None]
    v = s["v"].view(U8)[page, :, off // 64, :, off % 64].view(E4M3).float()
    v *= s["vs"].view(U8)[page, :, off].view(E5M2).float()[..., None]
    k, v = k.permute(0, 2, 3, 1), v.permute(0, 2, 1, 3)                                       # [n, n_kv, d, L], [n, n_kv, L, d]
    cu, lens = s["cu"].long(), s["lens"].long()
    new, t = cu[1:] - cu[:-1], torch.arange(M, device=dev)
    row = (cu[:-1, None] + t).clamp(max=T - 1)
    q = s["q"].float().view(T, nkv, G, d)[row].permute(0, 2, 3, 1, 4).reshape(n, nkv, G * M, d)
    p = torch.matmul(q, k).view(n, nkv, G, M, L)
    p *= 1.0 / math.sqrt(d)
    seen = at[None, None, :] <= ((lens - new)[:, None] + t)[..., None]                        # [n, M, L]
    p.masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p -= torch.where(top.isinf(), 0.0, top)
    p.exp_()
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, nkv, G * M, L), v).view(n, nkv, G, M, d) / torch.where(z == 0, 1.0, z)
    rows = torch.arange(T, device=dev)
    seq = torch.searchsorted(cu[1:], rows, right=True)
    o = o[seq, :, :, rows - cu[seq]].reshape(T, nh * d)
    if s["gate"] is not None:
        o *= 1.0 / (1.0 + torch.exp(-s["gate"]))
    return s["out"].copy_(o)


def _pages(s: dict) -> dict:
    c, src, dst = s["c"], s["src"].long(), s["dst"].long()
    n, nkv, d, B = c["pages"], c["nkv"], c["d"], c["block"]
    if c["to"] == "f16":
        k = s["k"].view(U8)[src].view(E4M3).float() * s["ks"].view(U8)[src].view(E5M2).float()[..., None]
        v = s["v"].view(U8)[src].view(E4M3).float() * s["vs"].view(U8)[src].view(E5M2).float().view(n, nkv, B // 64, 1, 64)
        s["k16"][dst] = k.half()
        s["v16"][dst] = v.view(n, nkv, B // 64, d, 2, 32).transpose(3, 4).reshape(n, nkv, B // 32, d, 32).half()
        return {"k": s["k16"], "v": s["v16"]}
    code, scale = _quantise(s["k16"][src].float())
    s["k"].view(U8)[dst], s["ks"].view(U8)[dst] = code.view(U8), scale.view(U8)
    code, scale = _quantise(s["v16"][src].float().transpose(-1, -2).reshape(n, nkv, B, d))
    s["v"].view(U8)[dst] = code.view(U8).view(n, nkv, B // 64, 64, d).transpose(-1, -2)
    s["vs"].view(U8)[dst] = scale.view(U8)
    return {"k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case: dict) -> dict:
    c, B = case, case["block"]
    nh, nkv, d = c["nh"], c["nkv"], c["d"]
    if c["kind"] == "pages":
        values = 2 * c["pages"] * nkv * B * d
        return {"bytes": 3 * values + values // d + 8 * c["pages"], "flops": (3 if c["to"] == "e4m3" else 1) * values}
    lens = _lengths(case)
    T = sum(m for _, m in lens)
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["kind"] == "store":
        span = N_ROT if c["rope"] == "mrope" else d
        return {"bytes": T * ((nh + 2 * nkv) * d * size[c["dtype"]] + nh * d * size[c["out"]] + 2 * nkv * (d + 1) + 8) + 8 * d,
                "flops": T * ((nh + nkv) * (4 * d + 3 * span) + 6 * nkv * d)}
    keys = sum(L for L, _ in lens)
    pairs = sum(m * (L - m) + m * (m + 1) // 2 for L, m in lens)
    return {"bytes": 2 * keys * nkv * (d + 1) + T * nh * d * (2 * size[c["dtype"]] + (4 if c["gated"] else 0))
            + 4 * sum(-(-L // B) for L, _ in lens) + 8 * len(lens),
            "flops": 4 * pairs * nh * d}


# ---- the same in 64 bits -------------------------------------------------------------------------

def _codes64(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales as numbers: of the candidates 2^k the smallest whose largest code holds the row, and
    of the steps 2^max(exponent - 3, -9) the nearest multiple, ties to even."""
    top, scale = x.abs().amax(-1), torch.full(x.shape[:-1], 2.0 ** 7, dtype=torch.float64, device=x.device)
    for k in range(6, -15, -1):
        scale = torch.where(top <= 448.0 * 2.0 ** k, 2.0 ** k, scale)
    y = (x / scale[..., None]).clamp(-448.0, 448.0)
    step = torch.full_like(y, 2.0 ** -9)
    for e in range(-5, 9):
        step = torch.where(y.abs() >= 2.0 ** e, 2.0 ** (e - 3), step)
    return (y / step).round() * step, scale


def exact(case: dict, seed: int):
    c = case
    s = prepare(case, seed)
    nh, nkv, d, B = c["nh"], c["nkv"], c["d"], c["block"]
    if c["kind"] == "pages":
        n, nb, src, dst = c["pages"], c["pages"] + 5, s["src"].tolist(), s["dst"].tolist()
        if c["to"] == "f16":
            K = torch.zeros((nb, nkv, B, d), dtype=torch.float64, device="cuda")
            V = torch.zeros((nb, nkv, B // 32, d, 32), dtype=torch.float64, device="cuda")
            for i in range(n):
                K[dst[i]] = s["k"][src[i]].double() * s["ks"][src[i]].double()[..., None]
                x = s["v"][src[i]].double().permute(0, 1, 3, 2).reshape(nkv, B, d) * s["vs"][src[i]].double()[..., None]
                V[dst[i]] = x.reshape(nkv, B // 32, 32, d).permute(0, 1, 3, 2)
            return {"k": K, "v": V}
        K = torch.zeros((nb, nkv, B, d), dtype=torch.float64, device="cuda")
        V = torch.zeros((nb, nkv, B // 64, d, 64), dtype=torch.float64, device="cuda")
        KS, VS = (torch.zeros((nb, nkv, B), dtype=torch.float64, device="cuda") for _ in range(2))
        for i in range(n):
            K[dst[i]], KS[dst[i]] = _codes64(s["k16"][src[i]].double())
            code, VS[dst[i]] = _codes64(s["v16"][src[i]].double().permute(0, 1, 3, 2).reshape(nkv, B, d))
            V[dst[i]] = code.reshape(nkv, B // 64, 64, d).permute(0, 1, 3, 2)
        return {"k": K, "v": V, "ks": KS, "vs": VS}
    if c["kind"] == "store":
        span = N_ROT if c["rope"] == "mrope" else d
        x = s["qkv"].double().reshape(s["T"], -1, d)
        w = torch.cat([s["q_norm"].double().expand(nh, d), s["k_norm"].double().expand(nkv, d)])
        y = x[:, :nh + nkv]
        y = y / (y.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w
        j = torch.arange(span // 2, device=x.device)
        a, b = (2 * j, 2 * j + 1) if c["rope"] == "pairs" else (j, j + span // 2)
        z = torch.polar(torch.ones(1, 1, dtype=torch.float64, device=x.device),
                        s["pos"].double()[:, None] * torch.exp(j.double() * (-2.0 * math.log(c["theta"]) / span)))
        r = torch.complex(y[..., a], y[..., b]) * z[:, None, :]
        y[..., a], y[..., b] = r.real, r.imag
        slot = s["slot"].long()
        K = torch.zeros(s["n_blocks"] * B, nkv, d, dtype=torch.float64, device=x.device)
        V, KS = torch.zeros_like(K), torch.zeros_like(K[..., 0])
        VS = torch.zeros_like(KS)
        K[slot], KS[slot] = _codes64(y[:, nh:])
        V[slot], VS[slot] = _codes64(x[:, nh + nkv:])
        return {"q": y[:, :nh].reshape(s["T"], nh * d), "k": K.view(-1, B, nkv, d).transpose(1, 2),
                "v": V.view(-1, B // 64, 64, nkv, d).permute(0, 3, 1, 4, 2),
                "ks": KS.view(-1, B, nkv).transpose(1, 2), "vs": VS.view(-1, B, nkv).transpose(1, 2)}
    out, cu = [], 0
    for i, (L, m) in enumerate(_lengths(c)):
        page = s["table"][i, :-(-L // B)].tolist()
        K = torch.cat([s["k"][p].double() * s["ks"][p].double()[..., None] for p in page], 1)[:, :L]
        V = torch.cat([s["v"][p].double().transpose(1, 2).reshape(nkv, d, B) * s["vs"][p].double()[:, None, :] for p in page], 2)
        V = V[..., :L].transpose(1, 2)
        q = s["q"][cu:cu + m].double().view(m, nh, d)
        ahead = torch.arange(L, device=q.device)[None, :] > torch.arange(L - m, L, device=q.device)[:, None]
        o = torch.empty_like(q)
        for h in range(nh):
            a = (q[:, h] @ K[h * nkv // nh].t() / math.sqrt(d)).masked_fill_(ahead, -math.inf)
            o[:, h] = a.softmax(-1) @ V[h * nkv // nh]
        out.append(o.reshape(m, nh * d))
        cu += m
    o = torch.cat(out)
    return o * s["gate"].double().sigmoid() if c["gated"] else o
