"""The operators of serving over a paged KV cache: what a scheduler's step asks of the backend.

Kinds:

  plan   block tables, slot map, positions and row offsets of one step, from the request lengths and the
         list of free blocks (paged_plan)
  rope   RMSNorm of every query and key head, the position rotation and the store of K and V into the
         pages, in one pass over the projected rows (qk_norm_rope_kv_store)
  attn   attention of each sequence's new tokens over its pages (paged_attn): decode tokens, chunks of a
         prompt, whole prompts, and batches of all of them

A pool holds f16 pages of `block` positions: K [n_blocks, n_kv, block, d] and V [n_blocks, n_kv, block/32,
d, 32].  Lengths and tables are int32 tensors on the GPU.  A case's lengths follow from its numbers alone;
its values, and which pages a sequence has, from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# (query heads, kv heads, head_dim, rope, theta): the head layouts of the benchmark's configurations
HEADS = [(14, 2, 64, "half", 1e6), (28, 4, 128, "half", 1e6), (32, 8, 128, "pairs", 5e5), (16, 2, 256, "mrope", 1e7)]
N_ROT = 64  # rotated dimensions of a qwen35 head
EPS = 1e-6


def _h(i: int) -> dict:
    nh, nkv, d, rope, theta = HEADS[i]
    return {"nh": nh, "nkv": nkv, "d": d, "rope": rope, "theta": theta}


def listed() -> list[dict]:
    return [
        # a decode step of 64 sequences between 1k and 32k tokens: latency
        {"name": "plan_decode_64", "kind": "plan", "n_seq": 64, "lo": 1024, "hi": 32768, "chunks": 0, "new": 1, "block": 64},
        # a step of 256 sequences, 16 of which bring up to 512 prompt tokens
        {"name": "plan_mixed_256", "kind": "plan", "n_seq": 256, "lo": 200, "hi": 16384, "chunks": 16, "new": 512, "block": 64},
        # one decode token of a qwen35 attention layer: the smallest call
        {"name": "rope_token", "kind": "rope", **_h(3), "n_seq": 1, "lo": 4223, "hi": 4223, "chunks": 0, "new": 1, "block": 64, "dtype": "f32", "out": "f32"},
        # the decode tokens of 64 sequences
        {"name": "rope_decode_64", "kind": "rope", **_h(2), "n_seq": 64, "lo": 1024, "hi": 32768, "chunks": 0, "new": 1, "block": 64, "dtype": "bf16", "out": "bf16"},
        # four chunks of a prompt and decode tokens, fp32 rows as the engine holds them
        {"name": "rope_mixed_f32", "kind": "rope", **_h(1), "n_seq": 32, "lo": 300, "hi": 8192, "chunks": 4, "new": 512, "block": 128, "dtype": "f32", "out": "f16"},
        # whole prompts of 8192 tokens in all
        {"name": "rope_prompts_8k", "kind": "rope", **_h(3), "n_seq": 3, "lo": 2700, "hi": 2760, "chunks": 3, "new": 2731, "block": 64, "dtype": "bf16", "out": "bf16"},
        # one decode token of the reference's CPU-runnable model over 512 keys: latency
        {"name": "attn_token_512", "kind": "attn", **_h(0), "n_seq": 1, "lo": 512, "hi": 512, "chunks": 0, "new": 1, "block": 64, "dtype": "f32", "gated": False},
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
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["plan", "rope", "rope", "attn", "attn", "attn"])
    block = rng.choice([64, 64, 128, 256])
    if kind == "plan":
        n = _log(rng, 1, 512)
        chunks = rng.choice([0, _log(rng, 1, 16)])
        hi = _log(rng, 64, 32768)
        return {"kind": kind, "n_seq": n, "lo": max(1, hi // 32), "hi": hi, "chunks": min(n, chunks),
                "new": 1 if chunks == 0 else _log(rng, 2, 1024), "block": block}
    h = _h(rng.randrange(len(HEADS)))
    if kind == "rope":
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


def prepare(case: dict, seed: int) -> dict:
    c, g, B = case, _gen(seed), case["block"]
    lens = _lengths(c)
    n, T = len(lens), sum(m for _, m in lens)
    most = max(-(-L // B) for L, _ in lens)
    s = {"c": c, "T": T, "max_len": max(L for L, _ in lens), "max_new": max(m for _, m in lens)}
    total = _i32([L for L, _ in lens])
    new = _i32([m for _, m in lens])
    # the pages of every sequence, anywhere in the pool; a plan's sequences hold those of their old tokens
    pages = sum(-(-L // B) for L, _ in lens)
    free = pages + 8
    order = torch.randperm(free, generator=g, device="cuda").int()
    held = (total - new + B - 1).div(B, rounding_mode="floor") if c["kind"] == "plan" else (total + B - 1).div(B, rounding_mode="floor")
    first = held.cumsum(0) - held
    at = torch.arange(most, device="cuda")[None, :]
    table = torch.where(at < held[:, None], order[(first[:, None] + at).clamp(max=free - 1)], -1).int()
    if c["kind"] == "plan":
        s.update(table=table, ctx=total - new, new=new, free=order.flip(0).contiguous(), n_free=(free - held.sum()).int().reshape(1))
        return s
    nh, nkv, d = c["nh"], c["nkv"], c["d"]
    s["n_blocks"] = free
    if c["kind"] == "rope":
        seq = torch.repeat_interleave(torch.arange(n, device="cuda"), new.long(), output_size=T)
        cu = new.cumsum(0) - new
        pos = ((total - new)[seq] + torch.arange(T, device="cuda") - cu[seq]).int()
        # the pool of the pages that this step writes: each sequence's last ones
        lo = (total - new).div(B, rounding_mode="floor")
        used = held - lo
        page = torch.randperm(int(used.sum()), generator=g, device="cuda").int()
        slot = page[(used.cumsum(0) - used)[seq] + pos // B - lo[seq]] * B + pos % B
        s["n_blocks"] = nb = page.numel()
        s.update(pos=pos, slot=slot.int(), qkv=_normal(g, T, (nh + 2 * nkv) * d).to(DTYPES[c["dtype"]]),
                 q_norm=1.0 + _normal(g, d, scale=0.1), k_norm=1.0 + _normal(g, d, scale=0.1),
                 q=torch.empty((T, nh * d), dtype=DTYPES[c["out"]], device="cuda"))
        s["k"] = torch.zeros((nb, nkv, B, d), dtype=torch.float16, device="cuda")
        s["v"] = torch.zeros((nb, nkv, B // 32, d, 32), dtype=torch.float16, device="cuda")
        return s
    dt = DTYPES[c["dtype"]]
    s.update(table=table, lens=total, cu=torch.cat([_i32([0]), new.cumsum(0).int()]),
             k=torch.randn((free, nkv, B, d), generator=g, device="cuda", dtype=torch.float16),
             v=torch.randn((free, nkv, B // 32, d, 32), generator=g, device="cuda", dtype=torch.float16),
             q=_normal(g, T, nh * d).to(dt), gate=_normal(g, T, nh * d) if c["gated"] else None,
             out=torch.empty((T, nh * d), dtype=dt, device="cuda"))
    return s


# ---- one pass ----------------------------------------------------------------------------------

def _own(s: dict):
    from yllm_amd import attention as A
    from yllm_amd import paged as P

    c = s["c"]
    if c["kind"] == "plan":
        step = P.paged_plan(s["table"], s["ctx"], s["new"], s["free"], s["n_free"], c["block"], s["T"])
        return {"table": step.block_table, "cu": step.cu_new, "lens": step.kv_lens, "slots": step.slots,
                "positions": step.positions, "counts": step.counts}
    cache = P.PagedKV(s["k"], s["v"])
    if c["kind"] == "rope":
        rope = {"half": A.ROPE_HALF, "pairs": A.ROPE_PAIRS, "mrope": A.ROPE_MROPE}[c["rope"]]
        kd, qd = c["nkv"] * c["d"], c["nh"] * c["d"]
        q, k, v = s["qkv"][:, :qd], s["qkv"][:, qd:qd + kd], s["qkv"][:, qd + kd:]
        P.qk_norm_rope_kv_store(cache, q, k, v, c["nh"], rope, c["theta"], N_ROT if c["rope"] == "mrope" else 0,
                                positions=s["pos"], slots=s["slot"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                                eps=EPS, q_out=s["q"])
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    if "ws" not in s:  # a program keeps one workspace for all its layers
        s["ws"] = P.paged_attn_workspace(s["T"], c["n_seq"], s["max_new"], s["max_len"], c["nh"], c["nkv"], c["d"])
    return P.paged_attn(s["q"], cache, s["table"], s["lens"], s["cu"], c["nh"], s["max_new"], s["max_len"],
                        gate=s["gate"], out=s["out"], workspace=s["ws"])


def run(s: dict):
    if own:
        return _own(s)
    return {"plan": _plan, "rope": _rope, "attn": _attn}[s["c"]["kind"]](s)


def _plan(s: dict) -> dict:
    """Sequences take their blocks in order from the end of the free list."""
    B, T, table, ctx, new = s["c"]["block"], s["T"], s["table"], s["ctx"], s["new"]
    n, width = table.shape
    held = torch.div(ctx + B - 1, B, rounding_mode="floor")
    need = torch.div(ctx + new + B - 1, B, rounding_mode="floor") - held
    took = need.cumsum(0)
    ends = new.cumsum(0)
    fits = (held + need <= width) & ((need == 0) | (took <= s["n_free"])) & (ends <= T)
    at = torch.arange(width, device=table.device)[None, :]
    fresh = fits[:, None] & (at >= held[:, None]) & (at < (held + need)[:, None])
    pick = s["n_free"] - 1 - ((took - need)[:, None] + at - held[:, None])
    table.copy_(torch.where(fresh, s["free"][pick.clamp(0, s["free"].numel() - 1)], table))
    row = torch.arange(T, device=table.device)
    seq = torch.searchsorted(ends, row, right=True).clamp(max=n - 1)
    pos = ctx[seq] + row - (ends - new)[seq]
    real = row < ends[-1]
    slot = table[seq, torch.div(pos, B, rounding_mode="floor").clamp(0, width - 1)] * B + pos % B
    lens = torch.where(fits, ctx + new, 0).int()
    used = torch.where(fits, need, 0).sum()
    short = (took[-1] - s["n_free"][0]).clamp(min=0)
    counts = torch.stack([s["n_free"][0] - used, ends[-1], (~fits).sum(), short]).int()
    return {"table": table, "cu": torch.cat([torch.zeros_like(new[:1]), ends.int()]), "lens": lens,
            "slots": torch.where(real & fits[seq], slot, -1).int(), "positions": torch.where(real, pos, 0).int(),
            "counts": counts}


def _turn(x: torch.Tensor, cs: torch.Tensor, sn: torch.Tensor, rope: str, span: int) -> torch.Tensor:
    if rope == "pairs":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cs - b * sn, a * sn + b * cs], -1).flatten(-2)
    a, b = x[..., :span // 2], x[..., span // 2:span]
    return torch.cat([a * cs - b * sn, a * sn + b * cs, x[..., span:]], -1)


def _rope(s: dict) -> dict:
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
    s["k"][page, :, off] = _turn(k, cs, sn, c["rope"], span).half()
    s["v"][page, :, off // 32, :, off % 32] = v.half()
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _attn(s: dict) -> torch.Tensor:
    """Every sequence padded to the longest context and the largest chunk."""
    c, T, M, L = s["c"], s["T"], s["max_new"], s["max_len"]
    nh, nkv, d, B = c["nh"], c["nkv"], c["d"], c["block"]
    G, n, dev = nh // nkv, s["table"].shape[0], s["q"].device
    at = torch.arange(L, device=dev)
    page = s["table"][:, at // B].clamp(min=0).long()
    k = s["k"][page, :, (at % B)[None, :]].permute(0, 2, 3, 1).float()                       # [n, n_kv, d, L]
    v = s["v"][page, :, (at % B // 32)[None, :], :, (at % 32)[None, :]].permute(0, 2, 1, 3).float()  # [n, n_kv, L, d]
    cu, lens = s["cu"].long(), s["lens"].long()
    new, t = cu[1:] - cu[:-1], torch.arange(M, device=dev)
    row = (cu[:-1, None] + t).clamp(max=T - 1)
    q = s["q"].float().view(T, nkv, G, d)[row].permute(0, 2, 3, 1, 4).reshape(n, nkv, G * M, d)
    p = torch.matmul(q, k).view(n, nkv, G, M, L)
    p *= 1.0 / math.sqrt(d)
    seen = at[None, None, :] <= ((lens - new)[:, None] + t)[..., None]                       # [n, M, L]
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


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case: dict) -> dict:
    c, lens, B = case, _lengths(case), case["block"]
    T = sum(m for _, m in lens)
    if c["kind"] == "plan":
        fresh = sum(-(-L // B) - -(-(L - m) // B) for L, m in lens)
        part = sum((L - m) % B != 0 for L, m in lens)  # a held block that new tokens fill up: its entry is read
        return {"bytes": 4 * (2 * len(lens) + 1 + part + 2 * fresh + 2 * len(lens) + 1 + 2 * T + 4), "flops": 0}
    nh, nkv, d = c["nh"], c["nkv"], c["d"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["kind"] == "rope":
        span = N_ROT if c["rope"] == "mrope" else d
        return {"bytes": T * ((nh + 2 * nkv) * d * size[c["dtype"]] + nh * d * size[c["out"]] + 4 * nkv * d + 8) + 8 * d,
                "flops": T * (nh + nkv) * (4 * d + 3 * span)}
    keys = sum(L for L, _ in lens)
    pairs = sum(m * (L - m) + m * (m + 1) // 2 for L, m in lens)
    return {"bytes": 4 * keys * nkv * d + T * nh * d * (2 * size[c["dtype"]] + (4 if c["gated"] else 0))
            + 4 * sum(-(-L // B) for L, _ in lens) + 8 * len(lens),
            "flops": 4 * pairs * nh * d}


# ---- the same in 64 bits -------------------------------------------------------------------------

def exact(case: dict, seed: int):
    c = case
    if c["kind"] == "plan":
        return None
    s = prepare(case, seed)
    nh, nkv, d, B = c["nh"], c["nkv"], c["d"], c["block"]
    if c["kind"] == "rope":
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
        V = torch.zeros_like(K)
        K[slot], V[slot] = y[:, nh:], x[:, nh + nkv:]
        K = K.view(-1, B, nkv, d).transpose(1, 2)
        V = V.view(-1, B // 32, 32, nkv, d).permute(0, 3, 1, 4, 2)
        return {"q": y[:, :nh].reshape(s["T"], nh * d), "k": K, "v": V}
    out, cu = [], 0
    for i, (L, m) in enumerate(_lengths(c)):
        page = s["table"][i, :-(-L // B)].long()
        K = s["k"][page].transpose(0, 1).reshape(nkv, -1, d)[:, :L].double()
        V = s["v"][page].permute(1, 0, 2, 4, 3).reshape(nkv, -1, d)[:, :L].double()
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
