"""Serving over a paged KV cache, on HIP: host-side mirror of the paged part of the C ABI.

    paged_plan(block_table, ctx_lens, ...)        block tables, slot map and row offsets of one step
    qk_norm_rope_kv_store(cache, q, k, v, ...)    QK norm, rotation and the K/V store in one pass
    paged_attn(q, cache, block_table, ...)        the new tokens of every sequence over its pages

A step of a layer, for sequences of any lengths (decode tokens and prompt chunks together):

    step = paged_plan(block_table, ctx_lens, new_lens, free_blocks, n_free, block, n_tok)
    q = qk_norm_rope_kv_store(cache, q, k, v, n_heads, rope, theta, positions=step.positions, slots=step.slots, ...)
    out = paged_attn(q, cache, step.block_table, step.kv_lens, step.cu_new, n_heads, max_new, max_len)

Tensors are torch tensors on one GPU; every call is queued on the current torch stream of that GPU.  Errors raise
YhipError; there is no CPU fallback.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ._lib import ENOSPC, F32, OK, YhipError, check, elsewhere, lib
from ._lib import current_stream as _stream
from .attention import _DT, ROPE_MROPE, ROPE_NONE, LayerKV, _dtype_code, _with_workspace

_I32 = torch.int32
_F16 = torch.float16


@dataclass
class PagedKV:
    """One layer's pool of KV pages in HBM, shared by all sequences.

    k: f16 [n_blocks, n_kv, block, head_dim]
    v: f16 [n_blocks, n_kv, block // 32, head_dim, 32] (32-position tiles, d-major)
    """

    k: torch.Tensor
    v: torch.Tensor

    @property
    def n_blocks(self) -> int:
        return self.k.shape[0]

    @property
    def n_kv(self) -> int:
        return self.k.shape[1]

    @property
    def block(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]

    @classmethod
    def empty(cls, n_blocks: int, n_kv: int, head_dim: int, block: int = 64, device: str | torch.device = "cuda",
              zero: bool = True) -> "PagedKV":
        if not 64 <= block <= 65536 or block & (block - 1):
            raise YhipError(-22, f"PagedKV: block {block} must be a power of two in 64..65536")
        alloc = torch.zeros if zero else torch.empty
        k = alloc((n_blocks, n_kv, block, head_dim), dtype=torch.float16, device=device)
        v = alloc((n_blocks, n_kv, block // 32, head_dim, 32), dtype=torch.float16, device=device)
        return cls(k, v)


# Small calls are bound by this module's own work (a decode step's kernels take 4 to 6 us), so the checks below ask a
# tensor for as little as they can, and build messages only when they fail.

def _pool(cache: PagedKV | LayerKV, fn: str) -> tuple[int, int, int, int]:
    """(n_blocks, n_kv, block, head_dim); a LayerKV is a pool of one page."""
    k, v = cache.k, cache.v
    shape = k.shape
    if len(shape) == 3:
        shape = (1, *shape)
    if len(shape) != 4 or k.dtype is not _F16 or v.dtype is not _F16 or not k.is_contiguous() \
            or not v.is_contiguous() or v.numel() != k.numel() or v.shape[-2:] != (shape[3], 32):
        raise YhipError(-22, f"{fn}: the cache must hold contiguous f16 K and V of one size, V in tiles of 32 positions")
    return shape


def _ints(fn: str, name: str, t: torch.Tensor, n: int) -> None:
    if t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous():
        raise YhipError(-22, f"{fn}: {name} must be contiguous int32 [{n}]")


def _table(fn: str, t: torch.Tensor) -> tuple[int, int, int]:
    """(rows, entries per row, row stride) of a block table."""
    if t.dtype is _I32 and t.dim() == 2:
        n, w = t.shape
        if w and t.is_contiguous():
            return n, w, w
        if w and (w == 1 or t.stride(1) == 1):
            return n, w, (t.stride(0) if n > 1 else w)
    raise YhipError(-22, f"{fn}: block_table must be int32 [n_seq, max_blocks] with unit column stride")


@dataclass
class PagedStep:
    """What paged_plan found for one step: the tensors the step's layers read (all int32)."""

    block_table: torch.Tensor  # [n_seq, max_blocks]
    cu_new: torch.Tensor       # [n_seq + 1]
    kv_lens: torch.Tensor      # [n_seq]
    slots: torch.Tensor        # [n_tok]
    positions: torch.Tensor    # [n_tok]
    counts: torch.Tensor       # [4]: free blocks left, rows, sequences not served, blocks missing


def paged_plan(block_table: torch.Tensor, ctx_lens: torch.Tensor, new_lens: torch.Tensor, free_blocks: torch.Tensor,
               n_free: torch.Tensor, block: int, n_tok: int, out: PagedStep | None = None) -> PagedStep:
    """Blocks, slots and positions of a step in which sequence i, with ctx_lens[i] positions stored, brings
    new_lens[i] tokens (all int32 on the GPU).  block_table [n_seq, max_blocks] gets the entries of the new blocks,
    which come from the end of free_blocks[:n_free[0]]; n_tok rows get a slot and a position (padding: -1 and 0).
    counts[:1] is the n_free of the next step; a sequence that could not be served in whole has kv_lens 0 and slots of
    -1 (yhip_paged_plan has the rules).  `out`: the tensors of an earlier step, overwritten; the inputs must not be among
    them, so its counts[:1] and kv_lens are first copied (n_free.copy_(out.counts[:1])) to tensors of their own."""
    fn = "paged_plan"
    n, w, stride = _table(fn, block_table)
    _ints(fn, "ctx_lens", ctx_lens, n)
    _ints(fn, "new_lens", new_lens, n)
    _ints(fn, "n_free", n_free, 1)
    n_list = free_blocks.numel()
    _ints(fn, "free_blocks", free_blocks, n_list)
    if out is None:
        # one allocation
        buf = torch.empty(2 * n + 2 * n_tok + 5, dtype=_I32, device=block_table.device)
        cu, lens, slots, pos, counts = buf.split_with_sizes([n + 1, n, n_tok, n_tok, 4])
        there = elsewhere(fn, block_table.get_device(), ctx_lens, new_lens, free_blocks, n_free)
    else:
        cu, lens, slots, pos, counts = out.cu_new, out.kv_lens, out.slots, out.positions, out.counts
        for name, t, m in (("cu_new", cu, n + 1), ("kv_lens", lens, n), ("slots", slots, n_tok),
                           ("positions", pos, n_tok), ("counts", counts, 4)):
            _ints(fn, name, t, m)
        there = elsewhere(fn, block_table.get_device(), ctx_lens, new_lens, free_blocks, n_free, cu, lens, slots, pos,
                          counts)
    args = (block_table.data_ptr(), w, stride, ctx_lens.data_ptr(), new_lens.data_ptr(), free_blocks.data_ptr(), n_list,
            n_free.data_ptr(), n, n_tok, block, cu.data_ptr(), lens.data_ptr(), slots.data_ptr(), pos.data_ptr(),
            counts.data_ptr())
    _launch(lib().yhip_paged_plan, args, there)
    if out is None:
        return PagedStep(block_table, cu, lens, slots, pos, counts)
    out.block_table = block_table
    return out


def _launch(f, args: tuple, there) -> None:
    if there is None:
        rc = f(*args, _stream())
    else:
        with there:
            rc = f(*args, _stream())
    if rc != OK:
        check(rc)


def _rows(fn: str, name: str, t: torch.Tensor, rows: int, width: int) -> int:
    """The row stride of a [rows, >= width] matrix with unit column stride."""
    shape, step = t.shape, t.stride()
    if len(step) == 2 and shape[0] == rows and shape[1] >= width and (step[1] == 1 or shape[1] == 1):
        return step[0] if rows > 1 else width
    raise YhipError(-22, f"{fn}: {name} must be [{rows}, >={width}] rows with unit column stride")


def qk_norm_rope_kv_store(cache: PagedKV | LayerKV, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                          n_heads: int, rope: int, theta: float, n_rot: int = 0, *,
                          positions: torch.Tensor | None = None, slots: torch.Tensor | None = None,
                          pos_start: int = 0, q_norm: torch.Tensor | None = None,
                          k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                          q_out: torch.Tensor | None = None,
                          q_out_dtype: torch.dtype | None = None) -> torch.Tensor | None:
    """RMSNorm of every query and key head with the weights q_norm and k_norm [head_dim] (f32 / f16; both None: no
    norm), RoPE by `positions`, and k and v stored into the cache at `slots` (int32 [T], as paged_plan gives them).
    Without slots the rows are the positions pos_start.. and slots of a contiguous cache (LayerKV).

    q [T, n_heads*head_dim], k and v [T, n_kv*head_dim] of one type (f32 / f16 / bf16); rows may be strided slices of
    one projection output.  rope: ROPE_PAIRS, ROPE_HALF, ROPE_MROPE (first n_rot dims) or ROPE_NONE.  Returns the
    rotated q (q_out, allocated in q_out_dtype or q's type if not given; q_out may be q itself), or None when q is
    None.  Rows without a slot (negative) are skipped."""
    fn = "qk_norm_rope_kv_store"
    n_blocks, n_kv, block, d = _pool(cache, fn)
    dt = k.dtype
    T = k.shape[0]
    ks, vs = _rows(fn, "k", k, T, n_kv * d), _rows(fn, "v", v, T, n_kv * d)
    if v.dtype is not dt or dt not in _DT or (q is not None and q.dtype is not dt):
        raise YhipError(-22, f"{fn}: q, k and v must have one type, f32, f16 or bf16")
    qs = qos = qp = qop = 0
    qdt = F32
    if q is not None:
        qs = _rows(fn, "q", q, T, n_heads * d)
        if q_out is None:
            q_out = torch.empty((T, n_heads * d), dtype=q_out_dtype or dt, device=q.device)
        qos = _rows(fn, "q_out", q_out, T, n_heads * d)
        qdt = _dtype_code(q_out)
        qp, qop = q.data_ptr(), q_out.data_ptr()
    else:
        q_out = None
    pp = sp = wq = wk = None
    if positions is not None:
        _ints(fn, "positions", positions, T)
        pp = positions.data_ptr()
    if slots is not None:
        if positions is None:
            raise YhipError(-22, f"{fn}: slots come with positions")
        _ints(fn, "slots", slots, T)
        sp = slots.data_ptr()
    norm = F32
    if q_norm is not None or k_norm is not None:
        if q_norm is None or k_norm is None or q_norm.shape != (d,) or k_norm.shape != (d,) \
                or not q_norm.is_contiguous() or not k_norm.is_contiguous() or k_norm.dtype is not q_norm.dtype \
                or q_norm.dtype not in (torch.float32, _F16):
            raise YhipError(-22, f"{fn}: q_norm and k_norm must both be [{d}], f32 or f16")
        norm = _DT[q_norm.dtype]
        wq, wk = q_norm.data_ptr(), k_norm.data_ptr()
    kc, vc = cache.k, cache.v
    args = (qop, qdt, qos, qp, qs, k.data_ptr(), ks, v.data_ptr(), vs, _DT[dt], wq, wk, norm, eps, kc.data_ptr(),
            vc.data_ptr(), n_blocks, block, pp, sp, pos_start, T, n_heads, n_kv, d, rope,
            n_rot if rope == ROPE_MROPE else 0, theta if rope != ROPE_NONE else 1.0)
    _launch(lib().yhip_qk_norm_rope_kv_store, args,
            elsewhere(fn, k.get_device(), kc, vc, q, v, q_out, positions, slots, q_norm, k_norm))
    return q_out


def paged_attn_workspace_bytes(n_tok: int, n_seq: int, max_new: int, max_len: int, n_heads: int, n_kv: int,
                               head_dim: int) -> int:
    """Workspace of every paged_attn call within these bounds."""
    return int(lib().yhip_paged_attn_workspace(n_tok, n_seq, max_new, max_len, n_heads, n_kv, head_dim))


def paged_attn_workspace(n_tok: int, n_seq: int, max_new: int, max_len: int, n_heads: int, n_kv: int, head_dim: int,
                         device: torch.device | str = "cuda") -> torch.Tensor:
    nbytes = paged_attn_workspace_bytes(n_tok, n_seq, max_new, max_len, n_heads, n_kv, head_dim)
    return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)


def paged_attn(q: torch.Tensor, cache: PagedKV, block_table: torch.Tensor, kv_lens: torch.Tensor, cu_new: torch.Tensor,
               n_heads: int, max_new: int, max_len: int | None = None, gate: torch.Tensor | None = None,
               out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of every sequence's new tokens, rows cu_new[i]..cu_new[i+1]-1 of q [T, n_heads*head_dim] (f32 /
    f16 / bf16), over its kv_lens[i] stored positions (the new ones included).  max_new and max_len bound the new
    tokens and lengths of every sequence (max_len None: what block_table can hold).  gate: None or fp32 rows (the
    output times sigmoid(gate)).  A workspace of paged_attn_workspace is allocated per call unless given."""
    fn = "paged_attn"
    if not isinstance(cache, PagedKV):
        raise YhipError(-22, f"{fn}: the cache must be a PagedKV")
    n_blocks, n_kv, block, d = _pool(cache, fn)
    n, w, stride = _table(fn, block_table)
    _ints(fn, "kv_lens", kv_lens, n)
    _ints(fn, "cu_new", cu_new, n + 1)
    width = n_heads * d
    T = q.shape[0]
    if q.shape[-1] != width:
        raise YhipError(-22, f"{fn}: q must be [T, n_heads*head_dim]")
    qs = _rows(fn, "q", q, T, width)
    if max_len is None:
        max_len = min(w * block, 0x7fffffff)
    if out is None:
        out = torch.empty((T, width), dtype=out_dtype or q.dtype, device=q.device)
    os_ = _rows(fn, "out", out, T, width)
    gp, gs = None, 0
    if gate is not None:
        gs = _rows(fn, "gate", gate, T, width)
        gp = gate.data_ptr()
        if gate.dtype is not torch.float32:
            raise YhipError(-22, f"{fn}: gate must be fp32")
    kc, vc = cache.k, cache.v
    dev = q.get_device()
    there = elsewhere(fn, dev, kc, vc, block_table, kv_lens, cu_new, out, gate)
    args = (out.data_ptr(), _dtype_code(out), os_, q.data_ptr(), _dtype_code(q), qs, kc.data_ptr(), vc.data_ptr(),
            n_blocks, block, block_table.data_ptr(), w, stride, kv_lens.data_ptr(), cu_new.data_ptr(), n, T, max_new,
            max_len, n_heads, n_kv, d, gp, gs)
    f = lib().yhip_paged_attn
    if there is None and workspace is not None and workspace.get_device() == dev:
        rc = f(*args, workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream())
        if rc == OK:
            return out
        if rc != ENOSPC:
            check(rc)
        workspace = None  # too short: allocated below
    need = lambda: paged_attn_workspace_bytes(T, n, max_new, max_len, n_heads, n_kv, d)  # noqa: E731
    if there is None:
        _with_workspace(f, args, workspace, need, q.device)
    else:
        with there:
            _with_workspace(f, args, workspace, need, q.device)
    return out
