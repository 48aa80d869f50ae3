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

from ._lib import F32, YhipError, _gpu_of, check, lib
from ._lib import current_stream as _stream
from .attention import ROPE_MROPE, ROPE_NONE, LayerKV, _dtype_code, _ptr, _with_workspace

_I32 = torch.int32


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
        if block < 64 or block & (block - 1):
            raise YhipError(-22, f"PagedKV: block {block} must be a power of two of at least 64")
        alloc = torch.zeros if zero else torch.empty
        k = alloc((n_blocks, n_kv, block, head_dim), dtype=torch.float16, device=device)
        v = alloc((n_blocks, n_kv, block // 32, head_dim, 32), dtype=torch.float16, device=device)
        return cls(k, v)


def _pool(cache: PagedKV | LayerKV, fn: str) -> tuple[int, int, int, int]:
    """(n_blocks, n_kv, block, head_dim); a LayerKV is a pool of one page."""
    k, v = cache.k, cache.v
    shape = (1, *k.shape) if isinstance(cache, LayerKV) else tuple(k.shape)
    if len(shape) != 4 or k.dtype != torch.float16 or v.dtype != torch.float16 or not k.is_contiguous() \
            or not v.is_contiguous() or v.numel() != k.numel():
        raise YhipError(-22, f"{fn}: the cache must hold contiguous f16 K and V of one size")
    return shape


def _ints(fn: str, name: str, t: torch.Tensor, n: int) -> torch.Tensor:
    if t.dtype != _I32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise YhipError(-22, f"{fn}: {name} must be contiguous int32 [{n}]")
    return t


def _table(fn: str, t: torch.Tensor) -> tuple[int, int, int]:
    """(rows, entries per row, row stride) of a block table."""
    if t.dtype != _I32 or t.dim() != 2 or t.shape[1] == 0 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise YhipError(-22, f"{fn}: block_table must be int32 [n_seq, max_blocks] with unit column stride")
    n, w = t.shape
    return n, w, (t.stride(0) if n > 1 else w)


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
    -1 (yhip_paged_plan has the rules).  `out`: the tensors of an earlier step, overwritten."""
    fn = "paged_plan"
    n, w, stride = _table(fn, block_table)
    _ints(fn, "ctx_lens", ctx_lens, n)
    _ints(fn, "new_lens", new_lens, n)
    _ints(fn, "n_free", n_free, 1)
    _ints(fn, "free_blocks", free_blocks, free_blocks.numel())
    if out is None:
        dev = block_table.device
        # one allocation: int32 parts of n + 1, n, n_tok, n_tok and 4
        buf = torch.empty(2 * n + 2 * n_tok + 5, dtype=_I32, device=dev)
        cu, lens, slots, pos, counts = buf.split([n + 1, n, n_tok, n_tok, 4])
        out = PagedStep(block_table, cu, lens, slots, pos, counts)
    else:
        out.block_table = block_table
        for name, t, m in (("cu_new", out.cu_new, n + 1), ("kv_lens", out.kv_lens, n), ("slots", out.slots, n_tok),
                           ("positions", out.positions, n_tok), ("counts", out.counts, 4)):
            _ints(fn, name, t, m)
    with _gpu_of(fn, block_table, ctx_lens, new_lens, free_blocks, n_free, out.cu_new, out.kv_lens, out.slots,
                 out.positions, out.counts):
        check(lib().yhip_paged_plan(block_table.data_ptr(), w, stride, ctx_lens.data_ptr(), new_lens.data_ptr(),
                                    free_blocks.data_ptr(), free_blocks.numel(), n_free.data_ptr(), n, n_tok, block,
                                    out.cu_new.data_ptr(), out.kv_lens.data_ptr(), out.slots.data_ptr(),
                                    out.positions.data_ptr(), out.counts.data_ptr(), _stream()))
    return out


def _rows(fn: str, name: str, t: torch.Tensor, width: int, dtype: torch.dtype | None = None) -> int:
    """The row stride of a [T, >= width] matrix with unit column stride."""
    if t.dim() != 2 or t.shape[1] < width or t.stride(1) != 1 or (dtype is not None and t.dtype != dtype):
        raise YhipError(-22, f"{fn}: {name} must be [T, >={width}] rows with unit column stride"
                             f"{'' if dtype is None else f' of {dtype}'}")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


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
    T = k.shape[0]
    ks, vs = _rows(fn, "k", k, n_kv * d), _rows(fn, "v", v, n_kv * d, k.dtype)
    qs = qos = 0
    qdt = F32
    if v.shape[0] != T or (q is not None and q.shape[0] != T):
        raise YhipError(-22, f"{fn}: q, k, v row counts differ")
    if q is not None:
        qs = _rows(fn, "q", q, n_heads * d, k.dtype)
        if q_out is None:
            q_out = torch.empty((T, n_heads * d), dtype=q_out_dtype or q.dtype, device=q.device)
        qos = _rows(fn, "q_out", q_out, n_heads * d)
        if q_out.shape[0] != T:
            raise YhipError(-22, f"{fn}: q_out must have the rows of q")
        qdt = _dtype_code(q_out)
    else:
        q_out = None
    if slots is not None:
        _ints(fn, "slots", slots, T)
        if positions is None:
            raise YhipError(-22, f"{fn}: slots come with positions")
    if positions is not None:
        _ints(fn, "positions", positions, T)
    norm = F32
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None and (w.shape != (d,) or not w.is_contiguous() or w.dtype not in (torch.float32, torch.float16)):
            raise YhipError(-22, f"{fn}: {name} must be [{d}], f32 or f16")
    if q_norm is not None and k_norm is not None:
        if q_norm.dtype != k_norm.dtype:
            raise YhipError(-22, f"{fn}: q_norm and k_norm must have one type")
        norm = _dtype_code(q_norm)
    with _gpu_of(fn, cache.k, cache.v, q, k, v, q_out, positions, slots, q_norm, k_norm):
        check(lib().yhip_qk_norm_rope_kv_store(
            _ptr(q_out), qdt, qos, _ptr(q), qs, k.data_ptr(), ks, v.data_ptr(), vs, _dtype_code(k), _ptr(q_norm),
            _ptr(k_norm), norm, eps, cache.k.data_ptr(), cache.v.data_ptr(), n_blocks, block, _ptr(positions),
            _ptr(slots), pos_start, T, n_heads, n_kv, d, rope, n_rot if rope == ROPE_MROPE else 0,
            theta if rope != ROPE_NONE else 1.0, _stream()))
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
    qs = _rows(fn, "q", q, width)
    T = q.shape[0]
    if q.shape[1] != width:
        raise YhipError(-22, f"{fn}: q must be [T, n_heads*head_dim]")
    if max_len is None:
        max_len = min(w * block, 0x7fffffff)
    if out is None:
        out = torch.empty((T, width), dtype=out_dtype or q.dtype, device=q.device)
    os_ = _rows(fn, "out", out, width)
    if out.shape[0] != T or (gate is not None and gate.shape[0] != T):
        raise YhipError(-22, f"{fn}: out and gate must have the rows of q")
    gs = _rows(fn, "gate", gate, width, torch.float32) if gate is not None else 0
    args = (out.data_ptr(), _dtype_code(out), os_, q.data_ptr(), _dtype_code(q), qs, cache.k.data_ptr(),
            cache.v.data_ptr(), n_blocks, block, block_table.data_ptr(), w, stride, kv_lens.data_ptr(),
            cu_new.data_ptr(), n, T, max_new, max_len, n_heads, n_kv, d, _ptr(gate), gs)
    with _gpu_of(fn, q, cache.k, cache.v, block_table, kv_lens, cu_new, out, gate):
        _with_workspace(lib().yhip_paged_attn, args, workspace,
                        lambda: paged_attn_workspace_bytes(T, n, max_new, max_len, n_heads, n_kv, d), q.device)
    return out
