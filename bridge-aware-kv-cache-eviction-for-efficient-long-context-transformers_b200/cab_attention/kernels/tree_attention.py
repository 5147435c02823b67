"""Attention of drafted tokens over a paged KV cache, on the sm_100a kernel
``cab_tree_attn_fwd``: a tree of draft nodes, a chain of new tokens, or one decoded token per
sequence. It takes the KV-cache steps of the reference's flash attention
(``cab_attention/kernels/flash_attention_accumulate.py:169-261``, whose cache is one dense
tensor) to pages and trees; ``cab_attention.cache.PagedKVCache.attend`` calls it on a cache.

With ``len`` tokens in a sequence's pages, the last ``m = num_nodes`` are its nodes (their
keys and values are in the cache already). Node t sees every earlier token and, of the nodes,
its ancestors and itself: ``out = softmax(scale * q k^T) v`` over what it sees. A query that
sees nothing, and the queries past ``m``, give 0 and a log-sum-exp of -inf. What a query does
not see cannot reach its output, whatever it holds (unused slots, NaN, infinities).
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _lib

_current_device = getattr(torch._C, "_cuda_getDevice", None)  # none in a torch without CUDA, where no call gets this far
_INTS, _BOOLS = (torch.int32, torch.int64), (torch.bool, torch.uint8)


def describe_cache(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                   ref_counts: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None):
    """Checks a cache's tensors and returns their ``cab_page_cache``. ``k_pages, v_pages``
    ``[L, P, Hkv, S, D]``; the tensors must stay alive as long as it is used."""
    if k_pages.dim() != 5 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError("k_pages and v_pages must be [layers, pages, Hkv, page_size, D] of one shape and dtype")
    if k_pages.numel() == 0:
        raise ValueError("the cache has no pages")
    if k_pages.stride(4) != 1 or v_pages.stride(4) != 1:
        raise ValueError("the pages' innermost dimension must be contiguous")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(1) != 1:
        raise ValueError("block_table must be int32 [rows, width] with contiguous rows")
    rows = block_table.shape[0]
    state = [("seq_lens", seq_lens, rows)]
    if ref_counts is not None:
        state += [("ref_counts", ref_counts, k_pages.shape[1]), ("status", status, 1)]
    for name, t, size in state:
        if t.dtype != torch.int32 or tuple(t.shape) != (size,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor [{size}]")
    for t in (v_pages, block_table, seq_lens, ref_counts, status):
        if t is not None and t.device != k_pages.device:
            raise ValueError("the cache's tensors must be on one device")
    c = _lib.PageCache()
    c.k_pages, c.v_pages = k_pages.data_ptr(), v_pages.data_ptr()
    c.layers, c.pages, c.heads, c.page_size, c.dim = k_pages.shape
    c.k_strides[:], c.v_strides[:] = k_pages.stride()[:4], v_pages.stride()[:4]
    c.block_table, c.seq_lens = block_table.data_ptr(), seq_lens.data_ptr()
    c.rows, c.width = block_table.shape
    c.table_stride = block_table.stride(0)
    c.ref_counts = None if ref_counts is None else ref_counts.data_ptr()
    c.status = None if status is None else status.data_ptr()
    c.dtype = _lib.dtype_code(k_pages)
    c.sizes = {}  # workspace bytes by call shape
    return c


def int32_vector(t: Optional[torch.Tensor], n: Optional[int], name: str, device) -> Optional[torch.Tensor]:
    """``t`` as a contiguous int32 vector of ``n`` entries on ``device`` (int64 is converted)."""
    if t is None:
        return None
    shape, dtype = t.shape, t.dtype
    if len(shape) != 1 or (n is not None and shape[0] != n) or (dtype is not torch.int32 and dtype is not torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 tensor [{'n' if n is None else n}]")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    if dtype is torch.int32 and t.is_contiguous():
        return t
    return to_int32(t)


def to_int32(t: torch.Tensor) -> torch.Tensor:
    """As contiguous int32; what does not fit stays out of range instead of wrapping around."""
    return (t if t.dtype is torch.int32 else t.clamp(-1, 2 ** 31 - 1).to(torch.int32)).contiguous()


def call_on(device: torch.device, name: str, fn, *args) -> None:
    """``fn(*args, stream)`` with ``device`` current, on its current stream."""
    index = device.index
    if _current_device() == index:
        rc = fn(*args, _lib.raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _lib.raw_stream(index))
    if rc:
        _lib.check(rc, name)


def attend_cache(cache, device, dtype, layer: int, q: torch.Tensor, parents=None, tree_mask=None, num_nodes=None,
                 rows=None, softmax_scale=None, out=None, return_lse: bool = False):
    """``tree_attention`` on a described cache (``describe_cache``). Written for few host
    microseconds: a decode step of a short cache takes less time on the device than here."""
    shape = q.shape
    if len(shape) != 4 or q.dtype is not dtype:
        raise ValueError(f"q must be [n, Hq, T, D] of the cache's dtype {dtype}")
    if q.device != device:
        raise ValueError(f"q must be on {device}")
    n, Hq, T, D = shape
    if D != cache.dim or Hq == 0 or Hq % cache.heads:
        raise ValueError(f"q must have D = {cache.dim} and a multiple of {cache.heads} heads")
    if not 0 <= layer < cache.layers:
        raise ValueError(f"layer {layer} of {cache.layers}")
    rows_ptr = nodes_ptr = parents_ptr = mask_ptr = None
    if rows is not None:
        rows = int32_vector(rows, n, "rows", device)
        rows_ptr = rows.data_ptr()
    elif n > cache.rows:
        raise ValueError(f"{n} sequences, {cache.rows} rows")
    if num_nodes is not None:
        num_nodes = int32_vector(num_nodes, n, "num_nodes", device)
        nodes_ptr = num_nodes.data_ptr()
    parents_stride = mask_stride = 0
    if parents is not None:
        if tree_mask is not None:
            raise ValueError("give parents or tree_mask, not both")
        if parents.dtype not in _INTS or parents.shape not in ((T,), (n, T)):
            raise ValueError(f"parents must be int32 or int64 [{T}] or [{n}, {T}]")
        if parents.device != device:
            raise ValueError(f"parents must be on {device}")
        if parents.dtype is not torch.int32 or not parents.is_contiguous():
            parents = to_int32(parents)
        parents_ptr, parents_stride = parents.data_ptr(), (T if parents.dim() == 2 else 0)
    elif tree_mask is not None:
        if tree_mask.dtype not in _BOOLS or tree_mask.shape not in ((T, T), (n, T, T)):
            raise ValueError(f"tree_mask must be bool [{T}, {T}] or [{n}, {T}, {T}]")
        if tree_mask.device != device:
            raise ValueError(f"tree_mask must be on {device}")
        if not tree_mask.is_contiguous():
            tree_mask = tree_mask.contiguous()
        mask_ptr, mask_stride = tree_mask.data_ptr(), (T * T if tree_mask.dim() == 3 else 0)
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("softmax_scale must be positive and finite")
    if out is None:
        out = torch.empty(n, Hq, T, D, dtype=dtype, device=device)  # sizes one by one parse faster than a tuple
    elif out.shape != shape or out.dtype is not dtype or out.device != device or out.stride(3) != 1:
        raise ValueError("out must be [n, Hq, T, D] of q's dtype and device with a dense last dimension")
    lse = torch.empty(n, Hq, T, dtype=torch.float32, device=device) if return_lse else None
    if n == 0 or T == 0:
        return (out, lse) if return_lse else out
    s0, s1, s2, s3 = q.stride()
    if s3 != 1 or (s0 | s1 | s2) & (16 // q.element_size() - 1) or not (s0 > 0 and s1 > 0 and s2 > 0) or q.data_ptr() & 15:
        q = q.clone(memory_format=torch.contiguous_format)  # contiguous() would return a misaligned dense view
        s0, s1, s2, _ = q.stride()
    L = _lib.lib()
    nbytes = cache.sizes.get((n, Hq, T))
    if nbytes is None:
        size = _lib._c_size(0)
        with torch.cuda.device(device.index):
            _lib.check(L.cab_tree_attn_workspace_size(cache, n, Hq, T, size), "cab_tree_attn_workspace_size")
        nbytes = cache.sizes[(n, Hq, T)] = size.value
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    o0, o1, o2, _ = out.stride()
    call_on(device, "cab_tree_attn_fwd", L.cab_tree_attn_fwd, cache, layer, q.data_ptr(), out.data_ptr(),
            lse.data_ptr() if return_lse else None, n, Hq, T, _lib.strides(s0, s1, s2), _lib.strides(o0, o1, o2),
            rows_ptr, nodes_ptr, parents_ptr, parents_stride, mask_ptr, mask_stride, scale,
            None if ws is None else ws.data_ptr(), nbytes)
    return (out, lse) if return_lse else out


def tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                   seq_lens: torch.Tensor, parents: Optional[torch.Tensor] = None,
                   tree_mask: Optional[torch.Tensor] = None, num_nodes: Optional[torch.Tensor] = None,
                   rows: Optional[torch.Tensor] = None, softmax_scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """``q [n, Hq, T, D]`` over one layer's ``k_pages, v_pages [P, Hkv, S, D]`` (innermost dim
    dense, other strides free), ``block_table [R, W]`` int32 (page numbers), ``seq_lens [R]``
    int32 (cached tokens, the nodes included). Sequence i is table row ``rows[i]`` (default i).

    ``parents`` int ``[n, T]`` or ``[T]`` (each node's parent, before it; negative: none), or
    ``tree_mask`` bool ``[n, T, T]`` or ``[T, T]`` (which node sees which), or neither: node t
    sees nodes 0..t, so ``T = 1`` is a decode step (``parents``: at most 1024 nodes). ``num_nodes [n]`` (default T): nodes of each
    sequence. Returns ``out [n, Hq, T, D]``, with ``return_lse`` also the natural-log sum-exp
    ``[n, Hq, T]`` fp32.

    bf16 / f16 with D 64 or 128 and a page size of 8, 16, 32, 64 or a multiple of 128 run on the
    tensor cores; float32, other page sizes and any D <= 256 on CUDA cores.
    """
    _lib.require_cuda(q, k_pages, v_pages, block_table, seq_lens, parents, tree_mask, num_nodes, rows, out)
    if k_pages.dim() != 4:
        raise ValueError("k_pages and v_pages must be [pages, Hkv, page_size, D]")
    cache = describe_cache(k_pages.unsqueeze(0), v_pages.unsqueeze(0), block_table, seq_lens)
    return attend_cache(cache, k_pages.device, k_pages.dtype, 0, q, parents, tree_mask, num_nodes,
                        rows, softmax_scale, out, return_lse)
