"""A paged KV cache for decoding with eviction and drafted tokens, on the sm_100a kernels
``cab_pages_update``, ``cab_pages_write`` and ``cab_tree_attn_fwd``.

The reference's ``CABCache`` (``cab_attention/cache/cab_cache.py:41-267``) keeps one dense
tensor per layer, grows it by concatenation (``:122-175``) and evicts by indexing it anew
(``:177-226``). Here K and V live in pages that a table assigns to sequence rows, so rows share
prefixes, grow without copies, and give up what eviction drops:

* ``extend`` / ``write``: room for new tokens, and their keys and values;
* ``attend``: their attention (one decoded token, a chunk of a prompt, a draft tree);
* ``compact``: keep the listed tokens only: the eviction policy's selection
  (``cab_attention.eviction.select_indices_batched``) or a draft tree's accepted path;
* ``fork``: rows that continue another row, sharing its full pages;
* ``truncate`` / ``free``: drop the newest tokens, or all.

Which pages a row gets is decided on the device (the free pages of lowest number, in order),
so no call waits for the host and all of them can be captured in a CUDA graph. What only the
device can refuse (no free page left, a position outside a row) sets ``status``, leaves the
cache as it was and stops later updates and writes; ``check()`` raises it.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from .. import _lib
from ..kernels.tree_attention import attend_cache, call_on, describe_cache, int32_vector

STATUS = {1: "not enough free pages", 2: "a row would hold more tokens than its table row has pages for",
          4: "a row outside the table, or named twice as a destination",
          8: "a length, count or kept position out of range",
          16: "a table entry outside the pages, or a partly filled page that two rows share"}
MAX_COUNT = 2 ** 31 - 1  # larger than any row: the device refuses it, and it does not wrap around on the way


class PagedKVCache:
    """The cache's state is the caller's tensors: ``k_pages, v_pages`` ``[L, P, Hkv, S, D]`` (innermost
    dim dense, other strides free), ``block_table [R, W]`` (-1 past a row's pages), ``seq_lens [R]``,
    ``ref_counts [P]`` (rows that use a page; 0: free) and ``status [1]``, the last four int32. A page
    whose content ends inside it must belong to one row alone. ``allocate`` makes an empty cache.

    ``rows`` of a method (int32 or int64 ``[n]``, on the device; default: all rows in order) are table
    rows; a call may change a row once. Counts may be given as a number or per row as a tensor. A page update
    (``extend``, ``truncate``, ``free``, ``fork``, ``compact``) takes at most 1024 rows: those of a larger cache
    are listed in several calls."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, ref_counts: torch.Tensor, status: torch.Tensor):
        _lib.require_cuda(k_pages, v_pages, block_table, seq_lens, ref_counts, status)
        self._c = describe_cache(k_pages, v_pages, block_table, seq_lens, ref_counts, status)
        self.k_pages, self.v_pages = k_pages, v_pages
        self.block_table, self.seq_lens, self.ref_counts, self.status = block_table, seq_lens, ref_counts, status
        self.device, self.dtype = k_pages.device, k_pages.dtype
        self.num_layers, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = k_pages.shape
        self.num_rows, self.max_pages = block_table.shape
        self._sizes: dict = {}

    @classmethod
    def allocate(cls, num_layers: int, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int,
                 num_rows: int, max_pages: int, dtype=torch.bfloat16, device="cuda") -> "PagedKVCache":
        """An empty cache of ``num_pages`` pages for ``num_rows`` sequences of at most ``max_pages`` pages."""
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device),
                   torch.full((num_rows, max_pages), -1, **i32), torch.zeros(num_rows, **i32),
                   torch.zeros(num_pages, **i32), torch.zeros(1, **i32))

    # ------------------------------------------------------------ page updates
    def _update(self, src, dst, n: int, start, keep, keep_num, grow, copies: bool) -> None:
        start_value = grow_value = 0
        if isinstance(start, torch.Tensor):
            start = int32_vector(start, n, "start", self.device)
        else:
            start_value, start = (-1 if start is None else min(int(start), MAX_COUNT)), None
        if isinstance(grow, torch.Tensor):
            grow = int32_vector(grow, n, "num_new", self.device)
        else:
            grow_value, grow = min(int(grow), MAX_COUNT), None
        L = _lib.lib()
        size = self._sizes.get(n)
        if size is None:
            nbytes = _lib._c_size(0)
            _lib.check(L.cab_pages_update_workspace_size(self._c, n, nbytes), "cab_pages_update_workspace_size")
            size = self._sizes[n] = nbytes.value
        ws = torch.empty(size, dtype=torch.uint8, device=self.device)
        keep_ptr = num_ptr = None
        keep_bytes = keep_stride = keep_cols = num_stride = 0
        if keep is not None:
            keep_ptr, keep_bytes, keep_stride, keep_cols = keep.data_ptr(), keep.element_size(), keep.stride(0), keep.shape[1]
        if keep_num is not None:
            num_ptr, num_stride = keep_num.data_ptr(), keep_num.stride(0)
        call_on(self.device, "cab_pages_update", L.cab_pages_update, self._c, None if src is None else src.data_ptr(),
                None if dst is None else dst.data_ptr(), n, None if start is None else start.data_ptr(), start_value,
                keep_ptr, keep_bytes, keep_stride, keep_cols, num_ptr, num_stride,
                None if grow is None else grow.data_ptr(), grow_value, copies, ws.data_ptr(), size)

    def _rows(self, rows, name: str = "rows"):
        if rows is None:
            return None, self.num_rows
        rows = int32_vector(rows, None, name, self.device)
        return rows, rows.shape[0]

    def extend(self, num_new: Union[int, torch.Tensor], rows: Optional[torch.Tensor] = None) -> None:
        """Room for ``num_new`` more tokens of each row, to be written by ``write``."""
        rows, n = self._rows(rows)
        if not isinstance(num_new, torch.Tensor) and num_new < 0:
            raise ValueError("num_new must not be negative")
        if n:
            self._update(rows, None, n, None, None, None, num_new, False)

    def truncate(self, new_lens: Union[int, torch.Tensor], rows: Optional[torch.Tensor] = None) -> None:
        """Keeps the first ``new_lens`` tokens of each row (at most its length)."""
        rows, n = self._rows(rows)
        if not isinstance(new_lens, torch.Tensor) and new_lens < 0:
            raise ValueError("new_lens must not be negative")
        if n:
            self._update(rows, None, n, new_lens, None, None, 0, True)

    def free(self, rows: Optional[torch.Tensor] = None) -> None:
        """Gives up all pages of the rows."""
        rows, n = self._rows(rows)
        if n:
            self._update(rows, None, n, 0, None, None, 0, False)

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Row ``dst[i]`` becomes a continuation of row ``src[i]`` (as both were before the call): full
        pages are shared, a partly filled last page is copied. Beam search reorders rows this way."""
        src, n = self._rows(src, "src")
        dst = int32_vector(dst, n, "dst", self.device)
        if src is None or dst is None:
            raise ValueError("fork needs src and dst")
        if n:
            self._update(src, dst, n, None, None, None, 0, True)

    def compact(self, keep: torch.Tensor, keep_num: Optional[torch.Tensor] = None,
                start: Union[int, torch.Tensor] = 0, src: Optional[torch.Tensor] = None,
                dst: Optional[torch.Tensor] = None) -> None:
        """Keeps, of each row, its first ``start`` tokens and then those at ``start + keep[i, x]`` for
        ``x < keep_num[i]``, in the order of the list. ``keep [n, K]`` int32 or int64, ``keep_num [n]`` int32
        (any stride; default K): the eviction policy's ``keep`` and ``counts[:, 0]`` as they are, or the
        accepted nodes of a draft tree with ``start`` the context length. With ``dst`` the result becomes
        row ``dst[i]`` and row ``src[i]`` stays. Tokens that move are copied into fresh pages, so as many
        pages as they fill must be free: for an eviction to ``budget`` tokens ``ceil(budget / page_size)`` for each
        row of the call; pages whose tokens stay in place are kept or shared."""
        src, n = self._rows(src, "src")
        dst = int32_vector(dst, n, "dst", self.device)
        if start is None:
            start = 0
        if keep.dim() != 2 or keep.shape[0] != n or keep.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"keep must be int32 or int64 [{n}, K]")
        if keep.device != self.device:
            raise ValueError(f"keep must be on {self.device}")
        if keep.shape[1] and keep.stride(1) != 1:
            keep = keep.contiguous()
        if keep_num is not None:
            if keep_num.dim() != 1 or keep_num.shape[0] != n or keep_num.device != self.device:
                raise ValueError(f"keep_num must be int32 or int64 [{n}] on {self.device}")
            if keep_num.dtype != torch.int32:
                keep_num = int32_vector(keep_num, n, "keep_num", self.device)
        if not isinstance(start, torch.Tensor) and start < 0:
            raise ValueError("start must not be negative")
        if n:
            self._update(src, dst, n, start, keep if keep.shape[1] else None, keep_num, 0, True)

    # ------------------------------------------------------------ tokens
    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, num_new: Optional[torch.Tensor] = None,
              rows: Optional[torch.Tensor] = None) -> None:
        """Keys and values ``[n, Hkv, T, D]`` of each row's newest ``num_new`` (default T) tokens; tokens
        t >= num_new[i] are not written. Rows must differ. Tokens that ``extend`` has made room for are in pages
        of the row alone; older ones may be in pages that rows share, and are then written for all of them (by the
        last of the sequences, where several do)."""
        if k.dim() != 4 or k.shape != v.shape or k.dtype is not self.dtype or v.dtype is not self.dtype:
            raise ValueError(f"k and v must be [n, Hkv, T, D] of the cache's dtype {self.dtype}")
        if k.device != self.device or v.device != self.device:
            raise ValueError(f"k and v must be on {self.device}")
        n, H, T, D = k.shape
        if H != self.num_kv_heads or D != self.head_dim:
            raise ValueError(f"k and v must have {self.num_kv_heads} heads of {self.head_dim}")
        if not 0 <= layer < self.num_layers:
            raise ValueError(f"layer {layer} of {self.num_layers}")
        rows = int32_vector(rows, n, "rows", self.device)
        if rows is None and n > self.num_rows:
            raise ValueError(f"{n} sequences, {self.num_rows} rows")
        num_new = int32_vector(num_new, n, "num_new", self.device)
        if n == 0 or T == 0:
            return
        ks, vs = k.stride(), v.stride()
        if ks[3] != 1:
            k = k.contiguous()
            ks = k.stride()
        if vs[3] != 1:
            v = v.contiguous()
            vs = v.stride()
        call_on(self.device, "cab_pages_write", _lib.lib().cab_pages_write, self._c, layer, k.data_ptr(), v.data_ptr(),
                n, T, _lib.strides(ks[0], ks[1], ks[2]), _lib.strides(vs[0], vs[1], vs[2]),
                None if rows is None else rows.data_ptr(), None if num_new is None else num_new.data_ptr(), T)

    def attend(self, layer: int, q: torch.Tensor, parents: Optional[torch.Tensor] = None,
               tree_mask: Optional[torch.Tensor] = None, num_nodes: Optional[torch.Tensor] = None,
               rows: Optional[torch.Tensor] = None, softmax_scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """Attention of each row's newest tokens over the layer's cache: ``tree_attention``
        (``cab_attention/kernels/tree_attention.py``) on this cache's pages."""
        return attend_cache(self._c, self.device, self.dtype, layer, q, parents, tree_mask, num_nodes, rows,
                            softmax_scale, out, return_lse)

    # ------------------------------------------------------------ host side
    def check(self) -> None:
        """Waits for the device (all its streams); raises and clears what it refused since the last check."""
        torch.cuda.synchronize(self.device)
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise RuntimeError("paged KV cache: " + "; ".join(text for bit, text in STATUS.items() if bits & bit))

    def free_pages(self) -> int:
        """Pages no row uses (waits for the device)."""
        torch.cuda.synchronize(self.device)
        return int((self.ref_counts == 0).sum().item())
