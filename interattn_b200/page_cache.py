"""Pages of a K/V cache that sequences share: hand out, write, fork, free, compact.

The reference keeps one sequence in one contiguous cache (``condition_block_triton_impl/core.py:319-329``); ``ops`` reads
paged pools through tables that its caller makes.  This is where such tables come from.  All layers share one table.
State lives on the device and every call is ordered by the current stream alone, without a host round trip, so a loop that
admits, forks and frees sequences can run ahead of the GPU or be captured into a graph.

Free pages are handed out lowest first, in the order of the list, so the same calls give the same tables every time.
What goes wrong on the device is refused for the list entry concerned and reported in ``ops.device_status()``:
``IA_DEV_STATUS_BAD_INDEX`` (a row or count out of range, a row named twice, a child that is not empty) or
``IA_DEV_STATUS_NO_PAGES`` (the entries from the first one that does not fit on were left as they were).  What was refused stays
refused in the calls that run ahead of that news: a row whose ``extend`` was refused takes no ``write`` until one is served.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .dense_attention import _raw_stream, _same_device, device_guard, wait_for
from .ops import PagedKV, _DTYPES, _need_cuda

PAGE = 16


class PageCache:
    """``pools``: one ``(k_pool, v_pool)`` pair per layer, ``[n_pages, Hkv, 16, D]``, all of the same shape, strides and dtype.
    ``block_table`` int32 ``[n_rows, max_pages]``, ``seq_lens`` int32 ``[n_rows]``, ``refs`` int32 ``[n_pages]``: how many table
    entries hold a page (a caller may add to it what it keeps for itself); 0 is free.  Lists of rows are int32 device
    tensors that name a row once.

    One cache is one state: calls that change it go to one stream, or are ordered by events."""

    def __init__(self, pools: Sequence[Tuple[torch.Tensor, torch.Tensor]], block_table: torch.Tensor, seq_lens: torch.Tensor,
                 refs: torch.Tensor):
        if not pools:
            raise ValueError("at least one layer's pools are needed")
        flat = [p for pair in pools for p in pair]
        k = flat[0]
        _need_cuda(*flat, block_table, seq_lens, refs)
        if k.dim() != 4 or k.shape[2] != PAGE or k.dtype not in _DTYPES:
            raise ValueError("pools are [n_pages, Hkv, 16, D] float32 or bfloat16 tensors")
        if any(p.shape != k.shape or p.dtype != k.dtype or p.stride() != k.stride() for p in flat):
            raise ValueError("the pools of all layers must have equal shape, dtype and strides")
        if k.stride(3) != 1 or k.stride(2) != k.shape[3]:
            raise ValueError("the [P, D] run of one (page, kv head) must be contiguous")
        if any(p.data_ptr() % 16 for p in flat):
            raise ValueError("pools must be 16-byte aligned")
        for name, t, dims in (("block_table", block_table, 2), ("seq_lens", seq_lens, 1), ("refs", refs, 1)):
            if t.dtype != torch.int32 or not t.is_contiguous() or t.dim() != dims:
                raise ValueError(f"{name} must be a contiguous int32 tensor with {dims} dimension(s)")
        if seq_lens.shape[0] != block_table.shape[0] or refs.shape[0] != k.shape[0]:
            raise ValueError("seq_lens has one entry per table row, refs one per page")
        self.device = k.device
        _same_device(self.device, block_table=block_table, seq_lens=seq_lens, refs=refs,
                     **{f"pool {i}": p for i, p in enumerate(flat)})
        self.pools = [tuple(pair) for pair in pools]
        self.block_table, self.seq_lens, self.refs = block_table, seq_lens, refs
        size = int(_lib.load().ia_pages_scratch_bytes(int(block_table.shape[0]), int(k.shape[0])))
        if size < 0:
            _lib.check(_lib.IA_ERR_BAD_ARG)
        # the copy of the addresses waits for its stream, so the scratch too is ready for any other
        self._scratch = torch.zeros((size + 256,), dtype=torch.uint8, device=self.device)
        self._addresses = torch.tensor([p.data_ptr() for p in flat], dtype=torch.int64, device=self.device)
        scratch = self._scratch.data_ptr()
        self._state = _lib.PageCacheState(
            block_table=block_table.data_ptr(), seq_lens=seq_lens.data_ptr(), refs=refs.data_ptr(),
            pools=self._addresses.data_ptr(), scratch=scratch + (-scratch) % 256, scratch_bytes=size,
            page_stride=k.stride(0), head_stride=k.stride(1), n_rows=int(block_table.shape[0]),
            max_pages=int(block_table.shape[1]), n_pages=int(k.shape[0]), n_pools=len(flat), n_kv_heads=int(k.shape[1]),
            head_dim=int(k.shape[3]), dtype=_DTYPES[k.dtype], reserved=0)
        self._held = (flat, block_table, seq_lens, refs)  # the attributes may be given other tensors
        self._c, self._index = ctypes.byref(self._state), self.device.index
        self._streams = {_raw_stream(self._index)}
        self._lib = _lib.load()
        self._token_shape, self._dtype = (int(k.shape[1]), int(k.shape[3])), k.dtype
        self._pool_addresses = [(a.data_ptr(), b.data_ptr()) for a, b in self.pools]

    @staticmethod
    def empty(n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, n_rows: int, max_pages: int, *,
              dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PageCache":
        """A cache of its own pools, all pages free, all rows empty."""
        shape = (n_pages, n_kv_heads, PAGE, head_dim)
        pools = [(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))
                 for _ in range(n_layers)]
        i32 = dict(dtype=torch.int32, device=device)
        return PageCache(pools, torch.full((n_rows, max_pages), -1, **i32), torch.zeros((n_rows,), **i32),
                         torch.zeros((n_pages,), **i32))

    def kv(self, layer: int, prefix_lens: Optional[torch.Tensor] = None) -> PagedKV:
        """One layer as the operators of ``ops`` and ``dense_attention`` take it; the tensors are the cache's own, so
        what later calls change shows there.  ``prefix_lens`` defaults to ``seq_lens``."""
        k, v = self.pools[layer]
        return PagedKV(k, v, self.block_table, self.seq_lens if prefix_lens is None else prefix_lens, self.seq_lens)

    def _list(self, name: str, t: torch.Tensor, n: Optional[int] = None) -> int:
        if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.get_device() != self._index \
                or (n is not None and t.numel() != n):
            _need_cuda(t)
            _same_device(self.device, **{name: t})
            raise ValueError(f"{name} must be a contiguous int32 list" + ("" if n is None else f" of {n} entries"))
        return t.data_ptr()

    def _call(self, function, *args) -> None:
        stream = _raw_stream(self._index)
        if stream not in self._streams:
            wait_for(stream, self._streams, self._index, self._scratch, self._addresses)
        with device_guard(self._index):
            _lib.check(function(self._c, *args, stream))

    def extend(self, rows: torch.Tensor, n_tokens: torch.Tensor) -> None:
        """``rows[i]`` becomes ``n_tokens[i]`` tokens longer and gets the pages for them."""
        n = rows.numel()
        self._call(self._lib.ia_pages_extend, self._list("rows", rows), self._list("n_tokens", n_tokens, n), n)

    def write(self, layer: int, rows: torch.Tensor, starts: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
        """Tokens ``[starts[i], starts[i + 1])`` of k and v ``[T, Hkv, D]`` (token and head strides of any multiple of 16 bytes)
        become the last tokens of ``rows[i]`` in this layer; tokens before the first start and from the last on belong to no row.
        Refused for a row whose last ``extend`` was refused, where a token would fall into a whole page that a fork shared
        while others still hold it, outside the tokens, and for all rows if a start lies below the one before it."""
        shape, ks, vs = k.shape, k.stride(), v.stride()
        if shape != v.shape:
            raise ValueError("k and v hold the same tokens")
        if len(shape) != 3 or (shape[1], shape[2]) != self._token_shape or ((ks[2] != 1 or vs[2] != 1) and shape[0] != 0) \
                or k.dtype is not self._dtype or v.dtype is not self._dtype or k.get_device() != self._index \
                or v.get_device() != self._index:
            for name, t in (("k", k), ("v", v)):
                _need_cuda(t)
                _same_device(self.device, **{name: t})
            raise ValueError("k and v must be [T, Hkv, D] tensors of the pools' dtype with contiguous heads")
        n = rows.numel()
        self._call(self._lib.ia_pages_write, self._list("rows", rows), self._list("starts", starts, n + 1), n, k.data_ptr(),
                   v.data_ptr(), ks[0], ks[1], vs[0], vs[1], shape[0], *self._pool_addresses[layer])

    def fork(self, parents: torch.Tensor, children: torch.Tensor, *, share: bool = True) -> None:
        """``children[i]``, an empty row, becomes a copy of ``parents[i]`` as it was before the call.  With ``share`` the two
        hold the same whole pages and a partly filled last page is copied, so both can be extended; without, every
        page is copied.  A parent may have any number of children."""
        n = parents.numel()
        self._call(self._lib.ia_pages_fork, self._list("parents", parents), self._list("children", children, n), n,
                   1 if share else 0)

    def free(self, rows: torch.Tensor) -> None:
        """The rows become empty (they may be already); pages that no row holds any more are free."""
        self._call(self._lib.ia_pages_free, self._list("rows", rows), rows.numel())

    def compact(self) -> None:
        """The pages in use move to the front of the pools, in all layers, and the table follows.  Pages that the caller holds
        by a count of its own move too: it finds them nowhere in the table, so it should hold none."""
        self._call(self._lib.ia_pages_compact)
