"""Attention over all keys, next to the block-sparse step of ``ops``: whole prompts, and single tokens of sequences that
share a prefix.

The reference leaves both to ``scaled_dot_product_attention``, one sequence at a time (``condition_block_triton_impl/
core.py:115-123, 1276-1290``).  Here the prompts of a batch lie one after the other whatever their lengths, and in the
decode step the pages of a common prefix are read once for all sequences of a group.  Conventions as in ``ops``: CUDA
tensors only, the current stream of the tensors' device, query head = kv * G + g, G up to 16, head_dim 64 or 128, bfloat16 or
float32, scale 1 / sqrt(D), softmax in fp32; no backward pass.

    cache = page_cache.PageCache.empty(...)                  # pages of all layers
    plan = PromptAttention(lens, n_q_heads, n_kv_heads, D)    # once per batch of prompts
    y = plan.run(q, k, v)                                     # every layer
    cache.extend(rows, lens); cache.write(layer, rows, starts, k, v); cache.fork(parents, children)
    step = SharedPrefixAttention(cache.kv(layer), group_sizes, shared_lens, n_q_heads)
    y = step.step(q)                                          # every token
"""

from __future__ import annotations

import contextlib
import ctypes
import struct
from typing import Optional, Sequence

import torch

from . import _lib
from .ops import PagedKV, _DTYPES, _need_cuda, _ptr


_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_NO_GUARD = contextlib.nullcontext()


def device_guard(index: int):
    """A context in which kernels go to the device."""
    return _NO_GUARD if index == _current_device() else torch.cuda.device(index)


def wait_for(stream: int, known: set, index: int, *held: torch.Tensor) -> None:
    """torch's allocator hears of a stream, the device's current one, whose kernels read `held`: memory whose owner is dropped waits
    for it too, as it does for those in `known`."""
    for t in held:
        t.record_stream(torch.cuda.current_stream(index))
    known.add(stream)


def _same_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def _host_lens(name: str, lens) -> torch.Tensor:
    given = torch.as_tensor(lens, device="cpu")
    t = given.to(torch.int64)
    if t.dim() != 1 or not torch.equal(t.to(given.dtype), given) or (t.numel() and (int(t.min()) < 0 or int(t.max()) > 0x7fffffff)):
        raise ValueError(f"{name} is a list of lengths, whole numbers, one per sequence, none negative")
    return t.to(torch.int32).contiguous()


_PROMPT_TENSORS = struct.Struct("=5Q6q6i").pack   # struct ia_prompt_tensors


class PromptAttention:
    """Causal attention over whole prompts packed one after the other.

    ``q_lens[i]`` query tokens and ``kv_lens[i]`` keys (as many, if not given) belong to sequence ``i``; its query token ``t``
    sees its first ``kv_lens[i] - q_lens[i] + t + 1`` keys, so with more keys than queries the queries continue a prompt
    that is partly read.  A row that sees no key comes out as zeros.  What a row does not see never reaches it, also
    where it is infinite or NaN.

    The lengths are host values; the work is cut and spread over the GPU once, here, and the object serves every layer
    and any number of streams and captured graphs (keep it as long as these): it holds nothing that a call writes.  Where
    there are few queries and many keys the keys are cut too, and ``run`` takes a workspace from torch's allocator."""

    def __init__(self, q_lens: Sequence[int], n_q_heads: int, n_kv_heads: int, head_dim: int, *,
                 kv_lens: Optional[Sequence[int]] = None, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if dtype not in _DTYPES:
            raise ValueError(f"dtype {dtype} not supported (float32, bfloat16)")
        if n_kv_heads <= 0 or n_q_heads <= 0 or n_q_heads % n_kv_heads != 0:
            raise ValueError("query heads must be a multiple of kv heads")
        q_lens = _host_lens("q_lens", q_lens)
        kv_lens = q_lens if kv_lens is None else _host_lens("kv_lens", kv_lens)
        if q_lens.numel() != kv_lens.numel():
            raise ValueError("q_lens and kv_lens describe the same sequences")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("interattn_b200 operators take CUDA tensors only (there is no CPU path)")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.dtype, self.n_q_heads, self.n_kv_heads, self.head_dim = dtype, int(n_q_heads), int(n_kv_heads), int(head_dim)
        self.n_q_tokens, self.n_kv_tokens = int(q_lens.sum()), int(kv_lens.sum())
        lib = _lib.load()
        group = self.n_q_heads // self.n_kv_heads
        args = (_ptr(q_lens), _ptr(kv_lens), q_lens.numel(), self.n_kv_heads, group, self.head_dim, _DTYPES[dtype])
        with torch.cuda.device(self.device):
            words = int(lib.ia_prompt_plan_ints(*args))
            if words < 0:
                _lib.check(_lib.IA_ERR_UNSUPPORTED)
            self._host = torch.empty((words,), dtype=torch.int32)
            _lib.check(lib.ia_prompt_plan(*args, _ptr(self._host), words))
            self._plan = self._host.to(self.device)
        self._host = self._host[:8].clone()
        self._ws_bytes = int(lib.ia_prompt_workspace_bytes(_ptr(self._host)))
        # run() is called once per layer: what it passes and checks against is made here
        self._call, self._index = lib.ia_prompt_attention, self.device.index
        self._streams = {_raw_stream(self._index)}
        self._plan_args = (self._host.data_ptr(), self._plan.data_ptr())
        self._sizes = (self.n_q_tokens, self.n_kv_tokens, self.n_kv_heads, group, self.head_dim, _DTYPES[dtype])
        self._q_shape = torch.Size((self.n_q_tokens, self.n_q_heads, self.head_dim))
        self._kv_shape = torch.Size((self.n_kv_tokens, self.n_kv_heads, self.head_dim))

    def _fits(self, t: torch.Tensor, shape: torch.Size) -> bool:
        return t.shape == shape and t.dtype is self.dtype and t.get_device() == self._index \
            and (t.stride(2) == 1 or t.numel() == 0)

    def _refuse(self, name: str, t: torch.Tensor, shape: torch.Size) -> None:
        _need_cuda(t)
        if t.shape != shape or t.dtype != self.dtype:
            raise ValueError(f"{name} must be a {list(shape)} {self.dtype} tensor")
        _same_device(self.device, **{name: t})
        raise ValueError(f"the {self.head_dim} elements of one head of {name} must be contiguous")

    def run(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, out: Optional[torch.Tensor] = None,
            return_lse: bool = False):
        """q ``[sum(q_lens), Hq, D]``, k and v ``[sum(kv_lens), Hkv, D]`` (token and head strides of any multiple of 16 bytes)
        -> ``[sum(q_lens), Hq, D]``, which may not overlap them; with ``return_lse`` also the log-sum-exp ``[sum(q_lens), Hq]`` f32 (-inf for a
        row without keys) that ``ops.finalize`` merges by."""
        for name, t, shape in (("q", q, self._q_shape), ("k", k, self._kv_shape), ("v", v, self._kv_shape)):
            if not self._fits(t, shape):
                self._refuse(name, t, shape)
        if out is None:
            out = q.new_empty(self._q_shape)
        elif not self._fits(out, self._q_shape):
            self._refuse("out", out, self._q_shape)
        elif not out.is_contiguous():
            raise ValueError("out must be contiguous")
        lse = torch.empty(self._q_shape[:2], dtype=torch.float32, device=self.device) if return_lse else None
        (qt, qh, _), (kt, kh, _), (vt, vh, _) = q.stride(), k.stride(), v.stride()
        tensors = _PROMPT_TENSORS(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                                  qt, qh, kt, kh, vt, vh, *self._sizes)
        ws = torch.empty((self._ws_bytes,), dtype=torch.uint8, device=self.device) if self._ws_bytes else None
        stream = _raw_stream(self._index)
        if stream not in self._streams:
            wait_for(stream, self._streams, self._index, self._plan)
        with device_guard(self._index):
            _lib.check(self._call(tensors, *self._plan_args, 0 if ws is None else ws.data_ptr(), self._ws_bytes, stream))
        return (out, lse) if return_lse else out


class SharedPrefixAttention:
    """One decode step, attending to every token, of a paged batch whose sequences share prefixes in groups.

    ``group_sizes`` cuts the batch of ``kv`` into consecutive groups (a group of one shares nothing).  The first
    ``shared_lens[g]`` tokens (int32, device) of group ``g`` are the same for all its sequences; of those, the whole pages are
    read once for the group, through the table row of its longest sequence, and the rest of every sequence through its own row.
    Every row is complete and valid by itself, as ``PageCache.fork`` leaves it; a member may leave (length 0: its row is
    not read and its output is zeros).  ``kv.prefix_lens`` is not used.

    ``step`` reads the lengths and tables on the device, allocates its workspace and output from torch's allocator and
    does not synchronise: it can be captured (keep the object as long as the graph), and calls on several streams do not
    meet.  The tensors of ``kv`` and ``shared_lens`` are bound at construction: update them in place."""

    def __init__(self, kv: PagedKV, group_sizes: Sequence[int], shared_lens: torch.Tensor, n_q_heads: int):
        if n_q_heads <= 0 or n_q_heads % kv.n_kv_heads != 0:
            raise ValueError("query heads must be a multiple of kv heads")
        sizes = _host_lens("group_sizes", group_sizes)
        _need_cuda(shared_lens)
        if shared_lens.dtype != torch.int32 or not shared_lens.is_contiguous() or shared_lens.shape != (sizes.numel(),):
            raise ValueError("shared_lens must be a contiguous int32 tensor with one entry per group")
        self.kv, self.shared_lens, self.device = kv, shared_lens, kv.k_pool.device
        _same_device(self.device, v_pool=kv.v_pool, block_table=kv.block_table, seq_lens=kv.seq_lens, shared_lens=shared_lens)
        if kv.seq_lens.numel() != kv.batch:
            raise ValueError("kv.seq_lens has one entry per row of the block table")
        lib = _lib.load()
        self.geom = kv.geom(n_q_heads // kv.n_kv_heads, kv.page_size, 1)
        self._shape, self._dtype = (kv.batch, int(n_q_heads), kv.head_dim), kv.k_pool.dtype
        with torch.cuda.device(self.device):
            words = int(lib.ia_shared_prefix_plan_ints(_ptr(sizes), sizes.numel(), ctypes.byref(self.geom)))
            if words < 0:
                _lib.check(_lib.IA_ERR_UNSUPPORTED)
            plan = torch.zeros((words,), dtype=torch.int32)
            _lib.check(lib.ia_shared_prefix_plan(_ptr(sizes), sizes.numel(), ctypes.byref(self.geom), _ptr(plan), words))
            self._plan, self._parts = plan.to(self.device), int(plan[0])
            self._ws_bytes = int(lib.ia_shared_prefix_workspace_bytes(self._parts, ctypes.byref(self.geom)))
        self._call, self._index, self._q_shape = lib.ia_shared_prefix_decode, self.device.index, torch.Size(self._shape)
        self._streams = {_raw_stream(self._index)}
        self._held = (kv.k_pool, kv.v_pool, kv.block_table, kv.seq_lens)  # kv's fields may be given other tensors
        self._args = (_ptr(kv.k_pool), _ptr(kv.v_pool), _ptr(kv.block_table), _ptr(kv.seq_lens), _ptr(shared_lens),
                      _ptr(self._plan), self._parts, ctypes.byref(self.geom))

    def step(self, q: torch.Tensor, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q ``[B, Hq, D]`` -> ``[B, Hq, D]``."""
        if q.shape != self._q_shape or q.dtype is not self._dtype or q.get_device() != self._index or not q.is_contiguous():
            self._refuse("q", q)
        if out is None:
            out = torch.empty_like(q)
        elif out.shape != self._q_shape or out.dtype is not self._dtype or out.get_device() != self._index or not out.is_contiguous():
            self._refuse("out", out)
        ws = torch.empty((self._ws_bytes,), dtype=torch.uint8, device=self.device)
        stream = _raw_stream(self._index)
        if stream not in self._streams:
            wait_for(stream, self._streams, self._index, self._plan)
        with device_guard(self._index):
            _lib.check(self._call(q.data_ptr(), *self._args, ws.data_ptr(), self._ws_bytes, out.data_ptr(), stream))
        return out

    def _refuse(self, name: str, t: torch.Tensor) -> None:
        if t.is_cuda and t.shape == self._q_shape and t.dtype == self._dtype and t.is_contiguous():
            _same_device(self.device, **{name: t})
        raise ValueError(f"{name} must be a contiguous CUDA {self._shape} {self._dtype} tensor")
