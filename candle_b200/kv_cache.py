"""A KV cache in pages, and the attention of a decode batch that reads it.

candle's quantized models keep one tensor [batch, heads, positions, head_dim] per layer (candle-transformers/src/models/quantized_llama.rs:235-245): every
sequence has its own copy of all it has read, and all have one length.  Here sequences ("slots") have their own lengths, their keys and values lie in pages
of one pool, and a sequence that goes on from another one shares its full pages:

    cache = PagedKvCache(layers, pages, page_size, kv_heads, head_dim, max_seqs, max_len)
    cache.reserve([0], n)                               # positions for a prompt of n tokens
    q = cache.append(layer, [0], k, v, q=q, rotary=(cos, sin))
    cache.fork([0] * 7, range(1, 8))                    # seven more continuations of it
    plan = cache.attention_plan(8, heads)               # one group: all eight share a prefix
    ...                                                 # per step:
    cache.reserve(slots, 1); plan.update(slots)
    out = cache.attention(layer, q, plan)               # per layer

Nothing here but `check()` waits for the device or looks at its numbers: a step can be captured into a CUDA graph (slots given as an
int32 tensor of the device).  What the device finds wrong - no page left, a slot named twice, ... - leaves the bookkeeping as it was, stops every later change, and is
raised by `check()`.  Calls on one cache are ordered by the caller: one stream, or events between several.
"""
from __future__ import annotations

import ctypes as C
import math
import operator

import numpy as np
import torch

from . import capi
from .capi import CandleQError

_ELEM = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}


def _whole(values, what: str) -> list[int]:
    try:
        return [operator.index(v) for v in values]
    except TypeError:
        raise CandleQError(f"{what} must be a list of whole numbers") from None


class PagedKvCache:
    """`pages` pages of `page_size` (16, 32, 64, 128) positions for all layers; at most `max_seqs` sequences of at most `max_len` positions.  `k`, `v`:
    [layers, pages, kv_heads, page_size, head_dim]; `refs` [pages], `lens` [max_seqs] and `tables` [max_seqs, max_pages] (-1 behind a sequence's pages) are views
    of the bookkeeping, int32.  `pools`: the two tensors, where the caller has made them."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, max_seqs: int, max_len: int, dtype: torch.dtype = torch.float32,
                 device="cuda:0", pools=None):
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise CandleQError("PagedKvCache needs a CUDA device: there is no CPU path")
        if dtype not in _ELEM:
            raise CandleQError(f"Expected f32/f16/bf16, got {dtype}")
        if page_size <= 0 or max_len <= 0:
            raise CandleQError("PagedKvCache: page_size and max_len must be positive")
        max_pages = -(-max_len // page_size)
        shape = (layers, pages, kv_heads, page_size, head_dim)
        if min(shape) <= 0 or max_seqs <= 0:
            raise CandleQError("PagedKvCache: sizes must be positive")
        if pools is None:
            pools = (torch.zeros(shape, dtype=dtype, device=self.device), torch.zeros(shape, dtype=dtype, device=self.device))
        for t in pools:
            if t.shape != shape or t.dtype != dtype or t.device != pools[0].device or not t.is_cuda or not t.is_contiguous():
                raise CandleQError(f"PagedKvCache: the pools must be contiguous CUDA tensors {list(shape)} of {dtype}")
        self.k, self.v = pools
        self.device = self.k.device
        self._index = self.device.index
        lib = capi.lib()
        # rounded up, so that a view of everything keeps its alignment
        self.state = torch.zeros(capi.pad(lib.cq_kv_state_ints(pages, max_seqs, max_pages), 4), dtype=torch.int32, device=self.device)
        self._c = capi.KvCache(self.k.data_ptr(), self.v.data_ptr(), self.state.data_ptr(), layers, pages, kv_heads, page_size, head_dim, max_seqs, max_pages,
                               _ELEM[dtype])
        self._p = C.byref(self._c)
        self.layers, self.pages, self.page_size, self.kv_heads, self.head_dim = layers, pages, page_size, kv_heads, head_dim
        self.max_seqs, self.max_len, self.dtype = max_seqs, max_pages * page_size, dtype
        at = 16
        self.refs, at = self.state[at:at + pages], at + pages
        self.lens, at = self.state[at:at + max_seqs], at + max_seqs
        self.tables = self.state[at:at + max_seqs * max_pages].view(max_seqs, max_pages)
        self.reset()

    # ---- helpers ----
    def _call(self, fn, *args) -> None:
        if torch.cuda.current_device() == self._index:
            fn(self._p, *args, capi.stream_of(self.device))
        else:
            with torch.cuda.device(self.device):
                fn(self._p, *args, capi.stream_of(self.device))
        capi.check("PagedKvCache")

    def slot_list(self, slots) -> torch.Tensor:
        """Slots as the device reads them: int32, contiguous, on the cache's device.  Such a tensor is taken as it is; numbers of the host are copied there."""
        if isinstance(slots, torch.Tensor):
            if slots.dtype == torch.int32 and slots.device == self.device and slots.dim() == 1 and slots.is_contiguous() and slots.shape[0] <= self.max_seqs:
                return slots
        else:
            slots = _whole([slots] if isinstance(slots, int) else slots, "PagedKvCache: slots")
            if any(not 0 <= s < self.max_seqs for s in slots):
                raise CandleQError(f"PagedKvCache: slots are 0 .. {self.max_seqs - 1}")
            if len(slots) <= self.max_seqs:
                return torch.tensor(slots, dtype=torch.int32).to(self.device, non_blocking=True)       # pageable memory: copied aside before this returns
            slots = torch.tensor(slots, dtype=torch.int32)
        if slots.dim() != 1 or slots.is_floating_point() or slots.is_complex() or slots.dtype == torch.bool:
            raise CandleQError("PagedKvCache: slots must be a list of whole numbers")
        if slots.numel() > self.max_seqs:
            raise CandleQError(f"PagedKvCache: {slots.numel()} slots named, the cache has {self.max_seqs}")
        if slots.dtype in (torch.int64, torch.uint32, torch.uint64):
            slots = slots.to(torch.int64).clamp(-1, self.max_seqs)         # what int32 does not hold stays out of range
        return slots.to(device=self.device, dtype=torch.int32).contiguous()

    # ---- pages ----
    def reset(self) -> None:
        """Every slot empty, every page free, no fault."""
        self._call(capi.lib().cq_kv_reset)

    def reserve(self, slots, tokens: int) -> None:
        """`tokens` more positions for each of the slots.  The lowest free pages are taken, in the order of the list."""
        s = self.slot_list(slots)
        if tokens < 0 or tokens > self.max_len:
            raise CandleQError(f"PagedKvCache.reserve: {tokens} tokens, a sequence holds 0 .. {self.max_len}")
        self._call(capi.lib().cq_kv_reserve, s.data_ptr(), s.numel(), tokens)

    def fork(self, src, dst) -> None:
        """The empty slots dst[i] go on from src[i] (one source may be named many times): full pages are shared, a part-full last page is copied."""
        self._fork(src, dst, 0)

    def copy(self, src, dst) -> None:
        """Like `fork`, with pages of their own for all positions."""
        self._fork(src, dst, 1)

    def _fork(self, src, dst, deep: int) -> None:
        a, b = self.slot_list(src), self.slot_list(dst)
        if a.numel() != b.numel():
            raise CandleQError("PagedKvCache.fork: one destination for each source")
        self._call(capi.lib().cq_kv_fork, a.data_ptr(), b.data_ptr(), a.numel(), deep)

    def free(self, slots) -> None:
        """The slots become empty; pages that no other slot shares are free."""
        s = self.slot_list(slots)
        self._call(capi.lib().cq_kv_free, s.data_ptr(), s.numel())

    def compact(self) -> None:
        """Moves the live pages to the front of the pool (n live pages: the numbers 0 .. n - 1), tables included."""
        self._call(capi.lib().cq_kv_compact)

    def check(self) -> None:
        """Raises if a call since the last check found a fault on the device (synchronises the stream)."""
        with capi.on_device(self.device):
            fault = capi.lib().cq_kv_take_fault(self._p, capi.stream_of(self.device))
        if fault:
            capi.check("PagedKvCache")
            raise CandleQError("PagedKvCache: the state could not be read")

    # ---- keys and values ----
    def _rows(self, t: torch.Tensor, name: str, batch: int, heads: int | None, tokens: int | None):
        """`t` as [batch, tokens, heads, head_dim] with heads side by side and aligned rows at one distance; (tensor, row distance)."""
        shape, d = t.shape, self.head_dim
        if len(shape) != 4 or shape[0] != batch or shape[3] != d or (heads is not None and shape[2] != heads) or (tokens is not None and shape[1] != tokens) or \
                t.get_device() != self._index:
            raise CandleQError(f"PagedKvCache: {name} must be [batch, tokens, heads, {d}] on {self.device}, got {list(shape)}")
        width = shape[2] * d
        if t.is_contiguous():
            return (t if t.data_ptr() % 16 == 0 else t.clone()), width
        stride = t.stride(1) if shape[1] > 1 else t.stride(0)
        if t.stride(3) != 1 or (shape[2] > 1 and t.stride(2) != d) or stride < width or (batch > 1 and t.stride(0) != stride * shape[1]) or \
                stride * t.element_size() % 16 or t.data_ptr() % 16:
            return t.contiguous(), width
        return t, stride

    def append(self, layer: int, slots, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None, rotary=None, neox: bool = False):
        """Keys and values [batch, tokens, kv_heads, head_dim] (f32, f16, bf16) of the last `tokens` positions of the slots, which `reserve` has added (a position in a
        page that other slots share is a fault; with a fault in any row nothing is stored, and zeros are returned).  With
        `rotary` = (cos, sin), each [positions, head_dim / 2] f32, k and q are rotated at their sequence's own positions: pairs (2i, 2i + 1), with `neox`
        (i, i + head_dim / 2).  Returns q [batch, tokens, heads, head_dim] in the cache's type, or None."""
        s = self.slot_list(slots)
        if not 0 <= layer < self.layers:
            raise CandleQError(f"PagedKvCache.append: layer {layer} of {self.layers}")
        elem = _ELEM.get(k.dtype)
        if elem is None or v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
            raise CandleQError("PagedKvCache.append: q, k and v must be of one type, f32, f16 or bf16")
        b = s.shape[0]
        if b == 0 or k.dim() != 4 or k.shape[1] == 0:
            raise CandleQError("PagedKvCache.append: no slots or no tokens")
        tokens = k.shape[1]
        k, ks = self._rows(k, "k", b, self.kv_heads, tokens)
        v, vs = self._rows(v, "v", b, self.kv_heads, tokens)
        qs, out, heads, q_at, out_at = 0, None, 0, None, None
        if q is not None:
            q, qs = self._rows(q, "q", b, None, tokens)
            heads = q.shape[2]
            out = torch.empty_like(q, dtype=self.dtype, memory_format=torch.contiguous_format)
            q_at, out_at = q.data_ptr(), out.data_ptr()
        cos_at = sin_at = None
        positions = 0
        if rotary is not None:
            cos, sin = rotary
            positions = cos.shape[0]
            cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
            want = (positions, self.head_dim // 2)
            if positions == 0 or cos.shape != want or sin.shape != want or cos.dtype != torch.float32 or sin.dtype != torch.float32 or not cos.is_contiguous() or \
                    not sin.is_contiguous() or cos.get_device() != self._index or sin.get_device() != self._index or (cos_at | sin_at) % 16:
                raise CandleQError(f"PagedKvCache.append: rotary tables must be contiguous, aligned f32 [positions, {self.head_dim // 2}] on {self.device}")
        self._call(capi.lib().cq_kv_append, layer, s.data_ptr(), b, tokens, q_at, k.data_ptr(), v.data_ptr(), elem, heads, qs, ks, vs, cos_at, sin_at, positions, int(neox),
                   out_at)
        return out

    # ---- attention ----
    def attention_plan(self, batch: int, heads: int, queries: int = 1, groups=None) -> "AttentionPlan":
        """What `attention` needs for a batch of this shape: `queries` tokens of each of `batch` sequences.  `groups`: how many neighbouring sequences go on from
        the same prompt, a list that adds up to `batch`; None: all of them."""
        return AttentionPlan(self, batch, heads, queries, groups)

    def attention(self, layer: int, q: torch.Tensor, plan: "AttentionPlan", scale: float | None = None) -> torch.Tensor:
        """softmax(scale q K^T) V of the last `queries` positions of the plan's slots, each over the positions up to its own; scale: 1 / sqrt(head_dim).
        q: [batch, queries, heads, head_dim] of the cache's type.  A sequence without positions gives zeros."""
        if plan.cache is not self:
            raise CandleQError("PagedKvCache.attention: the plan belongs to another cache")
        if not 0 <= layer < self.layers:
            raise CandleQError(f"PagedKvCache.attention: layer {layer} of {self.layers}")
        if not plan.updated:
            raise CandleQError("PagedKvCache.attention: the plan has no slots yet (AttentionPlan.update)")
        if q.dtype != self.dtype:
            raise CandleQError(f"PagedKvCache.attention: q must be of the cache's type, {self.dtype}")
        q, stride = self._rows(q, "q", plan.batch, plan.heads, plan.queries)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        self._call(capi.lib().cq_prefix_attention, layer, plan._p, q.data_ptr(), stride, out.data_ptr(), 1.0 / math.sqrt(self.head_dim) if scale is None else scale)
        return out


class AttentionPlan:
    """The division of a batch's attention into pieces, and the room for their results.  `update(slots)` makes it for the lengths and tables as they are, once a
    step; all layers use it.  One plan serves one stream at a time, and like any tensor it must outlive its use on a stream other than the one it was made on."""

    def __init__(self, cache: PagedKvCache, batch: int, heads: int, queries: int, groups):
        groups = [batch] if groups is None else _whole(groups, "attention_plan: groups")
        if any(g <= 0 for g in groups) or sum(groups) != batch:
            raise CandleQError(f"attention_plan: groups {groups} must be positive and add up to the batch of {batch}")
        self.cache, self.batch, self.heads, self.queries, self.updated = cache, batch, heads, queries, False
        self._c = capi.PrefixPlan(batch=batch, queries=queries, heads=heads, groups=len(groups))
        self._p = C.byref(self._c)
        sizes = np.array(groups, dtype=np.int32)
        shapes = np.zeros(4 * len(groups), dtype=np.int32)
        with capi.on_device(cache.device):
            if capi.lib().cq_prefix_plan_shape(cache._p, self._p, sizes.ctypes.data, shapes.ctypes.data):
                capi.check("attention_plan")
        self._ints = torch.zeros(self._c.n_ints, dtype=torch.int32, device=cache.device)
        self._scratch = torch.empty(self._c.n_floats, dtype=torch.float32, device=cache.device)
        self._ints[16:16 + shapes.size].copy_(torch.from_numpy(shapes))
        self._c.ints, self._c.scratch = self._ints.data_ptr(), self._scratch.data_ptr()

    def update(self, slots) -> None:
        s = self.cache.slot_list(slots)
        if s.numel() != self.batch:
            raise CandleQError(f"AttentionPlan.update: {s.numel()} slots for a batch of {self.batch}")
        self._slots = s             # read on the device after this returns
        self.cache._call(capi.lib().cq_prefix_plan_update, self._p, s.data_ptr())
        self.updated = True
