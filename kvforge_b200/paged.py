"""Paged cache of many growing sequences, the attention of new tokens on it,
and eviction by the attention weight that its tokens have received.

What a serving program does with a cache before it hands a layer to the codec:
tokens are appended as they come, attended to from single tokens up to long
chunks, and thrown out when a budget runs out; `gather` gives one sequence of
one layer as the KVCache that `compress` takes. The reference has no cache of
its own. Everything runs on the GPU through the C ABI (kvf_paged_*,
include/kvforge.h); this module keeps the page tables.
"""
from __future__ import annotations

import array
import ctypes as C
import math
from typing import List, NamedTuple, Optional, Sequence

import numpy as np
import torch

from . import _lib as L
from ._lib import KvForgeError

# the current stream's handle without making a Stream object (1.2 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)

_DTYPES = {torch.float32: L.IN_F32, torch.float16: L.IN_F16, torch.bfloat16: L.IN_BF16}


def _ints(rows):
    """Lists of whole numbers as one host array of 32-bit rows of equal length
    (filled up with 0), and that length."""
    n = max([1] + [len(r) for r in rows])
    a = array.array("i", [0]) if not rows else array.array("i")
    for r in rows:
        a.extend(r)
        if len(r) < n:
            a.frombytes(bytes(4 * (n - len(r))))
    return (C.c_int32 * len(a)).from_buffer(a), n


class Eviction(NamedTuple):
    """What PagedKVCache.evict did: the sequences that hold the kept tokens, and
    kept [num_layers, sequences, num_heads, budget] i32: their slots before the
    eviction, in order, -1 behind the last."""
    seqs: List[int]
    kept: torch.Tensor


class _Sequence:
    __slots__ = ("pages", "length", "alive")

    def __init__(self, pages, length):
        self.pages = pages
        self.length = length
        self.alive = True


class PagedBatch:
    """The sequences and new tokens of one step (PagedKVCache.extend or .batch):
    made once, used for every layer. tokens: new tokens of all sequences, one
    after another; starts: the first token of each sequence, and their number."""

    def __init__(self, handle, owner, seqs, states, query_heads: int, starts: np.ndarray):
        self._h = handle
        self._owner = owner  # what its cache is told by (not the cache: a batch keeps no pages)
        self._states = states  # (sequence, its page list) as the plan saw them
        self.seqs = seqs
        self.query_heads = query_heads
        self.starts = starts
        self.tokens = int(starts[-1])

    def __del__(self):
        h = getattr(self, "_h", None)
        if h and L is not None and L._lib is not None:  # module globals are gone at interpreter exit
            L.lib().kvf_paged_plan_free(h)
            self._h = None


class PagedKVCache:
    """Keys and values of `num_layers` layers in pages of `page_size` tokens.

    keys, values: [num_layers, num_pages, num_heads, page_size, head_dim] of
    `dtype` (float16, bfloat16 or float32); weights: f32 [num_layers, num_pages,
    num_heads, page_size], the attention weight that each token has received
    (zero when it is appended). A sequence's token j lies in row j % page_size of
    its page j // page_size, the same pages in every layer.

    Calls are stream-ordered on the current stream; a call on another stream
    than the one before first waits for that one. One host thread at a time.
    append and attend can be captured in a CUDA graph on the stream that the
    batch was made on, attend with `decay` after one call of that batch with a
    `decay` (its workspace is not made inside a capture; nor is a batch). The
    batch must outlive the graph."""

    def __init__(self, num_pages: int, num_heads: int, head_dim: int, page_size: int = 64, num_layers: int = 1,
                 dtype: torch.dtype = torch.float16, device=None):
        from . import _device_index
        if dtype not in _DTYPES:
            raise TypeError(f"expected float32, float16 or bfloat16, got {dtype}")
        if page_size not in (16, 32, 64, 128):
            raise KvForgeError(L.ERR_INVALID_CONFIG, "page_size must be 16, 32, 64 or 128")
        if not 1 <= head_dim <= 256:
            raise KvForgeError(L.ERR_SHAPE_MISMATCH, "head_dim must be in 1..256")
        if min(num_pages, num_heads, num_layers) < 1:
            raise KvForgeError(L.ERR_SHAPE_MISMATCH, "num_pages, num_heads and num_layers must be at least 1")
        self._dev = _device_index(device)
        self.num_layers, self.num_pages, self.num_heads = int(num_layers), int(num_pages), int(num_heads)
        self.page_size, self.head_dim, self.dtype = int(page_size), int(head_dim), dtype
        where = f"cuda:{self._dev}"
        shape = (self.num_layers, self.num_pages, self.num_heads, self.page_size)
        self.keys = torch.zeros(shape + (self.head_dim,), dtype=dtype, device=where)
        self.values = torch.zeros(shape + (self.head_dim,), dtype=dtype, device=where)
        self.weights = torch.zeros(shape, dtype=torch.float32, device=where)
        self._pool = L.PagedPool(_DTYPES[dtype], self.page_size, self.num_layers, self.num_pages, self.num_heads,
                                 self.head_dim, self.keys.data_ptr(), self.values.data_ptr(),
                                 self.weights.data_ptr())
        self._pool_ref = C.byref(self._pool)
        self._lib, self._ctx = L.lib(), L.context(self._dev)
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self._free = list(range(self.num_pages - 1, -1, -1))  # the lowest page is handed out first
        self._seqs = {}
        self._self = object()
        self._next = 0
        self._last = torch.cuda.current_stream(self._dev)
        self._last_raw = self._last.cuda_stream

    # ---- sequences ------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _seq(self, seq: int) -> _Sequence:
        s = self._seqs.get(seq)
        if s is None:
            raise KvForgeError(L.ERR_INVALID_CONFIG, f"no sequence {seq}")
        return s

    def _take(self, n: int) -> list:
        if n > len(self._free):
            raise KvForgeError(L.ERR_PIPELINE, f"{n} pages needed, {len(self._free)} free")
        taken = self._free[len(self._free) - n:][::-1]
        del self._free[len(self._free) - n:]
        return taken

    def _give(self, pages) -> None:
        self._free.extend(reversed(pages))

    def _pages_for(self, length: int) -> int:
        return -(-length // self.page_size)

    def add(self, length: int = 0, pages: Optional[Sequence[int]] = None) -> int:
        """A new sequence of `length` tokens whose rows the caller fills (0: an
        empty one). pages: the free pages to use, in order (more than `length`
        needs are kept for later tokens); by default any."""
        length = int(length)
        if length < 0:
            raise KvForgeError(L.ERR_SHAPE_MISMATCH, "negative length")
        if pages is None:
            pages = self._take(self._pages_for(length))
        else:
            pages = [int(p) for p in pages]
            if len(pages) < self._pages_for(length):
                raise KvForgeError(L.ERR_SHAPE_MISMATCH, "fewer pages than the length needs")
            want = set(pages)
            if len(want) != len(pages) or not want <= set(self._free):
                raise KvForgeError(L.ERR_INVALID_CONFIG, "pages must be free, each named once")
            self._free = [p for p in self._free if p not in want]
        seq = self._next
        self._next += 1
        self._seqs[seq] = _Sequence(pages, length)
        return seq

    def free(self, seqs) -> None:
        """Gives the sequences' pages back."""
        seqs = self._ids(seqs)
        for seq in reversed(seqs):
            s = self._seqs.pop(seq)
            s.alive = False
            self._give(s.pages)

    def length(self, seq: int) -> int:
        return self._seq(seq).length

    def pages(self, seq: int) -> List[int]:
        """The sequence's pages, in order."""
        return list(self._seq(seq).pages)

    def _ids(self, seqs) -> list:
        seqs = [int(seqs)] if isinstance(seqs, (int, np.integer)) else [int(s) for s in seqs]
        if len(set(seqs)) != len(seqs):
            raise KvForgeError(L.ERR_INVALID_CONFIG, "a sequence is named twice")
        for s in seqs:
            self._seq(s)
        return seqs

    # ---- one step's batch -------------------------------------------------------
    def extend(self, seqs, new_tokens, query_heads: int = 0, window: int = 0, sinks: int = 0) -> PagedBatch:
        """Makes room for new_tokens[i] tokens behind sequence seqs[i] and returns
        the batch that `append` and `attend` take. query_heads: heads of the
        queries (a multiple of num_heads), 0 when the batch is only appended.
        window: a query sees the last `window` tokens up to its own (0: all),
        and the first `sinks` tokens."""
        seqs = self._ids(seqs)
        new = [int(n) for n in ([new_tokens] if isinstance(new_tokens, (int, np.integer)) else new_tokens)]
        if len(new) != len(seqs) or any(n < 0 for n in new):
            raise KvForgeError(L.ERR_SHAPE_MISMATCH, "one number of new tokens, 0 or more, per sequence")
        states = [self._seqs[s] for s in seqs]
        need = [max(0, self._pages_for(s.length + n) - len(s.pages)) for s, n in zip(states, new)]
        if sum(need) > len(self._free):
            raise KvForgeError(L.ERR_PIPELINE, f"{sum(need)} pages needed, {len(self._free)} free")
        before = [s.length for s in states]
        for s, n, k in zip(states, new, need):
            if k:
                s.pages = s.pages + self._take(k)
            s.length += n
        try:
            return self.batch(seqs, new, query_heads, window, sinks)
        except Exception:
            for s, n in zip(states, before):  # the pages stay with the sequence
                s.length = n
            raise

    def batch(self, seqs, query_tokens, query_heads: int = 0, window: int = 0, sinks: int = 0) -> PagedBatch:
        """The batch of the last query_tokens[i] cached tokens of each sequence,
        without making room for more: `extend` after the fact, or another
        window on the same step. More queries than cached tokens are allowed;
        the first ones then see nothing."""
        seqs = self._ids(seqs)
        q = [int(n) for n in ([query_tokens] if isinstance(query_tokens, (int, np.integer)) else query_tokens)]
        if len(q) != len(seqs) or any(n < 0 for n in q):
            raise KvForgeError(L.ERR_SHAPE_MISMATCH, "one number of tokens, 0 or more, per sequence")
        states = [self._seqs[s] for s in seqs]
        h = self._plan(states, q, query_heads, window, sinks)
        starts = np.zeros(len(q) + 1, np.int64)
        np.cumsum(q, out=starts[1:])
        return PagedBatch(h, self._self, seqs, states, int(query_heads), starts)

    def _plan(self, states, q, query_heads, window, sinks) -> C.c_void_p:
        kv, _ = _ints([[s.length for s in states]])
        ql, _ = _ints([q])
        table, stride = _ints([s.pages for s in states])
        # ctypes cuts whole numbers to 32 bits: longer ones than any sequence mean the same as 2^31 - 1
        window, sinks = (max(-1, min(int(x), 2 ** 31 - 1)) for x in (window, sinks))
        h = C.c_void_p()
        L.check(self._lib.kvf_paged_plan_create(self._ctx, self._pool_ref, len(states), ql, kv, table, stride,
                                                int(query_heads), window, sinks, C.byref(h), self._enter()))
        return h

    def _enter(self) -> int:
        """The current stream, ordered behind the last call's."""
        raw = _raw_stream(self._dev)
        if raw != self._last_raw:
            s = torch.cuda.current_stream(self._dev)
            s.wait_stream(self._last)
            for t in (self.keys, self.values, self.weights):
                t.record_stream(s)  # the pool's memory is not reused before this stream is done with it
            self._last, self._last_raw = s, raw
        return raw

    def _handle(self, batch: PagedBatch):
        if batch._owner is not self._self:
            raise KvForgeError(L.ERR_INVALID_CONFIG, "the batch belongs to another cache")
        for s in batch._states:
            if not s.alive:
                raise KvForgeError(L.ERR_INVALID_CONFIG, "a sequence of the batch was freed or evicted")
        return batch._h

    def _rows(self, x: torch.Tensor, name: str, tokens: int, heads: int) -> torch.Tensor:
        if not isinstance(x, torch.Tensor) or x.dtype != self.dtype:
            raise TypeError(f"{name}: expected a {self.dtype} tensor, got {getattr(x, 'dtype', type(x))}")
        if x.shape != (tokens, heads, self.head_dim):
            raise KvForgeError(L.ERR_SHAPE_MISMATCH,
                               f"{name}: expected {(tokens, heads, self.head_dim)}, got {tuple(x.shape)}")
        if not x.is_cuda or x.device.index != self._dev:
            raise KvForgeError(L.ERR_INVALID_CONFIG, f"{name}: expected a tensor on cuda:{self._dev}")
        return x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.num_layers:
            raise KvForgeError(L.ERR_SHAPE_MISMATCH, f"layer {layer} of {self.num_layers}")
        return layer

    def sync(self) -> None:
        """Waits for the cache's calls so far, and raises KvForgeError when a
        kernel of theirs gave up a bounded wait (KVF_ERR_DEVICE_TIMEOUT: what it was
        to write is unfinished) or when one of the codec's reported an error: the
        device has one status word, which the first call that reads it clears.
        Nothing else here waits for the GPU or looks."""
        L.check(self._lib.kvf_sync(self._ctx, self._enter()))

    # ---- operators ----------------------------------------------------------------
    def append(self, batch: PagedBatch, keys: torch.Tensor, values: torch.Tensor, layer: int = 0) -> None:
        """Writes the batch's new tokens, keys and values [tokens, num_heads,
        head_dim] (any strides), into one layer; their weights become 0."""
        h = self._handle(batch)
        k = self._rows(keys, "keys", batch.tokens, self.num_heads)
        v = self._rows(values, "values", batch.tokens, self.num_heads)
        L.check(self._lib.kvf_paged_append(self._ctx, h, self._pool_ref, self._layer(layer), k.data_ptr(), k.stride(0),
                                           k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), self._enter()))

    def attend(self, batch: PagedBatch, query: torch.Tensor, layer: int = 0, scale: Optional[float] = None,
               decay: Optional[float] = None, return_lse: bool = False):
        """Attention of the batch's tokens, query [tokens, query_heads, head_dim]
        (any strides), over the cache, their own rows included (append them
        first): softmax(scale * q . k) v over what each token sees. scale
        defaults to 1/sqrt(head_dim). decay: None leaves `weights` alone;
        otherwise each token of the batch's sequences gets weight = decay *
        weight + the attention that it received here from all of its KV head's
        queries (1: the sum over all steps, 0: this step's alone). Returns the
        output, contiguous, of the cache's dtype, and with return_lse also the f32
        logarithm of the softmax's sum [tokens, query_heads]."""
        h = self._handle(batch)
        if not batch.query_heads:
            raise KvForgeError(L.ERR_INVALID_CONFIG, "the batch was made without query_heads")
        q = self._rows(query, "query", batch.tokens, batch.query_heads)
        if decay is not None and not 0.0 <= decay <= 1.0:
            raise KvForgeError(L.ERR_INVALID_CONFIG, "decay must be in 0..1")
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = self.weights.new_empty(q.shape[:2]) if return_lse else None
        L.check(self._lib.kvf_paged_attention(
            self._ctx, h, self._pool_ref, self._layer(layer), q.data_ptr(), q.stride(0), q.stride(1),
            self._scale if scale is None else float(scale), -1.0 if decay is None else float(decay),
            out.data_ptr(), lse.data_ptr() if return_lse else None, self._enter()))
        return (out, lse) if return_lse else out

    def evict(self, seqs, budget: int, recent: int = 0, sinks: int = 0, keep_source: bool = False) -> Eviction:
        """Shortens each sequence to `budget` tokens, in every layer and KV head on
        its own: the first `sinks`, the last `recent`, and of the others those
        with the largest weight (among equals the earliest; NaN below every
        number), in order, with their weights. A shorter sequence keeps all. The
        kept tokens move to free pages, which must be there; then the old pages
        are given back, or, with keep_source, stay as they are and the kept tokens
        become new sequences (a branch)."""
        seqs = self._ids(seqs)
        budget = int(budget)
        if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget:
            raise KvForgeError(L.ERR_INVALID_CONFIG, "budget must be at least 1 and hold the sinks and recent tokens")
        states = [self._seqs[s] for s in seqs]
        lens = [min(budget, s.length) for s in states]
        # (first: where memory runs out, no page has been taken)
        kept = self.weights.new_empty((self.num_layers, len(seqs), self.num_heads, budget), dtype=torch.int32)
        taken = self._take(sum(self._pages_for(n) for n in lens))
        lists, at = [], 0
        for n in lens:
            lists.append(taken[at:at + self._pages_for(n)])
            at += len(lists[-1])
        try:
            kv, _ = _ints([[s.length for s in states]])
            table, stride = _ints([s.pages for s in states])
            new, new_stride = _ints(lists)
            L.check(self._lib.kvf_paged_evict(self._ctx, self._pool_ref, len(states), kv, table, stride, budget,
                                              int(recent), int(sinks), new, new_stride, kept.data_ptr(),
                                              self._enter()))
        except Exception:
            self._give(taken)
            raise
        fresh = [_Sequence(p, n) for p, n in zip(lists, lens)]
        if keep_source:
            out = list(range(self._next, self._next + len(seqs)))
            self._next += len(seqs)
        else:
            out = seqs
            for s in reversed(states):
                s.alive = False
                self._give(s.pages)
        self._seqs.update(zip(out, fresh))
        return Eviction(out, kept)

    def gather(self, seq: int, layer: int = 0):
        """One sequence of one layer out of its pages, as a KVCache [num_heads,
        tokens, head_dim] of the cache's dtype: what `compress` takes (the codec
        reads float16 and float32)."""
        from . import KVCache
        s = self._seq(seq)
        shape = (self.num_heads, s.length, self.head_dim)
        k, v = self.keys.new_empty(shape), self.keys.new_empty(shape)
        pages, _ = _ints([s.pages])
        L.check(self._lib.kvf_paged_gather(self._ctx, self._pool_ref, self._layer(layer), pages, s.length,
                                           k.data_ptr(), v.data_ptr(), self._enter()))
        return KVCache(k, v, layer)
