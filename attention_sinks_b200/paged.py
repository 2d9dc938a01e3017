"""Paged K/V cache for a batch of sequences that may share a long prefix: append with the
rotation applied on the way, and decode attention that reads the shared rows once.

A sink cache gives every stream its own buffer of fixed length.  Here rows live in pages of a
pool, a sequence's pages are named by its row of a block table, and several sequences may name
the same pages: a prompt that a whole batch starts from is stored once, and
`PagedKVCache.attend(..., shared_len=P)` computes the attention over its P rows for all
queries together (one pass over those keys and values per kv head), merged with each
sequence's own rows.

One decode step of one layer:

    lens += 1                                     # once per step, for all layers
    q = cache.append(k, v, q=q)                   # rows lens - 1, rotated there; q rotated too
    out = cache.attend(q, shared_len=prefix)      # [B, 1, Hq, D]

Block table, lengths and counts are device tensors that the kernels read, so a captured CUDA
graph of the step serves every later token.  Its kernels read and write the cache's tensors:
keep the cache as long as the graph.
"""

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib
from .rope import device_frequencies, has_tangent, rotation


def _no_gradients(*inputs: torch.Tensor | None) -> None:
    """Refuse inputs that gradients or tangents are asked of: the cache keeps neither."""
    if (torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in inputs)) or has_tangent(*inputs):
        raise RuntimeError("the paged cache keeps no gradients or tangents: call it under torch.no_grad() or detach "
                           "its inputs (in forward mode, take their primals)")


def _scratch(nbytes: int, index: int, stream: int) -> torch.Tensor:
    """Scratch of `attend`, one buffer per (thread, device, stream): a call's two launches follow
    each other on their stream, so one thread's calls there can share one; another thread's
    launches may come between.  Inside a graph capture a fresh one comes from the graph's own
    pool, so that two graphs never share."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=index)
    buffers = _lib.forms("scratch")
    buf = buffers.get((index, stream))
    if buf is None or buf.numel() < nbytes:
        buf = buffers[index, stream] = torch.empty(nbytes, dtype=torch.uint8, device=index)
    return buf


class _AppendCall:
    """A checked form of `append` call, with the descriptors of its tensors."""

    def __init__(self, cache, k, v, q, counts):
        tokens = k.shape[2] if k.dim() == 4 else -1
        self.copy = [False] * 3
        for i, (name, x, heads) in enumerate((("k", k, cache.heads_kv), ("v", v, cache.heads_kv), ("q", q, None))):
            if x is not None:
                cache._check_rows(name, x, heads, tokens)
                self.copy[i] = x.stride(-1) != 1
        if counts is not None and (counts.shape != (cache.batch,) or counts.dtype != torch.int32
                                   or counts.device != cache.device or not counts.is_contiguous()):
            raise ValueError(f"counts is a contiguous int32 [{cache.batch}] tensor on {cache.device}")
        self.copies = any(self.copy)
        self.empty = not (tokens and cache.batch)
        k, v, q = (x if x is None else _lib.layout_of(x, c) for x, c in zip((k, v, q), self.copy))
        self.k, self.v = _lib.RowsArg(k), _lib.RowsArg(v)
        if q is not None:
            self.q, self.q_out = _lib.RowsArg(q), _lib.RowsArg(torch.empty_like(q))


class _AttendCall:
    """A checked form of `attend` call."""

    def __init__(self, cache, q, shared_len, aligned):
        cache._check_rows("q", q, None, 1)
        _lib.int32("shared_len", shared_len)
        b, hq, _, d = q.shape
        # the kernel's tiled copies start rows on 16-byte boundaries
        self.copy = (not aligned or q.stride(-1) != 1 or q.stride(0) % 8 or q.stride(1) % 8
                     or min(q.stride(0), q.stride(1)) < d)
        self.shape = (b, 1, hq, d)
        self.q = _lib.RowsArg(_lib.layout_of(q, self.copy))
        # shapes that the kernel refuses need nothing: the call says why
        self.workspace = max(256, _lib.paged_workspace_bytes(b, cache.heads_kv, hq, d, shared_len,
                                                             _lib.sm_count(cache.device)))


class PagedKVCache:
    """One layer's paged cache over tensors of the caller's.

    k_pages, v_pages: [pages, Hkv, page_size, D] pools (rows contiguous, page and head strides
    free), bfloat16, float16 or float32 (`attend` takes fewer forms than `append`: it says
    which).  block_table: int32 [B, width]; row p of sequence b is slot p % page_size of page
    block_table[b, p // page_size].  lens: int32 [B], the rows of each sequence, this step's
    tokens included; 0 for an idle sequence.  Both are read by the kernels when they run: update
    them in place.  Layers of one model share them, and may share `status` (a device int32 word
    that failures are recorded in).

    inv_freq (or None: keys and queries are stored and returned as they are), interleaved and
    attention_scaling are `rotary`'s.
    """

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                 inv_freq: torch.Tensor | None = None, interleaved: bool = False, attention_scaling: float = 1.0,
                 status: torch.Tensor | None = None):
        device = k_pages.device
        _lib.check_device(device)
        if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
            raise ValueError(f"pools are [pages, Hkv, page_size, D] of one shape and type, got {tuple(k_pages.shape)} "
                             f"{k_pages.dtype}, {tuple(v_pages.shape)} {v_pages.dtype}")
        pages, hkv, page, d = (_lib.int32("a pool's size", n) for n in k_pages.shape)
        for x in (k_pages, v_pages):
            if x.stride(-1) != 1 or (page > 1 and x.stride(-2) != d):
                raise ValueError("pages need contiguous rows (stride[-2] == head_dim, stride[-1] == 1)")
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(-1) != 1:
            raise ValueError("block_table is an int32 [B, width] tensor with a unit last stride")
        batch, width = (_lib.int32("a block table's size", n) for n in block_table.shape)
        if lens.shape != (batch,) or lens.dtype != torch.int32 or not lens.is_contiguous():
            raise ValueError(f"lens is a contiguous int32 [{batch}] tensor")
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=device)
        elif status.dtype != torch.int32 or status.numel() != 1:
            raise ValueError("status is one int32 word")
        for x in (v_pages, block_table, lens, status):
            if x.device != device:
                raise ValueError(f"the cache's tensors are on one device, got {device} and {x.device}")
        if inv_freq is not None and 2 * inv_freq.numel() > d:
            raise ValueError(f"{2 * inv_freq.numel()} rotated dims of a head of {d}")
        self.k_pages, self.v_pages, self.block_table, self.lens, self.status = k_pages, v_pages, block_table, lens, status
        self.device, self.dtype = device, k_pages.dtype
        self.batch, self.heads_kv, self.page_size, self.head_dim = batch, hkv, page, d
        self.inv_freq = None if inv_freq is None else device_frequencies(inv_freq, device)
        rot = None if inv_freq is None else rotation(self.inv_freq, interleaved, attention_scaling)
        self._kv = _lib.PagedKV(k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(), lens.data_ptr(),
                                status.data_ptr(), _lib.dtype_code(k_pages.dtype), batch, hkv, d, page, pages, width, 0,
                                block_table.stride(0), k_pages.stride(0), k_pages.stride(1), v_pages.stride(0),
                                v_pages.stride(1))
        self._rot = rot
        self._kv_ref, self._rot_ref = ctypes.byref(self._kv), None if rot is None else ctypes.byref(rot)
        self._index = device.index
        _lib.prepare_device(device)  # before any graph capture of this cache's steps
        self._like = (k_pages.dtype, batch, hkv, d, device)  # what a call's form depends on here
        self._fixed = frozenset((*self.__dict__, "_fixed"))

    _fixed = frozenset()  # names of the attributes that stay, once they are all there

    # The kernels read the memory that the attributes had when the cache was made, and the attributes
    # are what keeps it: they can be updated in place (`cache.lens += 1` too) and not replaced.
    def __setattr__(self, name: str, value) -> None:
        if name in self._fixed and value is not getattr(self, name):
            raise AttributeError(f"{name} of a paged cache cannot be replaced: update it in place, or make another "
                                 "cache over the new one")
        super().__setattr__(name, value)

    def __delattr__(self, name: str) -> None:
        if name in self._fixed:
            raise AttributeError(f"{name} of a paged cache cannot be removed")
        super().__delattr__(name)

    def _check_rows(self, name: str, x: torch.Tensor, heads: int | None, tokens: int) -> None:
        if (x.dim() != 4 or x.shape[0] != self.batch or (heads is not None and x.shape[1] != heads)
                or x.shape[2] != tokens or x.shape[3] != self.head_dim or x.dtype != self.dtype
                or x.device != self.device):
            raise ValueError(f"{name} is [{self.batch}, {heads or 'Hq'}, {tokens}, {self.head_dim}] {self.dtype} on "
                             f"{self.device}, got {tuple(x.shape)} {x.dtype} on {x.device}")

    def append(self, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None,
               counts: torch.Tensor | None = None) -> torch.Tensor | None:
        """Store the first counts[b] (all, when None) of the tokens k, v [B, Hkv, T, D] as the last
        rows of sequence b: rows lens[b] - counts[b] .. lens[b] - 1, k rotated to those
        positions.  Returns q [B, Hq, T, D] rotated to them too, in one launch (None without q).
        Tokens from counts[b] on, and all of an idle sequence's (lens 0), are not stored; their
        q rows come back as zeros.  counts: int32 [B] on the device.  Sequences may share pages that
        they read, not slots that they append to: a slot that two write in one call holds each
        value of its rows from one or the other."""
        if _lib.current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.append(k, v, q, counts)
        if forward_ad._current_level >= 0 or k.requires_grad or v.requires_grad or (q is not None and q.requires_grad):
            _no_gradients(k, v, q)
        form = (self._like, _lib.form_of(k), _lib.form_of(v), _lib.form_of(q), _lib.form_of(counts))
        known = _lib.forms("append")
        call = known.get(form)
        if call is None:
            call = known[form] = _AppendCall(self, k, v, q, counts)
        if call.copies:
            k, v, q = (x.contiguous() if c else x for x, c in zip((k, v, q), call.copy))
        q_out = None if q is None else torch.empty_like(q)
        if call.empty:
            return q_out
        rc = _lib.lib().sink_paged_append(self._kv_ref, call.k.at(k), call.v.at(v),
                                          None if counts is None else counts.data_ptr(),
                                          None if q is None else call.q.at(q),
                                          None if q is None else call.q_out.at(q_out), self._rot_ref,
                                          _lib.raw_stream(self._index))
        if rc:
            _lib._check(rc, "sink_paged_append")
        return q_out

    def attend(self, q: torch.Tensor, scale: float | None = None, shared_len: int = 0) -> torch.Tensor:
        """Attention of one query token per sequence, q [B, Hq, 1, D], over its rows
        [0, lens[b]): [B, 1, Hq, D] in q's type, zeros for an idle sequence.  `scale` defaults
        to D ** -0.5.  What is not finite comes out as the formula has it.

        The first `shared_len` rows (a multiple of the page size) are the same for all
        sequences: they are read through the first row of the block table, once per kv head
        for the whole batch.  bfloat16 or float16, head_dim 64 or 128, pages of 16, 32, 64 or
        128 rows, up to 8 query heads per kv head."""
        if _lib.current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.attend(q, scale, shared_len)
        if forward_ad._current_level >= 0 or q.requires_grad:
            _no_gradients(q)
        aligned = q.data_ptr() % 16 == 0
        form = (self._like, _lib.form_of(q), shared_len, aligned)
        known = _lib.forms("attend")
        call = known.get(form)
        if call is None:
            call = known[form] = _AttendCall(self, q, shared_len, aligned)
        if call.copy:
            q = q.clone(memory_format=torch.contiguous_format)
        out = q.new_empty(call.shape)
        if self.batch == 0:
            return out
        stream = _lib.raw_stream(self._index)
        work = _scratch(call.workspace, self._index, stream)
        rc = _lib.lib().sink_paged_attention(call.q.at(q), self._kv_ref, shared_len,
                                             self.head_dim ** -0.5 if scale is None else scale, out.data_ptr(),
                                             call.shape[2] * self.head_dim, self.head_dim, work.data_ptr(),
                                             work.numel(), stream)
        if rc:
            _lib._check(rc, "sink_paged_attention")
        return out

    def check_status(self) -> None:
        """Raise RuntimeError if a kernel met a position past the block table or a page outside
        the pool since the last check (nothing was accessed there); synchronises the stream."""
        st = ctypes.c_int32(0)
        with torch.cuda.device(self._index):
            _lib._check(_lib.lib().sink_read_status(self.status.data_ptr(), _lib.raw_stream(self._index),
                                                    ctypes.byref(st)), "sink_read_status")
        _lib.raise_status(st.value)
