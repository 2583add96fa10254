"""Paged KV cache of many sequences (fl_pages_* of include/flare_hip.h).

`PagedKv` holds a pool of pages and sequences that are lists of pages: forks
share what they have in common, a page is copied when one of them would write to
it, and `attention` reads a page that several of the batch's sequences hold once
for all of them.  Where flarellm's caches (flare-core/src/kv_cache.rs:431-546) hold
one sequence, this holds a batch: several answers to one prompt, beams, chats
behind one system prompt.

Work is enqueued on the backend's stream.  Calls made with another current torch
stream order the two streams by events, so tensors go in and come out as with any
torch operation; calls do not wait for the GPU (but where their lists outgrow their memory).
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import FL_KV_F16, FL_KV_F32, FL_KV_Q8, FlareError, PagesConfig, check


def _ids(x, what: str, n: int = -1) -> np.ndarray:
    a = np.asarray(x)
    if a.dtype != np.int32 or a.ndim != 1:
        if a.ndim != 1 or (a.size and a.dtype.kind not in "iu"):
            raise ValueError(f"{what}: a list of whole numbers")
        if a.size and (a.max() > 2**31 - 1 or a.min() < -(2**31)):
            raise ValueError(f"{what}: out of range")
        a = a.astype(np.int32)
    if n >= 0 and a.size != n:
        raise ValueError(f"{what}: {a.size} values for {n} sequences")
    return a


class PagedKv:
    """A pool of `pages` pages of `page_size` tokens for sequences 0..max_seqs-1."""

    def __init__(self, backend, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 kv_format: int = FL_KV_F16, max_seqs: int = 64, max_len: int = 0):
        import torch

        self._h = None
        self._b = backend
        self.lib = backend.lib
        self.layers, self.pages, self.page_size = layers, pages, page_size
        self.kv_heads, self.head_dim, self.kv_format = kv_heads, head_dim, kv_format
        self.max_seqs, self.max_len = max_seqs, max_len or min(pages * page_size, 1 << 24)
        cfg = PagesConfig(layers, kv_heads, head_dim, kv_format, pages, page_size, max_seqs, self.max_len)
        check(self.lib.fl_pages_bytes(C.byref(cfg), None, None))
        self.device = torch.device("cuda", self.lib.fl_ctx_device(backend.ctx))
        dtype = {FL_KV_F32: torch.float32, FL_KV_F16: torch.float16, FL_KV_Q8: torch.int8}[kv_format]
        kw = dict(dtype=dtype, device=self.device)
        #: K [layer, page, kv head, slot, head_dim], V [layer, page, kv head, slot / 32, head_dim, 32]
        self.k = torch.empty(layers, pages, kv_heads, page_size, head_dim, **kw)
        self.v = torch.empty(layers, pages, kv_heads, page_size // 32, head_dim, 32, **kw)
        #: 8-bit form: binary16 scale per 32 channels [layer, page, kv head, slot, head_dim / 32]
        self.k_scale = self.v_scale = None
        if kv_format == FL_KV_Q8:
            self.k_scale, self.v_scale = (torch.empty(layers, pages, kv_heads, page_size, head_dim // 32,
                                                      dtype=torch.float16, device=self.device) for _ in "kv")
        #: the backend's stream: with it as the current one, calls need no events
        self.stream = torch.cuda.ExternalStream(backend.stream, device=self.device)
        self._stream = self.stream.cuda_stream
        self._current, self._index = torch._C._cuda_getCurrentRawStream, self.device.index
        self._row = (kv_heads, head_dim)
        self._torch = torch  # (an import statement costs a call 0.3 us)
        self._before, self._behind = torch.cuda.Event(), torch.cuda.Event()  # (kept: making one costs 10 us)
        # the memory may be what earlier work of the current stream still uses
        self.stream.wait_stream(torch.cuda.current_stream(self.device))
        h = C.c_void_p()
        check(self.lib.fl_pages_create(backend.ctx, C.byref(cfg), *(None if t is None else t.data_ptr() for t in
                                       (self.k, self.v, self.k_scale, self.v_scale)), C.byref(h)), backend.ctx)
        self._h = h

    def close(self):
        if self._h:
            if self._b.ctx:
                self._b.sync()  # the tensors' memory goes back to torch
            self.lib.fl_pages_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _open(self):
        if not self._h or not self._b.ctx:
            raise FlareError("the paged cache or its backend is closed")

    def _call(self, fn, *args):
        self._open()
        rc = fn(self._h, *args)
        if rc:
            check(rc, self._b.ctx)

    def _enqueue(self, fn, *args):
        """_call behind the current torch stream's work, and before what follows there."""
        if self._current(self._index) == self._stream:
            return self._call(fn, *args)
        torch = self._torch
        current = torch.cuda.current_stream(self.device)
        self._before.record(current)
        self.stream.wait_event(self._before)
        try:
            self._call(fn, *args)
        finally:
            self._behind.record(self.stream)
            current.wait_event(self._behind)

    def _rows(self, t, what: str, shape):
        """A float32 tensor on this device whose last dimensions are `shape`, without gaps between them."""
        torch = self._torch
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.float32 or t.get_device() != self._index:
            raise ValueError(f"{what}: a float32 tensor on {self.device}")
        n = len(shape)
        if t.shape[-n:] != shape:
            raise ValueError(f"{what}: {tuple(t.shape)}, not [.., {', '.join(map(str, shape))}]")
        if t.is_contiguous():
            return
        want = 1
        for size, stride in zip(reversed(shape), reversed(t.stride()[-n:])):
            if size != 1 and stride != want:
                raise ValueError(f"{what}: gaps within a row")
            want *= size

    # ---- sequences ----------------------------------------------------------
    # (lists go to the library as bytes: their address is the cheapest that numpy gives)
    def fork(self, src, dst, lens=None):
        """dst[i] (empty) becomes the first lens[i] tokens (all of them) of src[i], on the same pages."""
        src = _ids(src, "src")
        n = src.size
        dst = _ids(dst, "dst", n)
        lens = None if lens is None else _ids(lens, "lens", n).tobytes()
        self._call(self.lib.fl_pages_fork, src.tobytes(), dst.tobytes(), lens, n)

    def copy(self, src, dst):
        """dst[i] (empty) becomes a copy of src[i] on pages of its own."""
        src = _ids(src, "src")
        dst = _ids(dst, "dst", src.size)
        self._enqueue(self.lib.fl_pages_copy, src.tobytes(), dst.tobytes(), src.size)

    def free(self, seqs):
        """Empties sequences; pages that none holds any more are free."""
        seqs = _ids(seqs, "seqs")
        self._call(self.lib.fl_pages_free, seqs.tobytes(), seqs.size)

    def truncate(self, seqs, lens):
        """Cuts sequences to their first lens[i] tokens."""
        seqs = _ids(seqs, "seqs")
        lens = _ids(lens, "lens", seqs.size)
        self._call(self.lib.fl_pages_truncate, seqs.tobytes(), lens.tobytes(), seqs.size)

    def extend(self, seqs, counts):
        """Reserves slots for counts[i] more tokens of each sequence; `write` fills them, layer by layer."""
        seqs = _ids(seqs, "seqs")
        counts = _ids(counts, "counts", seqs.size)
        self._enqueue(self.lib.fl_pages_extend, seqs.tobytes(), counts.tobytes(), seqs.size)

    def compact(self) -> int:
        """Moves pages so that those in use have the lowest numbers; returns how many moved."""
        n = C.c_int()
        self._enqueue(self.lib.fl_pages_compact, C.byref(n))
        return n.value

    def length(self, seq: int) -> int:
        n = self.lib.fl_pages_len(self._h, seq)
        if n < 0:
            self._open()
            raise ValueError(f"sequence {seq} of {self.max_seqs}")
        return n

    @property
    def free_pages(self) -> int:
        self._open()
        return self.lib.fl_pages_free_count(self._h)

    def tables(self) -> np.ndarray:
        """Page lists [max_seqs, pages of max_len], -1 where a sequence holds none."""
        t = np.empty((self.max_seqs, -(-self.max_len // self.page_size)), np.int32)
        self._call(self.lib.fl_pages_tables, t.ctypes.data, None)
        return t

    def lens(self) -> np.ndarray:
        n = np.empty(self.max_seqs, np.int32)
        self._call(self.lib.fl_pages_tables, None, n.ctypes.data)
        return n

    # ---- rows ---------------------------------------------------------------
    def write(self, k, v, layer: int = 0):
        """Keys and values of the last `extend`'s tokens, sequence by sequence: [tokens, kv_heads, head_dim]
        for one layer, or [layers, tokens, kv_heads, head_dim] for as many from `layer` on.  Token rows
        may be slices of wider ones."""
        self._rows(k, "k", self._row)
        self._rows(v, "v", self._row)
        if k.dim() not in (3, 4) or k.shape != v.shape or k.stride() != v.stride():
            raise ValueError("k and v: [tokens, kv_heads, head_dim] or [layers, ..], laid out alike")
        n = k.shape[-3]
        room = self.lib.fl_pages_pending(self._h) if self._h else n
        if room >= 0 and n != room:
            raise ValueError(f"{n} tokens, where the last extend() made room for {room}")
        if n == 0:
            return
        layers = k.shape[0] if k.dim() == 4 else 1
        row = self.kv_heads * self.head_dim
        stride = k.stride(-3) if n > 1 else max(k.stride(0), row) if layers > 1 else row
        if layers > 1 and k.stride(0) != n * stride:
            raise ValueError("k and v: gaps between layers")
        self._enqueue(self.lib.fl_pages_write, layer, layers, k.data_ptr(), v.data_ptr(), stride)

    def read(self, seqs, starts, counts, layer: int = 0):
        """The f32 keys and values [tokens, kv_heads, head_dim] of counts[i] tokens of each sequence, from starts[i] on."""
        torch = self._torch
        seqs = _ids(seqs, "seqs")
        starts, counts = _ids(starts, "starts", seqs.size), _ids(counts, "counts", seqs.size)
        shape = (max(0, int(counts.sum())), self.kv_heads, self.head_dim)
        k, v = (torch.empty(shape, dtype=torch.float32, device=self.device) for _ in "kv")
        self._enqueue(self.lib.fl_pages_read, layer, seqs.tobytes(), starts.tobytes(), counts.tobytes(), seqs.size,
                      k.data_ptr(), v.data_ptr())
        return k, v

    def attention(self, q, seqs, seen=None, layer: int = 0, out=None):
        """Attention of queries q [n, heads, head_dim] (RoPE applied; rows may be slices of wider ones): query i
        over the first seen[i] tokens (all of them) of sequence seqs[i].  -> [n, heads, head_dim] (out: apart from q)"""
        torch = self._torch
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise ValueError("q: [n, heads, head_dim]")
        n, heads, _ = shape = q.shape
        self._rows(q, "q", (heads, self.head_dim))
        seqs = _ids(seqs, "seqs", n)
        if seen is None:
            if n and (seqs.min() < 0 or seqs.max() >= self.max_seqs):
                raise ValueError(f"seqs: of {self.max_seqs}")
            seen = self.lens()[seqs]
        seen = _ids(seen, "seen", n)
        if out is None:
            out = torch.empty(shape, dtype=torch.float32, device=self.device)
        else:
            self._rows(out, "out", shape)
            if out.dim() != 3:
                raise ValueError("out: [n, heads, head_dim]")
        stride = q.stride(0) if n > 1 else heads * self.head_dim
        self._enqueue(self.lib.fl_pages_attention, layer, q.data_ptr(), stride, seqs.tobytes(), seen.tobytes(), n, heads,
                      out.data_ptr())
        return out
