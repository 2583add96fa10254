"""Paged KV cache of many sequences (fl_pages_* of include/flare_hip.h).

`PagedKv` holds a pool of pages and sequences that are lists of pages: forks
share what they have in common, a page is copied when one of them would write to
it, and `attention` reads a page that several of the batch's sequences hold once
for all of them.  Where flarellm's caches (flare-core/src/kv_cache.rs:431-546) hold
one sequence, this holds a batch: several answers to one prompt, beams, chats
behind one system prompt.

Work is enqueued on the backend's stream.  Calls made with another current torch
stream order the two streams by events, so tensors go in and come out as with any
torch operation; no call waits for the GPU.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import numpy as np

from . import _lib
from ._lib import FL_KV_F16, FL_KV_F32, FL_KV_Q8, FlareError, PagesConfig, check


def _ids(x, what: str) -> np.ndarray:
    a = np.asarray(x)
    if a.dtype == np.int32 and a.ndim == 1 and a.flags.c_contiguous:
        return a
    if a.ndim != 1 or (a.size and a.dtype.kind not in "iu"):
        raise ValueError(f"{what}: a list of whole numbers")
    if a.size and (a.max() > 2**31 - 1 or a.min() < -(2**31)):
        raise ValueError(f"{what}: out of range")
    return np.ascontiguousarray(a, np.int32)


def _ids_of(n: int, x, what: str) -> np.ndarray:
    a = _ids(x, what)
    if a.size != n:
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
        self.max_seqs, self.max_len = max_seqs, max_len or pages * page_size
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

    def _call(self, name: str, *args):
        if not self._h or not self._b.ctx:
            raise FlareError("the paged cache or its backend is closed")
        check(getattr(self.lib, name)(self._h, *args), self._b.ctx)

    @contextlib.contextmanager
    def _ordered(self):
        """The current torch stream's work before this, and this before what follows there."""
        import torch

        current = torch.cuda.current_stream(self.device)
        if current.cuda_stream == self.stream.cuda_stream:
            yield
            return
        self.stream.wait_stream(current)
        yield
        current.wait_stream(self.stream)

    def _rows(self, t, what: str, shape):
        """A float32 tensor on this device whose last dimensions are `shape`, without gaps between them."""
        import torch

        if not torch.is_tensor(t) or t.dtype != torch.float32 or t.device != self.device:
            raise ValueError(f"{what}: a float32 tensor on {self.device}")
        n = len(shape)
        if t.dim() < n or tuple(t.shape[-n:]) != tuple(shape):
            raise ValueError(f"{what}: {tuple(t.shape)}, not [.., {', '.join(map(str, shape))}]")
        want = 1
        for size, stride in zip(reversed(t.shape[-n:]), reversed(t.stride()[-n:])):
            if size != 1 and stride != want:
                raise ValueError(f"{what}: gaps within a row")
            want *= size

    # ---- sequences ----------------------------------------------------------
    def fork(self, src, dst, lens=None):
        """dst[i] (empty) becomes the first lens[i] tokens (all of them) of src[i], on the same pages."""
        src = _ids(src, "src")
        dst = _ids_of(len(src), dst, "dst")
        lens = None if lens is None else _ids_of(len(src), lens, "lens")
        self._call("fl_pages_fork", src.ctypes.data, dst.ctypes.data, None if lens is None else lens.ctypes.data, len(src))

    def copy(self, src, dst):
        """dst[i] (empty) becomes a copy of src[i] on pages of its own."""
        src = _ids(src, "src")
        dst = _ids_of(len(src), dst, "dst")
        with self._ordered():
            self._call("fl_pages_copy", src.ctypes.data, dst.ctypes.data, len(src))

    def free(self, seqs):
        """Empties sequences; pages that none holds any more are free."""
        seqs = _ids(seqs, "seqs")
        self._call("fl_pages_free", seqs.ctypes.data, len(seqs))

    def truncate(self, seqs, lens):
        """Cuts sequences to their first lens[i] tokens."""
        seqs = _ids(seqs, "seqs")
        lens = _ids_of(len(seqs), lens, "lens")
        self._call("fl_pages_truncate", seqs.ctypes.data, lens.ctypes.data, len(seqs))

    def extend(self, seqs, counts):
        """Reserves slots for counts[i] more tokens of each sequence; `write` fills them, layer by layer."""
        seqs = _ids(seqs, "seqs")
        counts = _ids_of(len(seqs), counts, "counts")
        with self._ordered():
            self._call("fl_pages_extend", seqs.ctypes.data, counts.ctypes.data, len(seqs))
        self._tokens = int(counts.sum())

    def compact(self) -> int:
        """Moves pages so that those in use have the lowest numbers; returns how many moved."""
        n = C.c_int()
        with self._ordered():
            self._call("fl_pages_compact", C.byref(n))
        return n.value

    def length(self, seq: int) -> int:
        n = self.lib.fl_pages_len(self._h, seq)
        if n < 0:
            raise ValueError(f"sequence {seq} of {self.max_seqs}")
        return n

    @property
    def free_pages(self) -> int:
        return self.lib.fl_pages_free_count(self._h)

    def tables(self) -> np.ndarray:
        """Page lists [max_seqs, pages of max_len], -1 where a sequence holds none."""
        t = np.empty((self.max_seqs, -(-self.max_len // self.page_size)), np.int32)
        self._call("fl_pages_tables", t.ctypes.data, None)
        return t

    def lens(self) -> np.ndarray:
        n = np.empty(self.max_seqs, np.int32)
        self._call("fl_pages_tables", None, n.ctypes.data)
        return n

    # ---- rows ---------------------------------------------------------------
    def write(self, k, v, layer: int = 0):
        """Keys and values of the last `extend`'s tokens, sequence by sequence: [tokens, kv_heads, head_dim]
        for one layer, or [layers, tokens, kv_heads, head_dim] for as many from `layer` on.  Token rows
        may be slices of wider ones."""
        row = (self.kv_heads, self.head_dim)
        for t, what in ((k, "k"), (v, "v")):
            self._rows(t, what, row)
        if k.dim() not in (3, 4) or k.shape != v.shape or k.stride() != v.stride():
            raise ValueError("k and v: [tokens, kv_heads, head_dim] or [layers, ..], laid out alike")
        n = k.shape[-3]
        if n != getattr(self, "_tokens", -1):
            raise ValueError(f"{n} tokens, where the last extend() made room for {getattr(self, '_tokens', 0)}")
        if n == 0:
            return
        layers = k.shape[0] if k.dim() == 4 else 1
        stride = k.stride(-3) if n > 1 else max(k.stride(-3), self.kv_heads * self.head_dim)
        if layers > 1 and k.stride(0) != n * stride:
            raise ValueError("k and v: gaps between layers")
        with self._ordered():
            self._call("fl_pages_write", layer, layers, k.data_ptr(), v.data_ptr(), stride)

    def read(self, seqs, starts, counts, layer: int = 0):
        """The f32 keys and values [tokens, kv_heads, head_dim] of counts[i] tokens of each sequence, from starts[i] on."""
        import torch

        seqs = _ids(seqs, "seqs")
        starts, counts = _ids_of(len(seqs), starts, "starts"), _ids_of(len(seqs), counts, "counts")
        shape = (max(0, int(counts.sum())), self.kv_heads, self.head_dim)
        k, v = (torch.empty(shape, dtype=torch.float32, device=self.device) for _ in "kv")
        with self._ordered():
            self._call("fl_pages_read", layer, seqs.ctypes.data, starts.ctypes.data, counts.ctypes.data, len(seqs),
                       k.data_ptr(), v.data_ptr())
        return k, v

    def attention(self, q, seqs, seen=None, layer: int = 0, out=None):
        """Attention of queries q [n, heads, head_dim] (RoPE applied; rows may be slices of wider ones): query i
        over the first seen[i] tokens (all of them) of sequence seqs[i].  -> [n, heads, head_dim]"""
        import torch

        if not torch.is_tensor(q) or q.dim() != 3:
            raise ValueError("q: [n, heads, head_dim]")
        n, heads, _ = q.shape
        self._rows(q, "q", (heads, self.head_dim))
        seqs = _ids_of(n, seqs, "seqs")
        if seen is None:
            if n and (seqs.min() < 0 or seqs.max() >= self.max_seqs):
                raise ValueError(f"seqs: of {self.max_seqs}")
            seen = self.lens()[seqs]
        seen = _ids_of(n, seen, "seen")
        if out is None:
            out = torch.empty(n, heads, self.head_dim, dtype=torch.float32, device=self.device)
        else:
            self._rows(out, "out", (n, heads, self.head_dim))
            if out.dim() != 3:
                raise ValueError("out: [n, heads, head_dim]")
        stride = q.stride(0) if n > 1 else max(q.stride(0), heads * self.head_dim)
        with self._ordered():
            self._call("fl_pages_attention", layer, q.data_ptr(), stride, seqs.ctypes.data, seen.ctypes.data, n, heads,
                       out.data_ptr())
        return out
