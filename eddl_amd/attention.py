"""What the attention operators of ``Backend`` take: the paged cache, the batch of sequences that reads and writes it, and the
plan of a rotary position."""
import ctypes

import numpy as np

_CACHE_TYPES = {"float32": 0, "bfloat16": 1}


class PagedCache:
    """A pool of pages of keys and values on the device (the layout stands in include/eddlhip.h).  ``storage`` = (keys, values): tensors of
    the caller's to use instead of new ones, which start as zeros."""

    def __init__(self, backend, pages, page_size, kv_heads, head_dim, dtype="float32", storage=None):
        if dtype not in _CACHE_TYPES:
            raise ValueError("a cache holds float32 or bfloat16, not %s" % dtype)
        self.backend, self.dtype = backend, dtype
        self.pages, self.page_size, self.kv_heads, self.head_dim = int(pages), int(page_size), int(kv_heads), int(head_dim)
        if self.page_size < 16 or self.page_size & (self.page_size - 1) or self.pages < 1 or self.kv_heads < 1 or not 16 <= self.head_dim <= 256 or self.head_dim % 16:
            raise ValueError("a cache of %d pages of %d tokens, %d heads of %d: the page size is a power of two from 16 on, the head dimension a "
                             "multiple of 16 up to 256" % (pages, page_size, kv_heads, head_dim))
        blocks, d = self.page_size // 16, self.head_dim
        k_shape, v_shape = (self.pages, self.kv_heads, blocks, d // 8, 16, 8), (self.pages, self.kv_heads, blocks, 2, d, 8)
        if storage is None:
            self.keys, self.values = backend.empty(k_shape, dtype), backend.empty(v_shape, dtype)
            for t in (self.keys, self.values):  # (zeros in either type)
                backend._check(backend.lib.eddlhip_fill(backend.dev, t.address, t.nbytes // 4, 0.0))
        else:
            self.keys, self.values = storage
            if tuple(self.keys.shape) != k_shape or tuple(self.values.shape) != v_shape or self.keys.dtype != dtype or self.values.dtype != dtype:
                raise ValueError("a cache of %d pages of %d tokens, %d heads of %d holds keys %s and values %s of %s, not %s %s and %s %s"
                                 % (pages, page_size, kv_heads, head_dim, k_shape, v_shape, dtype, self.keys.dtype, self.keys.shape, self.values.dtype,
                                    self.values.shape))
        self.arguments = (self.keys.address, self.values.address, _CACHE_TYPES[dtype], self.pages, self.page_size)


class PagedBatch:
    """The sequences of a call: int32 device tensors ``table`` [sequences, width], ``offsets`` [sequences + 1], ``lengths`` [sequences], and the
    host's bounds of the new tokens and the length of a sequence."""

    def __init__(self, table, offsets, lengths, max_new, max_length):
        if len(table.shape) != 2 or tuple(offsets.shape) != (table.shape[0] + 1,) or tuple(lengths.shape) != (table.shape[0],) \
                or any(t.dtype != "int32" for t in (table, offsets, lengths)):
            raise ValueError("a batch is int32 table [sequences, width], offsets [sequences + 1], lengths [sequences], not %s %s %s" % (table.shape, offsets.shape, lengths.shape))
        self.table, self.offsets, self.lengths = table, offsets, lengths
        self.max_new, self.max_length = int(max_new), int(max_length)
        self.arguments = (table.address, table.shape[1], offsets.address, lengths.address, table.shape[0])


class RotaryPlan:
    """Axis and frequency of every pair of dimensions of a head: arrays of rot_dim / 2 entries.  ``pairing``: "halves" pairs dimension n with
    n + rot_dim / 2, "adjacent" 2n with 2n + 1."""

    def __init__(self, head_dim, axis, freq, pairing="halves", axes=None):
        axis, freq = np.ascontiguousarray(axis, np.int32), np.ascontiguousarray(freq, np.float64)
        if axis.ndim != 1 or axis.shape != freq.shape or pairing not in ("halves", "adjacent"):
            raise ValueError("a rotary plan has an axis and a frequency for every pair, and pairs halves or adjacent dimensions, not %s %s %s"
                             % (axis.shape, freq.shape, pairing))
        self.head_dim, self.axis, self.freq, self.pairing = int(head_dim), axis, freq, pairing
        self.axes = int(axes) if axes is not None else int(axis.max(initial=0)) + 1
        self.rot_dim = 2 * len(axis)
        self.arguments = (self.rot_dim, int(pairing == "adjacent"), self.axes, ctypes.c_void_p(axis.ctypes.data), ctypes.c_void_p(freq.ctypes.data))

    @classmethod
    def sections(cls, head_dim, sections, theta=10000.0, pairing="halves", shared=True, interleaved=False):
        """``sections[a]`` pairs turn by axis ``a``, side by side or, ``interleaved``, in turns.  Frequencies fall as theta ** (-n / pairs) over all
        pairs (``shared``), or over the pairs of an axis."""
        counts = [int(c) for c in sections]
        axis = np.repeat(np.arange(len(counts)), counts)
        if interleaved:
            nth = np.concatenate([np.arange(c) for c in counts])
            axis = axis[np.lexsort((axis, nth))]
        if shared:
            freq = theta ** (-np.arange(len(axis), dtype=np.float64) / max(len(axis), 1))
        else:
            seen = np.array([np.sum(axis[:n] == a) for n, a in enumerate(axis)], np.float64)
            freq = theta ** (-seen / np.maximum(np.array(counts, np.float64)[axis], 1))
        return cls(head_dim, axis, freq, pairing, len(counts))
