"""The attention operators in 64 bits with numpy, from their formulas, and the cache's layout as index arithmetic."""
import numpy as np

EPS = 2.0 ** -24  # half a step of fp32, relative


def bf16_bits(x):
    """Nearest bfloat16, ties to even, as 16-bit patterns."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    out = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), out)


def bf16_value(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def key_index(place, head, d, page_size, kv_heads, dim, page):
    t = place % page_size
    return (((page * kv_heads + head) * (page_size // 16) + t // 16) * (dim // 8) + d // 8) * 128 + (t % 16) * 8 + d % 8


def value_index(place, head, d, page_size, kv_heads, dim, page):
    t = place % page_size
    return ((((page * kv_heads + head) * (page_size // 16) + t // 16) * 2 + t % 16 // 8) * dim + d) * 8 + t % 8


class Pool:
    """A cache's content and its batch on the host: random pages, ragged sequences, tokens behind a sequence's length NaN."""

    def __init__(self, rng, news, lengths, kv_heads, dim, page_size, dtype, spare=2, width=None, fill=np.nan, shared=None):
        self.news, self.lengths, self.kv_heads, self.dim, self.page_size, self.dtype = list(news), list(lengths), kv_heads, dim, page_size, dtype
        counts = [-(-n // page_size) for n in lengths]
        self.pages = sum(counts) + spare
        order = rng.permutation(self.pages)
        self.width = max(counts + [1]) if width is None else width
        self.table = np.full((len(news), self.width), -7, np.int32)
        at = 0
        for s, c in enumerate(counts):
            self.table[s, :c] = order[at:at + c]
            at += c
        if shared is not None:  # the first pages of all sequences are those of the first one
            for s in range(1, len(news)):
                self.table[s, :shared] = self.table[0, :shared]
        self.offsets = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.rows = int(self.offsets[-1])
        n = self.pages * page_size * kv_heads * dim
        self.k, self.v = np.full(n, fill, np.float32), np.full(n, fill, np.float32)
        for s, c in enumerate(lengths):
            for name in ("k", "v"):
                self.put(s, np.arange(c), name, rng.standard_normal((c, kv_heads, dim), dtype=np.float32))

    def index(self, s, places, name):
        places = np.asarray(places, np.int64)[:, None, None]
        head, d = np.arange(self.kv_heads)[None, :, None], np.arange(self.dim)[None, None, :]
        page = self.table[s, places // self.page_size].astype(np.int64)
        return (key_index if name == "k" else value_index)(places, head, d, self.page_size, self.kv_heads, self.dim, page)

    def put(self, s, places, name, x):
        if self.dtype == "bfloat16":
            x = bf16_value(bf16_bits(x))
        getattr(self, name)[self.index(s, places, name)] = x

    def get(self, s, places, name):
        return getattr(self, name)[self.index(s, places, name)]

    def on(self, hip, max_new=None, max_length=None):
        """(PagedCache, PagedBatch) on the device."""
        from eddl_amd.attention import PagedBatch, PagedCache
        put = (lambda x: hip.array(bf16_bits(x), "bfloat16")) if self.dtype == "bfloat16" else hip.array
        p, h, b, d = self.pages, self.kv_heads, self.page_size // 16, self.dim
        storage = put(self.k).reshape((p, h, b, d // 8, 16, 8)), put(self.v).reshape((p, h, b, 2, d, 8))
        cache = PagedCache(hip, p, self.page_size, h, d, self.dtype, storage)
        batch = PagedBatch(hip.array(self.table, "int32"), hip.array(self.offsets, "int32"), hip.array(np.array(self.lengths), "int32"),
                           max(self.news + [0]) if max_new is None else max_new, max(self.lengths + [0]) if max_length is None else max_length)
        return cache, batch

    def read(self, cache):
        """Keys and values of a device cache as flat float32 arrays."""
        out = [t.numpy().reshape(-1) for t in (cache.keys, cache.values)]
        return [bf16_value(x) for x in out] if self.dtype == "bfloat16" else out


def attention(q, pool, heads, scale, causal, window, dtype=np.float64):
    """(output, bound of its error) [rows, heads * dim].

    The bound: a score is a sum of D products over D / 16 instructions and three to six parts; with at most four roundings of
    fp32 an instruction's contribution and what the split leaves out (2^-24 of a product) it is off by 4 (D / 16 + 4) EPS sum |q k|, plus
    one rounding of the scaled query (EPS |q k|) and two of the exponential's argument (2 EPS (|s| + |m|) log2 e, in exponents of two), plus
    2 EPS of the exponential.  All weights off by a relative e move a weighted mean by at most 2 e max |v|; the sums over the tokens add 4
    roundings an instruction of 16 tokens and one a rescaling, and the joins and the division a few more."""
    dim, kv = pool.dim, pool.kv_heads
    out, tol = np.zeros((pool.rows, heads * dim), dtype), np.zeros((pool.rows, heads * dim))
    for s, (new, length) in enumerate(zip(pool.news, pool.lengths)):
        j = np.arange(length)
        k, v = pool.get(s, j, "k").astype(dtype), pool.get(s, j, "v").astype(dtype)
        for i in range(new):
            row, pos = int(pool.offsets[s]) + i, length - new + i
            seen = np.ones(length, bool)
            if causal:
                seen &= j <= pos
            if window > 0:
                seen &= j > pos - window
            if not seen.any():
                continue
            for h in range(heads):
                x, kk, vv = q[row, h * dim:(h + 1) * dim].astype(dtype), k[seen, h * kv // heads], v[seen, h * kv // heads]
                with np.errstate(all="ignore"):
                    sc = (kk @ x) * dtype(scale)
                    top = sc.max()
                    w = np.exp(sc - top)
                    out[row, h * dim:(h + 1) * dim] = (w @ vv) / w.sum()
                    if dtype == np.float64:
                        mag = (np.abs(kk) @ np.abs(x)).max() * scale
                        e = (4 * (dim / 16 + 4) + 1) * EPS * mag + 6 * EPS * mag + 2 * EPS
                        tol[row, h * dim:(h + 1) * dim] = (2 * e + (8 * (seen.sum() / 16 + 1) + 16) * EPS) * np.abs(vv).max()
    return out, tol


def turned(x, positions, heads, dim, axis, freq, adjacent):
    """Rotary positions in 64 bits."""
    y = x.astype(np.float64).reshape(len(x), heads, dim).copy()
    half = len(axis)
    for n in range(half):
        i, j = (2 * n, 2 * n + 1) if adjacent else (n, n + half)
        a = positions[:, axis[n]].astype(np.float64) * freq[n]
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        y[:, :, i], y[:, :, j] = y[:, :, i] * c - y[:, :, j] * s, y[:, :, j] * c + y[:, :, i] * s
    return y.reshape(len(x), heads * dim)


def normed(x, kind, w, b, eps):
    x = x.astype(np.float64)
    if kind is None:
        return x
    if kind == "layer":
        x = x - x.mean(1, keepdims=True)
    y = x / np.sqrt((x * x).mean(1, keepdims=True) + eps)
    if w is not None:
        y = y * w
    return y if b is None else y + b


def norm_residual(x, r, post, pre, gate, scale, mod, shift, group_rows):
    g = np.arange(len(x)) // group_rows
    n = normed(x, *post)
    if gate is not None:
        n = n * (gate[g] if len(gate) > 1 else gate).astype(np.float64)
    s = n if r is None else np.float64(np.float32(scale)) * r + n
    h = normed(s, *pre)
    if mod is not None:
        h = h * (1.0 + mod[g].astype(np.float64))
    return s, h if shift is None else h + shift[g]
