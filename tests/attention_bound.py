"""Attention in 64 bits with a bound of the error for every row and head, from the row's own visible tokens alone: what a row does not see, or
gives no weight, adds nothing to what it may be off by."""
import numpy as np

from attention_ref import EPS


def attention_rows(q, pool, heads, scale, causal, window, dtype=np.float64):
    """(output [rows, heads, dim], bound [rows, heads, 1], size [rows, heads, 1]); size: the largest of a row's sums of p_j |v_jd|.

    A score is off by e_j = (12 (D / 16) + 15) EPS sum |q k_j| + 24 EPS: three products for 16 dimensions, four roundings of fp32 each;
    8 EPS where numbers are pairs of fp16 (2 EPS a number, 4 EPS for the product of two low halves); a rounding of the scaled query or factor and six of the
    exponential's argument; and 24 EPS that no score exceeds through exponents shared with other tokens (2^-19 of a doubling, and the exponential's 2 EPS).
    An error common to a row's scores cancels, so the mean moves by at most sum_j p_j e_j (|v_jd| + |o_d|).  The sums over the tokens: 12 EPS for 16 tokens,
    2^-26 a token for weights and values that share exponents with others (of the row's largest sum), and 16 EPS for rescalings, joins and the
    division."""
    dim, kv = pool.dim, pool.kv_heads
    group = heads // kv
    out, tol, size = np.zeros((pool.rows, heads, dim), dtype), np.zeros((pool.rows, heads, 1)), np.zeros((pool.rows, heads, 1))
    q = q.reshape(len(q), heads, dim)
    for s, (new, length) in enumerate(zip(pool.news, pool.lengths)):
        if new == 0 or length == 0:
            continue
        j, rows = np.arange(length), slice(int(pool.offsets[s]), int(pool.offsets[s]) + new)
        pos = length - new + np.arange(new)[:, None]
        seen = np.ones((new, length), bool)
        if causal:
            seen &= j <= pos
        if window > 0:
            seen &= j > pos - window
        k, v = pool.get(s, j, "k").astype(dtype), pool.get(s, j, "v").astype(dtype)
        for h in range(heads):
            x, kk, vv = q[rows, h].astype(dtype), k[:, h // group], v[:, h // group]
            sc = np.where(seen, (x @ kk.T) * dtype(scale), dtype(-np.inf))
            top = sc.max(1, keepdims=True)
            w = np.exp(sc - np.where(np.isfinite(top), top, 0))
            p = w / np.where(seen.any(1, keepdims=True), w.sum(1, keepdims=True), 1)
            o = p @ np.where(seen.any(0)[:, None], vv, 0)
            out[rows, h] = o
            if dtype == np.float64:
                e = (12 * (dim / 16) + 15) * EPS * (np.abs(x) @ np.abs(kk).T) * abs(scale) + 24 * EPS
                mean, n = p @ np.abs(vv), length
                moved = (p * e) @ np.abs(vv) + (p * e).sum(1, keepdims=True) * np.abs(o)
                size[rows, h] = mean.max(1, keepdims=True)
                tol[rows, h] = moved.max(1, keepdims=True) + (12 * (n / 16 + 1) + n / 4 + 16) * EPS * size[rows, h]
    return out, tol, size


def check_rows(got, q, pool, heads, scale, causal, window, what=""):
    """Every number within its row's bound, and the rows' errors, each relative to its row, as small as those of the formula in fp32 arithmetic."""
    want, tol, size = attention_rows(q, pool, heads, scale, causal, window)
    got = got.reshape(want.shape)
    off = np.abs(got - want)
    assert np.all(off <= tol), (what, "of its row's size", float((off / np.where(size > 0, size, 1)).max()))
    plain = attention_rows(q, pool, heads, scale, causal, window, np.float32)[0]
    norm = lambda t: np.linalg.norm(t / np.where(size > 0, size, 1))
    assert norm(got - want) <= 4 * norm(plain - want) + 8 * EPS * norm(want), (what, norm(got - want), norm(plain - want), norm(want))
