"""Group norm, causal convolution and selective scan in 64 bits, each with a bound of what fp32 arithmetic may be off by."""
import numpy as np

EPS = 2.0 ** -24  # half a step of fp32, relative


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-x))


def activated(x, kind):
    return x if kind is None else np.where(x > 0, x, 0 * x) if kind == "relu" else x * sigmoid(x)


def activated_error(x, err, kind):
    """``err`` of x behind the activation: no slope is above 1.1; silu adds an exponential (4 EPS), a sum, a reciprocal (2 EPS) and a product."""
    return err if kind != "silu" else 1.1 * err + 10 * EPS * np.abs(x * sigmoid(x))


def group_norm(x, groups, w, b, eps, mod, shift, kind):
    """x [images, channels, pixels].  (result, bound).

    A mean is a sum over at most 100 numbers a thread, in turns or a tree, and a join of such sums: 128 EPS of the mean size of the numbers, and that moves every
    difference.  The squares' sum is off by 128 EPS of itself, half of it in the root, which with the division adds 4 EPS."""
    images, channels, pixels = x.shape
    x = x.astype(np.float64).reshape(images, groups, -1)
    mean = x.mean(2, keepdims=True)
    sd = np.sqrt(((x - mean) ** 2).mean(2, keepdims=True) + eps)
    n = (x - mean) / sd
    off = 128 * EPS * np.abs(x).mean(2, keepdims=True) / sd
    err = (off + (72 + 4) * EPS * np.abs(n) + off * np.abs(n) * np.abs(n).max(2, keepdims=True)).reshape(images, channels, pixels)
    n = n.reshape(images, channels, pixels)
    each = lambda t: t.astype(np.float64).reshape(-1, channels, 1)
    if w is not None:
        n, err = n * each(w), err * np.abs(each(w)) + 2 * EPS * np.abs(n * each(w))
    if b is not None:
        n = n + each(b)
        err = err + EPS * np.abs(n)
    if mod is not None:
        m = each(1.0 + mod.astype(np.float64))
        n, err = n * m, err * np.abs(m) + 2 * EPS * np.abs(n * m)
    if shift is not None:
        n = n + each(shift)
        err = err + EPS * np.abs(n)
    return activated(n, kind), activated_error(n, err, kind)


def sequences(offsets, rows, reverse):
    """The rows of every sequence in the order in which its tokens are taken; offsets out of range are cut."""
    out = []
    for a, b in zip(offsets[:-1], offsets[1:]):
        a = min(max(int(a), 0), rows)
        b = min(max(int(b), a), rows)
        out.append(np.arange(a, b)[::-1] if reverse else np.arange(a, b))
    return out


def reads(s, new, lengths, slots, pool):
    """The slot that sequence s continues: None where it begins, -1 where it lies outside the pool."""
    if pool is None or int(lengths[s]) <= new:
        return None
    return int(slots[s]) if 0 <= slots[s] < len(pool) else -1


def causal_conv(x, w, b, offsets, kind, reverse, pool=None, lengths=None, slots=None, out_slots=None):
    """(result, bound, pool afterwards); rows of no sequence are NaN in the result.  ``width`` products, each rounded with its sum."""
    channels, width = w.shape
    out, err = np.full(x.shape, np.nan), np.zeros(x.shape)
    after = None if pool is None else pool.copy()
    for s, rows in enumerate(sequences(offsets, len(x), reverse)):
        if not len(rows):
            continue
        slot = reads(s, len(rows), lengths, slots, pool)
        before = np.zeros((width - 1, channels), np.float32) if slot is None else np.full((width - 1, channels), np.nan, np.float32) if slot < 0 else pool[slot]
        full = np.concatenate([before, x[rows]])
        terms = np.stack([full[k:k + len(rows)].astype(np.float64) * w[:, k] for k in range(width)])
        with np.errstate(invalid="ignore"):
            y = terms.sum(0) + (0 if b is None else b)
            e = (width + 1) * EPS * (np.abs(terms).sum(0) + (0 if b is None else np.abs(b)))
            out[rows], err[rows] = activated(y, kind), activated_error(y, e, kind)
        if pool is not None and 0 <= out_slots[s] < len(pool):
            after[out_slots[s]] = full[len(full) - width + 1:]
    return out, err, after


def selective_scan(x, dt, A, B, C, offsets, skip=None, gate=None, dt_bias=None, softplus=True, reverse=False, pool=None, lengths=None, slots=None, out_slots=None):
    """(result, bound, pool afterwards, its bound); rows of no sequence are NaN in the result.

    The bounds follow the recurrence.  d: the sum with the bias rounds (EPS of it, through a slope of at most 1), softplus by 12 EPS of itself (exponential 4,
    logarithm 2, corrections and sums).  The factor e^(dA): its argument is off by 4 EPS of itself (A in base 2, the product) and what d is off by; the exponential 2.  A
    state: what it was off by and the factor's share of it, the product d x B and one rounding.  States that are joined from parts of the tokens are products and sums of the same factors,
    so twice these bounds cover them.  The sum over n states: n + 8 roundings."""
    channels, n = A.shape
    per = channels * n // B.shape[1]
    out, err = np.full(x.shape, np.nan), np.zeros(x.shape)
    after = None if pool is None else pool.astype(np.float64)
    after_err = None if pool is None else np.zeros(pool.shape)
    f = lambda t: t.astype(np.float64)
    A64 = f(A)
    group = np.arange(channels) // per
    for s, rows in enumerate(sequences(offsets, len(x), reverse)):
        if not len(rows):
            continue
        slot = reads(s, len(rows), lengths, slots, pool)
        h = np.zeros((channels, n)) if slot is None else np.full((channels, n), np.nan) if slot < 0 else f(pool[slot])
        eh = np.zeros((channels, n))
        raw = f(dt[rows]) + (0 if dt_bias is None else f(dt_bias))
        d, ed = raw, (EPS * np.abs(raw) if dt_bias is not None else 0 * raw)
        if softplus:
            d = np.logaddexp(raw, 0)
            ed = ed * sigmoid(raw) + 12 * EPS * d
        with np.errstate(invalid="ignore", over="ignore"):
            for t, row in enumerate(rows):
                b, c = f(B[row]).reshape(-1, n)[group], f(C[row]).reshape(-1, n)[group]
                arg = d[t][:, None] * A64
                a = np.exp(arg)
                put = (d[t] * f(x[row]))[:, None] * b
                rel = np.where(a > 0, ed[t][:, None] * np.abs(A64) + 4 * EPS * np.abs(arg) + 2 * EPS, 0)  # (a factor of 0 is exact)
                relative = (ed[t] / np.where(d[t] != 0, np.abs(d[t]), 1))[:, None] + 3 * EPS
                eh = a * (1 + rel) * eh + np.abs(h) * a * rel + np.abs(put) * relative
                h = a * h + put
                eh = eh + EPS * np.abs(h)
                y = (c * h).sum(1)
                ey = 2 * (np.abs(c) * eh).sum(1) + (n + 8) * EPS * np.abs(c * h).sum(1)
                if skip is not None:
                    y = y + f(skip) * f(x[row])
                    ey = ey + EPS * np.abs(y) + EPS * np.abs(f(skip) * f(x[row]))
                if gate is not None:
                    g = f(gate[row])
                    v = g * sigmoid(g)
                    ey = ey * np.abs(v) + 11 * EPS * np.abs(y * v)
                    y = y * v
                out[row], err[row] = y, ey
        if pool is not None and 0 <= out_slots[s] < len(pool):
            after[out_slots[s]], after_err[out_slots[s]] = h, 2 * eh
    return out, err, after, after_err
