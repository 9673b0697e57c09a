"""Group norm, causal convolution and selective scan against their formulas in 64 bits."""
import numpy as np
import pytest

from state_space_ref import EPS, causal_conv, group_norm, selective_scan

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -120  # what numbers below the normal ones may lose


def _check(got, want, err, what=""):
    """Every number within its bound; where the formula gives none (or rows are of no sequence) ``got`` is not looked at."""
    fine = np.isfinite(want)
    off = np.abs(got.astype(np.float64) - want)[fine]
    worst = float((off / (err[fine] + TINY)).max()) if off.size else 0.0
    assert np.all(off <= err[fine] + TINY), (what, worst)
    return worst


# ------------------------------------------------------------------------------------------------- group norm
SHAPES = [(1, 1, 1, 1, 1), (2, 4, 1, 1, 2), (1, 512, 7, 7, 32), (3, 6, 5, 1, 3), (2, 64, 33, 31, 8), (5, 30, 3, 4, 10), (1, 128, 64, 64, 1), (2, 66, 37, 37, 11), (4, 96, 14, 14, 32),
          (1, 2, 300, 301, 1), (1, 1, 1024, 1024, 1), (2, 320, 16, 16, 32), (65, 32, 2, 2, 4), (1, 4096, 3, 3, 4), (1, 8, 257, 255, 2), (1, 24, 1, 700, 24), (1, 7, 1, 40000, 7),
          (1, 2400, 20, 20, 1), (3000, 4, 1, 1, 2), (2, 1026, 9, 7, 1), (1, 48, 130, 131, 2), (1, 33, 150, 150, 3), (1, 51, 120, 100, 3), (1, 16, 200, 200, 4), (2, 40, 90, 90, 1)]


@pytest.mark.parametrize("images, channels, height, width, groups", SHAPES)
@pytest.mark.parametrize("kind", [None, "relu", "silu"])
def test_group_norm(hip, images, channels, height, width, groups, kind):
    rng = np.random.default_rng([images, channels, height, groups])
    n = lambda *s: rng.standard_normal(s, dtype=np.float32)
    pixels = height * width
    x = n(images, channels, pixels) * (0.5 + rng.random((1, channels, 1), dtype=np.float32)) + 0.5 * n(1, channels, 1)
    full = kind != "relu"
    w, b = (1 + 0.1 * n(channels), 0.1 * n(channels)) if full else (None, None)
    mod, shift = (0.2 * n(images, channels), 0.2 * n(images, channels)) if kind == "silu" else (None, None)
    want, err = group_norm(x, groups, w, b, 1e-5, mod, shift, kind)
    d = lambda t: None if t is None else hip.array(t)
    args = dict(weight=d(w), bias=d(b), eps=1e-5, activation=kind, mod=d(mod), shift=d(shift))
    X = hip.array(x.reshape(images, channels, height, width))
    Y = hip.full(X.shape, -7.0)
    hip.group_norm(X, Y, groups, **args)
    got = Y.numpy()
    _check(got.reshape(x.shape), want, err, "maps")
    hip.group_norm(X, X, groups, **args)
    assert np.array_equal(X.numpy(), got)
    # the same as rows of tokens, channels last, whole and as columns of a wider tensor, at even and odd distances
    rows = np.ascontiguousarray(x.transpose(0, 2, 1)).reshape(images * pixels, channels)
    R = hip.array(rows)
    Y = hip.full(R.shape, -7.0)
    hip.group_norm(R, Y, groups, image_rows=pixels, **args)
    got = Y.numpy()
    back = lambda t: t.reshape(images, pixels, channels).transpose(0, 2, 1)
    _check(back(got), want, err, "rows")
    hip.group_norm(R, R, groups, image_rows=pixels, **args)
    assert np.array_equal(R.numpy(), got)
    if rows.size > 1 << 20:
        return
    for before, behind in ((4, 8), (3, 2)):
        wide = np.full((len(rows), channels + before + behind), -7.0, np.float32)
        wide[:, before:before + channels] = rows
        W, O = hip.array(wide), hip.full((len(rows), channels + behind), -7.0)
        hip.group_norm(W.columns(before, before + channels), O.columns(behind, behind + channels), groups, image_rows=pixels, **args)
        o = O.numpy()
        _check(back(o[:, behind:]), want, err, ("columns", before, behind))
        assert np.all(o[:, :behind] == -7.0)


def test_group_norm_keeps_images_and_groups_apart(hip):
    """Infinities and NaN reach their own group of their own image only; a group that is constant is its bias, far from 0 too."""
    rng = np.random.default_rng(3)
    for channels, pixels, groups in ((8, 100, 4), (64, 1500, 4), (6, 40000, 2)):
        x = rng.standard_normal((3, channels, pixels), dtype=np.float32)
        b = rng.standard_normal(channels, dtype=np.float32)
        per = channels // groups
        x[0, 0, 3], x[1, per, 7], x[2, channels - 1, pixels - 1] = np.inf, np.nan, -np.inf
        x[1, :per] = 1e4
        want, err = group_norm(np.where(np.isfinite(x), x, 0), groups, None, b, 1e-5, None, None, None)
        for i, g in ((0, 0), (1, 1), (2, groups - 1)):
            want[i, g * per:(g + 1) * per] = np.nan
        X = hip.array(x.reshape(3, channels, pixels, 1))
        hip.group_norm(X, X, groups, bias=hip.array(b))
        got = X.numpy().reshape(x.shape)
        _check(got, want, err)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        R = hip.array(x.transpose(0, 2, 1).reshape(-1, channels))
        hip.group_norm(R, R, groups, bias=hip.array(b), image_rows=pixels)
        got = R.numpy().reshape(3, pixels, channels).transpose(0, 2, 1)
        _check(got, want, err)
        assert np.array_equal(np.isnan(got), np.isnan(want))


def test_group_norm_far_from_zero(hip):
    """A mean a thousand times the spread: the variance is that of the differences, not a difference of squares."""
    rng = np.random.default_rng(4)
    for channels, side, groups in ((16, 10, 2), (4, 400, 2)):
        x = (1000 + rng.standard_normal((2, channels, side * side))).astype(np.float32)
        want, err = group_norm(x, groups, None, None, 1e-5, None, None, None)
        X = hip.array(x.reshape(2, channels, side, side))
        hip.group_norm(X, X, groups)
        _check(X.numpy().reshape(x.shape), want, err)


# ------------------------------------------------------------------------------------------------- batches
class Ragged:
    """Sequences of ``news`` new tokens with rows before and behind them that belong to none, and a pool whose slots are in no order."""

    def __init__(self, rng, news, before=2, behind=3, kept=True, apart=True):
        self.news = np.asarray(news)
        self.offsets = (before + np.concatenate([[0], np.cumsum(self.news)])).astype(np.int32)
        self.rows, seqs = int(self.offsets[-1]) + behind, len(news)
        order = rng.permutation(2 * seqs + 1).astype(np.int32)
        self.pool = 2 * seqs + 1
        self.slots, self.out_slots = order[:seqs], order[seqs:2 * seqs] if apart else order[:seqs]
        self.lengths = (self.news + np.where(np.arange(seqs) % 3 == 1, 0, rng.integers(1, 90, seqs))).astype(np.int32)
        self.kept, self.apart = kept, apart

    def on(self, hip, max_new=None):
        from eddl_amd.state_space import StateBatch
        i = lambda t: hip.array(t, "int32")
        kept = dict(lengths=i(self.lengths), slots=i(self.slots), out_slots=i(self.out_slots) if self.apart else None) if self.kept else {}
        return StateBatch(i(self.offsets), max(1, int(self.news.max(initial=0))) if max_new is None else max_new, **kept)

    def reference(self, pool):
        return dict(offsets=self.offsets, **(dict(pool=pool, lengths=self.lengths, slots=self.slots, out_slots=self.out_slots) if self.kept else {}))

    def outside(self, y):
        return np.concatenate([y[:self.offsets[0]], y[self.offsets[-1]:]])


NEWS = [[1], [5], [0, 1, 2, 3], [1] * 9, [16, 17, 0, 15, 33], [130, 1, 64], [300], [129, 7, 0, 200, 128]]


# ------------------------------------------------------------------------------------------------- causal convolution
@pytest.mark.parametrize("width", [2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("channels", [1, 7, 64, 130, 260, 1028])
def test_causal_conv(hip, width, channels):
    rng = np.random.default_rng([width, channels])
    n = lambda *s: rng.standard_normal(s, dtype=np.float32)
    for turn, news in enumerate(NEWS):
        kind, reverse, bias = (None, "silu", "relu")[turn % 3], turn % 2 == 1, None if turn == 3 else n(channels)
        batch = Ragged(rng, news, kept=turn % 4 != 2, apart=turn % 3 != 1)
        x, w, pool = n(batch.rows, channels), n(channels, width), n(batch.pool, width - 1, channels)
        want, err, after, = causal_conv(x, w, bias, kind=kind, reverse=reverse, **batch.reference(pool))
        for at, ld in ((0, channels), (3, channels + 5), (4, channels + 8 - channels % 4)):  # whole tensors, and columns of wider ones
            X, S = np.full((batch.rows, ld), 9.0, np.float32), hip.array(pool)
            X[:, at:at + channels] = x
            X, Y = hip.array(X), hip.full((batch.rows, ld), -7.0)
            hip.causal_conv(X.columns(at, at + channels), hip.array(w), None if bias is None else hip.array(bias), Y.columns(0, channels), batch.on(hip, (None, 1, 1000)[turn % 3]),
                            states=S if batch.kept else None, activation=kind, reverse=reverse)
            y = Y.numpy()
            _check(y[:, :channels], want, err, (news, at))
            assert np.all(batch.outside(y) == -7.0) and np.all(y[:, channels:] == -7.0)
            assert np.array_equal(S.numpy(), after if batch.kept else pool)


def test_causal_conv_in_pieces(hip):
    """A sequence in calls of a few tokens each, its state kept in one slot: the bits of one call."""
    from eddl_amd.state_space import StateBatch
    rng = np.random.default_rng(5)
    n = lambda *s: rng.standard_normal(s, dtype=np.float32)
    tokens, channels, width = 70, 36, 4
    x, w, b = n(tokens, channels), n(channels, width), n(channels)
    i = lambda *t: hip.array(np.array(t), "int32")
    W, b, Y = hip.array(w), hip.array(b), hip.empty((tokens, channels))
    hip.causal_conv(hip.array(x), W, b, Y, StateBatch(i(0, tokens), tokens), activation="silu")
    S, at, got = hip.full((2, width - 1, channels), np.nan), 0, []
    for piece in (1, 1, 2, 16, 1, 30, 19):
        P = hip.empty((piece, channels))
        hip.causal_conv(hip.array(x[at:at + piece]), W, b, P, StateBatch(i(0, piece), piece, i(at + piece), i(1)), states=S, activation="silu")
        got.append(P.numpy())
        at += piece
    assert at == tokens and np.array_equal(np.concatenate(got), Y.numpy())
    assert np.array_equal(S.numpy()[1], x[-3:]) and np.all(np.isnan(S.numpy()[0]))


# ------------------------------------------------------------------------------------------------- selective scan
def _scan_case(rng, batch, channels, n, groups, softplus=True, gate=True, skip=True):
    r = lambda *s: rng.standard_normal(s, dtype=np.float32)
    rows = batch.rows
    steps = np.exp(rng.random(channels) * np.log(100) + np.log(0.001))
    return dict(x=r(rows, channels), dt=0.5 * r(rows, channels) if softplus else (steps * np.exp(0.3 * r(rows, channels))).astype(np.float32),
                dt_bias=(steps + np.log(-np.expm1(-steps))).astype(np.float32) if softplus else None,
                A=(-np.arange(1, n + 1) * (0.8 + 0.4 * rng.random((channels, n)))).astype(np.float32), B=r(rows, groups * n), C=r(rows, groups * n),
                skip=r(channels) if skip else None, gate=2 * r(rows, channels) if gate else None, softplus=softplus)


def _scan(hip, case, batch, pool, reverse, max_new=None, at=0, wider=0):
    """(output, pool afterwards) of the call on columns of tensors that are ``wider``."""
    def columns(t):
        if t is None:
            return None
        wide = np.full((len(t), t.shape[1] + wider), 9.0, np.float32)
        wide[:, at:at + t.shape[1]] = t
        return hip.array(wide).columns(at, at + t.shape[1])
    d = lambda t: None if t is None else hip.array(t)
    channels = case["x"].shape[1]
    Y, S = hip.full((batch.rows, channels + wider), -7.0), hip.array(pool)
    hip.selective_scan(columns(case["x"]), columns(case["dt"]), d(case["A"]), columns(case["B"]), columns(case["C"]), Y.columns(at, at + channels), batch.on(hip, max_new),
                       states=S if batch.kept else None, skip=d(case["skip"]), gate=columns(case["gate"]), dt_bias=d(case["dt_bias"]), softplus=case["softplus"], reverse=reverse)
    y = Y.numpy()
    outside = np.concatenate([y[:, :at], y[:, at + channels:]], 1)
    assert np.all(outside == -7.0)
    return y[:, at:at + channels], S.numpy()


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 12, 16, 17, 24, 32, 48, 64])
@pytest.mark.parametrize("channels, groups", [(1, 1), (6, 3), (64, 1), (130, 2), (264, 1)])
def test_selective_scan(hip, n, channels, groups):
    rng = np.random.default_rng([n, channels])
    for turn, news in enumerate(NEWS):
        batch = Ragged(rng, news, kept=turn % 4 != 2, apart=turn % 3 != 1)
        case = _scan_case(rng, batch, channels, n, groups, softplus=turn % 3 != 0, gate=turn % 4 != 3, skip=turn % 5 != 4)
        reverse, pool = turn % 2 == 1, rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
        want, err, after, after_err = selective_scan(reverse=reverse, **case, **batch.reference(pool))
        for at, wider in ((0, 0), (3, 5), (4, 8)):
            y, s = _scan(hip, case, batch, pool, reverse, (None, 1, 1000)[(turn + at) % 3], at, wider)
            _check(y, want, err, (news, at))
            assert np.all(batch.outside(y) == -7.0)
            if batch.kept:
                _check(s, after, after_err, (news, "state"))
                untouched = np.ones(batch.pool, bool)
                untouched[batch.out_slots[batch.news > 0]] = False
                assert np.array_equal(s[untouched], pool[untouched])


@pytest.mark.parametrize("channels, n, news", [(16, 16, [5000]), (5, 16, [3001, 40]), (64, 16, [2000]), (128, 4, [1500, 1000]), (40, 1, [4000]), (33, 64, [1025]), (600, 16, [700, 30, 2, 650]), (16, 16, [9000]), (24, 8, [2100, 1, 1030]), (3, 16, [33000]), (2, 1, [20000, 9]),
                                               (1500, 8, [400] * 3)])
def test_selective_scan_of_long_sequences(hip, channels, n, news):
    rng = np.random.default_rng([channels, n])
    batch = Ragged(rng, news, apart=False)
    case = _scan_case(rng, batch, channels, n, 1)
    pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
    for reverse in (False, True):
        want, err, after, after_err = selective_scan(reverse=reverse, **case, **batch.reference(pool))
        y, s = _scan(hip, case, batch, pool, reverse)
        _check(y, want, err)
        _check(s, after, after_err)
        assert np.all(batch.outside(y) == -7.0)
        again, t = _scan(hip, case, batch, pool, reverse)
        assert np.array_equal(y, again) and np.array_equal(s, t)


def test_selective_scan_of_growing_and_of_constant_states(hip):
    """A of 0 keeps what came, a positive one grows; steps of 0 leave the state as it is, steps of 40 wipe it."""
    rng = np.random.default_rng(6)
    for channels, n in ((20, 16), (64, 4), (3, 1)):
        batch = Ragged(rng, [150, 20])
        case = _scan_case(rng, batch, channels, n, 1, softplus=False)
        case["A"][:, 0] = 0
        case["A"][1, :] = 0.5
        case["dt"][:, 2 % channels] = 0
        case["dt"][10:60:7] = 40 / np.arange(1, channels + 1) ** 2
        case["A"][case["A"] > 0.4] = 0.02
        pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
        want, err, after, after_err = selective_scan(**case, **batch.reference(pool))
        y, s = _scan(hip, case, batch, pool, False)
        _check(y, want, err)
        _check(s, after, after_err)


def test_softplus_over_its_range(hip):
    """One token whose state starts from zeros and whose A is 0: the output is d itself, within 14 EPS from steps of e^-80 to steps of 100."""
    from eddl_amd.state_space import StateBatch
    v = np.concatenate([np.linspace(-80, 100, 3000), np.linspace(-1, 1, 500), -np.logspace(-8, 1, 300), np.logspace(-8, 1, 200)]).astype(np.float32)
    X, one = hip.full((1, len(v)), 1.0), hip.full((1, 1), 1.0)
    Y = hip.empty(X.shape)
    hip.selective_scan(X, hip.array(v[None]), hip.full((len(v), 1), 0.0), one, one, Y, StateBatch(hip.array(np.array([0, 1]), "int32"), 1))
    want = np.logaddexp(v.astype(np.float64), 0)
    off = np.abs(Y.numpy()[0] - want) / want
    assert off.max() <= 14 * EPS, (off.max() / EPS, v[off.argmax()])


def test_gate_over_its_range(hip):
    from eddl_amd.state_space import StateBatch
    v = np.concatenate([np.linspace(-80, 100, 3000), np.linspace(-1, 1, 500)]).astype(np.float32)
    X, one = hip.full((1, len(v)), 1.0), hip.full((1, 1), 0.0)
    Y = hip.empty(X.shape)
    hip.selective_scan(X, X, hip.full((len(v), 1), 0.0), one, one, Y, StateBatch(hip.array(np.array([0, 1]), "int32"), 1), skip=hip.full((len(v),), 1.0), gate=hip.array(v[None]),
                       softplus=False)
    v = v.astype(np.float64)
    want = v / (1 + np.exp(-v))
    off = np.abs(Y.numpy()[0] - want) / np.maximum(np.abs(want), 2.0 ** -100)
    assert off.max() <= 11 * EPS, off.max() / EPS


def test_an_infinite_factor_wipes_the_state(hip):
    """A of minus infinity: what a token finds is gone behind it, and the last token's product is what is kept, however many tokens fill the tiles."""
    rng = np.random.default_rng(12)
    for news in ([1, 2, 3], [5, 17, 130]):
        batch = Ragged(rng, news)
        case = _scan_case(rng, batch, 20, 6, 1)
        case["A"][:, 2], case["A"][3] = -np.inf, -3e38
        pool = rng.standard_normal((batch.pool, 20, 6), dtype=np.float32)
        want, err, after, after_err = selective_scan(**case, **batch.reference(pool))
        y, s = _scan(hip, case, batch, pool, False)
        assert np.all(np.isfinite(want[batch.offsets[0]:batch.offsets[-1]])) and np.all(np.isfinite(after))
        _check(y, want, err)
        _check(s, after, after_err)


@pytest.mark.parametrize("channels, n", [(20, 16), (64, 4), (7, 1), (130, 64)])
def test_infinities_and_nan_stay_in_their_channel(hip, channels, n):
    """An input that is not finite: from its token on the channel is infinite or NaN, before it and in other channels and sequences nothing changes by a bit.  A
    NaN among B or C reaches the channels that share them.  Slots that a sequence does not continue are not read."""
    rng = np.random.default_rng(7)
    batch = Ragged(rng, [140, 33, 1])
    case = _scan_case(rng, batch, channels, n, 1)
    case["A"] = np.maximum(case["A"], -2)
    pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
    pool[batch.slots[1]] = np.nan  # (sequence 1 begins)
    y, s = _scan(hip, case, batch, pool, False)
    assert np.all(np.isfinite(y[batch.offsets[0]:batch.offsets[-1]]))
    for value in (np.inf, np.nan):
        bad = dict(case, x=case["x"].copy())
        at = int(batch.offsets[0]) + 77
        bad["x"][at, 2] = value
        y2, s2 = _scan(hip, bad, batch, pool, False)
        end = int(batch.offsets[1])
        assert not np.any(np.isfinite(y2[at:end, 2])) and not np.any(np.isfinite(s2[batch.out_slots[0], 2]))
        y2[at:end, 2], s2[batch.out_slots[0], 2] = y[at:end, 2], s[batch.out_slots[0], 2]
        assert np.array_equal(y, y2) and np.array_equal(s, s2, equal_nan=True)
    bad = dict(case, C=case["C"].copy())
    bad["C"][at, n - 1] = np.nan
    y2, s2 = _scan(hip, bad, batch, pool, False)
    assert np.all(np.isnan(y2[at])) and np.array_equal(s, s2, equal_nan=True)
    y2[at] = y[at]
    assert np.array_equal(y, y2)


def test_slots_outside_the_pool(hip):
    """A sequence that continues a state outside the pool is NaN, one whose state goes there is right and not kept; nothing else changes.  Offsets that
    run backwards or out of range are cut."""
    rng = np.random.default_rng(8)
    for channels, n in ((12, 16), (70, 3)):
        for news in ([1, 1, 1, 1], [20, 200, 3, 150]):
            batch = Ragged(rng, news)
            batch.lengths[:] = batch.news + 5
            case = _scan_case(rng, batch, channels, n, 1)
            pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
            batch.slots[1], batch.out_slots[2], batch.out_slots[3] = batch.pool, -1, 1 << 30
            want, err, after, after_err = selective_scan(**case, **batch.reference(pool))
            y, s = _scan(hip, case, batch, pool, False)
            _check(y, want, err)
            _check(s, after, after_err)
            lost = slice(int(batch.offsets[1]), int(batch.offsets[2]))
            assert np.all(np.isnan(y[lost])) and np.all(np.isnan(s[batch.out_slots[1]])) and np.array_equal(np.isnan(s), np.isnan(after))
            x, w, states = case["x"], rng.standard_normal((channels, 4), dtype=np.float32), rng.standard_normal((batch.pool, 3, channels), dtype=np.float32)
            want, err, after = causal_conv(x, w, None, kind="silu", reverse=False, **batch.reference(states))
            Y, S = hip.full(x.shape, -7.0), hip.array(states)
            hip.causal_conv(hip.array(x), hip.array(w), None, Y, batch.on(hip), states=S, activation="silu")
            y = Y.numpy()
            _check(y, want, err)
            first = int(batch.offsets[1])
            assert np.all(np.isnan(y[first:first + min(news[1], 3)])) and np.array_equal(S.numpy(), after, equal_nan=True)
            batch.offsets[:] = [-5, 7, 3, 1 << 30, -(1 << 31)]
            batch.lengths[:] = 0
            batch.out_slots[:] = -1
            for reverse in (False, True):
                want, err = selective_scan(reverse=reverse, **case, **batch.reference(pool))[:2]
                y, s = _scan(hip, case, batch, pool, reverse)
                # (sequences 0 and 2 share rows 3 .. 6, whose results are those of either)
                _check(y[7:], want[7:], err[7:])
                assert np.array_equal(s, pool)


def test_single_tokens_continue_a_prompt(hip):
    """A prompt, then token by token and in small pieces, against the whole sequence at once: both within the bounds."""
    from eddl_amd.state_space import StateBatch
    rng = np.random.default_rng(9)
    for channels, n in ((48, 16), (20, 5), (256, 32)):
        tokens, batch = 160, Ragged(rng, [160], before=0, behind=0, kept=False)
        case = _scan_case(rng, batch, channels, n, 1)
        want, err = selective_scan(offsets=[0, tokens], **case)[:2]
        S = hip.full((3, channels, n), np.nan)
        at = 0
        i = lambda *t: hip.array(np.array(t), "int32")
        d = lambda t: hip.array(t[at:at + piece])
        for piece in (100, 1, 1, 1, 2, 7, 1, 17, 30):
            Y = hip.empty((piece, channels))
            hip.selective_scan(d(case["x"]), d(case["dt"]), hip.array(case["A"]), d(case["B"]), d(case["C"]), Y, StateBatch(i(0, piece), piece, i(at + piece), i(2)), states=S,
                               skip=hip.array(case["skip"]), gate=d(case["gate"]), dt_bias=hip.array(case["dt_bias"]))
            _check(Y.numpy(), want[at:at + piece], err[at:at + piece], at)
            at += piece
        assert at == tokens and np.all(np.isnan(S.numpy()[:2]))


def test_empty_calls(hip):
    from eddl_amd.state_space import StateBatch
    none, E, V = StateBatch(hip.array(np.zeros(3), "int32") if False else hip.array(np.zeros(3, np.int32), "int32"), 1), hip.empty((0, 8)), hip.empty((0, 4))
    hip.causal_conv(E, hip.full((8, 4), 1.0), None, E, none)
    hip.selective_scan(E, E, hip.full((8, 4), 1.0), V, V, E, none)
    hip.group_norm(E, E, 2)
    hip.group_norm(hip.empty((0, 8, 3, 3)), hip.empty((0, 8, 3, 3)), 2)
    X, Y, V = hip.full((5, 8), 1.0), hip.full((5, 8), -7.0), hip.full((5, 4), 1.0)
    hip.causal_conv(X, hip.full((8, 4), 1.0), None, Y, none)
    hip.selective_scan(X, X, hip.full((8, 4), 1.0), V, V, Y, none)
    assert np.all(Y.numpy() == -7.0)


# ------------------------------------------------------------------------------------------------- graphs, networks, large tensors
def test_recorded_steps_follow_the_batch(hip):
    """A recorded convolution and scan, replayed while offsets, lengths and slots change: every replay equals the eager calls on the same states, with the program's own
    work between the replays."""
    rng = np.random.default_rng(20)
    channels, n, width, seqs = 40, 16, 4, 3
    for most in (1, 40, 700):
        batch = Ragged(rng, [most] * seqs, before=0, behind=0, apart=False)
        case = _scan_case(rng, batch, channels, n, 1)
        d = lambda t: hip.array(t)
        X, W, U, Y, dt, A, B, C, D, G, bias = d(case["x"]), d(rng.standard_normal((channels, width))), hip.empty(case["x"].shape), hip.empty(case["x"].shape), d(case["dt"]), d(case["A"]), \
            d(case["B"]), d(case["C"]), d(case["skip"]), d(case["gate"]), d(case["dt_bias"])
        inputs, states = rng.standard_normal((batch.pool, width - 1, channels), dtype=np.float32), rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
        P, S, b = d(inputs), d(states), batch.on(hip, most)

        def step():
            hip.causal_conv(X, W, None, U, b, states=P, activation="silu")
            hip.selective_scan(U, dt, A, B, C, Y, b, states=S, skip=D, gate=G, dt_bias=bias)
            hip.group_norm(Y, Y, 8, image_rows=batch.rows)

        step()
        graph = hip.record(step)
        for turn in range(3):
            news = np.minimum(np.array([[most, most, most], [most, 0, most // 2], [1, most, 0]][turn]), most)
            b.offsets.copy_from(np.concatenate([[0], np.cumsum(news)]))
            b.lengths.copy_from(news + [5, 0, 7])
            b.slots.copy_from(rng.permutation(batch.pool)[:seqs])
            got = []
            for run in (step, graph.launch):
                P.copy_from(inputs)
                S.copy_from(states)
                hip.fill_(Y, 0.5)
                X.copy_from(case["x"] * (turn + 1))
                run()
                got.append((Y.numpy(), P.numpy(), S.numpy()))
            for e, g in zip(*got):
                assert np.array_equal(e, g), (most, turn)


def test_calls_on_changing_streams(hip):
    """Divided groups and divided sequences share the library's workspace: calls on two streams in turn give the bits of calls on one."""
    import ctypes
    rng = np.random.default_rng(21)
    streams = [ctypes.c_void_p() for _ in range(2)]
    for s in streams:
        assert hip.lib.hipStreamCreateWithFlags(ctypes.byref(s), 1) == 0
    batch = Ragged(rng, [3000], kept=False)
    case = _scan_case(rng, batch, 24, 16, 1)
    X = hip.array(rng.standard_normal((1, 2, 400, 300)))
    try:
        Y, want = hip.empty(X.shape), None
        for turn in range(6):
            hip._check(hip.lib.eddlhip_set_stream(hip.dev, streams[turn % 2]))
            hip.group_norm(X, Y, 2)
            got = (_scan(hip, case, batch, np.zeros((batch.pool, 24, 16), np.float32), False)[0], Y.numpy())
            want = want or got
            assert all(np.array_equal(a, b) for a, b in zip(want, got)), turn
    finally:
        hip._check(hip.lib.eddlhip_set_stream(hip.dev, None))
        for s in streams:
            hip.lib.hipStreamDestroy(s)


def test_net_of_state_space_blocks(hip):
    """A network that scans the tokens of images both ways between group norms: norm, dense, convolution, dense, scan forwards; the same backwards; Add, dense, Add, norm with
    SiLU.  The fused plan, the layer walk and a captured plan give the same bits, and the network in 64 bits within 2e-5 of its largest output (some tens of EPS a stage)."""
    from eddl_amd import net as L
    rng = np.random.default_rng(22)
    images, tokens, cols, inner, n, rank = 3, 49, 32, 48, 8, 4

    def build(fuse):
        x = L.Input([tokens, cols], images)
        xz = L.Dense(L.GroupNormalization(x, 8), 2 * inner, use_bias=False)
        sides = []
        for reverse in (False, True):
            u = L.CausalConvolution(xz, 4, channels=inner, reverse=reverse)
            proj = L.Dense(u, rank + 2 * n, use_bias=False)
            sides.append(L.SelectiveScan(u, L.Dense(u, inner, use_bias=False), proj, n, gate=xz, reverse=reverse))
        s = L.Add(x, L.Dense(L.Add(*sides), cols))
        net = L.Net([x], [L.GroupNormalization(s, 4, activation="silu"), L.ReLu(L.GroupNormalization(s, 1, affine=False))])
        r = np.random.default_rng(23)
        for l in net.layers:
            for k, v in l.params.items():
                if k != "A":
                    scale = 1 / np.sqrt(v.shape[0]) if l.kind == "dense" and k == "W" else 0.5 if k == "W" else 0.1
                    l.params[k] = ((1.0 if k in ("w", "skip") else -2.0 if k == "dt_bias" else 0.0) + scale * r.standard_normal(v.shape)).astype(np.float32)
        return net.build(hip, fuse=fuse)

    fused, walk = build(True), build(False)
    assert sum(op.kind == "relu" for op in walk.ops) == 1 and not any(op.kind == "relu" for op in fused.ops)
    x = rng.standard_normal((images, tokens, cols), dtype=np.float32)
    got = fused.predict(x)
    graph = fused.capture()
    for a, b in zip(walk.predict(x), got):
        assert np.array_equal(a, b)
    for turn in range(2):
        fused.input_tensor().copy_from(x)
        fused.run_graph()
        for o, b in zip(fused.lout, got):
            assert np.array_equal(fused.output_of(o).numpy(), b)
    # in 64 bits
    by = lambda kind: [{k: v.astype(np.float64) for k, v in l.params.items()} for l in fused.layers if l.kind == kind]
    norms, denses, convs, scans = by("group_norm"), [l for l in fused.layers if l.kind == "dense"], [l for l in fused.layers if l.kind == "causal_conv"], \
        [l for l in fused.layers if l.kind == "selective_scan"]
    W = lambda l: {k: v.astype(np.float64) for k, v in l.params.items()}

    def norm(t, groups, p, eps):
        v = t.reshape(images, tokens, groups, -1)
        v = (v - v.mean((1, 3), keepdims=True)) / np.sqrt(v.var((1, 3), keepdims=True) + eps)
        v = v.reshape(t.shape)
        return v * p["w"] + p["b"] if p else v
    layer = {id(l): l for l in fused.layers}
    assert len(layer) == len(fused.layers)
    first = [l for l in fused.layers if l.kind == "group_norm" and l.parents[0].kind == "input"][0]
    z = norm(x.astype(np.float64), 8, W(first), 1e-3) @ W([l for l in denses if l.parents[0] is first][0])["W"]
    total = 0
    for conv in convs:
        scan = [l for l in scans if l.parents[0] is conv][0]
        c, p, flip = W(conv), W(scan), slice(None, None, -1 if conv.attrs["reverse"] else 1)
        u = np.concatenate([np.zeros((images, 3, inner)), z[:, flip, :inner]], 1)
        u = sum(u[:, k:k + tokens] * c["W"][:, k] for k in range(4)) + c["bias"]
        u = u / (1 + np.exp(-u))
        dt = np.logaddexp(u @ W(scan.parents[1])["W"] + p["dt_bias"], 0)
        v = u @ W(scan.parents[2])["W"]
        h, out = np.zeros((images, inner, n)), []
        for t in range(tokens):
            h = np.exp(dt[:, t, :, None] * p["A"]) * h + (dt[:, t] * u[:, t])[:, :, None] * v[:, t, None, rank:rank + n]
            out.append((h * v[:, t, None, rank + n:]).sum(2) + p["skip"] * u[:, t])
        total = total + np.stack(out, 1)[:, flip] * (z[:, :, inner:] / (1 + np.exp(-z[:, :, inner:])))
    last = [l for l in denses if l.parents[0].kind == "sum"][0]
    s = x + total @ W(last)["W"] + W(last)["bias"]
    a = norm(s, 4, W([l for l in fused.layers if l.kind == "group_norm" and l.attrs["activation"]][0]), 1e-3)
    for g, w in zip(got, (a / (1 + np.exp(-a)), np.maximum(norm(s, 1, None, 1e-3), 0))):
        assert np.abs(g - w).max() <= 2e-5 * np.abs(w).max(), np.abs(g - w).max() / np.abs(w).max()


def test_net_of_group_norms_on_maps(hip):
    """Convolution, group norm, ReLU: one launch for the last two in a fused plan, the same bits as the layer walk, another batch size behind it."""
    from eddl_amd import net as L
    rng = np.random.default_rng(24)
    nets = []
    for fuse in (True, False):
        x = L.Input([6, 13, 11], 2)
        net = L.Net([x], [L.ReLu(L.GroupNormalization(L.Conv2D(x, 12, [3, 3]), 4))])
        r = np.random.default_rng(25)
        for l in net.layers:
            for k, v in l.params.items():
                l.params[k] = (0.3 * r.standard_normal(v.shape)).astype(np.float32)
        nets.append(net.build(hip, fuse=fuse))
    assert [op.kind for op in nets[0].ops] == ["conv2d", "group_norm"] and [op.kind for op in nets[1].ops][-1] == "relu"
    for batch in (2, 5):
        x = rng.standard_normal((batch, 6, 13, 11), dtype=np.float32)
        a, b = (net.predict(x)[0] for net in nets)
        conv = nets[1].output_of([l for l in nets[1].layers if l.kind == "conv2d"][0]).numpy()
        p = [l for l in nets[0].layers if l.kind == "group_norm"][0].params
        want, err = group_norm(conv.reshape(batch, 12, -1), 4, p["w"], p["b"], 1e-3, None, None, "relu")
        assert np.array_equal(a, b)
        _check(a.reshape(want.shape), want, err)


def test_places_beyond_32_bits(hip):
    """Columns of a tensor of 2.4e9 numbers: the last rows lie beyond what 32 bits count, in numbers and in bytes."""
    from eddl_amd.state_space import StateBatch
    rng = np.random.default_rng(26)
    rows, ld, channels, n = 600000, 4096, 8, 16
    wide = hip.empty((rows, ld))
    hip.fill_(wide, 1.0)
    tail = 300
    x = rng.standard_normal((tail, channels), dtype=np.float32)
    flat = wide.reshape((rows * ld,))
    for t in range(tail):  # the last rows, in the last columns
        at = ((rows - tail + t) * ld + ld - channels) * 4
        row = np.ascontiguousarray(x[t])
        hip._check(hip.lib.eddlhip_memcpy_h2d(hip.dev, wide.ptr + at, row.ctypes.data, row.nbytes))
    assert flat.size == rows * ld
    X = wide.columns(ld - channels, ld)
    offsets = np.array([rows - tail, rows - tail + 100, rows], np.int32)
    batch = StateBatch(hip.array(offsets, "int32"), 200)
    w = rng.standard_normal((channels, 4), dtype=np.float32)
    Y = hip.full((rows, channels), -7.0)
    hip.causal_conv(X, hip.array(w), None, Y, batch)
    want, err, _ = causal_conv(x, w, None, [0, 100, tail], None, False)
    y = Y.numpy()
    _check(y[-tail:], want, err)
    assert np.all(y[:-tail] == -7.0)
    A, vectors = -np.ones((channels, n), np.float32), np.ones((tail, n), np.float32)
    hip.fill_(Y, -7.0)
    V = wide.columns(0, n)  # (ones)
    hip.selective_scan(X, X, hip.array(A), V, V, Y, batch)
    want, err = selective_scan(x, x, A, vectors, vectors, [0, 100, tail])[:2]
    y = Y.numpy()
    _check(y[-tail:], want, err)
    assert np.all(y[:-tail] == -7.0)
    hip.group_norm(X, Y, 2, image_rows=tail)
    want, err = group_norm(np.ascontiguousarray(x.T)[None], 2, None, None, 1e-5, None, None, None)
    _check(Y.numpy()[-tail:].T[None], want, err)
    whole = hip.empty(wide.shape)  # and maps: a group of 1.2e9 numbers
    hip.group_norm(wide.reshape((1, 2, rows // 2, ld)), whole.reshape((1, 2, rows // 2, ld)), 2, eps=1.0)
    got = np.empty(4096, np.float32)
    hip._check(hip.lib.eddlhip_memcpy_d2h(hip.dev, got.ctypes.data, whole.ptr + 4 * (rows * ld - 4096), got.nbytes))
    # (the second group: ones, but for the tail's numbers)
    total, count = x.astype(np.float64), rows * ld // 2
    mean = 1 + (total - 1).sum() / count
    var = ((1 - mean) ** 2 * (count - x.size) + ((total - mean) ** 2).sum()) / count
    row = np.concatenate([np.ones(ld - channels), x[-1]])
    want = (row - mean) / np.sqrt(var + 1.0)
    assert np.abs(got - want).max() <= 128 * EPS * np.abs(row).max()


# ------------------------------------------------------------------------------------------------- sequences whose parts several workgroups take
@pytest.mark.parametrize("channels, n, news", [(12, 16, [1200, 0, 700]), (40, 3, [2100, 17, 900, 1]), (5, 40, [2500])])
def test_divided_sequences(hip, channels, n, news):
    """Sequences with tokens and without, short and long, whose states come from other slots than they go to; with a bound below and far above the new
    tokens, and several sequences that continue one slot."""
    rng = np.random.default_rng([channels, n, 1])
    batch = Ragged(rng, news)
    case = _scan_case(rng, batch, channels, n, 1)
    pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
    for fork in (False, True):
        if fork:
            batch.slots = np.full(len(news), batch.slots[0], np.int32)
            batch.lengths = (batch.news + 3).astype(np.int32)
        for reverse in (False, True):
            want, err, after, after_err = selective_scan(reverse=reverse, **case, **batch.reference(pool))
            for most in (None, 600, 1 << 20):
                y, s = _scan(hip, case, batch, pool, reverse, most)
                _check(y, want, err, (fork, most))
                _check(s, after, after_err, (fork, most, "state"))
                assert np.all(batch.outside(y) == -7.0)


def test_not_finite_numbers_of_divided_sequences(hip):
    """As in short sequences: nothing changes by a bit before the token, in other channels and in other sequences; a state outside the pool makes its sequence NaN."""
    rng = np.random.default_rng(31)
    channels, n = 20, 16
    batch = Ragged(rng, [3000, 900])
    batch.lengths[:] = batch.news + 2
    case = _scan_case(rng, batch, channels, n, 1)
    case["A"] = np.maximum(case["A"], -2)
    pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
    y, s = _scan(hip, case, batch, pool, False)
    for value in (np.inf, np.nan):
        for token in (0, 1234, 2999):
            bad = dict(case, x=case["x"].copy())
            at, end = int(batch.offsets[0]) + token, int(batch.offsets[1])
            bad["x"][at, 2] = value
            y2, s2 = _scan(hip, bad, batch, pool, False)
            assert not np.any(np.isfinite(y2[at:end, 2])) and not np.any(np.isfinite(s2[batch.out_slots[0], 2]))
            y2[at:end, 2], s2[batch.out_slots[0], 2] = y[at:end, 2], s[batch.out_slots[0], 2]
            assert np.array_equal(y, y2) and np.array_equal(s, s2)
    batch.slots[0], batch.out_slots[1] = -1, batch.pool
    y2, s2 = _scan(hip, case, batch, pool, False)
    first, second = (slice(*batch.offsets[k:k + 2]) for k in (0, 1))
    assert np.all(np.isnan(y2[first])) and np.array_equal(y2[second], y[second]) and np.all(np.isnan(s2[batch.out_slots[0]]))


def test_a_larger_call_outgrows_a_recorded_one(hip):
    """Divided sequences and groups take the workspace: one that would have to grow is refused while a graph is recorded, and a graph whose workspace was
    replaced is refused at its launch."""
    from eddl_amd.backend import EddlHipError
    rng = np.random.default_rng(32)
    batch = Ragged(rng, [2000], before=0, behind=0, kept=False)
    case = _scan_case(rng, batch, 16, 16, 1)
    d, b = (lambda t: hip.array(t)), batch.on(hip)
    X, dt, A, B, C, Y = d(case["x"]), d(case["dt"]), d(case["A"]), d(case["B"]), d(case["C"]), hip.empty(case["x"].shape)
    big = hip.empty((1, 4, 600, 512))
    hip.fill_(big, 1.0)

    def small():
        hip.selective_scan(X, dt, A, B, C, Y, b)

    hip.workspace_trim()
    small()
    want = Y.numpy()
    graph = hip.record(small)
    hip.group_norm(big, big, 2)  # (fits the workspace that stands)
    hip.fill_(Y, 0.0)
    graph.launch()
    assert np.array_equal(Y.numpy(), want)
    many = Ragged(rng, [600] * 6, before=0, behind=0, kept=False)
    wide = _scan_case(rng, many, 60, 64, 1)
    m = many.on(hip)
    W = [d(wide[k]) for k in ("x", "dt", "A", "B", "C")] + [hip.empty(wide["x"].shape)]
    with pytest.raises(EddlHipError, match="before recording"):
        hip.record(lambda: hip.selective_scan(*W, m))
    hip.selective_scan(*W, m)
    with pytest.raises(EddlHipError, match="record again"):
        graph.launch()
    graph = hip.record(small)
    hip.fill_(Y, 0.0)
    graph.launch()
    assert np.array_equal(Y.numpy(), want)


@pytest.mark.parametrize("most", [1, 9, 1 << 20])
def test_as_many_sequences_as_there_may_be(hip, most):
    """65535 sequences of no to three tokens, whatever bound the host gives; a last one of 400."""
    from eddl_amd.state_space import StateBatch
    rng = np.random.default_rng(41)
    seqs, channels, n = 65535, 5, 3
    news = rng.integers(0, 4, seqs)
    news[-1] = 400
    offsets = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    rows = int(offsets[-1])
    r = lambda *s: rng.standard_normal(s, dtype=np.float32)
    x, dt, A, B, C, w = r(rows, channels), np.exp(0.3 * r(rows, channels) - 1), -np.exp(r(channels, n)), r(rows, n), r(rows, n), r(channels, 4)
    token = np.arange(rows) - np.repeat(offsets[:-1], news)
    X, Y, batch = hip.array(x), hip.full((rows, channels), -7.0), StateBatch(hip.array(offsets, "int32"), most)
    hip.causal_conv(X, hip.array(w), None, Y, batch)
    want, size = np.zeros((rows, channels)), np.zeros((rows, channels))
    for back in range(4):
        there = np.flatnonzero(token >= back)
        product = x[there - back].astype(np.float64) * w[:, 3 - back]
        want[there] += product
        size[there] += np.abs(product)
    _check(Y.numpy(), want, 8 * EPS * size)
    hip.fill_(Y, -7.0)
    d = lambda t: hip.array(t)
    hip.selective_scan(X, d(dt), d(A), d(B), d(C), Y, batch, softplus=False)
    y = Y.numpy()
    for length in (1, 2, 3, 400):
        for s in np.flatnonzero(news == length)[::500]:
            rows_of = slice(int(offsets[s]), int(offsets[s + 1]))
            want, err = selective_scan(x[rows_of], dt[rows_of], A, B[rows_of], C[rows_of], [0, length], softplus=False)[:2]
            _check(y[rows_of], want, err, (length, s))
    assert np.all(np.isfinite(y)) and not np.any(y == -7.0)


MIXED = [(1500, 16, [1] * 20 + [300] + [2] * 20), (100, 16, [2] * 200 + [0] * 60 + [2000] + [1] * 100), (40, 40, [3] * 550 + [700, 600] + [0, 1] * 40), (520, 1, [1] * 90 + [129]),
         (300, 4, [150] + [7] * 150 + [140, 0])]


@pytest.mark.parametrize("channels, n, news", MIXED)
def test_long_sequences_among_short_ones(hip, channels, n, news):
    """A few long sequences are walked in a launch of their own, whatever the host's bound is and wherever they stand."""
    rng = np.random.default_rng([channels, n, 2])
    batch = Ragged(rng, news)
    case = _scan_case(rng, batch, channels, n, 1)
    pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
    for reverse in (False, True):
        want, err, after, after_err = selective_scan(reverse=reverse, **case, **batch.reference(pool))
        for most in (None, max(news) // 3, 1 << 20):
            y, s = _scan(hip, case, batch, pool, reverse, most)
            _check(y, want, err, (reverse, most))
            _check(s, after, after_err, (reverse, most, "state"))
            assert np.all(batch.outside(y) == -7.0)


def test_a_recorded_mixed_batch_follows_its_offsets(hip):
    """The long sequences are looked up when the kernels run: replays after the program moved them, made more of them or none equal the eager calls."""
    rng = np.random.default_rng(51)
    channels, n, seqs, most = 600, 16, 64, 400
    batch = Ragged(rng, [1] * (seqs - 1) + [most], before=0, behind=0, apart=False)
    case = _scan_case(rng, batch, channels, n, 1)
    d = lambda t: hip.array(t)
    X, dt, A, B, C, Y, b = d(case["x"]), d(case["dt"]), d(case["A"]), d(case["B"]), d(case["C"]), hip.empty(case["x"].shape), batch.on(hip, most)
    pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
    S = d(pool)
    step = lambda: hip.selective_scan(X, dt, A, B, C, Y, b, states=S)
    step()
    graph = hip.record(step)
    places = [[(5, 400)], [(0, 210), (63, 190)], [], [(k, 7) for k in range(seqs)]]
    for long in places:
        news = np.ones(seqs, int)
        for k, length in long:
            news[k] = length
        b.offsets.copy_from(np.minimum(np.concatenate([[0], np.cumsum(news)]), batch.rows))
        b.lengths.copy_from(news + 3)
        got = []
        for run in (step, graph.launch):
            S.copy_from(pool)
            hip.fill_(Y, 0.5)
            run()
            got.append((Y.numpy(), S.numpy()))
        assert all(np.array_equal(e, g) for e, g in zip(*got)), long
