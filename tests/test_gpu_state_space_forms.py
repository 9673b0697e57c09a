"""Every kernel that the rules of the selective scan and the group norm choose between, against 64 bits."""
import numpy as np
import pytest

import test_gpu_state_space as base
from state_space_ref import EPS, selective_scan
from test_gpu_state_space import Ragged, _check, _scan, _scan_case

pytestmark = pytest.mark.gpu

UNITS = 256  # compute units


def _form(channels, groups, n, seqs, tokens):
    """What the library's rule takes for sequences of up to ``tokens`` tokens."""
    lanes = 1 if n <= 4 else 2 if n <= 8 else 4 if n <= 16 else 8 if n <= 32 else 16
    tile, ch, per = 16 if lanes >= 4 else 8, 64 // lanes, channels // groups
    wide, narrow = groups * -(-per // (4 * ch)), groups * -(-per // ch)
    if tokens <= 3:
        return "tokens"
    if wide * seqs >= 2 * UNITS or tokens <= tile:
        return "one"
    if 2 * narrow * seqs >= 3 * UNITS:
        return "four"
    return "divided" if UNITS // (narrow * seqs) >= 2 and tokens > 3 * 8 * tile else "eight"


def _sizes(form, n):
    """(channels, groups, new tokens of the sequences) that take ``form``: the channels of a group are no multiple of those of a wavefront."""
    ch = 64 if n <= 4 else 32 if n <= 8 else 16 if n <= 16 else 8 if n <= 32 else 4
    rng = np.random.default_rng([n, len(form)])
    ragged = lambda seqs, low, high: [high, 0, 1] + list(rng.integers(low, high, seqs - 3))
    channels, news = {"tokens": (2 * ch + 2, ragged(9, 1, 3)), "one": (2 * (12 * ch + ch // 2 + 1), ragged(64, 3, 45)), "four": (2 * (12 * ch + ch // 4 + 1), ragged(16, 33, 90)),
                      "eight": (2 * (12 * ch + 3), ragged(6, 130, 300)), "divided": (2 * (6 * ch + 1), ragged(3, 0, 901)[:1] + [700, 40])}[form]
    assert _form(channels, 2, n, len(news), max(news)) == form
    return channels, 2, news


FORMS = ["tokens", "one", "four", "eight", "divided"]


@pytest.mark.parametrize("n", [1, 3, 7, 8, 13, 16, 31, 64])
@pytest.mark.parametrize("form", FORMS)
def test_every_form_of_the_scan(hip, form, n):
    """Odd channels, two groups, ragged sequences with and without tokens, states read from and written to slots, both directions; an input that is not finite stays in its
    channel and sequence, and no bit changes before it."""
    channels, groups, news = _sizes(form, n)
    rng = np.random.default_rng([n, channels])
    batch = Ragged(rng, news, apart=n % 2 == 1)
    case = _scan_case(rng, batch, channels, n, groups)
    case["A"] = np.maximum(case["A"], -3)
    pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
    for reverse in (False, True):
        want, err, after, after_err = selective_scan(reverse=reverse, **case, **batch.reference(pool))
        y, s = _scan(hip, case, batch, pool, reverse, at=3 * reverse, wider=5 * reverse)
        _check(y, want, err, reverse)
        _check(s, after, after_err, (reverse, "state"))
        assert np.all(batch.outside(y) == -7.0)
        untouched = np.setdiff1d(np.arange(batch.pool), batch.out_slots[batch.news > 0])
        assert np.array_equal(s[untouched], pool[untouched])
        at, end, c = int(batch.offsets[0]) + news[0] // 2, int(batch.offsets[1]), channels - 1
        bad = dict(case, x=case["x"].copy())
        bad["x"][at, c] = np.inf
        y2, s2 = _scan(hip, bad, batch, pool, reverse, at=3 * reverse, wider=5 * reverse)
        lost = slice(int(batch.offsets[0]), at + 1) if reverse else slice(at, end)
        assert not np.any(np.isfinite(y2[lost, c])) and not np.any(np.isfinite(s2[batch.out_slots[0], c]))
        y2[lost, c], s2[batch.out_slots[0], c] = y[lost, c], s[batch.out_slots[0], c]
        assert np.array_equal(y, y2) and np.array_equal(s, s2)


def _bounds_of_runs(case, batch, pool):
    """Bounds of outputs and states where runs of tokens are joined: F h + H, F a run's factor, H its state from zeros.

    The recurrence's own bound takes errors relative to the state that it has: a token's rel |h|.  Joined, F h and H are off relative to themselves.  Where they cancel and the
    state grows, F h may be large, and carry the errors of all of the run's tokens, beside a small F h + H: of h = 1 and a first product of -1 the recurrence carries one token's error
    on, F h those of 8 or 16.  But every term, h or a product, times the factors behind it, is off by at most the sum of these tokens' errors relative to itself, in any order of
    joining; and that is what the recurrence's bound is where nothing cancels: with the magnitudes of states, inputs, B and C."""
    sizes = dict(case, x=np.abs(case["x"]), B=np.abs(case["B"]), C=np.abs(case["C"]))
    _, err, _, after_err = selective_scan(**sizes, **batch.reference(np.abs(pool)))
    return err, after_err


@pytest.mark.parametrize("n", [1, 4, 8, 16, 32, 64])
@pytest.mark.parametrize("form", FORMS)
def test_growing_states_in_every_form(hip, form, n):
    """Positive A, whose factors over a tile's or a sequence's tokens pass the largest number: a state of zeros stays zeros until its first input, one of 1e-30 grows as the
    formula says, whichever kernel the batch takes."""
    channels, groups, news = _sizes(form, n)
    rng = np.random.default_rng([n, channels, 5])
    batch = Ragged(rng, news)
    case = _scan_case(rng, batch, channels, n, groups, softplus=False, gate=False, skip=False)
    case["A"] = (0.5 + rng.random((channels, n))).astype(np.float32)
    last = np.concatenate([np.arange(b - min(4, k), b) for b, k in zip(batch.offsets[1:], news)])  # four tokens of every sequence
    # steps of 9: a factor of up to e^13 a token; the inputs come last
    zero = dict(case, x=np.zeros_like(case["x"]), dt=np.full_like(case["dt"], 9.0))
    zero["x"][last], zero["dt"][last] = case["x"][last], 0.3
    batch.lengths[:] = batch.news  # (every sequence begins)
    pool = np.zeros((batch.pool, channels, n), np.float32)
    want, err, after, after_err = selective_scan(**zero, **batch.reference(pool))
    y, s = _scan(hip, zero, batch, pool, False)
    _check(y, want, err, "zeros")
    _check(s, after, after_err, "zeros, state")
    # states and inputs of 1e-30, a growth of e^60 to e^130 over the longest sequence
    tiny = dict(case, x=case["x"] * np.float32(1e-30), dt=np.full_like(case["dt"], 88.0 / max(news)))
    batch.lengths[:] = batch.news + 5
    pool = (1e-30 * rng.standard_normal((batch.pool, channels, n))).astype(np.float32)
    want, _, after, _ = selective_scan(**tiny, **batch.reference(pool))
    err, after_err = _bounds_of_runs(tiny, batch, pool)
    assert np.abs(want[batch.offsets[0]:batch.offsets[-1]]).max() < 1e32
    y, s = _scan(hip, tiny, batch, pool, False)
    _check(y, want, err, "1e-30")
    _check(s, after, after_err, "1e-30, state")


@pytest.mark.parametrize("n", [1, 4, 8, 16, 32, 64])
@pytest.mark.parametrize("form", FORMS)
def test_steps_whose_sum_passes_the_largest_number(hip, form, n):
    """Steps of 1e38: negative A leaves nothing of what came before, A of 0 all of it."""
    channels, groups, news = _sizes(form, n)
    rng = np.random.default_rng([n, channels, 6])
    batch = Ragged(rng, news)
    case = _scan_case(rng, batch, channels, n, groups, softplus=False)
    case["A"] = -np.exp(rng.standard_normal((channels, n), dtype=np.float32))
    case["A"][::2, 0] = 0
    case["dt"][:], case["x"] = 1e38, case["x"] * np.float32(1e-38)
    batch.lengths[:] = batch.news + 5
    pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
    for reverse in (False, True):
        want, err, after, after_err = selective_scan(reverse=reverse, **case, **batch.reference(pool))
        y, s = _scan(hip, case, batch, pool, reverse)
        _check(y, want, err, reverse)
        _check(s, after, after_err, (reverse, "state"))
        assert np.all(np.isfinite(s)) and np.all(np.isfinite(y[batch.offsets[0]:batch.offsets[-1]]))


@pytest.mark.parametrize("n", [1, 4, 8, 16, 32, 64])
@pytest.mark.parametrize("form", FORMS)
def test_steps_of_both_signs_in_every_form(hip, form, n):
    """Without softplus steps may be negative: states decay and grow in turns, by some e^9 over the longest sequence."""
    channels, groups, news = _sizes(form, n)
    rng = np.random.default_rng([n, channels, 7])
    batch = Ragged(rng, news)
    case = _scan_case(rng, batch, channels, n, groups, softplus=False)
    case["dt"], case["A"] = 0.3 * rng.standard_normal(case["dt"].shape, dtype=np.float32), -rng.random((channels, n), dtype=np.float32)
    pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
    want, _, after, _ = selective_scan(**case, **batch.reference(pool))
    err, after_err = _bounds_of_runs(case, batch, pool)
    y, s = _scan(hip, case, batch, pool, False)
    _check(y, want, err)
    _check(s, after, after_err, "state")


@pytest.mark.parametrize("form", FORMS)
def test_inputs_and_outputs_of_one_tensor(hip, form):
    """A block's numbers as columns of one tensor, the output's columns between the inputs'; a step without gate, skip and bias beside it gives other outputs, the states' bits."""
    n = 16
    channels, groups, news = _sizes(form, n)
    rng = np.random.default_rng([channels, 8])
    batch = Ragged(rng, news)
    case = _scan_case(rng, batch, channels, n, groups)
    pool = rng.standard_normal((batch.pool, channels, n), dtype=np.float32)
    y, s = _scan(hip, case, batch, pool, False)
    parts, at = {}, 1
    for k in ("x", "B", "y", "dt", "C", "gate"):
        width = channels if k == "y" else case[k].shape[1]
        parts[k], at = (at, at + width), at + width
    wide = np.full((batch.rows, at + 2), 5.0, np.float32)
    for k, (a, b) in parts.items():
        wide[:, a:b] = -7.0 if k == "y" else case[k]
    T, S, d = hip.array(wide), hip.array(pool), lambda k: hip.array(case[k])
    c = {k: T.columns(*ab) for k, ab in parts.items()}
    hip.selective_scan(c["x"], c["dt"], d("A"), c["B"], c["C"], c["y"], batch.on(hip), states=S, skip=d("skip"), gate=c["gate"], dt_bias=d("dt_bias"))
    wide[:, slice(*parts["y"])] = y
    assert np.array_equal(T.numpy(), wide) and np.array_equal(S.numpy(), s)
    S, Y = hip.array(pool), hip.full((batch.rows, channels), -7.0)
    hip.selective_scan(c["x"], c["dt"], d("A"), c["B"], c["C"], Y, batch.on(hip), states=S, dt_bias=d("dt_bias"))
    bare = dict(case, gate=None, skip=None)
    want, err, after, after_err = selective_scan(**bare, **batch.reference(pool))
    _check(Y.numpy(), want, err)
    assert np.array_equal(S.numpy(), s) and np.all(batch.outside(Y.numpy()) == -7.0)


# ------------------------------------------------------------------------------------------------- group norm
# odd wide rows, whole and divided; odd maps, divided; even wide rows, whole; short groups of rows two numbers at a time; one group of them
@pytest.mark.parametrize("images, channels, height, width, groups", [(2, 99, 9, 7, 3), (1, 45, 33, 31, 1), (1, 1, 257, 255, 1), (1, 3, 201, 199, 1), (2, 132, 5, 5, 2), (3, 30, 7, 5, 5),
                                                                     (2, 54, 9, 9, 3), (3, 1, 31, 37, 1), (1, 33, 40, 27, 1), (2, 28, 45, 41, 14)])
@pytest.mark.parametrize("kind", [None, "relu", "silu"])
def test_more_shapes_of_group_norm(hip, images, channels, height, width, groups, kind):
    base.test_group_norm(hip, images, channels, height, width, groups, kind)


@pytest.mark.parametrize("channels, pixels, groups", [(8, 100, 4), (6, 49, 6), (64, 1500, 4), (128, 16, 1), (30, 333, 2), (99, 63, 3), (6, 40000, 2), (33, 1300, 1), (24, 12000, 3),
                                                      (4, 2500, 4), (40, 4000, 40), (2, 60000, 1)])
def test_constant_groups_are_their_bias(hip, channels, pixels, groups):
    """A group of equal numbers has their value as its mean, to the bit, whatever the value and however the group is read: what is left is the bias."""
    rng = np.random.default_rng([channels, pixels])
    values = np.array([1234.567, -0.1, 3.3e7, 1e4, 7.7e-5, -98765.4], np.float32)
    per = channels // groups
    x = np.repeat(np.resize(values, (2, groups))[:, :, None], per * pixels, 2).reshape(2, channels, pixels)
    b = rng.standard_normal(channels, dtype=np.float32)
    want = np.broadcast_to(b[None, :, None], x.shape)
    X = hip.array(x.reshape(2, channels, pixels, 1))
    hip.group_norm(X, X, groups, bias=hip.array(b))
    assert np.array_equal(X.numpy().reshape(x.shape), want), "maps"
    R = hip.array(x.transpose(0, 2, 1).reshape(-1, channels))
    hip.group_norm(R, R, groups, bias=hip.array(b), image_rows=pixels)
    assert np.array_equal(R.numpy().reshape(2, pixels, channels).transpose(0, 2, 1), want), "rows"


def test_gate_where_its_exponential_passes_the_largest_number(hip):
    """silu from -80 to -300: its size falls from 1e-33 below the smallest normal number; off by 2^-119 at most there, not by a share of itself."""
    from eddl_amd.state_space import StateBatch
    v = np.concatenate([np.linspace(-89, -80, 4000), np.linspace(-300, -89, 1000)]).astype(np.float32)
    X, none, A = hip.full((1, len(v)), 1.0), hip.full((1, 1), 0.0), hip.full((len(v), 1), 0.0)
    Y = hip.empty(X.shape)
    hip.selective_scan(X, X, A, none, none, Y, StateBatch(hip.array(np.array([0, 1]), "int32"), 1), skip=hip.full((len(v),), 1.0), gate=hip.array(v[None]), softplus=False)
    x = v.astype(np.float64)
    want = x * np.exp(x) / (1 + np.exp(x))
    assert np.all(np.abs(Y.numpy()[0] - want) <= 11 * EPS * np.abs(want) + 2.0 ** -119)


@pytest.mark.parametrize("per", [1, 2, 3, 4, 7, 8, 9, 13, 14, 15, 16, 17, 19, 27, 32, 33, 62, 96, 124, 130])
def test_which_norms_take_the_workspace(hip, per):
    """Groups of more than 32768 numbers of maps, of about 32000 of rows, groups side by side of fewer than 16 channels from 704 rows an image on: what the header says."""
    def taken(rows, groups, tokens):
        X = hip.full((rows, groups * per) if tokens else (1, groups * per, rows, 1), 1.0)
        hip.workspace_trim()
        hip.group_norm(X, X, groups)
        return hip.workspace_bytes() > 0

    assert not taken(32768 // per, 2, False) and taken(32768 // per + 1, 2, False)
    assert not taken(31968 // per, 1, True) and taken(32768 // per + 1, 1, True)
    if per < 16:
        assert not taken(704, 40, True) and taken(1057, 40, True)
    else:
        assert not taken(31968 // per, 2, True) and taken(32768 // per + 1, 2, True)


@pytest.mark.parametrize("pixels", [50, 30000])
def test_large_numbers_of_small_spread(hip, pixels):
    """Numbers about 3e20, 1e17 apart: a mean whose square is beyond the largest number, differences whose squares are not.  And equal ones of 1e20."""
    rng = np.random.default_rng(pixels)
    x = (3e20 + 1e17 * rng.standard_normal((2, 4, pixels))).astype(np.float32)
    x[1, 2:] = 1e20
    b = rng.standard_normal(4, dtype=np.float32)
    want, err = base.group_norm(x, 2, None, b, 1e-5, None, None, None)
    err[1, 2:] = 0
    want[1, 2:] = b[2:, None]
    X = hip.array(x.reshape(2, 4, pixels, 1))
    hip.group_norm(X, X, 2, bias=hip.array(b))
    _check(X.numpy().reshape(x.shape), want, err, "maps")
    R = hip.array(x.transpose(0, 2, 1).reshape(-1, 4))
    hip.group_norm(R, R, 2, bias=hip.array(b), image_rows=pixels)
    _check(R.numpy().reshape(2, pixels, 4).transpose(0, 2, 1), want, err, "rows")


@pytest.mark.parametrize("pixels", [50, 30000])
def test_squares_beyond_the_largest_number(hip, pixels):
    """What the header says of numbers that fp32 sums do not hold: squares beyond it leave the bias, sums beyond it NaN; the other group is as it was."""
    rng = np.random.default_rng(pixels)
    x = rng.standard_normal((1, 4, pixels), dtype=np.float32)
    b = rng.standard_normal(4, dtype=np.float32)
    for scale, left in ((1e21, b), (2e38, np.nan * b)):
        big = x.copy()
        big[0, :2] = scale * (np.abs(x[0, :2]) / np.abs(x[0, :2]).max() if scale > 1e30 else x[0, :2])
        X, plain = hip.array(big.reshape(1, 4, pixels, 1)), hip.array(x.reshape(1, 4, pixels, 1))
        for t in (X, plain):
            hip.group_norm(t, t, 2, bias=hip.array(b))
        got = X.numpy()[0, :, :, 0]
        assert np.array_equal(got[:2], np.broadcast_to(left[:2, None], (2, pixels)), equal_nan=True)
        assert np.array_equal(got[2:], plain.numpy()[0, 2:, :, 0])
