"""Every kernel that the rules of the selective scan and the group norm choose between, against 64 bits."""
import numpy as np
import pytest

import test_gpu_state_space as base
from state_space_ref import selective_scan
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
