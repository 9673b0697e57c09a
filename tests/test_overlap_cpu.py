"""Outputs of the attention operators on what the same call reads: refused before a device is asked for."""
import ctypes

import numpy as np
import pytest

M = 1 << 20
FAR = 1 << 40


@pytest.fixture(scope="module")
def lib():
    from eddl_amd import _lib
    return _lib.load()


def _outcome(lib, rc):
    """The refusal's text; None where the call got as far as asking for device 99, which does not exist."""
    text = lib.eddlhip_last_error().decode()
    assert rc in (-1, -3), (rc, text)
    assert (rc == -3) == ("device index 99" in text), (rc, text)
    return text if rc == -1 else None


def _check(outcome, refused, text):
    assert (outcome is not None and text in outcome) if refused else outcome is None, outcome


@pytest.mark.parametrize("O, ldo, k, v, refused", [
    (FAR, 256, M, 2 * M, False), (M, 256, M, FAR, True), (M + 9 * 16 * 2 * 64 * 4 - 4, 256, M, FAR, True), (M + 9 * 16 * 2 * 64 * 4, 256, M, FAR, False),
    (FAR, 256, M, FAR + 4 * 256 * 4 - 16, True), (FAR, 256, M, FAR + 4 * 256 * 4, False), (FAR, 256, FAR - 9 * 16 * 2 * 64 * 4 + 16, M, True)])
def test_attention(lib, O, ldo, k, v, refused):
    rc = lib.eddlhip_paged_attention(99, 8 * FAR, 256, O, ldo, 4, k, v, 0, 9, 16, 4, 2, 64, M, 3, M, M, 2, 2, 40, 0.1, 1, 0)
    _check(_outcome(lib, rc), refused, "shares memory with the cache")


@pytest.mark.parametrize("change, text", [
    (dict(), None), (dict(K=M), "with the cache"), (dict(V=2 * M + 16), "with the cache"), (dict(Q=M, Qout=M), "with the cache"), (dict(Qout=2 * M), "with the cache"),
    (dict(positions=6 * FAR + 4 * 255), "on the positions"), (dict(positions=6 * FAR + 4 * 256, ldo=256 + 4, rows=1), None), (dict(positions=6 * FAR, rot=0), None)])
def test_append(lib, change, text):
    axis, freq = np.zeros(32, np.int32), np.ones(32)
    a = dict(dict(Q=5 * FAR, Qout=6 * FAR, ldo=256, K=7 * FAR, V=8 * FAR, rows=4, positions=9 * FAR, rot=64), **change)
    rc = lib.eddlhip_paged_append(99, a["Q"], 256, a["Qout"], a["ldo"], a["K"], 128, a["V"], 128, a["rows"], 4, 2, 64, a["positions"], a["rot"], 0, 1,
                                  ctypes.c_void_p(axis.ctypes.data), ctypes.c_void_p(freq.ctypes.data), M, 2 * M, 1, 9, 16, M, 3, M, M, 2, 2)
    _check(_outcome(lib, rc), text is not None, text)


@pytest.mark.parametrize("Y, ldy, positions, refused", [
    (FAR, 512, 9 * FAR, False), (FAR, 512, FAR, True), (FAR, 512, FAR - 4, True), (FAR, 512, FAR - 8 * 4, False), (FAR, 512, FAR + 4 * 512 * 4, False), (FAR, 520, FAR + 4 * 512, False),
    (FAR, 520, FAR + 4 * 513, True), (FAR, 516, FAR + 4 * 512, True)])
def test_rotary(lib, Y, ldy, positions, refused):
    """Eight positions beside the output, on it, and in the gap between two of its rows."""
    axis, freq = np.zeros(32, np.int32), np.ones(32)
    rc = lib.eddlhip_rotary_axes(99, 5 * FAR, 512, Y, ldy, 4, 8, 64, positions, 64, 0, 2, ctypes.c_void_p(axis.ctypes.data), ctypes.c_void_p(freq.ctypes.data))
    _check(_outcome(lib, rc), refused, "on the positions")


@pytest.mark.parametrize("name", ["post_w", "post_b", "gate", "pre_w", "pre_b", "mod", "shift"])
@pytest.mark.parametrize("out", ["S", "H"])
def test_norm(lib, name, out):
    where = dict(S=5 * FAR, H=6 * FAR)
    for at, refused in ((where[out], True), (where[out] + 4 * (9 * 64 - 1), True), (where[out] + 4 * 9 * 64, False), (9 * FAR, False)):
        a = dict(dict(post_w=None, post_b=None, gate=None, pre_w=None, pre_b=None, mod=None, shift=None), **{name: at})
        rc = lib.eddlhip_norm_residual(99, FAR, 64, 3 * FAR, 64, 1.0, where["S"], 64, where["H"], 64, 9, 64, 2, a["post_w"], a["post_b"], 1e-6, a["gate"], 3,
                                       2, a["pre_w"], a["pre_b"], 1e-6, a["mod"], a["shift"], 4)
        _check(_outcome(lib, rc), refused, "lies on a weight")
