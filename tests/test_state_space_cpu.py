"""Refusals of the group norm and state space operators, which need no device, and their host-side objects."""
import numpy as np
import pytest

M = 1 << 20
P = [n * M for n in range(1, 40)]  # (pointers that no refused call reads)


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


def _check(outcome, text):
    assert outcome is None if text is None else outcome is not None and text in outcome, outcome


NORM = dict(dev=99, X=P[0], ldx=64, Y=P[1], ldy=64, images=3, channels=64, pixels=49, last=1, groups=8, w=P[2], b=P[3], eps=1e-5, mod=P[4], shift=P[5], activation=0)


@pytest.mark.parametrize("change, text", [
    (dict(), None), (dict(groups=7), "64 channels in 7 groups"), (dict(groups=0), "in 0 groups"), (dict(groups=-8), "groups"), (dict(groups=1, channels=4097, ldx=5000, ldy=5000), "of up to 4096"), (dict(channels=0), "0 channels"), (dict(pixels=0), "0 pixels"),
    (dict(images=-1), "-1 images"), (dict(images=1 << 16, pixels=1 << 16), "out of range"), (dict(activation=3), "unknown activation 3"), (dict(activation=-1), "unknown activation"),
    (dict(ldx=63), "shorter"), (dict(ldy=63), "shorter"), (dict(ldx=1, ldy=1, last=0), None), (dict(X=None), "NULL"), (dict(Y=None), "NULL"), (dict(Y=P[0]), None),
    (dict(Y=P[0], ldy=80), "in place"), (dict(Y=P[0] + 16), "part of the input"), (dict(Y=P[0] + 64 * 4, ldx=128, ldy=128), None), (dict(Y=P[0] + 64 * 4, last=0), "part of the input"),
    (dict(w=P[1]), "lies on a weight"), (dict(b=P[1] + 4 * 64 * 146), "lies on a weight"), (dict(mod=P[1] - 3 * 64 * 4 + 4), "lies on a weight"), (dict(mod=P[1] - 3 * 64 * 4), None),
    (dict(shift=P[1] + 4), "lies on a weight"), (dict(w=None, b=None, mod=None, shift=None), None)])
def test_group_norm_refusals(lib, change, text):
    _check(_outcome(lib, lib.eddlhip_group_norm(*dict(NORM, **change).values())), text)


CONV = dict(dev=99, X=P[0], ldx=64, W=P[1], bias=P[2], Y=P[3], ldy=64, rows=20, channels=64, width=4, activation=2, reverse=0, states=P[4], pool=5, offsets=P[5], lengths=P[6], slots=P[7],
            out_slots=P[8], seqs=3, max_new=9)


@pytest.mark.parametrize("change, text", [
    (dict(), None), (dict(width=1), "a width of 1"), (dict(width=9), "a width of 9"), (dict(channels=0), "0 channels"), (dict(activation=4), "unknown activation"), (dict(ldx=60), "shorter"),
    (dict(ldy=60), "shorter"), (dict(rows=-1), "-1 rows"), (dict(seqs=65536), "at most 65535"), (dict(seqs=-1), "-1 sequences"), (dict(max_new=-1), "max_new -1"), (dict(pool=0), "a pool of 0"),
    (dict(states=None), "at NULL"), (dict(states=None, pool=0), None), (dict(states=None, pool=0, lengths=None, slots=None, out_slots=None), None), (dict(offsets=None), "NULL offsets"),
    (dict(lengths=None), "NULL"), (dict(out_slots=None), "NULL"), (dict(X=None), "NULL tensor"), (dict(W=None), "NULL tensor"), (dict(bias=None), None), (dict(Y=P[0]), "lies on the input"),
    (dict(Y=P[0] + 256, ldx=128, ldy=128), None), (dict(Y=P[4] + 5 * 3 * 64 * 4 - 4), "lies on the states"), (dict(Y=P[4] + 5 * 3 * 64 * 4), None), (dict(W=P[3] + 16), "lies on the states"),
    (dict(lengths=P[3]), "lies on the states"), (dict(states=P[0] + 16), "states lie on the input"), (dict(states=P[1]), "states lie on the weights"), (dict(states=P[8] - 64), "states lie on the weights"),
    (dict(rows=0, X=None), "ok"), (dict(seqs=0, offsets=None), "ok")])
def test_causal_conv_refusals(lib, change, text):
    rc = lib.eddlhip_causal_conv(*dict(CONV, **change).values())
    if text == "ok":
        assert rc == 0
    else:
        _check(_outcome(lib, rc), text)


SCAN = dict(dev=99, X=P[0], ldx=64, dt=P[1], lddt=64, A=P[2], B=P[3], ldb=32, C=P[4], ldc=32, skip=P[5], gate=P[6], ldg=64, dt_bias=P[7], Y=P[8], ldy=64, rows=20, channels=64, n=16, groups=2,
            softplus=1, reverse=0, states=P[9], pool=5, offsets=P[10], lengths=P[11], slots=P[12], out_slots=P[13], seqs=3, max_new=9)


@pytest.mark.parametrize("change, text", [
    (dict(), None), (dict(n=0), "of 0 states"), (dict(n=65), "of 65 states"), (dict(groups=3), "in 3 groups"), (dict(groups=0), "in 0 groups"), (dict(channels=-2), "-2 channels"),
    (dict(ldx=63), "shorter than 64"), (dict(lddt=63), "shorter than 64"), (dict(ldg=63), "shorter than 64"), (dict(ldy=0), "shorter than 64"), (dict(ldg=0, gate=None), None),
    (dict(ldb=31), "vectors of 16"), (dict(ldc=31), "vectors of 16"), (dict(rows=-1), "-1 rows"), (dict(seqs=70000), "at most 65535"), (dict(pool=-1), "a pool of -1"), (dict(states=None), "at NULL"),
    (dict(states=None, pool=0), None), (dict(slots=None), "NULL"), (dict(offsets=None), "NULL"), (dict(A=None), "NULL tensor"), (dict(dt=None), "NULL tensor"), (dict(skip=None, dt_bias=None), None),
    *[({"Y": P[k]}, "lies on an input") for k in (0, 1, 3, 4, 6)], *[({"Y": P[k]}, "lies on the states") for k in (2, 5, 7, 9, 10, 11, 12, 13)],
    *[({"states": P[k] + 4}, "states lie on an input") for k in (0, 1, 3, 4, 6)], *[({"states": P[k] - 4 * 5 * 64 * 16 + 4}, "states lie on the weights") for k in (2, 5, 7, 10, 11, 12, 13)],
    (dict(Y=P[0] + 256, ldx=128, ldy=128), None), (dict(rows=0, Y=None), "ok"), (dict(seqs=0), "ok")])
def test_selective_scan_refusals(lib, change, text):
    rc = lib.eddlhip_selective_scan(*dict(SCAN, **change).values())
    if text == "ok":
        assert rc == 0
    else:
        _check(_outcome(lib, rc), text)


class _Tensor:
    def __init__(self, shape, dtype="float32", ptr=M):
        self.shape, self.dtype, self.address, self.ptr = tuple(shape), dtype, ptr, ptr
        self.size = int(np.prod(shape))


def _int(*shape):
    return _Tensor(shape, "int32")


def test_batches():
    from eddl_amd.state_space import StateBatch
    assert StateBatch(_int(4), 9).arguments == (M, None, None, None, 3, 9)
    assert StateBatch(_int(4), 9, _int(3), _int(3)).arguments == (M, M, M, M, 3, 9)
    for bad in ((_int(4), 9, _int(4), _int(3)), (_int(4), 9, _int(3), None), (_int(4), 9, None, _int(3)), (_Tensor((4,)), 9), (_int(4, 1), 9), (_int(0), 9),
                (_int(4), 9, _int(3), _int(3), _int(2)), (_int(4), 9, _int(3), _Tensor((3,)))):
        with pytest.raises(ValueError):
            StateBatch(*bad)


@pytest.fixture()
def hip():
    """A backend without a device: calls that pass the checks of shapes end at the library's, with device 99."""
    from eddl_amd import _lib
    from eddl_amd.backend import Backend
    h = object.__new__(Backend)
    h.lib, h.dev = _lib.load(), 99
    return h


def _refused(call):
    with pytest.raises(ValueError):
        call()


def _passes(call):
    from eddl_amd.backend import EddlHipError
    with pytest.raises(EddlHipError, match="device index 99"):
        call()


def test_shapes_of_group_norm(hip):
    t = lambda k, *shape: _Tensor(shape, ptr=P[k])
    _passes(lambda: hip.group_norm(t(0, 2, 8, 3, 3), t(1, 2, 8, 3, 3), 4))
    _passes(lambda: hip.group_norm(t(0, 18, 8), t(1, 18, 8), 4, image_rows=9, mod=t(2, 2, 8)))
    _passes(lambda: hip.group_norm(t(0, 18, 8), t(1, 18, 8), 4, weight=t(2, 8), activation="silu"))
    for bad in (lambda: hip.group_norm(t(0, 2, 8, 3, 3), t(1, 2, 8, 3, 2), 4), lambda: hip.group_norm(t(0, 2, 8, 3, 3), t(1, 2, 8, 3, 3), 4, image_rows=9),
                lambda: hip.group_norm(t(0, 2, 8, 3), t(1, 2, 8, 3), 4), lambda: hip.group_norm(t(0, 18, 8), t(1, 18, 8), 4, image_rows=7), lambda: hip.group_norm(t(0, 18, 8), t(1, 18, 9), 4),
                lambda: hip.group_norm(t(0, 18, 8), t(1, 18, 8), 4, image_rows=0), lambda: hip.group_norm(t(0, 18, 8), t(1, 18, 8), 4, weight=t(2, 9)),
                lambda: hip.group_norm(t(0, 18, 8), t(1, 18, 8), 4, image_rows=9, mod=t(2, 3, 8)), lambda: hip.group_norm(t(0, 18, 8), t(1, 18, 8), 4, activation="gelu"),
                lambda: hip.group_norm(_Tensor((18, 8), "int32"), t(1, 18, 8), 4), lambda: hip.group_norm(t(0, 18, 8), t(1, 18, 8), 4, image_rows=-3)):
        _refused(bad)


def test_shapes_of_causal_conv(hip):
    from eddl_amd.state_space import StateBatch
    t = lambda k, *shape: _Tensor(shape, ptr=P[k])
    plain, kept = StateBatch(_Tensor((4,), "int32", P[20]), 9), StateBatch(*(_Tensor((4,), "int32", P[20]), 9, _Tensor((3,), "int32", P[21]), _Tensor((3,), "int32", P[22])))
    ok = dict(X=t(0, 20, 8), W=t(1, 8, 4), bias=t(2, 8), Y=t(3, 20, 8), batch=plain)
    _passes(lambda: hip.causal_conv(**ok))
    _passes(lambda: hip.causal_conv(**dict(ok, batch=kept, states=t(4, 5, 3, 8), activation="relu", reverse=True)))
    for bad in (dict(Y=t(3, 20, 9)), dict(W=t(1, 9, 4)), dict(W=t(1, 8, 1, 4)), dict(bias=t(2, 7)), dict(batch=kept, states=t(4, 5, 4, 8)), dict(states=t(4, 5, 3, 8)),
                dict(batch=kept, states=t(4, 3, 8)), dict(activation="tanh"), dict(X=t(0, 160))):
        _refused(lambda: hip.causal_conv(**dict(ok, **bad)))


def test_shapes_of_selective_scan(hip):
    from eddl_amd.state_space import StateBatch
    t = lambda k, *shape: _Tensor(shape, ptr=P[k])
    kept = StateBatch(*(_Tensor((4,), "int32", P[20]), 9, _Tensor((3,), "int32", P[21]), _Tensor((3,), "int32", P[22])))
    ok = dict(X=t(0, 20, 8), dt=t(1, 20, 8), A=t(2, 8, 5), B=t(3, 20, 10), C=t(4, 20, 10), Y=t(5, 20, 8), batch=kept)
    _passes(lambda: hip.selective_scan(**ok))
    _passes(lambda: hip.selective_scan(**dict(ok, states=t(6, 5, 8, 5), skip=t(7, 8), gate=t(8, 20, 8), dt_bias=t(9, 8), softplus=False)))
    for bad in (dict(dt=t(1, 20, 9)), dict(dt=t(1, 19, 8)), dict(A=t(2, 9, 5)), dict(A=t(2, 40)), dict(B=t(3, 20, 11)), dict(B=t(3, 20, 11), C=t(4, 20, 11)), dict(B=t(3, 19, 10), C=t(4, 19, 10)),
                dict(gate=t(8, 20, 4)), dict(skip=t(7, 9)), dict(dt_bias=t(7, 9)), dict(states=t(6, 5, 5, 8)), dict(Y=t(5, 21, 8)), dict(A=_Tensor((8, 5), "int32")), dict(A=t(2, 8, 0))):
        _refused(lambda: hip.selective_scan(**dict(ok, **bad)))


def test_layers_check_their_parents():
    from eddl_amd import net as L
    x, t = L.Input([8, 5, 7], 3), L.Input([9, 24], 3)
    g = L.GroupNormalization(x, 4)
    assert g.out_shape == [3, 8, 5, 7] and g.params["w"].shape == (8,) and not L.GroupNormalization(t, 8, affine=False).params
    assert L.GroupNormalization(t, 8, activation="silu").params["b"].shape == (24,)
    for parent, groups, activation in ((x, 3, None), (t, 5, None), (x, 0, None), (x, 4, "gelu"), (L.Input([24], 3), 4, None)):
        with pytest.raises(RuntimeError):
            L.GroupNormalization(parent, groups, activation=activation)
    c = L.CausalConvolution(t, 4, channels=16)
    assert c.out_shape == [3, 9, 16] and c.params["W"].shape == (16, 4) and "bias" not in L.CausalConvolution(t, 2, use_bias=False).params
    for parent, width, channels in ((t, 1, None), (t, 9, None), (t, 4, 25), (t, 4, 0), (x, 4, None)):
        with pytest.raises(RuntimeError):
            L.CausalConvolution(parent, width, channels)
    with pytest.raises(RuntimeError):
        L.CausalConvolution(t, 4, states=_Tensor((3, 3, 24)))
    d, v, z = (L.Dense(c, n) for n in (16, 2 * 2 * 5 + 3, 16))
    y = L.SelectiveScan(c, d, v, 5, groups=2, gate=z)
    assert y.out_shape == [3, 9, 16] and y.params["A"].shape == (16, 5) and list(y.params) == ["A", "skip", "dt_bias"] and len(y.parents) == 4
    assert y.params["A"][3].tolist() == [-1, -2, -3, -4, -5]
    for bad in (dict(state=6), dict(groups=3), dict(dt=v), dict(gate=L.Dense(c, 15)), dict(state=0), dict(vectors=L.Input([8, 40], 3)), dict(parent=t), dict(state=65)):
        with pytest.raises(RuntimeError):
            L.SelectiveScan(**dict(dict(parent=c, dt=d, vectors=v, state=5, groups=2, gate=z), **bad))
    with pytest.raises(RuntimeError):
        L.SelectiveScan(c, d, v, 5, states=_Tensor((3, 16, 5)))


def test_layer_refuses_an_unknown_activation():
    from eddl_amd import net as L
    with pytest.raises(RuntimeError):
        L.CausalConvolution(L.Input([9, 24], 3), 4, activation="gelu")
