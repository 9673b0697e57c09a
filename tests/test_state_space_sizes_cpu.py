"""Sizes beyond 32 bits are refused by the group norm and state space operators, whose library counts in ints; states by layers whose batch has no place for them."""
import pytest

from test_state_space_cpu import P, _Tensor, _passes, _refused, hip  # noqa: F401

BIG = 1 << 32


def _t(k, *shape):
    return _Tensor(shape, ptr=P[k])


def test_group_norm_of_more_pixels_images_or_rows_than_an_int_counts(hip):  # noqa: F811
    _passes(lambda: hip.group_norm(_t(0, 2, 8, 30, 30), _t(1, 2, 8, 30, 30), 4))
    far = lambda *shape: (_Tensor(shape, ptr=P[0]), _Tensor(shape, ptr=P[0]))
    for shape in ((1, 1, 65536, 65537), (BIG + 1, 1, 1, 1), (1, BIG + 2, 1, 1), (BIG + 9, 1), (9, BIG + 1)):
        _refused(lambda: hip.group_norm(*far(*shape), 1))
    _refused(lambda: hip.group_norm(*far(2 * (BIG + 9), 1), 1, image_rows=BIG + 9))
    _refused(lambda: hip.group_norm(*far(BIG + 9, 1), 1, image_rows=1))
    for groups in (BIG + 4, -BIG + 4):
        _refused(lambda: hip.group_norm(_t(0, 2, 8, 30, 30), _t(1, 2, 8, 30, 30), groups))


def test_rows_slots_and_bounds_of_a_batch(hip):  # noqa: F811
    from eddl_amd.state_space import StateBatch
    batch = lambda most: StateBatch(_Tensor((4,), "int32", P[30]), most, _Tensor((3,), "int32", P[31]), _Tensor((3,), "int32", P[32]))
    conv = lambda rows=20, channels=8, most=9, slots=5: hip.causal_conv(_t(0, rows, channels), _t(1, channels, 4), None, _Tensor((rows, channels), ptr=1 << 50), batch(most),
                                                                         states=_Tensor((slots, 3, channels), ptr=1 << 60))
    scan = lambda rows=20, channels=8, most=9, slots=5, n=4: hip.selective_scan(_t(0, rows, channels), _t(1, rows, channels), _t(2, channels, n), _t(3, rows, n), _t(4, rows, n),
                                                                              _Tensor((rows, channels), ptr=1 << 50), batch(most), states=_Tensor((slots, channels, n), ptr=1 << 60))
    for call in (conv, scan):
        _passes(call)
        for most in ((1 << 31) - 1, 1 << 31, BIG, BIG + 9):  # (a bound however high)
            _passes(lambda: call(most=most))
        for bad in (dict(rows=BIG + 20), dict(slots=BIG + 5), dict(channels=BIG + 8)):
            _refused(lambda: call(**bad))
    _refused(lambda: scan(n=BIG + 4))
    for most in (-1, -BIG + 9):
        with pytest.raises(ValueError):
            batch(most)
    with pytest.raises(ValueError):
        StateBatch(_Tensor((BIG + 4,), "int32", P[30]), 9)


def test_layers_refuse_states_without_slots():
    from eddl_amd import net as L
    from eddl_amd.state_space import StateBatch
    x, bare = L.Input([9, 24], 3), StateBatch(_Tensor((4,), "int32", P[30]), 9)
    kept = StateBatch(_Tensor((4,), "int32", P[30]), 9, _Tensor((3,), "int32", P[31]), _Tensor((3,), "int32", P[32]))
    layers = (lambda batch: L.CausalConvolution(x, 4, batch=batch, states=_Tensor((5, 3, 24))), lambda batch: L.SelectiveScan(x, x, x, 5, batch=batch, states=_Tensor((5, 24, 5))))
    for layer in layers:
        assert layer(kept).attrs["states"] is not None
        with pytest.raises(RuntimeError, match="slots"):
            layer(bare)
