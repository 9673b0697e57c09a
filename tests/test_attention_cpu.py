"""Refusals of the attention operators, which need no device, and their host-side objects."""
import ctypes

import numpy as np
import pytest

P = 4096  # (a pointer that no refused call reads)


@pytest.fixture(scope="module")
def lib():
    from eddl_amd import _lib
    return _lib.load()


def _refused(lib, rc, text):
    assert rc == -1 and text in lib.eddlhip_last_error().decode(), (rc, lib.eddlhip_last_error())


ATTEND = dict(dev=0, Q=P, ldq=256, O=2 * P, ldo=256, rows=4, k=P, v=P, kind=0, pages=9, page=16, q_heads=4, kv_heads=2, dim=64, table=P, width=3, offsets=P, lengths=P, seqs=2,
              max_new=2, max_length=40, scale=0.1, causal=1, window=0)


@pytest.mark.parametrize("change, text", [
    (dict(kind=2), "unknown cache type"), (dict(dim=40), "multiple of 16"), (dict(dim=272), "multiple of 16"), (dict(dim=0), "multiple of 16"),
    (dict(q_heads=5), "do not share"), (dict(kv_heads=0), "do not share"), (dict(page=24), "power of two"), (dict(page=8), "power of two"), (dict(pages=0), "pool of 0"),
    (dict(width=0), "table of 0"), (dict(width=1 << 27), "table of 134217728"), (dict(rows=1 << 29), "out of range"), (dict(ldq=255), "do not hold"), (dict(ldo=100), "do not hold"), (dict(max_new=-1), "negative"), (dict(scale=float("nan")), "not finite"), (dict(scale=float("inf")), "not finite"), (dict(window=-1), "negative"),
    (dict(rows=-1), "-1 rows"), (dict(seqs=70000), "at most 65535"), (dict(Q=None), "NULL"), (dict(lengths=None), "NULL"), (dict(k=P + 8), "aligned"), (dict(O=P), "lies on"), (dict(O=P + 1024), "lies on"), (dict(O=P + 64, ldo=300), "lies on")])
def test_paged_attention_refusals(lib, change, text):
    _refused(lib, lib.eddlhip_paged_attention(*dict(ATTEND, **change).values()), text)


def _append(**change):
    axis, freq = np.zeros(32, np.int32), np.ones(32)
    a = dict(dev=0, Q=P, ldq=256, Qout=2 * P, ldo=256, K=P, ldk=128, V=P, ldv=128, rows=4, q_heads=4, kv_heads=2, dim=64, positions=P, rot=64, adjacent=0, axes=1,
             axis=ctypes.c_void_p(axis.ctypes.data), freq=ctypes.c_void_p(freq.ctypes.data), k=P, v=P, kind=0, pages=9, page=16, table=P, width=3, offsets=P, lengths=P, seqs=2,
             max_new=2)
    for key, v in change.items():
        if key == "third":
            axis[2] = v
        else:
            a[key] = v
    return list(a.values()), (axis, freq)


@pytest.mark.parametrize("change, text", [
    (dict(kind=-1), "unknown cache type"), (dict(dim=24), "multiple of 16"), (dict(page=48), "power of two"), (dict(rot=72), "rot_dim"), (dict(rot=12), "rot_dim"),
    (dict(rot=-8), "rot_dim"), (dict(third=1), "turns by axis 1 of 1"), (dict(third=-1), "turns by axis -1"), (dict(axes=0), "0 axes"), (dict(positions=None), "NULL positions"),
    (dict(Q=None), "come together"), (dict(ldk=100), "do not hold"), (dict(ldo=200), "do not hold"), (dict(V=None), "NULL"), (dict(v=P + 4), "aligned"),
    (dict(Qout=P, ldo=300, K=9 * P, V=10 * P), "in place"), (dict(Qout=P + 16, K=9 * P, V=10 * P), "lie on"), (dict(K=2 * P + 64), "lie on"), (dict(kv_heads=0), "key heads"), (dict(max_new=-2), "max_new -2")])
def test_paged_append_refusals(lib, change, text):
    args, keep = _append(**change)
    _refused(lib, lib.eddlhip_paged_append(*args), text)


@pytest.mark.parametrize("change, text", [
    (dict(dim=12), "multiple of 8"), (dict(rot=264, dim=512, ldx=4096, ldy=4096), "rot_dim"), (dict(heads=0), "0 heads"), (dict(ldx=100), "do not hold"), (dict(X=None), "NULL tensor"),
    (dict(Y=P, ldy=640), "in place"), (dict(Y=P + 32), "lies on"), (dict(rows=-3), "-3 rows"), (dict(axis=None), "NULL positions")])
def test_rotary_refusals(lib, change, text):
    axis, freq = np.zeros(256, np.int32), np.ones(256)
    a = dict(dev=0, X=P, ldx=512, Y=2 * P, ldy=512, rows=4, heads=8, dim=64, positions=P, rot=64, adjacent=0, axes=1, axis=ctypes.c_void_p(axis.ctypes.data),
             freq=ctypes.c_void_p(freq.ctypes.data))
    _refused(lib, lib.eddlhip_rotary_axes(*dict(a, **change).values()), text)


@pytest.mark.parametrize("change, text", [
    (dict(cols=0), "0 columns"), (dict(cols=32769, ldx=40000, ldr=40000, lds=40000, ldh=40000), "32769 columns"), (dict(post=3), "unknown norm 3"), (dict(pre=-1), "unknown norm -1"),
    (dict(group=0), "groups of 0"), (dict(gate=P, gate_groups=2), "gates of 2 groups for 3"), (dict(ldx=63), "shorter"), (dict(ldh=63), "shorter"), (dict(X=None), "NULL"),
    (dict(S=None, H=None, pre=0), "NULL"), (dict(H=None, pre=1), "no output"), (dict(H=None, pre=0, shift=P), "no output"), (dict(S=P, lds=80), "in place"),
    (dict(H=3 * P, ldh=80), "in place"), (dict(S=5 * P, H=5 * P), "share"), (dict(S=5 * P, H=5 * P + 64), "share"), (dict(S=P + 16), "part of an input"), (dict(H=3 * P - 256), "part of an input")])
def test_norm_residual_refusals(lib, change, text):
    a = dict(dev=0, X=P, ldx=64, R=3 * P, ldr=64, scale=1.0, S=5 * P, lds=64, H=7 * P, ldh=64, rows=9, cols=64, post=0, post_w=None, post_b=None, post_eps=0.0, gate=None, gate_groups=0,
             pre=2, pre_w=None, pre_b=None, pre_eps=1e-6, mod=None, shift=None, group=4)
    _refused(lib, lib.eddlhip_norm_residual(*dict(a, **change).values()), text)


def test_columns_of_one_tensor_do_not_overlap(lib):
    """Outputs beside the inputs in rows of the same distance pass that check (and are refused for what comes after it)."""
    _refused(lib, lib.eddlhip_paged_attention(*dict(ATTEND, ldq=512, ldo=512, O=P + 4 * 256, k=P + 8).values()), "aligned")
    _refused(lib, lib.eddlhip_paged_attention(*dict(ATTEND, ldq=511, ldo=511, O=P + 4 * 256, k=P + 8).values()), "lies on")


def test_empty_calls_need_no_device(lib):
    assert lib.eddlhip_paged_attention(*dict(ATTEND, rows=0).values()) == 0
    assert lib.eddlhip_paged_attention(*dict(ATTEND, seqs=0).values()) == 0
    args, keep = _append(rows=0)
    assert lib.eddlhip_paged_append(*args) == 0


class _Tensor:
    def __init__(self, shape, dtype="float32", ptr=P):
        self.shape, self.dtype, self.address = shape, dtype, ptr
        self.size = int(np.prod(shape))


def test_host_objects_refuse():
    from eddl_amd.attention import PagedBatch, PagedCache, RotaryPlan
    for bad in (dict(page_size=24), dict(page_size=8), dict(head_dim=40), dict(head_dim=512), dict(pages=0), dict(dtype="float16")):
        with pytest.raises(ValueError):
            PagedCache(None, **dict(dict(pages=4, page_size=16, kv_heads=2, head_dim=64), **bad), storage=(None, None))
    k, v = _Tensor((4, 2, 1, 8, 16, 8)), _Tensor((4, 2, 1, 2, 64, 8))
    assert PagedCache(None, 4, 16, 2, 64, storage=(k, v)).arguments == (P, P, 0, 4, 16)
    with pytest.raises(ValueError):
        PagedCache(None, 4, 16, 2, 64, "bfloat16", storage=(k, v))
    with pytest.raises(ValueError):
        PagedCache(None, 4, 16, 2, 64, storage=(v, k))
    i = lambda *s: _Tensor(s, "int32")
    assert PagedBatch(i(3, 5), i(4), i(3), 1, 80).arguments == (P, 5, P, P, 3)
    for bad in ((i(3, 5), i(3), i(3)), (i(3), i(4), i(3)), (i(3, 5), i(4), _Tensor((3,)))):
        with pytest.raises(ValueError):
            PagedBatch(*bad, 1, 80)
    for axis, freq, pairing in (([0, 0], [1.0], "halves"), ([0], [1.0], "other"), ([[0]], [[1.0]], "halves")):
        with pytest.raises(ValueError):
            RotaryPlan(64, axis, freq, pairing)


def test_sections_of_a_rotary_plan():
    from eddl_amd.attention import RotaryPlan
    p = RotaryPlan.sections(32, (2, 3, 3), theta=16.0)
    assert p.axis.tolist() == [0, 0, 1, 1, 1, 2, 2, 2] and p.rot_dim == 16 and p.axes == 3
    assert np.allclose(p.freq, 16.0 ** (-np.arange(8) / 8))
    p = RotaryPlan.sections(32, (2, 3, 3), theta=16.0, shared=False, interleaved=True)
    assert p.axis.tolist() == [0, 1, 2, 0, 1, 2, 1, 2]
    assert np.allclose(p.freq, [1, 1, 1, 16.0 ** -0.5, 16.0 ** (-1 / 3), 16.0 ** (-1 / 3), 16.0 ** (-2 / 3), 16.0 ** (-2 / 3)])


def test_wrapped_memory_is_contiguous():
    from eddl_amd.backend import Backend, Columns

    class Lent:
        def __init__(self, shape, typestr="<f4", strides=None):
            self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "strides": strides, "data": (P, False), "version": 2}

    hip = object.__new__(Backend)
    hip.lib, hip.dev = type("Lib", (), {"eddlhip_relu": None, "eddlhip_fill": None}), 0
    t = Backend.wrap(hip, Lent((3, 5)))
    assert (t.ptr, t.shape, t.dtype, t.nbytes) == (P, (3, 5), "float32", 60)
    assert Backend.wrap(hip, Lent((3, 1, 5), strides=(20, 999, 4))).size == 15
    assert Backend.wrap(hip, Lent((4,), "<i2"), dtype="bfloat16").nbytes == 8
    for bad in (Lent((3, 5), strides=(24, 4)), Lent((3,), "<f8"), Lent((3,), "<i2")):
        with pytest.raises(ValueError):
            Backend.wrap(hip, bad)
    c = t.columns(1, 4)
    assert isinstance(c, Columns) and (c.at, c.ld, c.shape) == (P + 4, 5, (3, 3)) and not hasattr(c, "ptr")
    typed = Backend.wrap(hip, Lent((6, 4), "<i4"))
    assert (typed.address, typed.dtype, typed.reshape((4, 6)).shape) == (P, "int32", (4, 6))
    for operator in (lambda: hip.relu(typed, typed), lambda: hip.fill_(typed, 0.0), lambda: typed.columns(0, 2), lambda: typed.ptr):
        with pytest.raises(TypeError):
            operator()
    for lo, hi in ((2, 2), (-1, 3), (0, 6)):
        with pytest.raises(ValueError):
            t.columns(lo, hi)


def test_reference_layout_is_a_permutation():
    from attention_ref import Pool, bf16_bits, bf16_value
    pool = Pool(np.random.default_rng(0), [1, 2], [40, 33], 2, 32, 16, "float32", spare=0)
    for name in ("k", "v"):
        seen = np.concatenate([pool.index(s, np.arange(48), name).reshape(-1) for s in range(2)])
        assert sorted(seen) == list(range(pool.pages * 16 * 2 * 32))
    x = np.array([1.0, 1.00390625, 1.01171875, -3.14159, np.inf], np.float32)
    assert bf16_value(bf16_bits(x)).tolist() == [1.0, 1.0, 1.015625, -3.140625, np.inf]


def test_paged_attention_layer_checks_its_parent():
    from eddl_amd import net as L
    from eddl_amd.attention import PagedCache
    cache = PagedCache(None, 4, 16, 2, 64, storage=(_Tensor((4, 2, 1, 8, 16, 8)), _Tensor((4, 2, 1, 2, 64, 8))))
    ok = L.PagedAttention(L.Input([7, 8 * 64], 3), 4, cache, None)
    assert ok.out_shape == [3, 7, 256]
    for shape, heads in (([7, 8 * 64], 5), ([7, 500], 4), ([8 * 64], 4), ([7, 7 * 64], 3)):
        with pytest.raises(RuntimeError):
            L.PagedAttention(L.Input(shape, 3), heads, cache, None)
    n = L.LayerNormalization(L.Input([7, 24], 3))
    assert sorted(n.params) == ["b", "w"] and n.params["w"].shape == (24,) and not L.RMSNormalization(n, affine=False).params
