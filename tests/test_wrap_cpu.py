"""Backend.wrap: what it refuses of another library's memory."""
import pytest

P = 4096  # (a pointer that nobody reads)


class Lent:
    def __init__(self, read_only=False, **more):
        self.__cuda_array_interface__ = dict({"shape": (3, 5), "typestr": "<f4", "strides": None, "data": (P, read_only), "version": 3}, **more)


@pytest.fixture
def hip():
    from eddl_amd.backend import Backend
    hip = object.__new__(Backend)
    hip.dev = 0
    return hip


def test_memory_that_may_not_be_written_or_is_being_written_is_refused(hip):
    assert hip.wrap(Lent()).ptr == P
    assert hip.wrap(Lent(stream=None, mask=None)).ptr == P
    for lent, text in ((Lent(read_only=True), "read-only"), (Lent(mask=Lent()), "masked"), (Lent(stream=0), "stream 0"), (Lent(stream=2), "stream 2"), (Lent(stream=12345), "stream 12345")):
        with pytest.raises(ValueError, match=text):
            hip.wrap(lent)


def test_memory_of_another_device_is_refused_and_the_null_stream_waited_for(hip, monkeypatch):
    from eddl_amd import _lib

    class Library:
        answer, waits, failure = -1, [], 0

        def hipStreamSynchronize(self, stream):
            self.waits.append(stream)
            return self.failure

        def eddlhip_pointer_device(self, ptr, device):
            assert ptr == P
            device._obj.value = self.answer
            return 0

    library = Library()
    monkeypatch.setattr(_lib, "load", lambda: library)
    for answer, dev, fine in ((-1, 0, True), (0, 0, True), (1, 0, False), (0, 1, False), (3, 3, True)):
        library.answer, hip.dev = answer, dev
        if fine:
            assert hip.wrap(Lent()).shape == (3, 5)
        else:
            with pytest.raises(ValueError, match="device %d, not on device %d" % (answer, dev)):
                hip.wrap(Lent())
    assert library.waits == []
    assert hip.wrap(Lent(stream=1)).ptr == P and library.waits == [None]  # (the null stream is waited for)
    library.failure = 1
    with pytest.raises(ValueError, match="stream 1"):
        hip.wrap(Lent(stream=1))


def test_host_numbers_that_a_type_does_not_hold_are_refused(hip, monkeypatch):
    """Nothing is cast into other numbers on its way to an int32 or bfloat16 tensor; float32 tensors take every number, as before."""
    import numpy as np
    from eddl_amd import backend
    sent = []
    hip.empty = lambda shape, dtype="float32": type("Tensor", (), {"copy_from": lambda self, host: sent.append((host.dtype, host.tolist()))})()
    for host, dtype in (([1, 2], "bfloat16"), (np.array([0.5, 1.5]), "bfloat16"), (np.array([0.5], np.float32), "bfloat16"), (np.array([1], np.int16), "bfloat16"),
                        (np.array([1.0]), "int32"), ([0.5], "int32"), (np.array([2 ** 31]), "int32"), (np.array([-2 ** 31 - 1]), "int32"), (np.array([2 ** 32], np.uint64), "int32")):
        with pytest.raises(ValueError):
            hip.array(host, dtype)
        tensor = object.__new__(backend.TypedTensor)
        tensor.dtype, tensor.size = dtype, 1
        with pytest.raises(ValueError):
            tensor.copy_from(host)
    assert sent == []
    hip.array(np.array([0x3F80, 0xFFFF], np.uint16), "bfloat16")
    hip.array([-2 ** 31, 2 ** 31 - 1], "int32")
    hip.array(np.zeros((2, 0)), "int32")
    hip.array(np.array([True, False]), "int32")
    hip.array([1, 2], "float32")
    hip.array(np.array([0.1]))
    assert sent == [(np.uint16, [0x3F80, 0xFFFF]), (np.int32, [-2 ** 31, 2 ** 31 - 1]), (np.int32, [[], []]), (np.int32, [1, 0]), (np.float32, [1.0, 2.0]),
                    (np.float32, [float(np.float32(0.1))])]


def test_the_library_is_set_up_once():
    from eddl_amd import _lib
    assert _lib.load() is _lib.load()
