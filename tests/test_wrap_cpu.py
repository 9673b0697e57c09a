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
