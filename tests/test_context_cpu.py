"""Host side of Context without a GPU: the stream is the library's, whoever set it."""
import ctypes as C

import turt_b200.runtime as rt


class FakeLibrary:
    """Contexts as entries of a dict, the stream of each in it."""

    def __init__(self):
        self.streams = {}

    def turt_init(self, device, out):
        out._obj.value = 4096
        self.streams[4096] = 77
        return 0

    def turt_ctx_stream(self, h):
        return self.streams.get(h.value)

    def turt_ctx_set_stream(self, h, stream):
        self.streams[h.value] = stream
        return 0

    def turt_ctx_destroy(self, h):
        del self.streams[h.value]
        return 0


def test_stream_is_the_librarys(monkeypatch):
    fake = FakeLibrary()
    monkeypatch.setattr(rt, "lib", lambda: fake)
    c = rt.Context(0)
    assert c.stream == 77
    c.set_stream(5)
    assert c.stream == 5
    fake.turt_ctx_set_stream(c.handle, 9)  # through the C ABI
    assert c.stream == 9
    fake.turt_ctx_set_stream(c.handle, None)
    assert c.stream == 0
    c.close()
    assert c.stream == 0


def test_stream_of_no_context():
    assert not rt.lib().turt_ctx_stream(C.c_void_p())
