"""Host side of Context without a GPU: the stream is the library's, whoever set it."""
import ctypes as C

import turt_b200.runtime as rt


class FakeLibrary:
    """One context, its stream in a cell of its own."""

    def __init__(self):
        self.cell, self.gone = C.c_void_p(), False

    def turt_init(self, device, out):
        out._obj.value = 4096
        self.cell.value = 77
        return 0

    def turt_ctx_stream_cell(self, h):
        assert h.value == 4096 and not self.gone
        return C.addressof(self.cell)

    def turt_ctx_set_stream(self, h, stream):
        self.cell.value = stream
        return 0

    def turt_ctx_destroy(self, h):
        self.gone = True
        self.cell.value = 13  # the memory belongs to someone else now
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
    assert not rt.lib().turt_ctx_stream_cell(C.c_void_p())
