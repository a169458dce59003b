"""Host side of PagedDecoder without a GPU: an engine that only books its buffers."""
from types import SimpleNamespace

import pytest

from turt_b200._lib import ERR_CUDA, TurtError
from turt_b200.generate import PagedDecoder


class BookedEngine:
    """Every op is recorded and does nothing; a freed buffer is held until reclaim()."""

    def __init__(self):
        self.live, self.pending, self.next, self.peak, self.calls, self.uploads = {}, [], 64, 0, [], {}
        self.ctx = SimpleNamespace(upload=self._upload)

    def _upload(self, p, a):
        self.uploads[p] = a.copy()

    def buffer(self, elems):
        p, self.next = self.next, self.next + (1 << 40)
        self.live[p] = elems
        self.peak = max(self.peak, sum(self.live.values()))
        return p

    def indexBuffer(self, a):
        p = self.buffer(a.size)
        self._upload(p, a)
        return p

    def free(self, p):
        self.pending.append(p)

    def reclaim(self):
        for p in self.pending:
            del self.live[p]
        self.pending = []

    def pagedAttentionWorkspace(self, kv, heads):
        return 4096

    def __getattr__(self, name):
        return lambda *a, **kw: self.calls.append((name, a, kw))


def booked_gpt(layers, arch="modern", E=8, H=2, block=256):
    t = lambda: SimpleNamespace(buffer=1)  # noqa: E731
    names = ("ln1g", "ln1b", "qW", "qb", "kW", "kb", "vW", "vb", "projW", "projb", "ln2g", "ln2b", "gateW", "upW", "downW", "fcW",
             "fcb", "mpW", "mpb")
    return SimpleNamespace(fused=False, engine=BookedEngine(), modern=arch == "modern", hidden=4 * E, headScale=0.5, wte=t(),
                           wpe=None if arch == "modern" else t(), lnfg=t(), lnfb=t(), blocks=[{n: t() for n in names}] * layers,
                           config=dict(nEmbd=E, nHead=H, vocabSize=11, nLayer=layers, blockSize=block))


def prefill_peak(layers, prompts, arch="modern"):
    g = booked_gpt(layers, arch)
    dec = PagedDecoder(g, [len(p) + 4 for p in prompts])
    held = sum(g.engine.live.values())
    dec.prefill(prompts)
    assert sum(g.engine.live.values()) == held  # a forward leaves nothing behind
    dec.step([1] * len(prompts))
    assert sum(g.engine.live.values()) == held
    peak = g.engine.peak - held
    dec.close()
    assert not g.engine.live
    return peak


@pytest.mark.parametrize("arch", ["modern", "gpt2"])
def test_prefill_memory_does_not_grow_with_the_layers(arch):
    prompts = [[1] * 200, [2] * 7, [3] * 90]
    assert prefill_peak(12, prompts, arch) == prefill_peak(1, prompts, arch)


def test_prefill_memory_of_many_prompts():
    """One matrix of scores serves all prompts: what else there is grows with the rows (16 values of width E or hidden a
    row, at most, and a few indices)."""
    one, many = prefill_peak(2, [[1] * 200]), prefill_peak(2, [[1] * 200] * 16)
    assert one >= 2 * 200 * 200
    assert many - one <= 15 * 200 * 16 * 4 * 8 and many < one + 2 * 200 * 200 * 15 / 2


def test_a_forward_that_fails_keeps_no_buffer():
    """The next forward asks for its own sizes."""
    g = booked_gpt(2)
    dec = PagedDecoder(g, [40, 40])
    held = set(g.engine.live)
    g.engine.pagedAttention = lambda *a, **kw: 1 // 0
    dec.prefill([[1] * 3, [2]])
    with pytest.raises(ZeroDivisionError):
        dec.step([1, 1])
    g.engine.pagedAttention = lambda *a, **kw: None
    g.engine.reclaim()
    assert set(g.engine.live) == held
    g.engine.peak = 0
    dec.prefill([[1] * 30, [2] * 20])
    assert g.engine.peak - sum(g.engine.live.values()) >= 2 * 30 * 30  # scores of 30 rows


def test_no_position_beyond_the_pages():
    """A step or prompt that a sequence has no pages for is refused before anything runs: it would go to another
    sequence's page.  What its last page has room for is taken."""
    g = booked_gpt(2)
    dec = PagedDecoder(g, [18, 40], page_size=8)
    # table entries behind a sequence's pages name no page
    table = g.engine.uploads[dec.table].view("int32").reshape(2, 5)
    assert table.tolist() == [[0, 1, 2, -1, -1], [3, 4, 5, 6, 7]]
    with pytest.raises(ValueError, match="25 positions, its pages hold 24"):
        dec.prefill([[1] * 25, [2]])
    for bad in ([[1]], [[1], []], [[1], [2], [3]]):
        with pytest.raises(ValueError):
            dec.prefill(bad)
    dec.prefill([[1] * 23, [2]])
    dec.step([1, 1])
    n = len(g.engine.calls)
    with pytest.raises(ValueError, match="25 positions, its pages hold 24"):
        dec.step([1, 1])
    with pytest.raises(ValueError):
        dec.step([1])
    assert len(g.engine.calls) == n and dec.lens.tolist() == [24, 2]
    dec.step([None, 1])
    assert dec.lens.tolist() == [24, 3]


def test_a_step_that_fails_leaves_the_lengths():
    g = booked_gpt(1)
    dec = PagedDecoder(g, [18, 40])
    dec.prefill([[1] * 3, [2]])
    g.engine.pagedAttention = lambda *a, **kw: 1 // 0
    with pytest.raises(ZeroDivisionError):
        dec.step([None, 1])
    assert dec.lens.tolist() == [3, 1]


@pytest.mark.parametrize("after", range(9))
def test_a_reservation_that_fails_keeps_nothing(after):
    """Memory that runs out at any of the buffers: those taken before it are given back, and a smaller batch fits."""
    g = booked_gpt(3)
    e, left = g.engine, [after]
    take = e.buffer

    def buffer(n):
        if left[0] == 0:
            raise TurtError(ERR_CUDA, "out of memory")
        left[0] -= 1
        return take(n)
    e.buffer = buffer
    with pytest.raises(TurtError, match="out of memory"):
        PagedDecoder(g, [18, 40])
    assert not e.live
    left[0] = 100
    PagedDecoder(g, [18]).close()
    assert not e.live


def test_closing_twice_frees_once():
    g = booked_gpt(1)
    dec = PagedDecoder(g, [18])
    dec.close()
    dec.close()
    assert not g.engine.live
