"""Host side of LogitRules without a GPU: what it hands to the library for given rules and histories."""
import ctypes as C

import numpy as np
import pytest

import turt_b200.generate as gen
from turt_b200._lib import TurtLogitRules


class FakeContext:
    """Device buffers as host arrays."""
    handle = None

    def __init__(self):
        self.mem, self.next = {}, 64

    def buffer(self, elems):
        p, self.next = self.next, self.next + 1000003
        self.mem[p] = None
        return p

    def upload(self, p, a):
        self.mem[p] = np.array(a)

    def free(self, p):
        del self.mem[p]

    def download(self, p, n):
        return np.arange(n, dtype=np.float32)


@pytest.fixture
def calls(monkeypatch):
    seen = []

    class Lib:
        @staticmethod
        def turt_logit_rules_apply(h, x, ld, out, old, rows, vocab, rules):
            seen.append((x, ld, rows, vocab, TurtLogitRules.from_buffer_copy(rules._obj)))
            return 0
    monkeypatch.setattr(gen, "lib", lambda: Lib)
    return seen


def test_arrays_of_a_batch(calls):
    ctx = FakeContext()
    allowed = lambda r, ids: None if r == 1 else np.arange(40) % 3 == len(ids) % 3  # noqa: E731
    rules = gen.LogitRules(ctx, 40, 3, repetition=[1.5, 1.0, 2.0], frequency=0.25, bias=[{7: 1.0, 3: -2.0}, None, {39: 4.0}],
                           allowed=allowed)
    assert rules.active
    out = rules.apply(12345, [[1, 2], [3], [4, 5, 6]], [[9], [], [8, 8]])
    assert out.shape == (3, 40)
    (x, ld, rows, vocab, r), = calls
    assert (x, ld, rows, vocab) == (12345, 40, 3, 40)
    at = lambda p: ctx.mem[p].tolist()  # noqa: E731
    assert at(r.tokens) == [1, 2, 9, 3, 4, 5, 6, 8, 8]
    assert at(r.token_start) == [0, 3, 4, 9] and at(r.generated_start) == [2, 4, 7]
    assert at(r.repetition) == [1.5, 1.0, 2.0] and at(r.frequency) == [0.25] * 3 and at(r.presence) == [0.0] * 3
    assert at(r.bias_ids) == [3, 7, 39] and at(r.bias) == [-2.0, 1.0, 4.0] and at(r.bias_start) == [0, 2, 2, 3]
    assert r.n_masks == 2 and at(r.mask_row) == [0, 0xFFFFFFFF, 1]
    words = ctx.mem[r.mask].reshape(2, 2)
    for m, n in zip(words, (3, 5)):
        bits = [(int(m[i // 32]) >> (i % 32)) & 1 for i in range(64)]
        assert bits == [int(i < 40 and i % 3 == n % 3) for i in range(64)]
    rules.close()
    assert not ctx.mem


def test_rules_left_out(calls):
    rules = gen.LogitRules(FakeContext(), 10)
    assert not rules.active
    rules.apply(1, [[1]], [[2]])
    r = calls[0][4]
    assert all(getattr(r, f) in (None, 0) for f, _ in TurtLogitRules._fields_)


def test_refusals():
    for kw in (dict(repetition=0.0), dict(repetition=[1.0, -1.0], rows=2), dict(bias=[{}], rows=2), dict(frequency=[1, 2, 3])):
        with pytest.raises(ValueError):
            gen.LogitRules(FakeContext(), 10, **kw)
    rules = gen.LogitRules(FakeContext(), 10, allowed=lambda r, ids: np.ones(11, bool))
    with pytest.raises(ValueError):
        rules.apply(1, [[1]], [[2]])
    rules = gen.LogitRules(FakeContext(), 10, presence=1.0)
    with pytest.raises((ValueError, OverflowError)):
        rules.apply(1, [[-1]], [[2]])
