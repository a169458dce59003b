"""Host side of generate_batch without a GPU: which sequences it asks about, and what it hands to the rules."""
import numpy as np
import pytest

import turt_b200.generate as gen
from turt_b200._lib import TurtLogitRules
from test_generate_memory_cpu import DeferredContext
from test_paged_decoder_cpu import booked_gpt


@pytest.fixture
def rules(monkeypatch):
    seen = []

    class Lib:
        @staticmethod
        def turt_logit_rules_apply(h, x, ld, out, old, rows, vocab, r):
            seen.append(TurtLogitRules.from_buffer_copy(r._obj))
            return 0
    monkeypatch.setattr(gen, "lib", lambda: Lib)
    return seen


def test_stopped_sequences_are_left_alone(rules):
    g = booked_gpt(1)
    g.engine.ctx = DeferredContext()
    g.engine.ctx.upload = lambda p, a: None
    asked, made, stopped = [], [0, 0, 0], set()

    def allowed(row, ids):
        assert row not in stopped
        asked.append(row)
        return np.ones(11, bool)

    def on_token(i, token):
        assert i not in stopped
        made[i] += 1
        if made[i] == 2 + 2 * i:
            stopped.add(i)
            return False
    out = gen.generate_batch(g, [[1], [2, 3], [4]], 10, rngs=[lambda: 0.5] * 3, on_token=on_token, allowed=allowed)
    assert [len(s) for s in out] == [3, 6, 7] and made == [2, 4, 6]
    assert [asked.count(i) for i in range(3)] == made
    assert [r.n_masks for r in rules] == [3, 3, 2, 2, 1, 1]


def test_rules_refuse_another_number_of_rows(rules):
    """The device reads an entry per row of every array."""
    r = gen.LogitRules(DeferredContext(), 11, 3, frequency=0.5)
    for args in (([[1]] * 2, [[]] * 2), ([[1]] * 3, [[]] * 2), ([[1]] * 4, [[]] * 3), ([[1]] * 3, [[]] * 3, [True] * 2)):
        with pytest.raises(ValueError, match="expected 3 rows"):
            r.apply(64, *args)
    assert not rules and not r.ctx.live
    r.apply(64, [[1]] * 3, [[]] * 3, [True, False, True])
    assert len(rules) == 1
