"""Device memory of generation under rules, without a GPU: a context whose free() is deferred to reclaim(), as the
library's is, and a model that answers with fixed logits."""
import numpy as np
import pytest

import turt_b200.generate as gen
from turt_b200._lib import ERR_RANGE, TurtError

V = 50


class DeferredContext:
    """Buffers as host arrays; a freed one is held until reclaim()."""
    handle = None

    def __init__(self, fail=False):
        self.live, self.pending, self.next, self.fail = {}, [], 64, fail

    def buffer(self, elems):
        p, self.next = self.next, self.next + (1 << 20)
        self.live[p] = elems
        return p

    def upload(self, p, a):
        assert a.nbytes <= 4 * self.live[p]

    def free(self, p):
        self.pending.append(p)

    def reclaim(self):
        for p in self.pending:
            del self.live[p]
        self.pending = []
        if self.fail:
            raise TurtError(ERR_RANGE, "reported late")

    def download(self, p, n):
        return np.zeros(n, np.float32)


class FakeModel:
    class cfg:
        block_size, vocab_size = 512, V

    def __init__(self, ctx):
        self.ctx = ctx

    def generate_prefill(self, ids):
        return np.zeros(V, np.float32)

    def generate_step(self, token, pos):
        return np.zeros(V, np.float32)

    def generate_logits(self):
        return 64


@pytest.fixture(autouse=True)
def no_library(monkeypatch):
    class Lib:
        @staticmethod
        def turt_logit_rules_apply(*a):
            return 0
    monkeypatch.setattr(gen, "lib", lambda: Lib)


@pytest.mark.parametrize("kw", [dict(repetition_penalty=1.3), dict(bias={3: 1.0}), dict(allowed=lambda r, ids: np.ones(V, bool))])
def test_generate_gives_its_memory_back(kw):
    ctx = DeferredContext()
    model = FakeModel(ctx)
    for _ in range(3):
        ids = gen.generate(model, [1, 2], 200, rng=lambda: 0.5, **kw)  # long enough for a buffer to grow
        assert len(ids) == 202 and not ctx.live


def test_an_error_on_the_way_out_hides_none():
    def stop(_):
        raise KeyError("mine")
    ctx = DeferredContext(fail=True)
    with pytest.raises(KeyError):
        gen.generate(FakeModel(ctx), [1], 5, rng=lambda: 0.5, on_token=stop, presence_penalty=0.5)
    assert not ctx.live
    with pytest.raises(TurtError):  # alone it is raised
        gen.generate(FakeModel(ctx), [1], 5, rng=lambda: 0.5, presence_penalty=0.5)
    assert not ctx.live
