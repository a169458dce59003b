"""Several sequences at once through the paged cache, and rules on the logits, against the oracle.

* PagedDecoder: the logits of every prompt and of every step (ragged lengths, idle sequences) equal the
  oracle's full forward (maxRelErr <= 1e-3, the bound of the single-sequence cache), both architectures.
* generate_batch draws, per sequence, the oracle's GPT.generate tokens; stops a sequence on request.
* generate and generate_batch under penalties, biases and masks draw the tokens of a plain loop over the
  oracle's logits with the rules applied in 64 bits.
"""
import math

import numpy as np
import pytest

from oracle.oracle import Oracle, max_rel_err

pytestmark = pytest.mark.gpu
LOGIT_TOL = 1e-3
V, T, L = 60, 40, 2


@pytest.fixture(scope="module")
def eng():
    from turt_b200.engine import GpuEngine
    e = GpuEngine.create(0)
    yield e
    e.ctx.close()


@pytest.fixture(scope="module")
def orc():
    return Oracle()


def _gpt(eng, orc, arch, E=48, H=3, seed=7):
    from turt_b200.engine import GpuGPT
    c = orc.cfg(V, T, L, H, E, arch)
    p = orc.init(c, seed)
    g = GpuGPT(eng, dict(vocabSize=V, blockSize=T, nEmbd=E, nLayer=L, nHead=H, arch=arch))
    g.loadFlat(p)
    return c, p, g


@pytest.mark.parametrize("arch,E,H", [("modern", 48, 3), ("gpt2", 48, 3), ("modern", 64, 1), ("gpt2", 40, 4)])
def test_logits_of_prompts_and_steps(eng, orc, arch, E, H):
    from turt_b200.generate import PagedDecoder
    c, p, g = _gpt(eng, orc, arch, E, H)
    rs = np.random.default_rng(3)
    seqs = [[int(x) for x in rs.integers(0, V, n)] for n in (1, 17, 5, 16)]
    dec = PagedDecoder(g, [T, 30, 12, 32], page_size=8)
    try:
        live0 = eng.liveBuffers
        got = eng.read(dec.prefill(seqs), len(seqs) * V).reshape(len(seqs), V)
        for i, s in enumerate(seqs):
            assert max_rel_err(got[i], orc.logits(c, p, s, 1, len(s))[-1]) <= LOGIT_TOL
        for k in range(7):
            new = [int(x) for x in rs.integers(0, V, len(seqs))]
            new = [None if (i + k) % 3 == 0 else t for i, t in enumerate(new)]
            got = eng.read(dec.step(new), len(seqs) * V).reshape(len(seqs), V)
            for i, (s, t) in enumerate(zip(seqs, new)):
                if t is not None:
                    s.append(t)
                    assert max_rel_err(got[i], orc.logits(c, p, s, 1, len(s))[-1]) <= LOGIT_TOL, (k, i)
        assert eng.liveBuffers == live0  # a step leaves no buffers behind
    finally:
        dec.close()


@pytest.mark.parametrize("arch,temperature,top_k", [("modern", 1.0, None), ("gpt2", 0.9, 8), ("modern", 0.7, 4)])
def test_batch_matches_oracle(eng, orc, arch, temperature, top_k):
    from turt_b200.generate import generate_batch
    from turt_b200.pretrain import Mulberry32
    c, p, g = _gpt(eng, orc, arch)
    prompts = [[5, 9, 2], [1], [3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8, 9, 7, 9, 3, 2]]
    want = [orc.generate(c, p, s, 20, temperature=temperature, topk=top_k or 0, rng_state=orc.rng(123 + i))
            for i, s in enumerate(prompts)]
    got = generate_batch(g, prompts, 20, temperature=temperature, top_k=top_k, rngs=[Mulberry32(123 + i) for i in range(3)])
    assert got == want
    # sequence 1 stops after four tokens; the others do not notice
    seen = [0, 0, 0]

    def stop(i, _):
        seen[i] += 1
        return not (i == 1 and seen[1] == 4)
    got = generate_batch(g, prompts, 20, temperature=temperature, top_k=top_k, rngs=[Mulberry32(123 + i) for i in range(3)],
                         on_token=stop)
    assert got == [want[0], want[1][:5], want[2]]


@pytest.mark.parametrize("cache_type", ["f16", "bf16"])
def test_batch_with_a_16_bit_cache(eng, orc, cache_type):
    """Logits after a step through a 16-bit cache.  A key or value is off by at most half a step, u = 2^-11 or 2^-8
    relative.  With scores below 4 in size a score moves by at most 4 u, a weight by a factor exp(8 u) at most, an
    attention output (8 u + u) max|v|; with two layers of weights drawn at 0.02 the logits move by far less than their
    own size times 9 u."""
    from turt_b200.generate import PagedDecoder
    c, p, g = _gpt(eng, orc, "modern")
    u = 2.0 ** -11 if cache_type == "f16" else 2.0 ** -8
    dec = PagedDecoder(g, [20, 20], cache_type=cache_type)
    try:
        dec.prefill([[1, 2, 3, 4, 5], [7]])
        got = eng.read(dec.step([6, 8]), 2 * V).reshape(2, V)
        for row, s in zip(got, ([1, 2, 3, 4, 5, 6], [7, 8])):
            want = orc.logits(c, p, s, 1, len(s))[-1]
            assert np.abs(row - want).max() <= 9 * u * np.abs(want).max()
    finally:
        dec.close()


def _ruled(orc, c, p, prompt, n, rng, temperature, rep, freq, pres, bias, allowed, row=0):
    """GPT.generate's loop over the oracle's logits with the rules in 64 bits."""
    from turt_b200.generate import apply_temperature_top_k, sample_from_logits
    ids = list(prompt)
    for _ in range(n):
        x = orc.logits(c, p, ids, 1, len(ids))[-1].astype(np.float64)
        made = ids[len(prompt):]
        for t in set(ids):
            x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
        for t in set(made):
            x[t] -= freq * made.count(t) + pres
        for t, v in (bias or {}).items():
            x[t] += v
        if allowed is not None:
            m = allowed(row, ids)
            if m is not None:
                x[~np.asarray(m)] = -math.inf
        ids.append(sample_from_logits(apply_temperature_top_k(x, temperature), rng))
    return ids


def _grammar(row, ids):
    """Even and odd tokens by turns; sequence 1 is free."""
    return None if row == 1 else np.arange(V) % 2 == len(ids) % 2


RULES = dict(rep=1.3, freq=0.4, pres=0.25, bias={3: 2.0, 59: -1.0, 0: 1.0}, allowed=_grammar)
KW = dict(repetition_penalty=1.3, frequency_penalty=0.4, presence_penalty=0.25, bias={3: 2.0, 59: -1.0, 0: 1.0}, allowed=_grammar)


def test_generate_under_rules(eng, orc):
    from turt_b200.generate import generate
    from turt_b200.pretrain import Mulberry32
    from turt_b200.runtime import Model, make_config
    c = orc.cfg(V, T, L, 2, 32, "modern")
    p = orc.init(c, 11)
    m = Model(eng.ctx, make_config(V, T, L, 2, 32, "modern"))
    try:
        m.load_flat(p)
        want = _ruled(orc, c, p, [5, 9, 2], 20, Mulberry32(5), 0.5, **RULES)
        assert generate(m, [5, 9, 2], 20, temperature=0.5, rng=Mulberry32(5), **KW) == want
        assert all((t % 2) == (i % 2) for i, t in enumerate(want) if i >= 3)
        # rules that change nothing: the plain path's tokens
        plain = generate(m, [5, 9, 2], 20, rng=Mulberry32(5))
        assert generate(m, [5, 9, 2], 20, rng=Mulberry32(5), allowed=lambda r, ids: None) == plain
        assert generate(m, [5, 9, 2], 20, rng=Mulberry32(5), allowed=lambda r, ids: np.ones(V, bool)) == plain
    finally:
        m.close()


def test_batch_under_rules(eng, orc):
    from turt_b200.generate import generate_batch
    from turt_b200.pretrain import Mulberry32
    c, p, g = _gpt(eng, orc, "gpt2")
    prompts = [[5, 9, 2, 2], [1], [4, 4, 8]]
    want = [_ruled(orc, c, p, s, 15, Mulberry32(70 + i), 0.6, **RULES, row=i) for i, s in enumerate(prompts)]
    eng.reclaim()
    live0 = eng.liveBuffers
    got = generate_batch(g, prompts, 15, temperature=0.6, rngs=[Mulberry32(70 + i) for i in range(3)], **KW)
    assert got == want
    eng.reclaim()
    assert eng.liveBuffers == live0


def test_refusals(eng, orc):
    from turt_b200._lib import TurtError
    from turt_b200.engine import GpuGPT
    from turt_b200.generate import LogitRules, generate_batch
    from turt_b200.runtime import Model, make_config
    c, p, g = _gpt(eng, orc, "modern")
    assert generate_batch(g, [], 5) == []
    assert generate_batch(g, [[1, 2]], 0) == [[1, 2]]
    with pytest.raises(ValueError):
        generate_batch(g, [[1], []], 5)
    with pytest.raises(ValueError):
        generate_batch(g, [[1] * 30], T - 29)  # beyond the block
    with pytest.raises(ValueError):
        generate_batch(g, [[1]], 5, rngs=[])
    with pytest.raises(ValueError):
        generate_batch(g, [[1]], 5, cache_type="f64")
    with pytest.raises(ValueError):
        LogitRules(eng.ctx, V, 1, repetition=0.0)
    with pytest.raises(ValueError):
        LogitRules(eng.ctx, V, 2, bias=[{1: 1.0}])
    with pytest.raises(ValueError):
        generate_batch(g, [[1]], 5, allowed=lambda r, ids: np.ones(V + 1, bool))
    with pytest.raises(TurtError):
        generate_batch(g, [[1]], 5, bias={V: 1.0})  # a token that is not in the vocabulary
    with pytest.raises(TypeError):
        generate_batch(GpuGPT(eng, dict(vocabSize=V, blockSize=T, nEmbd=32, nLayer=1, nHead=2, arch="modern"), fused=True),
                       [[1]], 5)
    m = Model(eng.ctx, make_config(V, T, 1, 2, 32, "modern"))
    with pytest.raises(TurtError):
        m.generate_logits()  # nothing generated yet
    m.close()
    assert generate_batch(g, [[1]], 3, allowed=lambda r, ids: None)  # still usable
