"""Sampling continuations from a GPU model: GPT.generate with a KV cache.

GPT.generate (src/models/gpt.ts:291-321) re-runs the whole forward over the last blockSize
tokens for every new token and samples from the last position's logits.  Here the forward of
a context that still fits the block is split into one prefill (turt_generate_prefill, which
fills the per-layer key / value cache) and one decode step per new token
(turt_generate_step); once the context outgrows the block the window slides, every position
shifts, and each token re-prefills the cropped window, as the reference does.  The logits come
back to the host, where temperature, top-k and sampleFromLogits (gpt.ts:324-341) run with the
reference's arithmetic: f32 logits divided by the temperature into a Float32Array, the top-k
threshold taken from a descending sort, exp in double stored as f32 probabilities whose double
sum scales rng(), and a sequential subtraction scan.

Beyond the reference: LogitRules (penalties for repeated tokens, biases, masks) run on the device
before the logits come back, and generate_batch decodes several sequences at a time through a paged
cache (GpuEngine.pagedAppend / pagedAttention) on the op-by-op GpuGPT.
"""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Callable, Iterable, List, Optional

import numpy as np

from ._lib import CACHE_TYPES, TurtError, check, lib, u32
from .pretrain import Mulberry32
from .runtime import make_logit_rules, make_paged_kv

# The reference's module-level defaultRng (src/math/random.ts:27): one mulberry32(42) stream
# shared by every call that passes no rng.
default_rng = Mulberry32(42)


def apply_temperature_top_k(logits: np.ndarray, temperature: float = 1.0, top_k: Optional[int] = None) -> np.ndarray:
    """last[j] = logits[j] / temperature (stored as f32); with 0 < top_k < V, entries below the
    top_k-th largest become -inf (gpt.ts:306-314)."""
    last = (np.asarray(logits, dtype=np.float32).astype(np.float64) / float(temperature)).astype(np.float32)
    V = last.shape[0]
    if top_k and top_k < V:
        threshold = np.sort(last)[::-1][top_k - 1]
        last[last < threshold] = -np.inf
    return last


def sample_from_logits(logits: np.ndarray, rng: Callable[[], float]) -> int:
    """sampleFromLogits (gpt.ts:324-341): one index drawn from softmax(logits)."""
    last = np.asarray(logits, dtype=np.float32)
    mx = float(np.max(last)) if last.size else -np.inf
    e = np.exp(last.astype(np.float64) - mx)
    probs = e.astype(np.float32)
    total = float(np.cumsum(e)[-1])  # a sequential double sum, as the reference's loop
    r = rng() * total
    # r -= probs[j] one after another; the first j where r <= 0 is drawn
    scan = np.subtract.accumulate(np.concatenate(([r], probs.astype(np.float64))))[1:]
    hit = np.flatnonzero(scan <= 0)
    return int(hit[0]) if hit.size else last.shape[0] - 1


class _Grown:
    """A device buffer that is replaced by a larger one when an upload does not fit."""

    def __init__(self, ctx):
        self.ctx, self.ptr, self.bytes = ctx, None, 0

    def put(self, a: np.ndarray) -> int:
        a = np.ascontiguousarray(a)
        if a.nbytes > self.bytes or self.ptr is None:
            self.free()
            self.bytes = max(64, 2 * a.nbytes)
            self.ptr = self.ctx.buffer((self.bytes + 3) // 4)
        self.ctx.upload(self.ptr, a)
        return self.ptr

    def free(self) -> None:
        if self.ptr is not None:
            self.ctx.free(self.ptr)
        self.ptr = None


class LogitRules:
    """Rules on the logits of `rows` sequences, applied on the device (turt_logit_rules_apply).

    repetition (> 0), frequency and presence are numbers or one per row; bias is {token: value} or one
    such dict (or None) per row; allowed(row, ids) gives the tokens that may come next as a boolean array
    [vocab], or None for any.  ids of the prompt count for `repetition` only."""

    def __init__(self, ctx, vocab: int, rows: int = 1, repetition=1.0, frequency=0.0, presence=0.0, bias=None,
                 allowed: Optional[Callable] = None):
        self.ctx, self.vocab, self.rows, self.allowed = ctx, vocab, rows, allowed
        per_row = lambda v: np.broadcast_to(np.asarray(v, np.float32), (rows,))  # noqa: E731
        self.repetition, self.frequency, self.presence = per_row(repetition), per_row(frequency), per_row(presence)
        if not np.all(self.repetition > 0):
            raise ValueError("repetition penalties must be positive")
        self.bias = [bias] * rows if bias is None or isinstance(bias, dict) else list(bias)
        if len(self.bias) != rows:
            raise ValueError(f"expected {rows} bias dicts, got {len(self.bias)}")
        self.penalties = bool((self.repetition != 1).any() or self.frequency.any() or self.presence.any())
        self.active = self.penalties or any(self.bias) or allowed is not None
        self._bufs, self._out = {}, None

    def _put(self, name: str, a: np.ndarray) -> int:
        return self._bufs.setdefault(name, _Grown(self.ctx)).put(a)

    def apply(self, d_logits: int, prompts, generated, live=None) -> np.ndarray:
        """The logits [rows][vocab] at d_logits under the rules, on the host; prompts and generated hold
        each row's ids.  Rows that live (a truth value per row, default all) leaves out get no mask: allowed is
        not asked about them."""
        for what in (prompts, generated) if live is None else (prompts, generated, live):
            if len(what) != self.rows:
                raise ValueError(f"expected {self.rows} rows, got {len(what)}")
        kw = {}
        if self.penalties:
            lens = np.array([[len(p), len(g)] for p, g in zip(prompts, generated)], np.int64)
            start = np.concatenate(([0], np.cumsum(lens.sum(1))))
            kw = dict(tokens=self._put("tokens", u32([i for p, g in zip(prompts, generated) for i in (*p, *g)] or [0])),
                      token_start=self._put("start", u32(start)),
                      generated_start=self._put("generated", u32(start[:-1] + lens[:, 0])),
                      repetition=self._put("repetition", self.repetition),
                      frequency=self._put("frequency", self.frequency), presence=self._put("presence", self.presence))
        if any(self.bias):
            pairs = [sorted((b or {}).items()) for b in self.bias]
            kw.update(bias_ids=self._put("bias_ids", u32([i for p in pairs for i, _ in p])),
                      bias=self._put("bias", np.array([v for p in pairs for _, v in p], np.float32)),
                      bias_start=self._put("bias_start", u32(np.concatenate(([0], np.cumsum([len(p) for p in pairs]))))))
        if self.allowed is not None:
            masks = [self.allowed(r, [*prompts[r], *generated[r]]) if live is None or live[r] else None
                     for r in range(self.rows)]
            some = [np.asarray(m, bool) for m in masks if m is not None]
            for m in some:
                if m.shape != (self.vocab,):
                    raise ValueError(f"a mask must hold {self.vocab} truth values, got shape {m.shape}")
            if some:
                words = (self.vocab + 31) // 32
                bits = np.zeros((len(some), words * 32), bool)
                bits[:, :self.vocab] = some
                at = iter(range(len(some)))
                kw.update(mask=self._put("mask", np.packbits(bits, axis=1, bitorder="little").view(np.uint32)),
                          mask_row=self._put("mask_row", u32([0xFFFFFFFF if m is None else next(at) for m in masks])),
                          n_masks=len(some))
        if self._out is None:
            self._out = self.ctx.buffer(self.rows * self.vocab)
        check(lib().turt_logit_rules_apply(self.ctx.handle, d_logits, self.vocab, self._out, self.vocab, self.rows, self.vocab,
                                           C.byref(make_logit_rules(**kw))))
        return self.ctx.download(self._out, self.rows * self.vocab).reshape(self.rows, self.vocab)

    def close(self) -> None:
        """Frees the buffers; their memory comes back with the context's next reclaim()."""
        for b in self._bufs.values():
            b.free()
        if self._out is not None:
            self.ctx.free(self._out)
        self._bufs, self._out = {}, None


@contextlib.contextmanager
def _released(ctx, *things):
    """Closes `things` on the way out and gives their memory back.  An error that the device reports then does not
    take the place of the one that led out."""
    try:
        yield
    except BaseException:
        with contextlib.suppress(TurtError):
            for t in things:
                t.close()
            ctx.reclaim()
        raise
    for t in things:
        t.close()
    ctx.reclaim()


class Generator:
    """KV-cached decoding state of one model: which window of ids the cache holds."""

    def __init__(self, model):
        self.model = model
        self.block = model.cfg.block_size
        self.win_start = 0
        self.cached = 0

    def next_logits(self, ids: List[int]) -> np.ndarray:
        """Logits of the last position of ids[-block_size:]: one decode step when the cache
        already holds every earlier position of that window, else a prefill of the window."""
        if not ids:
            raise ValueError("generate: the prompt must hold at least one token")
        start = max(0, len(ids) - self.block)
        if self.cached > 0 and start == self.win_start and self.win_start + self.cached == len(ids) - 1:
            out = self.model.generate_step(ids[-1], self.cached)
            self.cached += 1
            return out
        out = self.model.generate_prefill(ids[start:])
        self.win_start, self.cached = start, len(ids) - start
        return out


def generate(model, prompt: Iterable[int], max_new_tokens: int, temperature: float = 1.0,
             top_k: Optional[int] = None, rng: Optional[Callable[[], float]] = None,
             on_token: Optional[Callable[[int], Optional[bool]]] = None, repetition_penalty: float = 1.0,
             frequency_penalty: float = 0.0, presence_penalty: float = 0.0, bias: Optional[dict] = None,
             allowed: Optional[Callable] = None) -> List[int]:
    """GPT.generate on the GPU model: returns prompt + sampled ids; on_token returning False
    stops early (gpt.ts:291-321).  The penalties, bias {token: value} and allowed(row, ids) are
    LogitRules on the logits before the temperature (none by default, as in the reference)."""
    rng = default_rng if rng is None else rng
    ids = [int(i) for i in prompt]
    n_prompt = len(ids)
    gen = Generator(model)
    rules, held = None, contextlib.nullcontext()
    if (repetition_penalty, frequency_penalty, presence_penalty) != (1.0, 0.0, 0.0) or bias or allowed is not None:
        rules = LogitRules(model.ctx, model.cfg.vocab_size, 1, repetition_penalty, frequency_penalty, presence_penalty, bias,
                           allowed)
        held = _released(model.ctx, rules)
    with held:
        for _ in range(max_new_tokens):
            logits = gen.next_logits(ids)
            if rules is not None:
                logits = rules.apply(model.generate_logits(), [ids[:n_prompt]], [ids[n_prompt:]])[0]
            last = apply_temperature_top_k(logits, temperature, top_k)
            nxt = sample_from_logits(last, rng)
            ids.append(nxt)
            if on_token is not None and on_token(nxt) is False:
                break
    return ids


class PagedDecoder:
    """Several sequences of an op-by-op GpuGPT at once: keys and values in pages, one page table for all
    layers.  prefill() takes the prompts, step() one more token of each sequence; both give the logits
    of every sequence's last position on the device."""

    def __init__(self, gpt, lengths, cache_type: str = "f32", page_size: int = 16):
        if gpt.fused:
            raise TypeError("PagedDecoder runs the op-by-op GpuGPT (fused=False)")
        self.gpt, self.e, self.batch = gpt, gpt.engine, len(lengths)
        if cache_type not in CACHE_TYPES:
            raise ValueError(f"cache type must be one of {list(CACHE_TYPES)}, got {cache_type!r}")
        c = gpt.config
        self.E, self.H, self.V, self.L = c["nEmbd"], c["nHead"], c["vocabSize"], c["nLayer"]
        self.hd = self.E // self.H
        if max(lengths) > c["blockSize"]:
            raise ValueError(f"{max(lengths)} positions exceed block size {c['blockSize']}")
        need = [-(-n // page_size) for n in lengths]
        self.n_pages, self.width = sum(need), max(need)
        self.room = np.array(need, np.int64) * page_size
        table = np.full((self.batch, self.width), 0xFFFFFFFF, np.uint32)  # no page
        page = 0
        for b, n in enumerate(need):
            table[b, :n] = np.arange(page, page + n)
            page += n
        self.lens = np.zeros(self.batch, np.int64)
        self.held, self.tmp, self.indices = [], {}, []
        try:
            self._reserve(table, cache_type, page_size)
        except BaseException:
            with contextlib.suppress(TurtError):
                self.close()
            raise

    def _reserve(self, table, cache_type, page_size) -> None:
        def keep(p):
            self.held.append(p)
            return p
        self.table = keep(self.e.indexBuffer(table))
        self.d_lens = keep(self.e.indexBuffer(np.zeros(self.batch, np.uint32)))
        per = self.n_pages * page_size * self.E
        words = per if cache_type == "f32" else (per + 1) // 2
        self.kv = [make_paged_kv(keep(self.e.buffer(words)), keep(self.e.buffer(words)), self.table, self.d_lens, cache_type,
                                 self.n_pages, page_size, self.H, self.hd, self.batch, self.width) for _ in range(self.L)]
        self.work = self.e.pagedAttentionWorkspace(self.kv[0], self.H)
        self.space = keep(self.e.buffer((self.work + 3) // 4))
        self.logits = keep(self.e.buffer(self.batch * self.V))

    def _new(self, name: str, n: int) -> int:
        """The forward's buffer `name`.  All layers and prompts use the same one after another, which the stream orders;
        the first use takes the largest size."""
        if name not in self.tmp:
            self.tmp[name] = self.e.buffer(n)
        return self.tmp[name]

    def _index(self, a) -> int:
        self.indices.append(self.e.indexBuffer(a))
        return self.indices[-1]

    def _lin(self, name, x, w, rows, k, n, bias=None) -> int:
        out = self._new(name, rows * n)
        self.e.matmulInto(x, w.buffer, out, rows, k, n, 1, False, False, False)
        if bias is not None:
            self.e.ewise(out, bias.buffer, out, rows * n, n, 0, False)
        return out

    def _norm(self, x, rows, g, b) -> int:
        out, stat = self._new("norm", rows * self.E), self._new("stat", 2 * rows)
        if self.gpt.modern:
            self.e.rmsFwd(x, g.buffer, out, stat, rows, self.E, 1e-5)
        else:
            self.e.lnFwd(x, g.buffer, b.buffer, out, stat, stat + 4 * rows, rows, self.E, 1e-5)
        return out

    def _add(self, name, a, b, n) -> int:
        out = self._new(name, n)
        self.e.ewise(a, b, out, n, n, 0, False)
        return out

    def _prompt_attention(self, q, k, v, out, t, longest) -> None:
        """Causal attention inside one prompt of t rows (q rotated already), with the ops of the tape."""
        e, H, hd, n = self.e, self.H, self.hd, t * self.E

        def heads(name, x):
            y = self._new(name, longest * self.E)
            e.permute4(x, y, [1, t, H, hd], [0, 2, 1, 3], n, False)
            return y
        qh, kh, vh = heads("qh", q), heads("kh", k), heads("vh", v)
        if self.gpt.modern:
            r = self._new("kr", longest * self.E)
            e.ropeInto(kh, r, H, t, hd, 10000.0)
            kh = r
        s, y = self._new("scores", H * longest * longest), self._new("yh", longest * self.E)
        e.matmulInto(qh, kh, s, t, hd, t, H, False, True, False)
        e.scale(s, s, H * t * t, self.gpt.headScale, False)
        e.maskInto(s, s, H, t)
        e.softmaxInto(s, s, H * t, t)
        e.matmulInto(s, vh, y, t, t, hd, H, False, False, False)
        e.permute4(y, out, [1, H, t, hd], [0, 2, 1, 3], n, False)

    def _forward(self, ids, pos, start) -> None:
        """One forward of rows (ids at positions pos): the prompts one after another (start: where each
        begins) or, start None, one new token per sequence."""
        try:
            self._run(ids, pos, start)
        finally:
            self._drop()  # the next forward's sizes are others
        self.e.reclaim()

    def _run(self, ids, pos, start) -> None:
        e, g, E, rows = self.e, self.gpt, self.E, len(ids)
        e.ctx.upload(self.d_lens, u32(self.lens))
        d_start = None if start is None else self._index(start)
        x = self._new("x", rows * E)
        e.gatherInto(g.wte.buffer, self._index(ids), x, rows, E, self.V)
        if g.wpe is not None:
            p = self._new("out", rows * E)
            e.gatherInto(g.wpe.buffer, self._index(pos), p, rows, E, g.config["blockSize"])
            self._add("x", x, p, rows * E)
        for blk, kv in zip(g.blocks, self.kv):
            y = self._norm(x, rows, blk["ln1g"], blk.get("ln1b"))
            q, k, v = (self._lin(n, y, blk[n + "W"], rows, E, E, blk.get(n + "b")) for n in "qkv")
            qr, att = self._new("qr", rows * E), self._new("att", rows * E)
            e.pagedAppend(kv, k, E, v, E, rows, start=d_start, q=q, qStride=E, qOut=qr, qOutStride=E, nHead=self.H,
                          rotDim=self.hd if g.modern else 0)
            if start is None:
                e.pagedAttention(kv, qr, E, att, E, self.H, self.space, self.work, scale=g.headScale)
            else:
                longest = int(np.diff(start).max())
                for lo, hi in zip(start[:-1], start[1:]):
                    at = 4 * int(lo) * E
                    self._prompt_attention(qr + at, k + at, v + at, att + at, int(hi - lo), longest)
            h = self._add("h", x, self._lin("out", att, blk["projW"], rows, E, E, blk.get("projb")), rows * E)
            y = self._norm(h, rows, blk["ln2g"], blk.get("ln2b"))
            n = g.hidden
            if g.modern:
                a, u = self._lin("gate", y, blk["gateW"], rows, E, n), self._lin("up", y, blk["upW"], rows, E, n)
                act = self._new("act", rows * n)
                e.siluInto(a, act, rows * n)
                e.ewise(act, u, act, rows * n, rows * n, 2, False)
                m = self._lin("out", act, blk["downW"], rows, n, E)
            else:
                f = self._lin("gate", y, blk["fcW"], rows, E, n, blk["fcb"])
                act = self._new("act", rows * n)
                e.geluInto(f, act, rows * n)
                m = self._lin("out", act, blk["mpW"], rows, n, E, blk["mpb"])
            self._add("x", h, m, rows * E)
        if start is not None:
            last = self._new("h", self.batch * E)
            e.gatherInto(x, self._index(start[1:] - 1), last, self.batch, E, rows)
            x = last
        y = self._norm(x, self.batch, g.lnfg, g.lnfb)
        e.matmulInto(y, g.wte.buffer, self.logits, self.batch, E, self.V, 1, False, True, False)

    def _drop(self) -> None:
        for b in (*self.tmp.values(), *self.indices):
            self.e.free(b)
        self.tmp, self.indices = {}, []

    def _fits(self, lens) -> None:
        for i in np.flatnonzero(lens > self.room):
            raise ValueError(f"sequence {i} would hold {lens[i]} positions, its pages hold {self.room[i]}")

    def prefill(self, prompts) -> int:
        if len(prompts) != self.batch or not all(len(p) for p in prompts):
            raise ValueError(f"expected {self.batch} prompts of one token or more")
        lens = np.array([len(p) for p in prompts])
        self._fits(lens)
        self.lens = lens
        ids = np.concatenate([np.asarray(p) for p in prompts])
        try:
            self._forward(u32(ids), u32(np.concatenate([np.arange(n) for n in lens])), np.concatenate(([0], np.cumsum(lens))))
        except BaseException:
            self.lens = np.zeros(self.batch, np.int64)  # what the pages hold is not known
            raise
        return self.logits

    def step(self, tokens) -> int:
        """One token per sequence; None leaves a sequence idle (its logits are then meaningless)."""
        if len(tokens) != self.batch:
            raise ValueError(f"expected {self.batch} tokens, got {len(tokens)}")
        live = np.array([t is not None for t in tokens])
        lens = np.where(live, self.lens + 1, 0)
        self._fits(lens)
        held, self.lens = self.lens, lens
        try:
            self._forward(u32([0 if t is None else t for t in tokens]), u32(np.maximum(lens - 1, 0)), None)
            held = np.where(live, lens, held)
        finally:
            self.lens = held
        return self.logits

    def close(self) -> None:
        for b in self.held:
            self.e.free(b)
        self.held = []
        self._drop()
        self.e.reclaim()


def generate_batch(gpt, prompts, max_new_tokens: int, temperature: float = 1.0, top_k: Optional[int] = None, rngs=None,
                   on_token: Optional[Callable[[int, int], Optional[bool]]] = None, repetition_penalty=1.0,
                   frequency_penalty=0.0, presence_penalty=0.0, bias=None, allowed: Optional[Callable] = None,
                   cache_type: str = "f32", page_size: int = 16) -> List[List[int]]:
    """generate() for several prompts at once on an op-by-op GpuGPT, through a paged cache; prompt and new
    tokens together must fit the block.  rngs holds one generator per sequence (default: each its own
    mulberry32(42 + i)); on_token(i, id) returning False stops sequence i.  The rules are LogitRules
    (numbers or one per sequence)."""
    seqs = [[int(i) for i in p] for p in prompts]
    if not seqs:
        return []
    if not all(seqs):
        raise ValueError("generate_batch: every prompt must hold at least one token")
    if max_new_tokens <= 0:
        return seqs
    rngs = [Mulberry32(42 + i) for i in range(len(seqs))] if rngs is None else list(rngs)
    if len(rngs) != len(seqs):
        raise ValueError(f"expected {len(seqs)} generators, got {len(rngs)}")
    n_prompt = [len(s) for s in seqs]
    rules = LogitRules(gpt.engine.ctx, gpt.config["vocabSize"], len(seqs), repetition_penalty, frequency_penalty,
                       presence_penalty, bias, allowed)
    dec = PagedDecoder(gpt, [n + max_new_tokens for n in n_prompt], cache_type, page_size)
    with _released(gpt.engine.ctx, rules, dec):
        logits = dec.prefill(seqs)
        live = [True] * len(seqs)
        for k in range(max_new_tokens):
            if rules.active:
                rows = rules.apply(logits, [s[:n] for s, n in zip(seqs, n_prompt)], [s[n:] for s, n in zip(seqs, n_prompt)],
                                   live)
            else:
                rows = gpt.engine.read(logits, len(seqs) * dec.V).reshape(len(seqs), dec.V)
            for i, s in enumerate(seqs):
                if live[i]:
                    s.append(sample_from_logits(apply_temperature_top_k(rows[i], temperature, top_k), rngs[i]))
                    if on_token is not None and on_token(i, s[-1]) is False:
                        live[i] = False
            if k + 1 == max_new_tokens or not any(live):
                break
            logits = dec.step([s[-1] if alive else None for s, alive in zip(seqs, live)])
    return seqs
