"""The serving operators of the framework, as they are measured: the paged key / value cache (append with
rotation, attention of one new token) and the rules on logits (penalties, biases, masks).

`own` false computes them from elementary torch operations in 32 bits; `own` true calls the framework.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_engines = {}


# ---------------------------------------------------------------------------------- cases

def listed():
    return [
        # one sequence's next token, the heads of the 6-layer 384-wide model, cache in fp32
        dict(name="append_token", op="append", heads=6, kv_heads=6, dim=64, rot=64, page=16, type="f32", batch=1,
             new=1, lo=200, hi=200, empty=0, base=10000.0),
        # the next token of a full batch, the heads of the 12-layer 768-wide model; some places of the batch idle
        dict(name="append_batch", op="append", heads=12, kv_heads=12, dim=64, rot=64, page=16, type="f32", batch=256,
             new=1, lo=1, hi=1024, empty=9, base=10000.0),
        # ragged prompts of grouped heads into bf16 pages, at the end of long contexts
        dict(name="append_prompts", op="append", heads=32, kv_heads=8, dim=128, rot=128, page=64, type="bf16", batch=12,
             new=683, lo=1000, hi=100000, empty=0, base=500000.0),
        # many short prompts, an odd page size, half of each head rotated, fp16 pages
        dict(name="append_partial", op="append", heads=15, kv_heads=5, dim=80, rot=40, page=24, type="f16", batch=61,
             new=97, lo=97, hi=2000, empty=0, base=10000.0),
        # one sequence's next token: the 6-layer 384-wide model inside its block of 256
        dict(name="attend_token", op="attend", heads=6, kv_heads=6, dim=64, page=16, type="f32", batch=1, lo=200, hi=200,
             empty=0, window=0),
        # a batch of the 12-layer 768-wide model, contexts up to its block of 1024, some places idle
        dict(name="attend_batch", op="attend", heads=12, kv_heads=12, dim=64, page=16, type="f32", batch=64, lo=1,
             hi=1024, empty=3, window=0),
        # one very long context, grouped heads, bf16 pages
        dict(name="attend_long", op="attend", heads=32, kv_heads=8, dim=128, page=64, type="bf16", batch=1, lo=131001,
             hi=131001, empty=0, window=0),
        # a large serving batch of ragged contexts, grouped heads, bf16 pages: the largest case
        dict(name="attend_grouped", op="attend", heads=32, kv_heads=8, dim=128, page=32, type="bf16", batch=96, lo=1,
             hi=8192, empty=2, window=0),
        # a sliding window over odd sizes, fp16 pages
        dict(name="attend_window", op="attend", heads=15, kv_heads=5, dim=80, page=24, type="f16", batch=33, lo=3,
             hi=5000, empty=1, window=700),
        # one row of the 8192-word vocabulary, penalties for a short history
        dict(name="rules_row", op="rules", rows=1, vocab=8192, prompt=120, made=80, biases=0, masks=False),
        # a batch with an odd vocabulary, biases, and masks on some rows
        dict(name="rules_batch", op="rules", rows=64, vocab=50001, prompt=700, made=300, biases=40, masks=True),
        # a large batch of a large vocabulary with long histories
        dict(name="rules_large", op="rules", rows=256, vocab=128000, prompt=3000, made=1000, biases=300, masks=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "rules"])
    if op == "rules":
        vocab = _log(rng, 500, 128000)
        rows = _log(rng, 1, 256)
        prompt, made = _log(rng, 1, 3000), _log(rng, 1, 1000)
        return dict(op=op, rows=rows, vocab=vocab, prompt=prompt, made=made, biases=rng.choice([0, _log(rng, 1, 300)]),
                    masks=rng.random() < 0.6)
    group = rng.choice([1, 1, 2, 3, 4, 5, 8])
    kv_heads = _log(rng, 1, 12)
    dim = rng.choice([16, 32, 40, 48, 64, 64, 72, 80, 96, 112, 128, 128])
    while group * kv_heads * dim > 4096:
        kv_heads -= 1
    case = dict(op=op, heads=group * kv_heads, kv_heads=kv_heads, dim=dim, page=rng.choice([8, 16, 24, 32, 37, 64, 128]),
                type=rng.choice(["f32", "f16", "bf16"]))
    if op == "append":
        batch = _log(rng, 1, 256)
        new = rng.choice([1, _log(rng, 1, max(1, 8192 // batch))])
        hi = new + _log(rng, 1, min(100000, 10 ** 8 // (kv_heads * dim)))
        return dict(case, batch=batch, rot=rng.choice([0, dim // 2, dim, dim]), new=new, lo=rng.randint(new, hi), hi=hi,
                    empty=rng.choice([0, batch // 10]), base=rng.choice([10000.0, 500000.0]))
    batch = _log(rng, 1, 96)
    size = 4 if case["type"] == "f32" else 2
    hi = _log(rng, 1, min(131072, 786432 // batch, 3 * 10 ** 9 // (4 * batch * kv_heads * dim * size)))
    return dict(case, batch=batch, lo=rng.randint(1, hi), hi=hi, empty=rng.choice([0, batch // 10]),
                window=rng.choice([0, 0, _log(rng, 1, 4096)]))


def _lengths(c):
    """The lengths of the batch, in increasing order; the first `empty` places are idle."""
    b = c["batch"]
    return [0 if i < c["empty"] else c["lo"] + (c["hi"] - c["lo"]) * (i + 1) // b for i in range(b)]


def _new(c):
    """How many new rows each sequence brings: one, or ragged prompts of `new` at most."""
    if c["new"] == 1:
        return [1 if n else 0 for n in _lengths(c)]
    return [min(n, c["new"] - (101 * i) % (c["new"] // 2 + 1)) if n else 0 for i, n in enumerate(_lengths(c))]


def work(c):
    if c["op"] == "rules":
        n, ids = c["rows"] * c["vocab"], c["rows"] * (c["prompt"] + c["made"] + 2 * c["biases"])
        return {"bytes": 8 * n + 4 * ids + (n // 8 if c["masks"] else 0), "flops": n}
    size = 4 if c["type"] == "f32" else 2
    if c["op"] == "append":
        n = sum(_new(c))
        wide = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": n * (4 * wide + 4 * c["heads"] * c["dim"] + 2 * size * c["kv_heads"] * c["dim"]),
                "flops": 3 * n * (c["heads"] + c["kv_heads"]) * c["rot"]}
    seen = sum(min(n, c["window"]) if c["window"] else n for n in _lengths(c))
    return {"bytes": 2 * seen * c["kv_heads"] * c["dim"] * size + 8 * c["batch"] * c["heads"] * c["dim"],
            "flops": 4 * seen * c["heads"] * c["dim"]}


# --------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.Generator().manual_seed(seed + 1)
    return (_prepare_rules if case["op"] == "rules" else _prepare_cache)(dict(case), g, h)


def _prepare_cache(c, g, h):
    dev, n_seq, page, dim = "cuda", c["batch"], c["page"], c["dim"]
    order = torch.randperm(n_seq, generator=h)
    lens = torch.tensor(_lengths(c))[order]
    pages = (lens + page - 1) // page
    width = int(pages.max())
    at = torch.arange(width)[None, :]
    # appended rows go to pages of their own, behind a prefix that the sequences share; attention reads its own pages
    first = (lens - torch.tensor(_new(c))[order]) // page if c["op"] == "append" else torch.zeros_like(lens)
    mine = (at >= first[:, None]) & (at < pages[:, None])
    shared = int(first.max())
    total = shared + int(mine.sum())
    n_pages = total + total // 16 + 1
    spare = torch.randperm(n_pages, generator=h)[:total].to(torch.int32)
    table = torch.full((n_seq, width), -1, dtype=torch.int32)  # -1: no position has reached the page
    table[:, :shared] = spare[:shared]
    table[at.expand(n_seq, -1) >= pages[:, None]] = -1
    table[mine] = spare[shared:]
    shape = (n_pages, c["kv_heads"], page, dim)
    s = {"case": c, "table": table.to(dev), "lens": lens.to(torch.int32).to(dev)}
    for name in ("k", "v"):
        s[name] = torch.randn(shape, generator=g, device=dev, dtype=TYPES[c["type"]])
    if c["op"] == "append":
        new = torch.tensor(_new(c))[order]
        start = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)])
        # one new row for each place of the batch, idle ones too, or the rows of the prompts one after another
        rows = n_seq if c["new"] == 1 else int(start[-1])
        s["start"] = None if c["new"] == 1 else start.to(torch.int32).to(dev)
        s["rows"] = rows
        wide = (c["heads"] + 2 * c["kv_heads"]) * dim
        s["qkv"] = torch.randn(rows, wide, generator=g, device=dev)
        s["q_out"] = torch.zeros(rows, c["heads"] * dim, device=dev)
    else:
        # queries in place, in the fused projection of the new tokens
        s["qkv"] = torch.randn(n_seq, (c["heads"] + 2 * c["kv_heads"]) * dim, generator=g, device=dev)
        s["out"] = torch.empty(n_seq, c["heads"] * dim, device=dev)
    if own:
        from turt_b200.runtime import make_paged_kv
        s["kv"] = make_paged_kv(s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), s["lens"].data_ptr(),
                                c["type"], shape[0], page, c["kv_heads"], dim, n_seq, width)
        if c["op"] == "attend":
            s["space"] = torch.zeros(_engine().pagedAttentionWorkspace(s["kv"], c["heads"]), dtype=torch.uint8, device=dev)
    return s


def _prepare_rules(c, g, h):
    dev, rows, vocab = "cuda", c["rows"], c["vocab"]
    # frequent words come again and again: ids fall off like 1 / rank
    made = torch.randint(max(1, c["made"] // 2), c["made"] + 1, (rows,), generator=h)
    prompt = torch.randint(c["prompt"] // 2, c["prompt"] + 1, (rows,), generator=h)
    start = torch.cat([torch.zeros(1, dtype=torch.int64), (made + prompt).cumsum(0)])
    rank = torch.exp(torch.rand(int(start[-1]), generator=h, dtype=torch.float64) * math.log(vocab))
    ids = ((rank.long() - 1).clamp(0, vocab - 1) * 7919) % vocab
    s = {"case": c, "logits": torch.randn(rows, vocab, generator=g, device=dev) * 3, "out": torch.empty(rows, vocab, device=dev),
         "ids": ids.to(torch.int32).to(dev), "start": start.to(torch.int32).to(dev),
         "made": (start[:-1] + prompt).to(torch.int32).to(dev),
         "repetition": (1 + torch.rand(rows, generator=h) / 2).to(dev), "frequency": (torch.rand(rows, generator=h) - 0.3).to(dev),
         "presence": (torch.rand(rows, generator=h) / 2).to(dev), "bias_ids": None, "mask": None}
    if c["biases"]:
        n = min(c["biases"], vocab)
        step = torch.randint(1, vocab // n + 1, (rows, n), generator=h)
        s["bias_ids"] = (step.cumsum(1) - 1).reshape(-1).to(torch.int32).to(dev)  # increasing in each row
        s["bias"] = (torch.randn(rows * n, generator=h) * 4).to(dev)
        s["bias_start"] = (torch.arange(rows + 1) * n).to(torch.int32).to(dev)
    if c["masks"]:
        # a third of the rows follows no grammar, the others allow from nearly everything to nearly nothing
        n_masks = max(1, rows * 2 // 3)
        words = (vocab + 31) // 32
        few = torch.rand(n_masks, 1, generator=h)
        bits = torch.rand(n_masks, words, 32, generator=g, device=dev) < few.to(dev)[:, :, None]
        weight = torch.bitwise_left_shift(torch.ones(32, dtype=torch.int64, device=dev), torch.arange(32, device=dev))
        word = (bits * weight).sum(-1)
        s["mask"] = torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)
        s["mask_row"] = torch.where(torch.arange(rows) < n_masks, torch.arange(rows), -1)[torch.randperm(rows, generator=h)].to(torch.int32).to(dev)
    if own:
        from turt_b200.runtime import make_logit_rules
        at = lambda name: s[name].data_ptr() if s.get(name) is not None else None  # noqa: E731
        s["rules"] = make_logit_rules(tokens=at("ids"), token_start=at("start"), generated_start=at("made"),
                                      repetition=at("repetition"), frequency=at("frequency"), presence=at("presence"),
                                      bias_ids=at("bias_ids"), bias=at("bias"), bias_start=at("bias_start"),
                                      mask=at("mask"), mask_row=at("mask_row"),
                                      n_masks=s["mask"].shape[0] if c["masks"] else 0)
    return s


# ----------------------------------------------------------------------------------- runs

def _engine():
    from turt_b200.engine import GpuEngine
    dev, stream = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream
    if dev not in _engines:
        _engines[dev] = GpuEngine.create(dev)
    e = _engines[dev]
    if e.ctx.stream != stream:
        e.ctx.set_stream(stream)
    return e


def run(s):
    return {"append": _append, "attend": _attend, "rules": _rules}[s["case"]["op"]](s)


def _append(s):
    c = s["case"]
    heads, kv_heads, dim, rows = c["heads"], c["kv_heads"], c["dim"], s["rows"]
    if own:
        p, wide = s["qkv"].data_ptr(), s["qkv"].shape[1]
        _engine().pagedAppend(s["kv"], p + 4 * heads * dim, wide, p + 4 * (heads + kv_heads) * dim, wide, rows,
                              start=None if s["start"] is None else s["start"].data_ptr(), q=p, qStride=wide,
                              qOut=s["q_out"].data_ptr(), qOutStride=heads * dim, nHead=heads, rotDim=c["rot"], base=c["base"])
        return {"k": s["k"], "v": s["v"], "q": s["q_out"]}
    lens, row = s["lens"].long(), torch.arange(rows, device="cuda")
    if s["start"] is None:
        seq, pos = row, lens - 1
    else:
        start = s["start"].long()
        seq = (row[:, None] >= start[None, 1:]).sum(1)
        pos = lens[seq] - start[seq + 1] + row
    live = pos >= 0
    new = s["qkv"].view(rows, heads + 2 * kv_heads, dim)
    q, k, v = new[:, :heads], new[:, heads:heads + kv_heads], new[:, heads + kv_heads:]
    q, k = _rotate(q, pos, c), _rotate(k, pos, c)
    page = s["table"][seq[live], pos[live] // c["page"]].long()
    slot = pos[live] % c["page"]
    s["k"][page, :, slot] = k[live].to(s["k"].dtype)
    s["v"][page, :, slot] = v[live].to(s["v"].dtype)
    q_out = torch.where(live[:, None, None], q, s["q_out"].view(rows, heads, dim)).reshape(rows, heads * dim)
    return {"k": s["k"], "v": s["v"], "q": q_out}


def _rotate(x, pos, c):
    rot = c["rot"]
    if not rot:
        return x
    inv = c["base"] ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = pos.double()[:, None] * inv
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _attend(s):
    c = s["case"]
    heads, kv_heads, dim, n_seq = c["heads"], c["kv_heads"], c["dim"], c["batch"]
    if own:
        _engine().pagedAttention(s["kv"], s["qkv"].data_ptr(), s["qkv"].shape[1], s["out"].data_ptr(), heads * dim, heads,
                                 s["space"].data_ptr(), s["space"].numel(), window=c["window"])
        return s["out"]
    at = torch.arange(s["table"].shape[1] * c["page"], device="cuda")
    lens = s["lens"].long()[:, None]
    seen = at < lens
    if c["window"]:
        seen &= at >= lens - c["window"]
    table = s["table"].clamp(min=0).long()
    k, v = (s[x][table].transpose(1, 2).flatten(2, 3).float() for x in ("k", "v"))
    q = s["qkv"][:, :heads * dim].reshape(n_seq, kv_heads, heads // kv_heads, dim)
    score = (q @ k.transpose(-1, -2)) * (1 / math.sqrt(dim))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - top.clamp(min=-3e38)).exp()
    o = (p @ v) / p.sum(-1, keepdim=True)
    return torch.where(lens[:, :, None, None] > 0, o, 0.0).reshape(n_seq, heads * dim)


def _rules(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    if own:
        _engine().logitRules(s["logits"].data_ptr(), vocab, s["out"].data_ptr(), vocab, rows, vocab, s["rules"])
        return s["out"]
    i = torch.arange(s["ids"].numel(), device="cuda")
    row = (torch.searchsorted(s["start"].long(), i, right=True) - 1)
    place = row * vocab + s["ids"].long()
    seen = torch.zeros(rows * vocab, dtype=torch.bool, device="cuda")
    seen[place] = True
    made = torch.zeros(rows * vocab, device="cuda")
    made.index_add_(0, place, (i >= s["made"].long()[row]).float())
    seen, made = seen.view(rows, vocab), made.view(rows, vocab)
    x, rho = s["logits"], s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rho, x * rho), x)
    x = x - made * s["frequency"][:, None] - (made > 0) * s["presence"][:, None]
    if s["bias_ids"] is not None:
        at = torch.arange(rows, device="cuda").repeat_interleave(s["bias_ids"].numel() // rows) * vocab + s["bias_ids"].long()
        x = x.reshape(-1).index_add(0, at, s["bias"]).view(rows, vocab)
    if s["mask"] is not None:
        v = torch.arange(vocab, device="cuda")
        bit = (s["mask"][:, v >> 5] >> (v & 31)) & 1
        owner = s["mask_row"].long()
        x = x.masked_fill((owner[:, None] >= 0) & (bit[owner.clamp(min=0)] == 0), -math.inf)
    return x


# --------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "append":
        lens, start = s["lens"].tolist(), None if s["start"] is None else s["start"].tolist()
        pos, seq = [], []
        for b in range(c["batch"]):
            n = (start[b + 1] - start[b]) if start else 1
            pos += [lens[b] - n + j for j in range(n)]
            seq += [b] * n
        seq, pos = torch.tensor(seq, device="cuda"), torch.tensor(pos, device="cuda", dtype=torch.float64)
        live = (pos >= 0).nonzero()[:, 0]
        k, v, q_out = s["k"].double(), s["v"].double(), s["q_out"].double()
        x = s["qkv"].double().view(-1, c["heads"] + 2 * c["kv_heads"], c["dim"])[live].clone()
        seq, pos = seq[live], pos[live]
        turned = c["heads"] + c["kv_heads"]
        for m in range(c["rot"] // 2):
            a = pos / c["base"] ** (2 * m / c["rot"])
            z = torch.polar(torch.ones_like(a), a)[:, None] * torch.complex(x[:, :turned, 2 * m], x[:, :turned, 2 * m + 1])
            x[:, :turned, 2 * m], x[:, :turned, 2 * m + 1] = z.real, z.imag
        whole = pos.long()
        page, slot = s["table"][seq, whole // c["page"]].long(), whole % c["page"]
        k[page, :, slot] = x[:, c["heads"]:turned]
        v[page, :, slot] = x[:, turned:]
        q_out[live] = x[:, :c["heads"]].reshape(len(live), -1)
        return {"k": k, "v": v, "q": q_out}
    if c["op"] == "attend":
        group, dim = c["heads"] // c["kv_heads"], c["dim"]
        out = torch.zeros(c["batch"], c["heads"], dim, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            lo = max(0, n - c["window"]) if c["window"] else 0
            if n:
                at = torch.arange(lo, n, device="cuda")
                page, slot = s["table"][b, at // c["page"]].long(), at % c["page"]
                k, v = s["k"][page, :, slot].double(), s["v"][page, :, slot].double()
                q = s["qkv"][b, :c["heads"] * dim].double().view(c["kv_heads"], group, dim)
                p = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(dim), -1)
                out[b] = torch.einsum("hgn,nhd->hgd", p, v).reshape(c["heads"], dim)
        return out.reshape(c["batch"], -1)
    x = s["logits"].double()
    start, made = s["start"].tolist(), s["made"].tolist()
    words = s["mask"].long() & 0xFFFFFFFF if s["mask"] is not None else None
    v = torch.arange(c["vocab"], device="cuda")
    for r in range(c["rows"]):
        known, counts = s["ids"][start[r]:start[r + 1]].long().unique(), torch.bincount(s["ids"][made[r]:start[r + 1]].long(), minlength=c["vocab"])
        y, rho = x[r, known], s["repetition"][r].double()
        x[r, known] = torch.where(y > 0, y / rho, y * rho)
        x[r] -= s["frequency"][r].double() * counts + s["presence"][r].double() * (counts > 0)
        if s["bias_ids"] is not None:
            n = s["bias_ids"].numel() // c["rows"]
            x[r, s["bias_ids"][r * n:(r + 1) * n].long()] += s["bias"][r * n:(r + 1) * n].double()
        if words is not None and int(s["mask_row"][r]) >= 0:
            x[r, ((words[int(s["mask_row"][r])][v // 32] >> (v % 32)) & 1) == 0] = -math.inf
    return x
