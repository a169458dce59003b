"""The serving operators on the GPU against plain 64-bit implementations: appending rotated keys and
values to a paged cache, attention of one new token over it, and rules on logits.

Tolerances follow from the arithmetic (u = 2^-24, one fp32 rounding; 2u where an addition may
truncate), never from what the kernels gave:
* attention: a score is a sum of head_dim products, off by at most (dim + 4) 2u scale sum|q k|; exp
  turns an absolute error d of its argument into a relative one d (plus 2^-21 of its own), and the
  weights, their sum and the output each add their rounding, (n + 64) 2u at most for n positions.  The
  output is off by at most that times sum p |v|.
* append: two products and a sum per element, and the cosine and sine off by 2^-23: 2^-21 (|x| + |y|);
  then half a step of the cache's type (eps / 2, and half the smallest subnormal).
* rules: at most six roundings of values no larger than the terms' sum.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U2 = 2.0 ** -23


@pytest.fixture(scope="module")
def eng():
    from turt_b200.engine import GpuEngine
    e = GpuEngine.create(0)
    e.ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield e
    torch.cuda.synchronize()
    e.ctx.close()


class Cache:
    """A paged cache on the GPU with its pages in random order; order "slot" is [page][slot][head][dim],
    "pad" has gaps between positions, heads and pages."""

    def __init__(self, lens, kvh, dim, page, dtype, seed=0, order="head", extra=2, fill=None, kv=None):
        from turt_b200.runtime import make_paged_kv
        g = torch.Generator().manual_seed(seed)
        self.lens_l, self.page, self.kvh, self.dim, self.dtype = list(lens), page, kvh, dim, dtype
        need = [-(-n // page) for n in lens]
        self.width = max(1, max(need, default=1)) + 1
        n_pages = sum(need) + extra
        perm = torch.randperm(n_pages, generator=g).tolist()
        table = torch.full((max(1, len(lens)), self.width), -1, dtype=torch.int32)
        for b, c in enumerate(need):
            for j in range(c):
                table[b, j] = perm.pop()
        pad = 8 if order == "pad" else 0
        if order == "slot":
            ss, hs, ps = kvh * dim, dim, kvh * dim * page
        else:
            ss = dim + pad
            hs = ss * page + pad
            ps = hs * kvh + pad
        self.ss, self.hs, self.ps, self.n_pages = ss, hs, ps, n_pages
        t = TYPES[dtype]
        self.k = torch.full((n_pages * ps,), float("nan"), dtype=t)
        self.v = torch.full((n_pages * ps,), float("nan"), dtype=t)
        self.table_cpu = table
        if fill != "empty":
            for b, n in enumerate(lens):
                kv_ = torch.randn(2, n, kvh, dim, generator=g)
                for which, buf in ((0, self.k), (1, self.v)):
                    self.view(buf)[self._at(b, n)] = kv_[which].to(t)
        self.k, self.v = self.k.cuda(), self.v.cuda()
        self.table, self.lens = table.cuda(), torch.tensor(list(lens) or [0], dtype=torch.int32).cuda()
        self.kv = make_paged_kv(self.k.data_ptr(), self.v.data_ptr(), self.table.data_ptr(), self.lens.data_ptr(), dtype,
                                n_pages, page, kvh, dim, len(lens), self.width,
                                *((ps, hs, ss) if order != "head" else ()))

    def view(self, buf):
        """[page][slot][head][dim] view of a flat buffer."""
        return buf.as_strided((self.n_pages, self.page, self.kvh, self.dim), (self.ps, self.ss, self.hs, 1))

    def _at(self, b, n):
        j = torch.arange(n)
        return self.table_cpu[b, j // self.page].long(), j % self.page

    def read(self, buf, b, n):
        """[n][head][dim] of sequence b in float64 on the CPU."""
        return self.view(buf.cpu())[self._at(b, n)].double()


def attend(eng, c, q, heads, window=0, scale=None, lse=True, space=None, qs=None):
    n_seq, dim = len(c.lens_l), c.dim
    out = torch.full((n_seq, heads * dim + 3), float("nan"), device="cuda")
    ls = torch.full((n_seq, heads), float("nan"), device="cuda")
    if space is None:
        space = torch.zeros(eng.pagedAttentionWorkspace(c.kv, heads), dtype=torch.uint8, device="cuda")
    eng.pagedAttention(c.kv, q.data_ptr(), q.stride(0) if qs is None else qs, out.data_ptr(), out.stride(0), heads,
                       space.data_ptr(), space.numel(), scale=scale, window=window, lse=ls.data_ptr() if lse else None)
    eng.ctx.synchronize()
    assert torch.isnan(out[:, heads * dim:]).all()  # behind each row: left as it was
    return out[:, :heads * dim].cpu(), ls.cpu()


def expect(c, q, heads, window=0, scale=None):
    """(out, lse, bound of out, bound of lse) in 64 bits."""
    dim, group = c.dim, heads // c.kvh
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out = torch.zeros(len(c.lens_l), heads, dim, dtype=torch.float64)
    lse = torch.full((len(c.lens_l), heads), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros(len(c.lens_l), heads, dtype=torch.float64)
    for b, n in enumerate(c.lens_l):
        lo = max(0, n - window) if window else 0
        if n == 0:
            continue
        k, v = c.read(c.k, b, n)[lo:], c.read(c.v, b, n)[lo:]
        for h in range(heads):
            qq = q[b, h * dim:(h + 1) * dim].cpu().double()
            s = scale * (k[:, h // group] @ qq)
            m = s.max()
            p = torch.exp(s - m)
            out[b, h] = (p @ v[:, h // group]) / p.sum()
            lse[b, h] = m + p.sum().log()
            d = ((dim + 4) * U2 * abs(scale) * (k[:, h // group].abs() @ qq.abs())).max() + 8 * U2 * (s - m).abs().max()
            w = 2 * d + 2.0 ** -20 + 2 * (n - lo + 64) * U2
            tol[b, h] = w * (p @ v[:, h // group].abs()) / p.sum() + 1e-30
            ltol[b, h] = w + 4 * U2 * lse[b, h].abs()
    return out.reshape(len(c.lens_l), -1), lse, tol.reshape(len(c.lens_l), -1), ltol


def close(got, want, tol):
    got = got.double()
    bad = ~((got - want).abs() <= tol) & ~((got == want) & torch.isinf(want))
    assert not bad.any(), (int(bad.sum()), float((got - want)[bad].abs().max()))


def check_attend(eng, c, heads, seed=0, **kw):
    g = torch.Generator().manual_seed(100 + seed)
    q = torch.randn(max(1, len(c.lens_l)), heads * c.dim, generator=g).cuda()
    out, lse = attend(eng, c, q, heads, **kw)
    want, wl, tol, ltol = expect(c, q, heads, **kw)
    close(out, want, tol)
    close(lse, wl, ltol)
    return out


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,dim,page,lens,window", [
    (6, 6, 64, 16, [200], 0), (12, 12, 64, 16, [1, 0, 17, 16, 15, 1000, 64], 0), (8, 2, 128, 64, [0, 63, 64, 65, 700], 0),
    (8, 1, 32, 8, [3, 0, 0, 129], 0), (15, 5, 80, 24, [5, 24, 25, 333, 1], 100), (4, 4, 2, 1, [1, 2, 9, 70], 0),
    (3, 1, 96, 37, [36, 37, 38, 500], 37), (2, 2, 250, 5, [11, 301], 0), (7, 7, 6, 3, [40, 0, 1], 1),
    (16, 1, 256, 128, [1, 129, 400], 0), (5, 5, 12, 7, [100], 99), (10, 2, 72, 16, [257], 256), (32, 2, 48, 32, [90, 31], 0),
    (4, 2, 16, 16, [2000], 3000), (9, 3, 112, 40, [41, 39], 0), (24, 1, 64, 16, [333], 0)])
def test_attention(eng, dtype, heads, kvh, dim, page, lens, window):
    check_attend(eng, Cache(lens, kvh, dim, page, dtype, seed=dim), heads, window=window)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [8, 24, 88, 104, 120, 136, 200, 248])
def test_attention_head_dims(eng, dtype, dim):
    check_attend(eng, Cache([70, 0, 1, 200], 2, dim, 16, dtype, seed=dim), 2 * (1 + dim % 5))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [1, 2, 4, 7, 8, 12, 16, 33, 40, 1000])
@pytest.mark.parametrize("dim", [32, 128])
def test_attention_page_sizes(eng, dtype, page, dim):
    check_attend(eng, Cache([1, page, page + 1, 150, 0, 2 * page + 3], 2, dim, page, dtype, seed=page), 4)
    check_attend(eng, Cache([90, 333], 1, dim, page, dtype, seed=page), 3, window=45)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("batch,empty", [(1024, 0), (1025, 1), (3000, 7), (2049, 2)])
def test_attention_large_batches(eng, dtype, batch, empty):
    lens = [0 if empty and i % empty == 0 else 1 + (i * 37) % 60 for i in range(batch)]
    check_attend(eng, Cache(lens, 1, 16, 16, dtype, seed=batch), 2)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8, 9, 16, 17])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_groups(eng, dtype, group):
    check_attend(eng, Cache([300, 20], 2, 64, 16, dtype, seed=group), 2 * group)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,heads,kvh", [([30000], 8, 8), ([20001, 3, 9000, 0, 0, 12345], 4, 1), ([1] * 300, 4, 2),
                                            (list(range(0, 700, 7)), 2, 2)])
def test_attention_splits(eng, dtype, lens, heads, kvh):
    """Long contexts, many short ones and ragged batches: every way a length is cut and joined."""
    check_attend(eng, Cache(lens, kvh, 64, 32, dtype, seed=3), heads)


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("f16", 128), ("bf16", 64), ("bf16", 20), ("f32", 36)])
@pytest.mark.parametrize("order", ["slot", "pad"])
def test_attention_orders(eng, dtype, dim, order):
    check_attend(eng, Cache([100, 0, 37, 513], 2, dim, 16, dtype, order=order), 8)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_unaligned(eng, dtype):
    """Pointers and strides that no 16-byte access fits."""
    from turt_b200.runtime import make_paged_kv
    c = Cache([100, 37], 2, 64, 16, dtype)
    k, v = (torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda") for x in (c.k, c.v))
    k[1:], v[1:] = c.k, c.v
    size = 4 if dtype == "f32" else 2
    c.kv = make_paged_kv(k.data_ptr() + size, v.data_ptr() + size, c.table.data_ptr(), c.lens.data_ptr(), dtype,
                         c.n_pages, 16, 2, 64, 2, c.width)
    check_attend(eng, c, 8)
    c = Cache([100, 37], 2, 64, 16, dtype)
    q = torch.randn(2, 8 * 64 + 1, device="cuda")
    out, lse = attend(eng, c, q[:, 1:], 8)
    want, wl, tol, ltol = expect(c, q[:, 1:], 8)
    close(out, want, tol)


def test_attention_of_a_fused_projection(eng):
    """Queries read in place from [row][q | k | v], without lse."""
    c = Cache([100, 7, 300], 2, 64, 16, "bf16")
    qkv = torch.randn(3, (8 + 4) * 64, device="cuda")
    out, lse = attend(eng, c, qkv, 8, lse=False)
    want, _, tol, _ = expect(c, qkv, 8)
    close(out, want, tol)
    assert torch.isnan(lse).all()


def test_attention_scale_and_large_scores(eng):
    c = Cache([300, 40], 1, 64, 16, "f32")
    q = 30 * torch.randn(2, 4 * 64, device="cuda")
    for scale in (1.0, -0.5, 0.0):
        out, lse = attend(eng, c, q, 4, scale=scale)
        want, wl, tol, ltol = expect(c, q, 4, scale=scale)
        close(out, want, tol)
        close(lse, wl, ltol)


@pytest.mark.parametrize("dtype,heads", [("f32", 2), ("bf16", 2), ("f16", 8), ("bf16", 16)])
def test_attention_infinities_and_nan(eng, dtype, heads):
    """A key at -infinity has no weight; all of them leave zeros; NaN and +infinity give NaN in their own heads only."""
    c = Cache([50, 50, 50, 50], 1, 64, 16, dtype)
    q = torch.ones(4, heads * 64, device="cuda")
    kv = c.view(c.k)
    at = c.table_cpu[:, 1].long()
    kv[at[0], 3] = -math.inf  # one position of sequence 0
    for page in range(4):
        kv[c.table_cpu[1, page].long()] = -math.inf  # all of sequence 1
    kv[at[2], 3, 0, 0] = math.nan
    kv[at[3], 3, 0, 0] = math.inf
    out, lse = attend(eng, c, q, heads)
    k, v = c.read(c.k, 0, 50)[:, 0], c.read(c.v, 0, 50)[:, 0]
    p = torch.softmax(k.sum(1) / 8, 0)
    close(out[0].view(heads, 64)[heads - 1], p @ v, 1e-4)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
    assert torch.isnan(out[2:]).all() and torch.isnan(lse[2]).all()


@pytest.mark.parametrize("dtype,dim,page", [("bf16", 64, 16), ("f32", 64, 8), ("bf16", 60, 16), ("f32", 6, 8), ("f16", 128, 8),
                                            ("bf16", 64, 4)])
def test_attention_garbage_behind_the_length(eng, dtype, dim, page):
    """NaN in the slots behind a sequence's end, in unused pages and in the window's past does not reach the result (the
    caches above are NaN there too); page numbers that are out of range outside the window are not read."""
    c = Cache([100, 61], 2, dim, page, dtype)
    c.table[0, :71 // page] = -1
    c.table[1, :32 // page] = 99999
    q = torch.randn(2, 4 * dim, device="cuda")
    out, lse = attend(eng, c, q, 4, window=29)
    want, wl, tol, ltol = expect(c, q, 4, window=29)
    close(out, want, tol)
    close(lse, wl, ltol)


@pytest.mark.parametrize("dtype,dim", [("f32", 6), ("bf16", 60), ("bf16", 64), ("f16", 128), ("f32", 128), ("f32", 200)])
@pytest.mark.parametrize("page", [3, 8, 16, 21, 64])
def test_attention_each_bad_page_is_reported(eng, dtype, dim, page):
    """A bad page anywhere in a sequence raises, its positions are left out, and the others count."""
    from turt_b200._lib import ERR_RANGE, TurtError
    c = Cache([200], 1, dim, page, dtype)
    q = torch.randn(1, 2 * dim, device="cuda")
    want = None
    for bad in sorted({0, 1, (200 - 1) // page // 2, (200 - 1) // page}):
        c.table.copy_(c.table_cpu)
        c.table[0, bad] = c.n_pages + bad
        out = torch.empty(1, 2 * dim, device="cuda")
        space = torch.zeros(eng.pagedAttentionWorkspace(c.kv, 2), dtype=torch.uint8, device="cuda")
        eng.pagedAttention(c.kv, q.data_ptr(), 2 * dim, out.data_ptr(), 2 * dim, 2, space.data_ptr(), space.numel())
        with pytest.raises(TurtError) as e:
            eng.ctx.synchronize()
        assert e.value.code == ERR_RANGE
        keep = torch.tensor([j for j in range(200) if j // page != bad])
        if len(keep):
            k, v = c.read(c.k, 0, 200)[keep, 0], c.read(c.v, 0, 200)[keep, 0]
            for h in range(2):
                p = torch.softmax(k @ q[0, h * dim:(h + 1) * dim].cpu().double() / math.sqrt(dim), 0)
                want = p @ v
                # the bound of expect(), at most (dim + 4) 2u 4 sqrt(dim) 5 and (200 + 64) 4u for values below 5
                close(out[0, h * dim:(h + 1) * dim].cpu(), want, 5 * (2 * (dim + 4) * U2 * 20 * math.sqrt(dim) + 600 * U2))
    assert want is not None


def test_attention_bad_pages_and_lengths(eng):
    from turt_b200._lib import ERR_RANGE, TurtError
    c = Cache([100, 61, 10], 2, 64, 16, "f32")
    q = torch.randn(3, 256, device="cuda")
    c.table[0, 2] = c.n_pages  # positions 32 .. 47 of sequence 0
    space = torch.zeros(eng.pagedAttentionWorkspace(c.kv, 4), dtype=torch.uint8, device="cuda")
    out = torch.empty(3, 256, device="cuda")
    args = (c.kv, q.data_ptr(), 256, out.data_ptr(), 256, 4, space.data_ptr(), space.numel())
    eng.pagedAttention(*args)
    with pytest.raises(TurtError) as e:
        eng.ctx.synchronize()
    assert e.value.code == ERR_RANGE and "page" in str(e.value)
    k, v = c.read(c.k, 0, 100), c.read(c.v, 0, 100)
    keep = torch.tensor([j for j in range(100) if j // 16 != 2])
    p = torch.softmax(k[keep, 0] @ q[0, :64].cpu().double() / 8, 0)
    close(out[0, :64].cpu(), p @ v[keep, 0], 1e-4)
    c.table[0, 2] = int(c.table_cpu[0, 2])
    c.lens[1] = c.width * 16 + 1
    eng.pagedAttention(*args)
    with pytest.raises(TurtError) as e:
        eng.ctx.synchronize()
    assert e.value.code == ERR_RANGE
    assert (out[1] == 0).all()
    c.lens[1] = 61
    eng.pagedAttention(*args)
    eng.ctx.synchronize()
    want, _, tol, _ = expect(c, q, 4)
    close(out.cpu(), want, tol)


def test_attention_offsets_past_32_bits(eng):
    """Pages 2^31 and more elements apart."""
    from turt_b200.runtime import make_paged_kv
    stride, page = (1 << 31) + 64, 16
    if torch.cuda.mem_get_info()[0] < 3 * stride * 2:
        pytest.skip("needs 13 GB of free device memory")
    buf = torch.empty(2 * stride + 2 * page * 64, dtype=torch.bfloat16, device="cuda")
    c = Cache([45], 1, 64, page, "bf16", extra=0)
    for i in range(3):
        at = i * stride
        buf[at:at + page * 64] = c.k[i * page * 64:(i + 1) * page * 64]
        buf[at + page * 64:at + 2 * page * 64] = c.v[i * page * 64:(i + 1) * page * 64]
    c.kv = make_paged_kv(buf.data_ptr(), buf.data_ptr() + 2 * page * 64, c.table.data_ptr(), c.lens.data_ptr(), "bf16", 3,
                         page, 1, 64, 1, c.width, stride, page * 64, 64)
    check_attend(eng, c, 4)
    # the append of position 44 goes through the same offsets
    row = torch.randn(1, 128, device="cuda")
    eng.pagedAppend(c.kv, row.data_ptr(), 128, row.data_ptr() + 256, 128, 1)
    eng.ctx.synchronize()
    at = int(c.table_cpu[0, 2]) * stride + (44 % page) * 64
    assert torch.equal(buf[at:at + 64], row[0, :64].bfloat16())
    assert torch.equal(buf[at + page * 64:at + page * 64 + 64], row[0, 64:].bfloat16())


def test_attention_equal_bits_and_shared_workspace(eng):
    """Equal calls give equal bits; one workspace serves calls of different sizes one after another."""
    a, b = Cache([5000, 1, 900], 2, 64, 16, "bf16", seed=1), Cache([70] * 40, 4, 128, 32, "f32", seed=2)
    qa, qb = torch.randn(3, 8 * 64, device="cuda"), torch.randn(40, 4 * 128, device="cuda")
    n = max(eng.pagedAttentionWorkspace(a.kv, 8), eng.pagedAttentionWorkspace(b.kv, 4))
    space = torch.zeros(n, dtype=torch.uint8, device="cuda")
    first = attend(eng, a, qa, 8, space=space)[0], attend(eng, b, qb, 4, space=space)[0]
    for _ in range(3):
        assert torch.equal(attend(eng, a, qa, 8, space=space)[0], first[0])
        assert torch.equal(attend(eng, b, qb, 4, space=space)[0], first[1])


def test_empty_batch(eng):
    c = Cache([5], 2, 64, 16, "f32")
    c.kv.batch = 0
    eng.pagedAttention(c.kv, None, 0, None, 0, 4, torch.zeros(1 << 20, dtype=torch.uint8, device="cuda").data_ptr(), 1 << 20)
    eng.pagedAppend(c.kv, None, 0, None, 0, 0)
    eng.ctx.synchronize()


# --------------------------------------------------------------------------------- append

def rotated(x, pos, rot, base):
    """x [n][head][dim] in float64, rotated at pos [n]; and the bound of the fp32 arithmetic."""
    y, tol = x.clone(), torch.zeros_like(x)
    for m in range(rot // 2):
        a = pos.double() * base ** (-2.0 * m / rot)
        c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
        x0, x1 = x[..., 2 * m], x[..., 2 * m + 1]
        y[..., 2 * m], y[..., 2 * m + 1] = x0 * c - x1 * s, x0 * s + x1 * c
        t = 2.0 ** -21 * (x0.abs() + x1.abs())
        tol[..., 2 * m], tol[..., 2 * m + 1] = t, t
    return y, tol


STEP = {"f32": (0.0, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}


def check_append(eng, lens, new, heads, kvh, dim, page, dtype, rot, base=1e4, order="head", tail=0, shift=0, in_place=False,
                 with_q=True):
    """new None: one row per sequence (idle ones take none); else how many rows each sequence brings, `tail` rows behind
    them.  shift: floats by which every input is moved off its alignment."""
    c = Cache(lens, kvh, dim, page, dtype, order=order, seed=5)
    before_k, before_v = c.k.cpu().clone(), c.v.cpu().clone()
    counts = [1 if n else 0 for n in lens] if new is None else new
    rows = len(lens) if new is None else sum(new) + tail
    wide = (heads + 2 * kvh) * dim
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(rows, wide + shift, generator=g).cuda()
    q_out = qkv if in_place else torch.full((rows, heads * dim + shift), 7.0).cuda()
    src = qkv.cpu().double()
    start = None
    if new is not None:
        start = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32).cuda()
    p, o = qkv.data_ptr() + 4 * shift, q_out.data_ptr() + 4 * shift
    eng.pagedAppend(c.kv, p + 4 * heads * dim, wide + shift, p + 4 * (heads + kvh) * dim, wide + shift, rows,
                    start=None if start is None else start.data_ptr(), q=p if with_q else None, qStride=wide + shift,
                    qOut=o if with_q else None, qOutStride=q_out.stride(0), nHead=heads, rotDim=rot, base=base)
    eng.ctx.synchronize()
    want_k, want_v = before_k.double(), before_v.double()
    tol_k, tol_v = torch.zeros_like(want_k), torch.zeros_like(want_v)
    rel, low = STEP[dtype]
    got_q = q_out.cpu().double()
    row = 0
    for b, n in enumerate(counts):
        if new is None:
            row = b
        r = torch.arange(row, row + n)
        row += n
        pos = torch.arange(lens[b] - n, lens[b])
        x = src[r][:, shift:].view(n, heads + 2 * kvh, dim)
        y, t = rotated(x[:, :heads + kvh], pos, rot, float(np.float32(base)))
        at = (c.table_cpu[b, pos // page].long(), pos % page)
        c.view(want_k)[at], c.view(tol_k)[at] = y[:, heads:], t[:, heads:] * 1.01 + y[:, heads:].abs() * rel + low
        c.view(want_v)[at], c.view(tol_v)[at] = x[:, heads + kvh:], x[:, heads + kvh:].abs() * rel + low
        if with_q:
            close(got_q[r][:, shift:shift + heads * dim], y[:, :heads].flatten(1), t[:, :heads].flatten(1))
    for got, want, tol in ((c.k, want_k, tol_k), (c.v, want_v, tol_v)):
        got = got.cpu().double()
        same = torch.isnan(want)
        assert torch.equal(torch.isnan(got), same)  # everything that no row went to is as it was
        close(got[~same], want[~same], tol[~same])
    left = [b for b, n in enumerate(counts) if n == 0] if new is None else list(range(sum(counts), rows))
    if not in_place:
        assert (q_out[left] == 7.0).all()
    else:
        assert torch.equal(q_out[left].cpu().double(), src[left])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,new,heads,kvh,dim,page,rot", [
    ([200], None, 6, 6, 64, 16, 64), ([1, 0, 17, 16, 0], None, 12, 12, 64, 16, 64), ([40, 7, 90], [40, 0, 9], 8, 2, 128, 32, 128),
    ([5, 1, 60, 61], [5, 1, 33, 2], 15, 5, 80, 24, 40), ([9, 3], None, 3, 1, 6, 1, 2), ([30, 30, 30], [0, 0, 0], 4, 4, 16, 8, 16),
    ([300], [299], 4, 2, 36, 37, 36), ([12, 13], [12, 1], 2, 2, 250, 5, 250), ([70, 1], [64, 1], 16, 1, 256, 64, 0)])
def test_append(eng, dtype, lens, new, heads, kvh, dim, page, rot):
    check_append(eng, lens, new, heads, kvh, dim, page, dtype, rot)


@pytest.mark.parametrize("order", ["slot", "pad"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_orders(eng, dtype, order):
    check_append(eng, [40, 7, 90], [40, 0, 9], 8, 2, 64, 16, dtype, 64, order=order)


def test_append_variants(eng):
    check_append(eng, [40, 7], [5, 7], 8, 2, 64, 16, "bf16", 64, tail=6)  # a padded batch of rows
    check_append(eng, [40, 7], [5, 7], 8, 2, 64, 16, "bf16", 64, shift=1)  # no 16-byte alignment
    check_append(eng, [40, 7], [5, 7], 8, 2, 64, 16, "f16", 32, in_place=True)
    check_append(eng, [40, 0, 7], None, 8, 2, 64, 16, "f32", 64, in_place=True)
    check_append(eng, [40, 7], [5, 7], 8, 2, 64, 16, "bf16", 64, with_q=False)
    check_append(eng, [90001, 130000], [3, 1], 2, 2, 64, 512, "f32", 64, base=5e5)  # far positions
    check_append(eng, list(range(1, 400)), None, 2, 2, 16, 8, "bf16", 16)
    check_append(eng, [3] * 1100, [(i * 7) % 4 for i in range(1100)], 2, 1, 8, 4, "f16", 8, tail=5)  # many prompts
    check_append(eng, [900, 901], [900, 700], 3, 3, 24, 16, "f32", 24)  # several rows to a block
    check_append(eng, [2000], [1999], 40, 8, 128, 16, "bf16", 64)


def test_append_bad_pages(eng):
    from turt_b200._lib import ERR_RANGE, TurtError
    c = Cache([40, 20, 5], 1, 16, 16, "f32")
    k0 = c.k.clone()
    c.table[0, 2] = c.n_pages  # position 39
    x = torch.randn(3, 48, device="cuda")
    q = torch.full((3, 16), 7.0, device="cuda")

    def call(rows=3, start=None):
        eng.pagedAppend(c.kv, x.data_ptr(), 48, x.data_ptr() + 64, 48, rows, start=start, q=x.data_ptr() + 128, qStride=48,
                        qOut=q.data_ptr(), qOutStride=16, nHead=1, rotDim=16)
    call()
    with pytest.raises(TurtError) as e:
        eng.ctx.synchronize()
    assert e.value.code == ERR_RANGE and "page" in str(e.value)
    assert (q[0] == 7).all() and not (q[1:] == 7).any()
    changed = (c.view(c.k) != c.view(k0)) & ~torch.isnan(c.view(c.k))
    assert changed.flatten(2).any(-1).sum() == 2  # the two good rows, and nothing else
    # more new rows than the sequence has positions: the two that would come before position 0 are left out
    c = Cache([1, 20, 5], 1, 16, 16, "f32")
    start = torch.tensor([0, 3, 3, 3], dtype=torch.int32, device="cuda")
    q.fill_(7.0)
    call(start=start.data_ptr())
    with pytest.raises(TurtError):
        eng.ctx.synchronize()
    assert (q[:2] == 7).all() and not (q[2] == 7).any()
    # a length beyond the page table
    c.lens[1] = c.width * 16 + 1
    call()
    with pytest.raises(TurtError):
        eng.ctx.synchronize()
    c.lens[1] = 20
    call()
    eng.ctx.synchronize()


# ---------------------------------------------------------------------------------- rules

def check_rules(eng, rows, vocab, seed=0, hist=(30, 20), biases=0, masks=None, pad=0, out_pad=None, shift=0, in_place=False,
                penalties=("repetition", "frequency", "presence"), made=True, special=False, bias_lists=None):
    from turt_b200.runtime import make_logit_rules
    rs = np.random.default_rng(seed)
    out_pad = pad if out_pad is None else out_pad
    ld, old = vocab + pad, vocab + out_pad
    x = torch.tensor(rs.standard_normal(rows * ld + shift) * 4, dtype=torch.float32)
    X = x[shift:].view(rows, ld)
    if special:
        X[:, ::5], X[:, 1::7], X[:, 2::11], X[:, 3::13] = math.nan, math.inf, -math.inf, -3.4e38
    x = x.cuda()
    y = x if in_place else torch.full((rows * old + shift,), 7.0, device="cuda")
    keep = {}

    def dev(a, dtype):
        t = torch.tensor(np.ascontiguousarray(a).astype(dtype)).cuda()
        keep[len(keep)] = t
        return t.data_ptr()
    kw, want = {}, X.double().clone()[:, :vocab]
    tol = want.abs()
    prompts = [rs.integers(0, vocab, rs.integers(0, hist[0] + 1)) for _ in range(rows)] if hist else []
    gens = [rs.integers(0, max(1, vocab // 3), rs.integers(0, hist[1] + 1)) for _ in range(rows)] if hist else []
    rep, fr, pr = (rs.uniform(lo, hi, rows).astype(np.float32) for lo, hi in ((0.7, 2), (-1, 1), (-1, 1)))
    if hist:
        ids = np.concatenate([np.concatenate([p, g]) for p, g in zip(prompts, gens)] or [[]])
        start = np.concatenate([[0], np.cumsum([len(p) + len(g) for p, g in zip(prompts, gens)])])
        kw.update(tokens=dev(np.concatenate([ids, [0]]), np.int32), token_start=dev(start, np.int32))
        if made:
            kw.update(generated_start=dev(start[:-1] + [len(p) for p in prompts], np.int32))
        for name, val in (("repetition", rep), ("frequency", fr), ("presence", pr)):
            if name in penalties:
                kw[name] = dev(val, np.float32)
        for r in range(rows):
            known = np.unique(np.concatenate([prompts[r], gens[r]])).astype(int)
            n = np.bincount(gens[r].astype(int), minlength=vocab).astype(np.float64) if made else np.zeros(vocab)
            z = want[r, known]
            if "repetition" in penalties:
                want[r, known] = torch.where(z > 0, z / float(rep[r]), z * float(rep[r]))
            tol[r] = torch.maximum(tol[r], want[r].abs())
            for name, val in (("frequency", float(fr[r]) * n), ("presence", float(pr[r]) * (n > 0))):
                if name in penalties:
                    want[r] -= torch.tensor(val)
                    tol[r] += torch.tensor(np.abs(val))
    lists = bias_lists or ([np.sort(rs.choice(vocab, min(biases, vocab), replace=False)) if r != 1 else np.zeros(0, int)
                            for r in range(rows)] if biases else None)
    if lists:
        val = rs.standard_normal(sum(len(b) for b in lists)) * 5
        val = val.astype(np.float32)
        bstart = np.concatenate([[0], np.cumsum([len(b) for b in lists])])
        kw.update(bias_ids=dev(np.concatenate(lists + [[0]]), np.int32), bias=dev(np.append(val, 0), np.float32),
                  bias_start=dev(bstart, np.int32))
        for r in range(rows):
            v = torch.tensor(val[bstart[r]:bstart[r + 1]]).double()
            want[r, lists[r].astype(int)] += v
            tol[r, lists[r].astype(int)] += v.abs()
    if masks is not None:
        n_masks = max(1, rows - 1)
        bits = rs.random((n_masks, (vocab + 31) // 32 * 32)) < rs.choice([0.0, 0.01, 0.5, 1.0], (n_masks, 1))
        words = (bits.reshape(n_masks, -1, 32) * (1 << np.arange(32, dtype=np.uint64))).sum(-1).astype(np.uint32).view(np.int32)
        if masks == "rows":
            owner = rs.integers(-1, n_masks, rows)
            kw.update(mask_row=dev(owner, np.int32))
        else:
            owner = np.zeros(rows, int)
            assert n_masks >= rows
        kw.update(mask=dev(words, np.int32), n_masks=n_masks)
        for r in range(rows):
            if owner[r] >= 0:
                want[r, ~torch.tensor(bits[owner[r], :vocab])] = -math.inf
    eng.logitRules(x.data_ptr() + 4 * shift, ld, y.data_ptr() + 4 * shift, old, rows, vocab, make_logit_rules(**kw))
    eng.ctx.synchronize()
    got = y[shift:].view(rows, ld if in_place else old).cpu()
    if not in_place:
        assert (got[:, vocab:] == 7.0).all()
    got = got[:, :vocab].double()
    # fp32 rounds magnitudes from 2^128 (1 - 2^-25) on to infinity
    want = torch.where(want.abs() >= 2.0 ** 128 * (1 - 2.0 ** -25), torch.sign(want) * math.inf, want)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fine = ~nan & ~inf
    close(got[fine], want[fine], (6 * 2.0 ** -24 * tol + 1e-37)[fine])
    return got


@pytest.mark.parametrize("rows,vocab", [(1, 8192), (3, 1), (2, 2), (5, 31), (4, 33), (2, 4095), (2, 4096), (2, 4097), (7, 50001),
                                        (33, 12345), (1, 128000)])
def test_rules(eng, rows, vocab):
    check_rules(eng, rows, vocab, biases=9, masks="rows")


@pytest.mark.parametrize("kw", [
    dict(hist=None), dict(hist=None, biases=40), dict(hist=None, masks="rows"), dict(hist=(0, 50)), dict(hist=(50, 0)),
    dict(hist=(20000, 9000), biases=2000), dict(made=False), dict(penalties=("repetition",)), dict(penalties=("frequency",)),
    dict(penalties=("presence",)), dict(penalties=()), dict(pad=3), dict(pad=4, out_pad=8), dict(pad=4, out_pad=5),
    dict(shift=1), dict(shift=3, pad=2, masks="rows", biases=5), dict(in_place=True, biases=5, masks="rows"),
    dict(special=True, biases=5, masks="rows")])
@pytest.mark.parametrize("rows,vocab", [(6, 10007), (310, 17001)])
def test_rules_variants(eng, kw, rows, vocab):
    """A few rows, and enough of them for the kernel of large batches (310 x 17001: three slices a row)."""
    check_rules(eng, rows, vocab, seed=4, **kw)


@pytest.mark.parametrize("rows,vocab", [(700, 7), (650, 8191), (601, 8192), (599, 8193), (300, 16385)])
def test_rules_of_large_batches(eng, rows, vocab):
    check_rules(eng, rows, vocab, seed=6, hist=(50, 30), biases=5, masks="rows")


def test_rules_of_very_large_vocabularies(eng):
    """More slices to a row than ids are sorted by."""
    check_rules(eng, 9, 600001, seed=7, hist=(3000, 2000), biases=700, masks="rows")


def test_rules_rows_without_ids_between(eng):
    """Rows with many ids, with none and with many again, one after another in the same block."""
    from turt_b200.runtime import make_logit_rules
    rows, vocab = 900, 6000
    rs = np.random.default_rng(8)
    lens = rs.choice([0, 0, 1, 500, 5000], rows)
    start = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32).cuda()
    ids = torch.tensor(rs.integers(0, vocab, int(start[-1])), dtype=torch.int32).cuda()
    rep = torch.full((rows,), 2.0, device="cuda")
    x = torch.randn(rows, vocab, device="cuda")
    y = torch.empty_like(x)
    eng.logitRules(x.data_ptr(), vocab, y.data_ptr(), vocab, rows, vocab,
                   make_logit_rules(tokens=ids.data_ptr(), token_start=start.data_ptr(), repetition=rep.data_ptr()))
    eng.ctx.synchronize()
    seen = torch.zeros(rows, vocab, dtype=torch.bool)
    row = np.repeat(np.arange(rows), lens)
    seen[torch.tensor(row), ids.cpu().long()] = True
    x = x.cpu()
    assert torch.equal(y.cpu(), torch.where(seen, torch.where(x > 0, x / 2, x * 2), x))


def test_rules_repeated_ids_count(eng):
    """The same id a hundred thousand times, in the prompt and generated."""
    from turt_b200.runtime import make_logit_rules
    n = 100000
    ids = torch.full((2 * n,), 5, dtype=torch.int32, device="cuda")
    x = torch.ones(1, 64, device="cuda")
    y = torch.empty_like(x)
    start, made = torch.tensor([0, 2 * n], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    f = torch.tensor([0.5], device="cuda")
    eng.logitRules(x.data_ptr(), 64, y.data_ptr(), 64, 1, 64,
                   make_logit_rules(tokens=ids.data_ptr(), token_start=start.data_ptr(), generated_start=made.data_ptr(),
                                    frequency=f.data_ptr()))
    eng.ctx.synchronize()
    assert y[0, 5].item() == 1 - 0.5 * n and (y[0, :5] == 1).all() and (y[0, 6:] == 1).all()


def test_rules_out_of_range(eng):
    from turt_b200._lib import ERR_RANGE, TurtError
    from turt_b200.runtime import make_logit_rules
    x = torch.ones(2, 100, device="cuda")
    y = torch.empty_like(x)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    rep = torch.tensor([2.0, 2.0], device="cuda")
    ids, start, bias = i32(5, 100, 7, -1), i32(0, 2, 4), torch.ones(4, device="cuda")
    mask, owner = i32(*[-1] * 4), i32(0, 1)
    for kw in (dict(tokens=ids.data_ptr(), token_start=start.data_ptr(), repetition=rep.data_ptr()),
               dict(bias_ids=ids.data_ptr(), bias=bias.data_ptr(), bias_start=start.data_ptr()),
               dict(bias_ids=i32(3, 3, 4, 2).data_ptr(), bias=bias.data_ptr(), bias_start=start.data_ptr()),
               dict(mask=mask.data_ptr(), mask_row=owner.data_ptr(), n_masks=1)):
        eng.logitRules(x.data_ptr(), 100, y.data_ptr(), 100, 2, 100, make_logit_rules(**kw))
        with pytest.raises(TurtError) as e:
            eng.ctx.synchronize()
        assert e.value.code == ERR_RANGE and "rule" in str(e.value)
    eng.logitRules(x.data_ptr(), 100, y.data_ptr(), 100, 2, 100, make_logit_rules())
    eng.ctx.synchronize()
    assert torch.equal(x, y)


# ------------------------------------------------------------------------ streams and graphs

def test_step_in_a_graph_with_new_lengths():
    """Append and attention captured once, replayed while lengths, page table and contents change; two graphs with a
    workspace each, replayed on two streams at a time; a context on a stream of its own."""
    from turt_b200.engine import GpuEngine
    heads, kvh, dim, page, batch = 8, 2, 64, 16, 5
    steps = []
    for which in range(2):
        e = GpuEngine.create(0)
        side = torch.cuda.Stream()
        e.ctx.set_stream(side.cuda_stream)
        c = Cache([400 + which] * batch, kvh, dim, page, "bf16", seed=which)
        qkv = torch.randn(batch, (heads + 2 * kvh) * dim, device="cuda")
        rot, out = torch.zeros(batch, heads * dim, device="cuda"), torch.zeros(batch, heads * dim, device="cuda")
        space = torch.zeros(e.pagedAttentionWorkspace(c.kv, heads), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            p, wide = qkv.data_ptr(), qkv.shape[1]
            e.pagedAppend(c.kv, p + 4 * heads * dim, wide, p + 4 * (heads + kvh) * dim, wide, batch, q=p, qStride=wide,
                          qOut=rot.data_ptr(), qOutStride=heads * dim, nHead=heads, rotDim=dim)
            e.pagedAttention(c.kv, rot.data_ptr(), heads * dim, out.data_ptr(), heads * dim, heads, space.data_ptr(),
                             space.numel())
        steps.append((e, side, c, qkv, rot, out, space, g))
    for lens in ([1, 2, 300, 0, 17], [399, 16, 0, 1, 80], [3, 3, 3, 3, 3]):
        for e, side, c, qkv, rot, out, space, g in steps:
            c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
            c.lens_l = lens
            qkv.normal_()
            out.fill_(math.nan)
        torch.cuda.synchronize()
        for _ in range(3):
            for e, side, c, qkv, rot, out, space, g in steps:
                with torch.cuda.stream(side):
                    g.replay()
        torch.cuda.synchronize()
        for e, side, c, qkv, rot, out, space, g in steps:
            e.ctx.synchronize()
            want, _, tol, _ = expect(c, rot, heads)
            live = torch.tensor([n > 0 for n in lens])
            close(out.cpu()[live], want[live], tol[live])
            assert (out.cpu()[~live] == 0).all()
    for s in steps:
        s[0].ctx.close()
