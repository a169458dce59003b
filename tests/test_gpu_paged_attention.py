"""Paged attention where it can go wrong: head sizes crossed with the ways a sequence is cut and joined, inputs
whose elements differ much in size, values and keys that are not finite.

References and tolerances are test_gpu_serving's (64 bits; derived from the arithmetic) unless a test says
otherwise.
"""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_serving import Cache, attend, close, eng, expect  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kvh", [(2, 1, 1), (2, 2, 2), (4, 1, 1), (6, 1, 1), (2, 2, 1), (2, 3, 1), (8, 1, 1), (60, 4, 1),
                                           (250, 2, 2), (256, 5, 1)])
def test_head_sizes_and_splits(eng, dtype, dim, heads, kvh):
    """Sequences that two, three and many blocks share.  The workspace holds what a call of other sizes left."""
    lens = [600, 2000, 1] if dim < 60 else [2000]
    space = None
    for n in (lens, [30000 if dim < 60 else 9000]):
        c = Cache(n, kvh, dim, 16, dtype, seed=dim)
        need = max(eng.pagedAttentionWorkspace(c.kv, heads), 1 << 24)
        if space is None:
            space = torch.zeros(need, dtype=torch.uint8, device="cuda")
            other = Cache([20000], 1, 64, 16, "f32", seed=9)
            attend(eng, other, 1000 * torch.randn(1, 8 * 64, device="cuda"), 8, space=space)
        q = torch.randn(len(n), heads * dim, generator=torch.Generator().manual_seed(dim)).cuda()
        out, lse = attend(eng, c, q, heads, space=space)
        want, wl, tol, ltol = expect(c, q, heads)
        close(out, want, tol)
        close(lse, wl, ltol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ratio", [8, 15, 22, 28])
@pytest.mark.parametrize("dim,heads", [(16, 1), (64, 4), (128, 8)])
def test_an_outlier_in_q(eng, dtype, ratio, dim, heads):
    """One element of q 2^ratio times the others, over a key element of 0: it adds nothing to the bound of a score, which
    the other elements have to keep."""
    c = Cache([700, 20], 1, dim, 16, dtype, seed=ratio)
    c.view(c.k)[..., 5] = 0
    q = torch.randn(2, heads * dim, generator=torch.Generator().manual_seed(ratio)).cuda()
    q[:, 5::dim] = 2.0 ** ratio
    out, lse = attend(eng, c, q, heads)
    want, wl, tol, ltol = expect(c, q, heads)
    close(out, want, tol)
    close(lse, wl, ltol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gap", [8, 12, 16, 20])
@pytest.mark.parametrize("at", [0, 333, 999])
@pytest.mark.parametrize("dim,heads", [(32, 1), (64, 4), (128, 8)])
def test_a_dominant_key_without_value(eng, dtype, gap, at, dim, heads):
    """One position has nearly all of the weight and a value of 0; the output is what the others add, whose weights are
    e^-gap of it, and its bound is relative to that."""
    c = Cache([1000, at % 16 + 5], 1, dim, 16, dtype, seed=gap)
    k, v = c.view(c.k), c.view(c.v)
    g = torch.Generator().manual_seed(gap)
    q = torch.randn(2, heads * dim, generator=g).cuda()
    q[:, 0::dim] = math.sqrt(dim)
    for b, n in enumerate(c.lens_l):
        pages, slots = c._at(b, n)
        k[pages, slots] *= 2.0 ** -7  # scores next to 0 ..
        k[pages, slots, :, 0] = 0
        j = at % 16 if b else at
        k[pages[j], slots[j], :, 0] = gap  # .. and one of them at `gap`
        v[pages[j], slots[j]] = 0
    out, lse = attend(eng, c, q, heads)
    want, wl, tol, ltol = expect(c, q, heads)
    close(out, want, tol)
    close(lse, wl, ltol)


NARROW_AND_WIDE = [("f32", 16, 1), ("f32", 64, 3), ("f32", 128, 2), ("f32", 200, 4), ("f32", 60, 8), ("f32", 6, 2), ("f16", 64, 3),
                   ("f16", 200, 2), ("bf16", 128, 8), ("bf16", 136, 4), ("bf16", 60, 2)]


@pytest.mark.parametrize("dtype,dim,heads", NARROW_AND_WIDE)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_no_weight_whatever_the_value(eng, dtype, dim, heads, value):
    """Positions with a key at -infinity do not count, be their values infinite or NaN."""
    c = Cache([50, 700], 1, dim, 16, dtype, seed=dim)
    q = torch.rand(2, heads * dim, generator=torch.Generator().manual_seed(dim)).cuda() + 0.5
    out_at = {0: [3, 17, 49], 1: [0, 333, 334, 699]}
    for b, js in out_at.items():
        pages, slots = c._at(b, c.lens_l[b])
        for j in js:
            c.view(c.k)[pages[j], slots[j]] = -math.inf
            c.view(c.v)[pages[j], slots[j]] = value
    out, lse = attend(eng, c, q, heads)
    # the same sequences without these positions
    left = {b: [j for j in range(n) if j not in out_at[b]] for b, n in enumerate(c.lens_l)}
    d = Cache([len(left[0]), len(left[1])], 1, dim, 16, dtype)
    for src, dst in ((c.k, d.k), (c.v, d.v)):
        for b in left:
            pages, slots = c._at(b, c.lens_l[b])
            d.view(dst)[d._at(b, len(left[b]))] = c.view(src)[pages[left[b]], slots[left[b]]]
    want, wl, tol, ltol = expect(d, q, heads)
    close(out, want, tol)
    close(lse, wl, ltol)


@pytest.mark.parametrize("dtype,dim,heads", [x for x in NARROW_AND_WIDE if x[0] != "f16"])
@pytest.mark.parametrize("size", [1e34, 3e34, 1e35])
def test_values_near_the_largest(eng, dtype, dim, heads, size):
    """Values from 1e34 on under scores that rise and fall by 5 (2^7.2) from one 16 positions to the next: sums of 32 or
    256 of them at a weight of 2^7.2 are past fp32's range, sums of 256 at a weight of 1 are not."""
    c = Cache([512], 1, dim, 16, dtype, seed=dim)
    q = torch.zeros(1, heads * dim, device="cuda")
    q[:, 0::dim] = math.sqrt(dim)
    pages, slots = c._at(0, 512)
    c.view(c.k)[pages, slots] = 0
    c.view(c.k)[pages, slots, :, 0] = (5.0 * ((torch.arange(512) // 16) % 2))[:, None].to(c.k)
    c.view(c.v)[pages, slots] = (c.view(c.v)[pages, slots].abs() + 1) * size
    out, lse = attend(eng, c, q, heads)
    want, wl, tol, ltol = expect(c, q, heads)
    close(out, want, tol)
    close(lse, wl, ltol)


@pytest.mark.parametrize("dtype,dim,heads", NARROW_AND_WIDE)
@pytest.mark.parametrize("window", [0, 70])
def test_sequences_that_are_not_finite_among_others(eng, dtype, dim, heads, window):
    """NaN in some sequences of a ragged batch, several of them in a warp's stretch: the others do not notice."""
    lens = [(i * 37) % 120 for i in range(150)] + [900, 2500, 0, 1]
    c = Cache(lens, 1, dim, 16, dtype, seed=dim)
    bad = [b for b, n in enumerate(lens) if n and b % 7 == 3]
    for b in bad:
        pages, slots = c._at(b, lens[b])
        c.view(c.v if b % 2 else c.k)[pages[-1], slots[-1], :, 1] = math.nan
    q = torch.randn(len(lens), heads * dim, generator=torch.Generator().manual_seed(dim)).cuda()
    out, lse = attend(eng, c, q, heads, window=window)
    want, wl, tol, ltol = expect(c, q, heads, window=window)
    good = [b for b in range(len(lens)) if b not in bad]
    close(out[good], want[good], tol[good])
    close(lse[good], wl[good], ltol[good])
    assert torch.isnan(out.view(len(lens), heads, dim)[bad][..., 1]).all()
    again, _ = attend(eng, c, q, heads, window=window)
    assert torch.equal(again[good], out[good])


def test_more_tiles_than_32_bits_count(eng):
    """One sequence of nearly 2^31 positions and 80 key heads, 5.4e9 tiles of 32 positions.  All pages but the last three
    are one page whose scores lie 10^4 below, e^-10000 of the weight and 0 in fp32; the last three are others, so the
    output is theirs alone."""
    from turt_b200.runtime import make_paged_kv
    kvh, dim, page = 80, 8, 4096
    width = (1 << 31) // page - 1
    g = torch.Generator().manual_seed(4)
    k = torch.randn(4, kvh, page, dim, generator=g).bfloat16()
    v = torch.randn(4, kvh, page, dim, generator=g).bfloat16()
    q = torch.randn(1, kvh * dim, generator=g)
    q[:, 0::dim] = math.sqrt(dim)
    k[..., 0] = 0
    k[0, ..., 0] = -10000
    table = torch.zeros(1, width, dtype=torch.int32)
    table[0, -3:] = torch.tensor([2, 1, 3])
    n = width * page - 100
    k_, v_, q_, t_ = k.cuda(), v.cuda(), q.cuda(), table.cuda()
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    kv = make_paged_kv(k_.data_ptr(), v_.data_ptr(), t_.data_ptr(), lens.data_ptr(), "bf16", 4, page, kvh, dim, 1, width)
    out = torch.full((1, kvh * dim), math.nan, device="cuda")
    space = torch.zeros(eng.pagedAttentionWorkspace(kv, kvh), dtype=torch.uint8, device="cuda")
    eng.pagedAttention(kv, q_.data_ptr(), kvh * dim, out.data_ptr(), kvh * dim, kvh, space.data_ptr(), space.numel())
    eng.ctx.synchronize()
    kk, vv = (x[[2, 1, 3]].transpose(1, 2).reshape(3 * page, kvh, dim)[:3 * page - 100].double() for x in (k, v))
    qq = q.double().view(kvh, dim)
    s = torch.einsum("nhd,hd->nh", kk, qq) / math.sqrt(dim)
    p = torch.softmax(s, 0)
    want = torch.einsum("nh,nhd->hd", p, vv).reshape(1, -1)
    # expect()'s bound with the positions that have a weight
    d = ((dim + 4) * 2.0 ** -23 / math.sqrt(dim) * torch.einsum("nhd,hd->nh", kk.abs(), qq.abs())).amax(0)
    d = d + 8 * 2.0 ** -23 * (s.amax(0) - s.amin(0))
    w = 2 * d + 2.0 ** -20 + 2 * (3 * page + 64) * 2.0 ** -23
    close(out.cpu(), want, (w[:, None] * torch.einsum("nh,nhd->hd", p, vv.abs())).reshape(1, -1))
