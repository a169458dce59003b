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
