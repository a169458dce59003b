"""Rules on logits where it can go wrong: bias ids out of order."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from test_gpu_serving import eng  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab", [(7, 10007), (310, 17001), (601, 8192)])
@pytest.mark.parametrize("penalties", [True, False])
@pytest.mark.parametrize("in_place", [False, True])
def test_bias_ids_out_of_order(eng, rows, vocab, penalties, in_place):
    """Rows whose bias ids come twice, side by side or apart, or fall, take none of their biases; the others, and the
    penalties of all rows, are as always (vocab 10007: one block per slice, 17001 and 8192: the pipeline)."""
    from turt_b200._lib import ERR_RANGE, TurtError
    from turt_b200.runtime import make_logit_rules
    rs = np.random.default_rng(rows)
    dev = lambda a, t: torch.tensor(np.asarray(a).astype(t)).cuda()  # noqa: E731
    lists, orderly = [], []
    for r in range(rows):
        ids = np.sort(rs.choice(vocab, 40, replace=False))
        if r % 3 == 1:
            ids[20] = ids[19]
        elif r % 3 == 2:
            ids[37] = ids[3]
        lists.append(ids)
        orderly.append(r % 3 == 0)
    val = (4 * rs.standard_normal(40 * rows)).astype(np.float32)
    # every second id of the biases is known, so that counts and biases meet
    known = [np.concatenate([lists[r][::2], rs.integers(0, vocab, 30)]) for r in range(rows)]
    x = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(rows)).cuda()
    want = x.cpu().double()
    bufs = dict(bias_ids=dev(np.concatenate(lists), np.int32), bias=dev(val, np.float32),
                bias_start=dev(40 * np.arange(rows + 1), np.int32))
    if penalties:
        start = 50 * np.arange(rows + 1)
        bufs.update(tokens=dev(np.concatenate(known), np.int32), token_start=dev(start, np.int32),
                    generated_start=dev(start[:-1] + 10, np.int32), frequency=dev(np.full(rows, 0.25), np.float32))
        for r in range(rows):
            want[r] -= torch.tensor(0.25 * np.bincount(known[r][10:], minlength=vocab))
    for r in range(rows):
        if orderly[r]:
            want[r, lists[r]] += torch.tensor(val[40 * r:40 * r + 40]).double()
    y = x if in_place else torch.empty_like(x)
    eng.logitRules(x.data_ptr(), vocab, y.data_ptr(), vocab, rows, vocab,
                   make_logit_rules(**{k: v.data_ptr() for k, v in bufs.items()}))
    with pytest.raises(TurtError) as e:
        eng.ctx.synchronize()
    assert e.value.code == ERR_RANGE and "rule" in str(e.value)
    # two roundings of values below 64
    assert (y.cpu().double() - want).abs().max() <= 2 * 64 * 2.0 ** -24
    # nothing is left behind for the next call
    z = torch.empty_like(y)
    eng.logitRules(y.data_ptr(), vocab, z.data_ptr(), vocab, rows, vocab, make_logit_rules())
    eng.ctx.synchronize()
    assert torch.equal(y, z)
