"""The device logits of the last prefill or step are there until another forward of the model."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_logits_until_another_forward():
    from oracle.oracle import Oracle
    from turt_b200._lib import ERR_INVALID, TurtError
    from turt_b200.runtime import Context, Model, make_config
    orc, ctx = Oracle(), Context(0)
    m = Model(ctx, make_config(60, 32, 2, 2, 32, "modern"))
    m.load_flat(orc.init(orc.cfg(60, 32, 2, 2, 32, "modern"), 1))
    ids = np.arange(4 * 32, dtype=np.int32) % 60
    try:
        for other in (lambda: m.forward(ids, ids, 4, 32), lambda: m.forward_backward(ids[:64], ids[:64], 2, 32)):  # larger, then smaller
            for run in (lambda: m.generate_prefill([1, 2, 3]), lambda: m.generate_step(4, 3)):
                want = run()
                assert np.array_equal(ctx.download(m.generate_logits(), 60), want)
            m.generate_prefill([1, 2, 3])
            other()
            with pytest.raises(TurtError) as e:
                m.generate_logits()
            assert e.value.code == ERR_INVALID
    finally:
        m.close()
        ctx.close()
