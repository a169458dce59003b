"""Device buffers of generation on the GPU: what a call took is back when it returns."""
import pytest

pytestmark = pytest.mark.gpu


def test_live_buffers_of_generate_under_rules():
    from oracle.oracle import Oracle
    from turt_b200.engine import GpuEngine
    from turt_b200.generate import generate
    from turt_b200.pretrain import Mulberry32
    from turt_b200.runtime import Model, make_config
    eng, orc = GpuEngine.create(0), Oracle()
    c = orc.cfg(60, 128, 2, 2, 32, "modern")
    m = Model(eng.ctx, make_config(60, 128, 2, 2, 32, "modern"))
    m.load_flat(orc.init(c, 1))
    live = None
    for _ in range(3):
        generate(m, [1, 2, 3], 60, rng=Mulberry32(5), repetition_penalty=1.2, bias={3: 1.0})
        assert live in (None, eng.liveBuffers)
        live = eng.liveBuffers
    m.close()
    eng.ctx.close()
