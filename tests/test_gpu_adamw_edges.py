"""AdamW's calls out of order and with what does not fit, and what torch is told of its writes."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

STATE = -6


@pytest.fixture(scope="module")
def learner():
    import omoknuni_small_amd as omk
    return omk.Learner()


def test_an_optimizer_outlives_its_learner(learner):
    """It only waits to be destroyed then: its other calls are refused."""
    import omoknuni_small_amd as omk
    from omoknuni_small_amd import learn
    own = omk.Learner()
    p = torch.ones(300, device="cuda")
    opt = omk.AdamW(own, [p])
    opt.step([p.clone()], lr=0.1)
    assert opt.steps() == 1
    own.close()
    lib, n = learn._library(), C.c_int64()
    assert lib.omk_adamw_set_steps(opt._h, 5) == STATE
    assert lib.omk_adamw_get_steps(opt._h, C.byref(n)) == STATE
    assert lib.omk_adamw_step(opt._h, (C.c_void_p * 1)(p.data_ptr()), 0.1, None, None) == STATE
    opt.close()
