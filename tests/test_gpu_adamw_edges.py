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


@pytest.mark.parametrize("states", ["f32", "f8"])
def test_a_state_is_taken_over_whole_or_not_at_all(learner, states):
    import omoknuni_small_amd as omk
    p = torch.ones(300, device="cuda")
    opt = omk.AdamW(learner, [p], states=states)
    opt.step([p.clone()], lr=0.1)
    before = {name: x.clone().view(torch.uint8) for name, x in opt.state().items()}
    other = {name: torch.zeros_like(x) for name, x in opt.state().items()}
    for steps in (-1, 1 << 31, (1 << 64) + 5):
        with pytest.raises(omk.OmkError, match="steps"):
            opt.load_state(steps=steps, **other)
    assert opt.steps() == 1
    assert all(torch.equal(before[name], x.view(torch.uint8)) for name, x in opt.state().items())
    opt.load_state(steps=7, **other)
    assert opt.steps() == 7 and all((x.view(torch.uint8) == 0).all() for x in opt.state().values())
