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


def test_torch_is_told_of_what_is_written(learner):
    """A weight, a copy or logits that change between a forward pass and its backward pass: the backward pass is refused, and
    gradients through what was not written are right."""
    import omoknuni_small_amd as omk
    gen = torch.Generator().manual_seed(2)
    flat = torch.randn(2 * 64, generator=gen).cuda()
    for make in (lambda: [torch.nn.Parameter(flat[:64].clone().view(8, 8)), torch.nn.Parameter(flat[64:].clone().view(8, 8))],
                 lambda: [x.view(8, 8) for x in flat.clone().split(64)]):
        for frozen in (False, True):
            params = make()
            copies = [p.detach().bfloat16() for p in params]
            opt = omk.AdamW(learner, params, copies=copies)
            x = torch.randn(4, 8, device="cuda", requires_grad=True)
            last = (x @ params[0] @ params[1]).sum()
            of_copies = (x.bfloat16() @ copies[1]).sum()
            grads = [torch.ones(8, 8, device="cuda"), None if frozen else torch.ones(8, 8, device="cuda")]
            versions = [p._version for p in params + copies]
            opt.step(grads, lr=0.1)
            assert params[0]._version > versions[0] and copies[0]._version > versions[2]
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                last.backward()
            if not frozen:
                with pytest.raises(RuntimeError, match="modified by an inplace"):
                    of_copies.backward()
            else:
                of_copies.backward()
                assert torch.equal(x.grad, (torch.ones(4, 8, device="cuda").bfloat16() @ copies[1].t()).float())
            (x @ params[0] @ params[1]).sum().backward()  # a new forward pass has the new weights
    w = torch.randn(8, 225, device="cuda", requires_grad=True)
    moves, f = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    begin = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    x = torch.randn(4, 8, device="cuda")
    for call in (lambda y, grad: learner.policy_loss(y, moves, f, f + 1, grad=grad), lambda y, grad: learner.preference_loss(y, moves, begin, grad=grad)):
        logits = x @ w
        again = (logits * logits).sum()  # saves the logits
        got = call(logits.detach(), True)
        given = torch.empty_like(got.grad)
        before = given._version
        call(logits.detach(), given)
        assert given._version > before and torch.equal(given, got.grad)
        call(logits.detach(), logits.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            again.backward()
        logits = x @ w
        got = call(logits.detach(), logits.detach())
        w.grad = None
        logits.backward(got.grad)  # the product has saved its operands, not the logits: its gradient is right
        assert torch.equal(w.grad, x.t() @ got.grad)
    out = torch.empty(4, 225, device="cuda")
    before = out._version
    learner.priors(x @ w.detach(), out=out)
    assert out._version > before


def test_tensors_made_in_inference_mode(learner):
    import omoknuni_small_amd as omk
    with torch.inference_mode():
        p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
        opt = omk.AdamW(learner, [p, torch.ones(600, device="cuda")[300:]], weight_decay=0.0)
        opt.step([g, g], lr=0.5)
        opt.step([g, None], lr=0.5)
        out = torch.empty(3, 300, device="cuda")
        learner.priors(torch.zeros(3, 300, device="cuda"), out=out)
        assert (p != 1).all() and opt.steps() == 2 and (out > 0).all()
