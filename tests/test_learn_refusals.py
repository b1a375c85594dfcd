"""Refusals of include/omk_learn.h beyond those of test_learn_host.py, without a GPU: each before anything is enqueued."""
import ctypes as C

import pytest

from omoknuni_small_amd import learn
from tests.test_learn_host import INVALID, address, handle, message, policy, preference, rows  # noqa: F401  (handle: a fixture)


def test_gradients_are_looked_at_without_pairs(handle):  # noqa: F811
    for change in (dict(grad_stride=224), dict(d_grad=address(3) + 1), dict(d_grad=address(0) + 4)):
        assert preference(handle, out=dict(zero_rest=1, **change), pairs=0) == INVALID, change


def across(rc):
    return rc == INVALID and "across" in message()


LOGITS, LEGAL = 8 * 225 * 2, 8 * 8 * 4  # bytes of what rows() gives


def test_priors_and_log_probabilities_lie_apart(handle):  # noqa: F811
    lib, r = learn._library(), rows()
    priors = lambda at, work=None, n=0: lib.omk_policy_priors(handle, C.byref(r), at, 225, work, n)  # noqa: E731
    for at in (address(1), address(1) + LEGAL - 4, address(1) - 8 * 225 * 4 + 4):
        assert across(priors(at)), hex(at)
    logprobs = lambda moves, lp, ent: lib.omk_policy_logprobs(handle, C.byref(r), moves, lp, ent, None, 0)  # noqa: E731
    for n, size in ((0, LOGITS), (1, LEGAL), (5, 32)):
        for at in (address(n), address(n) + size - 4, address(n) - 28):
            assert across(logprobs(address(5), at, None)), (n, at)
            assert across(logprobs(address(5), address(2), at)), (n, at)
    assert across(logprobs(address(5), address(2), address(2) + 28))
    wide = rows(actions=100000, row_stride=100000, d_legal=None)
    need = lib.omk_policy_work(8, 100000)
    for work in (address(0), address(2)):
        assert across(lib.omk_policy_logprobs(handle, C.byref(wide), address(5), address(2), None, work, need))
    assert across(lib.omk_policy_priors(handle, C.byref(wide), address(3), 100000, address(3) + 16, need))


def test_results_of_the_losses_lie_apart(handle):  # noqa: F811
    for n, size in ((0, LOGITS), (1, LEGAL), (5, 32), (6, 32), (7, 32), (8, 32), (9, 32)):
        for name in ("d_loss", "d_logprob", "d_kl"):
            for at in (address(n), address(n) + size - 4):
                assert across(policy(handle, out={name: at}, samples=dict(d_weight=address(9)))), (n, name)
        if n:
            assert across(policy(handle, out=dict(d_grad=address(n)), samples=dict(d_weight=address(9)))), n
    for out in (dict(d_loss=address(4) + 28), dict(d_kl=address(4) - 28), dict(d_loss=address(3) + 4), dict(d_logprob=address(3) + LOGITS - 4),
                dict(d_kl=address(2)), dict(d_logprob=address(11) + 32), dict(d_grad=address(11) - LOGITS + 4)):
        assert across(policy(handle, out=out)), out
    for n, size in ((0, LOGITS), (1, LEGAL), (5, 32), (6, 28)):
        for name in ("d_loss", "d_margin", "d_line_logprob"):
            for at in (address(n), address(n) + size - 4):
                assert across(preference(handle, out={name: at})), (n, name)
        if n:
            assert across(preference(handle, out=dict(d_grad=address(n)))), n
    for out in (dict(d_margin=address(3)), dict(d_loss=address(3)), dict(d_margin=address(4), d_line_logprob=address(4) + 8),
                dict(d_margin=address(11)), dict(d_line_logprob=address(11) + 16)):
        assert across(preference(handle, out=out)), out


def test_what_lies_between_rows_is_free(handle):  # noqa: F811
    """Rows of 225 bf16 with 31 behind each: a loss there is taken (these calls get as far as the device, which there is none of), one in
    a row is not."""
    r = rows(row_stride=256)
    for row in (0, 3, 7):
        begin = address(0) + row * 512
        assert across(policy(handle, out=dict(d_loss=begin + 448), r=r)) and across(policy(handle, out=dict(d_loss=begin), r=r))
        got = policy(handle, out=dict(d_loss=begin + 452), r=r)
        assert got not in (0, INVALID) and "across" not in message()


def test_masks_of_numbers():
    """Masks that are no truth values: what is not 0 is legal, whatever its size."""
    torch = pytest.importorskip("torch")
    mask = torch.rand(5, 70, generator=torch.Generator().manual_seed(1)) < 0.5
    want = learn.pack_legal(mask)
    for values in (mask.to(torch.uint8) * 255, mask.int() * 2, mask.long() * -7, mask.float() * 0.25, mask.half() * 3.5):
        assert torch.equal(learn.pack_legal(values), want), values.dtype


def test_results_lie_apart_without_pairs(handle):  # noqa: F811
    for at in (address(3), address(3) + LOGITS - 4, address(0), address(0) + LOGITS - 4):
        assert across(preference(handle, out=dict(d_loss=at, zero_rest=1), pairs=0)), hex(at)
