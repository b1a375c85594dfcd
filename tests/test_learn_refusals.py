"""Refusals of include/omk_learn.h beyond those of test_learn_host.py, without a GPU: each before anything is enqueued."""

from tests.test_learn_host import INVALID, address, handle, preference  # noqa: F401  (handle: a fixture)

def test_gradients_are_looked_at_without_pairs(handle):  # noqa: F811
    for change in (dict(grad_stride=224), dict(d_grad=address(3) + 1), dict(d_grad=address(0) + 4)):
        assert preference(handle, out=dict(zero_rest=1, **change), pairs=0) == INVALID, change
