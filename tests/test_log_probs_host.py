"""CPU: log_probs answers and refuses what its kernels answer and refuse."""
import pytest
import torch

from multiagentperception_amd import loss
from multiagentperception_amd._native import W2CError


@pytest.mark.parametrize("shape,dim,target", [((4, 16), -1, (3,)), ((4, 16), -1, (4, 1)), ((4, 16), -1, ()), ((2, 5, 3, 4), 1, (2, 3, 3)), ((2, 5, 3, 4), 1, (2, 5, 3))])
def test_a_target_of_another_shape_is_refused(shape, dim, target):
    with pytest.raises(W2CError, match="shape"):
        loss.log_probs(torch.randn(shape), torch.zeros(target, dtype=torch.int64), dim=dim)


@pytest.mark.parametrize("dim", [2, -3])
def test_a_dimension_that_is_not_there_is_refused(dim):
    with pytest.raises(W2CError, match="dim"):
        loss.log_probs(torch.randn(4, 16), dim=dim)


def test_a_target_outside_gives_its_row_no_number_for_a_gradient_and_an_ignored_one_none():
    x = torch.randn(5, 6, generator=torch.Generator().manual_seed(1)).requires_grad_()
    t = torch.tensor([0, 6, -100, -1, 5])
    r = loss.log_probs(x, t)
    r.logp.sum().backward()
    assert r.logp.isnan().tolist() == [False, True, False, True, False] and float(r.logp.detach()[2]) == 0.0
    assert x.grad.isnan().all(1).tolist() == [False, True, False, True, False] and not x.grad[2].any() and not x.grad[[0, 4]].isnan().any()
