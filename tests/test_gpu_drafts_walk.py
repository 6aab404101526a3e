"""The walk through drafted tokens: requests that begin outside of them."""
import pytest
import torch

from easy_gpt.cpp_amd import kernels

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("far", [-1, -(2 ** 31), 3, 4, 2 ** 31 - 1])
def test_a_request_that_begins_nowhere_has_no_tokens(far):
    path, count, accepted = kernels.backend().accept_drafts(i32([1, 2, 3]), i32([-1, 0, 1]), i32([2, 3, 9]), i32([far, 0]), i32([3, 3]))
    assert count.tolist() == [0, 3]
    assert bool((path[0] == -1).all()) and bool((accepted[0] == -1).all())
    assert path[1].tolist() == [0, 1, 2] + [-1] * 61 and accepted[1].tolist() == [2, 3, 9] + [-1] * 61
