"""rope_axes with its numbers given as tensors: the values at the time of the call count."""
import pytest
import torch

from pasa_b200 import ops

pytestmark = pytest.mark.gpu


def test_numbers_in_tensors(cuda_device):
    q = torch.randn(1, 2, 20, 32, device="cuda")
    theta = torch.tensor(100.0)
    for value in (100.0, 10000.0, 7.0):
        theta.fill_(value)
        assert torch.equal(ops.rope_axes(q, axes=(8, 8), grid=(4, 5), theta=theta),
                           ops.rope_axes(q, axes=(8, 8), grid=(4, 5), theta=value))
    pair, axes, grid, origin = torch.tensor([100.0, 50.0]), torch.tensor([8, 16]), torch.tensor([4, 5]), torch.tensor([1, 2])
    for i in range(3):
        pair.add_(10.0)
        origin.add_(1)
        assert torch.equal(ops.rope_axes(q, axes=list(axes), grid=list(grid), origin=list(origin), theta=list(pair)),
                           ops.rope_axes(q, axes=(8, 16), grid=(4, 5), origin=(2 + i, 3 + i),
                                         theta=(110.0 + 10 * i, 60.0 + 10 * i)))
