"""The differentiable decoder operators on the GPU: what torch's differentiation may ask of them."""
import pytest
import torch

from tdgs_amd import appearance, decoder

pytestmark = pytest.mark.gpu


def test_gradient_penalty_raises(gpu):
    """The image reaches the corrected one by the operators and past them: a penalty on its gradient would lack the operators'
    part. The first derivative is the same with and without a graph."""
    dec = appearance.AppearanceDecoder(2, channels=32, groups=4)
    rgb = torch.rand((17, 9, 3), generator=torch.Generator().manual_seed(0)).cuda().requires_grad_(True)
    want, = torch.autograd.grad((dec(rgb, 1) ** 2).sum(), rgb)
    got, = torch.autograd.grad((dec(rgb, 1) ** 2).sum(), rgb, create_graph=True)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="differentiated again"):
        got.pow(2).sum().backward()
