"""Arguments at the ends of their ranges: weights whose sum leaves the range of fp32."""

import pytest
import torch

from ossa_b200 import top_logit_distillation_loss

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("scale", [2.0 ** -138, 2.0 ** 125])
@pytest.mark.parametrize("upstream", [1.0, -0.75])
def test_weights_of_any_size(scale, upstream):
    """The mean does not change when all weights are scaled, be their sum below 1 / FLT_MAX or above FLT_MAX.  The
    scaled weights are multiples of 2^-8 times the scale, exact in fp32; the mean's unit is rounded once either way."""
    T, V, K = 40, 500, 8
    g = _gen(2)
    z = torch.randn(T, V, generator=g).to(DEV).requires_grad_()
    ids = torch.rand(T, V, generator=g).topk(K, dim=-1).indices.to(DEV)
    t = torch.randn(T, K, generator=g).to(DEV)
    w = (torch.randint(0, 256, (T,), generator=g).float() / 256).to(DEV)

    def run(weight):
        loss = top_logit_distillation_loss(z, t, ids, row_weight=weight)
        return loss.detach(), torch.autograd.grad(loss, z, torch.tensor(upstream, device=DEV))[0]

    loss, dz = run(w)
    got, dgot = run(w * scale)
    assert abs(got.item() - loss.item()) <= 2.0 ** -22 * abs(loss.item())
    assert ((dgot - dz).abs() <= 2.0 ** -22 * dz.abs() + 2.0 ** -126).all()
