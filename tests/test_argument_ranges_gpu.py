"""Arguments at the ends of their ranges: prefix lengths past 32 bits, weights whose sum leaves the range of fp32."""

import pytest
import torch

from ossa_b200 import top_logit_distillation_loss, topk_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def test_prefix_lengths_past_32_bits():
    """An int64 length is compared as the number it is: past the last key it opens every key."""
    B, H, N, D, K = 4, 2, 30, 64, 9
    g = _gen(1)
    q, k, v = (torch.randn(B, H, N, D, generator=g).to(DEV) for _ in range(3))
    idx = torch.randint(0, N, (B, H, N, K), generator=g).to(DEV)
    lengths = torch.tensor([2 ** 31, 2 ** 40 + 3, -2 ** 40 + 5, 7])
    want = topk_attention(q, k, v, topk_indices=idx, prefix_len=torch.tensor([N, N, 0, 7], device=DEV))
    assert torch.equal(topk_attention(q, k, v, topk_indices=idx, prefix_len=lengths.to(DEV)), want)
    assert torch.equal(want[0], topk_attention(q[:1], k[:1], v[:1], topk_indices=idx[:1], causal=False)[0])


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
