"""The teacher's softmax of the top-logit distillation does not depend on a common shift of its logits, nor on
their size: offsets, rows of the lowest value, temperatures from small to large, against 64 bits.

Tolerances are those of test_top_logit_distill_gpu: p = exp((t - max) / tau) / sum takes the difference first, which
is exact to 2^-24 of itself, so |d| e^d keeps its rounding below 2^-23 of a row's p, whatever the logits' size.
At temperatures below 1/2 the student's exponents leave the range for which 2^-18 was derived (up to ~30): with
x = (max - z) / tau the kernel's exponent x log2 e is a difference, a constant log2 e / tau and a product, each rounded by
2^-24 of itself, so q = e^-x is off by 3 x 2^-24 of itself besides (x = 80: 1.4e-5 of a q of 1e-35); that is added."""

import pytest
import torch

from ossa_b200 import top_logit_distillation_loss
from test_top_logit_distill_gpu import DEV, FINE, _case, _check, _gen, _ref

pytestmark = pytest.mark.gpu
LOW = torch.finfo(torch.float32).min


@pytest.mark.parametrize("offset", [300.0, -300.0, 1e4, -1e4, 3e5, 1e30])
@pytest.mark.parametrize("tau", [0.5, 1.0, 3.0])
def test_offsets(offset, tau):
    z, t, ids = _case(torch.float32, (12,), 700, 64, seed=3)
    t = (torch.randn(12, 64, generator=_gen(9)) * 3).sort(dim=-1, descending=True).values + offset
    _check(z, t, ids, tau=tau)
    _check(z, t, ids, tau=tau, reduction="none")


@pytest.mark.parametrize("tau", [0.25, 0.5, 1.0, 4.0])
def test_lowest_and_largest(tau):
    """Rows whose entries are all the lowest value (each weighs 1 / K), all the largest, or both."""
    z, t, ids = _case(torch.float32, (5,), 400, 24, seed=4, holes=False)
    t[0] = LOW
    t[1] = -LOW
    t[2, ::2] = LOW
    t[3, 5] = -LOW
    t[4, 3:] = -float("inf")
    want, size, p, q, scale = _ref(z, t, ids, tau)
    leaf = z.to(DEV).requires_grad_()
    loss = top_logit_distillation_loss(leaf, t.to(DEV), ids.to(DEV), temperature=tau)
    assert abs(loss.item() - want.item()) <= FINE * size.item()
    dz = torch.autograd.grad(loss, leaf)[0].double().cpu()
    x = (z.double().amax(-1, keepdim=True) - z.double()) / tau
    ref = scale.unsqueeze(-1) * (q - p)
    bound = scale.unsqueeze(-1) * (FINE * (q + p) + 3 * 2.0 ** -24 * x * q) + 2.0 ** -24 * ref.abs() + 2.0 ** -126
    assert ((dz - ref).abs() <= bound).all()
    # each of the lowest or of the largest weighs the same
    assert torch.equal(p[0][ids[0]], torch.full((24,), 1 / 24, dtype=torch.float64))
    assert torch.equal(p[1][ids[1]], p[0][ids[0]])


@pytest.mark.parametrize("tau", [1e-3, 1e-10, 1e-30, 2.0 ** -126, 1e4, 1e15])
def test_temperatures(tau):
    """Small temperatures leave the teacher's largest entry alone, large ones weigh all alike."""
    z, t, ids = _case(torch.float32, (6,), 300, 16, seed=6)
    ids[:, 0] = torch.arange(6) + 1
    z = z * 0.5
    rows = top_logit_distillation_loss(z.to(DEV), t.to(DEV), ids.to(DEV), temperature=tau, reduction="none").double().cpu()
    zd, td = z.double(), t.double()
    ok = (ids >= 0) & (ids < 300)
    p = torch.softmax((td / tau).masked_fill(~ok, -float("inf")), -1)
    lq = torch.log_softmax(zd / tau, -1).gather(-1, ids.clamp(0, 299))
    lp = torch.log(p.clamp_min(1e-300))
    want = tau * tau * torch.where(p > 0, p * (lp - lq), 0.0).sum(-1)
    # each term is tau times a difference of logits, or tau^2 times a logarithm: 2^-18 of their sizes; what lies below
    # the normal range keeps absolute precision, tau times it
    size = tau * tau * torch.where(p > 0, p * (lp.abs() + lq.abs()), 0.0).sum(-1)
    assert ((rows - want).abs() <= 2.0 ** -18 * size + 2.0 ** -126).all(), (rows, want)
