"""Operators that are differentiable once refuse a second derivative where it would not be zero, also when the
incoming gradient is a constant (a penalty on a gradient); where an operator is linear the second is zero."""

import pytest
import torch

from ossa_b200 import qk_norm_rope, rope_to_heads, top_logit_distillation_loss, topk_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _calls():
    g = _gen(31)
    q, k, v = (torch.randn(1, 2, 20, 64, generator=g).to(DEV).requires_grad_() for _ in range(3))
    slopes = torch.rand(2, generator=g).to(DEV).requires_grad_()
    idx = torch.randint(0, 20, (1, 2, 20, 4), generator=g).to(DEV)
    x, y = (torch.randn(1, 5, 2 * 64, generator=g).to(DEV).requires_grad_() for _ in range(2))
    w = torch.rand(64, generator=g).to(DEV).requires_grad_()
    z = torch.randn(6, 50, generator=g).to(DEV).requires_grad_()
    ids = torch.rand(6, 50, generator=g).topk(3, dim=-1).indices.to(DEV)
    t = torch.randn(6, 3, generator=g).to(DEV)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2).detach().requires_grad_()
    return {"q": (q, lambda: topk_attention(q, k, v, topk_indices=idx)),
            "k": (k, lambda: topk_attention(q.detach(), k, v.detach(), topk_indices=idx, softcap=3.0)),
            "strided q": (turned, lambda: topk_attention(turned, k.detach(), v.detach(), topk_indices=idx)),
            "slopes": (slopes, lambda: topk_attention(q.detach(), k.detach(), v.detach(), topk_indices=idx, slopes=slopes)),
            "norm x": (x, lambda: qk_norm_rope(x, y, 2, 2, w, w)[0]),
            "norm y": (y, lambda: qk_norm_rope(x, y, 2, 2, None, w.detach())[1]),
            "norm w": (w, lambda: qk_norm_rope(x, y, 2, 2, w, w)[1]),
            "logits": (z, lambda: top_logit_distillation_loss(z, t, ids)),
            "rows": (z, lambda: top_logit_distillation_loss(z, t, ids, reduction="none"))}


@pytest.mark.parametrize("name", ["q", "k", "strided q", "slopes", "norm x", "norm y", "norm w", "logits", "rows"])
def test_refused(name):
    leaf, call = _calls()[name]
    (plain,) = torch.autograd.grad(call().sum(), leaf)
    (first,) = torch.autograd.grad(call().sum(), leaf, create_graph=True)
    assert torch.equal(first.detach(), plain)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        (first.square().sum() + leaf.sum()).backward()


def test_linear_operators():
    """The gradient of a linear operator does not depend on its input: nothing to refuse."""
    g = _gen(7)
    x, y = (torch.randn(1, 5, 2 * 64, generator=g).to(DEV).requires_grad_() for _ in range(2))
    w = torch.rand(64, generator=g).to(DEV).requires_grad_()
    for call, leaf in ((lambda: rope_to_heads(x, 2), x), (lambda: qk_norm_rope(x, y, 2, 2)[1], y),
                       (lambda: qk_norm_rope(x.detach(), y.detach(), 2, 2, w)[0], w)):
        (first,) = torch.autograd.grad(call().sum(), leaf, create_graph=True)
        assert not first.requires_grad


def test_a_graph_of_the_first_derivative_alone():
    """create_graph without a second backward pass gives the gradients it gave."""
    for name, (leaf, call) in _calls().items():
        leaf.grad = None
        call().sum().backward(create_graph=True)
        (plain,) = torch.autograd.grad(call().sum(), leaf)
        assert torch.equal(leaf.grad.detach(), plain), name
        leaf.grad = None
