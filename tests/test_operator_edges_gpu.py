"""Training calls at their edges: gradients and inputs off 16-byte boundaries, saved tensors that come back in
another layout, rows that are not finite beside rows that are, lists in any order."""

import pytest
import torch

from mod_attention_ref import attention, rel, score_step
from ossa_b200 import qk_norm_rope, rope_to_heads, top_logit_distillation_loss, topk_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
STEP = 2.0 ** -8


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distillation_of_offloaded_slices(dtype, reduction):
    """Logits that are a slice of a larger tensor, saved by a hook that packs them: the backward pass reads
    them in the layout in which they come back."""
    g = _gen(3)
    B, N, V, K = 3, 9, 333, 7
    whole = (torch.randn(B, N, V, generator=g) * 2).to(dtype).to(DEV).requires_grad_()
    ids = torch.rand(B, N - 1, V, generator=g).topk(K, dim=-1).indices.to(DEV)
    teacher = torch.randn(B, N - 1, K, generator=g).to(DEV)
    dl = torch.rand((B, N - 1) if reduction == "none" else (), generator=g).to(DEV) + 1.5  # not 1: computed anew

    def run():
        loss = top_logit_distillation_loss(whole[:, :-1], teacher, ids, temperature=2.0, reduction=reduction)
        return torch.autograd.grad(loss, whole, dl)[0]

    want = run()
    with torch.autograd.graph.save_on_cpu():
        got = run()
    # Not the same bits: a row of 333 values begins elsewhere between 16-byte boundaries in the packed copy, and its
    # sum is split at those.  Either result is within 2^-18 (softmax + p) scale and half a step of the gradient.
    z = whole.detach()[:, :-1].double()
    p = torch.zeros_like(z).scatter_add_(-1, ids, torch.softmax(teacher.double() / 2.0, -1))
    scale = 2.0 * (dl.double().unsqueeze(-1) if reduction == "none" else dl.double() / ids[..., 0].numel())
    bound = 2 * (2.0 ** -18 * (torch.softmax(z / 2.0, -1) + p) * scale + want[:, :-1].double().abs() * torch.finfo(dtype).eps)
    assert ((want - got)[:, :-1].double().abs() <= bound).all()
    assert (want[:, :-1] != 0).any(-1).all() and (want[:, -1] == 0).all() and (got[:, -1] == 0).all()


def _shifted(t):
    """t's values as a contiguous tensor one element off a 16-byte boundary."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.flatten()
    x = flat[1:].view(t.shape)
    assert x.is_contiguous() and x.data_ptr() % 16
    return x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 6, 2, 40, 128, 9), (1, 2, 2, 33, 64, 5)])
def test_attention_off_boundaries(dtype, shape):
    B, H, Hkv, N, D, K = shape
    g = _gen(5)
    q, do = ((torch.randn(B, H, N, D, generator=g)).to(dtype).to(DEV) for _ in range(2))
    k, v = ((torch.randn(B, Hkv, N, D, generator=g)).to(dtype).to(DEV) for _ in range(2))
    idx = torch.randint(0, N, (B, H, N, K), generator=g).to(DEV)

    def run(place):
        leaves = [place(t).detach().requires_grad_() for t in (q, k, v)]
        out = topk_attention(*leaves, topk_indices=idx, softcap=4.0)
        return (out.detach(), *torch.autograd.grad(out, leaves, place(do)))

    assert all(torch.equal(a, b) for a, b in zip(run(lambda t: t), run(_shifted)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 40])
def test_norms_off_boundaries(dtype, D):
    B, N, Hq, Hk = 2, 11, 4, 2
    g = _gen(7)
    q, k = (torch.randn(B, N, h * D, generator=g).to(dtype).to(DEV) for h in (Hq, Hk))
    wq, wk = (torch.rand(D, generator=g).to(DEV) + 0.5 for _ in range(2))
    cos, sin = (torch.randn(1, N, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    gq, gk = (torch.randn(B, h, N, D, generator=g).to(dtype).to(DEV) for h in (Hq, Hk))

    def run(place):
        leaves = [place(t).detach().requires_grad_() for t in (q, k, wq, wk)]
        c, s = place(cos), place(sin)
        out = qk_norm_rope(leaves[0], leaves[1], Hq, Hk, leaves[2], leaves[3], c, s)
        grads = torch.autograd.grad(out, leaves, (place(gq), place(gk)))
        x = q.clone().requires_grad_()
        rope = rope_to_heads(x, Hq, cos, sin)
        return (*[t.detach() for t in out], *grads, *torch.autograd.grad(rope, x, place(gq)))

    assert all(torch.equal(a, b) for a, b in zip(run(lambda t: t), run(_shifted)))
