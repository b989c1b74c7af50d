"""Saved tensors that a hook brings back in another layout (twice as wide, every other element) or off a 16-byte
boundary: the gradients are those of the tensors as they were saved."""

import pytest
import torch

from ossa_b200 import qk_norm_rope, rope_to_heads, top_logit_distillation_loss, topk_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _wide(t):
    x = torch.zeros(*t.shape, 2, dtype=t.dtype, device=t.device)
    x[..., 0] = t
    return x[..., 0]


def _off(t):
    x = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
    x[1:] = t.flatten()
    return x[1:].view(t.shape)


def _calls(dtype):
    g = torch.Generator().manual_seed(3)
    B, H, Hkv, N, D, K, V = 2, 4, 2, 40, 128, 9, 301
    q = torch.randn(B, H, N, D, generator=g).to(dtype).to(DEV).requires_grad_()
    k, v = (torch.randn(B, Hkv, N, D, generator=g).to(dtype).to(DEV).requires_grad_() for _ in range(2))
    slopes = torch.rand(H, generator=g).to(DEV).requires_grad_()
    idx = torch.randint(-1, N, (B, H, N, K), generator=g).to(DEV)
    seg = torch.sort(torch.randint(0, 2, (B, N), generator=g), dim=1).values.to(DEV)
    x, y = (torch.randn(B, N, h * D, generator=g).to(dtype).to(DEV).requires_grad_() for h in (H, Hkv))
    w = torch.rand(D, generator=g).to(DEV).requires_grad_()
    cs = [torch.randn(B, N, D, generator=g).to(dtype).to(DEV) for _ in range(2)]
    z = torch.randn(B, N, V, generator=g).to(dtype).to(DEV).requires_grad_()
    ids = torch.rand(B, N, V, generator=g).topk(K, dim=-1).indices.to(DEV)
    t = torch.randn(B, N, K, generator=g).to(DEV)
    return {"attention": ((q, k, v, slopes), lambda: topk_attention(q, k, v, topk_indices=idx, slopes=slopes, segments=seg,
                                                                   prefix_len=torch.tensor([3, 0], device=DEV))),
            "norms": ((x, y, w), lambda: torch.cat([o.flatten() for o in qk_norm_rope(x, y, H, Hkv, w, w, *cs)])),
            "rope": ((x,), lambda: rope_to_heads(x, H, *cs)),
            "mean": ((z,), lambda: top_logit_distillation_loss(z, t, ids)),
            "scaled mean": ((z,), lambda: 3.0 * top_logit_distillation_loss(z, t, ids)),
            "rows": ((z,), lambda: top_logit_distillation_loss(z, t, ids, reduction="none"))}


@pytest.mark.parametrize("place", [_wide, _off])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["attention", "norms", "rope", "mean", "scaled mean", "rows"])
def test_another_layout(name, dtype, place):
    leaves, call = _calls(dtype)[name]

    def grads():
        out = call()
        up = torch.randn(out.shape, generator=torch.Generator().manual_seed(5)).to(out) if out.dim() else torch.ones_like(out)
        return torch.autograd.grad(out, leaves, up)

    want = grads()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, place):
        got = grads()
    for a, b in zip(want, got):
        if name in ("scaled mean", "rows") and place is _off:
            # rows begin elsewhere between 16-byte boundaries: their sums are split there (2^-18 of softmax + p)
            assert (a.double() - b.double()).abs().max() <= 2.0 ** -17 * a.abs().max() + 2 * torch.finfo(dtype).eps * a.abs().max()
        else:
            assert torch.equal(a, b), name
