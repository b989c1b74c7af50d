"""A row that sees nothing adds nothing to any gradient, whatever its query, its list and its incoming gradient hold."""

import pytest
import torch

from ossa_b200 import topk_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype,H,Hkv,D,K", [(torch.bfloat16, 6, 2, 128, 20), (torch.bfloat16, 2, 2, 128, 40),
                                             (torch.bfloat16, 9, 1, 128, 20), (torch.bfloat16, 4, 2, 128, 150),
                                             (torch.bfloat16, 4, 2, 64, 20), (torch.float32, 4, 2, 128, 33)])
def test_rows_without_a_key(dtype, H, Hkv, D, K, bad):
    B, N = 2, 70
    g = torch.Generator().manual_seed(K + H)
    q, do = (torch.randn(B, H, N, D, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(B, Hkv, N, D, generator=g).to(dtype) for _ in range(2))
    slopes = torch.rand(H, generator=g) * 0.1
    idx = torch.randint(0, N, (B, H, N, K), generator=g)
    seg = torch.zeros(B, N, dtype=torch.int32)
    seg[:, 60:] = 1  # rows of the second document list keys of the first only, row 7 keys behind it, row 9 nothing
    idx[:, :, 60:] = torch.randint(0, 60, (B, H, 10, K), generator=g)
    idx[:, :, 7] = torch.randint(8, N, (B, H, K), generator=g)
    idx[:, :, 9] = -1
    empty = [7, 9] + list(range(60, 70))
    res = []
    for value in (0.0, bad):
        qq, dd = q.clone(), do.clone()
        qq[:, :, empty] = value
        dd[:, :, empty] = value
        leaves = [t.to(DEV).requires_grad_() for t in (qq, k, v, slopes)]
        out = topk_attention(*leaves[:3], topk_indices=idx.to(DEV), slopes=leaves[3], segments=seg.to(DEV), softcap=7.0)
        res.append([out.detach(), *torch.autograd.grad(out, leaves, dd.to(DEV))])
    assert (res[0][0][:, :, empty] == 0).all() and (res[0][1][:, :, empty] == 0).all() and res[0][4].ne(0).all()
    for name, a, b in zip(("out", "dq", "dk", "dv", "dslopes"), *res):
        assert torch.equal(a, b), name
