"""The plain gather: what a head does not list, or does not see, may hold NaN or infinities.  Rows and heads that list
such a key show it, all others get what they get without it."""

import pytest
import torch

from mod_attention_ref import attention
from ossa_b200 import topk_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# dtype, H, Hkv, N, D, K: the heads together (2, 3, 4, 6, 8 a kv head; few and many keys), per head, other head dims
CASES = [(torch.bfloat16, 6, 2, 300, 128, 32), (torch.bfloat16, 12, 2, 5000, 128, 64), (torch.bfloat16, 8, 1, 200, 128, 100),
         (torch.bfloat16, 4, 2, 90, 128, 17), (torch.bfloat16, 2, 2, 90, 128, 17), (torch.bfloat16, 5, 1, 90, 128, 40),
         (torch.bfloat16, 4, 2, 90, 128, 150), (torch.bfloat16, 4, 2, 90, 64, 17), (torch.float32, 4, 2, 90, 128, 33)]


def _lists(H, N, K, g):
    """Ascending distinct keys of about half the listed places, -1 behind, key 0 and key 7 in none."""
    idx = torch.rand(1, H, N, N, generator=g).topk(min(K, N), dim=-1).indices
    keep = torch.rand(idx.shape, generator=g) < 0.6
    idx = torch.where((idx == 0) | (idx == 7) | ~keep, N, idx).sort(dim=-1).values
    return torch.nn.functional.pad(torch.where(idx == N, -1, idx), (0, K - idx.shape[-1]), value=-1)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_keys_that_nobody_lists(case, bad):
    dtype, H, Hkv, N, D, K = case
    g = torch.Generator().manual_seed(N + K)
    q = torch.randn(1, H, N, D, generator=g).to(dtype).to(DEV)
    k, v = (torch.randn(1, Hkv, N, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    idx = _lists(H, N, K, g).to(DEV)
    want = topk_attention(q, k, v, topk_indices=idx)
    for t in (k, v):
        t[:, :, 0] = bad
        t[:, :, 7] = bad
    assert torch.isfinite(want).all() and torch.equal(topk_attention(q, k, v, topk_indices=idx), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_a_key_that_one_head_lists(case, bad):
    """Key 7's value row (and for NaN its key row) in the lists of head 0 alone, at every fifth row."""
    dtype, H, Hkv, N, D, K = case
    g = torch.Generator().manual_seed(N + K + 1)
    q = torch.randn(1, H, N, D, generator=g).to(dtype)
    k, v = (torch.randn(1, Hkv, N, D, generator=g).to(dtype) for _ in range(2))
    idx = _lists(H, N, K, g)
    idx[:, 0, 10::5, 0] = 7
    v[:, :, 7] = bad
    if bad != bad:
        k[:, :, 7] = bad
    ref = attention(q.double(), k.double(), v.double(), idx)[0]
    out = topk_attention(q.to(DEV), k.to(DEV), v.to(DEV), topk_indices=idx.to(DEV)).cpu()
    odd = ~torch.isfinite(ref)
    assert odd[0, 0, 10::5].all() and odd.sum() == odd[0, 0, 10::5].sum()
    assert torch.equal(~torch.isfinite(out), odd)  # an infinity may have met a weight of 0 on its way
    # p and the output are rounded to the type: two steps in the norm, and fp32 sums
    step = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -16
    diff = (out.double() - ref)[~odd]
    assert diff.norm() <= 2 * step * ref[~odd].norm()
