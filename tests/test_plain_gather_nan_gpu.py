"""NaN in what a query sees shows in the plain gather too (no modifiers, no gradient), in every form."""

import pytest
import torch

from mod_attention_ref import attention
from ossa_b200 import topk_attention
from test_not_finite_attention_gpu import DEV, LARGE, NAN, SMALL, _gen, _same_places

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("case", SMALL + LARGE + [(torch.bfloat16, 12, 2, 5000, 128, 20), (torch.bfloat16, 4, 2, 200, 128, 100)],
                         ids=lambda c: "-".join(map(str, c)))
def test_plain_gather(case, rows):
    dtype, H, Hkv, N, D, K = case
    g = _gen(N + D + K)
    q = torch.randn(1, H, N, D, generator=g).to(dtype)
    k, v = (torch.randn(1, Hkv, N, D, generator=g).to(dtype) for _ in range(2))
    idx = torch.randint(0, N, (1, H, N, K), generator=g)
    idx[idx == 5] = 6
    idx = idx.sort(dim=-1).values  # ascending with repeats; the first rows see few of them
    idx[:, :, ::4, -1] = 5
    idx[:, 0, 11] = -1
    q[0, 0, [3, 11, 17]] = NAN
    q[0, H - 1, N - 1, 1] = NAN
    k[0, Hkv - 1, 5] = NAN
    for causal in (True, False):
        ref = attention(q.double(), k.double(), v.double(), idx, causal=causal)[0]
        kw = {"q_start": 0} if rows else {}
        out = topk_attention(q.to(DEV), k.to(DEV), v.to(DEV), topk_indices=idx.to(DEV), causal=causal, **kw)
        _same_places("out", out, ref)
        assert (out[0, 0, 11] == 0).all()


def test_distinct_lists():
    """Lists in the selectors' form (distinct, ascending, -1 behind): the heads taken together."""
    for N, K in ((300, 64), (300, 100), (5000, 64)):
        g = _gen(N + K)
        q = torch.randn(1, 12, N, 128, generator=g).bfloat16()
        k, v = (torch.randn(1, 2, N, 128, generator=g).bfloat16() for _ in range(2))
        near = torch.arange(N).view(N, 1) - torch.arange(K - 1, -1, -1)
        idx = torch.where(near < 0, N, near).sort(dim=-1).values
        idx = torch.where(idx == N, -1, idx).expand(1, 12, N, K).contiguous()
        q[0, 3, 40] = NAN
        q[0, 11, N - 1, 5] = NAN
        k[0, 1, N - 50] = NAN
        ref = attention(q.double(), k.double(), v.double(), idx)[0]
        _same_places("out", topk_attention(q.to(DEV), k.to(DEV), v.to(DEV), topk_indices=idx.to(DEV)), ref)
