"""NaN in what a query sees shows in its output and gradients, in every form of the gathered attention and
nowhere else; a row that sees nothing is 0 whatever its query holds.  The places are those of the 64-bit
definition."""

import pytest
import torch

from mod_attention_ref import attention
from ossa_b200 import topk_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN = float("nan")

# dtype, H, Hkv, N, D, K.  bf16 with D = 128: up to 2^17 listed keys few rows, more with 2-8 heads per kv head the
# tensor cores, one head per kv head or K > 128 the per-head form; every other row the per-head form.
SMALL = [(torch.bfloat16, 6, 2, 40, 128, 17), (torch.bfloat16, 2, 2, 33, 128, 40), (torch.bfloat16, 9, 1, 20, 128, 150),
         (torch.bfloat16, 4, 2, 40, 64, 17), (torch.float32, 4, 2, 50, 64, 33), (torch.float32, 3, 1, 30, 256, 5),
         (torch.float32, 2, 2, 30, 16, 20), (torch.float32, 6, 2, 45, 128, 34)]
LARGE = [(torch.bfloat16, 6, 2, 400, 128, 64), (torch.bfloat16, 2, 2, 1100, 128, 64), (torch.bfloat16, 4, 2, 300, 128, 150)]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _case(dtype, H, Hkv, N, D, K):
    """Rows 3, 11 and 17 of head 0 hold NaN (row 11 lists nothing); key 5 of the last kv head does, and one value of
    value row 7 of the first.  The last listed key of every fourth row is key 5, alone in its step of the list."""
    g = _gen(N + D + K)
    q = torch.randn(1, H, N, D, generator=g).to(dtype)
    k, v = (torch.randn(1, Hkv, N, D, generator=g).to(dtype) for _ in range(2))
    idx = torch.rand(1, H, N, N, generator=g).topk(min(K, N), dim=-1).indices
    idx = torch.nn.functional.pad(idx, (0, K - idx.shape[-1]), value=-1)
    idx[(idx == 5) | (idx == 7)] = -1
    idx[:, :, ::4, -1] = 5
    idx[:, :, 1::6, 0] = 7
    idx[:, 0, 11] = -1
    idx[:, 0, 17, 0] = 0
    q[0, 0, [3, 17]] = NAN
    q[0, 0, 11, 2] = NAN
    k[0, Hkv - 1, 5] = NAN
    v[0, 0, 7, D // 2 + 1] = NAN
    return q, k, v, idx.int()


def _same_places(name, got, want):
    got = got.detach().cpu()
    assert torch.equal(got.isnan(), want.isnan()), f"{name}: NaN in {got.isnan().sum()} places, {want.isnan().sum()} wanted"
    assert torch.isfinite(got[~want.isnan()]).all(), name


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", SMALL + LARGE, ids=lambda c: "-".join(map(str, c)))
def test_training_form(case, causal):
    q, k, v, idx = _case(*case)
    ref_in = [t.double().requires_grad_() for t in (q, k, v)]
    ref, p, _ = attention(*ref_in, idx, causal=causal, softcap=6.0)
    do = torch.randn(ref.shape, generator=_gen(1)).to(q.dtype)
    want = torch.autograd.grad(ref, ref_in, do.double())
    # a row that sees nothing is 0 and has no gradient; torch's tanh makes 0 times NaN of it
    want[0][p.sum(-1) == 0] = 0.0
    dev = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = topk_attention(*dev, topk_indices=idx.to(DEV), causal=causal, softcap=6.0)
    _same_places("out", out, ref.detach())
    assert (out[0, 0, 11] == 0).all()
    # a row whose softmax is not a number has no gradient that is one; neither have the keys that it sees
    for name, got, w in zip(("dq", "dk", "dv"), torch.autograd.grad(out, dev, do.to(DEV)), want):
        _same_places(name, got, w)


@pytest.mark.parametrize("mods", ["slopes", "prefix"])
@pytest.mark.parametrize("case", SMALL + LARGE, ids=lambda c: "-".join(map(str, c)))
def test_modifiers_without_gradient(case, mods):
    q, k, v, idx = _case(*case)
    m = {"slopes": torch.rand(case[1], generator=_gen(2))} if mods == "slopes" else {"prefix_len": 9}
    ref = attention(q.double(), k.double(), v.double(), idx, **m)[0]
    m = {n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in m.items()}
    _same_places("out", topk_attention(q.to(DEV), k.to(DEV), v.to(DEV), topk_indices=idx.to(DEV), **m), ref)


@pytest.mark.parametrize("H,K", [(6, 17), (6, 64)])
def test_single_tokens(H, K):
    """One new token against a cache, its last listed key NaN or its query."""
    B, Hkv, N, D = 3, 2, 900, 128
    g = _gen(K)
    q = torch.randn(B, H, 1, D, generator=g).bfloat16()
    k, v = (torch.randn(B, Hkv, N, D, generator=g).bfloat16() for _ in range(2))
    idx = torch.rand(B, H, 1, N, generator=g).topk(K, dim=-1).indices
    idx[idx == 5] = -1
    idx[0, ..., -1] = 5
    k[0, :, 5] = NAN
    q[1, 2] = NAN
    ref = attention(q.double(), k.double(), v.double(), idx, q_start=N - 1, softcap=5.0)[0]
    out = topk_attention(q.to(DEV), k.to(DEV), v.to(DEV), topk_indices=idx.to(DEV), q_start=N - 1, softcap=5.0)
    _same_places("out", out, ref)
    assert out[0].isnan().all() and out[1, 2].isnan().all() and torch.isfinite(out[2]).all()
