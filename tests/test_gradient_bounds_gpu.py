"""Gradients of the modified gather within bounds near their own rounding, so that a lost part shows: the slopes'
gradient head by head, and bf16 gradients against the rounding of an exact result.

Slopes.  -dslope_h = sum over rows of sum_j dS_j far_j, dS_j = p_j (dP_j - Delta).  With e the relative error of a p
(twice the score's rounding, (D + 8) 2^-24 (1 + max |q||k| scale) of the row, for the score and for the row's
statistic, and 8 steps for the exponential and what surrounds it) and d the error of a dP ((D + 8) 2^-24 |dO||v|),
a row's share is off by at most
    e (A + P F) + 2 d F + K 2^-24 A,   A = sum p |dP - Delta| far,  P = sum p |dP - Delta|,  F = sum p far,
the second term for Delta, an average under the same p.  The errors of different rows are independent, and n
independent errors of at most b_i add up to more than 6 sqrt(sum b_i^2) once in 10^7 (Hoeffding).  Every head is held to
that over its rows, and it is at most a twentieth of the largest head's value: a kernel that loses the term, or a
head, fails.

bf16.  A result rounded once to bf16 is off by a uniform error of half a step, 2^-8 / m relative for a mantissa m in
[1, 2): in the norm of many such values 2^-8 sqrt(E[1 / (3 m^2)]) = 2^-8 * 0.425 = 1.66e-3 for mantissas spread
over their logarithm (1 % either way for as many values as here).  What enters it as two bf16 parts adds 2^-17, scores
and sums some 1e-5.  Evaluated in 64 bits with one mistake planted: weights without their rests 2.35e-3, Delta from
an output without its rest 1.89e-3 to 2.0e-3.  The bound is 1.8e-3."""

import math

import pytest
import torch

from mod_attention_ref import attention, rel
from ossa_b200 import topk_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROUNDED = 1.8e-3


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _lists(B, H, N, K, repeats, g):
    """Distinct keys of a row in ascending order, keys at or before it; with repeats, one listed twice."""
    near = (torch.rand(B, H, N, N, generator=g) * (torch.arange(N).view(1, N) <= torch.arange(N).view(N, 1))).topk(K, dim=-1)
    idx = torch.where(near.values > 0, near.indices, N).sort(dim=-1).values
    idx = torch.where(idx == N, -1, idx)
    if repeats:
        idx[..., 1] = idx[..., 0]
    return idx


def _case(dtype, B, H, Hkv, N, D, K, repeats, seed):
    g = _gen(seed)
    q, do = (torch.randn(B, H, N, D, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(B, Hkv, N, D, generator=g).to(dtype) for _ in range(2))
    idx = _lists(B, H, N, K, repeats, g)
    slopes = torch.rand(H, generator=g) * 0.1
    seg = torch.sort(torch.randint(0, 2, (B, N), generator=g), dim=1).values
    return q, k, v, do, idx, slopes, seg


def _slope_bound(q, k, do, idx, p, vg, out, q_start=0):
    """(H,) bounds on the error of dslopes."""
    B, H, N, D = q.shape
    K = idx.shape[-1]
    q, k, do = q.double(), k.double(), do.double()
    far = (q_start + torch.arange(N).view(1, 1, N, 1) - idx.clamp_min(0)).abs().double()
    dp = (vg @ do.unsqueeze(-1)).squeeze(-1)
    delta = (out * do).sum(-1, keepdim=True)
    size = p * (dp - delta).abs()
    A, P, F = (size * far).sum(-1), size.sum(-1), (p * far).sum(-1)
    kn = k.norm(dim=-1).amax(dim=2).repeat_interleave(H // k.shape[1], dim=1).unsqueeze(-1)  # (B, H, 1)
    score = (D + 8) * 2.0 ** -24 * (1 + q.norm(dim=-1) * kn / math.sqrt(D))
    e = 2 * score + 8 * 2.0 ** -24
    d = (D + 8) * 2.0 ** -24 * do.norm(dim=-1) * vg.norm(dim=-1).amax(dim=-1)
    return 6 * (e * (A + P * F) + 2 * d * F + K * 2.0 ** -24 * A).square().sum(dim=(0, 2)).sqrt()


def _run(dtype, B, H, Hkv, N, D, K, repeats, opts, docs, seed):
    q, k, v, do, idx, slopes, seg = _case(dtype, B, H, Hkv, N, D, K, repeats, seed)
    ref_in = [t.double().requires_grad_() for t in (q, k, v, slopes)]
    m = dict(opts, **({"segments": seg} if docs else {}))
    ref, p, vg = attention(*ref_in[:3], idx, slopes=ref_in[3], **m)
    want = torch.autograd.grad(ref, ref_in, do.double())
    p, vg, ref = p.detach(), vg.detach(), ref.detach()
    dev = [t.to(DEV).requires_grad_() for t in (q, k, v, slopes)]
    m = {n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in m.items()}
    out = topk_attention(*dev[:3], topk_indices=idx.to(DEV), slopes=dev[3], **m)
    got = [t.cpu() for t in torch.autograd.grad(out, dev, do.to(DEV))]
    bound = _slope_bound(q, k, do, idx, p, vg, ref)
    assert (bound <= 0.05 * want[3].abs().max()).all()  # the check below says something
    err = (got[3].double() - want[3]).abs()
    assert (err <= bound).all(), (err / bound).max()
    if dtype == torch.bfloat16:
        for name, a, b in zip(("out", "dq", "dk", "dv"), [out.detach().cpu()] + got[:3], [ref, *want[:3]]):
            assert rel(a, b) <= ROUNDED, f"{name}: {rel(a, b):.3e}"


@pytest.mark.parametrize("repeats", [False, True])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 6, 7, 8])
def test_tensor_core_passes(G, repeats):
    """Every group size, the heads' keys together and (a repeated key) head by head."""
    _run(torch.bfloat16, 2, 2 * G, 2, 160, 128, 48, repeats, {}, G % 2 == 0, seed=G)


@pytest.mark.parametrize("repeats", [False, True])
@pytest.mark.parametrize("B,H,Hkv,N,K", [(1, 12, 2, 400, 64), (2, 4, 2, 300, 128)])
def test_more_rows(B, H, Hkv, N, K, repeats):
    """More listed keys than the forward's few-row form takes."""
    assert B * H * N * K > 1 << 17
    _run(torch.bfloat16, B, H, Hkv, N, 128, K, repeats, {"softcap": 8.0}, True, seed=N)


@pytest.mark.parametrize("dtype,H,Hkv,D,K", [(torch.bfloat16, 9, 1, 128, 40), (torch.bfloat16, 4, 2, 128, 150),
                                             (torch.bfloat16, 4, 2, 64, 33), (torch.bfloat16, 2, 2, 256, 20),
                                             (torch.float32, 6, 3, 64, 33), (torch.float32, 4, 2, 128, 64),
                                             (torch.float32, 2, 1, 16, 10), (torch.float32, 3, 1, 256, 12)])
def test_per_head_passes(dtype, H, Hkv, D, K):
    _run(dtype, 2, H, Hkv, 200, D, K, False, {"softcap": 8.0}, True, seed=D)


@pytest.mark.parametrize("Nk", [300, 9000])
def test_rows_far_from_their_keys(Nk):
    """Distances up to the cache's length: the slopes' gradient where they are large."""
    B, H, Hkv, Nq, D, K = 2, 6, 2, 40, 128, 32
    g = _gen(Nk)
    q, do = (torch.randn(B, H, Nq, D, generator=g).bfloat16() for _ in range(2))
    k, v = (torch.randn(B, Hkv, Nk, D, generator=g).bfloat16() for _ in range(2))
    idx = torch.rand(B, H, Nq, Nk - Nq, generator=g).topk(K, dim=-1).indices.sort(dim=-1).values
    slopes = torch.rand(H, generator=g) * (3.0 / Nk)
    q0 = Nk - Nq
    ref_in = [t.double().requires_grad_() for t in (q, k, v, slopes)]
    ref, p, vg = attention(*ref_in[:3], idx, q_start=q0, slopes=ref_in[3])
    (want,) = torch.autograd.grad(ref, ref_in[3:], do.double())
    dev = [t.to(DEV).requires_grad_() for t in (q, k, v, slopes)]
    out = topk_attention(*dev[:3], topk_indices=idx.to(DEV), slopes=dev[3], q_start=q0)
    (got,) = torch.autograd.grad(out, dev[3:], do.to(DEV))
    bound = _slope_bound(q, k, do, idx, p.detach(), vg.detach(), ref.detach(), q_start=q0)
    assert (bound <= 0.05 * want.abs().max()).all()
    assert ((got.cpu().double() - want).abs() <= bound).all()
