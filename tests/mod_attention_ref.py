"""Gathered attention with score modifiers in 64 bits, and the error bounds its tests use."""

import math

import torch


def attention(q, k, v, idx, *, causal=True, q_start=0, softcap=None, slopes=None, segments=None, prefix_len=None):
    """(out, p, s) of q (B, H, Nq, D), k, v (B, Hkv, Nk, D) over the listed keys, differentiable.

    The definition entry by entry: each listed key inside [0, Nk) that the row sees takes part
    once for every time it is listed; a row without any is 0."""
    B, H, Nq, D = q.shape
    Hkv, Nk = k.shape[1], k.shape[2]
    G = H // Hkv
    idx = idx.long()
    j = idx.clamp(0, Nk - 1)
    i = (q_start + torch.arange(Nq, device=q.device)).view(1, 1, Nq, 1)
    ok = (idx >= 0) & (idx < Nk)
    if causal:
        see = j <= i
        if prefix_len is not None:
            see = see | (j < torch.as_tensor(prefix_len, device=q.device).expand(B).view(B, 1, 1, 1))
        ok = ok & see
    b = torch.arange(B, device=q.device).view(B, 1, 1, 1)
    if segments is not None:
        seg = segments.expand(B, Nk)
        ok = ok & (seg[b, j] == seg[b, i.expand(B, 1, Nq, 1)])
    g = (torch.arange(H, device=q.device) // G).view(1, H, 1, 1)
    kg, vg = k[b, g, j], v[b, g, j]
    # masked places may hold anything
    kg = torch.where(ok.unsqueeze(-1), kg, torch.zeros_like(kg))
    vg = torch.where(ok.unsqueeze(-1), vg, torch.zeros_like(vg))
    s = torch.einsum("bhnd,bhnkd->bhnk", q, kg) / math.sqrt(D)
    if softcap is not None:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        s = s - slopes.view(1, H, 1, 1) * (i - j).abs()
    s = s.masked_fill(~ok, -1e300)
    e = torch.exp(s - s.amax(dim=-1, keepdim=True).detach()) * ok
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    return torch.einsum("bhnk,bhnkd->bhnd", p, vg), p, vg


def score_step(q, k):
    """Largest rounding of a score in fp32: a chain of D products and the few operations after it, each
    within 2^-24 of sum |q_d k_d| / sqrt(D) (Cauchy-Schwarz)."""
    D = q.shape[-1]
    most = q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max() / math.sqrt(D)
    return (D + 8) * 2.0 ** -24 * (1.0 + most.item())


def rel(got, ref):
    ref = ref.double()
    return ((got.double() - ref).norm() / ref.norm().clamp_min(1e-300)).item()
