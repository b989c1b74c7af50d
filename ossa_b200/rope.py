"""RoPE fused with the head transpose of the patched layer.

The patched forward (ossa/bench/sparse_forward.py:166-178) views each q/k/v
projection (B, N, Hx*D) as (B, Hx, N, D), applies Qwen2's
``apply_rotary_pos_emb`` to q and k, and the selection and gather read
contiguous rows.  ``rope_to_heads`` does that in one kernel pass, with the same
rounding as the eager expression ``x*cos + rotate_half(x)*sin``; the result is
bit-identical to it.  Additive: the reference runs the eager ops.

``qk_norm_rope`` serves layers that norm every query and key head before the rotation:
norm, rotation and head transpose of both tensors in one kernel pass.  Both functions are
differentiable (csrc/autograd.cpp; one backward kernel, ``ossa_qk_norm_rope_bwd``).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib


def rope_to_heads(x: torch.Tensor, n_heads: int, cos: Optional[torch.Tensor] = None,
                  sin: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x: (B, N, n_heads * D) or (B, N, n_heads, D); cos, sin: (B or 1, N, D)
    (Qwen2's position embeddings) or both None (layout only).  Returns the
    contiguous (B, n_heads, N, D) tensor, rotated when cos/sin are given.
    Differentiable in x (head dims up to 512), once, not in cos and sin."""
    if (cos is None) != (sin is None):
        raise ValueError("pass both cos and sin, or neither")
    B, N = x.shape[0], x.shape[1]
    D = x.shape[-1] if x.dim() == 4 else x.shape[-1] // n_heads
    if x.dim() not in (3, 4) or x.shape[2:] not in ((n_heads * D,), (n_heads, D)):
        raise ValueError(f"x of shape {tuple(x.shape)} is not (B, N, {n_heads} heads x D)")
    ts = [x] if cos is None else [x, cos, sin]
    dev = _lib.require_cuda(*ts)
    xc = x.contiguous()
    code = _lib.dtype_code(xc)
    cs = None
    if cos is not None:
        cos = cos.to(xc.dtype)
        sin = sin.to(xc.dtype)
        if cos.dim() == 2:
            cos, sin = cos.unsqueeze(0), sin.unsqueeze(0)
        if cos.shape != sin.shape or cos.shape[0] not in (1, B) or tuple(cos.shape[1:]) != (N, D):
            raise ValueError(f"cos/sin of shape {tuple(cos.shape)} do not match (B or 1, {N}, {D})")
        cs = (cos.contiguous(), sin.contiguous())
    if torch.is_grad_enabled() and x.requires_grad:
        return _lib.native().rope_to_heads(x, *([t.detach() for t in cs] if cs else (None, None)), n_heads)
    out = torch.empty((B, n_heads, N, D), dtype=xc.dtype, device=dev)
    if out.numel() == 0:
        return out
    with torch.cuda.device(dev):
        st = _lib.lib().ossa_rope_to_heads(xc.data_ptr(), _lib.ptr(cs[0] if cs else None),
                                           _lib.ptr(cs[1] if cs else None),
                                           1 if cs is not None and cs[0].shape[0] == B and B > 1 else 0, code,
                                           B, N, n_heads, D, out.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(st)
    return out


def _tables(cos, sin, B, N, D, dtype):
    """cos, sin as (B or 1, N, D) of the rows' type."""
    if cos.requires_grad or sin.requires_grad:
        cos, sin = cos.detach(), sin.detach()
    if cos.dtype != dtype or sin.dtype != dtype:
        cos, sin = cos.to(dtype), sin.to(dtype)
    if cos.dim() == 2:
        cos, sin = cos.unsqueeze(0), sin.unsqueeze(0)
    if cos.shape != sin.shape or cos.dim() != 3 or cos.shape[0] not in (1, B) or tuple(cos.shape[1:]) != (N, D):
        raise ValueError(f"cos/sin of shapes {tuple(cos.shape)}, {tuple(sin.shape)} do not match (B or 1, {N}, {D})")
    return cos, sin


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, n_heads: int, n_kv_heads: int,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, *,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head, rotation and head transpose in one pass.

    q: (B, N, n_heads * D) or (B, N, n_heads, D), k alike with n_kv_heads, float32 or
    bfloat16; views whose (b, n) rows lie in one piece (slices of a joint projection) are read
    where they are.  q_weight, k_weight: (D,) norm weights, None for no norm of that tensor;
    cos, sin: (B or 1, N, D) or (N, D), cast to the rows' type, or both None for no rotation.
    Returns the contiguous (B, n_heads, N, D) and (B, n_kv_heads, N, D) tensors
    ``rope(x * rsqrt(mean(x**2) + eps) * weight)``, computed in fp32 and rounded once.  D is a
    multiple of 8, at most 512.

    Differentiable in q, k and the weights, once; not in cos and sin.  Gradients are the same
    bits in every call."""
    if (cos is None) != (sin is None):
        raise ValueError("pass both cos and sin, or neither")
    if q.dtype != k.dtype:
        raise TypeError(f"q and k dtypes differ: {q.dtype}, {k.dtype}")
    _lib.dtype_code(q)
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and >= 0, got {eps}")
    if q.dim() not in (3, 4) or k.dim() not in (3, 4) or q.shape[:2] != k.shape[:2]:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} are not (B, N, heads x D) of one B and N")
    D = q.shape[3] if q.dim() == 4 else q.shape[2] // max(n_heads, 1)
    Dk = k.shape[3] if k.dim() == 4 else k.shape[2] // max(n_kv_heads, 1)
    if n_heads <= 0 or n_kv_heads <= 0 or D != Dk or \
            (q.shape[2] != n_heads if q.dim() == 4 else q.shape[2] != n_heads * D) or \
            (k.shape[2] != n_kv_heads if k.dim() == 4 else k.shape[2] != n_kv_heads * D):
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} do not hold {n_heads} and {n_kv_heads} heads of one D")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (tuple(w.shape) != (D,) or not w.is_floating_point()):
            raise ValueError(f"{name} must be ({D},) floating point; got {tuple(w.shape)} {w.dtype}")
    kinds = {w.dtype for w in (q_weight, k_weight) if w is not None}
    if kinds and kinds not in ({torch.float32}, {torch.bfloat16}):  # one storage type for both weights
        q_weight = None if q_weight is None else q_weight.float()
        k_weight = None if k_weight is None else k_weight.float()
    q_weight = None if q_weight is None else q_weight.contiguous()
    k_weight = None if k_weight is None else k_weight.contiguous()
    _lib.require_cuda(*[t for t in (q, k, q_weight, k_weight, cos, sin) if t is not None])
    if cos is not None:
        cos, sin = _tables(cos, sin, q.shape[0], q.shape[1], D, q.dtype)
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight))
    return _lib.native().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, n_heads, n_kv_heads, eps, grad)
