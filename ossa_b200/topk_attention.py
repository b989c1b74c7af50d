"""Top-K sparse attention forward on sm_100a (the reference's ``topk_attention``).

Drop-in for ``ossa.triton_kernel.topk_attention`` (ossa/triton_kernel.py:41-70):
same signature and result.  The reference dispatches between a Triton kernel
(never launched on hardware) and a PyTorch fallback; here there is exactly one
implementation, ``ossa_topk_attention_fwd`` in libossa_b200.so, and CPU tensors
are rejected.  Differences, all additive:

* k and v may carry Hkv < H heads (GQA, query head h reads kv head h // (H/Hkv));
  the reference needs them repeated to H heads first (sparse_forward.py:175-178).
* indices may be int32 or int64; an index outside [0, N) (for example the -1
  padding of ossa_b200's selectors) is treated as masked.
* ``block_m`` and ``use_triton`` are accepted for signature compatibility and
  ignored (there is no Triton path to select).
* (additive) score modifiers: ``softcap`` (a tanh cap), ``slopes`` (a bias that falls
  with distance), ``segments`` (documents packed in one row) and ``prefix_len`` (keys
  that every query may see).
* (additive) gradients: where q, k, v or slopes require them, the output carries
  autograd history (csrc/autograd.cpp, ``ossa_topk_attention_bwd``); the forward's values are then the
  same to rounding (a bf16 output sums its keys in another order).
"""

from __future__ import annotations

import math
from typing import Optional, Union

import torch

from . import _lib

# Import-compatibility name: the reference exports whether its fused GPU kernel
# is usable.  Here the fused sm_100a kernel is the only implementation.
HAS_TRITON = True

_F32 = torch.finfo(torch.float32)


def _check(q, k, v, idx, rows=False):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k and v must be 4-D (B, H, N, D)")
    B, H, N, D = q.shape
    if k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have the same shape")
    Bk, Hkv, Nk, Dk = k.shape
    if (B, D) != (Bk, Dk) or (not rows and N != Nk):
        raise ValueError(f"q {tuple(q.shape)} and k/v {tuple(k.shape)} disagree on B, N or D")
    if Hkv <= 0 or H % Hkv != 0:
        raise ValueError(f"query heads {H} must be a multiple of key/value heads {Hkv}")
    if idx.dim() != 4 or tuple(idx.shape[:3]) != (B, H, N):
        raise ValueError(f"topk_indices must be (B, H, N, K) = ({B}, {H}, {N}, K); got {tuple(idx.shape)}")
    if idx.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"topk_indices must be int32 or int64, got {idx.dtype}")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"q, k, v dtypes differ: {q.dtype}, {k.dtype}, {v.dtype}")
    return B, H, Hkv, N, D, idx.shape[-1]


def topk_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    topk_indices: torch.Tensor,
    causal: bool = True,
    block_m: int = 32,
    use_triton: Optional[bool] = None,
    q_start: Optional[int] = None,
    softcap: Optional[float] = None,
    slopes: Optional[torch.Tensor] = None,
    segments: Optional[torch.Tensor] = None,
    prefix_len: Union[torch.Tensor, int, None] = None,
) -> torch.Tensor:
    """Top-K sparse attention, forward and (by autograd) backward.

    q: (B, H, N, D); k, v: (B, Hkv, N, D); topk_indices: (B, H, N, K).
    Returns (B, H, N, D) in q's dtype: per query, softmax over the K listed keys
    of (q . k) / sqrt(D) (keys > i masked when ``causal``), times V; rows with
    no unmasked key are 0.

    ``q_start`` (additive, for sequence sharding): q and topk_indices then hold
    Nq query rows at positions q_start .. q_start + Nq - 1 of a sequence whose
    Nk keys k, v hold in full; row l is masked causally against q_start + l.

    Score modifiers (additive), x the scaled score of a query at position i and key j:
    ``softcap``: x becomes softcap * tanh(x / softcap); at least 2^-126 and finite in float32.
    ``slopes`` (H,): slopes[h] * abs(i - j) is subtracted after the cap.
    ``segments`` (B, Nk) or (Nk,), int32 or int64 (compared as 32-bit values): a key is
    seen only from its own segment; every query position must be below Nk.
    ``prefix_len`` (B,) int32 or int64, or one int: keys j < prefix_len[b] are seen by
    every query of batch element b, whatever the causal mask says of them.

    Differentiable in q, k, v and slopes, once; indices, segments and prefix_len are not.
    An index listed twice in a row counts twice.  The gradients are the same bits in every
    call; they need (H / Hkv) * Nq * K <= 2**30.
    """
    del block_m, use_triton
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                        (slopes is not None and slopes.requires_grad))
    if grad or softcap is not None or slopes is not None or segments is not None or prefix_len is not None:
        return _topk_attention_modified(q, k, v, topk_indices, causal, q_start, softcap, slopes, segments, prefix_len,
                                        grad)
    if q_start is not None:
        return _topk_attention_rows(q, k, v, topk_indices, causal, int(q_start))
    B, H, Hkv, N, D, K = _check(q, k, v, topk_indices)
    dev = _lib.require_cuda(q, k, v, topk_indices)
    code = _lib.dtype_code(q)
    qc, kc, vc = q.contiguous(), k.contiguous(), v.contiguous()
    ic = topk_indices.contiguous()
    out = torch.empty_like(qc)
    if out.numel() == 0:
        return out
    with torch.cuda.device(dev):
        st = _lib.lib().ossa_topk_attention_fwd(
            qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), ic.data_ptr(),
            1 if ic.dtype == torch.int64 else 0, code, B, H, Hkv, N, D, K,
            float(1.0 / math.sqrt(D)), 1 if causal else 0, out.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(st)
    return out


def _topk_attention_rows(q, k, v, topk_indices, causal, q_start):
    if q_start < 0:
        raise ValueError(f"q_start must be >= 0, got {q_start}")
    B, H, Hkv, Nq, D, K = _check(q, k, v, topk_indices, rows=True)
    Nk = k.shape[2]
    dev = _lib.require_cuda(q, k, v, topk_indices)
    code = _lib.dtype_code(q)
    qc, kc, vc = q.contiguous(), k.contiguous(), v.contiguous()
    ic = topk_indices.contiguous()
    out = torch.empty_like(qc)
    if out.numel() == 0:
        return out
    with torch.cuda.device(dev):
        st = _lib.lib().ossa_topk_attention_fwd_rows(
            qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), ic.data_ptr(),
            1 if ic.dtype == torch.int64 else 0, code, B, H, Hkv, Nq, Nk, D, K,
            float(1.0 / math.sqrt(D)), 1 if causal else 0, q_start, out.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(st)
    return out


def _int32(name, t, shapes):
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be an int32 or int64 tensor, got {getattr(t, 'dtype', type(t).__name__)}")
    if tuple(t.shape) not in shapes:
        raise ValueError(f"{name} of shape {tuple(t.shape)} is not {' or '.join(map(str, shapes))}")
    return t.to(torch.int32)


def _topk_attention_modified(q, k, v, idx, causal, q_start, softcap, slopes, segments, prefix_len, grad):
    q0 = 0 if q_start is None else int(q_start)
    if q0 < 0:
        raise ValueError(f"q_start must be >= 0, got {q0}")
    B, H, Hkv, Nq, D, K = _check(q, k, v, idx, rows=q_start is not None)
    Nk = k.shape[2]
    cap = 0.0
    if softcap is not None:
        cap = float(softcap)
        if not (_F32.tiny <= cap <= _F32.max):  # as the kernels hold it
            raise ValueError(f"softcap must lie in the normal range of float32, got {softcap}")
    if slopes is not None:
        if tuple(slopes.shape) != (H,) or not slopes.is_floating_point():
            raise ValueError(f"slopes must be ({H},) floating point; got {tuple(slopes.shape)} {slopes.dtype}")
        slopes = slopes.float().contiguous()
    if segments is not None:
        segments = _int32("segments", segments, [(B, Nk), (Nk,)])
        if q0 + Nq > Nk:
            raise ValueError(f"segments need every query position below {Nk}; rows end at {q0 + Nq}")
        segments = segments.expand(B, Nk).contiguous()
    if prefix_len is not None:
        if isinstance(prefix_len, int):
            if prefix_len < 0:
                raise ValueError(f"prefix_len must be >= 0, got {prefix_len}")
            prefix_len = torch.full((B,), min(prefix_len, Nk), dtype=torch.int32, device=q.device)
        elif isinstance(prefix_len, torch.Tensor) and prefix_len.dtype == torch.int64:
            prefix_len = prefix_len.clamp(0, Nk)  # a length past 32 bits is still one
        prefix_len = _int32("prefix_len", prefix_len, [(B,)]).contiguous()
    _lib.dtype_code(q)
    _lib.require_cuda(*[t for t in (q, k, v, idx, slopes, segments, prefix_len) if t is not None])
    return _lib.native().topk_attention(q, k, v, slopes, idx, segments, prefix_len, bool(causal), q0, cap, grad)
