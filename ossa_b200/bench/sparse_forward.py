"""Patched ``Qwen2Attention.forward`` running the sm_100a sparse path.

Mirrors ``PatchPlan`` / ``_patch_layer`` / ``_load_router`` of
ossa/bench/sparse_forward.py:122-239, 272-294, so code that patches a Hugging
Face Qwen2 model with the reference keeps working.  The patched forward
(reference :157-229) does q/k/v projections and RoPE with the layer's own
modules, then:

* selection in fp32 by one fused kernel (router: ContentRouter scores, :185-193;
  oracle: exact q.k/sqrt(D), :194-196), causal, no N x N selector in memory;
* the gathered sparse forward (reference :204-208) on GQA-native K/V
  (no ``repeat_interleave``, :175-178);
* ``impl="mask"`` keeps the reference's mask-path semantics (top-K set plus the
  forced diagonal, :209-222) but evaluates them on the same O(N*K) kernel by
  appending the diagonal to each index row instead of a dense N x N softmax;
* o_proj and the ``(out, None)`` return as the reference;
* (additive) RoPE and the head transpose of q/k/v run as one kernel pass per
  tensor (``rope_to_heads``), bit-identical to ``apply_rotary_pos_emb`` plus the
  layout copies; a layer that norms its query and key heads (``q_norm``, ``k_norm``
  RMS modules) has norm, RoPE and transpose of both in one pass (``qk_norm_rope``);
* (additive) the layer trains: every step but the selection is differentiable
  (gradients flow through the selected keys' attention, the selection is a
  constant), and ``PatchPlan`` carries the score modifiers of ``topk_attention``.

Deliberate difference: the reference casts router logits to the model dtype
before ``torch.topk`` (:193), which ties ~15% of rows at the K-th boundary in
bf16; selection here is in fp32 (ties broken toward the lower key index).
Like the reference, the forward is prefill-only: ``attention_mask`` (padding)
and ``past_key_values`` are ignored.
"""

from __future__ import annotations

from dataclasses import dataclass
from pathlib import Path
from typing import Optional, Union

import torch

from .. import select
from ..rope import qk_norm_rope, rope_to_heads
from ..router import ContentRouter, ContentRouterConfig
from ..topk_attention import topk_attention


@dataclass
class PatchPlan:
    mode: str                          # "dense" | "oracle" | "router"
    k: int = 64
    layers: tuple[int, ...] = ()       # which layers to patch; empty = none
    routers: dict[int, ContentRouter] | None = None  # layer_idx -> router
    impl: str = "mask"                 # "mask" (top-K + forced diagonal) | "gather"
    # Score modifiers of every patched layer, as topk_attention takes them (additive).  They act on the
    # attention, not on the selection: a row's K keys may lie in other documents, which hides them (a row of
    # impl "gather" whose keys all do gives 0).
    softcap: Optional[float] = None
    slopes: Optional[torch.Tensor] = None                    # (H,)
    segments: Optional[torch.Tensor] = None                  # (B, N) or (N,)
    prefix_len: Union[torch.Tensor, int, None] = None        # (B,) or one int


def _norms_as(norm, weight, eps):
    """Whether the module is the norm that qk_norm_rope computes (others store their weight as an offset from 1)."""
    with torch.no_grad():
        x = torch.linspace(-1.0, 1.5, weight.numel(), device=weight.device, dtype=weight.dtype)
        want = x.float() * torch.rsqrt(x.float().pow(2).mean() + eps) * weight.float()
        got = norm(x.unsqueeze(0)).squeeze(0).float()
        # as many roundings of its type as a norm may make; an offset shows far above them
        return bool(((got - want).abs() <= 16 * torch.finfo(weight.dtype).eps * want.abs() + 1e-30).all())


def _head_norms(layer_module):
    """(q weight, k weight, eps) of the layer's query and key head norms, None if it has none."""
    norms = [getattr(layer_module, name, None) for name in ("q_norm", "k_norm")]
    if all(norm is None or isinstance(norm, torch.nn.Identity) for norm in norms):
        return None
    eps = []
    for norm in norms:
        weight = getattr(norm, "weight", None)
        e = getattr(norm, "variance_epsilon", getattr(norm, "eps", None))
        if weight is None or weight.shape != (layer_module.head_dim,) or e is None or \
                getattr(norm, "bias", None) is not None or isinstance(norm, torch.nn.LayerNorm):
            raise TypeError("q_norm and k_norm must both be RMS norms over head_dim (weight and eps, no bias); "
                            f"got {type(norm).__name__}")
        eps.append(float(e))
        if not _norms_as(norm, weight, float(e)):
            raise TypeError(f"{type(norm).__name__} does not compute x * rsqrt(mean(x**2) + eps) * weight")
    if eps[0] != eps[1]:
        raise TypeError(f"q_norm and k_norm must have one eps, got {eps[0]} and {eps[1]}")
    return norms[0].weight, norms[1].weight, eps[0]


def _router_params(router):
    """(wq, wk, pos_bias, seq_len) of a ContentRouter-shaped module (this package's
    or the reference's: both expose q_proj[0], k_proj[0], pos_bias, cfg.seq_len)."""
    try:
        return (router.q_proj[0].weight, router.k_proj[0].weight, router.pos_bias.weight,
                int(router.cfg.seq_len))
    except AttributeError as e:
        raise TypeError(
            "only ContentRouter-style routers (q_proj, k_proj, pos_bias) are supported; "
            f"got {type(router).__name__}") from e


def select_indices(plan: PatchPlan, layer_idx: int, q: torch.Tensor, k: torch.Tensor) -> torch.Tensor:
    """Causal top-K indices (B, H, N, K') for one patched layer, int32, -1 padded."""
    N = q.shape[2]
    k_eff = min(plan.k, N)
    if plan.mode == "router":
        if plan.routers is None or layer_idx not in plan.routers:
            raise KeyError(f"no router for layer {layer_idx}")
        wq, wk, pb, seq_len = _router_params(plan.routers[layer_idx])
        idx = select.router_topk(q, k, wq, wk, pb, seq_len, k_eff, causal=True)
    elif plan.mode == "oracle":
        idx = select.oracle_topk(q, k, k_eff, causal=True)
    else:
        raise ValueError(plan.mode)
    if plan.impl == "mask":
        idx = select.with_diagonal(idx)
    elif plan.impl != "gather":
        raise ValueError(f"unknown impl {plan.impl!r}")
    return idx


def _patch_layer(model, plan: PatchPlan):
    """Monkey-patches ``self_attn.forward`` of the chosen layers; returns a
    callable that undoes every patch."""
    if plan.mode == "dense" or not plan.layers:
        return lambda: None

    restores: list = []
    for layer_idx in plan.layers:
        layer_module = model.model.layers[layer_idx].self_attn
        original_forward = layer_module.forward
        head_norms = _head_norms(layer_module)

        def make_forward(layer_module=layer_module, captured_idx=layer_idx, eps=head_norms and head_norms[2]):
            def new_forward(hidden_states, attention_mask=None, position_ids=None,
                            past_key_values=None, output_attentions=False,
                            use_cache=False, cache_position=None,
                            position_embeddings=None, **kwargs):
                B, N, _ = hidden_states.shape
                head_dim = layer_module.head_dim
                n_heads = layer_module.config.num_attention_heads
                n_kv_heads = layer_module.config.num_key_value_heads

                # projections, then RoPE and the (B, heads, N, D) layout in one kernel
                # pass per tensor (bit-identical to apply_rotary_pos_emb + contiguous)
                cos, sin = position_embeddings if position_embeddings is not None else (None, None)
                q, k = layer_module.q_proj(hidden_states), layer_module.k_proj(hidden_states)
                if eps is not None:
                    wq, wk = layer_module.q_norm.weight, layer_module.k_norm.weight
                    q, k = qk_norm_rope(q, k, n_heads, n_kv_heads, wq, wk, cos, sin, eps=eps)
                else:
                    q = rope_to_heads(q, n_heads, cos, sin)
                    k = rope_to_heads(k, n_kv_heads, cos, sin)
                v = rope_to_heads(layer_module.v_proj(hidden_states), n_kv_heads)

                with torch.no_grad():
                    idx = select_indices(plan, captured_idx, q, k)
                out = topk_attention(q, k, v, topk_indices=idx, causal=True, softcap=plan.softcap,
                                     slopes=plan.slopes, segments=plan.segments, prefix_len=plan.prefix_len)

                out = out.transpose(1, 2).reshape(B, N, n_heads * head_dim)
                out = layer_module.o_proj(out)
                return out, None
            return new_forward

        layer_module.forward = make_forward()
        restores.append((layer_module, original_forward))

    def restore() -> None:
        for lm, orig in restores:
            lm.forward = orig

    return restore


def _load_router(checkpoint: Path, model, layer: int, seq_len: int, *, pos_bias: str = "exact"):
    """Loads a ContentRouter checkpoint ({"state_dict", "cfg"}, the reference's
    format, bench/content_train.py:172-175) sized for ``seq_len`` as the reference
    does (sparse_forward.py:272-294).  With ``pos_bias="exact"`` (the reference's
    behaviour) a checkpoint trained at another seq_len does not fit.  With
    ``pos_bias="extend"`` (additive) the router is built at its trained seq_len
    and resized with ``ContentRouter.with_seq_len``: its scores at any offset
    equal the trained router's clamped ones."""
    if pos_bias not in ("exact", "extend"):
        raise ValueError(f"pos_bias must be 'exact' or 'extend', got {pos_bias!r}")
    state = torch.load(checkpoint, map_location=next(model.parameters()).device, weights_only=False)
    cfg_dict = state["cfg"]
    state_dict = state["state_dict"]
    if not any(key.startswith("q_proj") or key.startswith("k_proj") for key in state_dict):
        raise TypeError("only ContentRouter checkpoints are supported (PerLayerRouter is out of scope)")
    layer_module = model.model.layers[layer].self_attn
    trained = state_dict["pos_bias.weight"].shape[0] // 2
    cfg = ContentRouterConfig(
        head_dim=layer_module.head_dim,
        n_heads=layer_module.config.num_attention_heads,
        seq_len=trained if pos_bias == "extend" else seq_len,
        proj_dim=cfg_dict.get("proj_dim", 64),
    )
    router = ContentRouter(cfg).to(next(model.parameters()).device)
    router.load_state_dict(state_dict)
    router.eval()
    if pos_bias == "extend" and trained != seq_len:
        router = router.with_seq_len(seq_len).eval()
    return router


def patch_all_layers(model, mode: str, k: int, routers: Optional[dict] = None, impl: str = "gather"):
    """Convenience: patch every decoder layer (the full-model configuration)."""
    n = len(model.model.layers)
    return _patch_layer(model, PatchPlan(mode=mode, k=k, layers=tuple(range(n)), routers=routers, impl=impl))
