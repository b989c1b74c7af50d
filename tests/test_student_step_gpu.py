"""A training step of the sparse model against its dense teacher, the operators together: patched
decoder layers (head norms with rotation, selection, gathered attention with a score cap and packed
documents) and the top-logit distillation loss, forward and backward, against 64 bits.

The 64-bit model takes the key lists that the fp32 run selected (a near-tie may order otherwise).
Tolerance: three fp32 layers of products up to 256 terms; each step's relative error is below
(256 + 8) 2^-24 (1 + |score|), about 1e-4 with scores up to 6, and some ten of them follow one another
on the way to any gradient: 1e-3 in the norm of each parameter's gradient."""

import copy

import pytest
import torch

from mod_attention_ref import attention, rel
from ossa_b200 import ContentRouter, ContentRouterConfig, top_logit_distillation_loss
from ossa_b200.bench import sparse_forward
from ossa_b200.bench.sparse_forward import PatchPlan, _patch_layer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class HeadNorm(torch.nn.Module):
    def __init__(self, dim, eps=1e-5):
        super().__init__()
        self.weight = torch.nn.Parameter(1.0 + 0.3 * torch.randn(dim, generator=torch.Generator().manual_seed(dim)))
        self.eps = eps

    def forward(self, x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.eps) * self.weight


def _model(norms, seed=0):
    from transformers import Qwen2Config, Qwen2ForCausalLM

    cfg = Qwen2Config(hidden_size=256, intermediate_size=320, num_hidden_layers=3, num_attention_heads=4,
                      num_key_value_heads=2, vocab_size=301, max_position_embeddings=256, rope_theta=1e4)
    torch.manual_seed(seed)
    model = Qwen2ForCausalLM(cfg).eval()
    if norms:
        for layer in model.model.layers:
            layer.self_attn.q_norm = HeadNorm(layer.self_attn.head_dim)
            layer.self_attn.k_norm = HeadNorm(layer.self_attn.head_dim)
    return model


def _patch_64(model, lists, opts):
    """The patched layers' mathematics in the model's own type, over recorded key lists."""
    from transformers.models.qwen2.modeling_qwen2 import apply_rotary_pos_emb

    for li, layer in enumerate(model.model.layers):
        attn = layer.self_attn

        def fwd(hidden_states, position_embeddings=None, _attn=attn, _li=li, **kw):
            B, N, _ = hidden_states.shape
            D, H, Hkv = _attn.head_dim, _attn.config.num_attention_heads, _attn.config.num_key_value_heads
            q = _attn.q_proj(hidden_states).view(B, N, H, D)
            k = _attn.k_proj(hidden_states).view(B, N, Hkv, D)
            v = _attn.v_proj(hidden_states).view(B, N, Hkv, D).transpose(1, 2)
            if hasattr(_attn, "q_norm"):
                q, k = _attn.q_norm(q), _attn.k_norm(k)
            cos, sin = position_embeddings
            q, k = apply_rotary_pos_emb(q.transpose(1, 2), k.transpose(1, 2), cos, sin)
            out, _, _ = attention(q, k, v, lists[_li], **opts)
            return _attn.o_proj(out.transpose(1, 2).reshape(B, N, H * D)), None

        attn.forward = fwd


@pytest.mark.parametrize("mode,impl", [("router", "gather"), ("oracle", "mask")])
@pytest.mark.parametrize("norms", [True, False])
@pytest.mark.parametrize("modified", [True, False])
def test_step(mode, impl, norms, modified, monkeypatch):
    B, N, K = 2, 120, 16
    model = _model(norms)
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 301, (B, N), generator=g)
    teacher_ids = torch.rand(B, N, 301, generator=g).topk(24, dim=-1).indices
    teacher = torch.randn(B, N, 24, generator=g) * 2
    weight = (torch.rand(B, N, generator=g) < 0.8).float()
    opts = {}
    if modified:
        opts = dict(softcap=4.0, slopes=torch.tensor([0.0, 0.02, 0.05, 0.1]),
                    segments=torch.sort(torch.randint(0, 3, (B, N), generator=g), dim=1).values, prefix_len=7)
    routers = None
    if mode == "router":
        routers = {}
        for li in range(3):
            torch.manual_seed(li)
            routers[li] = ContentRouter(ContentRouterConfig(head_dim=64, n_heads=4, seq_len=N, proj_dim=64)).to(DEV)

    lists = {}
    plain = sparse_forward.select_indices

    def record(plan, li, q, k):
        idx = plain(plan, li, q, k)
        lists[li] = idx.cpu()
        return idx

    monkeypatch.setattr(sparse_forward, "select_indices", record)
    gpu = copy.deepcopy(model).to(DEV)
    dev = {n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in opts.items()}
    restore = _patch_layer(gpu, PatchPlan(mode=mode, k=K, layers=(0, 1, 2), routers=routers, impl=impl, **dev))
    logits = gpu(input_ids=ids.to(DEV), use_cache=False).logits
    loss = top_logit_distillation_loss(logits[:, :-1], teacher[:, :-1].to(DEV), teacher_ids[:, :-1].to(DEV), temperature=2.0,
                                       row_weight=weight[:, :-1].to(DEV))
    loss.backward()
    restore()

    ref = copy.deepcopy(model).double()
    _patch_64(ref, lists, {n: t.double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t
                           for n, t in opts.items()})
    z = ref(input_ids=ids, use_cache=False).logits[:, :-1].double()
    p = torch.softmax(teacher[:, :-1].double() / 2, -1)
    lq = torch.log_softmax(z / 2, -1).gather(-1, teacher_ids[:, :-1])
    w = weight[:, :-1].double()
    want = 4 * ((p * (torch.log(p) - lq)).sum(-1) * w).sum() / w.sum()
    want.backward()
    assert rel(logits.detach().cpu()[:, :-1], z) < 1e-3
    assert abs(loss.item() - want.item()) < 1e-3 * abs(want.item())
    checked = 0
    named = dict(ref.named_parameters())
    for name, param in gpu.named_parameters():
        grad = named[name].grad
        if grad is None or grad.norm() == 0:
            assert param.grad is None or param.grad.norm() == 0, name
            continue
        if name.endswith("k_proj.bias") and not norms and not modified:
            # a common shift of a row's keys changes no softmax where rotation leaves it common: the true
            # gradient is what the rotation's spread leaves, compared on the scale of the weight's gradient
            scale = named[name.replace("bias", "weight")].grad.norm()
            assert (param.grad.double().cpu() - grad).norm() < 1e-3 * scale, name
        else:
            assert rel(param.grad.cpu(), grad) < 1e-3, (name, rel(param.grad.cpu(), grad))
        checked += 1
    assert checked >= 30
    for r in (routers or {}).values():
        assert all(t.grad is None for t in r.parameters())  # the selection is a constant


def test_norms_that_are_not_rms_are_refused():
    model = _model(True)
    model.model.layers[1].self_attn.k_norm = torch.nn.LayerNorm(64)
    with pytest.raises(TypeError):
        _patch_layer(model, PatchPlan(mode="oracle", k=4, layers=(0, 1, 2)))
    model.model.layers[1].self_attn.k_norm = HeadNorm(64, eps=1e-3)
    with pytest.raises(TypeError):
        _patch_layer(model, PatchPlan(mode="oracle", k=4, layers=(0, 1, 2)))


def test_prefill_then_single_tokens():
    """Serving with the modifiers: a prompt's rows in one call and the following tokens one by one, against
    the whole sequence in one call (bf16; both round p at most and the output: 4 steps)."""
    from ossa_b200 import qk_norm_rope, topk_attention
    from ossa_b200.select import oracle_topk

    B, H, Hkv, N, D, K, n0 = 2, 6, 2, 260, 128, 32, 250
    g = torch.Generator().manual_seed(3)
    x = [torch.randn(B, N, h * D, generator=g).bfloat16().to(DEV) for h in (H, Hkv, Hkv)]
    w = (1 + 0.1 * torch.randn(D, generator=g)).bfloat16().to(DEV)
    pos = torch.arange(N).double()[:, None] / 1e4 ** (torch.arange(0, D, 2) / D)
    cos, sin = (torch.cat([f(pos), f(pos)], -1).bfloat16().to(DEV) for f in (torch.cos, torch.sin))
    q, k = qk_norm_rope(x[0], x[1], H, Hkv, w, w, cos, sin)
    v = x[2].view(B, N, Hkv, D).transpose(1, 2).contiguous()
    idx = oracle_topk(q, k, K)
    opts = dict(softcap=10.0, slopes=torch.linspace(0, 0.1, H).to(DEV), prefix_len=torch.tensor([5, 9], device=DEV))
    full = topk_attention(q, k, v, topk_indices=idx, **opts)
    kc, vc = torch.full_like(k, float("nan")), torch.full_like(v, float("nan"))  # a cache that fills up
    qp, kp = qk_norm_rope(x[0][:, :n0], x[1][:, :n0], H, Hkv, w, w, cos[:n0], sin[:n0])
    kc[:, :, :n0], vc[:, :, :n0] = kp, v[:, :, :n0]
    out = [topk_attention(qp, kc[:, :, :n0].contiguous(), vc[:, :, :n0].contiguous(),
                          topk_indices=idx[:, :, :n0].contiguous(), **opts)]
    for t in range(n0, N):
        q1, k1 = qk_norm_rope(x[0][:, t:t + 1], x[1][:, t:t + 1], H, Hkv, w, w, cos[t:t + 1], sin[t:t + 1])
        assert torch.equal(q1, q[:, :, t:t + 1]) and torch.equal(k1, k[:, :, t:t + 1])
        kc[:, :, t:t + 1], vc[:, :, t:t + 1] = k1, v[:, :, t:t + 1]
        out.append(topk_attention(q1, kc, vc, topk_indices=idx[:, :, t:t + 1].contiguous(), q_start=t, **opts))
    assert rel(torch.cat(out, dim=2), full) < 4 * 2.0 ** -8


def _step_of_all(q, k, v, w, table, idx, segments, teacher, teacher_ids, out_w):
    """The operators one after another, from projections to a loss."""
    from ossa_b200 import qk_norm_rope, rope_to_heads, topk_attention

    qr, kr = qk_norm_rope(q, k, 4, 2, w, w, table[0], table[1])
    vr = rope_to_heads(v, 2)
    out = topk_attention(qr, kr, vr, topk_indices=idx, softcap=5.0, segments=segments)
    return top_logit_distillation_loss(out.transpose(1, 2).flatten(2) @ out_w, teacher, teacher_ids)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_checkpointed_offloaded_and_two_at_once(dtype):
    """Saved tensors that come back as other tensors (non-reentrant checkpointing, offloading to the
    host), joint projections whose slices are read in place, two steps on two streams at once: the same
    bits as the plain step."""
    from torch.utils.checkpoint import checkpoint

    B, N, D = 2, 90, 128
    g = torch.Generator().manual_seed(11)

    def make(seed):
        g.manual_seed(seed)
        joint = torch.randn(B, N, 8 * D, generator=g).to(dtype).to(DEV).requires_grad_()
        w = torch.randn(D, generator=g).to(dtype).to(DEV).requires_grad_()
        table = torch.randn(2, 1, N, D, generator=g).to(dtype).to(DEV)
        idx = torch.randint(-1, N, (B, 4, N, 20), generator=g).int().to(DEV)
        seg = torch.sort(torch.randint(0, 2, (B, N), generator=g), dim=1).values.to(DEV)
        teacher = torch.randn(B, N, 12, generator=g).to(DEV)
        ids = torch.randint(0, 77, (B, N, 12), generator=g).to(DEV)
        out_w = torch.randn(4 * D, 77, generator=g).to(dtype).to(DEV).requires_grad_()
        return joint, w, out_w, (table, idx, seg, teacher, ids)

    def loss_of(joint, w, out_w, rest):
        table, idx, seg, teacher, ids = rest
        return _step_of_all(joint[..., :4 * D], joint[..., 4 * D:6 * D], joint[..., 6 * D:], w, table, idx, seg, teacher, ids,
                            out_w)

    def grads(run, args):
        loss = run(args)
        return [loss.detach()] + list(torch.autograd.grad(loss, args[:3]))

    args, other = make(1), make(2)
    want = grads(lambda a: loss_of(*a), args)
    want_other = grads(lambda a: loss_of(*a), other)
    got = grads(lambda a: checkpoint(loss_of, *a, use_reentrant=False), args)
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    def offloaded(a):
        with torch.autograd.graph.save_on_cpu():
            return loss_of(*a)

    assert all(torch.equal(a, b) for a, b in zip(want, grads(offloaded, args)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    both = []
    for s, a in zip(streams, (args, other)):
        with torch.cuda.stream(s):
            both.append(grads(lambda x: loss_of(*x), a))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, both[0]))
    assert all(torch.equal(a, b) for a, b in zip(want_other, both[1]))


def test_an_unaligned_index_slice():
    """Index rows that begin off any 16-byte boundary (K = 5, a slice of the batch)."""
    from ossa_b200 import topk_attention

    g = torch.Generator().manual_seed(1)
    q = torch.randn(3, 2, 7, 64, generator=g).to(DEV)
    idx = torch.randint(0, 7, (3, 2, 7, 5), generator=g).int().to(DEV)
    whole = topk_attention(q, q, q, topk_indices=idx, softcap=3.0)
    x = q[1:].clone().requires_grad_()
    part = topk_attention(x, x, x, topk_indices=idx[1:], softcap=3.0)
    assert torch.equal(part.detach(), whole[1:])
    assert torch.isfinite(torch.autograd.grad(part.sum(), x)[0]).all()
