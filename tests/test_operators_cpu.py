"""Refusals of the modified attention, the head norm and the top-logit distillation: bad arguments are
turned down before anything reaches a device, by the C ABI and by the Python entry points."""

import pytest
import torch

from ossa_b200 import _lib, qk_norm_rope, rope_to_heads, top_logit_distillation_loss, topk_attention

INV, UNS, WS, OK = _lib.OSSA_ERR_INVALID, _lib.OSSA_ERR_UNSUPPORTED, _lib.OSSA_ERR_WORKSPACE, _lib.OSSA_OK
BF, F32 = _lib.OSSA_BF16, _lib.OSSA_F32
INF, NAN = float("inf"), float("nan")


def _mod_fwd(**kw):
    a = dict(q=16, k=16, v=16, idx=16, i64=0, dtype=BF, B=1, H=4, Hkv=2, Nq=8, Nk=8, D=128, K=4, scale=0.1, causal=1,
             q0=0, cap=0.0, slopes=None, seg=None, prefix=None, out=16, lse=16, rest=None, stream=None)
    a.update(kw)
    return _lib.lib().ossa_topk_attention_mod_fwd(*a.values())


def _mod_bwd(**kw):
    a = dict(q=16, k=16, v=16, idx=16, i64=0, dtype=BF, B=1, H=4, Hkv=2, Nq=8, Nk=8, D=128, K=4, scale=0.1, causal=1,
             q0=0, cap=0.0, slopes=None, seg=None, prefix=None, out=16, lse=16, rest=None, dout=16, dq=16, dk=16, dv=16,
             dslopes=None, ws=256, wsb=1 << 30, stream=None)
    a.update(kw)
    return _lib.lib().ossa_topk_attention_bwd(*a.values())


BAD_MOD = [(dict(H=5), INV), (dict(D=96), UNS), (dict(dtype=3), INV), (dict(K=-1), INV), (dict(i64=2), INV),
           (dict(scale=NAN), INV), (dict(cap=-1.0), INV), (dict(cap=INF), INV), (dict(cap=NAN), INV),
           (dict(q0=-1), INV), (dict(seg=16, q0=1), INV), (dict(B=40000, H=2, Hkv=2), UNS), (dict(q=None), INV),
           (dict(k=8), INV), (dict(idx=18), INV), (dict(idx=None), INV), (dict(Nk=0), INV),
           (dict(rest=24), INV), (dict(rest=16, dtype=F32), INV)]


@pytest.mark.parametrize("kw,code", BAD_MOD)
def test_modified_attention_refusals(kw, code):
    assert _mod_fwd(**kw) == code
    assert _mod_bwd(**kw) == code


def test_attention_backward_refusals():
    assert _mod_bwd(dslopes=16) == INV  # without slopes
    assert _mod_bwd(lse=None) == INV and _mod_bwd(dq=None) == INV and _mod_bwd(dv=24) == INV
    need = _lib.lib().ossa_topk_attention_bwd_workspace_size(BF, 1, 4, 2, 8, 8, 128, 4, 0)
    assert need > 0 and _mod_bwd(wsb=need - 1) == WS and _mod_bwd(ws=None) == WS
    assert _mod_bwd(Nq=1 << 20, Nk=1 << 20, K=1024) == UNS  # more than 2^30 listed keys per kv head
    assert _mod_fwd(B=0) == OK and _mod_fwd(Nq=0) == OK
    assert _lib.lib().ossa_topk_attention_bwd_workspace_size(BF, 1, 4, 3, 8, 8, 128, 4, 0) == 0


def _norm(fn="fwd", **kw):
    a = dict(q=16, k=16, wq=16, wk=16, cos=16, sin=16, batched=0, dtype=BF, wdtype=BF, B=1, N=4, Hq=4, Hk=2, D=128,
             qsb=0, qsn=512, ksb=0, ksn=256, eps=1e-6)
    tail = dict(qo=16, ko=16, stream=None) if fn == "fwd" else dict(gq=16, gk=16, dq=16, dk=16, dwq=None, dwk=None,
                                                                     ws=256, wsb=1 << 30, stream=None)
    a.update(tail)
    a.update(kw)
    return getattr(_lib.lib(), f"ossa_qk_norm_rope_{fn}")(*a.values())


@pytest.mark.parametrize("kw,code", [(dict(dtype=5), INV), (dict(wdtype=5), INV), (dict(D=12), INV), (dict(D=520), UNS),
                                     (dict(Hq=0), INV), (dict(Hk=-1), INV), (dict(N=-1), INV), (dict(eps=-1.0), INV),
                                     (dict(eps=NAN), INV), (dict(sin=None), INV), (dict(qsn=4), INV),
                                     (dict(ksb=3), INV), (dict(q=8), INV), (dict(q=None), INV)])
@pytest.mark.parametrize("fn", ["fwd", "bwd"])
def test_norm_rope_refusals(kw, code, fn):
    assert _norm(fn, **kw) == code


def test_norm_rope_more():
    assert _norm("fwd", qo=None) == INV and _norm("fwd", ko=8) == INV and _norm("fwd", B=0) == OK
    assert _norm("bwd", gq=None) == INV and _norm("bwd", dwq=16, wq=None) == INV
    need = _lib.lib().ossa_qk_norm_rope_bwd_workspace_size(128)
    assert need > 0 and _norm("bwd", wsb=need - 1) == WS and _norm("bwd", ws=None) == WS


def _distill(fn="fwd", **kw):
    a = dict(z=16, dtype=BF, outer=1, inner=4, V=100, so=0, si=100)
    if fn == "fwd":
        a.update(teacher=16, ids=16, i64=0, K=8, tau=1.0, w=None, mean=1, rows=None, loss=16, dz=16, ws=256, wsb=1 << 20,
                 stream=None)
    else:
        a.update(ids=16, i64=0, K=8, tau=1.0, mean=1, grad=16, per_row=0, skip=0, dz=16, ws=256, wsb=1 << 20, stream=None)
    a.update(kw)
    return getattr(_lib.lib(), f"ossa_top_logit_distill_{fn}")(*a.values())


@pytest.mark.parametrize("kw,code", [(dict(dtype=9), INV), (dict(V=0), INV), (dict(K=0), INV), (dict(K=1025), UNS),
                                     (dict(inner=0), INV), (dict(outer=-1), INV), (dict(outer=1 << 20, inner=1 << 20), UNS),
                                     (dict(i64=3), INV), (dict(tau=0.0), INV), (dict(tau=-1.0), INV), (dict(tau=NAN), INV),
                                     (dict(tau=INF), INV), (dict(z=None), INV), (dict(z=17), INV), (dict(ids=None), INV),
                                     (dict(wsb=10), WS), (dict(ws=None), WS)])
@pytest.mark.parametrize("fn", ["fwd", "bwd"])
def test_distill_refusals(kw, code, fn):
    assert _distill(fn, **kw) == code


def test_distill_more():
    assert _distill("fwd", teacher=None) == INV and _distill("fwd", loss=None) == INV
    assert _distill("bwd", grad=None) == INV and _distill("bwd", dz=None) == INV
    assert _distill("bwd", per_row=1, skip=1) == INV
    assert _lib.lib().ossa_top_logit_distill_workspace_size(10, 0) == 0


# ------------------------------------------------------------------ Python entry points


def _qkv(H=4, Hkv=2, Nq=8, Nk=8, D=64, K=4, dtype=torch.float32):
    return (torch.zeros(1, H, Nq, D, dtype=dtype), torch.zeros(1, Hkv, Nk, D, dtype=dtype),
            torch.zeros(1, Hkv, Nk, D, dtype=dtype), torch.zeros(1, H, Nq, K, dtype=torch.int32))


@pytest.mark.parametrize("kw,err", [
    (dict(softcap=0.0), ValueError), (dict(softcap=-2.0), ValueError), (dict(softcap=INF), ValueError),
    (dict(softcap=NAN), ValueError), (dict(slopes=torch.zeros(3)), ValueError),
    (dict(slopes=torch.zeros(4, dtype=torch.int32)), ValueError),
    (dict(segments=torch.zeros(1, 7, dtype=torch.int32)), ValueError), (dict(segments=torch.zeros(1, 8)), TypeError),
    (dict(segments=torch.zeros(8, dtype=torch.int32), q_start=1), ValueError), (dict(prefix_len=-1), ValueError),
    (dict(prefix_len=torch.zeros(2, dtype=torch.int32)), ValueError), (dict(prefix_len=torch.zeros(1)), TypeError),
    (dict(prefix_len=1.5), TypeError), (dict(softcap=1.0, q_start=-1), ValueError),
    (dict(softcap=1.0), RuntimeError),  # CPU tensors
])
def test_topk_attention_refusals(kw, err):
    q, k, v, idx = _qkv()
    with pytest.raises(err):
        topk_attention(q, k, v, topk_indices=idx, **kw)


def test_topk_attention_types():
    q, k, v, idx = _qkv(dtype=torch.float16)
    with pytest.raises(TypeError):
        topk_attention(q, k, v, topk_indices=idx, softcap=2.0)
    q, k, v, idx = _qkv()
    with pytest.raises(TypeError):
        topk_attention(q, k, v, topk_indices=idx.float(), softcap=2.0)
    with pytest.raises(TypeError):
        topk_attention(q, k.bfloat16(), v, topk_indices=idx, softcap=2.0)


def test_qk_norm_rope_refusals():
    q, k, w = torch.zeros(1, 3, 4 * 64), torch.zeros(1, 3, 2 * 64), torch.zeros(64)
    cos = torch.zeros(1, 3, 64)
    for args, kw, err in [((q, k, 4, 2, w, w, cos, None), {}, ValueError), ((q, k, 3, 2, w, w), {}, ValueError),
                          ((q, k, 4, 1, w, w), {}, ValueError), ((q, k, 0, 2, w, w), {}, ValueError),
                          ((q, k[:, :2], 4, 2, w, w), {}, ValueError), ((q, k, 4, 2, w[:32], w), {}, ValueError),
                          ((q, k, 4, 2, w.int(), w), {}, ValueError), ((q, k.bfloat16(), 4, 2, w, w), {}, TypeError),
                          ((q.half(), k.half(), 4, 2, w, w), {}, TypeError), ((q, k, 4, 2, w, w), {"eps": -1.0}, ValueError),
                          ((q, k, 4, 2, w, w), {"eps": NAN}, ValueError), ((q[0], k[0], 4, 2, w, w), {}, ValueError),
                          ((q, k, 4, 2, w, w, cos, cos), {}, RuntimeError)]:
        with pytest.raises(err):
            qk_norm_rope(*args, **kw)


def test_rope_to_heads_refuses_cpu_under_autograd():
    with pytest.raises(RuntimeError):
        rope_to_heads(torch.zeros(1, 3, 128, requires_grad=True), 2)


@pytest.mark.parametrize("kw,err", [
    (dict(temperature=0.0), ValueError), (dict(temperature=NAN), ValueError), (dict(reduction="avg"), ValueError),
    (dict(teacher_indices=torch.zeros(5, 3)), TypeError), (dict(teacher_indices=torch.zeros(4, 3, dtype=torch.int64)), ValueError),
    (dict(teacher_logits=torch.zeros(5, 2)), ValueError), (dict(row_weight=torch.zeros(4)), ValueError),
    (dict(logits=torch.zeros(5, 9, dtype=torch.int64)), ValueError), ({}, RuntimeError),
])
def test_distillation_loss_refusals(kw, err):
    a = dict(logits=torch.zeros(5, 9), teacher_logits=torch.zeros(5, 3), teacher_indices=torch.zeros(5, 3, dtype=torch.int64))
    a.update(kw)
    with pytest.raises(err):
        top_logit_distillation_loss(**a)


def test_patching_refuses_other_norms():
    """A norm that stores its weight as an offset from 1 is not the one that the patched layer computes."""
    from types import SimpleNamespace

    from ossa_b200.bench.sparse_forward import _head_norms

    class Norm(torch.nn.Module):
        def __init__(self, offset, dtype):
            super().__init__()
            self.offset, self.eps = offset, 1e-6
            self.weight = torch.nn.Parameter((0.9 + 0.2 * torch.rand(64, generator=torch.Generator().manual_seed(1))).to(dtype))

        def forward(self, x):
            return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.eps) * (self.offset + self.weight)

    for dtype in (torch.float32, torch.bfloat16):
        good, other = Norm(0.0, dtype), Norm(1.0, dtype)
        wq, wk, eps = _head_norms(SimpleNamespace(q_norm=good, k_norm=good, head_dim=64))
        assert wq is good.weight and wk is good.weight and eps == 1e-6
        with pytest.raises(TypeError):
            _head_norms(SimpleNamespace(q_norm=good, k_norm=other, head_dim=64))


def test_the_backward_workspace_of_refused_sizes():
    assert _lib.lib().ossa_topk_attention_bwd_workspace_size(BF, 1, 4, 2, 1 << 20, 1 << 20, 128, 1024, 0) == 0
