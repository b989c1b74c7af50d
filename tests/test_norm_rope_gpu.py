"""qk_norm_rope and the gradient of rope_to_heads against the 64-bit definition.

Tolerances: a row is fp32 arithmetic of a few roundings and a sum of D squares (its relative
error (D / 2 + 8) 2^-24 at most), rounded once at the end: |error| <= c 2^-24 size + step |value|,
step = half a step of the type, size the sum of the absolute terms.  Gradients of the weights sum
n = B N Hx terms: rel <= (sqrt(n) + D) 2^-24 + step in the norm."""

import pytest
import torch

from mod_attention_ref import rel
from ossa_b200 import qk_norm_rope, rope_to_heads

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _ref(x, w, cos, sin, heads, eps):
    B, N = x.shape[:2]
    h = x.reshape(B, N, heads, -1).transpose(1, 2)
    D = h.shape[-1]
    if w is not None:
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * w
    if cos is not None:
        c, s = cos.unsqueeze(1), sin.unsqueeze(1)
        h = h * c + torch.cat([-h[..., D // 2:], h[..., :D // 2]], dim=-1) * s
    return h


def _tables(B, N, D, seed):
    """Any values: the halves of the tables need not agree."""
    g = _gen(seed)
    return torch.randn(B, N, D, generator=g), torch.randn(B, N, D, generator=g)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _check(dtype, B, N, H, Hkv, D, *, wdtype=None, norm=(True, True), rope=True, cs_batch=None, eps=1e-6, seed=0):
    g = _gen(seed)
    q = (torch.randn(B, N, H * D, generator=g) * 3).to(dtype)
    k = (torch.randn(B, N, Hkv * D, generator=g) * 0.5).to(dtype)
    wdtype = wdtype or dtype
    wq = torch.randn(D, generator=g).to(wdtype) if norm[0] else None
    wk = torch.randn(D, generator=g).to(wdtype) if norm[1] else None
    cos = sin = None
    if rope:
        cos, sin = (t.to(dtype) for t in _tables(cs_batch or B, N, D, seed + 1))
    gq = torch.randn(B, H, N, D, generator=g).to(dtype)
    gk = torch.randn(B, Hkv, N, D, generator=g).to(dtype)
    dbl = lambda t: None if t is None else t.double()  # noqa: E731
    ref_leaves = [t.requires_grad_() for t in (dbl(q), dbl(k), dbl(wq), dbl(wk)) if t is not None]
    rl = iter(ref_leaves)
    rq, rk = next(rl), next(rl)
    rwq = next(rl) if norm[0] else None
    rwk = next(rl) if norm[1] else None
    yq = _ref(rq, rwq, dbl(cos), dbl(sin), H, eps)
    yk = _ref(rk, rwk, dbl(cos), dbl(sin), Hkv, eps)
    want = torch.autograd.grad((yq, yk), ref_leaves, (gq.double(), gk.double()))
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    dq, dk = dev(q).requires_grad_(), dev(k).requires_grad_()
    dwq = dev(wq).requires_grad_() if norm[0] else None
    dwk = dev(wk).requires_grad_() if norm[1] else None
    leaves = [t for t in (dq, dk, dwq, dwk) if t is not None]
    oq, ok = qk_norm_rope(dq, dk, H, Hkv, dwq, dwk, dev(cos), dev(sin), eps=eps)
    got = torch.autograd.grad((oq, ok), leaves, (dev(gq), dev(gk)))
    with torch.no_grad():
        nq, nk = qk_norm_rope(dq, dk, H, Hkv, dwq, dwk, dev(cos), dev(sin), eps=eps)
    assert torch.equal(nq, oq) and torch.equal(nk, ok)
    fine, step = (D / 2 + 16) * 2.0 ** -24, _half(dtype)
    for o, y in ((oq, yq), (ok, yk)):
        assert o.dtype == dtype and o.is_contiguous() and o.shape == y.shape
        err = (o.double().cpu() - y).abs()
        size = y.abs() + y.abs().amax(-1, keepdim=True)
        assert (err <= fine * size + step * y.abs() + 1e-30).all(), (err / size).max()
    for n, (a, w) in enumerate(zip(got, want)):
        a = a.cpu()
        st = step if n < 2 else _half(wdtype)
        terms = 1 if n < 2 else (B * N * max(H, Hkv)) ** 0.5
        assert a.shape == w.shape
        if w.numel():
            assert rel(a, w) <= 4 * (terms * 2.0 ** -24 + fine) + st, (n, rel(a, w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,N,H,Hkv,D", [(1, 1, 1, 1, 16), (2, 3, 12, 2, 128), (1, 77, 4, 4, 64), (3, 130, 6, 3, 32),
                                         (2, 33, 3, 1, 256), (1, 65, 5, 2, 80), (2, 9, 2, 1, 8), (1, 20, 3, 2, 512),
                                         (8, 1, 12, 2, 128), (1, 700, 8, 2, 96)])
def test_norm_and_rotation(dtype, B, N, H, Hkv, D):
    _check(dtype, B, N, H, Hkv, D, seed=D + N)


@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
def test_weight_types(dtype, wdtype):
    _check(dtype, 2, 40, 6, 2, 128, wdtype=wdtype, seed=4)


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("norm,rope", [((True, False), True), ((False, True), True), ((False, False), True),
                                       ((True, True), False), ((False, False), False)])
def test_parts_left_out(norm, rope, D):
    for dtype in (torch.bfloat16, torch.float32):
        _check(dtype, 2, 31, 4, 2, D, norm=norm, rope=rope, seed=2)


def test_one_table_for_all_and_large_eps():
    _check(torch.bfloat16, 3, 25, 4, 2, 128, cs_batch=1, eps=0.25, seed=9)


def test_row_of_zeros():
    """A head row of zeros is 0 with a positive eps, forward and backward."""
    q = torch.zeros(1, 3, 2 * 64, device=DEV, requires_grad=True)
    k = torch.randn(1, 3, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    oq, ok = qk_norm_rope(q, k, 2, 1, w, w)
    gq, gk, gw = torch.autograd.grad((oq, ok), (q, k, w), (torch.ones_like(oq), torch.ones_like(ok)))
    assert (oq == 0).all() and all(torch.isfinite(t).all() for t in (ok, gq, gk, gw))


def test_views_of_a_joint_projection():
    """Queries and keys as slices of one (B, N, (H + 2 Hkv) D) projection, read in place; other layouts
    are copied; the gradient flows into the joint tensor."""
    B, N, H, Hkv, D = 2, 37, 4, 2, 128
    g = _gen(3)
    joint = torch.randn(B, N, (H + 2 * Hkv) * D, generator=g).bfloat16().to(DEV)
    w = torch.randn(D, generator=g).bfloat16().to(DEV)
    cos, sin = (t.bfloat16().to(DEV) for t in _tables(B, N, D, 5))
    q, k = joint[..., :H * D], joint[..., H * D:(H + Hkv) * D]
    want = qk_norm_rope(q.contiguous(), k.contiguous(), H, Hkv, w, w, cos, sin)
    for qq, kk in ((q, k), (q.view(B, N, H, D), k.view(B, N, Hkv, D)),
                   (q.transpose(0, 1).contiguous().transpose(0, 1), k)):
        got = qk_norm_rope(qq, kk, H, Hkv, w, w, cos, sin)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.randn(B, N, H * D + 1, generator=g).bfloat16().to(DEV)[..., 1:]  # rows off any 16-byte boundary
    got = qk_norm_rope(odd, k, H, Hkv, w, w, cos, sin)
    assert torch.equal(got[0], qk_norm_rope(odd.contiguous(), k, H, Hkv, w, w, cos, sin)[0])
    leaf = joint.clone().requires_grad_()
    oq, ok = qk_norm_rope(leaf[..., :H * D], leaf[..., H * D:(H + Hkv) * D], H, Hkv, w, w, cos, sin)
    (gj,) = torch.autograd.grad((oq, ok), leaf, (torch.ones_like(oq), torch.ones_like(ok)))
    a, b = q.contiguous().requires_grad_(), k.contiguous().requires_grad_()
    oq, ok = qk_norm_rope(a, b, H, Hkv, w, w, cos, sin)
    ga, gb = torch.autograd.grad((oq, ok), (a, b), (torch.ones_like(oq), torch.ones_like(ok)))
    assert torch.equal(gj[..., :H * D], ga) and torch.equal(gj[..., H * D:(H + Hkv) * D], gb)
    assert (gj[..., (H + Hkv) * D:] == 0).all()


@pytest.mark.parametrize("which", [0, 1])
def test_one_output_unused(which):
    B, N, H, Hkv, D = 2, 19, 4, 2, 64
    g = _gen(8)
    leaves = [torch.randn(B, N, H * D, generator=g), torch.randn(B, N, Hkv * D, generator=g),
              torch.randn(D, generator=g), torch.randn(D, generator=g)]
    leaves = [t.to(DEV).requires_grad_() for t in leaves]
    cos, sin = (t.to(DEV) for t in _tables(B, N, D, 1))
    both = qk_norm_rope(leaves[0], leaves[1], H, Hkv, leaves[2], leaves[3], cos, sin)
    grads = torch.autograd.grad(both[which].sum(), leaves, allow_unused=True, retain_graph=True)
    full = torch.autograd.grad(both[which].sum() + 0 * both[1 - which].sum(), leaves)
    for n in (which, 2 + which):
        assert rel(grads[n], full[n]) < 1e-5
    for n in (1 - which, 3 - which):
        assert grads[n] is None or (grads[n] == 0).all()


def test_same_bits_and_differences():
    B, N, H, Hkv, D = 2, 300, 6, 2, 128
    g = _gen(5)
    base = [torch.randn(B, N, H * D, generator=g), torch.randn(B, N, Hkv * D, generator=g),
            torch.randn(D, generator=g), torch.randn(D, generator=g)]
    base = [t.to(DEV) for t in base]
    cos, sin = (t.to(DEV) for t in _tables(B, N, D, 2))
    gq = torch.randn(B, H, N, D, generator=g).to(DEV)
    gk = torch.randn(B, Hkv, N, D, generator=g).to(DEV)

    def grads():
        leaves = [t.clone().requires_grad_() for t in base]
        o = qk_norm_rope(leaves[0], leaves[1], H, Hkv, leaves[2], leaves[3], cos, sin)
        return torch.autograd.grad(o, leaves, (gq, gk))

    first = grads()
    assert all(torch.equal(a, b) for _ in range(4) for a, b in zip(first, grads()))

    def f(t):
        o = qk_norm_rope(t[0], t[1], H, Hkv, t[2], t[3], cos, sin)
        return ((o[0].double() * gq).sum() + (o[1].double() * gk).sum()).item()

    h = 2.0 ** -8  # error: h^2/6 third derivative (order 1 per unit of the direction) + 2^-24 sqrt(n) / h
    for n in range(4):
        d = torch.randn(base[n].shape, generator=_gen(30 + n)).to(DEV)
        diff = (f([t + h * d if i == n else t for i, t in enumerate(base)]) -
                f([t - h * d if i == n else t for i, t in enumerate(base)])) / (2 * h)
        want = (first[n].double() * d).sum().item()
        assert abs(diff - want) <= 1e-3 * first[n].double().norm().item() * d.abs().max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,rope", [(128, True), (64, False), (40, True)])
def test_rope_to_heads_gradient(dtype, D, rope):
    """rope_to_heads under autograd: the same values as without, and the transposed rotation back."""
    B, N, H = 2, 45, 3
    g = _gen(D)
    x = torch.randn(B, N, H * D, generator=g).to(dtype)
    cos, sin = (t.to(dtype) for t in _tables(1, N, D, 3)) if rope else (None, None)
    go = torch.randn(B, H, N, D, generator=g).to(dtype)
    xr = x.double().requires_grad_()
    y = _ref(xr, None, None if cos is None else cos.double(), None if sin is None else sin.double(), H, 0.0)
    (want,) = torch.autograd.grad(y, xr, go.double())
    dev = [None if t is None else t.to(DEV) for t in (cos, sin)]
    leaf = x.to(DEV).requires_grad_()
    out = rope_to_heads(leaf, H, *dev)
    assert torch.equal(out.detach(), rope_to_heads(x.to(DEV), H, *dev))
    (got,) = torch.autograd.grad(out, leaf, go.to(DEV))
    assert rel(got.cpu(), want) <= _half(dtype) + 4 * 2.0 ** -24


def test_captured_step_replays():
    B, N, H, Hkv, D = 2, 64, 12, 2, 128
    g = _gen(5)
    q, k = (torch.randn(B, N, h * D, generator=g).bfloat16().to(DEV) for h in (H, Hkv))
    w = torch.randn(D, generator=g).bfloat16().to(DEV)
    cos, sin = (t.bfloat16().to(DEV) for t in _tables(B, N, D, 2))

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, w)]
        o = qk_norm_rope(leaves[0], leaves[1], H, Hkv, leaves[2], leaves[2], cos, sin)
        return list(o) + list(torch.autograd.grad(o, leaves, o))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    q.copy_(torch.randn(q.shape, generator=_gen(77)).to(q))
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a.detach(), b.detach()) for a, b in zip(kept, want))


def test_empty():
    q = torch.zeros(2, 0, 4 * 64, device=DEV, requires_grad=True)
    k = torch.zeros(2, 0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    oq, ok = qk_norm_rope(q, k, 4, 1, w, w)
    assert oq.shape == (2, 4, 0, 64) and ok.shape == (2, 1, 0, 64)
    grads = torch.autograd.grad((oq, ok), (q, k, w), (torch.empty_like(oq), torch.empty_like(ok)))
    assert grads[0].shape == q.shape and (grads[2] == 0).all()
