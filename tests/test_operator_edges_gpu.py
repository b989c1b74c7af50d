"""Training calls at their edges: gradients and inputs off 16-byte boundaries, saved tensors that come back in
another layout, rows that are not finite beside rows that are, lists in any order."""

import gc

import pytest
import torch

from mod_attention_ref import attention, rel, score_step
from ossa_b200 import qk_norm_rope, rope_to_heads, top_logit_distillation_loss, topk_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
STEP = 2.0 ** -8


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distillation_of_offloaded_slices(dtype, reduction):
    """Logits that are a slice of a larger tensor, saved by a hook that packs them: the backward pass reads
    them in the layout in which they come back."""
    g = _gen(3)
    B, N, V, K = 3, 9, 333, 7
    whole = (torch.randn(B, N, V, generator=g) * 2).to(dtype).to(DEV).requires_grad_()
    ids = torch.rand(B, N - 1, V, generator=g).topk(K, dim=-1).indices.to(DEV)
    teacher = torch.randn(B, N - 1, K, generator=g).to(DEV)
    dl = torch.rand((B, N - 1) if reduction == "none" else (), generator=g).to(DEV) + 1.5  # not 1: computed anew

    def run():
        loss = top_logit_distillation_loss(whole[:, :-1], teacher, ids, temperature=2.0, reduction=reduction)
        return torch.autograd.grad(loss, whole, dl)[0]

    want = run()
    with torch.autograd.graph.save_on_cpu():
        got = run()
    # Not the same bits: a row of 333 values begins elsewhere between 16-byte boundaries in the packed copy, and its
    # sum is split at those.  Either result is within 2^-18 (softmax + p) scale and half a step of the gradient.
    z = whole.detach()[:, :-1].double()
    p = torch.zeros_like(z).scatter_add_(-1, ids, torch.softmax(teacher.double() / 2.0, -1))
    scale = 2.0 * (dl.double().unsqueeze(-1) if reduction == "none" else dl.double() / ids[..., 0].numel())
    bound = 2 * (2.0 ** -18 * (torch.softmax(z / 2.0, -1) + p) * scale + want[:, :-1].double().abs() * torch.finfo(dtype).eps)
    assert ((want - got)[:, :-1].double().abs() <= bound).all()
    assert (want[:, :-1] != 0).any(-1).all() and (want[:, -1] == 0).all() and (got[:, -1] == 0).all()


def _shifted(t):
    """t's values as a contiguous tensor one element off a 16-byte boundary."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.flatten()
    x = flat[1:].view(t.shape)
    assert x.is_contiguous() and x.data_ptr() % 16
    return x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 6, 2, 40, 128, 9), (1, 2, 2, 33, 64, 5)])
def test_attention_off_boundaries(dtype, shape):
    B, H, Hkv, N, D, K = shape
    g = _gen(5)
    q, do = ((torch.randn(B, H, N, D, generator=g)).to(dtype).to(DEV) for _ in range(2))
    k, v = ((torch.randn(B, Hkv, N, D, generator=g)).to(dtype).to(DEV) for _ in range(2))
    idx = torch.randint(0, N, (B, H, N, K), generator=g).to(DEV)

    def run(place):
        leaves = [place(t).detach().requires_grad_() for t in (q, k, v)]
        out = topk_attention(*leaves, topk_indices=idx, softcap=4.0)
        return (out.detach(), *torch.autograd.grad(out, leaves, place(do)))

    assert all(torch.equal(a, b) for a, b in zip(run(lambda t: t), run(_shifted)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 40])
def test_norms_off_boundaries(dtype, D):
    B, N, Hq, Hk = 2, 11, 4, 2
    g = _gen(7)
    q, k = (torch.randn(B, N, h * D, generator=g).to(dtype).to(DEV) for h in (Hq, Hk))
    wq, wk = (torch.rand(D, generator=g).to(DEV) + 0.5 for _ in range(2))
    cos, sin = (torch.randn(1, N, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    gq, gk = (torch.randn(B, h, N, D, generator=g).to(dtype).to(DEV) for h in (Hq, Hk))

    def run(place):
        leaves = [place(t).detach().requires_grad_() for t in (q, k, wq, wk)]
        c, s = place(cos), place(sin)
        out = qk_norm_rope(leaves[0], leaves[1], Hq, Hk, leaves[2], leaves[3], c, s)
        grads = torch.autograd.grad(out, leaves, (place(gq), place(gk)))
        x = q.clone().requires_grad_()
        rope = rope_to_heads(x, Hq, cos, sin)
        return (*[t.detach() for t in out], *grads, *torch.autograd.grad(rope, x, place(gq)))

    assert all(torch.equal(a, b) for a, b in zip(run(lambda t: t), run(_shifted)))


def _bounds(q, k, D, K, dtype):
    """(of the output, of a gradient) in the norm of a tensor: two and three roundings of the type."""
    fine = score_step(q, k) + (K + D) * 2.0 ** -24
    step = STEP if dtype == torch.bfloat16 else 0.0
    return 2 * step + 8 * fine, 3 * step + 8 * fine


@pytest.mark.parametrize("dtype,H,Hkv", [(torch.bfloat16, 6, 2), (torch.bfloat16, 8, 1), (torch.bfloat16, 2, 2),
                                         (torch.bfloat16, 9, 1), (torch.float32, 4, 2)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("repeats", [False, True])
def test_padding_that_is_not_finite(dtype, H, Hkv, bad, repeats):
    """Behind the sequence lies padding, a segment of its own, whose rows hold anything; its first keys share a
    block of 8 with the last real ones.  Real rows and keys get what they get without it."""
    B, N, real, D, K = 1, 700, 687, 128, 32
    g = _gen(11)
    q, do = (torch.randn(B, H, N, D, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(B, Hkv, N, D, generator=g).to(dtype) for _ in range(2))
    idx = torch.rand(B, H, N, N, generator=g).topk(K, dim=-1).indices
    idx[:, :, real:, :3] = torch.tensor([real, real + 1, 5])  # padding lists padding (and what it does not see)
    idx = idx.sort(dim=-1).values
    if repeats:
        idx[..., 1] = idx[..., 0]
    seg = (torch.arange(N) >= real).int()
    clean = [t[:, :, :real].double().requires_grad_() for t in (q, k, v)]
    lists = torch.where(idx[:, :, :real] < real, idx[:, :, :real], -1)
    ref = attention(*clean, lists, causal=False)[0]
    want = torch.autograd.grad(ref, clean, do[:, :, :real].double())
    for t in (q, k, v, do):
        t[:, :, real:] = bad
    dev = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = topk_attention(*dev, topk_indices=idx.to(DEV), causal=False, segments=seg.to(DEV))
    got = torch.autograd.grad(out, dev, do.to(DEV))
    of_out, of_grad = _bounds(q[:, :, :real], k[:, :, :real], D, K, dtype)
    assert rel(out.detach().cpu()[:, :, :real], ref.detach()) <= of_out
    for name, x, w in zip(("dq", "dk", "dv"), got, want):
        assert rel(x.cpu()[:, :, :real], w) <= of_grad, name


@pytest.mark.parametrize("H,N,K", [(3, 1400, 32), (8, 520, 32), (4, 13000, 8)])
def test_a_key_that_one_head_lists_is_not_finite(H, N, K):
    """The other heads of the group get what they get without it."""
    B, D, key = 1, 128, 5
    dtype = torch.bfloat16
    g = _gen(13)
    q, do = (torch.randn(B, H, N, D, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(B, 1, N, D, generator=g).to(dtype) for _ in range(2))
    idx = torch.randint(0, N, (B, H, N, K), generator=g).sort(dim=-1).values
    idx[idx == key] = -1
    ref_in = [t.double() for t in (q, k, v)]
    ref_in[0].requires_grad_()
    ref = attention(*ref_in, idx, causal=False)[0]
    (want,) = torch.autograd.grad(ref, ref_in[:1], do.double())
    of_out, of_grad = _bounds(q, k, D, K, dtype)
    idx[:, 0, :, 3] = key
    k[0, 0, key] = float("inf")
    v[0, 0, key] = float("nan")
    dev = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = topk_attention(*dev, topk_indices=idx.to(DEV), causal=False)
    dq = torch.autograd.grad(out, dev, do.to(DEV))[0]
    assert rel(out.detach().cpu()[:, 1:], ref.detach()[:, 1:]) <= of_out
    assert rel(dq.cpu()[:, 1:], want[:, 1:]) <= of_grad


@pytest.mark.parametrize("dtype,H,Hkv,D", [(torch.bfloat16, 6, 2, 128), (torch.float32, 2, 2, 64)])
def test_lists_in_any_order(dtype, H, Hkv, D):
    """Many entries of a row in one block of keys, in any order, repeats among them: the same gradients for
    the same lists, to rounding for another order."""
    B, N, K = 2, 300, 40
    g = _gen(17)
    q, do = (torch.randn(B, H, N, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    k, v = (torch.randn(B, Hkv, N, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    idx = torch.randint(-1, 48, (B, H, N, K), generator=g)

    def run(i):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = topk_attention(*leaves, topk_indices=i.to(DEV), causal=True)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    first = run(idx)
    assert all(torch.equal(a, b) for _ in range(3) for a, b in zip(first, run(idx)))
    _, of_grad = _bounds(q.cpu(), k.cpu(), D, K, dtype)
    for a, b in zip(first, run(idx.sort(dim=-1).values)):
        assert rel(a, b) <= 2 * of_grad


def test_attention_far_into_a_long_cache():
    """Key rows more than 2^31 elements behind the first: the last 64 keys of every head, against a cache of
    those alone.  Nothing else is written before or listed."""
    B, H, Hkv, N, D, K, near = 2, 4, 2, 4_200_003, 128, 24, 64
    assert B * Hkv * N * D > 2 ** 31
    g = _gen(19)
    for Nq in (1, 300):
        q, do = (torch.randn(B, H, Nq, D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
        small = [torch.randn(B, Hkv, near, D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
        k, v = (torch.empty(B, Hkv, N, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        for far, t in zip((k, v), small):
            far[:, :, N - near:] = t
        idx = torch.randint(0, near, (B, H, Nq, K), generator=g).to(DEV)
        res = []
        for (kk, vv), off in ((small, 0), ((k, v), N - near)):
            leaves = [t.detach().requires_grad_() for t in (q, kk, vv)]
            out = topk_attention(*leaves, topk_indices=idx + off, causal=False, q_start=off, softcap=5.0)
            dq, dk, dv = torch.autograd.grad(out, leaves, do)
            if off:
                assert not dk[:, :, :off].any() and not dv[:, :, :off].any()
                dk, dv = dk[:, :, off:].clone(), dv[:, :, off:].clone()
            res.append((out.detach(), dq, dk, dv))
            del leaves, out
        del k, v
        _, of_grad = _bounds(q.cpu(), small[0].cpu(), D, K, torch.bfloat16)
        for a, b in zip(*res):  # other blocks of keys, other tiles: equal to rounding
            assert rel(a, b) <= 2 * of_grad


def test_distillation_of_many_rows():
    """Rows more than 2^31 logits behind the first; those before weigh nothing and are not read."""
    T, V, K, near = 16_500, 131_072, 9, 5
    assert (T - near) * V > 2 ** 31
    g = _gen(23)
    z = torch.empty(T, V, dtype=torch.bfloat16, device=DEV)
    z[T - near:] = (torch.randn(near, V, generator=g) * 2).to(DEV)
    ids = torch.randint(0, V, (T, K), generator=g).to(DEV)
    teacher = torch.randn(T, K, generator=g).to(DEV)
    weight = torch.zeros(T, device=DEV)
    weight[T - near:] = 1.0
    z.requires_grad_()
    loss = top_logit_distillation_loss(z, teacher, ids, row_weight=weight)
    (dz,) = torch.autograd.grad(loss, z)
    part = z.detach()[T - near:].clone().requires_grad_()
    small = top_logit_distillation_loss(part, teacher[T - near:], ids[T - near:])
    (want,) = torch.autograd.grad(small, part)
    # few rows are split over more thread blocks: the sums in another order
    assert abs(loss.item() - small.item()) <= 2.0 ** -16 * abs(small.item())
    assert rel(dz[T - near:], want) <= 2.0 ** -8 + 2.0 ** -16
    assert not dz[:T - near].any()


def test_norms_of_many_rows():
    """Tokens more than 2^31 elements behind the first, bit for bit as in a call of their own."""
    N, Hq, Hk, D, near = 1_400_000, 12, 2, 128, 37
    assert (N - near) * Hq * D > 2 ** 31
    g = _gen(29)
    q, k = (torch.empty(1, N, h, D, dtype=torch.bfloat16, device=DEV) for h in (Hq, Hk))
    cos, sin = (torch.empty(1, N, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for t in (q, k, cos, sin):
        t[:, N - near:] = torch.randn(t[:, N - near:].shape, generator=g).to(DEV)
    wq, wk = (torch.rand(D, generator=g).to(DEV) + 0.5 for _ in range(2))
    gq, gk = (torch.empty(1, h, N, D, dtype=torch.bfloat16, device=DEV) for h in (Hq, Hk))
    for t in (gq, gk):
        t[:, :, N - near:] = torch.randn(t[:, :, N - near:].shape, generator=g).to(DEV)
    res = []
    for n0 in (N - near, 0):
        leaves = [t[:, n0:].clone().requires_grad_() for t in (q, k)]
        out = qk_norm_rope(*leaves, Hq, Hk, wq, wk, cos[:, n0:], sin[:, n0:])
        grads = torch.autograd.grad(out, leaves, (gq[:, :, n0:], gk[:, :, n0:]))
        res.append([t.detach()[:, :, -near:].clone() for t in out] + [t[:, -near:].clone() for t in grads])
        del leaves, out, grads
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_differentiable_once():
    """A second derivative is refused, not taken for zero."""
    g = _gen(31)
    q = torch.randn(1, 2, 20, 64, generator=g).to(DEV).requires_grad_()
    idx = torch.randint(0, 20, (1, 2, 20, 4), generator=g).to(DEV)
    x = torch.randn(1, 5, 2 * 64, generator=g).to(DEV).requires_grad_()
    z = torch.randn(6, 50, generator=g).to(DEV).requires_grad_()
    ids = torch.rand(6, 50, generator=g).topk(3, dim=-1).indices.to(DEV)
    t = torch.randn(6, 3, generator=g).to(DEV)
    w = torch.rand(64, generator=g).to(DEV)
    calls = [(q, lambda: topk_attention(q, q, q, topk_indices=idx)),
             (x, lambda: qk_norm_rope(x, x, 2, 2, w, w)[0]),
             (x, lambda: rope_to_heads(x, 2)),
             (z, lambda: top_logit_distillation_loss(z, t, ids))]
    for leaf, call in calls:
        out = call()
        up = torch.ones_like(out).requires_grad_()
        (first,) = torch.autograd.grad(out, leaf, up, create_graph=True)
        (plain,) = torch.autograd.grad(call(), leaf, torch.ones_like(out))
        assert torch.equal(first.detach(), plain)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            first.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_of_the_norm_weights(dtype):
    """Each weight without the other, each wanted or not: its gradient is the one that both have together."""
    B, N, Hq, Hk, D = 2, 9, 3, 2, 64
    g = _gen(37)
    q, k = (torch.randn(B, N, h * D, generator=g).to(dtype).to(DEV) for h in (Hq, Hk))
    gq, gk = (torch.randn(B, h, N, D, generator=g).to(dtype).to(DEV) for h in (Hq, Hk))
    wq, wk = (torch.rand(D, generator=g).to(DEV) + 0.5 for _ in range(2))

    def grads(uq, uk, want):
        out = qk_norm_rope(q, k, Hq, Hk, uq, uk)
        return torch.autograd.grad(out, want, (gq, gk))

    a, b = wq.clone().requires_grad_(), wk.clone().requires_grad_()
    dq, dk = grads(a, b, [a, b])
    for got, want in ((grads(a, None, [a]), dq), (grads(None, b, [b]), dk), (grads(a, wk, [a]), dq), (grads(wq, b, [b]), dk)):
        assert rel(got[0], want) <= 2.0 ** -18  # the rows of one tensor may go to more thread blocks


def test_errors_keep_their_type():
    from ossa_b200._lib import OSSA_ERR_UNSUPPORTED, OssaError

    q = torch.zeros(1, 1, 4, 96, device=DEV, requires_grad=True)
    idx = torch.zeros(1, 1, 4, 2, dtype=torch.int32, device=DEV)
    with pytest.raises(OssaError, match="head_dim") as e:
        topk_attention(q, q, q, topk_indices=idx)
    assert e.value.status == OSSA_ERR_UNSUPPORTED


def _all_calls(dtype=torch.bfloat16):
    g = _gen(41)
    x = torch.randn(2, 30, 4 * 128, generator=g).to(dtype).to(DEV)
    y = torch.randn(2, 30, 2 * 128, generator=g).to(dtype).to(DEV)
    w = (torch.rand(128, generator=g) + 0.5).to(DEV)
    cs = [torch.randn(1, 30, 128, generator=g).to(dtype).to(DEV) for _ in range(2)]
    idx = torch.randint(-1, 30, (2, 4, 30, 7), generator=g).to(DEV)
    seg = (torch.arange(30) // 9).int().to(DEV)
    z = torch.randn(2, 30, 77, generator=g).to(dtype).to(DEV)
    ids = torch.rand(2, 30, 77, generator=g).topk(5, dim=-1).indices.to(DEV)
    t = torch.randn(2, 30, 5, generator=g).to(DEV)

    def attend(a, b, c):
        q, k = qk_norm_rope(a, b, 4, 2, w, w, *cs)
        return topk_attention(q, k, rope_to_heads(b, 2), topk_indices=idx, segments=seg, softcap=5.0), c

    return (x, y, z), lambda a, b, c: (attend(a, b, c)[0], top_logit_distillation_loss(c, t, ids, temperature=2.0))


def test_inference_mode():
    """In inference mode, and without gradients on tensors made there, the calls give what they give without it."""
    leaves, call = _all_calls()
    with torch.no_grad():
        want = call(*leaves)
    with torch.inference_mode():
        inner = [t.clone() for t in leaves]
        assert all(torch.equal(a, b) for a, b in zip(want, call(*inner)))
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(want, call(*inner)))
    assert not any(t.requires_grad for t in call(*leaves))


@pytest.mark.parametrize("backward", [False, True])
def test_nothing_stays_behind(backward):
    """Calls whose results are dropped, with or without their backward pass, leave no memory held."""
    leaves, call = _all_calls()
    leaves = [t.requires_grad_() for t in leaves]

    def step():
        out, loss = call(*leaves)
        if backward:
            torch.autograd.grad(out.float().sum() + loss, leaves)

    for _ in range(3):
        step()
    torch.cuda.synchronize()
    gc.collect()  # what earlier tests left in reference cycles would go during the loop below
    held = torch.cuda.memory_allocated()
    for _ in range(20):
        step()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == held


def test_from_several_threads():
    """Two threads on streams of their own, each with its leaves: what each gets alone."""
    import threading

    leaves, call = _all_calls()

    def grads():
        own = [t.detach().clone().requires_grad_() for t in leaves]
        out, loss = call(*own)
        return torch.autograd.grad(out.float().sum() + loss, own)

    want = grads()
    torch.cuda.synchronize()
    got = {}

    def work(n):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(10):
                got[n] = grads()
        s.synchronize()

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for n in range(2) for a, b in zip(want, got[n]))


def test_positions_past_32_bits_are_refused():
    q = torch.zeros(1, 1, 4, 64, device=DEV)
    idx = torch.zeros(1, 1, 4, 2, dtype=torch.int32, device=DEV)
    for q_start in (2 ** 31, 2 ** 32, 2 ** 31 - 2):
        with pytest.raises((ValueError, RuntimeError)):
            topk_attention(q, q, q, topk_indices=idx, q_start=q_start, softcap=2.0)
