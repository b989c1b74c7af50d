"""topk_attention with score modifiers, and its gradients, against the 64-bit definition.

Tolerances.  fp32: every probability is off by at most twice the scores' rounding (score_step),
sums over K entries and D values add (K + D) 2^-24; gradients are products of three such factors:
rel <= 8 (score_step + (K + D) 2^-24).
bf16 (half a step is 2^-8 of a value): the output rounds p for p.v and itself, 2 steps; a gradient
rounds its weights, itself, and through Delta = out . dout the forward's output, 3 steps, in the
norm of the whole tensor.  Element by element the output is held to
2^-8 (sum p |v| + |out|) plus the fp32 part."""

import math

import pytest
import torch

from mod_attention_ref import attention, rel, score_step
from ossa_b200 import topk_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
STEP = 2.0 ** -8


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _lists(B, H, Nq, Nk, K, q0, seed, kind="causal"):
    """Index lists: "causal" (ascending, distinct, at or before the row, -1 behind), "any" (any order,
    repeats, -1 and values outside the range anywhere)."""
    g = _gen(seed)
    if kind == "any":
        return torch.randint(-2, Nk + 2, (B, H, Nq, K), generator=g).int()
    score = torch.rand(B, H, Nq, Nk, generator=g)
    pos = q0 + torch.arange(Nq).view(Nq, 1)
    score = score.masked_fill(torch.arange(Nk).view(1, Nk) > pos, -1.0)
    kk = min(K, Nk)
    val, idx = score.topk(kk, dim=-1)
    idx = torch.where(val < 0, torch.full_like(idx, Nk), idx).sort(dim=-1).values
    idx = torch.where(idx >= Nk, torch.full_like(idx, -1), idx)
    if kk < K:
        idx = torch.cat([idx, torch.full((B, H, Nq, K - kk), -1)], dim=-1)
    return idx.int()


def _inputs(dtype, B, H, Hkv, Nq, Nk, D, seed):
    g = _gen(seed)
    q = (torch.randn(B, H, Nq, D, generator=g) * 1.5).to(dtype)
    k = torch.randn(B, Hkv, Nk, D, generator=g).to(dtype)
    v = torch.randn(B, Hkv, Nk, D, generator=g).to(dtype)
    do = torch.randn(B, H, Nq, D, generator=g).to(dtype)
    return q, k, v, do


def _mods(names, B, H, Nk, seed):
    g = _gen(seed)
    m = {}
    if "cap" in names:
        m["softcap"] = 3.0
    if "slopes" in names:
        m["slopes"] = torch.rand(H, generator=g) * 0.2
    if "docs" in names:
        m["segments"] = torch.sort(torch.randint(0, 4, (B, Nk), generator=g), dim=1).values.int()
    if "prefix" in names:
        m["prefix_len"] = torch.randint(0, Nk + 1, (B,), generator=g).int()
    return m


def _on(m, dev=DEV):
    return {n: t.to(dev) if isinstance(t, torch.Tensor) else t for n, t in m.items()}


def _check(dtype, q, k, v, do, idx, m, *, causal=True, q0=0):
    D, K = q.shape[-1], idx.shape[-1]
    rq, rk, rv = (t.double().requires_grad_() for t in (q, k, v))
    rm = dict(m)
    leaves = [rq, rk, rv]
    if "slopes" in m:
        rm["slopes"] = m["slopes"].double().requires_grad_()
        leaves.append(rm["slopes"])
    ref, p, vg = attention(rq, rk, rv, idx, causal=causal, q_start=q0, **rm)
    rgrads = torch.autograd.grad(ref, leaves, do.double())
    dev = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    dm = _on(m)
    if "slopes" in m:
        dm["slopes"].requires_grad_()
        dev.append(dm["slopes"])
    rows = {} if q0 == 0 and q.shape[2] == k.shape[2] else {"q_start": q0}
    out = topk_attention(dev[0], dev[1], dev[2], topk_indices=idx.to(DEV), causal=causal, **rows, **dm)
    grads = torch.autograd.grad(out, dev, do.to(DEV))
    with torch.no_grad():
        again = topk_attention(dev[0], dev[1], dev[2], topk_indices=idx.to(DEV), causal=causal, **rows, **dm)
    if m:
        assert torch.equal(out.detach(), again)  # the statistic for the backward pass changes nothing
    out = out.detach().cpu()
    fine = score_step(q, k) + (K + D) * 2.0 ** -24
    step = 0.0 if dtype == torch.float32 else STEP
    mass = torch.einsum("bhnk,bhnkd->bhnd", p, vg.abs())
    bound = step * (mass + ref.abs()) + 8 * fine * mass
    assert ((out.double() - ref).abs() <= bound + 1e-300).all()
    empty = p.sum(-1) == 0
    assert (out[empty] == 0).all()
    assert out.dtype == dtype
    # Exact zeros: rows that see nothing, keys that no row sees (their dv is an empty sum).  A row
    # that sees one key only has dP - Delta = 0 by the cancellation of two rounded values, which
    # leaves up to the rounding of Delta: its dq is held by the norm alone.
    unseen = rgrads[2] == 0
    for name, got, want, zero in zip(("dq", "dk", "dv", "dslopes"), grads, rgrads, (empty, unseen, unseen, None)):
        got = got.cpu()
        assert torch.isfinite(got).all(), name
        assert zero is None or (got[zero] == 0).all(), name
        if want.norm() == 0 and name == "dv":
            assert (got == 0).all(), name
            continue
        s = 0.0 if name == "dslopes" else 3 * step  # dslopes is fp32 and takes the exact Delta
        if name == "dslopes":
            # terms of both signs: the bound is on the sum of their sizes
            size = (p * (vg @ do.double().unsqueeze(-1)).squeeze(-1).abs()).sum() * k.shape[2]
            assert (got.double() - want).abs().max() <= 8 * fine * size, name
        else:
            assert rel(got, want) <= s + 8 * fine, f"{name}: {rel(got, want):.3g}"


CASES = [
    # B, H, Hkv, Nq, Nk, D, K, modifiers
    (1, 1, 1, 1, 1, 16, 1, ""),
    (1, 2, 1, 3, 3, 32, 5, "cap"),
    (2, 4, 2, 65, 65, 64, 16, "cap slopes"),
    (1, 6, 3, 130, 130, 128, 33, "docs"),
    (2, 12, 2, 97, 97, 128, 64, "cap slopes docs prefix"),
    (1, 8, 1, 70, 70, 128, 100, "prefix"),
    (2, 4, 4, 50, 50, 128, 40, "slopes"),
    (1, 5, 1, 40, 40, 128, 20, "cap docs"),
    (1, 4, 1, 33, 33, 256, 9, "cap prefix"),
    (1, 6, 2, 60, 60, 128, 150, "slopes docs"),
    (1, 8, 4, 200, 200, 128, 24, "cap"),
    (1, 7, 1, 150, 150, 128, 100, "cap slopes"),
    (2, 14, 2, 90, 90, 128, 64, "docs"),
    (1, 10, 2, 140, 140, 128, 128, ""),
    (1, 3, 3, 600, 600, 128, 90, "cap docs"),
    (1, 9, 1, 70, 70, 128, 40, "slopes"),
    (1, 16, 2, 260, 260, 128, 128, "prefix"),
]


@pytest.mark.parametrize("Nk", [12288, 12289, 20000])
def test_many_keys(Nk):
    """On either side of what the heads' union covers with a byte per key; lists with and without repeats."""
    B, H, Hkv, Nq, D, K = 1, 6, 2, 100, 128, 64
    q, k, v, do = _inputs(torch.bfloat16, B, H, Hkv, Nq, Nk, D, seed=Nk)
    idx = _lists(B, H, Nq, Nk, K, Nk - Nq, seed=4)
    idx[:, :, ::3, 5] = idx[:, :, ::3, 4]
    idx[:, :, 1::7] = idx[:, :, 1::7].flip(-1)
    _check(torch.bfloat16, q, k, v, do, idx, _mods(["cap", "docs"], B, H, Nk, seed=1), q0=Nk - Nq)


@pytest.mark.parametrize("kind", ["causal", "any"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_gradients(case, dtype, kind):
    B, H, Hkv, Nq, Nk, D, K, names = case
    q, k, v, do = _inputs(dtype, B, H, Hkv, Nq, Nk, D, seed=Nq + D)
    idx = _lists(B, H, Nq, Nk, K, 0, seed=K, kind=kind)
    idx[:, 0, Nq // 2] = -1  # a row that lists nothing
    _check(dtype, q, k, v, do, idx, _mods(names.split(), B, H, Nk, seed=7))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Nq,Nk,q0", [(1, 300, 299), (3, 9000, 8997), (20, 500, 100), (5, 5, 0), (4, 64, 200)])
def test_query_rows(Nq, Nk, q0, causal, dtype):
    """Rows at positions q0.. against a longer (or, without segments, a shorter) key sequence."""
    B, H, Hkv, D, K = 2, 6, 2, 128, 48
    q, k, v, do = _inputs(dtype, B, H, Hkv, Nq, Nk, D, seed=Nk)
    idx = _lists(B, H, Nq, Nk, K, q0, seed=3)
    names = ["cap", "slopes", "prefix"] + (["docs"] if q0 + Nq <= Nk else [])
    _check(dtype, q, k, v, do, idx, _mods(names, B, H, Nk, seed=5), causal=causal, q0=q0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_key_that_every_row_lists(dtype):
    """Key 0 (and 1) in every row: its run spans many tiles of the key pass; int64 lists."""
    B, H, Hkv, N, D, K = 1, 4, 2, 700, 128, 12
    q, k, v, do = _inputs(dtype, B, H, Hkv, N, N, D, seed=1)
    idx = _lists(B, H, N, N, K, 0, seed=2).long()
    idx[..., -1] = 0
    idx[..., -2] = 1
    _check(dtype, q, k, v, do, idx, _mods(["cap"], B, H, N, seed=5))


def test_masked_places_hold_anything():
    """Keys that no row sees (another segment, behind the row, not listed) may hold NaN or infinities:
    outputs and gradients are those of finite ones, and their own gradients are 0."""
    for dtype in (torch.float32, torch.bfloat16):
        for H, Hkv in ((4, 2), (2, 2), (5, 1)):
            B, N, D, K = 1, 90, 128, 30
            q, k, v, do = _inputs(dtype, B, H, Hkv, N, N, D, seed=4)
            idx = _lists(B, H, N, N, K, 0, seed=9)
            seg = torch.zeros(B, N, dtype=torch.int32)
            seg[:, :6] = 1  # the first document: its rows are left out below
            idx[:, :, :6] = -1
            idx = torch.where(idx == 50, torch.full_like(idx, -1), idx)  # key 50 is never listed
            res = []
            for bad in (0.0, float("nan"), float("inf")):
                kk, vv = k.clone(), v.clone()
                for t in (kk, vv):
                    t[:, :, :6] = bad
                    t[:, :, 50] = bad
                leaves = [t.to(DEV).requires_grad_() for t in (q, kk, vv)]
                out = topk_attention(*leaves, topk_indices=idx.to(DEV), segments=seg.to(DEV), softcap=9.0)
                res.append([out.detach()] + list(torch.autograd.grad(out, leaves, do.to(DEV))))
            for other in res[1:]:
                for a, b in zip(res[0], other):
                    assert torch.equal(a, b)
            assert (res[0][2][:, :, 50] == 0).all() and (res[0][3][:, :, :6] == 0).all()


def test_plain_call_and_training_form_agree():
    """Without modifiers and gradients the plain kernels run.  The training form and neutral modifiers
    give the same values to rounding: both round p and the output, 2 steps each."""
    B, H, Hkv, N, D, K = 2, 12, 2, 300, 128, 64
    q, k, v, do = (t.to(DEV) for t in _inputs(torch.bfloat16, B, H, Hkv, N, N, D, seed=6))
    idx = _lists(B, H, N, N, K, 0, seed=1).to(DEV)
    plain = topk_attention(q, k, v, topk_indices=idx)
    assert not plain.requires_grad
    leaf = q.clone().requires_grad_()
    out = topk_attention(leaf, k, v, topk_indices=idx)
    assert out.requires_grad and rel(out.detach(), plain) < 4 * STEP
    neutral = topk_attention(q, k, v, topk_indices=idx, slopes=torch.zeros(H, device=DEV))
    assert rel(neutral, plain) < 4 * STEP
    for dtype, d in ((torch.float32, 128), (torch.bfloat16, 64)):  # per-head forms: the same bits
        q, k, v, do = (t.to(DEV) for t in _inputs(dtype, B, H, Hkv, N, N, d, seed=6))
        out = topk_attention(q.requires_grad_(), k, v, topk_indices=idx)
        assert torch.equal(out.detach(), topk_attention(q.detach(), k, v, topk_indices=idx))


def test_same_bits_every_call():
    B, H, Hkv, N, D, K = 2, 12, 2, 513, 128, 64
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v, do = (t.to(DEV) for t in _inputs(dtype, B, H, Hkv, N, N, D, seed=8))
        idx = _lists(B, H, N, N, K, 0, seed=2).to(DEV)
        idx[..., -1] = 0
        slopes = torch.rand(H, generator=_gen(1)).to(DEV)
        first = None
        for _ in range(5):
            leaves = [t.clone().requires_grad_() for t in (q, k, v, slopes)]
            out = topk_attention(*leaves[:3], topk_indices=idx, slopes=leaves[3])
            got = [out.detach()] + list(torch.autograd.grad(out, leaves, do))
            first = first or got
            assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_gradients_against_differences():
    """Directional derivatives of the fp32 kernel: central differences at h = 2^-7.  Their error is
    h^2/6 times the third derivative (the inputs are scaled so that derivatives stay around 1) plus
    the output's rounding over h, 2^-24 sqrt(n) 2^7: 1e-3 of the derivative's scale covers both."""
    B, H, Hkv, N, D, K = 1, 4, 2, 48, 64, 16
    q, k, v, do = (t.to(DEV) for t in _inputs(torch.float32, B, H, Hkv, N, N, D, seed=3))
    q = q * 0.5
    idx = _lists(B, H, N, N, K, 0, seed=5).to(DEV)
    m = _on(_mods(["cap", "docs"], B, H, N, seed=2))
    slopes = torch.rand(H, generator=_gen(2)).to(DEV) * 0.1

    def f(*t):
        o = topk_attention(t[0], t[1], t[2], topk_indices=idx, slopes=t[3], **m)
        return (o.double() * do.double()).sum().item()

    base = [q, k, v, slopes]
    leaves = [t.clone().requires_grad_() for t in base]
    out = topk_attention(*leaves[:3], topk_indices=idx, slopes=leaves[3], **m)
    grads = torch.autograd.grad(out, leaves, do)
    h = 2.0 ** -7
    for n in range(4):
        d = torch.randn(base[n].shape, generator=_gen(n + 20)).to(DEV)
        up = [t + h * d if i == n else t for i, t in enumerate(base)]
        down = [t - h * d if i == n else t for i, t in enumerate(base)]
        diff = (f(*up) - f(*down)) / (2 * h)
        want = (grads[n].double() * d.double()).sum().item()
        scale = (grads[n].double().norm()).item()
        assert abs(diff - want) <= 1e-3 * scale * max(1.0, d.abs().max().item()), (n, diff, want)


def test_strided_inputs_other_stream_and_retained_graph():
    B, H, Hkv, N, D, K = 2, 6, 2, 70, 128, 16
    q, k, v, do = _inputs(torch.bfloat16, B, H, Hkv, N, N, D, seed=2)
    idx = _lists(B, H, N, N, K, 0, seed=2).to(DEV)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = topk_attention(*leaves, topk_indices=idx, softcap=4.0)
    want = torch.autograd.grad(out, leaves, do.to(DEV), retain_graph=True)
    again = torch.autograd.grad(out, leaves, do.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    # (B, N, H, D) storage seen as (B, H, N, D), a strided dout, a stream of its own
    strided = [t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for t in (q, k, v)]
    dos = do.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        o2 = topk_attention(*strided, topk_indices=idx.transpose(2, 3).contiguous().transpose(2, 3), softcap=4.0)
        got = torch.autograd.grad(o2, strided, dos)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(o2, out) and all(torch.equal(a, b) for a, b in zip(want, got))


def test_captured_training_step_replays():
    B, H, Hkv, N, D, K = 1, 12, 2, 256, 128, 32
    q, k, v, do = (t.to(DEV) for t in _inputs(torch.bfloat16, B, H, Hkv, N, N, D, seed=12))
    idx = _lists(B, H, N, N, K, 0, seed=3).to(DEV)

    def step(q, k, v):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = topk_attention(*leaves, topk_indices=idx, softcap=6.0)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step(q, k, v)
    q.copy_(torch.randn(q.shape, generator=_gen(99)).to(q))
    graph.replay()
    want = step(q, k, v)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_empty_shapes():
    k = torch.randn(1, 2, 8, 64, device=DEV, requires_grad=True)
    q = torch.randn(1, 4, 0, 64, device=DEV, requires_grad=True)
    idx = torch.zeros(1, 4, 0, 3, dtype=torch.int32, device=DEV)
    out = topk_attention(q, k, k, topk_indices=idx, q_start=0, softcap=2.0)
    dq, dk = torch.autograd.grad(out, (q, k), torch.empty_like(out))
    assert out.shape == q.shape and dq.shape == q.shape and (dk == 0).all()
    q = torch.randn(1, 4, 8, 64, device=DEV, requires_grad=True)
    idx = torch.zeros(1, 4, 8, 0, dtype=torch.int32, device=DEV)
    out = topk_attention(q, k, k, topk_indices=idx)
    dq, dk = torch.autograd.grad(out, (q, k), torch.ones_like(out))
    assert (out == 0).all() and (dq == 0).all() and (dk == 0).all()
