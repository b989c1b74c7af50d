"""top_logit_distillation_loss and its gradient against the 64-bit definition.

Tolerances: exponents and logarithms of fp32 values up to ~30 (relative error about 2^-22 times
the exponent's size), sums of V terms in trees and short chains: the loss within 2^-18 of the sum
of its terms' sizes; a gradient entry within 2^-18 (softmax + p) scale plus half a step of its type."""

import pytest
import torch

from ossa_b200 import top_logit_distillation_loss

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FINE = 2.0 ** -18


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _ref(z, teacher, ids, tau, weight=None, reduction="mean"):
    """(loss, the size of its terms, p as a (rows, V) tensor, row scale) in 64 bits."""
    V = z.shape[-1]
    ids = ids.long()
    ok = (ids >= 0) & (ids < V)
    t = (teacher.double() / tau).masked_fill(~ok, -float("inf"))
    p = torch.softmax(torch.where(ok.any(-1, keepdim=True), t, torch.zeros_like(t)), -1) * ok
    w = ok.any(-1).double()
    if weight is not None:
        w = w * weight.double()
    zz = torch.where((w > 0).unsqueeze(-1), z.double(), torch.zeros_like(z, dtype=torch.float64))
    logq = torch.log_softmax(zz / tau, -1)
    lp = torch.where(p > 0, torch.log(p.clamp_min(1e-300)), torch.zeros_like(p))
    lq = logq.gather(-1, ids.clamp(0, V - 1))
    terms = torch.where(p > 0, p * (lp - lq), torch.zeros_like(p))
    rows = tau * tau * terms.sum(-1) * (w > 0)
    size = tau * tau * torch.where(p > 0, p * (lp.abs() + lq.abs()), torch.zeros_like(p)).sum(-1)
    if reduction == "none":
        unit = torch.ones((), dtype=torch.float64)
        loss, size = rows * w, size * w
    else:
        unit = 1.0 / w.sum() if reduction == "mean" and w.sum() > 0 else torch.tensor(float(w.sum() > 0 or reduction == "sum"))
        loss, size = (rows * w).sum() * unit, (size * w).sum() * unit
    dense = torch.zeros(z.shape, dtype=torch.float64).scatter_add_(-1, ids.clamp(0, V - 1), p)
    return loss, size, dense, torch.exp(logq), tau * w * unit


def _case(dtype, lead, V, K, seed, repeats=False, holes=True):
    g = _gen(seed)
    z = (torch.randn(*lead, V, generator=g) * 3).to(dtype)
    ids = torch.randint(0, V, (*lead, K), generator=g)
    if not repeats:
        ids = torch.rand(*lead, V, generator=g).topk(min(K, V), dim=-1).indices
        ids = torch.nn.functional.pad(ids, (0, K - ids.shape[-1]), value=-1)
    if holes:
        ids[torch.rand(ids.shape, generator=g) < 0.15] = -1
        ids[torch.rand(ids.shape, generator=g) < 0.05] = V + 3
    t = torch.randn(*lead, K, generator=g) * 3
    return z, t, ids


def _check(z, t, ids, tau=1.0, weight=None, reduction="mean", upstream=None):
    dtype = z.dtype
    step = torch.finfo(dtype).eps / 2
    want, size, p, q, scale = _ref(z, t, ids, tau, weight, reduction)
    leaf = z.to(DEV).requires_grad_()
    loss = top_logit_distillation_loss(leaf, t.to(DEV), ids.to(DEV), temperature=tau, reduction=reduction,
                                       row_weight=None if weight is None else weight.to(DEV))
    with torch.no_grad():
        again = top_logit_distillation_loss(leaf, t.to(DEV), ids.to(DEV), temperature=tau, reduction=reduction,
                                            row_weight=None if weight is None else weight.to(DEV))
    assert torch.equal(loss.detach(), again) and loss.dtype == torch.float32
    assert ((loss.detach().double().cpu() - want).abs() <= FINE * size + 1e-30).all()
    up = torch.ones(loss.shape) if upstream is None else upstream
    first = torch.autograd.grad(loss, leaf, up.to(DEV), retain_graph=True)[0]
    second = torch.autograd.grad(loss, leaf, up.to(DEV))[0]
    assert torch.equal(first, second) and first.dtype == dtype and first.shape == z.shape
    s = (scale * up.double()).abs().unsqueeze(-1) if reduction == "none" else (scale * up.double().abs()).unsqueeze(-1)
    sign = up.double().unsqueeze(-1).sign() if reduction == "none" else up.double().sign()
    ref = sign * s * (q - p)
    err = (first.double().cpu() - ref).abs()
    tiny = torch.finfo(dtype).tiny  # below the normal range a store keeps absolute precision
    assert (err <= FINE * s * (q + p) + step * ref.abs() + tiny).all(), (err / (s * (q + p) + 1e-30)).max()
    return loss, first


SHAPES = [((1,), 1, 1), ((3,), 5, 3), ((7,), 33, 8), ((16,), 1000, 40), ((5,), 8191, 64), ((2, 9), 4096, 10),
          ((300,), 257, 16), ((3,), 40001, 100), ((4,), 151936, 64), ((2,), 700001, 20)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead,V,K", SHAPES)
def test_loss_and_gradient(lead, V, K, dtype):
    z, t, ids = _case(dtype, lead, V, K, seed=V + K)
    _check(z, t, ids, tau=2.0)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_reductions_weights_and_upstream(dtype, reduction):
    lead, V, K = (4, 11), 3001, 24
    z, t, ids = _case(dtype, lead, V, K, seed=3, repeats=True)
    ids[1, 2] = -1  # rows that list nothing
    ids[3, 5] = V
    g = _gen(1)
    weight = torch.rand(lead, generator=g)
    weight[0, :4] = 0.0
    up = torch.randn(lead, generator=g) if reduction == "none" else torch.tensor(-1.75)
    for w in (None, weight):
        _check(z, t, ids.int(), tau=1.5, weight=w, reduction=reduction, upstream=up)
        _check(z, t, ids, tau=0.7, weight=w, reduction=reduction)


def test_repeated_entries():
    """All listed entries the same, and pairs: p adds up, the gradient is that of the sum."""
    z, t, _ = _case(torch.float32, (6,), 500, 40, seed=4)
    for ids in (torch.full((6, 40), 17), torch.arange(40).div(2, rounding_mode="floor").expand(6, 40) + 3):
        _check(z, t, ids)


def test_rows_of_weight_zero_hold_anything():
    z, t, ids = _case(torch.bfloat16, (12,), 2049, 16, seed=6)
    w = torch.ones(12)
    w[[2, 7]] = 0
    ids[9] = -1
    z[2] = float("nan")
    z[7] = float("inf")
    z[9] = float("nan")
    loss, dz = _check(z, t, ids, weight=w)
    assert torch.isfinite(loss) and (dz[[2, 7, 9]] == 0).all()
    w[:] = 0
    loss, dz = _check(z, t, ids, weight=w)
    assert loss.item() == 0 and (dz == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lowest_values_and_infinities(dtype):
    """Entries (and whole stretches) at the type's lowest value or -inf weigh nothing; a row whose first
    8192 entries are all lowest, at a temperature below 1, stays finite."""
    low = torch.finfo(dtype).min
    z, t, ids = _case(dtype, (6,), 20000, 12, seed=8, holes=False)
    ids = ids.clamp_min(16000)
    z[0, :15000] = low
    z[1, :15000] = -float("inf")
    z[2, 5:] = torch.where(torch.rand(19995, generator=_gen(1)) < 0.5, torch.tensor(low, dtype=dtype), z[2, 5:])
    z[2].scatter_(0, ids[2], torch.ones(12, dtype=dtype))
    t[3, 2] = -float("inf")
    for tau in (1.0, 0.5, 3.0):
        _check(z, t, ids, tau=tau)


def test_not_finite_rows_show():
    z, t, ids = _case(torch.float32, (3,), 100, 4, seed=2, holes=False)
    z[1, 50] = float("nan")
    rows = top_logit_distillation_loss(z.to(DEV), t.to(DEV), ids.to(DEV), reduction="none")
    assert torch.isnan(rows[1]) and torch.isfinite(rows[[0, 2]]).all()


def test_strided_logits():
    """Shifted sequences (B, N - 1, V) of a (B, N, V) tensor are read in place; a transposed tensor
    and odd offsets give the same values."""
    z, t, ids = _case(torch.bfloat16, (3, 9), 1003, 8, seed=5)
    full = torch.randn(3, 10, 1003, generator=_gen(1)).bfloat16()
    full[:, :-1] = z
    want = top_logit_distillation_loss(z.to(DEV), t.to(DEV), ids.to(DEV))
    leaf = full.to(DEV).requires_grad_()
    got = top_logit_distillation_loss(leaf[:, :-1], t.to(DEV), ids.to(DEV))
    assert torch.equal(want, got.detach())
    (gf,) = torch.autograd.grad(got, leaf)
    zl = z.to(DEV).requires_grad_()
    (gz,) = torch.autograd.grad(top_logit_distillation_loss(zl, t.to(DEV), ids.to(DEV)), zl)
    assert torch.equal(gf[:, :-1], gz) and (gf[:, -1] == 0).all()
    off = torch.randn(3, 9, 1005, generator=_gen(1)).bfloat16()
    off[..., 1:-1] = z
    assert torch.equal(top_logit_distillation_loss(off.to(DEV)[..., 1:-1], t.to(DEV), ids.to(DEV)), want)
    lt = z.to(DEV).transpose(0, 2).contiguous().transpose(0, 2)
    assert torch.equal(top_logit_distillation_loss(lt, t.to(DEV), ids.to(DEV)), want)
    one = top_logit_distillation_loss(z[0, 0].to(DEV), t[0, 0].to(DEV), ids[0, 0].to(DEV))
    assert one.shape == ()


def test_same_bits_and_differences():
    z, t, ids = _case(torch.float32, (64,), 5000, 32, seed=11)
    args = (t.to(DEV), ids.to(DEV))
    leaf = z.to(DEV).requires_grad_()
    res = []
    for _ in range(5):
        loss = top_logit_distillation_loss(leaf, *args, temperature=2.0, reduction="sum")
        res.append((loss.detach(), torch.autograd.grad(loss, leaf)[0]))
    assert all(torch.equal(a, b) for r in res[1:] for a, b in zip(res[0], r))
    # rows are differenced one by one and added in 64 bits; h^2/6 and 2^-18 |loss| / h stay below 2e-3
    d = torch.randn(z.shape, generator=_gen(5)).to(DEV)
    h = 2.0 ** -5

    def f(x):
        return top_logit_distillation_loss(x, *args, temperature=2.0, reduction="none").double()

    diff = (f(leaf.detach() + h * d) - f(leaf.detach() - h * d)) / (2 * h)
    want = (res[0][1].double() * d).sum(-1)
    assert ((diff - want).abs() <= 2e-3 * (1 + want.abs())).all()


def test_captured_step_replays():
    z, t, ids = _case(torch.bfloat16, (32,), 9000, 16, seed=12)
    z, t, ids = z.to(DEV), t.to(DEV), ids.to(DEV)

    def step():
        leaf = z.detach().requires_grad_()
        loss = top_logit_distillation_loss(leaf, t, ids, temperature=2.0)
        return loss.detach(), torch.autograd.grad(loss * 3.0, leaf)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    z.copy_(torch.randn(z.shape, generator=_gen(70)).to(z))
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_no_rows():
    z = torch.zeros(0, 50, device=DEV, requires_grad=True)
    t, ids = torch.zeros(0, 4, device=DEV), torch.zeros(0, 4, dtype=torch.int64, device=DEV)
    loss = top_logit_distillation_loss(z, t, ids)
    assert loss.item() == 0 and torch.autograd.grad(loss, z)[0].shape == z.shape
