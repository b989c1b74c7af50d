"""Measured cases of the trainable sparse student's operators.

Three operators, each in its plain form (elementary torch operations, ``own`` false) and
as a user calls it in ossa_b200 (``own`` true):

* attention: the gathered top-K attention with a tanh cap on its scores, a bias that falls
  with distance, documents packed in one row and a bidirectional prefix; the forward for
  prefill and single tokens, forward and backward for training
  (``ossa_b200.topk_attention``);
* norm_rope: the RMS norm of every query and key head with the rotation and the head
  transpose in the same pass, forward and backward (``ossa_b200.qk_norm_rope``);
* distill: the distillation loss against a teacher's top logits and its gradient
  (``ossa_b200.train.top_logit_distillation_loss``).
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}


# ------------------------------------------------------------------------------- cases


def _attention(name, **kw):
    case = dict(name=name, op="attention", dtype="bf16", B=1, H=12, Hkv=2, D=128, Nq=1, Nk=1, K=64, train=False,
                softcap=0.0, slopes=False, docs=0, prefix=0)
    case.update(kw)
    return case


def _norm_rope(name, **kw):
    case = dict(name=name, op="norm_rope", dtype="bf16", B=1, N=1, H=12, Hkv=2, D=128, train=False)
    case.update(kw)
    return case


def _distill(name, **kw):
    case = dict(name=name, op="distill", dtype="bf16", T=16, V=151936, K=64, temperature=1.0, weighted=False)
    case.update(kw)
    return case


def listed():
    return [
        # one new token for each of 8 sequences against a cache of 32768 positions
        _attention("attention decode", B=8, Nq=1, Nk=32768, softcap=20.0),
        # prefill of two packed rows, four documents each, scores biased by distance
        _attention("attention prefill packed", B=2, Nq=4096, Nk=4096, slopes=True, docs=4),
        # a training step of one layer at the full-model length, capped scores, packed documents
        _attention("attention train", B=2, Nq=4096, Nk=4096, softcap=20.0, docs=3, train=True),
        # the long training step: K = 128 at twice the length, no modifier
        _attention("attention train long", B=1, Nq=8192, Nk=8192, K=128, train=True),
        # fp32 with odd sizes: a prefix that all may see, learned slopes (their gradient too)
        _attention("attention train fp32 odd", dtype="fp32", B=2, H=6, Hkv=3, D=64, Nq=517, Nk=517, K=33,
                   slopes=True, prefix=37, train=True),
        # the queries and keys of one decoding step
        _norm_rope("norm_rope decode", B=8, N=1),
        # the queries and keys of a prefill
        _norm_rope("norm_rope prefill", B=8, N=4096),
        # a training step of one layer
        _norm_rope("norm_rope train", B=4, N=4096, train=True),
        # fp32 with odd sizes
        _norm_rope("norm_rope train fp32 odd", dtype="fp32", B=3, N=1021, H=6, Hkv=3, D=64, train=True),
        # a few rows of a large vocabulary, as an evaluation of one short answer gives
        _distill("distill few rows", T=16),
        # the loss of a training step: one row of 4096 tokens, the full-model vocabulary
        _distill("distill train", T=4096, temperature=2.0),
        # fp32, odd sizes, weighted rows (padding weighs nothing)
        _distill("distill fp32 odd", dtype="fp32", T=999, V=32003, K=20, weighted=True),
    ]


def _log_between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "norm_rope", "distill"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    H, Hkv = rng.choice([(12, 2), (12, 2), (8, 2), (6, 3), (4, 4)])
    if op == "attention":
        D = 128 if dtype == "bf16" else rng.choice([64, 128])
        K = _log_between(rng, 16, 128)
        train = rng.random() < 0.6
        case = dict(op=op, dtype=dtype, B=rng.randint(1, 3), H=H, Hkv=Hkv, D=D, K=K, train=train,
                    softcap=rng.choice([0.0, 5.0, 20.0, 50.0]), slopes=rng.random() < 0.4,
                    docs=rng.choice([0, 0, 2, 5]), prefix=rng.choice([0, 0, 19, 64]))
        if not train and rng.random() < 0.5:  # single tokens or a few of them against a cache
            case.update(Nq=rng.randint(1, 4), Nk=_log_between(rng, 200, 40000))
        else:
            # at most 12 heads * 8192 * 128 entries in all
            most = min(8192, 12 * 8192 * 128 // (case["B"] * H * K))
            n = _log_between(rng, 150, most)
            case.update(Nq=n, Nk=n)
        return case
    if op == "norm_rope":
        return dict(op=op, dtype=dtype, B=rng.randint(1, 6), N=_log_between(rng, 1, 4096), H=H, Hkv=Hkv,
                    D=rng.choice([64, 128, 128]), train=rng.random() < 0.6)
    return dict(op=op, dtype=dtype, T=_log_between(rng, 4, 2048), V=_log_between(rng, 8000, 152000),
                K=_log_between(rng, 8, 128), temperature=rng.choice([1.0, 2.0, 4.0]), weighted=rng.random() < 0.5)


# ------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _key_lists(case, g):
    """Key lists as the selectors give them: ascending, distinct, causal, -1 where a row has
    fewer keys than K.  Half of a row's keys are its most recent positions, the others lie
    anywhere before them; of those, half are common to the heads of a kv head."""
    B, H, Hkv, Nq, Nk, K = (case[x] for x in ("B", "H", "Hkv", "Nq", "Nk", "K"))
    near = K // 2
    far = K - near
    pos = torch.arange(Nk - Nq, Nk, device="cuda").view(1, 1, Nq, 1)
    room = (pos + 1 - near).clamp_min(0).double()  # keys before the recent ones
    slot = torch.arange(far, device="cuda").view(1, 1, 1, far)
    mine = torch.rand(B, H, Nq, far, device="cuda", generator=g)
    common = torch.rand(B, Hkv, Nq, far, device="cuda", generator=g).repeat_interleave(H // Hkv, dim=1)
    u = torch.where(slot % 2 == 0, common, mine).double()
    lo, hi = (slot * room / far).ceil(), ((slot + 1) * room / far).ceil()  # one key of each stratum
    j = (lo + (u * (hi - lo)).floor()).clamp_max(Nk).minimum(hi - 1)
    j = torch.where(hi > lo, j, torch.full_like(j, -1)).long()
    recent = (pos + 1 - near + torch.arange(near, device="cuda").view(1, 1, 1, near)).expand(B, H, Nq, near)
    rows = torch.cat([j, torch.where(recent >= 0, recent, torch.full_like(recent, -1))], dim=-1)
    # -1 last, the others ascending
    rows = torch.where(rows < 0, torch.full_like(rows, Nk), rows).sort(dim=-1).values
    return torch.where(rows >= Nk, torch.full_like(rows, -1), rows).int()


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dt)

    st = {"case": case}
    if case["op"] == "attention":
        B, H, Hkv, Nq, Nk, D = (case[x] for x in ("B", "H", "Hkv", "Nq", "Nk", "D"))
        st["q"] = randn(B, H, Nq, D, scale=1.5)
        st["k"], st["v"] = randn(B, Hkv, Nk, D), randn(B, Hkv, Nk, D)
        st["idx"] = _key_lists(case, g)
        st["q_start"] = Nk - Nq
        st["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda") / H).float() if case["slopes"] else None
        st["segments"] = None
        if case["docs"]:  # documents of unequal lengths, packed one after another
            cuts = torch.rand(B, Nk, device="cuda", generator=g).argsort(dim=1)[:, : case["docs"] - 1]
            starts = torch.zeros(B, Nk, device="cuda", dtype=torch.int32).scatter_(1, cuts, 1)
            st["segments"] = starts.cumsum(1).int()
        st["prefix"] = None
        if case["prefix"]:
            st["prefix"] = torch.randint(0, 2 * case["prefix"], (B,), device="cuda", generator=g).int()
            # a row of the prefix lists keys of the prefix behind it too
            behind = st["idx"][:, :, :, -1:].clamp_min(0) + 5
            st["idx"][:, :, :, -1:] = torch.where(behind < Nk, behind, torch.full_like(behind, -1))
        if case["train"]:
            st["dout"] = randn(B, H, Nq, D)
    elif case["op"] == "norm_rope":
        B, N, H, Hkv, D = (case[x] for x in ("B", "N", "H", "Hkv", "D"))
        st["q"], st["k"] = randn(B, N, H * D, scale=2.0), randn(B, N, Hkv * D, scale=2.0)
        st["wq"] = (1.0 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(dt)
        st["wk"] = (1.0 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(dt)
        first = torch.randint(0, 30000, (B, 1), device="cuda", generator=g)  # a position for each sequence
        pos = (first + torch.arange(N, device="cuda")).double()
        inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, device="cuda").double() / D))
        ang = torch.cat([pos[..., None] * inv, pos[..., None] * inv], dim=-1)
        st["cos"], st["sin"] = ang.cos().to(dt), ang.sin().to(dt)
        if case["train"]:
            st["dq"], st["dk"] = randn(B, H, N, D), randn(B, Hkv, N, D)
    else:
        T, V, K = case["T"], case["V"], case["K"]
        st["logits"] = randn(T, V, scale=3.0)
        # distinct entries in any order; the teacher mostly agrees with the student's raised ones
        ids = torch.arange(K, device="cuda") * (V // K) + torch.randint(0, V // K, (T, K), device="cuda", generator=g)
        ids = ids.gather(1, torch.rand(T, K, device="cuda", generator=g).argsort(dim=1))
        st["teacher"] = (torch.randn(T, K, device="cuda", generator=g) * 2 + 8).sort(dim=1, descending=True).values
        st["logits"].scatter_(1, ids, (st["teacher"] + torch.randn(T, K, device="cuda", generator=g)).to(dt))
        tail = torch.rand(T, K, device="cuda", generator=g) < 0.02  # lists of a teacher that keeps fewer
        st["ids"] = torch.where(tail, torch.full_like(ids, -1), ids).int()
        st["weight"] = None
        if case["weighted"]:
            w = torch.rand(T, device="cuda", generator=g)
            st["weight"] = torch.where(w < 0.2, torch.zeros_like(w), w)
    return st


# ------------------------------------------------------------------------------- plain forms


def _plain_attention(st):
    case = st["case"]
    B, H, Hkv, Nq, Nk, D = (case[x] for x in ("B", "H", "Hkv", "Nq", "Nk", "D"))
    G, cap, scale = H // Hkv, case["softcap"], 1.0 / math.sqrt(D)
    dt = st["q"].dtype
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    pos = (st["q_start"] + torch.arange(Nq, device="cuda")).view(1, 1, Nq, 1)
    listed_key = st["idx"].long()
    inside = (listed_key >= 0) & (listed_key < Nk)
    j = listed_key.clamp(0, Nk - 1)
    seen = j <= pos
    if st["prefix"] is not None:
        seen = seen | (j < st["prefix"].view(B, 1, 1, 1))
    seen = seen & inside
    b = torch.arange(B, device="cuda").view(B, 1, 1, 1)
    if st["segments"] is not None:
        seen = seen & (st["segments"][b, j] == st["segments"][b, pos])
    head = (torch.arange(H, device="cuda") // G).view(1, H, 1, 1)
    kg, vg = k[b, head, j], v[b, head, j]  # (B, H, Nq, K, D)
    s = (kg @ q.unsqueeze(-1)).squeeze(-1) * scale
    t = None
    if cap > 0:
        t = torch.tanh(s / cap)
        s = cap * t
    far = (pos - j).abs().float()
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, H, 1, 1) * far
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    out = {"out": (p.unsqueeze(-2) @ vg).squeeze(-2).to(dt)}
    if case["train"]:
        do = st["dout"].float()
        dp = (vg @ do.unsqueeze(-1)).squeeze(-1)
        ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True))
        if st["slopes"] is not None:
            out["dslopes"] = -(ds.double() * far).sum(dim=(0, 2, 3)).float()
        if cap > 0:
            ds = ds * (1 - t * t)
        ds = ds * scale
        out["dq"] = (ds.unsqueeze(-2) @ kg).squeeze(-2).to(dt)
        del kg, vg
        flat = ((b * Hkv + head) * Nk + j).reshape(-1)
        rows = (B * Hkv * Nk, D)
        out["dk"] = torch.zeros(rows, device="cuda").index_add_(
            0, flat, (ds.unsqueeze(-1) * q.unsqueeze(3)).view(-1, D)).view(B, Hkv, Nk, D).to(dt)
        out["dv"] = torch.zeros(rows, device="cuda").index_add_(
            0, flat, (p.unsqueeze(-1) * do.unsqueeze(3)).view(-1, D)).view(B, Hkv, Nk, D).to(dt)
    return out


def _plain_norm_rope_one(x, w, cos, sin, heads, dy):
    B, N = x.shape[:2]
    dt = x.dtype
    xf = x.float().view(B, N, heads, -1)
    D = xf.shape[-1]
    wf, c, s = w.float(), cos.float().unsqueeze(2), sin.float().unsqueeze(2)
    r = torch.rsqrt((xf * xf).mean(dim=-1, keepdim=True) + 1e-6)
    n = xf * r
    y = n * wf
    turned = torch.cat([-y[..., D // 2:], y[..., : D // 2]], dim=-1)
    out = (y * c + turned * s).transpose(1, 2).contiguous().to(dt)
    if dy is None:
        return out, None, None
    g = dy.float().transpose(1, 2)
    gs = g * s
    gy = g * c + torch.cat([gs[..., D // 2:], -gs[..., : D // 2]], dim=-1)
    dw = (gy * n).double().sum(dim=(0, 1, 2)).to(dt)
    gn = gy * wf
    dx = (r * (gn - n * (gn * n).mean(dim=-1, keepdim=True))).reshape(x.shape).to(dt)
    return out, dx, dw


def _plain_norm_rope(st):
    case = st["case"]
    q, dq, dwq = _plain_norm_rope_one(st["q"], st["wq"], st["cos"], st["sin"], case["H"], st.get("dq"))
    k, dk, dwk = _plain_norm_rope_one(st["k"], st["wk"], st["cos"], st["sin"], case["Hkv"], st.get("dk"))
    out = {"q": q, "k": k}
    if case["train"]:
        out.update(dq=dq, dk=dk, dwq=dwq, dwk=dwk)
    return out


def _plain_distill(st):
    case = st["case"]
    V, tau = case["V"], case["temperature"]
    z = st["logits"].float() / tau
    ok = (st["ids"] >= 0) & (st["ids"] < V)
    at = st["ids"].long().clamp(0, V - 1)
    t = (st["teacher"].float() / tau).masked_fill(~ok, float("-inf"))
    any_ok = ok.any(dim=1, keepdim=True)
    t_top = torch.where(any_ok, t.amax(dim=1, keepdim=True), torch.zeros_like(t[:, :1]))
    te = torch.exp(t - t_top)
    t_sum = te.sum(dim=1, keepdim=True).clamp_min(1e-30)
    p = te / t_sum
    log_p = torch.where(ok, t - t_top - torch.log(t_sum), torch.zeros_like(t))
    top = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    log_q = z.gather(1, at) - top - torch.log(total)
    rows = tau * tau * torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(dim=1)
    w = any_ok[:, 0].float() if st["weight"] is None else st["weight"] * any_ok[:, 0]
    weight = w.double().sum().clamp_min(1e-30)
    loss = ((rows.double() * w).sum() / weight).float()
    dz = (e / total).scatter_add_(1, at, -p) * (tau * w / weight.float()).unsqueeze(1)
    return {"loss": loss, "dlogits": dz.to(st["logits"].dtype)}


# ------------------------------------------------------------------------------- the framework's calls


def _own_attention(st):
    from ossa_b200 import topk_attention

    case = st["case"]
    opts = dict(q_start=st["q_start"], softcap=case["softcap"] or None, slopes=st["slopes"],
                segments=st["segments"], prefix_len=st["prefix"])
    if not case["train"]:
        return {"out": topk_attention(st["q"], st["k"], st["v"], topk_indices=st["idx"], **opts)}
    q, k, v = (st[x].detach().requires_grad_() for x in ("q", "k", "v"))
    leaves = [q, k, v]
    if st["slopes"] is not None:
        opts["slopes"] = st["slopes"].detach().requires_grad_()
        leaves.append(opts["slopes"])
    out = topk_attention(q, k, v, topk_indices=st["idx"], **opts)
    grads = torch.autograd.grad(out, leaves, st["dout"])
    res = dict(zip(("dq", "dk", "dv", "dslopes"), grads))
    res["out"] = out.detach()
    return res


def _own_norm_rope(st):
    from ossa_b200 import qk_norm_rope

    case = st["case"]
    if not case["train"]:
        q, k = qk_norm_rope(st["q"], st["k"], case["H"], case["Hkv"], st["wq"], st["wk"], st["cos"], st["sin"])
        return {"q": q, "k": k}
    leaves = [st[x].detach().requires_grad_() for x in ("q", "k", "wq", "wk")]
    q, k = qk_norm_rope(leaves[0], leaves[1], case["H"], case["Hkv"], leaves[2], leaves[3], st["cos"], st["sin"])
    dq, dk, dwq, dwk = torch.autograd.grad((q, k), leaves, (st["dq"], st["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def _own_distill(st):
    from ossa_b200.train import top_logit_distillation_loss

    z = st["logits"].detach().requires_grad_()
    loss = top_logit_distillation_loss(z, st["teacher"], st["ids"], temperature=st["case"]["temperature"],
                                       row_weight=st["weight"])
    (dz,) = torch.autograd.grad(loss, z)
    return {"loss": loss.detach(), "dlogits": dz}


def run(state):
    op = state["case"]["op"]
    if own:
        call = {"attention": _own_attention, "norm_rope": _own_norm_rope, "distill": _own_distill}[op]
    else:
        call = {"attention": _plain_attention, "norm_rope": _plain_norm_rope, "distill": _plain_distill}[op]
    return call(state)


# ------------------------------------------------------------------------------- work


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "attention":
        B, H, Hkv, Nq, Nk, K, D = (case[x] for x in ("B", "H", "Hkv", "Nq", "Nk", "K", "D"))
        G = H // Hkv
        rows = B * H * Nq
        # keys that some head lists: the recent ones and half of the others are common to a group
        keys = B * Hkv * min(Nk, (Nq - 1) + K // 2 + (K - K // 2) // 2 * (G + 1) * Nq)
        qo, kv, ix = rows * D * size, 2 * keys * D * size, rows * K * 4
        small = (H * 4 if case["slopes"] else 0) + (B * Nk * 4 if case["docs"] else 0)
        if not case["train"]:
            return {"bytes": 2 * qo + kv + ix + small, "flops": 4 * rows * K * D}
        # q, k, v, dout and the lists in; out, dq, dk, dv out (dk, dv for every key)
        return {"bytes": 4 * qo + kv + 2 * B * Hkv * Nk * D * size + ix + small, "flops": 12 * rows * K * D}
    if case["op"] == "norm_rope":
        B, N, H, Hkv, D = (case[x] for x in ("B", "N", "H", "Hkv", "D"))
        x = B * N * (H + Hkv) * D
        table = 2 * B * N * D * size
        if not case["train"]:
            return {"bytes": 2 * x * size + table, "flops": 8 * x}
        return {"bytes": 4 * x * size + table, "flops": 24 * x}
    T, V, K = case["T"], case["V"], case["K"]
    return {"bytes": 2 * T * V * size + T * K * 8 + 4 * T, "flops": 8 * T * V}


# ------------------------------------------------------------------------------- 64 bits


def _exact_attention(case, st):
    """Dense: every key of a row, weighted by how often the row lists it."""
    B, H, Hkv, Nq, Nk, D = (case[x] for x in ("B", "H", "Hkv", "Nq", "Nk", "D"))
    G = H // Hkv
    q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
    k, v = k.repeat_interleave(G, dim=1), v.repeat_interleave(G, dim=1)
    i = torch.arange(Nk - Nq, Nk, device="cuda")[:, None]
    j = torch.arange(Nk, device="cuda")[None, :]
    visible = (j <= i)[None].expand(B, Nq, Nk)
    if case["prefix"]:
        visible = visible | (j[None] < st["prefix"].view(B, 1, 1))
    if case["docs"]:
        seg = st["segments"]
        visible = visible & (seg[:, Nk - Nq:, None] == seg[:, None, :])
    times = torch.zeros(B, H, Nq, Nk + 1, device="cuda", dtype=torch.uint8)
    ids = st["idx"].long()
    ids = torch.where((ids >= 0) & (ids < Nk), ids, torch.full_like(ids, Nk))
    times = times.scatter_add_(3, ids, torch.ones_like(ids, dtype=torch.uint8))[..., :Nk]
    times = times * visible[:, None]
    x = torch.matmul(q, k.transpose(2, 3)).div_(math.sqrt(D))
    slope = None
    if case["softcap"] > 0:
        x = x.div_(case["softcap"]).tanh_()
        slope = 1 - x.square()
        x.mul_(case["softcap"])
    dist = (i - j).abs().double()
    if case["slopes"]:
        x.addcmul_(st["slopes"].double().view(1, H, 1, 1), dist, value=-1)
    x.masked_fill_(times == 0, float("-inf"))
    x.sub_(torch.nan_to_num(x.amax(dim=3, keepdim=True), neginf=0.0)).exp_().mul_(times)
    norm = x.sum(dim=3, keepdim=True)
    x.div_(norm.masked_fill_(norm == 0, 1.0))  # the probabilities
    res = {"out": torch.matmul(x, v)}
    if case["train"]:
        do = st["dout"].double()
        res["dv"] = torch.matmul(x.transpose(2, 3), do).view(B, Hkv, G, Nk, D).sum(dim=2)
        y = torch.matmul(do, v.transpose(2, 3))
        y.sub_((res["out"] * do).sum(dim=3, keepdim=True)).mul_(x)
        del x, times
        if case["slopes"]:
            res["dslopes"] = -(y * dist).sum(dim=(0, 2, 3))
        if slope is not None:
            y.mul_(slope)
        y.div_(math.sqrt(D))
        res["dq"] = torch.matmul(y, k)
        res["dk"] = torch.matmul(y.transpose(2, 3), q).view(B, Hkv, G, Nk, D).sum(dim=2)
    return res


def _exact_norm_rope(case, st):
    def one(x, w, heads, dy):
        B, N, D = case["B"], case["N"], case["D"]
        xd = x.double().requires_grad_(case["train"])
        wd = w.double().requires_grad_(case["train"])
        with torch.enable_grad():
            h = xd.view(B, N, heads, D).permute(0, 2, 1, 3)
            h = h / (h.square().sum(-1, keepdim=True) / D + 1e-6).sqrt() * wd
            # a rotation of the pairs (d, d + D/2) as complex numbers, where the table's halves agree
            c, s = st["cos"].double()[:, None], st["sin"].double()[:, None]
            a, b = h[..., : D // 2], h[..., D // 2:]
            y = torch.cat([a * c[..., : D // 2] - b * s[..., : D // 2], b * c[..., D // 2:] + a * s[..., D // 2:]], -1)
        if not case["train"]:
            return y, None, None
        gx, gw = torch.autograd.grad(y, (xd, wd), dy.double())
        return y.detach(), gx, gw

    q, dq, dwq = one(st["q"], st["wq"], case["H"], st.get("dq"))
    k, dk, dwk = one(st["k"], st["wk"], case["Hkv"], st.get("dk"))
    res = {"q": q, "k": k}
    if case["train"]:
        res.update(dq=dq, dk=dk, dwq=dwq, dwk=dwk)
    return res


def _exact_distill(case, st):
    tau = case["temperature"]
    ids = st["ids"].long()
    ok = (ids >= 0) & (ids < case["V"])
    p = torch.softmax((st["teacher"].double() / tau).masked_fill(~ok, -1e300), dim=1).masked_fill(~ok, 0.0)
    log_q = torch.log_softmax(st["logits"].double() / tau, dim=1)
    w = ok.any(dim=1).double()
    if st["weight"] is not None:
        w = w * st["weight"].double()
    if float(w.sum()) == 0.0:
        return {"loss": torch.zeros((), dtype=torch.float64), "dlogits": torch.zeros_like(log_q)}
    kl = (torch.special.xlogy(p, p) - p * log_q.gather(1, ids.clamp(0, case["V"] - 1))).sum(dim=1)
    dz = log_q.exp_()
    dz.scatter_add_(1, ids.clamp(0, case["V"] - 1), -p)
    dz.mul_((tau * w / w.sum())[:, None])
    return {"loss": tau * tau * (w * kl).sum() / w.sum(), "dlogits": dz}


def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "norm_rope": _exact_norm_rope, "distill": _exact_distill}[case["op"]](case, st)
