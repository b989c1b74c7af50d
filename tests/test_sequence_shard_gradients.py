"""Gradients through the sharded attention: each rank's gradients of its own blocks of q, k and v are the matching
rows of the unsharded gradients (gloo ranks on the CPU, a plain attention in the kernels' place)."""

import os
import socket

import pytest
import torch
import torch.multiprocessing as mp

from mod_attention_ref import attention
from ossa_b200.sequence_shard import gather_sequence, local_rows, zigzag_blocks
from shard_workers import _init, shard_inputs


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _select(q, k, wq, wk, pos_bias, seq_len, top_k, causal=True, q_start=0):
    """Any fixed choice of keys: the row's last ones and some before them."""
    pos = q_start + torch.arange(q.shape[2]).view(-1, 1)
    step = torch.arange(top_k).view(1, -1)
    idx = pos - step * (1 + step // 3)
    return idx.clamp_min(-1).expand(q.shape[0], q.shape[1], -1, -1)


def _attend(q, k, v, topk_indices, causal=True, q_start=0):
    return attention(q.double(), k.double(), v.double(), topk_indices, causal=causal, q_start=q_start)[0].to(q.dtype)


def _inputs(shape, dtype):
    B, H, Hkv, N, D, r, L, K = shape
    q, k, v, wq, wk, pb = shard_inputs(B, H, Hkv, N, D, r, L, seed=3)
    do = torch.randn(B, H, N, D, generator=torch.Generator().manual_seed(5))
    return [t.to(dtype) for t in (q, k, v, do)], (wq, wk, pb)


def _worker(rank, world, port, shape, dtype, wanted, out_dir):
    from ossa_b200.sequence_shard import sharded_routed_attention

    _init(rank, world, port, "gloo")
    try:
        (q, k, v, do), (wq, wk, pb) = _inputs(shape, dtype)
        parts = [local_rows(t, world, rank).requires_grad_(n in wanted) for n, t in zip("qkv", (q, k, v))]
        out = sharded_routed_attention(*parts, wq, wk, pb, shape[6], shape[7], select_fn=_select, attend_fn=_attend)
        leaves = [t for t in parts if t.requires_grad]
        grads = torch.autograd.grad(out, leaves, local_rows(do, world, rank)) if leaves else ()
        torch.save((out.detach(), [t.detach() for t in grads]), os.path.join(out_dir, f"rank{rank}.pt"))
        with torch.no_grad():
            again = sharded_routed_attention(*parts, wq, wk, pb, shape[6], shape[7], select_fn=_select, attend_fn=_attend)
        assert not again.requires_grad and torch.equal(again, out.detach())
    finally:
        torch.distributed.destroy_process_group()


@pytest.mark.parametrize("world,dtype,wanted", [(2, torch.float64, "qkv"), (3, torch.float64, "qkv"), (2, torch.float64, "k"),
                                                (2, torch.float64, "qv"), (2, torch.bfloat16, "qkv"), (2, torch.float64, "")])
def test_gradients_match_unsharded(world, dtype, wanted, tmp_path):
    shape = (2, 4, 2, 16 * world, 8, 4, 64, 5)  # B, H, Hkv, N, D, r, seq_len, K
    mp.spawn(_worker, args=(world, _free_port(), shape, dtype, wanted, str(tmp_path)), nprocs=world, join=True)
    (q, k, v, do), _ = _inputs(shape, dtype)
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    idx = _select(q, k, None, None, None, None, shape[7])
    out = _attend(*leaves, idx)
    want = dict(zip("qkv", torch.autograd.grad(out, leaves, do.double())))
    # 64 bits: equal to the order of sums.  bf16: a key's gradient is rounded (half a step is 2^-8) for each of a rank's
    # two blocks, where these are added and where the ranks' parts are
    bound = 1e-12 if dtype == torch.float64 else 3 * 2.0 ** -8
    for rank in range(world):
        got_out, got = torch.load(tmp_path / f"rank{rank}.pt")
        ref = local_rows(out.detach(), world, rank)
        assert (got_out.double() - ref).norm() <= bound * ref.norm()
        assert len(got) == len(wanted)
        for n, g in zip(wanted, got):
            ref = local_rows(want[n], world, rank)
            assert g.dtype == dtype and (g.double() - ref).norm() <= bound * ref.norm(), n


def _sum_worker(rank, world, port, out_dir):
    """The adjoint of the gather alone: every rank's gradient of the whole sequence, summed in fp32 and rounded once."""
    _init(rank, world, port, "gloo")
    try:
        x = torch.zeros(1, 2, 8, 4, dtype=torch.bfloat16, requires_grad=True)
        full = gather_sequence(x, world)
        up = torch.full(full.shape, 1.0 if rank == 0 else 2.0 ** -8, dtype=torch.bfloat16)
        (g,) = torch.autograd.grad(full, x, up, create_graph=False)
        torch.save(g, os.path.join(out_dir, f"rank{rank}.pt"))
    finally:
        torch.distributed.destroy_process_group()


def test_parts_are_summed_in_fp32(tmp_path):
    """1 + 2^-8 + 2^-8: rounded to bf16 after each addition it stays 1, summed first it is 1 + 2^-7."""
    mp.spawn(_sum_worker, args=(3, _free_port(), str(tmp_path)), nprocs=3, join=True)
    for rank in range(3):
        assert (torch.load(tmp_path / f"rank{rank}.pt") == 1 + 2.0 ** -7).all()


def test_single_rank_is_differentiable():
    x = torch.randn(2, 3, 16, 4, dtype=torch.float64, requires_grad=True)
    up = torch.randn(2, 3, 16, 4, dtype=torch.float64)
    (g,) = torch.autograd.grad(gather_sequence(local_rows(x, 1, 0), 1), x, up)
    assert torch.equal(g, up)
    assert zigzag_blocks(16, 1, 0) == [(0, 8), (8, 16)]
