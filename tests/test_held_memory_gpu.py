"""What the training calls hold: nothing of the backward pass behind it while the losses live on, and nothing under
checkpointing or offloading that these were asked to drop."""

import gc

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from ossa_b200 import top_logit_distillation_loss

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T, V, K = 512, 32000, 64
SIZE = T * V * 2  # bytes of the logits, and of their gradient


def _case():
    g = torch.Generator().manual_seed(3)
    z = torch.randn(T, V, generator=g).bfloat16().to(DEV).requires_grad_()
    ids = torch.randint(0, V, (T, K), generator=g).to(DEV)
    teacher = torch.randn(T, K, generator=g).to(DEV)
    return z, teacher, ids


def _held():
    torch.cuda.synchronize()
    gc.collect()
    return torch.cuda.memory_allocated()


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_losses_that_are_kept(reduction):
    z, teacher, ids = _case()
    up = torch.ones((T,) if reduction == "none" else (), device=DEV)

    def step():
        loss = top_logit_distillation_loss(z, teacher, ids, reduction=reduction)
        torch.autograd.grad(loss, z, up)
        return loss

    step()
    before = _held()
    losses = [step() for _ in range(5)]
    # a loss of its own each, in blocks of 512 bytes
    assert _held() - before <= 5 * max(512, 4 * losses[0].numel())


def test_checkpointed_forward():
    """Behind a checkpointed forward pass only the loss is held; the backward pass makes one gradient."""
    z, teacher, ids = _case()

    def call(x):
        return top_logit_distillation_loss(x, teacher, ids)

    (want,) = torch.autograd.grad(call(z), z)
    before = _held()
    loss = checkpoint(call, z, use_reentrant=False)
    assert _held() - before <= 4096
    torch.cuda.reset_peak_memory_stats()
    (got,) = torch.autograd.grad(loss, z)
    # the recomputed gradient is the one returned; the rest is the workspace, 16 bytes an entry
    assert torch.cuda.max_memory_allocated() - before <= SIZE + 24 * T * K + (1 << 20)
    assert torch.equal(got, want)


def test_offloaded_gradient():
    z, teacher, ids = _case()
    (want,) = torch.autograd.grad(top_logit_distillation_loss(z, teacher, ids), z)
    before = _held()
    with torch.autograd.graph.save_on_cpu():
        loss = top_logit_distillation_loss(z, teacher, ids)
    assert _held() - before <= 4096
    (got,) = torch.autograd.grad(loss, z)
    assert torch.equal(got, want)


def test_backward_twice():
    """A graph that is kept: the first and later passes accumulate into the leaf; a gradient changed in place does not
    change the next one."""
    z, teacher, ids = _case()
    loss = top_logit_distillation_loss(z, teacher, ids)
    (want,) = torch.autograd.grad(top_logit_distillation_loss(z, teacher, ids), z)
    (first,) = torch.autograd.grad(loss, z, retain_graph=True)
    assert torch.equal(first, want)
    first.mul_(3.0)
    loss.backward(retain_graph=True)
    assert torch.equal(z.grad, want)
    loss.backward()
    assert torch.equal(z.grad, want + want)
    with pytest.raises(RuntimeError, match="second time|already been freed"):
        torch.autograd.grad(loss, z)
