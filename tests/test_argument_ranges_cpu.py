"""Arguments that fp32 cannot hold are refused, not rounded to another meaning; sizes that are refused get no workspace."""

import pytest
import torch

from ossa_b200 import _lib, top_logit_distillation_loss, topk_attention
from test_operators_cpu import BF, INF, INV, _distill, _mod_bwd, _mod_fwd, _qkv


@pytest.mark.parametrize("cap", [1e-50, 1e-40, 2.0 ** -127, 1e39])
def test_caps_outside_fp32(cap):
    """A cap that rounds to 0 would be no cap at all; one below the normal range has no finite inverse."""
    q, k, v, idx = _qkv()
    with pytest.raises(ValueError, match="softcap"):
        topk_attention(q, k, v, topk_indices=idx, softcap=cap)
    if cap < 1:
        small = float(torch.tensor(cap, dtype=torch.float32))
        if small:
            assert _mod_fwd(cap=small) == INV and _mod_bwd(cap=small) == INV


@pytest.mark.parametrize("tau", [1e-50, 1e-40, 2.0 ** -127, 1e39])
def test_temperatures_outside_fp32(tau):
    z, t, ids = torch.zeros(5, 9), torch.zeros(5, 3), torch.zeros(5, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="temperature"):
        top_logit_distillation_loss(z, t, ids, temperature=tau)
    if tau < 1:
        small = float(torch.tensor(tau, dtype=torch.float32))
        for fn in ("fwd", "bwd"):
            assert _distill(fn, tau=small) == INV


def test_the_distillation_workspace_of_refused_sizes():
    size = _lib.lib().ossa_top_logit_distill_workspace_size
    assert size(10, 1024) > 0 and size(10, 1025) == 0 and size((1 << 30) + 1, 4) == 0
