"""A layer whose head norms are switched off (identity modules) is patched as one without."""

from types import SimpleNamespace

import pytest
import torch

from ossa_b200.bench.sparse_forward import _head_norms


def test_identity_is_no_norm():
    off = torch.nn.Identity()
    for q_norm, k_norm in ((off, off), (off, None), (None, off), (None, None)):
        assert _head_norms(SimpleNamespace(q_norm=q_norm, k_norm=k_norm, head_dim=64)) is None


def test_one_norm_alone_is_refused():
    norm = torch.nn.RMSNorm(64, eps=1e-6)
    for q_norm, k_norm in ((norm, torch.nn.Identity()), (None, norm)):
        with pytest.raises(TypeError):
            _head_norms(SimpleNamespace(q_norm=q_norm, k_norm=k_norm, head_dim=64))
