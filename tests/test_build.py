"""The autograd module is bound to one interpreter and one torch: a module built for others is not taken for it."""

import importlib.util
import sysconfig

import torch

from ossa_b200 import build


def test_module_names_its_abi():
    assert sysconfig.get_config_var("SOABI") in build.AUTOGRAD_PATH.name
    assert torch.__version__ in build.AUTOGRAD_PATH.name
    assert build.AUTOGRAD_PATH.parent == build.PKG_DIR


def test_another_torch_needs_another_module(monkeypatch):
    """With a module for this torch in place, the next version looks for its own and finds none."""
    build.build_autograd()
    assert not build.autograd_is_stale()
    spec = importlib.util.spec_from_file_location("other_build", build.__file__)
    other = importlib.util.module_from_spec(spec)
    monkeypatch.setattr(torch, "__version__", "99.0")
    spec.loader.exec_module(other)
    assert other.AUTOGRAD_PATH != build.AUTOGRAD_PATH and other.autograd_is_stale()
