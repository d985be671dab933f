"""The package imports where torch has no GPU support: the operators refuse
tensors at the call, not the module at its import."""
import importlib.util
import sys

import pytest
import torch

from conftest import PKG_DIR


def test_ops_import_without_gpu_support(monkeypatch):
    for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
        monkeypatch.delattr(torch._C, name)
    name = "g4mi_cpu_torch"
    spec = importlib.util.spec_from_file_location(name, PKG_DIR / "__init__.py", submodule_search_locations=[str(PKG_DIR)])
    mod = importlib.util.module_from_spec(spec)
    try:
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
        ops = importlib.import_module(name + ".ops")
        x = torch.zeros(4, 64)
        with pytest.raises(ValueError, match="device tensors"):
            ops.pre_rmsnorm_i8(x, torch.zeros(64), M=4, D=64)
    finally:
        for n in [n for n in sys.modules if n == name or n.startswith(name + ".")]:
            del sys.modules[n]
