"""The torch module belongs to the torch that it was built for."""
import subprocess

import pytest
import torch

from roofline_decoding_b200 import _build, _lib


def test_a_module_of_another_torch_is_not_used(monkeypatch):
    monkeypatch.setattr(_lib, "_torch_module", None)
    assert _lib.torch_module().torch_version == torch.__version__
    monkeypatch.setattr(_lib, "_torch_module", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    with pytest.raises(ImportError, match="built for torch"):
        _lib.torch_module()
    assert _lib._torch_module is None


def test_a_module_of_another_torch_is_built_again(monkeypatch, tmp_path):
    """With the compiler replaced: once, then not again, then for every torch of its own."""
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        (tmp_path / "_w4torch.so").write_bytes(b"")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(_build, "BUILD_DIR", tmp_path / "objects")
    monkeypatch.setattr(_build, "TORCH_MODULE_PATH", tmp_path / "_w4torch.so")
    monkeypatch.setattr(_build.subprocess, "run", run)
    for version, builds in ((torch.__version__, 1), (torch.__version__, 1), ("9.9.9", 2), ("9.9.9", 2),
                            (torch.__version__, 3)):
        monkeypatch.setattr(torch, "__version__", version)
        _build.build_torch_module()
        assert len(calls) == builds
        assert any(f'-DW4_TORCH_VERSION="{version}"' == a for a in calls[-1])
    (tmp_path / "_w4torch.so").unlink()
    _build.build_torch_module()
    assert len(calls) == 4
