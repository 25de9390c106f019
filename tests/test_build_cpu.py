"""When the build takes the tensor-level entry points' library for current (no GPU)."""
import importlib.util
import os
import subprocess
from types import SimpleNamespace

import pytest
import torch

from conftest import PKG_ROOT


@pytest.fixture
def build(monkeypatch, tmp_path):
    """The build module with its outputs under ``tmp_path`` and a compiler that notes its calls."""
    spec = importlib.util.spec_from_file_location("spx_build", os.path.join(PKG_ROOT, "csrc", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.FRONT, mod.BUILD = str(tmp_path / "_spx_front.so"), str(tmp_path / "_build")
    mod.calls = []

    def compiler(cmd, **kw):
        mod.calls.append(cmd)
        if mod.works:
            open(mod.FRONT, "w").close()
        return SimpleNamespace(returncode=0 if mod.works else 1, stdout="", stderr="")

    mod.works = True
    monkeypatch.setattr(subprocess, "run", compiler)
    return mod


@pytest.mark.parametrize("what", ["torch", "abi", "python"])
def test_another_torch_or_python_rebuilds_the_front(build, monkeypatch, what):
    build.build_front()
    build.build_front()
    assert len(build.calls) == 1
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "9.9.9")
    elif what == "abi":
        now = torch.compiled_with_cxx11_abi()
        monkeypatch.setattr(torch, "compiled_with_cxx11_abi", lambda: not now)
    else:
        import sysconfig
        real = sysconfig.get_config_var
        monkeypatch.setattr(sysconfig, "get_config_var", lambda n: "other" if n == "SOABI" else real(n))
    build.works = False
    with pytest.raises(RuntimeError):
        build.build_front()
    build.works = True
    build.build_front()             # a build that failed is not taken for done
    build.build_front()
    assert len(build.calls) == 3


def test_a_front_without_a_record_is_rebuilt(build):
    open(build.FRONT, "w").close()
    build.build_front()
    assert len(build.calls) == 1
    build.build_front(force=True)
    assert len(build.calls) == 2
