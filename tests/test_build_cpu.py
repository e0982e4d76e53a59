"""The native build: what it needs, and when the torch module is made again."""

import os
import subprocess
import sys
import time
import types

import pytest
import torch

from kvserve_hpdps_b200.ops import build as B
from kvserve_hpdps_b200.ops import paged as P


@pytest.fixture
def fake(monkeypatch, tmp_path):
    """A build in an empty folder whose compiler only writes its output; returns the commands."""
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write(" ".join(cmd))
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")
    monkeypatch.setattr(B, "BUILD", str(tmp_path))
    monkeypatch.setattr(B, "BIND_PATH", str(tmp_path / "mod.so"))
    monkeypatch.setattr(B, "_build_library", lambda *a: None)
    monkeypatch.setattr(subprocess, "run", run)
    return calls


def _links(calls):
    return [c for c in calls if "-shared" in c]


def test_the_library_does_not_need_a_torch_for_cuda(fake, monkeypatch):
    monkeypatch.setattr(torch.version, "cuda", None)
    with pytest.warns(UserWarning, match="not built for CUDA"):
        assert B.build() == B.LIB_PATH
    monkeypatch.setitem(sys.modules, "torch", None)
    with pytest.warns(UserWarning, match="cannot be imported"):
        assert B.build() == B.LIB_PATH
    assert not fake


@pytest.mark.skipif(torch.version.cuda is None, reason="needs a torch for CUDA")
def test_another_torch_makes_the_module_again(fake, monkeypatch):
    for n, version in enumerate(["2.0", "2.0", "2.1", "2.0", "2.0"]):
        monkeypatch.setattr(torch, "__version__", version)
        B.build()
        assert len(_links(fake)) == (1, 1, 2, 3, 3)[n]
        last = _links(fake)[-1]
        assert any(f"torch_{version}_" in x for x in last)
        time.sleep(0.01)


@pytest.mark.skipif(torch.version.cuda is None, reason="needs a torch for CUDA")
def test_the_module_is_named_for_the_interpreter(fake):
    import sysconfig
    name = f"{B.BIND_NAME}{sysconfig.get_config_var('EXT_SUFFIX')}"
    assert name != B.BIND_NAME + ".so"
    P._native()
    assert os.path.basename(P._ops.__file__) == name


def test_a_module_for_another_torch_is_refused(monkeypatch):
    import kvserve_hpdps_b200.ops as ops
    P._native()
    monkeypatch.setattr(P, "_ops", None)
    other = types.SimpleNamespace(torch_version="1.0")
    monkeypatch.setitem(sys.modules, "kvserve_hpdps_b200.ops._paged_ops", other)
    monkeypatch.setattr(ops, "_paged_ops", other, raising=False)
    with pytest.raises(RuntimeError, match="built for torch 1.0"):
        P._native()
