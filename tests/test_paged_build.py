"""The compiled entry of the paged-cache calls is made for one torch and one Python: when it is built again, and that the package
does without it where it does not fit.  No GPU."""
import subprocess
import sys
import types
from pathlib import Path

import pytest
import torch

from lvar_b200 import build as B

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def made(tmp_path, monkeypatch):
    """_build_host over a folder of its own and a compiler that only writes its output: what it was called with."""
    calls = []
    (tmp_path / "paged_host.cpp").write_text("")
    (tmp_path / "lvar_b200.h").write_text("")
    for name, value in {"CSRC": tmp_path, "INCLUDE": tmp_path, "BUILD_DIR": tmp_path / "build", "PKG_DIR": tmp_path,
                        "HOST_PATH": tmp_path / "_paged_host.so"}.items():
        monkeypatch.setattr(B, name, value)
    (tmp_path / "build").mkdir()

    def run(cmd, **_):
        calls.append(cmd)
        rc = 1 if getattr(run, "fails", False) else 0
        if rc == 0:
            Path(cmd[cmd.index("-o") + 1]).write_text("module")
        return types.SimpleNamespace(returncode=rc, stdout="", stderr="")
    monkeypatch.setattr(B.subprocess, "run", run)
    calls_and_run = types.SimpleNamespace(calls=calls, run=run)
    return calls_and_run


def test_built_once_and_again_for_another_torch(made, monkeypatch):
    B._build_host(False)
    B._build_host(False)
    assert len(made.calls) == 1
    monkeypatch.setattr(torch, "__version__", "2.99.0")
    B._build_host(False)
    B._build_host(False)
    assert len(made.calls) == 2
    monkeypatch.setattr(B.sysconfig, "get_config_var", lambda name: "cpython-399-somewhere" if name == "SOABI" else None)
    B._build_host(False)
    B._build_host(False)
    assert len(made.calls) == 3
    B._build_host(True)
    assert len(made.calls) == 4


def test_a_build_that_failed_is_tried_again(made, monkeypatch):
    B._build_host(False)
    monkeypatch.setattr(torch, "__version__", "2.99.0")
    made.run.fails = True
    for n in (2, 3):
        with pytest.raises(RuntimeError):
            B._build_host(False)
        assert len(made.calls) == n
    made.run.fails = False
    B._build_host(False)
    B._build_host(False)
    assert len(made.calls) == 4


def _child(prepare: str) -> str:
    code = f"""
import sys, types, warnings
sys.path.insert(0, {str(ROOT)!r})
{prepare}
with warnings.catch_warnings(record=True) as w:
    warnings.simplefilter("always")
    from lvar_b200 import kernels as K
assert K._paged_host is None, K._paged_host
assert any("python -m lvar_b200.build" in str(x.message) for x in w), [str(x.message) for x in w]
import lvar_b200.policy, lvar_b200.sparse_attn_ops, lvar_b200.paged
import torch
k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
table, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
x = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
for call in (lambda: K.paged_kv_append(x, x, k, k, table, n), lambda: K.paged_qkv_prologue(x, x, x, k, k, table, n),
             lambda: K.paged_kv_read(k, k, table, n, 1), lambda: K.paged_attn_fwd(x, k, k, table, n)):
    try:
        call()
    except RuntimeError as e:
        assert "CUDA" in str(e)
    else:
        raise SystemExit("not refused")
print("fine")
"""
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert res.returncode == 0, res.stderr
    return res.stdout


def test_the_package_imports_without_it():
    assert "fine" in _child("sys.modules['lvar_b200._paged_host'] = None")


def test_one_for_another_torch_is_left_alone():
    fake = "m = types.ModuleType('lvar_b200._paged_host'); m.built_for = 'torch 1.0'; sys.modules['lvar_b200._paged_host'] = m"
    assert "fine" in _child(fake + "; import lvar_b200; lvar_b200._paged_host = m")


def test_the_one_that_is_built_fits():
    from lvar_b200 import kernels
    assert kernels._paged_host is not None and kernels._paged_host.built_for == B.host_key()
