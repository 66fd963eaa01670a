"""What is built where: the C library needs nvcc alone, the torch side of text
generation belongs to the interpreter that asks for it."""
import importlib
import importlib.util
import subprocess
import sys
import sysconfig

import pytest


def dry_run(pkg, *args):
    r = subprocess.run(["make", "-n", "-B", "-C", str(pkg.PKG_DIR), *args], capture_output=True, text=True)
    return r.returncode, r.stdout, r.stderr


def test_the_library_builds_without_python_or_torch(pkg):
    code, out, err = dry_run(pkg, "PYTHON=/nonexistent/python")
    assert code == 0 and not err, err
    assert "-o libbark3_b200.so" in out and "textgen_ext" not in out


def test_the_torch_side_is_named_for_its_interpreter(pkg):
    code, out, _ = dry_run(pkg, "textgen", f"PYTHON={sys.executable}")
    assert code == 0
    assert f"-o _textgen{sysconfig.get_config_var('EXT_SUFFIX')}" in out
    assert f"-I{sysconfig.get_paths()['include']} " in out


@pytest.mark.parametrize("torch_there", [True, False])
def test_build_asks_for_what_this_interpreter_can_use(pkg, monkeypatch, torch_there):
    calls = []
    monkeypatch.setattr(subprocess, "run", lambda cmd, **kw: calls.append(cmd))
    found = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec",
                        lambda name, *a: found(name, *a) if name != "torch" or torch_there else None)
    assert pkg.build(force=True) == pkg.LIB_PATH
    (cmd,) = calls
    assert cmd[:3] == ["make", "-C", str(pkg.PKG_DIR)] and f"PYTHON={sys.executable}" in cmd
    assert "libbark3_b200.so" in cmd and ("textgen" in cmd) == torch_there


def test_a_missing_torch_side_is_said(pkg, monkeypatch):
    tg = importlib.import_module("bark3_b200.textgen")
    monkeypatch.delitem(sys.modules, "bark3_b200._textgen", raising=False)
    monkeypatch.delattr(pkg, "_textgen", raising=False)
    monkeypatch.setattr(pkg, "__path__", [])
    with pytest.raises(pkg.B3Error, match="not built") as ei:
        tg._load()
    assert ei.value.code == pkg.B3_ESTATE
