"""The build's rules, without building: what the default target takes for an interpreter with and without torch."""
import os
import subprocess
import sys

from conftest import ROOT


def _dry_run(python):
    out = subprocess.run(["make", "-Bn", "-C", os.path.join(ROOT, "luisaml_b200"), f"PYTHON={python}"], capture_output=True, text=True)
    return out.returncode, out.stdout, out.stderr


def test_the_libraries_build_without_torch():
    rc, out, err = _dry_run(f"{sys.executable} -I -S")  # no site-packages
    assert rc == 0, err
    assert "-o lib/liblcml_fp8.so" in out and "-o lib/liblcml_onnx.so" in out and "-o _decoder_bind.so" not in out
    assert "Traceback" not in err


def test_the_binding_is_built_for_the_interpreter_at_hand():
    rc, out, err = _dry_run(sys.executable)
    assert rc == 0, err
    import torch
    assert "-o _decoder_bind.so" in out and os.path.dirname(torch.__file__) in out


def test_build_names_its_own_interpreter(monkeypatch):
    sys.path.insert(0, ROOT)
    import __graft_entry__ as entry
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(entry.subprocess, "run", run)
    entry.build()
    mine = [c for c in calls if any(str(a).endswith("luisaml_b200") for a in c)]
    assert len(mine) == 1 and f"PYTHON={sys.executable}" in mine[0]
