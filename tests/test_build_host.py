"""CPU: when the Python extension of the dense operators is built again."""
import importlib.util
import os
import subprocess
import types

import pytest
import torch


@pytest.fixture()
def build(tmp_path, monkeypatch):
    """csrc/build.py with its outputs in a folder of the test and a compiler that only writes the output file."""
    import __graft_entry__ as g
    spec = importlib.util.spec_from_file_location("csrc_build_under_test", os.path.join(g.PKG_DIR, "csrc", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    monkeypatch.setattr(mod, "FASTCALL", str(tmp_path / "_fastcall.so"))
    if hasattr(mod, "FASTCALL_KEY"):
        monkeypatch.setattr(mod, "FASTCALL_KEY", str(tmp_path / "obj" / "fastcall.key"))
    mod.runs, mod.code = [], 0

    def run(cmd, **kw):
        mod.runs.append(cmd)
        if mod.code == 0:
            with open(mod.FASTCALL, "w"):
                pass
        return types.SimpleNamespace(returncode=mod.code, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    return mod


def test_built_once_for_a_torch_and_again_for_another(build, monkeypatch):
    build.build_fastcall()
    build.build_fastcall()
    assert len(build.runs) == 1
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build.build_fastcall()
    build.build_fastcall()
    assert len(build.runs) == 2


def test_a_failed_build_is_tried_again(build, monkeypatch):
    build.build_fastcall()
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build.code = 1
    with pytest.raises(RuntimeError, match="g\\+\\+ failed"):
        build.build_fastcall()
    build.code = 0
    assert os.path.exists(build.FASTCALL) and not build.fastcall_up_to_date()
    build.build_fastcall()
    assert len(build.runs) == 3 and build.fastcall_up_to_date()
