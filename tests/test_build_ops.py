"""The Python extension is rebuilt for another torch or Python (no compiler or
GPU needed: the compilation itself is left out)."""
import importlib.util
import os

import pytest

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hy_mt_rs_b200", "build.py")


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("hyq_build", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "BUILD", str(tmp_path))
    monkeypatch.setattr(module, "OPS", str(tmp_path / "_ops.so"))
    module.compiled = []

    def compiler(cmd):
        module.compiled.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()

    monkeypatch.setattr(module.subprocess, "check_call", compiler)
    return module


def test_rebuilt_for_another_torch(build, monkeypatch):
    build._build_ops(False)
    build._build_ops(False)
    assert len(build.compiled) == 1
    monkeypatch.setattr(build.metadata, "version", lambda name: "99.0")
    build._build_ops(False)
    build._build_ops(False)
    assert len(build.compiled) == 2
    monkeypatch.setattr(build.sys, "version", "9.9")
    build._build_ops(False)
    assert len(build.compiled) == 3
    build._build_ops(True)
    assert len(build.compiled) == 4
