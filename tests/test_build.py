"""CPU: what the build does where torch is missing or another one."""
from __future__ import annotations

import importlib.util
import subprocess
import sys

import pytest

from mini_triton_nvgpu_v1_b200 import build


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """The compilers' commands, recorded instead of run; outputs in tmp_path."""
    ran = []

    def run(cmd, verbose):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return ""

    monkeypatch.setattr(build, "_run", run)
    monkeypatch.setattr(build, "LIB", tmp_path / "libtbgemm.so")
    monkeypatch.setattr(build, "TORCH_LIB", tmp_path / "_tbtorch.so")
    monkeypatch.setattr(build, "TORCH_TAG", tmp_path / "_tbtorch.so.tag")
    return ran


def _kinds(commands):
    return sorted({"torch" if "-ltorch_python" in c else "library" for c in commands})


def test_the_c_library_is_built_without_torch(commands, monkeypatch, capsys):
    monkeypatch.setattr(build, "ROOT", build.TORCH_LIB.parent)   # objects go there too
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: None)
    monkeypatch.setattr(build, "_stale", lambda out, inputs: True)
    assert build.build() == build.LIB and build.LIB.exists()
    assert _kinds(commands) == ["library"]
    assert "torch is not installed" in capsys.readouterr().err
    assert build.build_torch() is None


def test_another_torch_or_python_is_built_for_anew(commands):
    assert build.build_torch() == build.TORCH_LIB and len(commands) == 1
    assert build.build_torch() == build.TORCH_LIB and len(commands) == 1   # up to date
    build.TORCH_TAG.write_text(build.TORCH_TAG.read_text().replace("version", "verslon"))
    assert build.build_torch() == build.TORCH_LIB and len(commands) == 2
    build.TORCH_TAG.unlink()
    build.build_torch()
    assert len(commands) == 3 and _kinds(commands) == ["torch"]


def test_a_failed_command_is_named():
    with pytest.raises(RuntimeError, match="false failed"):
        build._run(["false"], False)


@pytest.mark.parametrize("torch", [True, False])
def test_star_import(torch):
    """All names with torch; without it the ones that do not need it."""
    code = ("import sys\n" + ("" if torch else "sys.modules['torch'] = None\n") +
            "from mini_triton_nvgpu_v1_b200 import *\n"
            "assert matmul and plan_for and KernelConfig and version()\n"
            f"assert ('grouped_matmul' in globals()) is {torch}\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=build.ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
