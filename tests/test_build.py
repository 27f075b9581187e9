"""What the build does where a compiler fails or torch is not installed (no compiler runs)."""
import subprocess
import sys

import pytest

from sparsesam_b200 import build


@pytest.mark.parametrize("tool", ["nvcc", "g++"])
def test_the_failing_tool_is_named(monkeypatch, tool):
    def run(cmd, **_):
        failed = cmd[0].rsplit("/", 1)[-1] == tool
        return subprocess.CompletedProcess(cmd, int(failed), "", "no such header" if failed else "")

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    with pytest.raises(RuntimeError, match=f"^{tool.replace('+', '[+]')} failed") as e:
        build.build(force=True)
    assert "no such header" in str(e.value)


def test_the_library_needs_no_torch(monkeypatch):
    """The C ABI is built alone; the extension module of a torch that is not there is not."""
    ran, placed = [], []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **_: ran.append(cmd) or subprocess.CompletedProcess(cmd, 0, "", ""))
    monkeypatch.setattr(build.os, "replace", lambda a, b: placed.append(b))
    monkeypatch.setattr(build, "_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build(force=True) == build.LIB_PATH
    assert placed == [build.LIB_PATH] and not any("torch" in word for cmd in ran for word in cmd)
