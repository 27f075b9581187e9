"""What the build says when a compiler fails (no compiler runs)."""
import subprocess

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
