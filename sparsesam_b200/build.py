"""Builds libsparsesam_b200.so in-tree with nvcc for sm_100a.

The library is a plain C-ABI shared object (no torch headers), linked from the
translation units UNITS, which are compiled at the same time. Beside it the Python
extension module _torch_ops (csrc/torch_ops.cpp, torch headers, no device code; linked to
the library, which it finds beside itself) gives the decoder's operators their torch
form. Both are rebuilt when any csrc/ or include/ file is newer than they are. Where
torch is not installed, the library is built alone.
"""
from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(REPO_DIR, "include")
LIB_NAME = "libsparsesam_b200.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
TORCH_OPS_PATH = os.path.join(PKG_DIR, "_torch_ops.so")

UNITS = ["lib.cu", "cross_attention.cu", "cross_attention_fp16.cu", "cross_attention_bf16.cu", "norms.cu"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: set NVCC or install the CUDA toolkit")


def _sources() -> list[str]:
    out = []
    for d in (CSRC, INCLUDE):
        for name in sorted(os.listdir(d)):
            if name.endswith((".cu", ".cuh", ".h", ".cpp")):
                out.append(os.path.join(d, name))
    return out


def _torch_ops_commands(obj: str, lib: str, out: str) -> tuple[list[str], list[str]]:
    """Compile _torch_ops, and link it against this interpreter's torch and the library `lib`."""
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-DTORCH_EXTENSION_NAME=_torch_ops",
             "-I", os.path.join(root, "include"), "-I", os.path.join(root, "include", "torch", "csrc", "api", "include"),
             "-I", os.path.join(cuda, "include"), "-I", sysconfig.get_paths()["include"], "-I", INCLUDE,
             "-c", "-o", obj, os.path.join(CSRC, "torch_ops.cpp")],
            ["g++", "-shared", "-o", out, obj, lib, "-Wl,-rpath,$ORIGIN",
             "-L", os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"])


def _with_torch() -> bool:
    return importlib.util.find_spec("torch") is not None


def needs_build() -> bool:
    targets = [LIB_PATH, TORCH_OPS_PATH] if _with_torch() else [LIB_PATH]
    if not all(os.path.exists(t) for t in targets):
        return True
    t = min(os.path.getmtime(t) for t in targets)
    return any(os.path.getmtime(s) > t for s in _sources())


def build(force: bool = False, verbose: bool = False, extra_flags: list[str] | None = None) -> str:
    """Compile the library if it is missing or stale; return its path."""
    if not force and not needs_build():
        return LIB_PATH
    def run(cmd: list[str]) -> None:
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
        if verbose and (res.stdout or res.stderr):
            print(res.stdout, res.stderr, file=sys.stderr)

    tmp, tmp_ops = LIB_PATH + ".tmp", TORCH_OPS_PATH + ".tmp"
    with tempfile.TemporaryDirectory(prefix="ssam_build_") as work:
        objects = [os.path.join(work, unit + ".o") for unit in UNITS]
        units = [[_nvcc(), *NVCC_FLAGS, *(extra_flags or []), "-I", INCLUDE, "-c", "-o", obj, os.path.join(CSRC, unit)]
                 for unit, obj in zip(UNITS, objects)]
        link_ops = None
        if _with_torch():
            compile_ops, link_ops = _torch_ops_commands(os.path.join(work, "torch_ops.o"), tmp, tmp_ops)
            units.append(compile_ops)
        with ThreadPoolExecutor(len(units)) as pool:
            list(pool.map(run, units))
        run([_nvcc(), *NVCC_FLAGS, "-shared", "-Xlinker", f"-soname={LIB_NAME}", "-o", tmp, *objects])
        if link_ops is not None:
            run(link_ops)
    os.replace(tmp, LIB_PATH)
    if link_ops is not None:
        os.replace(tmp_ops, TORCH_OPS_PATH)
    return LIB_PATH


if __name__ == "__main__":
    force = "--force" in sys.argv
    extra = ["-Xptxas", "-v"] if "--ptxas-v" in sys.argv else None
    print(build(force=force, verbose=True, extra_flags=extra))
