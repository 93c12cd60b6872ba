"""Builds and runs a C++ program against libipus.so with host_runtime.h in place of
the HIP runtime (no device)."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
PACKAGE = os.path.join(ROOT, "ipu-stack_amd")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


def run_program(tmp_path, source):
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None or not os.path.isdir(os.path.join(ROCM, "include", "hip")):
        pytest.skip("no host compiler or no HIP headers")
    if not os.path.exists(os.path.join(PACKAGE, "libipus.so")):
        pytest.skip("the library is not built")
    (tmp_path / "program.cpp").write_text(source)
    # The program's own HIP functions come before the runtime's in the search.
    subprocess.run([compiler, "-std=c++20", "-g", "-O1", "-D__HIP_PLATFORM_AMD__", "-rdynamic", "-pthread",
                    "-I", HERE, "-I", os.path.join(ROOT, "include"), "-I", os.path.join(PACKAGE, "csrc"),
                    "-isystem", os.path.join(ROCM, "include"), "-Wno-unused-result",
                    "-o", str(tmp_path / "program"), str(tmp_path / "program.cpp"),
                    "-L", PACKAGE, "-l:libipus.so", f"-Wl,-rpath,{PACKAGE}", f"-Wl,-rpath,{ROCM}/lib",
                    "-Wl,--allow-shlib-undefined"], check=True)
    done = subprocess.run([str(tmp_path / "program")], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr
    return done.stdout
