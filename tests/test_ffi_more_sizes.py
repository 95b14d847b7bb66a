"""The XLA handlers of the changed scores, the normed rotary positions and the clipping, compiled against a stand-in for
XLA's header (``tests/ffi``) and called on the CPU: a buffer whose size or type does not fit the others is refused before
the library is called."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HERE = os.path.join(ROOT, "tests", "ffi")
PACKAGE = os.path.join(ROOT, "rf-detr-jax_b200")


@pytest.fixture(scope="module")
def lines(pkg, tmp_path_factory):
    compiler = shutil.which("g++")
    cuda = next((d for d in (os.environ.get("CUDA_HOME", ""), "/usr/local/cuda")
                 if os.path.exists(os.path.join(d, "include", "cuda_runtime.h"))), None)
    if compiler is None or cuda is None:
        pytest.skip("needs g++ and the CUDA headers")
    pkg._native.lib()
    program = str(tmp_path_factory.mktemp("ffi") / "sizes")
    lib = os.path.join(cuda, "lib64")
    made = subprocess.run(
        [compiler, "-std=c++17", "-o", program, os.path.join(HERE, "more_sizes.cc"), f"-I{HERE}",
         f"-I{os.path.join(ROOT, 'include')}", f"-I{os.path.join(cuda, 'include')}", f"-L{PACKAGE}",
         "-l:librfdetr_b200.so", f"-L{lib}", "-lcudart", f"-Wl,-rpath,{PACKAGE}:{lib}"],
        capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    out = subprocess.run([program], capture_output=True, text=True, check=True).stdout
    return [line.split("|") for line in out.splitlines()]


def test_sizes_that_fit_reach_the_library(lines):
    fit = [x for x in lines if x[1] == "fit"]
    assert len(fit) == 7 and all(x[2:] == ["ok", "1"] for x in fit), fit


def test_sizes_that_do_not_fit_are_refused(lines):
    others = [x for x in lines if x[1] != "fit"]
    assert len(others) > 80
    assert [x for x in others if x[2:] != ["refused", "0"]] == []
