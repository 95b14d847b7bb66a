"""Orders in ``csrc/attention.cu`` on which it depends that no wait runs out and none lasts for good: they are read
here, since what they prevent must not be brought about on a GPU."""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _body(name):
    """The text of the definition of function `name`, comments left out."""
    text = open(os.path.join(ROOT, "rf-detr-jax_b200", "csrc", "attention.cu")).read()
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(rf"\b{name}\(", text):
        brace, end = text.find("{", m.end()), text.find(";", m.end())
        if brace < 0 or 0 <= end < brace:
            continue  # a call or a declaration
        depth = 0
        for i in range(brace, len(text)):
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            if depth == 0:
                return text[brace:i + 1]
    raise AssertionError(f"{name} is not defined")


@pytest.mark.parametrize("name", ["bwd_load", "bwd_mma_loop", "bwd_grads"])
def test_bounded_waits_cover_this_block_only(name):
    """The dK/dV kernel starts while the dQ kernel still runs.  A warp that polls for a step's tiles or products, which
    come only once the other has ended, has to wait for that end first, without a limit of polls."""
    body = _body(name)
    passed = body.find("wait_for_primary()")
    assert passed >= 0
    polls = [m.start() for m in re.finditer(r"wait_warp\(&sh\.(?!x_full)", body)]
    assert polls
    # A lambda's polls count from its first call.
    calls = [m.start() for m in re.finditer(r"!scores\(", body)] or polls
    assert passed < min(calls)


def test_no_dependent_before_tensor_memory():
    """A dQ block lets dK/dV blocks in once it has its tensor memory: they hold theirs until its whole launch ends."""
    body = _body("attn_backward_kernel")
    alloc, lets_in = body.find("tmem_alloc("), body.find("launch_dependents()")
    assert 0 <= alloc < body.find("__syncthreads()", alloc) < lets_in
    assert body.count("launch_dependents()") == 1


def test_no_wait_for_the_cluster_with_tensor_memory():
    """A block that holds tensor memory waits for no block that may still have to get its own."""
    body = _body("attn_backward_kernel")
    joins = [m.start() for m in re.finditer(r"share_acc<|cluster_sync\(", body)]
    assert joins and 0 <= body.find("tmem_dealloc(") < min(joins)
    assert "cluster_sync(" not in _body("stage_acc") and "cluster_sync(" in _body("share_acc")


def test_registers_that_warps_hand_over():
    """Warps that ask for more registers take them from what the launch gave the block's others: with fewer to a thread
    than the shares were reckoned from they would wait for good.  So many the compiler has to use."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    package = os.path.join(ROOT, "rf-detr-jax_b200")
    made = subprocess.run(
        [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
         "--expt-relaxed-constexpr", f"-I{os.path.join(ROOT, 'include')}", f"-I{os.path.join(package, 'csrc')}",
         "-Xptxas", "-v", "-c", os.path.join(package, "csrc", "attention.cu"), "-o", os.devnull],
        capture_output=True, text=True, check=True)
    used = dict(re.findall(r"Compiling entry function '(\w+)'.*?Used (\d+) registers", made.stderr, re.S))
    shares = {"attn_forward_long_kernelILi32E": 168, "attn_forward_long_kernelILi64E": 168,
              "attn_forward_long_kernelILi128E": 168, "attn_backward_kernelILi64E": 80,
              "attn_backward_kernelILi128E": 96}
    for kernel, registers in shares.items():
        counts = {int(n) for name, n in used.items() if kernel in name}
        assert counts == {registers}, kernel
