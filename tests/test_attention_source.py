"""Orders in ``csrc/attention.cu`` on which it depends that no wait runs out and none lasts for good: they are read
here, since what they prevent must not be brought about on a GPU."""

from __future__ import annotations

import os
import re

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
