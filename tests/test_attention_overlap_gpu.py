"""The backward kernels where the second starts long before the first has ended."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import attention as OA

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_few_queries_over_very_many_keys(pkg, dim):
    """One tile of queries walks all keys, for milliseconds, while the blocks of most keys already wait for it."""
    rng = np.random.default_rng(dim)
    n, m = 24, 300_000
    f64 = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
    q, k, v, g = (torch.tensor(rng.standard_normal((x, 1, dim)).astype(np.float32), device=DEV).to(torch.bfloat16)
                  for x in (n, m, m, n))
    off = lambda x: torch.tensor([0, x], dtype=torch.int32, device=DEV)  # noqa: E731
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = pkg.packed_attention(*leaves, off(n), off(m))
    r = OA.attention(f64(q), f64(k), f64(v), [0, n], [0, m], grad=f64(g))
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, g))):
        # (What the sums' float32 adds to the bound, 2^-24 of them a step, is far below bf16's.)
        assert (np.abs(f64(got) - r[name]) <= r[name + "_bound"] + 1e-30).all(), name
    assert pkg._native.lib().rfdetr_take_device_fault(torch.cuda.current_stream().cuda_stream) == 0
