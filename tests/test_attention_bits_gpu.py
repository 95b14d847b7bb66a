"""A sequence's bits depend on its own rows alone: not on what shared memory held before, nor on the rows of
a tile that are another sequence's."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
KERNELS = ["1", "2", "3", "3,2"]


def _bf16(rng, *shape):
    return torch.tensor(rng.standard_normal(shape).astype(np.float32), device=DEV).to(torch.bfloat16)


def _offsets(lengths):
    return torch.tensor(np.cumsum([0, *lengths]), dtype=torch.int32, device=DEV)


def _ramp(rng, n, heads, dim):
    """Keys whose scores grow along the sequence by about a power of two a tile, so that rows are near the
    step at which their maximum's reference moves."""
    k = rng.standard_normal((n, heads, dim)) * (1.0 + np.arange(n)[:, None, None] / 128.0)
    return torch.tensor(k.astype(np.float32), device=DEV).to(torch.bfloat16)


@pytest.mark.parametrize("knob", KERNELS)
@pytest.mark.parametrize("group", [3, 5, 6, 7])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_rows_that_no_copy_fills(pkg, tuning, knob, group, dim):
    """A group that does not divide a tile leaves rows of it as the block before left them: large queries."""
    tuning("RFDETR_ATTN_FWD", knob)
    rng = np.random.default_rng(group)
    lengths = (500, 77)
    off = _offsets(lengths)
    q, k, v = _bf16(rng, 577, group, dim), _ramp(rng, 577, 1, dim), _bf16(rng, 577, 1, dim)
    wide = [_bf16(rng, 20000, 4, dim) * s for s in (300.0, 1.0, 1.0)]

    def run():
        return pkg.packed_attention(q, k, v, off, return_lse=True)

    def fill(scale):
        pkg.packed_attention(wide[0] * scale, wide[1][:, :1], wide[2][:, :1], _offsets((200,) * 100))

    fill(0.0)
    want = run()
    for scale in (1.0, -1.0, 0.01, 1e30):
        fill(scale)
        for a, b in zip(run(), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("knob", KERNELS)
@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1), (5, 1)])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_the_next_sequences_queries(pkg, tuning, knob, heads, kv, dim):
    """Rows past a ragged end are the next sequence's queries: large ones, or a single infinite element."""
    tuning("RFDETR_ATTN_FWD", knob)
    rng = np.random.default_rng(dim)
    lengths = (400, 400)
    off = _offsets(lengths)
    q, k, v = _bf16(rng, 800, heads, dim), _ramp(rng, 800, kv, dim), _bf16(rng, 800, kv, dim)
    want = pkg.packed_attention(q, k, v, off, return_lse=True)

    def check(other):
        out, lse = pkg.packed_attention(other, k, v, off, return_lse=True)
        assert torch.equal(out[:400], want[0][:400]) and torch.equal(lse[:, :400], want[1][:, :400])

    for scale in (300.0, -300.0, 0.0):
        other = q.clone()
        other[400:] *= scale
        check(other)
    for value in (float("inf"), -float("inf"), float("nan")):
        other = q.clone()
        other[400::7, :, 3] = value
        check(other)
