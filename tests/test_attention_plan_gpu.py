"""Which forward kernel the sizes choose, seen from its bits: each adds in another order."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _bf16(rng, *shape):
    return torch.tensor(rng.standard_normal(shape).astype(np.float32), device=DEV).to(torch.bfloat16)


def _offsets(lengths):
    return torch.tensor(np.cumsum([0, *lengths]), dtype=torch.int32, device=DEV)


def _chosen(pkg, tuning, lengths, keys, heads, dim, causal):
    """"halves" or "pairs"."""
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the plan depends on the SM count")
    rng = np.random.default_rng(0)
    own = keys is None
    q = _bf16(rng, sum(lengths), heads, dim)
    k, v = (_bf16(rng, sum(lengths if own else keys), heads, dim) for _ in range(2))

    def call(knob):
        tuning("RFDETR_ATTN_FWD", knob)
        return pkg.packed_attention(q, k, v, _offsets(lengths), None if own else _offsets(keys), causal=causal)

    got, pairs, halves = call(None), call("1"), call("3")
    assert not torch.equal(pairs, halves)
    assert torch.equal(got, pairs) or torch.equal(got, halves)
    return "pairs" if torch.equal(got, pairs) else "halves"


@pytest.mark.parametrize("lengths,keys,want", [((3000,), (2000,), "pairs"), ((3000,), (1000,), "pairs"),
                                               ((300,) * 8, (576, 2304, 0, 1600, 33, 1, 900, 4000), "halves")])
def test_other_tokens(pkg, tuning, lengths, keys, want):
    """192 row tiles.  The keys of a single sequence are of one count, whatever their number is next to the queries':
    no row tile's work is longer than another's."""
    assert _chosen(pkg, tuning, lengths, keys, 8, 80, False) == want


@pytest.mark.parametrize("lengths,heads,want", [((1024,) * 4, 8, "pairs"), ((900,) * 6, 6, "pairs"),
                                                ((1024,) * 4, 6, "halves"), ((1300,) * 2, 12, "halves"),
                                                ((2048,) * 2, 8, "halves")])
def test_causal(pkg, tuning, lengths, heads, want):
    """More row tiles than SMs: halves pay up to one and a half an SM, and with ten key tiles up to two."""
    assert _chosen(pkg, tuning, lengths, None, heads, 64, True) == want
