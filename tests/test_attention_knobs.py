"""What the forward kernel's knob selects, seen from the workspace that keys shared out over blocks need."""

from __future__ import annotations

import pytest


@pytest.mark.parametrize("sizes", [(5, 882, 882, 6, 2), (4, 180, 1046, 4, 1), (2, 135, 1030, 2, 2)])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_keys_are_shared_out_by_single_row_tiles_alone(pkg, tuning, sizes, dim):
    """A second number shares keys out with the alternating kernel (3), whatever the sizes would choose; with the others
    there is nothing to share, and it changes nothing."""
    size = pkg._native.lib().rfdetr_packed_attention_workspace_bytes
    n, tokens, keys, heads, kv = sizes
    for knob in ("1", "1,1", "1,3", "1,64", "2", "2,3", "3", "3,1"):
        tuning("RFDETR_ATTN_FWD", knob)
        assert size(n, tokens, keys, heads, kv, dim) == 0, knob
    needs = []
    for knob in ("3,2", "3,3", "3,64"):
        tuning("RFDETR_ATTN_FWD", knob)
        needs.append(size(n, tokens, keys, heads, kv, dim))
    assert 0 < needs[0] < needs[1] < needs[2]
    # A float32 result and log-sum-exp for each row of each block.
    assert needs[1] * 2 == needs[0] * 3 and needs[0] % (4 * (dim + 1)) == 0
