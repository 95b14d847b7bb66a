"""Integers of 64 bits whose values do not fit 32."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import rotary as OR

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_past_32_bits(pkg, dtype, interleaved):
    """Within 2^-21 (|x1| + |x2|) as for near positions: up to 2^33, times a frequency of at most 2^-7, the
    float64 angle is off by three roundings of 2^-53 2^26, 2^-25.4 radians."""
    rng = np.random.default_rng(0)
    tokens = 65
    pos = rng.integers(-2 ** 33, 2 ** 33, (tokens, 2))
    pos[0] = (2 ** 32 + 5, 5)
    freq = torch.tensor(rng.uniform(1e-3, 2.0 ** -7, 16).astype(np.float32), device=DEV)
    x = torch.tensor(rng.standard_normal((tokens, 3, 40)).astype(np.float32), device=DEV).to(dtype)
    got, key = pkg.axial_rotary(x, x[:, :1], torch.tensor(pos, device=DEV), freq, (8, 8), interleaved=interleaved)
    want = OR.rotary(x.double().cpu().numpy(), pos, freq.cpu().numpy(), (8, 8), interleaved)
    size = np.abs(x.double().cpu().numpy())
    i = np.arange(16)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + 16)
    size[..., first] = size[..., second] = size[..., first] + size[..., second]
    bound = 2.0 ** -21 * size + (2.0 ** -8 * np.abs(want) if dtype == torch.bfloat16 else 0.0)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()
    assert torch.equal(key, got[:, :1])


def test_positions_of_both_widths_agree(pkg):
    rng = np.random.default_rng(1)
    x = torch.randn((300, 2, 64), device=DEV)
    pos = torch.tensor(rng.integers(-1000, 100000, (300, 3)), device=DEV)
    freq = torch.rand(32, device=DEV)
    a, _ = pkg.axial_rotary(x, None, pos, freq, (10, 11, 11))
    b, _ = pkg.axial_rotary(x, None, pos.to(torch.int32), freq, (10, 11, 11))
    c, _ = pkg.axial_rotary(x, None, pos.repeat(1, 2)[:, :3], freq, (10, 11, 11))  # rows apart
    assert torch.equal(a, b) and torch.equal(a, c)


def test_addresses_of_wide_positions(pkg):
    """The library refuses int64 positions that are not aligned to 8 bytes."""
    N = pkg._native
    sections = N.int64_array((2,))
    call = lambda at: N.lib().rfdetr_axial_rotary(None, 16, 8, 4, None, 0, 0, N.F32, at, N.I64, 16, sections, 1, 16,  # noqa: E731
                                                  None, 1, 1, 0, 4, 0, 0)
    assert call(20) == N.ERR_ALIGN and call(18) == N.ERR_ALIGN


def test_offsets_past_32_bits(pkg):
    """They are clamped to the tensors like any others, and `check` sees them as they are."""
    q, k, v = (torch.randn((100, 2, 32), device=DEV).to(torch.bfloat16) for _ in range(3))
    near = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    far = lambda *x: torch.tensor(x, dtype=torch.int64, device=DEV)  # noqa: E731
    want = pkg.packed_attention(q, k, v, near(0, 60, 100))
    assert torch.equal(pkg.packed_attention(q, k, v, far(0, 60, 2 ** 32 + 70)), want)
    assert torch.equal(pkg.packed_attention(q, k, v, far(-2 ** 32 + 7, 60, 2 ** 62)), want)
    assert torch.equal(pkg.packed_attention(q, k, v, far(0, 60, 100), far(0, 60, 2 ** 33), check=False), want)
    assert torch.equal(pkg.packed_attention(q, k, v, far(0, 60, 100), check=True), want)
    for offsets in (far(0, 60, 2 ** 32 + 100), far(2 ** 32, 60, 100), far(-2 ** 32, 60, 100)):
        with pytest.raises(ValueError, match="ascend"):
            pkg.packed_attention(q, k, v, offsets, check=True)
        with pytest.raises(ValueError, match="ascend"):
            pkg.packed_attention(q, k, v, near(0, 60, 100), offsets, check=True)
