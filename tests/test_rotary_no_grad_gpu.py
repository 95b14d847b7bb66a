"""Positions and frequencies that are parameters: no gradient reaches them, which matters only where one is wanted."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_parameters_at_inference(pkg):
    x = torch.randn((9, 2, 16), device=DEV)
    pos, freq = torch.rand((9, 2), device=DEV), torch.rand(8, device=DEV)
    want, _ = pkg.axial_rotary(x, None, pos, freq, (4, 4))
    learned, moved = torch.nn.Parameter(freq), pos.clone().requires_grad_(True)
    with torch.no_grad():
        got, _ = pkg.axial_rotary(x, None, moved, learned, (4, 4))
    assert torch.equal(got, want)
    for p, f in ((pos, learned), (moved, freq)):
        with pytest.raises(ValueError, match="no gradient"):
            pkg.axial_rotary(x, None, p, f, (4, 4))
