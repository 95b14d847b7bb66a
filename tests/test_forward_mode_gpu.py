"""Forward-mode derivatives: no operator here has them, and none may drop a tangent in silence."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [False, True])
def test_packed_attention_refuses_tangents(pkg, which, grad):
    off = torch.tensor([0, 5, 9], dtype=torch.int32, device=DEV)
    x = [torch.randn((9, 2, 64), device=DEV).to(torch.bfloat16) for _ in range(3)]
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        x[which] = fwAD.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(NotImplementedError):
            pkg.packed_attention(*x, off)
    # Without a tangent a level changes nothing.
    x = [fwAD.unpack_dual(t).primal for t in x]
    want = pkg.packed_attention(*x, off)
    with fwAD.dual_level():
        assert torch.equal(pkg.packed_attention(*x, off), want)


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_axial_rotary_refuses_tangents(pkg, which):
    x = [torch.randn((9, 2, 8), device=DEV), torch.randn((9, 1, 8), device=DEV), torch.rand((9, 1), device=DEV),
         torch.rand(4, device=DEV)]
    with fwAD.dual_level():
        x[which] = fwAD.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(NotImplementedError):
            pkg.axial_rotary(*x, (4,))
