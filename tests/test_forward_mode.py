"""Whether a tensor carries a forward-mode derivative, with and without torch's own note of an open level."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD


@pytest.mark.parametrize("noted", [True, False])
def test_tangents_are_seen(pkg, monkeypatch, noted):
    N = pkg._native
    x, y = torch.randn(3), torch.randn(3, requires_grad=True)
    if not noted:
        public = fwAD.unpack_dual
        monkeypatch.setattr(N, "forward_ad", type("forward_ad", (), {"unpack_dual": staticmethod(public)}))
    assert not N.has_tangent(x, None, y)
    with fwAD.dual_level():
        assert not N.has_tangent(x, None, y)
        for t in (x, y):
            dual = fwAD.make_dual(t, torch.ones(3))
            assert N.has_tangent(dual) and N.has_tangent(x, None, dual) and N.has_tangent(dual * 2)
    assert not N.has_tangent(x, y)
