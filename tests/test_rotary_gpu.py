"""Rotary positions on the device against the float64 oracle.

Tolerances: the cosine and sine are right to 2 units in the last place of float32 and the two
products and their sum round three times, so a float32 result is off by at most 2^-21 (|x1| + |x2|);
a bf16 one by 2^-8 of itself more.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import rotary as OR

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _values(rng, dtype, *shape):
    return torch.tensor(rng.standard_normal(shape).astype(np.float32), device=DEV).to(dtype)


def _f64(t):
    return t.detach().double().cpu().numpy()


def _close(got, x, want, sections, interleaved, dtype):
    half = sum(sections)
    x = np.abs(_f64(x))
    size = x.copy()
    i = np.arange(half)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    size[..., first] = size[..., second] = x[..., first] + x[..., second]
    bound = 2.0 ** -21 * size + (2.0 ** -8 * np.abs(want) if dtype == torch.bfloat16 else 0.0)
    assert (np.abs(_f64(got) - want) <= bound).all()
    assert np.array_equal(_f64(got)[..., 2 * half:], want[..., 2 * half:])  # copied


def _check(pkg, tokens, heads, kv, dim, sections, interleaved, dtype, pos_dtype=torch.int32, extent=50, seed=0):
    rng = np.random.default_rng(seed)
    q, k = _values(rng, dtype, tokens, heads, dim), _values(rng, dtype, tokens, kv, dim)
    if pos_dtype == torch.float32:
        pos = torch.tensor(rng.uniform(-extent, extent, (tokens, len(sections))).astype(np.float32), device=DEV)
    else:
        pos = torch.tensor(rng.integers(0, extent, (tokens, len(sections))), device=DEV).to(pos_dtype)
    freq = torch.tensor(rng.uniform(1e-3, 1.0, sum(sections)).astype(np.float32), device=DEV)
    gq, gk = _values(rng, dtype, tokens, heads, dim), _values(rng, dtype, tokens, kv, dim)
    how = (pos.cpu().numpy(), freq.cpu().numpy(), sections, interleaved)
    q.requires_grad_(True)
    k.requires_grad_(True)
    yq, yk = pkg.axial_rotary(q, k, pos, freq, sections, interleaved=interleaved)
    assert yq.dtype == dtype and yk.dtype == dtype
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    for got, x, inverse in ((yq, q, False), (yk, k, False), (dq, gq, True), (dk, gk, True)):
        _close(got, x, OR.rotary(_f64(x), *how, inverse), sections, interleaved, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(("tokens", "heads", "kv", "dim", "sections"), [
    (1, 1, 1, 2, (1,)), (7, 3, 1, 10, (2, 3)), (33, 4, 2, 32, (8, 8)), (577, 6, 6, 64, (16, 16)),
    (130, 16, 4, 128, (16, 24, 24)), (65, 7, 1, 80, (8, 8, 8)), (19, 2, 2, 72, (18, 18)), (40, 2, 1, 48, (0, 5, 0, 3)),
    (9, 1, 1, 1024, (512,)), (5, 3, 3, 12, (1, 1, 1, 1, 1, 1))])
def test_against_oracle(pkg, tokens, heads, kv, dim, sections, interleaved, dtype):
    _check(pkg, tokens, heads, kv, dim, sections, interleaved, dtype, seed=tokens + dim)


@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64, torch.float32])
def test_positions(pkg, pos_dtype):
    """Far positions too: the angle's error does not grow with them."""
    _check(pkg, 90, 2, 2, 64, (16, 16), False, torch.float32, pos_dtype, extent=1_000_000)


def test_views_and_odd_addresses(pkg):
    rng = np.random.default_rng(1)
    sections, freq = (4, 4), torch.linspace(0.1, 1, 8, device=DEV)
    pos = torch.tensor(rng.integers(0, 9, (30, 2)), dtype=torch.int32, device=DEV)
    for dtype in (torch.float32, torch.bfloat16):
        fused = _values(rng, dtype, 30, 6, 24)
        q, k = fused.split((4, 2), 1)
        for interleaved in (False, True):
            want = pkg.axial_rotary(q.contiguous(), k.contiguous(), pos, freq, sections, interleaved=interleaved)
            for a, b in zip(pkg.axial_rotary(q, k, pos, freq, sections, interleaved=interleaved), want):
                assert torch.equal(a, b) and a.is_contiguous()
            odd = torch.empty(30, 4, 25, device=DEV, dtype=dtype)[..., 1:]  # no vector fits
            odd.copy_(q)
            turned = k.transpose(0, 1).contiguous().transpose(0, 1)
            strided = torch.empty(30, 4, 48, device=DEV, dtype=dtype)[..., ::2]  # channels not contiguous
            strided.copy_(q)
            wide = pos.repeat(1, 2)[:, :2]
            for x in (odd, strided):
                for a, b in zip(pkg.axial_rotary(x, turned, wide, freq, sections, interleaved=interleaved), want):
                    assert torch.equal(a, b)
            alone, none = pkg.axial_rotary(q, None, pos, freq, sections, interleaved=interleaved)
            assert none is None and torch.equal(alone, want[0])
            same = q[:, :1].expand(30, 4, 24)  # one head broadcast
            got, _ = pkg.axial_rotary(same, None, pos, freq, sections, interleaved=interleaved)
            ref, _ = pkg.axial_rotary(same.contiguous(), None, pos, freq, sections, interleaved=interleaved)
            assert torch.equal(got, ref)


def test_turns_add_up_and_keep_relative_places(pkg):
    """q at m against k at n depends on m - n alone."""
    rng = np.random.default_rng(2)
    q, k = _values(rng, torch.float32, 1, 1, 64), _values(rng, torch.float32, 1, 1, 64)
    freq = torch.tensor(1.0 / 50.0 ** (np.arange(32) / 32), dtype=torch.float32, device=DEV)
    dots = []
    for shift in (0, 5, 1000):
        p = lambda n: torch.tensor([[n + shift, 2 * shift]], dtype=torch.int32, device=DEV)  # noqa: E731
        yq, _ = pkg.axial_rotary(q, None, p(7), freq, (16, 16))
        yk, _ = pkg.axial_rotary(k, None, p(3), freq, (16, 16))
        dots.append(float((yq.double() * yk.double()).sum()))
    # 64 products of values up to about 3, each turned twice with 2^-21 of error.
    assert max(dots) - min(dots) < 64 * 2 * 10 * 2.0 ** -21


def test_non_finite_values_stay_in_their_pair(pkg):
    x = torch.ones((1, 1, 8), device=DEV)
    x[0, 0, 1] = float("inf")
    y, _ = pkg.axial_rotary(x, None, torch.ones((1, 1), device=DEV), torch.ones(3, device=DEV), (3,))
    assert torch.isfinite(y[0, 0, [0, 2, 3, 5, 6, 7]]).all() and not torch.isfinite(y[0, 0, [1, 4]]).any()


def test_empty_and_another_stream(pkg):
    pos, freq = torch.empty((0, 1), device=DEV), torch.ones(2, device=DEV)
    q, k = pkg.axial_rotary(torch.empty((0, 3, 4), device=DEV), torch.empty((0, 1, 4), device=DEV), pos, freq, (2,))
    assert q.shape == (0, 3, 4) and k.shape == (0, 1, 4)
    x = torch.randn((1000, 4, 64), device=DEV)
    p = torch.rand((1000, 1), device=DEV)
    f = torch.rand(32, device=DEV)
    want, _ = pkg.axial_rotary(x, None, p, f, (32,))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = pkg.axial_rotary(x, None, p, f, (32,))
    side.synchronize()
    assert torch.equal(got, want)


def test_gradient_of_one_of_the_two(pkg):
    x = torch.randn((10, 2, 16), device=DEV)
    q, k = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    pos, freq = torch.rand((10, 1), device=DEV), torch.rand(8, device=DEV)
    yq, yk = pkg.axial_rotary(q, k, pos, freq, (8,))
    (dk,) = torch.autograd.grad(yk, (k,), torch.ones_like(yk))
    want, _ = pkg.axial_rotary(torch.ones_like(x), None, -pos, freq, (8,))
    # The same angle negated: cos and sin are even and odd, so equal up to the sign of rounding.
    assert (dk - want).abs().max() <= 2.0 ** -20


def test_refusals(pkg):
    t = lambda *s, dtype=torch.float32: torch.zeros(s, device=DEV, dtype=dtype)  # noqa: E731
    q, k, p, f = t(4, 2, 8), t(4, 1, 8), t(4, 2), t(4)
    for args in [(t(4, 8), k, p, f, (2, 2)), (q, t(3, 1, 8), p, f, (2, 2)), (q, t(4, 1, 6), p, f, (2, 2)),
                 (q, k.bfloat16(), p, f, (2, 2)), (q.half(), None, p, f, (2, 2)), (q, k, t(4, 3), f, (2, 2)),
                 (q, k, p.double(), f, (2, 2)), (q, k, p, t(3), (2, 2)), (q, k, p, f.double(), (2, 2)),
                 (q, k, p, t(5), (2, 3)), (q, k, p, f, (5, -1)), (q, k, t(4, 9), f, (4,) + (0,) * 8),
                 (q.cpu(), k, p, f, (2, 2)), (q, k, p.requires_grad_(True), f, (2, 2))]:
        with pytest.raises(ValueError):
            pkg.axial_rotary(*args)
    with pytest.raises(ValueError):
        pkg.axial_rotary(t(4, 2, 7), None, t(4, 1), t(3), (3,), interleaved=True)
