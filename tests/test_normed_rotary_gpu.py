"""Norms of queries and keys with rotary positions, on the device against the float64 oracle.

Tolerances, in parts of the sums of absolute values that the oracle gives.  The float32 sum of squares has at most 16
terms to a lane (a lane that reads single values has 8, one of whole pieces up to 16) and 5 steps of shuffles
after them: 21 roundings of 2^-24, halved by the root; the mean's product, eps and the root a few more: the
norm's factor is right to 2^-19.  A turn: three roundings, sine and cosine right to two units of float32 and
an angle to 2^-25 of a turn: 2^-20.  So a result is off by 2^-18 of its sizes at most, the gradient of x, whose inner
sum passes the same roundings again, by 2^-16, that of the weights by 2^-15 (up to 300 sums in a row).  Results in bf16
are off by 2^-8 of themselves more.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.normed_rotary import normed_rotary

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
Y, DX, DW = 2.0 ** -18, 2.0 ** -16, 2.0 ** -15


def _values(rng, dtype, *shape):
    return torch.tensor(rng.standard_normal(shape).astype(np.float32), device=DEV).to(dtype)


def _f64(t):
    return t.detach().double().cpu().numpy()


def _close(name, got, want, size, part):
    bound = part * size + (2.0 ** -8 * np.abs(want) if got.dtype == torch.bfloat16 else 0.0)
    off = np.abs(_f64(got) - want)
    assert got.shape == want.shape
    assert (off <= bound).all(), f"{name}: {off.max()} at {np.argwhere(~(off <= bound))[0]}"


def _inputs(rng, tokens, heads, kv, dim, sections, dtype, pos_dtype=torch.int32, extent=50, weight=torch.float32):
    q, k = _values(rng, dtype, tokens, heads, dim), _values(rng, dtype, tokens, kv, dim)
    if pos_dtype == torch.float32:
        pos = torch.tensor(rng.uniform(-extent, extent, (tokens, len(sections))).astype(np.float32), device=DEV)
    else:
        pos = torch.tensor(rng.integers(-extent, extent, (tokens, len(sections))), device=DEV).to(pos_dtype)
    freq = torch.tensor(rng.uniform(1e-3, 1.0, sum(sections)).astype(np.float32), device=DEV)
    ws = [None if weight is None else (1.0 + 0.3 * _values(rng, torch.float32, dim)).to(weight) for _ in range(2)]
    return q, k, pos, freq, ws


def _check_all(pkg, q, k, pos, freq, sections, ws, gq, gk, eps=1e-6, interleaved=False):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (q, k, *ws)]
    plain = pkg.normed_axial_rotary(q, k, pos, freq, sections, *ws, eps=eps, interleaved=interleaved)
    outs = pkg.normed_axial_rotary(leaves[0], leaves[1], pos, freq, sections, *leaves[2:], eps=eps,
                                   interleaved=interleaved)
    got = torch.autograd.grad([o for o in outs if o is not None], [t for t in leaves if t is not None],
                              [gq] + ([gk] if k is not None else []))
    got = iter(got)
    grads = [None if t is None else next(got) for t in leaves]
    for i, (x, g) in enumerate(((q, gq), (k, gk))):
        if x is None:
            continue
        assert torch.equal(plain[i], outs[i])
        w = ws[i]
        y, ys, dx, dxs, dw, dws = normed_rotary(_f64(x), None if w is None else _f64(w), eps, pos.cpu().numpy(),
                                                freq.cpu().numpy(), sections, interleaved, _f64(g))
        _close("y", outs[i], y, ys, Y)
        _close("dx", grads[i], dx, dxs, DX)
        if w is not None:
            assert grads[2 + i].dtype == w.dtype
            _close("dw", grads[2 + i], dw, dws, DW)


def _check(pkg, tokens, heads, kv, dim, sections, interleaved, dtype, seed=0, **more):
    rng = np.random.default_rng(seed)
    q, k, pos, freq, ws = _inputs(rng, tokens, heads, kv, dim, sections, dtype, **more)
    gq, gk = _values(rng, dtype, tokens, heads, dim), _values(rng, dtype, tokens, kv, dim)
    _check_all(pkg, q, k, pos, freq, sections, ws, gq, gk, interleaved=interleaved)


# Whole and single pieces, both partners in a lane or not, parts of the channels, more tokens than one chunk.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(("tokens", "heads", "kv", "dim", "sections"), [
    (1, 1, 1, 2, (1,)), (7, 3, 1, 10, (2, 3)), (33, 4, 2, 32, (8, 8)), (577, 6, 6, 64, (16, 16)),
    (1301, 16, 4, 128, (16, 24, 24)), (65, 7, 1, 80, (8, 8, 8)), (19, 2, 2, 72, (18, 18)), (40, 2, 1, 48, (0, 5, 0, 3)),
    (90, 5, 2, 80, (11, 12)), (9, 1, 1, 256, (128,)), (31, 3, 2, 256, (37, 20)), (5, 3, 3, 12, (1, 1, 1, 1, 1, 1)),
    (700, 2, 1, 33, (7, 4)), (300, 1, 1, 8, (4,)), (25, 40, 40, 16, (3, 2))])
def test_against_oracle(pkg, tokens, heads, kv, dim, sections, interleaved, dtype):
    _check(pkg, tokens, heads, kv, dim, sections, interleaved, dtype, seed=tokens + dim)


@pytest.mark.parametrize("extent", [1000, 40_000_000])
@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64, torch.float32])
def test_positions(pkg, pos_dtype, extent):
    """Far positions too, beyond what float32 counts: the angle's error does not grow with them."""
    _check(pkg, 90, 2, 2, 64, (16, 16), False, torch.float32, pos_dtype=pos_dtype, extent=extent)


@pytest.mark.parametrize("weight", [None, torch.bfloat16])
def test_weights(pkg, weight):
    _check(pkg, 130, 4, 2, 64, (16, 16), False, torch.bfloat16, weight=weight)


def test_no_key_and_one_weight(pkg):
    rng = np.random.default_rng(2)
    q, _, pos, freq, ws = _inputs(rng, 60, 3, 1, 64, (20, 12), torch.float32)
    _check_all(pkg, q, None, pos, freq, (20, 12), [ws[0], None], torch.randn_like(q), None)
    out, none = pkg.normed_axial_rotary(q, None, pos, freq, (20, 12))
    assert none is None and out.shape == q.shape


def test_views_broadcasts_and_odd_addresses(pkg):
    """Views of a fused projection, strides and addresses off 16 bytes, cotangents of stride 0."""
    rng = np.random.default_rng(1)
    sections = (8, 8)
    pos = torch.tensor(rng.integers(0, 9, (50, 2)), dtype=torch.int32, device=DEV)
    freq = torch.linspace(0.1, 1, 16, device=DEV)
    for dtype in (torch.float32, torch.bfloat16):
        fused = _values(rng, dtype, 50, 9, 64)
        q, k, _ = fused.split((4, 2, 3), 1)
        ws = [1.0 + 0.1 * _values(rng, torch.float32, 64) for _ in range(2)]
        want = pkg.normed_axial_rotary(q.contiguous(), k.contiguous(), pos, freq, sections, *ws)
        for a, b in zip(pkg.normed_axial_rotary(q, k, pos, freq, sections, *ws), want):
            assert torch.equal(a, b)
        turned = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k)]
        for a, b in zip(pkg.normed_axial_rotary(*turned, pos, freq, sections, *ws), want):
            assert torch.equal(a, b)
        odd = torch.empty(50, 4, 65, device=DEV, dtype=dtype)[..., 1:]
        odd.copy_(q)
        one = torch.ones((), device=DEV, dtype=dtype)
        _check_all(pkg, odd, k, pos, freq, sections, ws, one.expand(50, 4, 64), one.expand(50, 2, 64))
        _check_all(pkg, q, k, pos, freq, sections, ws, _values(rng, dtype, 50, 7, 64)[:, 1:5],
                   _values(rng, dtype, 50, 2, 70)[..., 3:67])


def test_rows_of_zeros_and_eps(pkg):
    rng = np.random.default_rng(4)
    q, k, pos, freq, ws = _inputs(rng, 20, 2, 1, 64, (16, 16), torch.float32)
    q[3], k[5] = 0.0, 0.0
    for eps in (1e-6, 0.25):
        _check_all(pkg, q, k, pos, freq, (16, 16), ws, torch.randn_like(q), torch.randn_like(k), eps=eps)
    with_nan = q.clone()
    with_nan[7, 1, 3] = float("nan")
    a, b = (pkg.normed_axial_rotary(x, k, pos, freq, (16, 16), *ws)[0] for x in (q, with_nan))
    rest = torch.ones(20, 2, dtype=torch.bool, device=DEV)
    rest[7, 1] = False
    assert torch.equal(a[rest], b[rest]) and b[7, 1].isnan().all()


def test_gradient_against_differences(pkg):
    """Along one direction of all inputs: (f(x + h d) - f(x - h d)) / 2h = grad . d up to the third derivative (h^2) and
    float32 roundings of f (2^-18 of its sum's size, over h)."""
    rng = np.random.default_rng(6)
    q, k, pos, freq, ws = _inputs(rng, 40, 3, 2, 32, (7, 6), torch.float32)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, *ws)]
    ways = [torch.randn_like(t) for t in leaves]

    def value(by):
        y = pkg.normed_axial_rotary(leaves[0] + by * ways[0], leaves[1] + by * ways[1], pos, freq, (7, 6),
                                    leaves[2] + by * ways[2], leaves[3] + by * ways[3])
        return (y[0].double() * gq).sum() + (y[1].double() * gk).sum(), sum(float(x.detach().abs().sum()) for x in y)

    f, size = value(0.0)
    grads = torch.autograd.grad(f, leaves)
    along = sum(float((g.double() * w).sum()) for g, w in zip(grads, ways))
    h = 2.0 ** -7
    with torch.no_grad():
        got = float(value(h)[0] - value(-h)[0]) / (2 * h)
    # |third derivative| of a normed row along d: a few of its size, |d|^3 / rms^3 about 1 to 10.
    assert abs(got - along) <= 10 * h * h * size + 2.0 ** -18 * size / h


def test_nothing_to_do(pkg):
    freq, pos = torch.ones(4, device=DEV), torch.zeros(0, 1, device=DEV)
    q = torch.zeros(0, 2, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    out, _ = pkg.normed_axial_rotary(q, None, pos, freq, (4,), w)
    dq, dw = torch.autograd.grad(out.sum(), (q, w))
    assert out.shape == q.shape and dq.shape == q.shape and not dw.any()


def test_captured_and_side_by_side(pkg):
    """Bits of a replayed graph, beside another stream's calls, are those of calls in turn."""
    rng = np.random.default_rng(8)
    q, k, pos, freq, ws = _inputs(rng, 400, 4, 2, 64, (16, 16), torch.bfloat16)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, *ws)]
    gq, gk = torch.randn_like(q), torch.randn_like(k)

    def step():
        outs = pkg.normed_axial_rotary(leaves[0], leaves[1], pos, freq, (16, 16), *leaves[2:])
        return [*outs, *torch.autograd.grad(outs, leaves, (gq, gk))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    with torch.cuda.stream(side):
        beside = step()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, beside):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals(pkg):
    q = torch.zeros(4, 2, 64, device=DEV)
    pos, freq, w = torch.zeros(4, 1, device=DEV), torch.ones(8, device=DEV), torch.ones(64, device=DEV)
    f = pkg.normed_axial_rotary
    for bad in (lambda: f(q.half(), None, pos, freq, (8,)), lambda: f(q, q[:3], pos, freq, (8,)),
                lambda: f(q, q.bfloat16(), pos, freq, (8,)), lambda: f(q, None, pos, freq, (9,)),
                lambda: f(q, None, pos[:3], freq, (8,)), lambda: f(q, None, pos, freq, (40,)),
                lambda: f(q, None, pos.double(), freq, (8,)), lambda: f(q, None, pos, freq, (8,), w[:8]),
                lambda: f(q, None, pos, freq, (8,), w.half()), lambda: f(q, None, pos, freq, (8,), w, w),
                lambda: f(q, q, pos, freq, (8,), eps=-1.0), lambda: f(q, q, pos, freq, (8,), eps=float("nan")),
                lambda: f(q.expand(4, 2, 64)[0], None, pos, freq, (8,)),
                lambda: f(torch.zeros(4, 1, 264, device=DEV), None, pos, freq, (8,)),
                lambda: f(q.cpu(), None, pos, freq, (8,)),
                lambda: f(q, q, pos.requires_grad_(True), freq, (8,))):
        with pytest.raises(ValueError):
            bad()
    with torch.no_grad():
        f(q, q, pos, freq, (8,))


# Float32 rows with two pieces to a lane, where one piece each would be more than a warp's lanes, and the widest with one.
@pytest.mark.parametrize("dim", [136, 160, 192, 256])
@pytest.mark.parametrize("turned", [8, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_heads_turned_in_part(pkg, dim, turned, dtype):
    sections = (turned // 2 - turned // 4, turned // 4)
    for tokens, heads, kv in ((1, 1, 1), (41, 3, 2), (1500, 2, 1)):
        _check(pkg, tokens, heads, kv, dim, sections, False, dtype, seed=dim + turned + tokens)
