"""Gradient clipping on the device against float64.

Tolerances: squares and sums are float64, so the norm is right to its rounding to float32, 2^-24; a clipped value has the factor's
rounding and its own, 2^-23 relative, and in bf16 2^-8 more.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.float32, torch.bfloat16)]


def _tensors(rng, counts, dtype):
    return [torch.tensor(rng.standard_normal(n).astype(np.float32) * 10.0 ** rng.uniform(-4, 1), device=DEV).to(dtype)
            for n in counts]


def _norm(tensors):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in tensors))


def _check(norm, outs, before, max_norm):
    want = _norm(before)
    assert norm.dtype == torch.float32 and norm.shape == ()
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    factor = 1.0 if want <= max_norm else max_norm / want
    for y, x in zip(outs, before):
        exact = x.double() * factor
        bound = exact.abs() * (2.0 ** -23 + (2.0 ** -8 if y.dtype == torch.bfloat16 else 0.0)) + 2.0 ** -126
        assert ((y.double() - exact).abs() <= bound).all()


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize(("dtype", "out"), TYPES)
@pytest.mark.parametrize("counts", [(1,), (7, 0, 1, 3), (1023, 1024, 1025, 4097), (300_007, 5, 70_001), (33,) * 40,
                                    tuple(range(1, 500)), (2,) * 2600, (9_000_001,)])
def test_into_other_tensors(pkg, counts, dtype, out, kept):
    rng = np.random.default_rng(len(counts) + counts[0])
    gradients = _tensors(rng, counts, dtype)
    for share in (0.3, 2.0):
        outs = [torch.full((n,), 7.0, device=DEV, dtype=out) for n in counts]
        limit = share * _norm(gradients)
        if kept:
            norm = pkg.GradientClipper(gradients, outs).clip(limit)
        else:
            norm = pkg.clip_gradients(gradients, limit, out=outs)
        _check(norm, outs, gradients, limit)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_in_place(pkg, dtype):
    rng = np.random.default_rng(3)
    gradients = _tensors(rng, (50, 1, 20_000, 333), dtype)
    gradients[2] = gradients[2].view(100, 200).t()  # dense, in another order
    before = [t.clone() for t in gradients]
    limit = 2.0 * _norm(before)
    norm = pkg.clip_gradients(gradients, limit)
    _check(norm, gradients, before, limit)
    assert all(torch.equal(a, b) for a, b in zip(gradients, before))
    versions = [t._version for t in gradients]
    norm = pkg.clip_gradients(gradients, limit / 8)
    _check(norm, gradients, before, limit / 8)
    assert all(t._version > v for t, v in zip(gradients, versions))
    assert pkg.clip_gradients(gradients[0], 1.0).shape == ()


@pytest.mark.parametrize(("dtype", "out"), TYPES)
def test_views_at_odd_places(pkg, dtype, out):
    """Every misalignment of input against output."""
    rng = np.random.default_rng(5)
    for a, b in ((0, 0), (1, 1), (3, 0), (0, 5), (2, 7), (8, 4)):
        flat = _tensors(rng, (9000,), dtype)[0]
        room = torch.full((9000,), 7.0, device=DEV, dtype=out)
        counts = (1, 2, 301, 4000, 17, 3)
        starts = np.cumsum((0,) + counts[:-1])
        gradients = [flat[a + s:a + s + n] for s, n in zip(starts, counts)]
        outs = [room[b + s:b + s + n] for s, n in zip(starts, counts)]
        limit = 0.5 * _norm(gradients)
        norm = pkg.clip_gradients(gradients, limit, out=outs)
        _check(norm, outs, gradients, limit)
        assert (room[:b] == 7).all() and (room[b + sum(counts):] == 7).all()


def test_limits(pkg):
    gradients = _tensors(np.random.default_rng(6), (100, 3000), torch.float32)
    before = [t.clone() for t in gradients]
    assert abs(float(pkg.clip_gradients(gradients, math.inf)) - _norm(before)) <= 2.0 ** -23 * _norm(before)
    assert all(torch.equal(a, b) for a, b in zip(gradients, before))
    pkg.clip_gradients(gradients, 0.0)
    assert not any(t.any() for t in gradients)
    assert float(pkg.clip_gradients(gradients, 0.0)) == 0.0  # a norm of 0 is within any limit
    assert float(pkg.clip_gradients([torch.zeros(0, device=DEV)], 1.0)) == 0.0


def test_sizes_past_float32_squares(pkg):
    """Squares that float32 cannot hold, large and small."""
    for size in (1e30, 1e-30):
        x = torch.full((5000,), size, device=DEV)
        out = torch.empty_like(x)
        norm = pkg.clip_gradients(x, size, out=out)
        _check(norm, [out], [x], size)


def test_values_that_are_no_numbers(pkg):
    for value in (float("nan"), float("inf")):
        gradients = [torch.ones(1000, device=DEV), torch.ones(70, device=DEV)]
        gradients[1][3] = value
        norm = pkg.clip_gradients(gradients, 1.0)
        if math.isnan(value):
            assert norm.isnan() and all(t.isnan().all() for t in gradients)
        else:
            assert norm.isinf() and gradients[1][3].isnan()
            gradients[1][3] = 0
            assert not any(t.any() for t in gradients)


def test_equal_calls_and_captured_ones_give_equal_bits(pkg):
    gradients = _tensors(np.random.default_rng(7), (100_000, 7, 3_000_001, 64), torch.float32)
    outs = [torch.empty_like(t) for t in gradients]
    clipper = pkg.GradientClipper(gradients, outs)
    limit = 0.25 * _norm(gradients)
    norm = clipper.clip(limit)
    want = [t.clone() for t in outs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pkg.clip_gradients(gradients, limit, out=[torch.empty_like(t) for t in gradients])
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, replayed side by side
        other = [torch.empty_like(t) for t in gradients]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = pkg.clip_gradients(gradients, limit, out=other)
        graphs.append((graph, got, other))
    side.wait_stream(torch.cuda.current_stream())
    graphs[0][0].replay()
    with torch.cuda.stream(side):
        graphs[1][0].replay()
    torch.cuda.synchronize()
    for _, got, other in graphs:
        assert torch.equal(got, norm) and all(torch.equal(a, b) for a, b in zip(other, want))


def test_kept_tensors_are_read_anew(pkg):
    """A clipper works on what its tensors hold at the call."""
    x = torch.ones(2000, device=DEV)
    clipper = pkg.GradientClipper([x[:1500], x[1500:]])
    for scale in (1.0, 3.0):
        x.fill_(scale)
        norm = clipper.clip(1.0)
        assert abs(float(norm) - scale * math.sqrt(2000)) <= 2.0 ** -22 * scale * 45
        assert abs(float(x.norm()) - 1.0) <= 1e-5


def test_refusals(pkg):
    x = torch.ones(10, device=DEV)
    f = pkg.clip_gradients
    for bad in (lambda: f([], 1.0), lambda: f(x, -1.0), lambda: f(x, float("nan")), lambda: f(x.half(), 1.0),
                lambda: f([x, x], 1.0), lambda: f(x.clone().requires_grad_(True), 1.0), lambda: f(x.cpu(), 1.0),
                lambda: f([x, x.cpu()], 1.0), lambda: f(torch.ones((), device=DEV).expand(4), 1.0),
                lambda: f(torch.ones(4, 4, device=DEV)[:, :2], 1.0), lambda: f(x, 1.0, out=x[:9]),
                lambda: f(x, 1.0, out=[x, x]), lambda: f(x, 1.0, out=torch.ones(20, device=DEV)[::2]),
                lambda: f(x, 1.0, out=torch.ones(10, device=DEV, dtype=torch.float16)),
                lambda: pkg.GradientClipper(torch.ones(20, device=DEV)[::2], x)):
        with pytest.raises(ValueError):
            bad()
    y = torch.empty(10, device=DEV)
    f(torch.ones(20, device=DEV)[::2], math.inf, out=y)  # strided gradients are read where there is somewhere to put them
    assert (y == 1).all()


def test_results_that_share_memory_are_refused(pkg):
    x = torch.ones(100, device=DEV)
    a, b = x[:40], x[40:80]
    f = pkg.clip_gradients
    for bad in (lambda: f([x[:10], x[5:20]], 1.0), lambda: f([x, b], 1.0), lambda: f([a, b], 1.0, out=[b, a]),
                lambda: f([a, b], 1.0, out=[x[1:41], x[50:90]]), lambda: f(a, 1.0, out=x[:80].view(torch.bfloat16)[2:42]),
                lambda: pkg.GradientClipper([b, x[20:60]]).clip(1.0)):
        with pytest.raises(ValueError):
            bad()
    y = torch.empty(100, device=DEV)
    f([a, a], 1e9, out=[y[:40], y[40:80]])  # gradients alike, results apart
    f([a, b], 1e9, out=[a, y[:40]])
    assert torch.equal(y[:80], x[:80])
