"""Packed attention with capped scores, a bias by distance and prefix masks, on the device against the float64 oracle,
elementwise within the bounds that the oracle derives from the operator's roundings."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.scored_attention import scored_attention

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _bf16(rng, *shape, size=1.0):
    return torch.tensor((size * rng.standard_normal(shape)).astype(np.float32), device=DEV).to(torch.bfloat16)


def _f64(t):
    return t.detach().double().cpu().numpy()


def _offsets(lengths):
    return torch.tensor(np.cumsum([0, *lengths]), dtype=torch.int32, device=DEV)


def _close(name, got, want, bound):
    got = _f64(got)
    assert got.shape == want.shape
    same = got == want  # infinities
    off = np.where(same, 0.0, np.abs(got - np.where(same, 0.0, want)))
    bad = ~(off <= bound + 1e-30)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.size} outside the bound; first at {np.argwhere(bad)[0]}, " \
                          f"{got[bad][0]} for {want[bad][0]} within {bound[bad][0]:.3e}"


def _fault_free(pkg):
    assert pkg._native.lib().rfdetr_take_device_fault(torch.cuda.current_stream().cuda_stream) == 0


def _check(pkg, lengths, keys=None, heads=4, kv=2, dim=64, causal=False, cap=None, slopes=None, prefix=None, seed=0,
           size=3.0, scale=None, with_lse_grad=False, grad=True):
    rng = np.random.default_rng(seed)
    own = keys is None
    tk = sum(lengths if own else keys)
    q, k, v = _bf16(rng, sum(lengths), heads, dim, size=size), _bf16(rng, tk, kv, dim), _bf16(rng, tk, kv, dim)
    g = _bf16(rng, sum(lengths), heads, dim)
    gl = torch.tensor(rng.standard_normal((heads, sum(lengths))).astype(np.float32), device=DEV)
    off, koff = _offsets(lengths), None if own else _offsets(keys)
    m = None if slopes is None else torch.tensor(slopes, dtype=torch.float32, device=DEV)
    pre = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=DEV)
    r = scored_attention(_f64(q), _f64(k), _f64(v), off.cpu().numpy(), None if own else koff.cpu().numpy(), causal,
                         scale, cap, None if m is None else _f64(m), prefix, _f64(g) if grad else None,
                         _f64(gl) if with_lse_grad else None)
    how = dict(causal=causal, scale=scale, score_cap=cap, distance_slopes=m, prefix=pre)
    plain = pkg.packed_attention(q, k, v, off, koff, **how)
    _close("out", plain, r["out"], r["out_bound"])
    if not grad:
        _fault_free(pkg)
        return
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out, lse = pkg.packed_attention(*leaves, off, koff, return_lse=True, **how)
    _close("out", out, r["out"], r["out_bound"])
    _close("lse", lse, r["lse"], r["lse_bound"])
    outs, gs = ((out, lse), (g, gl)) if with_lse_grad else ((out,), (g,))
    for name, d in zip(("dq", "dk", "dv"), torch.autograd.grad(outs, leaves, gs)):
        _close(name, d, r[name], r[name + "_bound"])
    _fault_free(pkg)


def _slopes(heads):
    return 2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("lengths", [(1,), (7,), (64,), (129,), (300, 300), (5, 0, 257, 1, 130)])
@pytest.mark.parametrize("what", ["cap", "slopes", "both"])
def test_lengths(pkg, lengths, dim, causal, what):
    _check(pkg, lengths, dim=dim, causal=causal, cap=None if what == "slopes" else 20.0,
           slopes=None if what == "cap" else _slopes(4), seed=sum(lengths) + dim)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("prefix", [(0, 0), (1, 1), (2, 150), (700, 128), (5000, 129)])
def test_prefix(pkg, prefix, dim):
    """None, one key (rows before it see that alone), inside a tile, a whole tile, past the sequence."""
    _check(pkg, (700, 150), dim=dim, causal=True, prefix=prefix, seed=dim + prefix[1], with_lse_grad=True)


@pytest.mark.parametrize("dim", [32, 128])
@pytest.mark.parametrize(("lengths", "keys", "prefix"), [
    ((300, 300, 4), (576, 0, 1), (100, 3, 1)), ((1, 1, 1), (700, 1, 0), (10, 0, 2)), ((200, 10), (30, 200), (1, 0)),
    ((200, 10), (30, 200), (0, 7)), ((3, 5), (0, 64), (2, 2)), ((900, 2), (129, 2000), (40, 0))])
def test_queries_of_other_tokens(pkg, lengths, keys, prefix, dim):
    """Rows whose mask leaves nothing but a prefix, or nothing at all: no keys, or more queries than keys."""
    _check(pkg, lengths, keys, dim=dim, causal=True, prefix=prefix, cap=15.0, slopes=_slopes(4), seed=sum(keys))
    _check(pkg, lengths, keys, dim=dim, causal=False, cap=15.0, slopes=_slopes(4), seed=sum(keys))


@pytest.mark.parametrize("cap", [0.01, 1.0, 4.0, 9.0, 50.0, 1e4])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_caps(pkg, cap, dim):
    """From caps that most scores pass, through those that a few tiles pass, to one that changes nothing."""
    _check(pkg, (400, 77), heads=2, kv=1, dim=dim, causal=True, cap=cap, seed=int(cap))


@pytest.mark.parametrize("what", ["cap", "slopes"])
def test_scales(pkg, what):
    for scale in (0.02, 1.0):
        _check(pkg, (400, 77), heads=2, kv=1, causal=True, scale=scale, cap=25.0 if what == "cap" else None,
               slopes=(0.5, 0.01) if what == "slopes" else None, size=1.0)


@pytest.mark.parametrize(("heads", "kv"), [(1, 1), (6, 2), (7, 1), (5, 5), (71, 1), (96, 1)])
def test_grouped_heads(pkg, heads, kv):
    """Each head has its own slope, heads of a group in one tile."""
    _check(pkg, (33, 150, 2), heads=heads, kv=kv, causal=True, cap=20.0, slopes=_slopes(heads), prefix=(4, 0, 2),
           seed=heads)


def test_slopes_of_either_sign(pkg):
    """Steep, none, and negative (scores that rise with distance)."""
    for causal in (False, True):
        _check(pkg, (500, 90), heads=4, kv=4, causal=causal, slopes=(8.0, 0.0, -0.01, -0.5), size=1.0)


@pytest.mark.parametrize("dim", [8, 40, 72, 120])
def test_channels_that_fill_no_tile(pkg, dim):
    _check(pkg, (70, 200), dim=dim, causal=True, cap=12.0, slopes=_slopes(4), prefix=(30, 0), seed=dim)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_long(pkg, dim, causal):
    _check(pkg, (1700, 900), dim=dim, causal=causal, cap=18.0, slopes=_slopes(4), prefix=(600, 0) if causal else None,
           seed=dim)


@pytest.mark.parametrize("knob", ["1", "2", "3", "3,4"])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_every_forward_kernel(pkg, tuning, knob, dim):
    """The kernel for long sequences, the short one, halves in turn, keys shared out."""
    tuning("RFDETR_ATTN_FWD", knob)
    for cap, slopes in ((9.0, None), (None, _slopes(4)), (30.0, _slopes(4))):
        _check(pkg, (310, 100), (1000, 400), dim=dim, causal=True, cap=cap, slopes=slopes, prefix=(300, 0), grad=False)


@pytest.mark.parametrize("knob", ["1,1", "2,2", "4,4"])
def test_every_backward_split(pkg, tuning, knob):
    tuning("RFDETR_ATTN_BWD", knob)
    for dim in (32, 64, 128):
        _check(pkg, (600, 100), dim=dim, causal=True, cap=12.0, slopes=_slopes(4), prefix=(200, 1))


def test_single_tokens_over_a_long_cache(pkg):
    _check(pkg, (1,) * 5, (9000, 1, 0, 4097, 130), heads=16, kv=4, dim=128, causal=True, cap=30.0, slopes=_slopes(16),
           grad=False)


def test_without_a_change_the_bits_are_the_plain_call_s(pkg):
    """A prefix of no keys, slopes of 0 and a cap that is far from all scores leave the values, within a step of rounding;
    no change at all leaves the bits."""
    rng = np.random.default_rng(1)
    q, k, v = _bf16(rng, 300, 4, 64), _bf16(rng, 300, 2, 64), _bf16(rng, 300, 2, 64)
    off = _offsets((200, 100))
    want = pkg.packed_attention(q, k, v, off, causal=True)
    assert torch.equal(want, pkg.packed_attention(q, k, v, off, causal=True, score_cap=None, distance_slopes=None,
                                                  prefix=None))
    r = scored_attention(_f64(q), _f64(k), _f64(v), [0, 200, 300], causal=True)
    for how in (dict(prefix=torch.zeros(2, dtype=torch.int64, device=DEV)),
                dict(distance_slopes=torch.zeros(4, device=DEV)), dict(score_cap=1e4)):
        _close("out", pkg.packed_attention(q, k, v, off, causal=True, **how), r["out"], r["out_bound"])


def test_one_key_has_no_score_gradient(pkg):
    """A row that sees one key has P = 1: dS is 0 whatever the roundings; with a prefix of one, many rows do."""
    rng = np.random.default_rng(2)
    q, k, v = (_bf16(rng, 40, 2, 64).requires_grad_(True) for _ in range(3))
    key, value = k.detach()[:10].clone().requires_grad_(True), v.detach()[:10].clone().requires_grad_(True)
    out = pkg.packed_attention(q, key, value, _offsets((40,)), _offsets((10,)), causal=True, score_cap=5.0,
                               prefix=torch.ones(1, dtype=torch.int32, device=DEV))
    dq, dk, _ = torch.autograd.grad(out, (q, key, value), _bf16(rng, 40, 2, 64))
    assert not dq[:31].any() and dq[31:].any()


@pytest.mark.parametrize("knob", ["1", "2", "3", "3,2"])
def test_one_key_gives_its_value(pkg, tuning, knob):
    """A row that sees one key is that key's value, whatever its score, distance and cap: bit for bit."""
    tuning("RFDETR_ATTN_FWD", knob)
    rng = np.random.default_rng(7)
    for dim in (32, 64, 128):
        for how in (dict(score_cap=40.0), dict(score_cap=2.0), dict(score_cap=1e3),
                    dict(distance_slopes=torch.tensor([0.7, 0.01], device=DEV)),
                    dict(score_cap=40.0, distance_slopes=torch.tensor([0.7, 0.01], device=DEV))):
            q, k, v = (_bf16(rng, 150, 2, dim, size=3.0) for _ in range(3))
            out = pkg.packed_attention(q, k[:3], v[:3], _offsets((100, 0, 50)), _offsets((1, 1, 1)), **how)
            assert torch.equal(out[:100], v[:1].expand(100, 2, dim)) and torch.equal(out[100:], v[2:3].expand(50, 2, dim))
            out = pkg.packed_attention(q, k, v, _offsets((150,)), causal=True, **how)
            assert torch.equal(out[0], v[0])


def test_rows_without_a_query_choose_nothing(pkg):
    """A tile's rows behind its sequence's last query hold the next sequence's: their products, out of every polynomial's
    reach, change no bit of its gradients, in tiles whose last warp has one live row."""
    rng = np.random.default_rng(8)
    for dim in (32, 64, 128):
        q, k, v, g = (_bf16(rng, 500, 2, dim) for _ in range(4))
        off = _offsets((257, 243))
        loud = q.clone()
        loud[257:] *= 100.0
        got = []
        for x in (q, loud):
            leaves = [y.clone().requires_grad_(True) for y in (x, k, v)]
            out = pkg.packed_attention(*leaves, off, score_cap=12.0)
            got.append([out, *torch.autograd.grad(out, leaves, g)])
        for a, b in zip(*got):
            assert torch.equal(a[:257], b[:257])


def test_foreign_rows_change_nothing(pkg):
    """NaN, infinities and large values in rows outside the sequences, and in other sequences, change no bit."""
    rng = np.random.default_rng(3)
    slopes = torch.tensor(_slopes(4), dtype=torch.float32, device=DEV)
    for dim in (32, 64, 128):
        q, k, v = _bf16(rng, 400, 4, dim), _bf16(rng, 400, 2, dim), _bf16(rng, 400, 2, dim)
        g = _bf16(rng, 400, 4, dim)
        off = torch.tensor([10, 170, 300], dtype=torch.int32, device=DEV)

        def call(q, k, v):
            leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
            out = pkg.packed_attention(*leaves, off, causal=True, score_cap=10.0, distance_slopes=slopes,
                                       prefix=torch.tensor([20, 30], dtype=torch.int32, device=DEV))
            return [out, *torch.autograd.grad(out, leaves, g)]

        want = call(q, k, v)
        for value in (float("nan"), float("inf"), 1e30):
            other = [x.clone() for x in (q, k, v)]
            for x in other:
                x[:10], x[300:] = value, value
            for a, b in zip(call(*other), want):
                assert torch.equal(a[10:300], b[10:300])
        other = [x.clone() for x in (q, k, v)]
        for x in other:
            x[170:300] *= 50.0
        for a, b in zip(call(*other), want):
            assert torch.equal(a[10:170], b[10:170])


def test_infinite_products_are_capped(pkg):
    """A key whose products are infinite counts like one at the cap."""
    rng = np.random.default_rng(4)
    q, k, v = _bf16(rng, 1, 1, 64), _bf16(rng, 5, 1, 64), _bf16(rng, 5, 1, 64)
    q[0, 0, 0] = 1.0
    k[2, 0, 0] = float("inf")
    out, lse = pkg.packed_attention(q, k, v, _offsets((1,)), _offsets((5,)), score_cap=3.0, return_lse=True)
    s = 0.125 * (_f64(q)[0, 0] @ np.where(np.isinf(_f64(k)[:, 0]), 0.0, _f64(k)[:, 0]).T)
    s = 3.0 * np.tanh(s / 3.0)
    s[2] = 3.0
    assert abs(float(lse) - np.log(np.exp(s).sum())) <= 1e-5
    p = np.exp(s) / np.exp(s).sum()
    want, bound = p @ _f64(v)[:, 0], 2.0 ** -7 * (p @ np.abs(_f64(v)[:, 0]))
    assert (np.abs(_f64(out)[0, 0] - want) <= bound).all()


def test_gradient_against_differences(pkg):
    """The derivative along a direction of q against differences of the float64 definition: the difference's third-order
    part is taken out by halving the step; what is left is the operator's own bound."""
    rng = np.random.default_rng(5)
    q, k, v = _bf16(rng, 60, 2, 32, size=3.0), _bf16(rng, 60, 2, 32), _bf16(rng, 60, 2, 32)
    g = _bf16(rng, 60, 2, 32)
    how = dict(causal=True, cap=6.0, slopes=np.array([0.25, 0.03]), prefix=(13,))
    way = rng.standard_normal(q.shape)

    def value(by):
        return float((scored_attention(_f64(q) + by * way, _f64(k), _f64(v), [0, 60], **how)["out"] * _f64(g)).sum())

    slope = [(value(h) - value(-h)) / (2 * h) for h in (1e-3, 5e-4)]
    want = (4 * slope[1] - slope[0]) / 3
    r = scored_attention(_f64(q), _f64(k), _f64(v), [0, 60], grad=_f64(g), **how)
    assert abs(want - (r["dq"] * way).sum()) <= 1e-6 * np.abs(r["dq"] * way).sum()
    leaf = q.clone().requires_grad_(True)
    out = pkg.packed_attention(leaf, k, v, _offsets((60,)), causal=True, score_cap=6.0,
                               distance_slopes=torch.tensor(how["slopes"], dtype=torch.float32, device=DEV),
                               prefix=torch.tensor([13], dtype=torch.int32, device=DEV))
    got = float((torch.autograd.grad(out, leaf, g)[0].double().cpu().numpy() * way).sum())
    assert abs(got - want) <= (r["dq_bound"] * np.abs(way)).sum()


def test_captured(pkg):
    """A captured pass, replayed with other inputs and prefixes in place, gives the bits of a plain one."""
    rng = np.random.default_rng(6)
    q, k, v, g = (_bf16(rng, 500, 4, 64) for _ in range(4))
    k, v = k[:, :2].contiguous(), v[:, :2].contiguous()
    off, pre = _offsets((300, 200)), torch.tensor([50, 7], dtype=torch.int32, device=DEV)
    slopes = torch.tensor(_slopes(4), dtype=torch.float32, device=DEV)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]

    def step():
        out = pkg.packed_attention(*leaves, off, causal=True, score_cap=8.0, distance_slopes=slopes, prefix=pre)
        return [out, *torch.autograd.grad(out, leaves, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for change in (lambda: None, lambda: pre.fill_(120), lambda: slopes.mul_(2.0)):
        change()
        graph.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_refusals(pkg):
    q = torch.zeros(10, 4, 64, device=DEV, dtype=torch.bfloat16)
    off = _offsets((4, 6))
    m, pre = torch.zeros(4, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    f = lambda **how: pkg.packed_attention(q, q, q, off, **how)  # noqa: E731
    for bad in (dict(score_cap=0.0), dict(score_cap=-3.0), dict(score_cap=float("nan")), dict(score_cap=float("inf")),
                dict(score_cap=1e30), dict(distance_slopes=m[:3]), dict(distance_slopes=m.double()),
                dict(distance_slopes=m.cpu()), dict(distance_slopes=m.clone().requires_grad_(True)),
                dict(prefix=pre), dict(prefix=pre[:1], causal=True), dict(prefix=pre.float(), causal=True),
                dict(prefix=pre.cpu(), causal=True)):
        with pytest.raises(ValueError):
            f(**bad)
    f(score_cap=1.0, distance_slopes=m, prefix=pre, causal=True)


def _tiers(rng, heads, kv, dim, queries, values, cap=50.0):
    """Queries, keys and values whose scores lie in runs of 64 keys around these parts of the cap, low ones first, so that
    a row's largest score comes late and far above its first ones; `values`: the values' size."""
    at = np.repeat([-1.5, -1.2, -1.4, -0.6, 0.1, -1.0, 0.4, 1.2, -0.5, 2.5, 1.4, -2.5, 0.0, 3.0, 1.6], 64)
    one = dim ** -0.25 * np.ones(dim)
    q = 20.0 * one + 0.5 * rng.standard_normal((queries, heads, dim))
    k = cap / 20.0 * at[:, None, None] * one + 0.05 * rng.standard_normal((len(at), kv, dim))
    v = values * rng.standard_normal((len(at), kv, dim))
    return [torch.tensor(x.astype(np.float32), device=DEV).to(torch.bfloat16) for x in (q, k, v)]


@pytest.mark.parametrize("knob", ["1", "2", "3", "3,4"])
@pytest.mark.parametrize("values", [2.0 ** -60, 1.0, 2.0 ** 80])
def test_values_of_any_size(pkg, tuning, knob, values):
    """Weights stay near 1 whatever the first keys' scores: results are as far from float64 as their values' sizes say,
    be those tiny or large."""
    tuning("RFDETR_ATTN_FWD", knob)
    rng = np.random.default_rng(9)
    for dim, cap, slopes, causal, prefix in ((32, 50.0, None, False, None), (64, 50.0, None, True, (960,)),
                                             (128, 50.0, None, True, None), (64, 35.0, (0.01, -0.02), True, (300,)),
                                             (128, 50.0, (0.05, 0.004), False, None), (32, 60.0, (0.01, 0.0), True, None),
                                             (128, 60.0, None, True, None)):
        for queries in (1, 150, 960):
            q, k, v = _tiers(rng, 2, 1, dim, queries, values)
            m = None if slopes is None else torch.tensor(slopes, dtype=torch.float32, device=DEV)
            pre = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=DEV)
            out, lse = pkg.packed_attention(q, k, v, _offsets((queries,)), _offsets((960,)), causal=causal, score_cap=cap,
                                            distance_slopes=m, prefix=pre, return_lse=True)
            r = scored_attention(_f64(q), _f64(k), _f64(v), [0, queries], [0, 960], causal, None, cap,
                                 None if m is None else _f64(m), prefix)
            assert out.isfinite().all()
            _close("lse", lse, r["lse"], r["lse_bound"])
            _close("out", out.double() / values, r["out"] / values, r["out_bound"] / values)
    _fault_free(pkg)


@pytest.mark.parametrize("slope", [0.5, 8.0, 1e3, 1e6, 3e38])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_steep_slopes(pkg, dim, slope):
    """A bias is slope times distance rounded once: exactly 0 for the key that a row is level with, wherever in its tile
    that lies (at the end of one, for a single query over whole tiles of keys), and steep slopes leave that key alone."""
    for cap in (None, 20.0, 60.0):
        _check(pkg, (1, 1, 1, 1), (128, 64, 640, 131), heads=2, kv=1, dim=dim, causal=True, cap=cap, slopes=(slope, 0.25),
               seed=dim)
        _check(pkg, (40, 3), (168, 130), heads=2, kv=1, dim=dim, causal=False, cap=cap, slopes=(slope, 0.25), seed=dim)
        _check(pkg, (300, 64), heads=2, kv=1, dim=dim, causal=True, cap=cap, slopes=(0.25, slope), prefix=(150, 3), seed=dim)


@pytest.mark.parametrize("knob", ["1", "2", "3", "3,4"])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("cap", [8.0, 35.0, 50.0, 51.0, 60.0, 100.0])
def test_scores_past_the_cap_in_every_forward_kernel(pkg, tuning, knob, dim, cap):
    """Products of up to about one and up to about three caps, so that all forms of the cap are met in every kernel, with
    and without slopes and prefixes, in whole tiles and masked ones."""
    tuning("RFDETR_ATTN_FWD", knob)
    for part in (0.35, 1.0):
        for slopes, causal, prefix in ((None, False, None), (None, True, (300, 0)), ((0.5, 0.004, -0.01, 0.1), True, None),
                                       ((0.03, 0.0, 0.2, 0.01), False, None), ((0.1, 0.02, 0.3, 0.0), True, (129, 400))):
            _check(pkg, (310, 100), (1000, 400), dim=dim, causal=causal, cap=cap, slopes=slopes, prefix=prefix,
                   size=part * cap, grad=False, seed=int(cap) + dim)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("cap", [8.0, 50.0, 60.0])
def test_gradients_of_scores_past_the_cap(pkg, dim, cap):
    for part in (0.35, 1.0):
        for slopes, causal, prefix in ((None, False, None), ((0.5, 0.004, -0.01, 0.1), True, None),
                                       ((0.03, 0.0, 0.2, 0.01), True, (150, 3))):
            _check(pkg, (310, 64, 1), dim=dim, causal=causal, cap=cap, slopes=slopes,
                   prefix=None if prefix is None else (*prefix, 0), size=part * cap, seed=dim, with_lse_grad=True)


@pytest.mark.parametrize("knob", ["1", "2", "3", "3,4"])
def test_the_entries_without_a_change_are_the_plain_ones(pkg, tuning, knob):
    """``rfdetr_packed_attention`` and its gradients, and the entries with changed scores given none: equal bits."""
    tuning("RFDETR_ATTN_FWD", knob)
    N = pkg._native
    lib, stream = N.lib(), torch.cuda.current_stream().cuda_stream
    rng = np.random.default_rng(11)
    for dim in (32, 64, 128):
        T, Tk, H, Hkv, lengths, keys = 410, 1400, 4, 2, (310, 100), (1000, 400)
        q, k, v, g = (_bf16(rng, n, h, dim) for n, h in ((T, H), (Tk, Hkv), (Tk, Hkv), (T, H)))
        off, koff = _offsets(lengths), _offsets(keys)
        sizes = (2, T, Tk, H, Hkv, dim, 1, dim ** -0.5)
        rows = lambda x: (x.data_ptr(), x.stride(0), x.stride(1))  # noqa: E731
        results = []
        for forward, backward, more in (
                (lib.rfdetr_packed_attention, lib.rfdetr_packed_attention_backward, ()),
                (lib.rfdetr_packed_attention_scored, lib.rfdetr_packed_attention_scored_backward, (0.0, None, None))):
            out, low, dq = (torch.zeros_like(q) for _ in range(3))
            dk, dv = torch.zeros_like(k), torch.zeros_like(v)
            lse = torch.zeros(H, T, device=DEV)
            room = torch.zeros(max(lib.rfdetr_packed_attention_workspace_bytes(*sizes[:6]),
                                   lib.rfdetr_packed_attention_backward_workspace_bytes(T, H)), dtype=torch.uint8,
                               device=DEV)
            assert forward(stream, *rows(q), *rows(k), *rows(v), off.data_ptr(), koff.data_ptr(), out.data_ptr(),
                           low.data_ptr(), lse.data_ptr(), room.data_ptr(), room.numel(), *sizes, *more) == N.OK
            assert backward(stream, *rows(q), *rows(k), *rows(v), off.data_ptr(), koff.data_ptr(), out.data_ptr(),
                            low.data_ptr(), lse.data_ptr(), *rows(g), None, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                            room.data_ptr(), room.numel(), *sizes, *more) == N.OK
            results.append((out, low, lse, dq, dk, dv))
        for a, b in zip(*results):
            assert a.any() and torch.equal(a, b)
    _fault_free(pkg)


@pytest.mark.parametrize("knob", ["1", "2", "3", "3,2"])
@pytest.mark.parametrize("keys", [5, 128, 300])
def test_products_that_are_all_minus_infinity(pkg, tuning, knob, keys):
    """They are capped like any others: equal scores of minus the cap, whatever the tile's size."""
    tuning("RFDETR_ATTN_FWD", knob)
    rng = np.random.default_rng(keys)
    for cap in (3.0, 40.0, 70.0):
        q, k, v = _bf16(rng, 3, 1, 64), _bf16(rng, keys, 1, 64), _bf16(rng, keys, 1, 64)
        q[:, 0, 0], k[:, 0, 0] = 1.0, -float("inf")
        out, lse = pkg.packed_attention(q, k, v, _offsets((3,)), _offsets((keys,)), score_cap=cap, return_lse=True)
        assert (lse - (np.log(keys) - cap)).abs().max() <= 2.0 ** -20 * (cap + 10)
        want, size = _f64(v).mean(0), np.abs(_f64(v)).mean(0)
        assert (np.abs(_f64(out) - want) <= 2.0 ** -8 * (np.abs(want) + size)).all()
