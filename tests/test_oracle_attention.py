"""The attention and rotary oracles against independent evaluations: torch's float64 autograd of the
textbook softmax, central differences, and rotation matrices."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import attention as OA
from oracle import rotary as OR


def _inputs(seed, lengths, keys, heads, kv, dim):
    rng = np.random.default_rng(seed)
    tq, tk = sum(lengths), sum(keys)
    q = rng.standard_normal((tq, heads, dim))
    k, v = rng.standard_normal((2, tk, kv, dim))
    return (q, k, v, np.cumsum([0, *lengths]), np.cumsum([0, *keys]), rng.standard_normal((tq, heads, dim)),
            rng.standard_normal((heads, tq)))


def _torch_attention(q, k, v, off, koff, causal, scale):
    outs, lses = [], []
    for s in range(len(off) - 1):
        a, b = q[off[s]:off[s + 1]], k[koff[s]:koff[s + 1]]
        c = v[koff[s]:koff[s + 1]]
        b, c = (x.repeat_interleave(q.shape[1] // k.shape[1], 1) for x in (b, c))
        n, m = a.shape[0], b.shape[0]
        x = scale * torch.einsum("nhd,mhd->hnm", a, b)
        if causal:
            x = x.masked_fill(~torch.ones(n, m, dtype=torch.bool).tril(m - n), -torch.inf)
        lses.append(torch.logsumexp(x, -1))
        outs.append(torch.einsum("hnm,mhd->nhd", torch.softmax(x, -1), c))
    return torch.cat(outs), torch.cat(lses, 1)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize(("lengths", "keys", "heads", "kv"), [((3, 1, 5), (3, 1, 5), 2, 2), ((2, 4), (6, 4), 6, 2)])
def test_against_autograd(lengths, keys, heads, kv, causal):
    q, k, v, off, koff, g, gl = _inputs(1, lengths, keys, heads, kv, 8)
    r = OA.attention(q, k, v, off, koff, causal, 0.3, g, gl)
    t = [torch.tensor(x, requires_grad=True) for x in (q, k, v)]
    out, lse = _torch_attention(*t, off, koff, causal, 0.3)
    ((out * torch.tensor(g)).sum() + (lse * torch.tensor(gl)).sum()).backward()
    for name, want in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *(x.grad for x in t))):
        np.testing.assert_allclose(r[name], want.detach().numpy(), rtol=1e-12, atol=1e-13)


def test_against_differences():
    q, k, v, off, koff, g, gl = _inputs(2, (3, 2), (4, 2), 4, 2, 8)
    args = [q, k, v]

    def value():
        r = OA.attention(*args, off, koff, True, 0.4)
        return (r["out"] * g).sum() + (r["lse"] * gl).sum()

    r = OA.attention(*args, off, koff, True, 0.4, g, gl)
    rng = np.random.default_rng(3)
    for x, name in zip(args, ("dq", "dk", "dv")):
        for _ in range(12):
            at = tuple(rng.integers(0, n) for n in x.shape)
            keep, h = x[at], 1e-5
            x[at] = keep + h
            up = value()
            x[at] = keep - h
            down = value()
            x[at] = keep
            # Central difference: h^2 truncation, 1e-16 / h rounding.
            assert abs((up - down) / (2 * h) - r[name][at]) < 1e-7


def test_rows_without_keys():
    q, k, v, off, koff, g, _ = _inputs(4, (3, 4), (0, 2), 2, 1, 8)
    r = OA.attention(q, k, v, off, koff, True, None, g)
    assert not r["out"][:5].any() and np.isneginf(r["lse"][:, :5]).all()  # 3 rows, then 2 before key 0
    assert not r["dq"][:5].any() and np.isfinite(r["lse"][:, 5:]).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_is_a_rotation(interleaved):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((4, 3, 10))
    pos = rng.integers(0, 50, (4, 2))
    freq = rng.uniform(0.01, 1.0, 4)
    y = OR.rotary(x, pos, freq, (1, 3), interleaved)
    for t in range(4):
        for i in range(4):
            theta = pos[t, 0 if i < 1 else 1] * freq[i]
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 4)
            m = np.array([[np.cos(theta), -np.sin(theta)], [np.sin(theta), np.cos(theta)]])
            np.testing.assert_allclose(y[t][:, [a, b]], x[t][:, [a, b]] @ m.T, atol=1e-13)
    np.testing.assert_array_equal(y[..., 8:], x[..., 8:])
    np.testing.assert_allclose(OR.rotary(y, pos, freq, (1, 3), interleaved, inverse=True), x, atol=1e-13)
