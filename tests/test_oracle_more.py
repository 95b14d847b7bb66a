"""The oracles of the changed scores and of the normed rotary positions on the CPU: their gradients against differences of
their own outputs, and, without a change, the plain oracles."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import attention as OA
from oracle import rotary as OR
from oracle.normed_rotary import normed_rotary
from oracle.scored_attention import scored_attention


def _inputs(rng, tokens=23, heads=4, kv=2, dim=6):
    return (rng.standard_normal((tokens, heads, dim)) * 2, rng.standard_normal((tokens, kv, dim)),
            rng.standard_normal((tokens, kv, dim)), rng.standard_normal((tokens, heads, dim)))


@pytest.mark.parametrize("how", [dict(cap=2.0), dict(slopes=(0.5, 0.1, 0.0, -0.2)), dict(causal=True, prefix=(4, 1)),
                                 dict(causal=True, cap=3.0, slopes=(0.5, 0.1, 0.02, 1.0), prefix=(0, 30))])
def test_scored_attention_gradients(how):
    rng = np.random.default_rng(0)
    q, k, v, g = _inputs(rng)
    off = [0, 11, 23]
    gl = rng.standard_normal((4, 23))
    r = scored_attention(q, k, v, off, grad=g, grad_lse=gl, **how)

    def value(q, k, v):
        x = scored_attention(q, k, v, off, **how)
        return (x["out"] * g).sum() + (x["lse"] * gl).sum()

    for i, name in enumerate(("dq", "dk", "dv")):
        way = rng.standard_normal((q, k, v)[i].shape)
        moved = lambda h: value(*(x + h * way if j == i else x for j, x in enumerate((q, k, v))))  # noqa: E731
        got = (4 * (moved(5e-5) - moved(-5e-5)) / 1e-4 - (moved(1e-4) - moved(-1e-4)) / 2e-4) / 3
        want = (r[name] * way).sum()
        assert abs(got - want) <= 1e-7 * np.abs(r[name] * way).sum()


def test_without_a_change_it_is_plain_attention():
    rng = np.random.default_rng(1)
    q, k, v, g = _inputs(rng)
    a = OA.attention(q, k, v, [0, 9, 23], causal=True, grad=g)
    for how in (dict(), dict(cap=1e7), dict(slopes=np.zeros(4)), dict(prefix=(0, 0))):
        b = scored_attention(q, k, v, [0, 9, 23], causal=True, grad=g, **how)
        for name in ("out", "lse", "dq", "dk", "dv"):
            np.testing.assert_allclose(b[name], a[name], rtol=1e-9, atol=1e-12)


def test_a_prefix_of_all_keys_is_no_mask():
    rng = np.random.default_rng(2)
    q, k, v, _ = _inputs(rng)
    a = scored_attention(q, k, v, [0, 23], causal=True, prefix=(40,))
    np.testing.assert_allclose(a["out"], OA.attention(q, k, v, [0, 23])["out"], rtol=1e-12)


@pytest.mark.parametrize("interleaved", [False, True])
def test_normed_rotary_gradients(interleaved):
    rng = np.random.default_rng(3)
    x, w = rng.standard_normal((7, 2, 10)), rng.standard_normal(10)
    pos, freq, sections = rng.uniform(0, 5, (7, 2)), rng.uniform(0.1, 1, 3), (1, 2)
    g = rng.standard_normal(x.shape)
    y, _, dx, _, dw, _ = normed_rotary(x, w, 1e-6, pos, freq, sections, interleaved, g)
    for d, name in ((dx, "x"), (dw, "w")):
        way = rng.standard_normal(d.shape)
        at = lambda h: (normed_rotary(x + h * way if name == "x" else x, w + h * way if name == "w" else w, 1e-6,  # noqa: E731
                                      pos, freq, sections, interleaved)[0] * g).sum()
        got = (4 * (at(5e-5) - at(-5e-5)) / 1e-4 - (at(1e-4) - at(-1e-4)) / 2e-4) / 3
        assert abs(got - (d * way).sum()) <= 1e-7 * np.abs(d * way).sum()
    # A row of root mean square 1 is turned alone.
    unit = x / np.sqrt((x * x).mean(-1, keepdims=True))
    np.testing.assert_allclose(normed_rotary(unit, None, 0.0, pos, freq, sections, interleaved)[0],
                               OR.rotary(unit, pos, freq, sections, interleaved), rtol=1e-12, atol=1e-14)
