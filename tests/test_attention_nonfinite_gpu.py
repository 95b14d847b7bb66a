"""Scores that are NaN or infinite, in every column of a key tile and in every forward kernel."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import attention as OA

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
KERNELS = ["1", "2", "3", "3,2"]


def _bf16(rng, *shape):
    return torch.tensor(rng.standard_normal(shape).astype(np.float32), device=DEV).to(torch.bfloat16)


def _f64(t):
    return t.detach().double().cpu().numpy()


def _offsets(lengths):
    return torch.tensor(np.cumsum([0, *lengths]), dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("knob", KERNELS)
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_a_nan_key_shows_in_every_row_that_sees_it(pkg, tuning, knob, dim):
    """One key of each sequence is NaN, another column of the first tile in each: the definition has NaN in
    every row's output and log-sum-exp."""
    tuning("RFDETR_ATTN_FWD", knob)
    rng = np.random.default_rng(dim)
    count, n = 32, 150
    q, k, v = (_bf16(rng, count * n, 2, dim) for _ in range(3))
    for s in range(count):
        k[s * n + s] = float("nan")
    out, lse = pkg.packed_attention(q, k, v, _offsets((n,) * count), return_lse=True)
    assert torch.isnan(lse).all()
    assert torch.isnan(out).all()


@pytest.mark.parametrize("knob", KERNELS)
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_rows_whose_scores_are_all_minus_infinity(pkg, tuning, knob, dim):
    """They count as rows without keys: output 0, log-sum-exp -inf, and (where the scores got there by overflow,
    so that no operand is infinite) gradients 0."""
    tuning("RFDETR_ATTN_FWD", knob)
    rng = np.random.default_rng(dim + 1)
    lengths = (300, 129, 200)
    off = _offsets(lengths)
    q, k, v, g = (_bf16(rng, sum(lengths), 2, dim) for _ in range(4))
    q[300:429] = 0.0
    k[300:429] = 0.0
    q[300:429, :, 0] = 2.0 ** 100
    k[300:429, :, 0] = -2.0 ** 100  # their product is past float32
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out, lse = pkg.packed_attention(*leaves, off, return_lse=True)
    assert torch.isneginf(lse[:, 300:429]).all() and not out[300:429].any()
    for d in torch.autograd.grad(out, leaves, g):
        assert not d[300:429].any()
        assert torch.isfinite(d).all() and d[:300].any() and d[429:].any()


@pytest.mark.parametrize("knob", KERNELS)
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_keys_at_minus_infinity_weigh_nothing(pkg, tuning, knob, dim):
    """Every other pair of keys has the score -inf: the result is that of the keys left, within the same bounds."""
    tuning("RFDETR_ATTN_FWD", knob)
    rng = np.random.default_rng(dim + 2)
    n = 400
    q, k, v = (_bf16(rng, n, 2, dim) for _ in range(3))
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    left = (np.arange(n) // 2) % 2 == 0
    k[torch.tensor(~left, device=DEV), :, 0] = -float("inf")
    out, lse = pkg.packed_attention(q, k, v, _offsets((n,)), return_lse=True)
    r = OA.attention(_f64(q), _f64(k)[left], _f64(v)[left], [0, n], [0, int(left.sum())])
    assert (np.abs(_f64(out) - r["out"]) <= r["out_bound"]).all()
    assert (np.abs(_f64(lse) - r["lse"]) <= r["lse_bound"]).all()
