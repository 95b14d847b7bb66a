"""The decoder layer example with normed queries and keys, capped scores and clipped gradients: the operators together,
as a training step uses them."""

from __future__ import annotations

import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"


@pytest.fixture(scope="module")
def example(pkg):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import decoder_layer
    finally:
        sys.path.pop(0)
    return decoder_layer


def test_steps_run(example):
    losses = example.fit(images=1, groups=3, per_group=50, steps=4, normed=True, score_cap=30.0, clip=0.01)
    assert len(losses) == 4 and all(x == x for x in losses)


def test_clipped_gradients(example, pkg):
    """After clipping the gradients' norm is the limit, up to each value's rounding to bf16 (2^-8 at most)."""
    torch.manual_seed(3)
    layer = example.DecoderLayer(normed=True, score_cap=20.0).to(device=DEV, dtype=torch.bfloat16)
    queries, boxes, memory = example.inputs(1, 2, 40, (8, 8), 256, DEV)
    layer(queries, boxes, memory, (8, 8), example.group_offsets(1, 2, 40, DEV)).float().square().mean().backward()
    grads = [p.grad for p in layer.parameters()]
    assert all(g is not None and g.isfinite().all() for g in grads)
    assert all(p.grad.any() for p in layer.head_norms)
    norm = pkg.clip_gradients(grads, float("inf"))
    pkg.clip_gradients(grads, 0.5 * float(norm))
    after = torch.stack([g.double().norm() for g in grads]).norm()
    assert abs(float(after) - 0.5 * float(norm)) <= 2.0 ** -8 * float(norm)


def test_self_attention_gradients(example, pkg):
    """The chain norm, turn, capped attention against the same steps in float64, in the 2-norm.  Queries and keys are rounded to
    bf16 after the turn: at |q| = |k| = sqrt(32) that moves a score by 2 x 2^-8 x sqrt(32) = 0.044 at most, so the
    weights, and what is linear in them, by 4.5%; the gradients pass them twice, and six roundings of 2^-8 of values between:
    0.09 + 0.024."""
    torch.manual_seed(4)
    layer = example.DecoderLayer(normed=True, score_cap=6.0).to(device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        for w in layer.head_norms:
            w.add_(0.2 * torch.randn_like(w))
    n, sizes = 66, (33, 33)
    qkv = torch.randn(n, 24, 32, device=DEV).to(torch.bfloat16)
    centers = torch.rand(n, 2, device=DEV)
    g = torch.randn(n, 8, 32, device=DEV).to(torch.bfloat16)
    offsets = example.group_offsets(1, 2, 33, DEV)
    leaves = [qkv.clone().requires_grad_(True), *(w.detach().clone().requires_grad_(True) for w in layer.head_norms)]
    q, k, v = leaves[0].split(8, 1)
    q, k = pkg.normed_axial_rotary(q, k, centers, layer.inv_freq, (8, 8), *leaves[1:])
    out = pkg.packed_attention(q, k, v, offsets, score_cap=6.0)
    got = [out, *torch.autograd.grad(out, leaves, g)]

    leaves = [x.detach().double().requires_grad_(True) for x in leaves]
    q, k, v = leaves[0].split(8, 1)
    theta = torch.cat([centers[:, a:a + 1].double() * layer.inv_freq[a * 8:a * 8 + 8].double() for a in (0, 1)], -1)
    cos, sin = theta.cos()[:, None], theta.sin()[:, None]

    def turned(x, w):
        x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        a, b = x[..., :16], x[..., 16:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    q, k = turned(q, leaves[1]), turned(k, leaves[2])
    parts = []
    for qs, ks, vs in zip(q.split(sizes), k.split(sizes), v.split(sizes)):
        s = 6.0 * torch.tanh(torch.einsum("ihd,jhd->hij", qs, ks) / 32 ** 0.5 / 6.0)
        parts.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), vs))
    want = torch.cat(parts)
    for a, b in zip(got, [want, *torch.autograd.grad(want, leaves, g.double())]):
        assert (a.double() - b).norm() <= 0.115 * b.norm()
