"""The decoder layer example: rotary, packed self-attention, prologue and sampler together."""

from __future__ import annotations

import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(pkg):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import decoder_layer
    finally:
        sys.path.pop(0)
    return decoder_layer


def test_it_learns(example):
    losses = example.fit(images=1, groups=3, per_group=50, steps=12)
    assert all(x == x for x in losses) and losses[-1] < 0.9 * losses[0]


def test_groups_do_not_see_each_other(example):
    """Other queries in one group leave the other groups' outputs bit for bit as they were."""
    dev = "cuda:0"
    torch.manual_seed(1)
    layer = example.DecoderLayer().to(device=dev, dtype=torch.bfloat16)
    queries, boxes, memory = example.inputs(2, 3, 40, (8, 8), 256, dev)
    offsets = example.group_offsets(2, 3, 40, dev)
    with torch.no_grad():
        want = layer(queries, boxes, memory, (8, 8), offsets)
        queries[0, 40:80] = torch.randn_like(queries[0, 40:80])
        got = layer(queries, boxes, memory, (8, 8), offsets)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0, :40], want[0, :40])
    assert torch.equal(got[0, 80:], want[0, 80:]) and not torch.equal(got[0, 40:80], want[0, 40:80])


def test_self_attention_matches_plain_operations(example):
    """The layer's self-attention against the same steps in float32 torch operations: one group at a
    time, rotation by explicit cosines.  Both start from the same bf16 projection; q and k rounded to
    bf16 after the turn, the weights and the result to bf16: a few 2^-8 of values of order one."""
    dev = "cuda:0"
    torch.manual_seed(2)
    layer = example.DecoderLayer().to(device=dev, dtype=torch.bfloat16)
    queries, boxes, _ = example.inputs(2, 2, 33, (4, 4), 256, dev)
    with torch.no_grad():
        got = layer.self_attention(queries, boxes[..., :2], example.group_offsets(2, 2, 33, dev))
        qkv = layer.qkv(queries).float().view(2, 2, 33, 24, 32)
        theta = torch.cat([boxes[..., a:a + 1] * layer.inv_freq[a * 8:a * 8 + 8].float() for a in (0, 1)], -1)
        cos, sin = (f(theta).view(2, 2, 33, 1, 16) for f in (torch.cos, torch.sin))

        def turned(x):
            a, b = x[..., :16], x[..., 16:]
            return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

        q, k, v = (x.transpose(2, 3) for x in qkv.split(8, 3))
        q, k = turned(qkv[..., :8, :]).transpose(2, 3), turned(qkv[..., 8:16, :]).transpose(2, 3)
        out = torch.softmax(q @ k.transpose(-1, -2) / 32 ** 0.5, -1) @ v
        want = layer.out(out.transpose(2, 3).reshape(2, 66, 256).to(torch.bfloat16))
    assert (got.float() - want.float()).abs().max() <= 8 * 2.0 ** -8
