"""A decoder layer in training form on this package's operators: grouped self-attention of the
detection groups' queries, then deformable cross-attention over a feature map.

The groups attend only within themselves, so they are packed sequences (:func:`packed_attention`
with offsets instead of a mask or a padded batch); the queries' reference points enter the attention
as rotary positions on two axes (:func:`axial_rotary`); the sampler's prologue and the sampler
follow.  Run it on a GPU: ``python examples/decoder_layer.py [--images N] [--groups G] [--steps K]``;
it fits random targets and prints the loss.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from __graft_entry__ import load_package  # noqa: E402

rf = load_package()


class DecoderLayer(nn.Module):
    """Self-attention (8 heads of 32) within groups, cross-attention (16 heads of 16, 2 points) and a
    feed-forward network, each with its residual and LayerNorm, hidden size 256."""

    def __init__(self, hidden=256, heads=8, sampler_heads=16, points=2):
        super().__init__()
        self.heads, self.sampler_heads, self.points = heads, sampler_heads, points
        self.qkv = nn.Linear(hidden, 3 * hidden)
        self.out = nn.Linear(hidden, hidden)
        self.offsets = nn.Linear(hidden, sampler_heads * points * 2)
        self.weights = nn.Linear(hidden, sampler_heads * points)
        self.value = nn.Linear(hidden, hidden)
        self.cross = nn.Linear(hidden, hidden)
        self.up, self.down = nn.Linear(hidden, 4 * hidden), nn.Linear(4 * hidden, hidden)
        self.norms = nn.ModuleList(nn.LayerNorm(hidden) for _ in range(3))
        # 8 frequencies to each of x and y: turns of up to 64 radians across the image.
        freq = 64.0 * 100.0 ** (-torch.arange(8) / 8)
        self.register_buffer("inv_freq", torch.cat((freq, freq)), persistent=False)

    def _apply(self, fn, recurse=True):
        """Conversions of the layer: the frequencies follow its device, not its type (in bf16 their turns
        would be off by up to 0.011 radians across the image)."""
        freq = self.inv_freq
        super()._apply(fn, recurse)
        self.inv_freq = freq.to(self.inv_freq.device)
        return self

    def self_attention(self, queries, centers, group_offsets):
        """``queries [B, G * Q, C]`` with ``centers [B, G * Q, 2]`` in [0, 1]; every group a sequence."""
        batch, count, hidden = queries.shape
        qkv = self.qkv(queries).view(batch * count, 3 * self.heads, hidden // self.heads)
        q, k, v = qkv.split(self.heads, 1)
        # Frequencies 0 to 7 turn by x, 8 to 15 by y.
        q, k = rf.axial_rotary(q, k, centers.reshape(batch * count, 2), self.inv_freq, (8, 8))
        return self.out(rf.packed_attention(q, k, v, group_offsets).view(batch, count, hidden))

    def cross_attention(self, queries, boxes, memory, shape):
        batch, _, hidden = queries.shape
        dim = hidden // self.sampler_heads
        loc, attn = rf.msda_prologue(queries, boxes[:, :, None], (shape,), self.offsets.weight, self.offsets.bias,
                                     self.weights.weight, self.weights.bias, self.sampler_heads, 1, self.points)
        value = self.value(memory).view(batch, -1, self.sampler_heads, dim).transpose(1, 2)
        value = value.reshape(batch * self.sampler_heads, -1, dim)
        return self.cross(rf.ms_deform_attn_core_rows(value, (shape,), loc, attn))

    def forward(self, queries, boxes, memory, shape, group_offsets):
        queries = self.norms[0](queries + self.self_attention(queries, boxes[..., :2], group_offsets))
        queries = self.norms[1](queries + self.cross_attention(queries, boxes, memory, shape))
        return self.norms[2](queries + self.down(torch.relu(self.up(queries))))


def group_offsets(images, groups, per_group, device):
    """Offsets of ``images * groups`` sequences of ``per_group`` queries."""
    return torch.arange(0, images * groups * per_group + 1, per_group, dtype=torch.int32, device=device)


def inputs(images, groups, per_group, shape, hidden, device, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, device=device).to(torch.bfloat16)  # noqa: E731
    boxes = torch.rand((images, groups * per_group, 4), generator=gen, device=device) * 0.8 + 0.1
    return normal(images, groups * per_group, hidden), boxes, normal(images, shape[0] * shape[1], hidden)


def fit(images=2, groups=13, per_group=300, steps=20, shape=(24, 24), device="cuda:0"):
    """Trains one layer towards random targets; returns the losses."""
    torch.manual_seed(0)
    layer = DecoderLayer().to(device=device, dtype=torch.bfloat16)
    queries, boxes, memory = inputs(images, groups, per_group, shape, 256, device)
    target = torch.randn_like(queries)
    offsets = group_offsets(images, groups, per_group, device)
    optimizer = torch.optim.AdamW(layer.parameters(), lr=1e-3)
    losses = []
    for _ in range(steps):
        optimizer.zero_grad(set_to_none=True)
        loss = (layer(queries, boxes, memory, shape, offsets) - target).float().square().mean()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return [float(x) for x in losses]


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--images", type=int, default=2)
    parser.add_argument("--groups", type=int, default=13)
    parser.add_argument("--steps", type=int, default=20)
    args = parser.parse_args()
    for i, value in enumerate(fit(args.images, args.groups, steps=args.steps)):
        print(f"step {i}: loss {value:.4f}")
