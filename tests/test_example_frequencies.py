"""The decoder layer example's rotary frequencies stay float32 whatever type the layer is given."""

from __future__ import annotations

import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(pkg):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import decoder_layer
    finally:
        sys.path.pop(0)
    return decoder_layer


def test_frequencies_are_not_rounded(example):
    freq = (64.0 * 100.0 ** (-torch.arange(8, dtype=torch.float64) / 8)).repeat(2)
    for convert in (lambda x: x, lambda x: x.to(torch.bfloat16), lambda x: x.half().bfloat16(), lambda x: x.double()):
        layer = convert(example.DecoderLayer())
        assert layer.inv_freq.dtype == torch.float32
        assert ((layer.inv_freq.double() - freq).abs() <= 2.0 ** -21 * freq).all()
