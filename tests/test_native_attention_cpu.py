"""CPU-only checks of the packed attention's and rotary's entry points: bad arguments are refused
before any device call, and the Python functions refuse CPU tensors."""

from __future__ import annotations

import pytest
import torch


def _attention(N, T=4, Tk=4, H=2, Hkv=2, D=64, n=1, scale=0.1, q=16, strides=(128, 64), out=16, off=16):
    return N.lib().rfdetr_packed_attention(None, q, *strides, 16, Hkv * D, D, 16, Hkv * D, D, off, None, out, None,
                                           None, None, 0, n, T, Tk, H, Hkv, D, 0, scale)


def test_attention_arguments(pkg):
    N = pkg._native
    assert _attention(N, T=0, q=None, out=None) == N.OK  # nothing to do
    for bad in ({"H": 3}, {"H": 1}, {"Hkv": 0}, {"D": 60}, {"D": 136}, {"D": 0}, {"T": -1}, {"Tk": 1 << 31},
                {"n": -1}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}, {"scale": float("inf")}):
        assert _attention(N, **bad) == N.ERR_SHAPE, bad
    for bad in ({"q": None}, {"q": 24}, {"strides": (129, 64)}, {"strides": (128, 0)}, {"strides": (128, -64)},
                {"out": None}, {"out": 8}, {"off": None}):
        assert _attention(N, **bad) == N.ERR_ALIGN, bad
    lib = N.lib()
    assert lib.rfdetr_packed_attention_backward_workspace_bytes(100, 6) == 2400
    assert lib.rfdetr_packed_attention_backward_workspace_bytes(-1, 6) == 0
    assert lib.rfdetr_packed_attention_workspace_bytes(1, 4, 4, 3, 2, 64) == 0
    back = lambda ws, nbytes, g=16, low=16: lib.rfdetr_packed_attention_backward(  # noqa: E731
        None, 16, 128, 64, 16, 128, 64, 16, 128, 64, 16, None, 16, low, 16, g, 128, 64, None, 16, 16, 16, ws,
        nbytes, 1, 4, 4, 2, 2, 64, 0, 0.1)
    assert back(None, 0) == N.ERR_WORKSPACE
    assert back(16, 31) == N.ERR_WORKSPACE
    assert back(16, 32, None) == N.ERR_ALIGN
    assert back(16, 32, low=None) == N.ERR_ALIGN and back(16, 32, low=8) == N.ERR_ALIGN


def test_rotary_arguments(pkg):
    N = pkg._native

    def call(T=4, H=2, Hkv=1, D=8, sections=(2, 2), dtype=0, pos_dtype=0, q=16, interleaved=0, strides=(16, 8)):
        return N.lib().rfdetr_axial_rotary(None, q, *strides, 16, 8, 8, dtype, 16, pos_dtype, 16,
                                           N.int64_array(sections), len(sections), 16, 16, T, H, Hkv, D, interleaved,
                                           0)

    assert call(T=0) == N.OK
    assert call(H=0, Hkv=0) == N.OK
    assert call(dtype=5) == N.ERR_DTYPE and call(dtype=2) == N.ERR_DTYPE and call(pos_dtype=1) == N.ERR_DTYPE
    for bad in ({"T": -1}, {"D": 1}, {"D": 2000}, {"sections": (3, 2)}, {"sections": (-1, 3)}, {"sections": (0, 0)},
                {"sections": (1,) * 9}, {"strides": (-16, 8)}):
        assert call(**bad) == N.ERR_SHAPE, bad
    assert call(q=None) == N.ERR_ALIGN and call(q=18) == N.ERR_ALIGN
    assert call(interleaved=1, strides=(17, 8)) == N.ERR_ALIGN


def test_cpu_tensors_are_refused(pkg):
    x = torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA tensors"):
        pkg.packed_attention(x, x, x, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA tensors"):
        pkg.axial_rotary(x, x, torch.zeros((4, 1)), torch.zeros(2), (2,))
