"""CPU-only checks of the entry points of the changed scores, the normed rotary positions and the clipping: bad
arguments are refused before any device call, and the Python functions refuse CPU tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch


def _scored(N, T=4, causal=1, scale=0.1, cap=30.0, slopes=16, prefix=16):
    return N.lib().rfdetr_packed_attention_scored(None, 16, 128, 64, 16, 128, 64, 16, 128, 64, 16, None, 16, None, None,
                                                  None, 0, 1, T, 4, 2, 2, 64, causal, scale, cap, slopes, prefix)


def test_scored_attention_arguments(pkg):
    N = pkg._native
    assert _scored(N, T=0) == N.OK
    for bad in (-1.0, float("nan"), float("inf"), 1e-30, 1e30, 2.0 ** 21, 2.0 ** -24):
        assert _scored(N, T=0, cap=bad) == N.ERR_SHAPE, bad
    assert _scored(N, T=0, cap=0.0, slopes=None, prefix=None) == N.OK
    assert _scored(N, T=0, slopes=18) == N.ERR_ALIGN and _scored(N, T=0, prefix=18) == N.ERR_ALIGN
    back = lambda cap, slopes=None, ws=16: N.lib().rfdetr_packed_attention_scored_backward(  # noqa: E731
        None, 16, 128, 64, 16, 128, 64, 16, 128, 64, 16, None, 16, 16, 16, 16, 128, 64, None, 16, 16, 16, ws, 32 if ws else 0,
        1, 4, 4, 2, 2, 64, 1, 0.1, cap, slopes, None)
    assert back(-1.0) == N.ERR_SHAPE and back(30.0, 18) == N.ERR_ALIGN and back(30.0, None, None) == N.ERR_WORKSPACE


def test_normed_rotary_arguments(pkg):
    N = pkg._native

    def call(T=4, H=2, Hkv=1, D=8, sections=(2, 2), dtype=0, pos_dtype=0, q=16, w=16, w_dtype=0, eps=1e-6, stride=16):
        return N.lib().rfdetr_normed_rotary(None, q, stride, 8, 16, 8, 8, dtype, w, w_dtype, None, 0, eps, 16, pos_dtype,
                                            16, N.int64_array(sections), len(sections), 16, 16, T, H, Hkv, D, 0)

    assert call(T=0) == N.OK and call(H=0, Hkv=0) == N.OK
    assert call(dtype=5) == N.ERR_DTYPE and call(pos_dtype=1) == N.ERR_DTYPE and call(w_dtype=2) == N.ERR_DTYPE
    for bad in ({"T": -1}, {"D": 1}, {"D": 257}, {"sections": (3, 2)}, {"sections": (-1, 3)}, {"sections": (0, 0)},
                {"sections": (1,) * 9}, {"stride": -16}, {"eps": -1.0}, {"eps": float("nan")}, {"H": 65537}):
        assert call(**bad) == N.ERR_SHAPE, bad
    assert call(q=None) == N.ERR_ALIGN and call(q=18) == N.ERR_ALIGN and call(w=18) == N.ERR_ALIGN

    def back(ws=16, nbytes=1 << 20, dw=16, g=16, D=8):
        return N.lib().rfdetr_normed_rotary_backward(
            None, 16, 16, 8, 16, 8, 8, g, 16, 8, 16, 8, 8, 0, 16, 0, None, 0, 1e-6, 16, 0, 16, N.int64_array((2, 2)), 2, 16,
            16, dw, None, ws, nbytes, 4, 2, 1, D, 0)

    assert back(ws=None) == N.ERR_WORKSPACE and back(nbytes=16) == N.ERR_WORKSPACE
    assert back(g=None) == N.ERR_ALIGN and back(dw=18) == N.ERR_ALIGN
    size = N.lib().rfdetr_normed_rotary_backward_workspace_bytes
    assert size(64) > 0 and size(128) == 2 * size(64) and size(1) == 0 and size(300) == 0


def test_clip_arguments(pkg):
    N = pkg._native

    def call(ins=(16,), outs=(16,), types=(0,), out_types=(0,), counts=(4,), limit=1.0, norm=16, ws=16, nbytes=1 << 24):
        p = lambda t, v: (t * len(v))(*v)  # noqa: E731
        return N.lib().rfdetr_clip_gradients(None, p(ctypes.c_void_p, ins), p(ctypes.c_int32, types),
                                             p(ctypes.c_void_p, outs), p(ctypes.c_int32, out_types),
                                             p(ctypes.c_int64, counts), len(ins), limit, norm, ws, nbytes)

    assert call(limit=-1.0) == N.ERR_SHAPE and call(limit=float("nan")) == N.ERR_SHAPE
    assert call(counts=(-1,)) == N.ERR_SHAPE and call(counts=(1 << 41,)) == N.ERR_SHAPE
    assert call(types=(7,)) == N.ERR_DTYPE and call(out_types=(2,)) == N.ERR_DTYPE
    assert call(out_types=(1,)) == N.ERR_DTYPE  # in place, of another type
    assert call(ins=(None,)) == N.ERR_ALIGN and call(ins=(18,)) == N.ERR_ALIGN and call(outs=(18,)) == N.ERR_ALIGN
    assert call(norm=None) == N.ERR_ALIGN
    assert call(ws=None) == N.ERR_WORKSPACE and call(nbytes=64) == N.ERR_WORKSPACE and call(ws=20) == N.ERR_WORKSPACE
    size = N.lib().rfdetr_clip_gradients_workspace_bytes
    assert 0 < size(1) == size(999) < size(5000) and size(-1) == 0


def test_cpu_tensors_are_refused(pkg):
    x, off = torch.zeros((4, 2, 64), dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    for call in (lambda: pkg.packed_attention(x, x, x, off, score_cap=3.0),
                 lambda: pkg.normed_axial_rotary(x, x, torch.zeros((4, 1)), torch.zeros(2), (2,)),
                 lambda: pkg.clip_gradients([x], 1.0), lambda: pkg.GradientClipper(x)):
        with pytest.raises(ValueError, match="CUDA tensors"):
            call()


def test_another_device_is_made_current(pkg, monkeypatch):
    """A launch on a stream of a device that is not the current one fails: the call goes through a guard."""
    N = pkg._native
    order = []

    class Guard:
        def __init__(self, device):
            order.append(("device", device))

        def __enter__(self):
            order.append("in")

        def __exit__(self, *exc):
            order.append("out")

    class Fake:
        device = "the tensor's"

        def get_device(self):
            return 1

    monkeypatch.setattr(N.torch.cuda, "device", Guard)
    monkeypatch.setattr(N, "_current_device", lambda: 0)
    assert N.on_device(Fake(), lambda x: order.append(x) or 7, "call") == 7
    assert order == [("device", "the tensor's"), "in", "call", "out"]
    order.clear()
    monkeypatch.setattr(N, "_current_device", lambda: 1)
    N.on_device(Fake(), order.append, "call")
    assert order == ["call"]


def test_a_prefix_needs_a_causal_mask(pkg):
    """As the Python function says: without a mask every query sees all keys, and a prefix would be ignored."""
    N = pkg._native
    assert _scored(N, T=0, causal=0) == N.ERR_SHAPE and _scored(N, T=0, causal=0, prefix=None) == N.OK
    back = lambda causal, prefix: N.lib().rfdetr_packed_attention_scored_backward(  # noqa: E731
        None, 16, 128, 64, 16, 128, 64, 16, 128, 64, 16, None, 16, 16, 16, 16, 128, 64, None, 16, 16, 16, None, 0,
        1, 4, 4, 2, 2, 64, causal, 0.1, 30.0, None, prefix)
    assert back(0, 16) == N.ERR_SHAPE and back(1, 16) == back(0, None) == N.ERR_WORKSPACE
