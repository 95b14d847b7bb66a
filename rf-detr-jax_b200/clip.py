"""The norm of all gradients together, and their clipping to a limit of it, on B200.

For the training step, between the gradients' all-reduce (:class:`.collective.PeerAllReduce`) and the
optimizer: two launches for up to a thousand tensors, no synchronisation, no copy of pointers to the device.
"""

from __future__ import annotations

from array import array
from operator import attrgetter

import torch

from . import _native as N

_CODES = {torch.float32: N.F32, torch.bfloat16: N.BF16}

# What a call asks every tensor, as functions to map: a third less of its time than in comprehensions.
_device, _count, _place = torch.Tensor.get_device, torch.Tensor.numel, torch.Tensor.data_ptr
_dtype, _leaf, _whole = attrgetter("dtype"), attrgetter("requires_grad"), torch.Tensor.is_contiguous


def _is_dense(t: torch.Tensor) -> bool:
    """Whether the values fill a range of memory without gaps or repeats, in whatever order of axes."""
    return t.is_contiguous() or t.permute(sorted(range(t.dim()), key=t.stride, reverse=True)).is_contiguous()


def _types(name: str, tensors) -> array:
    found = set(map(_dtype, tensors))
    if not found <= _CODES.keys():
        raise ValueError(f"{name} must be float32 or bfloat16, got {sorted(map(str, found))}")
    if len(found) == 1:
        return array("i", [_CODES[found.pop()]]) * len(tensors)
    return array("i", [_CODES[t.dtype] for t in tensors])


def _list(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


class GradientClipper:
    """:func:`clip_gradients` for tensors that stay: checks and lays out a program's gradient buffers (and those that
    the results go to) once, so that a step's call does not look at every tensor again.

    The clipper keeps the tensors; each must keep its memory (be written in place, as the views of a flat buffer are,
    or a captured graph's gradients).  ``out`` as for :func:`clip_gradients`; the gradients have to be contiguous with
    it.
    """

    def __init__(self, gradients, out=None):
        tensors = _list(gradients)
        if not tensors:
            raise ValueError("there is no gradient to clip")
        device = tensors[0].get_device()
        if device < 0 or set(map(_device, tensors)) != {device}:
            N.require_cuda(*tensors)
        self._types = self._out_types = _types("gradients", tensors)
        self._counts = array("q", list(map(_count, tensors)))
        if out is None:
            outs = tensors
            if not all(map(_is_dense, tensors)):
                raise ValueError("gradients that are clipped in place must fill their memory: pass out")
        else:
            outs = _list(out)
            if not set(map(_device, outs)) <= {device}:
                raise ValueError("all tensors must be on the same device")
            self._out_types = _types("out", outs)
            if array("q", list(map(_count, outs))) != self._counts:
                raise ValueError("out must have as many values as the gradients, tensor by tensor")
            if not all(map(_whole, tensors)) or not all(map(_whole, outs)):
                raise ValueError("gradients and out must be contiguous")
        if torch.is_grad_enabled() and (any(map(_leaf, tensors)) or any(map(_leaf, outs))):
            raise ValueError("clipping is not differentiable: gradients and out must need no gradient")
        self._from = self._to = array("q", list(map(_place, tensors)))
        if out is not None:
            self._to = array("q", list(map(_place, outs)))
        if len(set(self._to)) < len(outs):
            places = [p for p, n in zip(self._to, self._counts) if n]
            if len(set(places)) < len(places):
                raise ValueError("a tensor is given twice")
        self._tensors, self._outs = tensors, outs
        self._written = None

    def clip(self, max_norm: float) -> torch.Tensor:
        """One step's clipping, on the current stream; returns the norm before it."""
        max_norm = float(max_norm)
        if not max_norm >= 0.0:
            raise ValueError(f"max_norm must not be negative, got {max_norm}")
        if self._written is None:  # views of a tensor count its writes together
            self._written = list({id(t): t for t in (t if t._base is None else t._base for t in self._outs)}.values())
        return self._launch(max_norm, self._written)

    def _launch(self, max_norm, written):
        first, lib, count = self._tensors[0], N.lib(), len(self._counts)
        ws_bytes = lib.rfdetr_clip_gradients_workspace_bytes(count)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=first.device)
        norm = torch.empty((), dtype=torch.float32, device=first.device)
        status = N.on_device(first, lib.rfdetr_clip_gradients, N.stream_of(first), self._from.buffer_info()[0],
                             self._types.buffer_info()[0], self._to.buffer_info()[0],
                             self._out_types.buffer_info()[0], self._counts.buffer_info()[0], count, max_norm,
                             norm.data_ptr(), workspace.data_ptr(), ws_bytes)
        if status:
            N.check(status, "rfdetr_clip_gradients")
        torch.autograd.graph.increment_version(written)
        return norm


def clip_gradients(gradients, max_norm: float, *, out=None) -> torch.Tensor:
    """Scales gradients so that their norm, taken over all values of all of them, is at most ``max_norm``.

    Args:
        gradients: a tensor or a sequence of them, float32 or bfloat16, on one device.  Views of a flat buffer, at
            any place, pass as they are.
        max_norm: the limit, not negative; ``inf`` for the norm alone.
        out: where the results go: None for the gradients themselves, or tensors with as many values each, contiguous,
            float32 or bfloat16 (bfloat16 gradients clipped into float32 ones, for instance).  They may be the
            gradients themselves; results that share memory with one another, or with a gradient otherwise, are refused.

    Returns:
        The norm before clipping, a float32 scalar on the device.  Where it is ``max_norm`` at most the values stay
        as they are; otherwise each is multiplied by ``max_norm / norm``.  A NaN among the gradients makes all
        results NaN; an infinite one makes itself NaN and the finite ones 0.  Squares and their sum are float64.
        Not differentiable.  (Looking at each tensor is most of a call's time on the host: a program whose
        tensors stay keeps a :class:`GradientClipper`.)
    """
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    if out is not None:
        gradients = list(map(torch.Tensor.contiguous, _list(gradients)))
    clipper = GradientClipper(gradients, out)
    return clipper._launch(max_norm, clipper._outs)
