"""Rotary positions with several axes on B200: queries and keys turned in one launch.

For attention over image or video tokens whose place is told by angles (time, height, width), next
to :func:`.attention.packed_attention`.  The gradient is the inverse turn, by the same kernel.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native as N


_POSITION_CODES = {torch.float32: N.F32, torch.int32: N.I32, torch.int64: N.I64}


def _rows(name: str, t: torch.Tensor) -> torch.Tensor:
    strides = t.stride()
    if len(strides) != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {list(t.shape)}")
    return t if strides[2] == 1 else t.contiguous()


def _pairs(t: torch.Tensor) -> torch.Tensor:
    """Interleaved pairs are read as one: aligned to a pair, or copied."""
    token, head, _ = t.stride()
    if (token | head) & 1 or t.data_ptr() % (2 * t.element_size()):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def rotary_launch(query, key, positions, inv_freq, sections, interleaved, inverse):
    """One launch over checked inputs; ``key`` may be None."""
    tokens, heads, dim = query.shape
    if interleaved:
        query, key = _pairs(query), None if key is None else _pairs(key)
    out = query.new_empty(tokens, heads, dim)
    key_out, kv_heads, key_strides = None, 0, (0, 0)
    if key is not None:
        kv_heads, key_strides = key.shape[1], key.stride()[:2]
        key_out = key.new_empty(tokens, kv_heads, dim)
    status = N.lib().rfdetr_axial_rotary(
        N.stream_of(query), query.data_ptr(), *query.stride()[:2], N.ptr(key), *key_strides,
        N.dtype_code(query.dtype), positions.data_ptr(), _POSITION_CODES[positions.dtype],
        inv_freq.data_ptr(), N.const_int64_array(sections), len(sections), out.data_ptr(), N.ptr(key_out), tokens, heads,
        kv_heads, dim, interleaved, inverse)
    if status:
        N.check(status, "rfdetr_axial_rotary")
    return out, key_out


class AxialRotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, positions, inv_freq, sections, interleaved):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = (sections, interleaved)
        return rotary_launch(query, key, positions, inv_freq, sections, interleaved, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_query, grad_key):
        positions, inv_freq = ctx.saved_tensors
        grads = rotary_launch(_rows("grad_query", grad_query), None if grad_key is None else _rows("grad_key", grad_key),
                              positions, inv_freq, *ctx.how, True)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None, None)


def axial_rotary(query: torch.Tensor, key: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor,
                 sections, *, interleaved: bool = False):
    """Turns the channels of queries and keys by their tokens' positions.

    Args:
        query, key: ``[tokens, heads, head_dim]`` and ``[tokens, kv_heads, head_dim]`` float32 or
            bfloat16 (views of a fused projection are read in place); ``key`` may be None.
        positions: ``[tokens, axes]`` float32, int32 or int64.
        inv_freq: ``[sum(sections)]`` float32, radians per unit of position.
        sections: frequencies per axis, in order; ``2 * sum(sections) <= head_dim`` and the channels
            beyond are copied.
        interleaved: pairs of channels ``(2i, 2i + 1)`` instead of ``(i, i + sum(sections))``.

    Returns:
        ``(query, key)`` turned, contiguous, in their own type; differentiable (in reverse mode) with
        respect to both (not to the positions or frequencies).
    """
    N.same_device(query, key, positions, inv_freq)
    query = _rows("query", query)
    tokens, _, dim = query.shape
    if query.dtype != torch.float32 and query.dtype != torch.bfloat16:
        raise ValueError(f"query must be float32 or bfloat16, got {query.dtype}")
    if key is not None:
        key = _rows("key", key)
        if key.shape[0] != tokens or key.shape[2] != dim or key.dtype != query.dtype:
            raise ValueError("key must have the query's tokens, head_dim and type")
    sections = tuple(map(int, sections))
    half = sum(sections)
    if not 1 <= len(sections) <= 8 or min(sections) < 0 or half < 1 or 2 * half > dim:
        raise ValueError(f"sections {sections} do not fit head_dim {dim}")
    if positions.shape != (tokens, len(sections)):
        raise ValueError(f"positions must be [{tokens}, {len(sections)}], got {list(positions.shape)}")
    if positions.dtype not in _POSITION_CODES:
        raise ValueError(f"positions must be float32, int32 or int64, got {positions.dtype}")
    if inv_freq.shape != (half,) or inv_freq.dtype != torch.float32:
        raise ValueError(f"inv_freq must be float32 [{half}]")
    if torch.is_grad_enabled() and (positions.requires_grad or inv_freq.requires_grad):
        raise ValueError("positions and inv_freq have no gradient")
    if dim > 1024:
        raise ValueError(f"head_dim must be at most 1024, got {dim}")
    if interleaved and dim % 2:
        raise ValueError("interleaved pairs need an even head_dim")
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    if ((torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad)))
            or N.has_tangent(query, key, positions, inv_freq)):
        return AxialRotaryFunction.apply(query, key, positions, inv_freq, sections, bool(interleaved))
    return rotary_launch(query, key, positions, inv_freq, sections, bool(interleaved), False)
