"""Norms of queries and keys for each head, with the rotary positions of their tokens, in one pass on B200.

For attention whose scores are kept in bounds by norming queries and keys (:func:`.attention.packed_attention`
reads the results): what :func:`.rotary.axial_rotary` does, after a root-mean-square norm.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .rotary import _POSITION_CODES, _rows


def _weight(name: str, w: torch.Tensor | None, dim: int) -> torch.Tensor | None:
    if w is None:
        return None
    if w.shape != (dim,) or (w.dtype != torch.float32 and w.dtype != torch.bfloat16):
        raise ValueError(f"{name} must be float32 or bfloat16 [{dim}], got {w.dtype} {list(w.shape)}")
    return w.contiguous()


def _weight_code(w: torch.Tensor | None) -> int:
    return N.F32 if w is None else N.dtype_code(w.dtype)


def normed_rotary_launch(query, key, query_weight, key_weight, positions, inv_freq, sections, interleaved, eps):
    """One launch over checked inputs; ``key`` may be None."""
    tokens, heads, dim = query.shape
    out = query.new_empty(tokens, heads, dim)
    key_out, kv_heads, key_strides = None, 0, (0, 0)
    if key is not None:
        kv_heads, key_strides = key.shape[1], key.stride()[:2]
        key_out = key.new_empty(tokens, kv_heads, dim)
    status = N.on_device(
        query, N.lib().rfdetr_normed_rotary, N.stream_of(query), query.data_ptr(), *query.stride()[:2], N.ptr(key),
        *key_strides, N.dtype_code(query.dtype), N.ptr(query_weight), _weight_code(query_weight), N.ptr(key_weight),
        _weight_code(key_weight), eps, positions.data_ptr(), _POSITION_CODES[positions.dtype], inv_freq.data_ptr(),
        N.const_int64_array(sections), len(sections), out.data_ptr(), N.ptr(key_out), tokens, heads, kv_heads, dim,
        interleaved)
    if status:
        N.check(status, "rfdetr_normed_rotary")
    return out, key_out


def normed_rotary_backward(query, key, query_weight, key_weight, positions, inv_freq, sections, interleaved, eps,
                           grad_query, grad_key, want_weights):
    """Gradients of query, key and (those of them that are wanted) of their weights."""
    tokens, heads, dim = query.shape
    grad_query = _rows("grad_query", grad_query)
    dq, dk, kv_heads, key_strides, grad_strides = query.new_empty(tokens, heads, dim), None, 0, (0, 0), (0, 0)
    if key is not None:
        grad_key = _rows("grad_key", grad_key)
        kv_heads, key_strides, grad_strides = key.shape[1], key.stride()[:2], grad_key.stride()[:2]
        dk = key.new_empty(tokens, kv_heads, dim)
    weights = [w.new_empty(dim) if want else None for w, want in zip((query_weight, key_weight), want_weights)]
    lib = N.lib()
    ws_bytes, workspace = 0, None
    if any(want_weights):
        ws_bytes = lib.rfdetr_normed_rotary_backward_workspace_bytes(dim)
        workspace = query.new_empty(ws_bytes, dtype=torch.uint8)
    status = N.on_device(
        query, lib.rfdetr_normed_rotary_backward, N.stream_of(query), query.data_ptr(), *query.stride()[:2],
        N.ptr(key), *key_strides, grad_query.data_ptr(), *grad_query.stride()[:2],
        N.ptr(grad_key) if key is not None else None, *grad_strides, N.dtype_code(query.dtype), N.ptr(query_weight),
        _weight_code(query_weight), N.ptr(key_weight), _weight_code(key_weight), eps, positions.data_ptr(),
        _POSITION_CODES[positions.dtype], inv_freq.data_ptr(), N.const_int64_array(sections), len(sections),
        dq.data_ptr(), N.ptr(dk), N.ptr(weights[0]), N.ptr(weights[1]), N.ptr(workspace), ws_bytes, tokens, heads,
        kv_heads, dim, interleaved)
    if status:
        N.check(status, "rfdetr_normed_rotary_backward")
    return dq, dk, *weights


class NormedRotaryFunction(torch.autograd.Function):
    """Keeps its inputs alone: backward forms the norms again."""

    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, positions, inv_freq, sections, interleaved, eps):
        ctx.save_for_backward(query, key, query_weight, key_weight, positions, inv_freq)
        ctx.how = (sections, interleaved, eps)
        return normed_rotary_launch(query, key, query_weight, key_weight, positions, inv_freq, sections, interleaved,
                                    eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_query, grad_key):
        need = ctx.needs_input_grad
        grads = normed_rotary_backward(*ctx.saved_tensors, *ctx.how, grad_query, grad_key, need[2:4])
        return (*(g if want else None for g, want in zip(grads, need)), None, None, None, None, None)


def normed_axial_rotary(query: torch.Tensor, key: torch.Tensor | None, positions: torch.Tensor,
                        inv_freq: torch.Tensor, sections, query_weight: torch.Tensor | None = None,
                        key_weight: torch.Tensor | None = None, *, eps: float = 1e-6, interleaved: bool = False):
    """Norms every head of queries and keys, ``x / sqrt(mean(x^2) + eps) * weight``, and turns it by its token's
    positions.

    Args:
        query, key: ``[tokens, heads, head_dim]`` and ``[tokens, kv_heads, head_dim]`` float32 or
            bfloat16 (views of a fused projection are read in place); ``key`` may be None.
            ``head_dim`` is 256 at most; what is a multiple of 16 bytes goes fastest.
        positions, inv_freq, sections, interleaved: as :func:`.rotary.axial_rotary` takes them.  The mean is over all of
            a head's channels, whether they are turned or not.
        query_weight, key_weight: ``[head_dim]`` float32 or bfloat16, shared by the heads; None for ones.
        eps: not negative.

    Returns:
        ``(query, key)``, contiguous, in their own type (rounded once, after the turn); differentiable (in reverse mode)
        with respect to both and to the weights (not to the positions or frequencies).
    """
    N.same_device(query, key, positions, inv_freq, query_weight, key_weight)
    query = _rows("query", query)
    tokens, _, dim = query.shape
    if query.dtype != torch.float32 and query.dtype != torch.bfloat16:
        raise ValueError(f"query must be float32 or bfloat16, got {query.dtype}")
    if key is not None:
        key = _rows("key", key)
        if key.shape[0] != tokens or key.shape[2] != dim or key.dtype != query.dtype:
            raise ValueError("key must have the query's tokens, head_dim and type")
    elif key_weight is not None:
        raise ValueError("key_weight needs a key")
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
    if dim > 256:
        raise ValueError(f"head_dim must be at most 256, got {dim}")
    if query.shape[1] > 65536 or (key is not None and key.shape[1] > 65536):
        raise ValueError("at most 65536 heads")
    eps = float(eps)
    if not 0.0 <= eps <= 3.4028234663852886e38:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    query_weight, key_weight = _weight("query_weight", query_weight, dim), _weight("key_weight", key_weight, dim)
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    inputs = (query, key, query_weight, key_weight, positions, inv_freq, sections, bool(interleaved), eps)
    if ((torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in inputs[:4]]))
            or N.has_tangent(*inputs[:6])):
        return NormedRotaryFunction.apply(*inputs)
    return normed_rotary_launch(*inputs)
