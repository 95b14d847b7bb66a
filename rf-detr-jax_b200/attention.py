"""Softmax attention over packed sequences on B200, forward and backward on the tensor cores.

The decoder's grouped self-attention (every detection group of queries attends within itself) and
the backbone's windows, or images of unequal size, are sequences of different lengths in one
packed tensor; the reference computes them as padded batches
(``src/rfdetr_jax/models/layers.py:54-98``).  :func:`packed_attention` takes the rows of all
sequences and their offsets, with grouped heads and an optional causal mask.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native as N


def _packed(name: str, t: torch.Tensor) -> torch.Tensor:
    """Checks ``[tokens, heads, dim]`` bf16 and returns it with strides the kernels take (a view of
    a fused projection passes as it is; anything else is made contiguous)."""
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
    strides = t.stride()
    if len(strides) != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {list(t.shape)}")
    token, head, channel = strides
    if channel != 1 or token <= 0 or head <= 0 or (token | head) & 7 or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _offsets(name: str, t: torch.Tensor) -> torch.Tensor:
    dtype = t.dtype
    if t.dim() != 1 or t.numel() < 1 or (dtype != torch.int32 and dtype != torch.int64):
        raise ValueError(f"{name} must be int32 [sequences + 1]")
    if dtype == torch.int64:  # clamped like any others, to the tensors by the kernels
        return t.clamp(0, 0x7fffffff).to(torch.int32).contiguous()
    return t.contiguous()


def _check_offsets(name: str, t: torch.Tensor, total: int) -> None:
    """Reads the offsets on the host (synchronises)."""
    values = t.tolist()
    if values[0] < 0 or values[-1] > total or any(b < a for a, b in zip(values, values[1:])):
        raise ValueError(f"{name} must ascend within [0, {total}]")


def attention_forward(query, key, value, offsets, key_offsets, causal, scale, want_lse, want_low):
    """One forward call; inputs already checked.  Returns ``(output, lse or None, low or None)``, low being
    what the output lost in its rounding to bf16 (the backward pass reads it)."""
    tokens, heads, dim = query.shape
    key_tokens, kv_heads, _ = key.shape
    sequences = offsets.numel() - 1
    out = query.new_empty(tokens, heads, dim)
    lse = query.new_empty(heads, tokens, dtype=torch.float32) if want_lse else None
    low = query.new_empty(tokens, heads, dim) if want_low else None
    lib = N.lib()
    ws_bytes = lib.rfdetr_packed_attention_workspace_bytes(sequences, tokens, key_tokens, heads, kv_heads, dim)
    workspace = query.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    status = lib.rfdetr_packed_attention(
        N.stream_of(query), query.data_ptr(), *query.stride()[:2], key.data_ptr(), *key.stride()[:2],
        value.data_ptr(), *value.stride()[:2], offsets.data_ptr(), N.ptr(key_offsets),
        out.data_ptr(), N.ptr(low), N.ptr(lse), N.ptr(workspace), ws_bytes, sequences, tokens, key_tokens, heads,
        kv_heads, dim, causal, scale)
    if status:
        N.check(status, "rfdetr_packed_attention")
    return out, lse, low


def attention_backward(query, key, value, offsets, key_offsets, causal, scale, out, low, lse, grad_output, grad_lse):
    """One backward call; returns ``(grad_query, grad_key, grad_value)``, contiguous."""
    tokens, heads, dim = query.shape
    key_tokens, kv_heads, _ = key.shape
    grad_output = _packed("grad_output", grad_output.to(query.dtype))
    if grad_lse is not None:
        grad_lse = grad_lse.to(torch.float32).contiguous()
    grads = query.new_empty(tokens, heads, dim), key.new_empty(key.shape), value.new_empty(key.shape)
    lib = N.lib()
    ws_bytes = lib.rfdetr_packed_attention_backward_workspace_bytes(tokens, heads)
    workspace = query.new_empty(max(1, ws_bytes), dtype=torch.uint8)
    status = lib.rfdetr_packed_attention_backward(
        N.stream_of(query), query.data_ptr(), *query.stride()[:2], key.data_ptr(), *key.stride()[:2],
        value.data_ptr(), *value.stride()[:2], offsets.data_ptr(), N.ptr(key_offsets),
        out.data_ptr(), N.ptr(low), lse.data_ptr(), grad_output.data_ptr(), *grad_output.stride()[:2],
        N.ptr(grad_lse), grads[0].data_ptr(), grads[1].data_ptr(), grads[2].data_ptr(), workspace.data_ptr(), ws_bytes,
        offsets.numel() - 1, tokens, key_tokens, heads, kv_heads, dim, int(causal), scale)
    if status:
        N.check(status, "rfdetr_packed_attention_backward")
    return grads


class PackedAttentionFunction(torch.autograd.Function):
    """Forward keeps the output (and what its rounding lost) and the log-sum-exp; backward forms the weights
    again from them."""

    @staticmethod
    def forward(ctx, query, key, value, offsets, key_offsets, causal, scale):
        out, lse, low = attention_forward(query, key, value, offsets, key_offsets, causal, scale, True, True)
        ctx.save_for_backward(query, key, value, offsets, key_offsets, out, low, lse)
        ctx.how = (causal, scale)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output, grad_lse):
        query, key, value, offsets, key_offsets, out, low, lse = ctx.saved_tensors
        if grad_output is None and grad_lse is None:
            return (None,) * 7
        if grad_output is None:
            grad_output = torch.zeros_like(out)
        grads = attention_backward(query, key, value, offsets, key_offsets, *ctx.how, out, low, lse, grad_output,
                                   grad_lse)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None, None)


def packed_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, offsets: torch.Tensor,
                     key_offsets: torch.Tensor | None = None, *, causal: bool = False, scale: float | None = None,
                     return_lse: bool = False, check: bool = False):
    """``softmax(scale * q k^T) v`` within each sequence of packed tensors.

    Args:
        query: ``[tokens, heads, head_dim]`` bfloat16, ``head_dim`` a multiple of 8 up to 128.  Views
            of a fused projection are read in place (channels contiguous, strides multiples of 8).
        key, value: ``[key_tokens, kv_heads, head_dim]``; head ``h`` reads key head
            ``h // (heads // kv_heads)``.
        offsets: int32 (or int64) ``[sequences + 1]`` on the device: sequence ``s`` is rows ``offsets[s]`` to
            ``offsets[s + 1] - 1`` of ``query``.
        key_offsets: the same for ``key`` and ``value``; None where they are the queries' own tokens.
        causal: query ``i`` of ``Lq`` sees keys ``j <= i + Lk - Lq`` (the last query sees all).
        scale: of the scores, positive; ``head_dim ** -0.5`` by default.
        return_lse: also return the scores' log-sum-exp ``[heads, tokens]`` float32.
        check: read the offsets on the host (synchronises) and raise ``ValueError`` unless they
            ascend within the tensors; otherwise the kernels clamp them.

    Returns:
        ``[tokens, heads, head_dim]`` bfloat16, differentiable (in reverse mode) with respect to query, key and
        value (and through the log-sum-exp).  A query without any key (or with all scores ``-inf``), and rows
        outside all sequences, give 0 (log-sum-exp ``-inf``) and gradient 0.
    """
    N.same_device(query, key, value, offsets, key_offsets)
    query, key, value = _packed("query", query), _packed("key", key), _packed("value", value)
    tokens, heads, dim = query.shape
    key_tokens, kv_heads, key_dim = key.shape
    if key_dim != dim or value.shape != key.shape:
        raise ValueError(f"key and value must be [key_tokens, kv_heads, {dim}], got {list(key.shape)} and "
                         f"{list(value.shape)}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads are not a multiple of {kv_heads} key heads")
    if dim % 8 or not 8 <= dim <= 128:
        raise ValueError(f"head_dim must be a multiple of 8 up to 128, got {dim}")
    if tokens > 1 << 30 or key_tokens > 1 << 30 or heads > 65536:
        raise ValueError("at most 2^30 tokens and 65536 heads")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale <= 3.4028234663852886e38:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    given, given_keys = offsets, key_offsets
    offsets = _offsets("offsets", offsets)
    if key_offsets is not None:
        key_offsets = _offsets("key_offsets", key_offsets)
        if key_offsets.numel() != offsets.numel():
            raise ValueError("offsets and key_offsets must have the same length")
    elif key_tokens != tokens:
        raise ValueError("key_offsets is needed where keys and queries are not the same tokens")
    if check:
        _check_offsets("offsets", given, tokens)
        if key_offsets is not None:
            _check_offsets("key_offsets", given_keys, key_tokens)
    if ((torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad))
            or N.has_tangent(query, key, value)):
        out, lse = PackedAttentionFunction.apply(query, key, value, offsets, key_offsets, bool(causal), scale)
    else:
        out, lse, _ = attention_forward(query, key, value, offsets, key_offsets, bool(causal), scale, return_lse,
                                        False)
    return (out, lse) if return_lse else out
