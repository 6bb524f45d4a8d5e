"""Rows of a table by token, scaled, and the table's gradient by sorted tokens: the input side of the table that
``token_log_probs`` and ``MemoryEfficientDistillLoss`` score features against.  Not part of the reference.

``embed_tokens(tokens, table, scale=1.0)`` is ``scale * table[tokens]``; the gradient of the table is dense, in the
table's dtype, summed in fp32 in ascending order of position, so it is the same from run to run.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _EmbedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale):
        ctx.save_for_backward(tokens)
        ctx.embed = (table.shape, scale)
        return ops.embed(tokens, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        (tokens,) = ctx.saved_tensors
        shape, scale = ctx.embed
        return None, ops.embed_grad(tokens, grad_output, shape[0], scale), None


def embed_tokens(tokens, table, scale=1.0):
    """scale * table[tokens], of shape tokens.shape + [D] in the table's dtype (rounded once).

    tokens: any shape, int64 or int32; a negative token is padding: its row is zero and it gets no gradient.  A token
    behind the table gives a row of NaN and gets none either.  table: [V, D] float32, bfloat16 or float16, any D, pitch and alignment.
    """
    ops._check_matrix(table, "table")
    assert tokens.get_device() == table.get_device(), "tokens and table must be on one device"
    assert tokens.dtype in (torch.int64, torch.int32), f"tokens: dtype {tokens.dtype} not supported (int64 or int32)"
    assert not isinstance(scale, torch.Tensor) and math.isfinite(scale), "scale must be a finite Python number"
    tokens = tokens if tokens.dtype == torch.int64 else tokens.to(torch.int64)
    tokens = tokens if tokens.is_contiguous() else tokens.contiguous()
    table = ops.row_major(table)
    if (table.requires_grad and torch.is_grad_enabled()) or ops.has_tangent(table):
        return _EmbedFn.apply(tokens, table, float(scale))
    return ops.embed(tokens, table, float(scale))
