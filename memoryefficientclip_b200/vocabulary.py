"""Softmax over a vocabulary with O((N + V) * D) memory on B200: scores of features against a table of V rows,

    z_ij = <x_i, y_j> / T,    p_ij = exp(z_ij) / sum_j exp(z_ij),

whose N x V matrix is never stored.  Not part of the reference (which has the contrastive losses only); it runs on the
same tile kernels.

``token_log_probs(features, table, tokens, temperature=1.0, top_k=0)`` gives the log probabilities of given tokens, the
entropy of every row and its top alternatives; gradients flow to the features and the table through the first two.
``MemoryEfficientDistillLoss(temperature, normalized_inputs, teacher_temperature, reduction)`` is the KL divergence from
a teacher that is known by its top logits; ``MemoryEfficientDistillLossFn.apply`` is its autograd node.

Features [N, D] and table [V, D]: float32, bfloat16 or float16 with any D, pitch and alignment.  Two float16 inputs are
scored as they are; otherwise, and wherever inputs are normalised inside, the operands are bf16 (rounded as in the
contrastive losses; there is no tf32 route, MECLIP_TF32 does not count here).  All sums are fp32, gradients come back in the
inputs' dtypes, there are no second or forward-mode derivatives.  Features and table must be finite: a row of NaN gives
NaN for that row, and NaN gradients for the table.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import ops

MAX_ENTRIES = 256       # given tokens or teacher entries per row
MAX_TOP = 32            # top alternatives per row


class TokenLogProbs(NamedTuple):
    """log_probs: shape of `tokens`; entropy [N]; top_log_probs, top_tokens [N, top_k] (None without top_k)."""
    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def _check_inputs(features, table, temperature):
    ops._check_matrix(features, "features")
    ops._check_matrix(table, "table")
    assert features.get_device() == table.get_device(), "features and table must be on one device"
    assert features.shape[1] == table.shape[1], \
        f"features have {features.shape[1]} columns, the table has {table.shape[1]}"
    assert not isinstance(temperature, torch.Tensor), "the temperature of a vocabulary softmax is a Python number"
    assert 0.0 < temperature < math.inf, "temperature must be positive"


def _check_tokens(tokens, features, name):
    """The tokens as contiguous int64."""
    assert tokens.get_device() == features.get_device(), f"{name} must be on the features' device"
    assert tokens.dtype in (torch.int64, torch.int32), f"{name}: dtype {tokens.dtype} not supported (int64 or int32)"
    assert tokens.dim() in (1, 2) and tokens.shape[0] == features.shape[0], \
        f"{name} must be [{features.shape[0]}] or [{features.shape[0]}, k]"
    assert tokens.dim() == 1 or 1 <= tokens.shape[1] <= MAX_ENTRIES, f"{name}: 1 to {MAX_ENTRIES} entries per row"
    tokens = tokens if tokens.dtype == torch.int64 else tokens.to(torch.int64)
    return tokens if tokens.is_contiguous() else tokens.contiguous()


def _grad_dtype(dtype, d):
    """(dtype the contraction writes, whether a conversion follows) for an input of this dtype and width."""
    return (dtype, False) if ops.direct_grad_dtype(dtype, d) else (torch.float32, True)


def _f32(g):
    """An incoming gradient as contiguous fp32."""
    if g is None or (g.dtype == torch.float32 and g.is_contiguous()):
        return g
    return g.to(torch.float32).contiguous()


class _TokenLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, table, tokens, temperature, top_k):
        status = ops.status_word(features.device)
        x, y = ops.vocab_operands(features, table)
        lp, entropy, top_lp, top, saved = ops.token_log_probs(x, y, tokens, temperature, top_k, True, status)
        ctx.save_for_backward(x, y, tokens, entropy, saved)
        ctx.vocab = (temperature, features.dtype, table.dtype, features.shape[1])
        ctx.set_materialize_grads(False)
        if top_k:
            ctx.mark_non_differentiable(top_lp, top)
        return lp, entropy, top_lp, top

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_log_probs, grad_entropy, _top_lp, _top):
        x, y, tokens, entropy, saved = ctx.saved_tensors
        temperature, x_dtype, y_dtype, d = ctx.vocab
        need = ctx.needs_input_grad
        if (grad_log_probs is None and grad_entropy is None) or not (need[0] or need[1]):
            return None, None, None, None, None
        dx_t, post_x = _grad_dtype(x_dtype, d)
        dy_t, post_y = _grad_dtype(y_dtype, d)
        dx, dy = ops.token_log_probs_grad(x, y, tokens, temperature, saved, entropy, _f32(grad_log_probs),
                                          _f32(grad_entropy), dx_t, dy_t, need[0], need[1], ops.status_word(x.device))
        if dx is not None and post_x:
            dx = ops.normalize_bwd(dx, None, None, x_dtype, d)
        if dy is not None and post_y:
            dy = ops.normalize_bwd(dy, None, None, y_dtype, d)
        ops.post_status(x.device)
        return dx, dy, None, None, None


def token_log_probs(features, table, tokens, temperature=1.0, top_k=0) -> TokenLogProbs:
    """Log probabilities of given tokens under softmax(features @ table^T / temperature).

    tokens: [N], or [N, k] with k up to 256 tokens per row, int64 or int32.  A negative token is absent: its log
    probability is 0 and it gets no gradient.  A token behind the table gives NaN and gets none either.
    top_k: 0 to 32 alternatives per row, best first; of equal scores the lower token comes first.  They carry no gradient.
    The order is that of exact scores unless a table row more than twice as long as the best one is among the close ones.
    """
    _check_inputs(features, table, temperature)
    tokens = _check_tokens(tokens, features, "tokens")
    assert isinstance(top_k, int) and 0 <= top_k <= min(MAX_TOP, table.shape[0]), \
        f"top_k must be between 0 and {min(MAX_TOP, table.shape[0])}"
    device = features.device
    ops.poll_status(device)
    if ((features.requires_grad or table.requires_grad) and torch.is_grad_enabled()) or ops.has_tangent(features, table):
        return TokenLogProbs(*_TokenLogProbsFn.apply(features, table, tokens, float(temperature), top_k))
    x, y = ops.vocab_operands(features, table)
    lp, entropy, top_lp, top, _saved = ops.token_log_probs(x, y, tokens, float(temperature), top_k, False,
                                                           ops.status_word(device))
    ops.post_status(device)
    return TokenLogProbs(lp, entropy, top_lp, top)


class MemoryEfficientDistillLossFn(torch.autograd.Function):
    """apply(features, table, teacher_tokens, teacher_logits, temperature, teacher_temperature, reduction, normalize)."""

    @staticmethod
    def forward(ctx, features, table, teacher_tokens, teacher_logits, temperature, teacher_temperature, reduction,
                normalize):
        _check_inputs(features, table, temperature)
        tokens = _check_tokens(teacher_tokens, features, "teacher_tokens")
        assert teacher_tokens.shape == teacher_logits.shape, "teacher_tokens and teacher_logits must have one shape"
        assert teacher_logits.device == features.device, "teacher_logits must be on the features' device"
        assert teacher_logits.dtype in ops._DT, f"teacher_logits: dtype {teacher_logits.dtype} not supported"
        assert not isinstance(teacher_temperature, torch.Tensor) and 0.0 < teacher_temperature < math.inf, \
            "teacher_temperature must be a positive Python number"
        assert reduction in ("mean", "sum", "none"), f"unknown reduction {reduction!r}"
        status = ops.status_word(features.device)
        ops.poll_status(features.device)
        inv_x = inv_y = None
        if normalize:
            x, inv_x = ops.normalize_fwd(features, True)
            y, inv_y = ops.normalize_fwd(table, True)
        else:
            x, y = ops.vocab_operands(features, table)
        result, saved = ops.distill_forward(x, y, tokens, teacher_logits.contiguous(), float(temperature),
                                            float(teacher_temperature), reduction, status)
        if not any(ctx.needs_input_grad[:2]):
            ops.post_status(features.device)
        ctx.save_for_backward(x, y, tokens, saved, inv_x, inv_y)
        ctx.vocab = (float(temperature), features.dtype, table.dtype, features.shape[1])
        return result

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        x, y, tokens, saved, inv_x, inv_y = ctx.saved_tensors
        temperature, x_dtype, y_dtype, d = ctx.vocab
        need = ctx.needs_input_grad
        if inv_x is None:
            dx_t, post_x = _grad_dtype(x_dtype, d)
            dy_t, post_y = _grad_dtype(y_dtype, d)
        else:                       # the Jacobian of the normalisation follows: fp32 until it rounds once
            dx_t, post_x, dy_t, post_y = torch.float32, True, torch.float32, True
        dx, dy = ops.distill_backward(x, y, tokens, temperature, saved, _f32(grad_output), dx_t, dy_t, need[0], need[1],
                                      ops.status_word(x.device))
        if dx is not None and post_x:
            dx = ops.normalize_bwd(dx, x if inv_x is not None else None, inv_x, x_dtype, d)
        if dy is not None and post_y:
            dy = ops.normalize_bwd(dy, y if inv_y is not None else None, inv_y, y_dtype, d)
        ops.post_status(x.device)
        return dx, dy, None, None, None, None, None, None


class MemoryEfficientDistillLoss(nn.Module):
    """KL(teacher || student) for a teacher that is known by the top entries of each row.

    The student's distribution is softmax(features @ table^T / temperature) over all rows of the table, the teacher's
    softmax(teacher_logits / teacher_temperature) over the entries that are present in the row.  ``forward(features,
    table, teacher_tokens, teacher_logits)``: teacher_tokens [N, k] (k up to 256, int64 or int32) name rows of the table,
    teacher_logits [N, k] are their logits (float32, bfloat16 or float16; no gradient).  An entry with a negative token or
    a logit of -inf is absent, whatever else stands in its place (the lowest finite value is a logit like any other); a row
    without entries adds nothing and gets no gradient; an entry counts by itself where a row names a token twice.
    reduction: "mean" over the rows that have entries, "sum", or "none" for the [N] losses.  With normalized_inputs=False features and table are L2-normalised inside, as in the contrastive
    losses: the table is then the other tower's output and the teacher's entries its best pairs.
    """

    def __init__(self, temperature=0.07, normalized_inputs=False, teacher_temperature=1.0, reduction="mean"):
        super().__init__()
        self.temperature = temperature
        self.normalized_inputs = normalized_inputs
        self.teacher_temperature = teacher_temperature
        self.reduction = reduction

    def forward(self, features, table, teacher_tokens, teacher_logits):
        return MemoryEfficientDistillLossFn.apply(features, table, teacher_tokens, teacher_logits, self.temperature,
                                                  self.teacher_temperature, self.reduction, not self.normalized_inputs)
