"""Differentiable forms of the operators that keep a training step small: layer norm of any width, a linear map and a
layer norm whose input is kept in 8 bits for the backward pass, and the loss of a linear classifier over many classes.

``checkpoint_bits``: 32 keeps the input itself (as the reference's autograd graph does), 8 its 8-bit checkpoint
(``supergnn_ops.checkpoint_pack_rows``): the forward results are the same, the gradients are those of the restored
input where the formula asks for it.  Nothing is kept, and no gradient computed with a loss, where no backward pass can
follow (under ``torch.no_grad()``, or when no argument requires a gradient).
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .. import supergnn_ops as ops


def check_bits(checkpoint_bits) -> int:
    if checkpoint_bits not in (8, 32):
        raise ValueError(f"checkpoint_bits must be 8 or 32, got {checkpoint_bits}")
    return int(checkpoint_bits)


def _backward_can_follow(*tensors) -> bool:
    """Asked before ``apply``: a parameter's ``needs_input_grad`` stays true inside it when gradients are off."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, bits):
        ctx.bits, ctx.has_bias = bits, bias is not None
        if bits == 8:
            y, stats, codes, params = ops.layer_norm_forward(x, weight, bias, eps, checkpoint=True)
            ctx.save_for_backward(stats, weight, codes, params)
        else:
            y, stats = ops.layer_norm_forward(x, weight, bias, eps)
            ctx.save_for_backward(stats, weight, x)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        stats, weight, *kept = ctx.saved_tensors
        if ctx.bits == 8:
            gx, g_weight, g_bias = ops.layer_norm_backward_checkpoint(gy, *kept, stats, weight)
        else:
            gx, g_weight, g_bias = ops.layer_norm_backward(gy, *kept, stats, weight)
        return gx, g_weight if weight is not None else None, g_bias if ctx.has_bias else None, None, None


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, checkpoint_bits: int = 32):
    """Layer norm over the last dimension of a CUDA tensor (fp32, bf16 or fp16); weight and bias fp32 or of x's type,
    or None."""
    bits, rows = check_bits(checkpoint_bits), x.reshape(-1, x.size(-1))
    if _backward_can_follow(x, weight, bias):
        y = _LayerNorm.apply(rows, weight, bias, float(eps), bits)
    else:
        y = ops.layer_norm_forward(rows, weight, bias, float(eps))[0]
    return y.reshape(x.shape)


class _CheckpointLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight):
        ctx.save_for_backward(weight, *ops.checkpoint_pack_rows(x))
        return F.linear(x, weight)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        weight, codes, params = ctx.saved_tensors
        gx = g @ weight if ctx.needs_input_grad[0] else None
        gw = ops.checkpoint_weight_grad(g, codes, params).to(weight.dtype) if ctx.needs_input_grad[1] else None
        return gx, gw


def linear(x, weight, checkpoint_bits: int = 32):
    """``x @ weight.T`` for ``x`` [n, K]; with ``checkpoint_bits=8`` the weight gradient is taken from the 8-bit
    checkpoint of ``x``, and ``x`` itself is not kept."""
    if check_bits(checkpoint_bits) == 32 or not _backward_can_follow(x, weight):
        return F.linear(x, weight)
    return _CheckpointLinear.apply(x, weight)


class _LinearNLL(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, labels, mask, inv_count):
        loss, gx, gw, gb = ops.linear_nll_loss_grad(x, weight, bias, labels, mask, inv_count)
        ctx.save_for_backward(gx, gw, gb)
        return loss.reshape(())

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        gx, gw, gb = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (gx * g if need[0] else None, gw * g if need[1] else None,
                gb * g if need[2] and gb is not None else None, None, None, None)


def linear_nll_loss(x, weight, bias, labels, mask, inv_count: float):
    """``-sum_{mask} log_softmax(x @ weight.T + bias)[r, labels[r]] * inv_count`` as a differentiable scalar, without the
    logits in memory (``supergnn_ops.linear_nll_loss_grad``); the gradients are computed with the loss."""
    if not _backward_can_follow(x, weight, bias):
        return ops.linear_nll_loss(x, weight, bias, labels, mask, float(inv_count))[0].reshape(())
    return _LinearNLL.apply(x, weight, bias, labels, mask, float(inv_count))
