"""Nearest-code lookup with the reference's call signatures
(reference src/inverter/utils_vq_vae/util_function.py), computed by the HIP library.

Forward only: the reference wraps these in ``torch.autograd.Function`` for VQ-VAE training
(straight-through gradient, codebook gradient); training is outside the PSO path, so the
results carry no autograd graph.  The soft assignment (``code_logits``) and the losses over it
(``balance``, ``distill``) are differentiable, forward and backward in the HIP library; they have no
counterpart in the reference.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ... import engine


def vq(inputs, codebook):
    """inputs [..., D], codebook [K, D] -> int64 indices [...] of the nearest code
    (reference util_function.py:6-23)."""
    return engine.vq_nearest(inputs, codebook)[0]


def vq_st(inputs, codebook):
    """-> (codes shaped like ``inputs``, flat int64 indices)  (reference util_function.py:34-44)."""
    idx, codes, _ = engine.vq_nearest(inputs, codebook, want_codes=True)
    return codes.view_as(inputs), idx.reshape(-1)


class _CodeLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, inputs, codebook, temperature):
        ctx.save_for_backward(inputs, codebook)
        ctx.temperature = temperature
        return engine.code_logits(inputs, codebook, temperature)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        inputs, codebook = ctx.saved_tensors
        d_inputs, d_codebook = engine.code_logits_grad(grad, inputs, codebook, ctx.temperature, want_inputs=ctx.needs_input_grad[0],
                                                       want_codebook=ctx.needs_input_grad[1])
        return d_inputs, d_codebook, None


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, indices, mask):
        loss, counts, mean_prob, _, ws = engine._balance(logits, indices, mask, None)
        ctx.save_for_backward(logits, counts, ws[:2].clone(), mask)
        ctx.mark_non_differentiable(counts, mean_prob)
        return loss, counts, mean_prob

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, _counts, _mean_prob):
        logits, counts, totals, mask = ctx.saved_tensors
        return engine.balance_grad(logits, counts, totals, grad, mask), None, None


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_indices, mask, temperature):
        loss, loss_rows, _, stats = engine._distill(logits, teacher_logits, teacher_indices, mask, temperature, None)
        ctx.save_for_backward(logits, teacher_logits, teacher_indices, mask, stats[:2 * loss_rows.numel() + 1])
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        logits, teacher_logits, teacher_indices, mask, stats = ctx.saved_tensors
        return engine.distill_grad(logits, teacher_logits, teacher_indices, stats, grad, mask, ctx.temperature), None, None, None, None


def code_logits(inputs, codebook, temperature=1.0):
    """inputs [..., D], codebook [K, D] of one floating-point type -> float32 logits [..., K] of the soft assignment,
    (2 <x, code> - |code|^2) / temperature; gradients reach both."""
    return _CodeLogits.apply(inputs, codebook, temperature)


def balance(logits, indices, mask=None):
    """logits [..., E], choices indices [..., k] or [...] -> (balance loss, int64 choices per expert [E], mean softmax [E]);
    gradients reach the logits through the loss.  See ``engine.balance``."""
    return _Balance.apply(logits, indices, mask)


def distill(logits, teacher_logits, teacher_indices, mask=None, temperature=1.0):
    """Student logits [..., V] against a teacher's top logits and their indices [..., k] -> distillation loss; gradients
    reach the student.  See ``engine.distill``."""
    return _Distill.apply(logits, teacher_logits, teacher_indices, mask, temperature)


__all__ = ["vq", "vq_st", "code_logits", "balance", "distill"]
