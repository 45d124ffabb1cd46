"""Rotary positions of queries and keys (no counterpart in the reference, whose positions are learned: model.py:54, 74).

A Rope (kernels.Rope) holds the angle of each pair of a head's elements for one position; rotate() turns queries and keys by
their positions' angles, differentiably.  rope_frequencies() gives the angles, also those of a model stretched past the
length it was trained at.
"""
import math

import torch

from . import kernels as K

SCALINGS = ('', 'linear', 'ntk', 'bands')


def rope_frequencies(rot, base=10000.0, scaling='', factor=1.0, trained=0, low=1.0, high=32.0):
    """(inv_freq, amplitude) for rot turned elements of a head: inv_freq[i] = base^(-2i / rot) radians a position, and for a
    context `factor` times the trained one
      'linear'  every angle divided by factor (positions pressed together);
      'ntk'     the base raised to base * factor^(rot / (rot - 2)): the slowest pair slowed by factor, the fastest not at all;
      'bands'   pairs that turn less than `low` times in the `trained` length slowed by factor, those that turn more than `high`
                times left, in between by parts; the amplitude is 0.1 ln(factor) + 1."""
    if rot < 2 or rot % 2 or not base > 0 or not factor >= 1:
        raise ValueError('rope_frequencies: an even number of elements, a positive base and a factor of at least 1')
    if scaling not in SCALINGS:
        raise ValueError('rope_frequencies: scaling one of %s' % (SCALINGS,))
    if scaling == 'ntk':
        if rot < 4:
            raise ValueError("rope_frequencies: 'ntk' needs at least two pairs")
        base = base * factor ** (rot / (rot - 2))
    w = [base ** (-2 * i / rot) for i in range(rot // 2)]
    amplitude = 1.0
    if scaling == 'linear':
        w = [x / factor for x in w]
    elif scaling == 'bands':
        if trained < 1 or not high > low:
            raise ValueError("rope_frequencies: 'bands' needs the trained length and high > low")
        keep = [min(1.0, max(0.0, (trained * x / (2 * math.pi) - low) / (high - low))) for x in w]
        w = [x / factor * (1 - r) + x * r for x, r in zip(w, keep)]
        amplitude = 0.1 * math.log(factor) + 1
    return w, amplitude


class _Rotate(torch.autograd.Function):
    """The turn; its gradient is the turn back."""

    @staticmethod
    def forward(ctx, x, pos, rope, inverse):
        ctx.save_for_backward(pos)
        ctx.rope, ctx.inverse = rope, inverse
        return K.rope(x if x.stride(-1) == 1 else x.contiguous(), pos, rope, inverse=inverse)

    @staticmethod
    def backward(ctx, dy):
        return _Rotate.apply(dy, ctx.saved_tensors[0], ctx.rope, not ctx.inverse), None, None, None


def rotate(x, pos, rope):
    """x (B,H,T,D), each row turned by the angles of its position (pos (T,) or (B,T)); differentiable in x."""
    if torch.is_grad_enabled() and x.requires_grad:
        return _Rotate.apply(x, pos, rope, False)
    return K.rope(x if x.stride(-1) == 1 else x.contiguous(), pos, rope)
