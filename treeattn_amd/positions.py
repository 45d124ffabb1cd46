"""Rotary positions of queries and keys (Su et al. 2021, arXiv:2104.09864; no counterpart in the reference, whose positions are
learned: model.py:54, 74).

A Rope (kernels.Rope) holds the angle of each pair of a head's elements for one position; rotate() turns queries and keys by
their positions' angles, differentiably.  rope_frequencies() gives the angles, also those of a model stretched past the
length it was trained at.  Models with Config.rope have them in place of learned positions: the attention modules turn what
their projection gives (heads), the decoder what it stores and asks with.
"""
import math

import torch
from torch.autograd import forward_ad

from . import kernels as K

SCALINGS = ('', 'linear', 'ntk', 'bands')


def rope_frequencies(rot, base=10000.0, scaling='', factor=1.0, trained=0, low=1.0, high=32.0):
    """(inv_freq, amplitude) for rot turned elements of a head: inv_freq[i] = base^(-2i / rot) radians a position, and for a
    context `factor` times the trained one
      'linear'  every angle divided by factor (positions pressed together: position interpolation, Chen et al. 2023,
                arXiv:2306.15595);
      'ntk'     the base raised to base * factor^(rot / (rot - 2)): the slowest pair slowed by factor, the fastest not at all (the
                "NTK-aware" change of base, as Peng et al. 2023, arXiv:2309.00071, section 3.1, give it);
      'bands'   pairs that turn less than `low` times in the `trained` length slowed by factor, those that turn more than `high`
                times left, in between by parts; the amplitude is 0.1 ln(factor) + 1 (by parts and with that factor on queries
                and keys both: the same paper, sections 3.2 to 3.4)."""
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
    """The turn, linear in x: its gradient is the turn back, its forward derivative the turn of the tangent."""

    @staticmethod
    def forward(ctx, x, pos, rope, inverse):
        ctx.save_for_backward(pos)
        ctx.save_for_forward(pos)
        ctx.rope, ctx.inverse = rope, inverse
        return K.rope(x if x.stride(-1) == 1 else x.contiguous(), pos, rope, inverse=inverse)

    @staticmethod
    def backward(ctx, dy):
        return _turn(dy, ctx.saved_tensors[0], ctx.rope, not ctx.inverse), None, None, None

    @staticmethod
    def jvp(ctx, dx, *_):
        return _turn(dx, ctx.saved_tensors[0], ctx.rope, ctx.inverse)


def _turn(x, pos, rope, inverse):
    # (outside a level of forward_ad no tensor has a tangent, and the second question costs nothing)
    if (torch.is_grad_enabled() and x.requires_grad) or forward_ad.unpack_dual(x).tangent is not None:
        return _Rotate.apply(x, pos, rope, inverse)
    return K.rope(x if x.stride(-1) == 1 else x.contiguous(), pos, rope, inverse=inverse)


def rotate(x, pos, rope):
    """x (B,H,T,D), each row turned by the angles of its position (pos (T,) or (B,T)); differentiable in x, backwards and
    forwards."""
    return _turn(x, pos, rope, False)


def _settings(cfg, device):
    """What a Rope of rope_of is made from."""
    return (cfg.rope, cfg.rope_dim, cfg.rope_base, cfg.rope_scaling, cfg.rope_factor, cfg.rope_trained, cfg.seq_len, cfg.n_embd,
            cfg.n_head, device)


def rope_of(cfg, device):
    """The Rope of a model configuration on `device`, None when its positions are learned."""
    if not getattr(cfg, 'rope', ''):
        return None
    dh = cfg.n_embd // cfg.n_head
    rot = cfg.rope_dim or dh
    if rot > dh:
        raise ValueError('rope_dim %d: heads have %d elements' % (rot, dh))
    freq, amplitude = rope_frequencies(rot, cfg.rope_base, cfg.rope_scaling, cfg.rope_factor, cfg.rope_trained or cfg.seq_len)
    return K.Rope(freq, device, layout=cfg.rope, amplitude=amplitude)


def heads(module, qkv):
    """The projection qkv (b,T,3C) of an attention module as its queries, keys and values (b,H,T,dh), queries and keys turned
    by their positions where the module's configuration has rotary positions (one call for both; differentiable)."""
    b, T, C3 = qkv.shape
    C, H = C3 // 3, module.H
    if not getattr(module.cfg, 'rope', ''):
        return [t.view(b, T, H, C // H).transpose(1, 2) for t in qkv.split(C, dim=2)]
    made, r = module.__dict__.get('_rope_made', (None, None))
    now = _settings(module.cfg, qkv.device)
    if made != now:
        r = rope_of(module.cfg, qkv.device)
        module.__dict__['_rope_made'] = now, r
    qk, v = qkv.split((2 * C, C), dim=2)
    pos = torch.arange(T, device=qkv.device, dtype=torch.int32)
    qk = rotate(qk.view(b, T, 2 * H, C // H).transpose(1, 2), pos, r)
    return [qk[:, :H], qk[:, H:], v.view(b, T, H, C // H).transpose(1, 2)]
