"""Rotary positions: the heads of queries and keys turned by their position, so that their products depend on relative positions only.

Beside SinusoidalPositionalEmbedding, which adds or projects positions: here nothing is added, and the same module serves sequences
(integer positions, one axis) and point clouds (coordinates, one frequency set per axis)."""
import math

import torch
import torch.nn as nn

from ... import kernels

SCALINGS = (None, 'linear', 'ntk', 'yarn')


def rotary_frequencies(pairs, base=10000.0, scaling=None, scaling_factor=1.0, original_length=None, beta_fast=32.0, beta_slow=1.0):
    """(radians per unit of position (pairs,) float64, factor on cosine and sine) of one axis: base^(-j / pairs), stretched for positions
    beyond those a model was trained on:
    'linear': every frequency divided by scaling_factor;
    'ntk':    a larger base, such that the slowest pair slows down by scaling_factor and the fastest keeps its rate;
    'yarn':   by parts (YaRN, Peng et al. 2023): pairs that turn beta_fast times or more within original_length keep their rate, pairs that
              turn beta_slow times or less are divided by scaling_factor, a linear ramp between; factor 0.1 ln(scaling_factor) + 1.  The ramp
              is in turns, as the formula is published; a program that ramps in the pair's index has other frequencies inside the ramp."""
    if scaling not in SCALINGS:
        raise ValueError(f'Unsupported scaling of rotary positions: {scaling}.')
    if not scaling_factor >= 1.0 or not base > 1.0:
        raise ValueError(f'rotary positions: base {base} (above 1), scaling_factor {scaling_factor} (1 or more)')
    if scaling == 'ntk' and pairs > 1:
        base = base * scaling_factor ** (pairs / (pairs - 1.0))
    freq = base ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    gain = 1.0
    if scaling == 'linear':
        freq = freq / scaling_factor
    elif scaling == 'yarn':
        if original_length is None or not beta_fast > beta_slow:
            raise ValueError("scaling='yarn' needs original_length, and beta_fast above beta_slow")
        keep = ((original_length * freq / (2.0 * math.pi) - beta_slow) / (beta_fast - beta_slow)).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / scaling_factor)
        gain = 0.1 * math.log(scaling_factor) + 1.0
    return freq, gain


class _Rotary(torch.autograd.Function):
    """The rotation is linear: its gradient is the transposed rotation, by the same function."""

    @staticmethod
    def forward(ctx, q, k, positions, turns, axis, how, inverse):
        ctx.save_for_backward(positions, turns, axis)
        ctx.how, ctx.inverse = how, inverse
        ctx.set_materialize_grads(False)
        return kernels.rotary(q, k, positions, turns, axis, *how, inverse=inverse, checked=True)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, turns, axis = ctx.saved_tensors
        if dq is None and dk is None:
            return (None,) * 7
        first, second = (dk, None) if dq is None else (dq, dk)
        if torch.is_grad_enabled():  # a graph of the gradient is wanted
            first, second = _Rotary.apply(first, second, positions, turns, axis, ctx.how, not ctx.inverse)
        else:
            first, second = kernels.rotary(first, second, positions, turns, axis, *ctx.how, inverse=not ctx.inverse)
        return (None, first, None, None, None, None, None) if dq is None else (first, second, None, None, None, None, None)


class RotaryPositionalEmbedding(nn.Module):
    """q, k = rope(q, k, positions): q (rows, H, head_dim) or (batch, rows, H, head_dim), k likewise with its own number of heads (or None),
    float32, bfloat16 or float16; positions (rows,) / (batch, rows) integers or floats, for num_axes > 1 with a last dimension of num_axes.
    Differentiable in q and k (in reverse mode).  The angles are taken in 64 bits, the rotation in 32, and the result is rounded once.

    rotary_dim: channels that are turned (the first ones; default: the largest multiple of 2 num_axes); interleaved: pairs (2i, 2i + 1)
    instead of (i, i + rotary_dim / 2).  Axis a turns the pairs a F .. (a + 1) F - 1, F = rotary_dim / (2 num_axes).
    base, scaling ...: see rotary_frequencies."""

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, interleaved=False, num_axes=1, scaling=None, scaling_factor=1.0,
                 original_length=None, beta_fast=32.0, beta_slow=1.0):
        super().__init__()
        if num_axes < 1:
            raise ValueError(f'num_axes {num_axes}')
        if rotary_dim is None:
            rotary_dim = head_dim // (2 * num_axes) * (2 * num_axes)
        if rotary_dim % (2 * num_axes) != 0 or not 2 * num_axes <= rotary_dim <= head_dim:
            raise ValueError(f'rotary_dim {rotary_dim}: a multiple of {2 * num_axes} (pairs x axes) up to the head\'s {head_dim} channels')
        self.head_dim, self.rotary_dim, self.num_axes, self.interleaved = head_dim, rotary_dim, num_axes, bool(interleaved)
        freq, self.gain = rotary_frequencies(rotary_dim // (2 * num_axes), base, scaling, scaling_factor, original_length, beta_fast, beta_slow)
        # the bits of float64 turns per unit: a module cast to half keeps integer buffers as they are
        self.register_buffer('turn_bits', (freq / (2.0 * math.pi)).repeat(num_axes).view(torch.int64), persistent=False)
        self.register_buffer('axis', torch.arange(num_axes, dtype=torch.int32).repeat_interleave(rotary_dim // (2 * num_axes)), persistent=False)

    def forward(self, q, k, positions):
        kernels.check_rotary_heads(q, k)
        lead = q.dim() - 2
        if q.shape[-1] != self.head_dim:
            raise ValueError(f'heads of {q.shape[-1]} channels, built for {self.head_dim}')
        if (positions.shape[-1] if positions.dim() == lead + 1 else 1) != self.num_axes:
            raise ValueError(f'positions {tuple(positions.shape)} of rows {tuple(q.shape[:lead])}, built for {self.num_axes} axes')
        if positions.requires_grad:
            raise NotImplementedError('rotary positions are not differentiable in the positions: pass positions.detach()')
        kernels.refuse_tangents('RotaryPositionalEmbedding', q, k, positions)
        how, turns = (self.rotary_dim, self.interleaved, self.gain), self.turn_bits
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            return _Rotary.apply(q, k, positions, turns, self.axis, how, False)
        return kernels.rotary(q, k, positions, turns, self.axis, *how, checked=True)
