"""Differential attention (Differential Transformer, Ye et al. 2024): a head's weights are the difference of two softmax maps, which cancels
what both maps give to every key.  Beside MultiHeadAttention / RPEMultiHeadAttention: the same layer structure, positions by rotation of the
heads instead of a pairwise embedding, no (heads, n, m) weights in memory.

`differential_attention` is the operator, differentiable and for stacked clouds or batches; the modules are built from it for inference on
one cloud per call, like the other layers of this package."""
import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from ... import kernels
from .attention_core import FusedProjection, _one
from .output_layer import AttentionOutput
from .rotary_embedding import RotaryPositionalEmbedding


class _DifferentialAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, q_lengths, k_lengths, key_masks, causal, scale):
        out, state = kernels.diff_attention(q, k, v, lam, q_lengths, k_lengths, key_masks, causal, scale, want_state=True, checked=True)
        ctx.save_for_backward(q, k, v, lam, *state, q_lengths, k_lengths, key_masks)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, lam, maps, lse, q_lengths, k_lengths, key_masks = ctx.saved_tensors
        grads = kernels.diff_attention_backward(dout, q, k, v, lam, (maps, lse), q_lengths, k_lengths, key_masks, ctx.causal, ctx.scale, checked=True)
        return grads + (None,) * 5


def differential_attention(q, k, v, lam, q_lengths=None, k_lengths=None, key_masks=None, causal=False, scale=None):
    """out[i, h] = sum_j (softmax_j(scale q[i, 2h] . k[j, 2c]) - lam[h] softmax_j(scale q[i, 2h+1] . k[j, 2c+1])) v[j, c].

    Stack mode: q (rows, 2 H, d), k (keys, 2 Hk, d), v (keys, Hk, d_v) of clouds one behind the other, q_lengths and k_lengths (clouds,)
    int64 on the device (both None: one cloud).  Batches: (batch, rows, ...), lengths optional -- a cache of keys and values filled to
    k_lengths.  H is a multiple of Hk: query heads h of a group share key and value head c = h Hk / H.  One query row over many keys is
    spread over the device.  d up to 128, d_v up to 256, multiples of 8; float32 (products in fp32), bfloat16, float16.

    lam: float32 tensor, one value or one per head; key_masks: truth values of the key rows, True = ignored (what an ignored row, or one
    beyond its length, holds is never read into a result); causal: query i sees keys j <= i + keys - queries of its cloud; scale: default
    1 / sqrt(d).  Rows without any key, beyond their length or behind the last cloud give zeros.
    In 16-bit types the weights are rounded to the type before their product with v; a call that keeps what a gradient needs adds the rest in a
    second product, so its output differs from the same call without gradients in the last bits.
    Returns (rows, H, d_v) / (batch, rows, H, d_v).  Differentiable in q, k, v and lam (once, in reverse mode); gradients do not depend on scheduling."""
    kernels.check_diff_attention(q, k, v, lam, q_lengths, k_lengths, key_masks, scale)
    kernels.refuse_tangents('differential_attention', q, k, v, lam)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, lam)):
        lam = lam.expand(q.shape[-2] // 2)  # the gradient of a shared value is the sum over its heads
        return _DifferentialAttention.apply(q, k, v, lam, q_lengths, k_lengths, key_masks, causal, scale)
    return kernels.diff_attention(q, k, v, lam, q_lengths, k_lengths, key_masks, causal, scale, checked=True)


class DifferentialMultiHeadAttention(nn.Module):
    """num_heads pairs of maps of d_model / num_heads / 2 channels each, values of d_model / num_heads.  lam = exp(a1 . b1) - exp(a2 . b2) +
    lambda_init with learned vectors; the heads are normalised one by one and scaled by 1 - lambda_init.  positions_* (1, N, 3): points
    whose coordinates turn the heads (None: no positions).

    The heads' norm is this package's LayerNorm, with a mean and a bias; the published layer divides each head by its root mean square alone.
    Weights trained with that layer are not this module's: use differential_attention and their own norm."""

    def __init__(self, d_model, num_heads, dropout=None, lambda_init=0.5, rotary_base=10000.0):
        super().__init__()
        if d_model % (2 * num_heads) != 0 or (d_model // num_heads // 2) % 8 != 0:
            raise ValueError('`d_model` ({}) must be a multiple of 16 `num_heads` ({}).'.format(d_model, num_heads))
        if dropout is not None:
            raise NotImplementedError('inference path: dropout=None')
        self.d_model, self.num_heads, self.lambda_init = d_model, num_heads, lambda_init
        self.d_map = d_model // num_heads // 2
        self.proj_q = nn.Linear(d_model, d_model)
        self.proj_k = nn.Linear(d_model, d_model)
        self.proj_v = nn.Linear(d_model, d_model)
        self.lambda_q1, self.lambda_k1, self.lambda_q2, self.lambda_k2 = (nn.Parameter(0.1 * torch.randn(self.d_map)) for _ in range(4))
        self.head_norm = nn.LayerNorm(2 * self.d_map)
        self.rotary = RotaryPositionalEmbedding(self.d_map, rotary_dim=self.d_map // 6 * 6 if self.d_map < 24 else self.d_map // 24 * 24,
                                                base=rotary_base, num_axes=3)
        self._qkv = FusedProjection(self.proj_q, self.proj_k, self.proj_v)
        self._kv = FusedProjection(self.proj_k, self.proj_v)

    def lam(self):
        return torch.exp(torch.dot(self.lambda_q1, self.lambda_k1)) - torch.exp(torch.dot(self.lambda_q2, self.lambda_k2)) + self.lambda_init

    def forward(self, input_q, input_k, input_v, positions_q=None, positions_k=None, key_masks=None):
        """input_* (1, N|M, C), positions_* (1, N|M, 3), key_masks (1, M) -> hidden (1, N, C)."""
        if input_q.shape[0] != 1:
            raise NotImplementedError('batch size 1 (one cloud per call), as in the reference model')
        if (positions_q is None) != (positions_k is None):
            raise ValueError('positions of both sides or of none')
        with torch.no_grad():
            if input_q is input_k and input_k is input_v:
                q, k, v = self._qkv(input_q[0])
            else:
                q = kernels.linear(input_q[0], self.proj_q.weight, self.proj_q.bias)
                if input_k is input_v:
                    k, v = self._kv(input_k[0])
                else:
                    k = kernels.linear(input_k[0], self.proj_k.weight, self.proj_k.bias)
                    v = kernels.linear(input_v[0], self.proj_v.weight, self.proj_v.bias)
            h, d = self.num_heads, self.d_map
            q, k, v = q.unflatten(1, (2 * h, d)), k.unflatten(1, (2 * h, d)), v.unflatten(1, (h, 2 * d))
            if positions_q is not None:
                if positions_q is positions_k and q.shape[0] == k.shape[0]:
                    q, k = self.rotary(q, k, positions_q[0])  # one launch, the angles once
                else:
                    q, k = self.rotary(q, None, positions_q[0])[0], self.rotary(k, None, positions_k[0])[0]
            out = differential_attention(q, k, v, self.lam().reshape(1), key_masks=_one(key_masks))
            out = kernels.layer_norm(out, self.head_norm.weight * (1.0 - self.lambda_init), self.head_norm.bias * (1.0 - self.lambda_init),
                                     self.head_norm.eps)
            return out.reshape(1, -1, self.d_model)


class DifferentialAttentionLayer(nn.Module):
    def __init__(self, d_model, num_heads, dropout=None, lambda_init=0.5, rotary_base=10000.0):
        super().__init__()
        self.attention = DifferentialMultiHeadAttention(d_model, num_heads, dropout=dropout, lambda_init=lambda_init, rotary_base=rotary_base)
        self.linear = nn.Linear(d_model, d_model)
        self.norm = nn.LayerNorm(d_model)

    def forward(self, input_states, memory_states, input_positions=None, memory_positions=None, memory_masks=None):
        hidden = self.attention(input_states, memory_states, memory_states, input_positions, memory_positions, key_masks=memory_masks)
        hidden = kernels.linear(hidden, self.linear.weight, self.linear.bias)
        return kernels.layer_norm(hidden, self.norm.weight, self.norm.bias, self.norm.eps, residual=input_states)


class DifferentialTransformerLayer(nn.Module):
    def __init__(self, d_model, num_heads, dropout=None, activation_fn='ReLU', lambda_init=0.5, rotary_base=10000.0):
        super().__init__()
        self.attention = DifferentialAttentionLayer(d_model, num_heads, dropout=dropout, lambda_init=lambda_init, rotary_base=rotary_base)
        self.output = AttentionOutput(d_model, dropout=dropout, activation_fn=activation_fn)

    def forward(self, input_states, memory_states, input_positions=None, memory_positions=None, memory_masks=None):
        return self.output(self.attention(input_states, memory_states, input_positions, memory_positions, memory_masks=memory_masks))


class DifferentialConditionalTransformer(nn.Module):
    """The interleaved self / cross stack of RPEConditionalTransformer with differential attention: 'self' blocks turn the heads by the
    superpoints' coordinates (points0 / points1 (1, N, 3)), 'cross' blocks use no positions, the two clouds being in frames of their own.
    lambda_init of layer l: 0.8 - 0.6 exp(-0.3 l)."""

    def __init__(self, blocks, d_model, num_heads, dropout=None, activation_fn='ReLU', parallel=False, rotary_base=10000.0):
        super().__init__()
        self.blocks = blocks
        for block in self.blocks:
            if block not in ('self', 'cross'):
                raise ValueError('Unsupported block type "{}".'.format(block))
        self.layers = nn.ModuleList(
            DifferentialTransformerLayer(d_model, num_heads, dropout=dropout, activation_fn=activation_fn,
                                         lambda_init=0.8 - 0.6 * math.exp(-0.3 * i), rotary_base=rotary_base) for i in range(len(blocks)))
        self.parallel = parallel

    def forward(self, feats0, feats1, points0, points1, masks0=None, masks1=None):
        for layer, block in zip(self.layers, self.blocks):
            if block == 'self':
                feats0 = layer(feats0, feats0, points0, points0, memory_masks=masks0)
                feats1 = layer(feats1, feats1, points1, points1, memory_masks=masks1)
            else:
                new0 = layer(feats0, feats1, memory_masks=masks1)
                feats1 = layer(feats1, feats0 if self.parallel else new0, memory_masks=masks0)
                feats0 = new0
        return feats0, feats1
