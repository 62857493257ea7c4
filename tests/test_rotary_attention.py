"""CPU: refusals of the rotary positions and the differential attention, their host logic, and the oracle's gradients against differences."""
import ctypes
import math

import pytest
import torch

import attention_oracle as oracle
from geotransformer_amd import _lib, kernels
from geotransformer_amd.modules.transformer import (DifferentialConditionalTransformer, DifferentialMultiHeadAttention, RotaryPositionalEmbedding,
                                                    differential_attention, rotary_frequencies)


def _qkv(rows=5, keys=7, heads=4, kv=2, d=16, dv=32, dtype=torch.float32, lead=()):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    return r(*lead, rows, 2 * heads, d), r(*lead, keys, 2 * kv, d), r(*lead, keys, kv, dv), torch.rand(heads, generator=g)


@pytest.mark.parametrize('change,error,text', [
    (dict(q=torch.zeros(5, 8)), ValueError, 'stack mode or'),
    (dict(k=torch.zeros(7, 4, 16, dtype=torch.float64)), TypeError, 'all of one type'),
    (dict(q=torch.zeros(5, 7, 16)), ValueError, '2 H heads'),
    (dict(q=torch.zeros(5, 6, 16)), ValueError, 'a multiple of Hk'),
    (dict(v=torch.zeros(6, 2, 32)), ValueError, 'do not fit'),
    (dict(q=torch.zeros(5, 8, 12), k=torch.zeros(7, 4, 12)), ValueError, 'multiples of 8'),
    (dict(v=torch.zeros(7, 2, 264)), ValueError, 'multiples of 8'),
    (dict(lam=torch.zeros(3)), ValueError, 'lam is'),
    (dict(lam=torch.zeros(4, dtype=torch.float64)), ValueError, 'lam is'),
    (dict(scale=0.0), ValueError, 'scale'),
    (dict(scale=float('nan')), ValueError, 'scale'),
    (dict(q_lengths=torch.tensor([5])), ValueError, 'both lengths'),
    (dict(q_lengths=torch.tensor([5], dtype=torch.int32), k_lengths=torch.tensor([7])), TypeError, 'int64'),
    (dict(q_lengths=torch.tensor([2, 3]), k_lengths=torch.tensor([7])), ValueError, 'sequences'),
    (dict(key_masks=torch.zeros(7)), ValueError, 'truth values'),
    (dict(key_masks=torch.zeros(6, dtype=torch.bool)), ValueError, 'truth values'),
    (dict(), RuntimeError, 'no CPU fallback'),
])
def test_attention_refuses(change, error, text):
    q, k, v, lam = _qkv()
    args = dict(dict(q=q, k=k, v=v, lam=lam), **change)
    with pytest.raises(error, match=text):
        differential_attention(**args)


@pytest.mark.parametrize('change,error,text', [
    (dict(q=torch.zeros(5, 16)), ValueError, 'rows, heads, channels'),
    (dict(k=torch.zeros(4, 2, 16)), ValueError, 'of the same rows'),
    (dict(q=torch.zeros(5, 2, 16, dtype=torch.float64), k=None), TypeError, 'float32, bfloat16 or float16'),
    (dict(q=torch.zeros(5, 2, 24), k=None), ValueError, 'built for 16'),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), ValueError, 'positions of rows'),
    (dict(positions=torch.zeros(5, 3)), ValueError, 'axes'),
    (dict(positions=torch.zeros(5, dtype=torch.float16)), TypeError, 'positions are'),
    (dict(positions=torch.zeros(5, requires_grad=True)), NotImplementedError, 'not differentiable'),
    (dict(), RuntimeError, 'no CPU fallback'),
])
def test_rotary_refuses(change, error, text):
    args = dict(dict(q=torch.zeros(5, 4, 16), k=torch.zeros(5, 2, 16), positions=torch.arange(5)), **change)
    with pytest.raises(error, match=text):
        RotaryPositionalEmbedding(16)(**args)


@pytest.mark.parametrize('kw', [dict(rotary_dim=18), dict(rotary_dim=7), dict(rotary_dim=0), dict(num_axes=9), dict(num_axes=0), dict(scaling='half'),
                                dict(scaling='yarn', scaling_factor=2.0), dict(scaling='linear', scaling_factor=0.5), dict(base=1.0)])
def test_rotary_module_refuses(kw):
    with pytest.raises(ValueError):
        RotaryPositionalEmbedding(16, **kw)


def test_frequencies():
    plain, gain = rotary_frequencies(8)
    assert gain == 1.0 and plain[0] == 1.0 and math.isclose(float(plain[-1]), 10000.0 ** (-7 / 8), rel_tol=1e-14)
    linear, _ = rotary_frequencies(8, scaling='linear', scaling_factor=4.0)
    assert torch.allclose(linear * 4, plain, rtol=1e-15)
    ntk, _ = rotary_frequencies(8, scaling='ntk', scaling_factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1] * 4), float(plain[-1]), rel_tol=1e-12)
    yarn, gain = rotary_frequencies(8, scaling='yarn', scaling_factor=4.0, original_length=2048)
    assert yarn[0] == plain[0] and math.isclose(float(yarn[-1] * 4), float(plain[-1]), rel_tol=1e-12) and math.isclose(gain, 0.1 * math.log(4) + 1)
    assert bool((yarn <= plain).all()) and bool((yarn >= plain / 4).all())


def test_a_cast_module_keeps_its_angles():
    rope = RotaryPositionalEmbedding(16)
    bits = rope.turn_bits.clone()
    assert rope.half().turn_bits.dtype == torch.int64 and torch.equal(rope.turn_bits, bits) and not rope.state_dict()


def test_entry_points_check_their_arguments():
    """The C entry points refuse before any launch (no GPU needed)."""
    lib = _lib.load()
    one = 1 << 20  # a non-null, aligned address that is never read
    view = kernels.Heads(one, 4, 0, 64, 16)
    call = lambda q, k, **kw: lib.geotr_rotary(ctypes.byref(q), ctypes.byref(q), k, k, kw.get('dtype', 0), 1, kw.get('rows', 4), 16, kw.get('rot', 16),  # noqa: E731
                                               0, one, kw.get('pos', 1), 0, 1, 0, one, one, 1.0, 0, None)
    assert call(view, None, dtype=3) == -1 and b'dtype' in lib.geotr_last_error()
    assert call(view, None, rot=17) == -1 and b'rotary dimension' in lib.geotr_last_error()
    assert call(view, None, pos=4) == -1 and b'position type' in lib.geotr_last_error()
    assert call(kernels.Heads(None, 4, 0, 64, 16), None) == -1 and b'null pointer' in lib.geotr_last_error()
    assert call(view, None, rows=0) == 0

    def op(**kw):
        a = dict(q=kernels.Heads(one, 8, 0, 128, 16), k=kernels.Heads(one, 4, 0, 64, 16), v=kernels.Heads(one, 2, 0, 64, 32), dtype=0, stacked=0, batch=1,
                 n=5, m=7, dim=16, v_dim=32, lam=one, scale=0.25)
        a.update(kw)
        return kernels.DiffAttn(**a)
    fwd = lambda o: lib.geotr_diff_attn_forward(ctypes.byref(o), one, None, None, None, 0, None)  # noqa: E731
    for change, text in ((dict(dtype=5), b'dtype'), (dict(dim=12), b'head dimensions'), (dict(v_dim=320), b'head dimensions'), (dict(scale=-1.0), b'scale'),
                         (dict(lam=None), b'lam'), (dict(stacked=1), b'both lengths'), (dict(q=kernels.Heads(one, 6, 0, 128, 16)), b'query'),
                         (dict(k=kernels.Heads(one, 2, 0, 64, 16)), b'k has 2 heads'), (dict(v=kernels.Heads(None, 2, 0, 64, 32)), b'v is a null'),
                         (dict(q=kernels.Heads(one + 4, 8, 0, 128, 16)), b'16-byte'), (dict(k=kernels.Heads(one, 4, 0, 66, 16)), b'16-byte'),
                         (dict(k=kernels.Heads(one, 4, 0, 1 << 24, 16)), b'strides'), (dict(n=1 << 31), b'query rows'), (dict(n=-1), b'rows')):
        assert fwd(op(**change)) == -1 and text in lib.geotr_last_error(), (change, lib.geotr_last_error())
    assert lib.geotr_diff_attn_forward(ctypes.byref(op()), None, None, None, None, 0, None) == -1
    assert lib.geotr_diff_attn_forward(ctypes.byref(op()), one, one, None, None, 0, None) == -1 and b'go together' in lib.geotr_last_error()
    big = op(n=1, m=100000)
    assert lib.geotr_diff_attn_workspace_bytes(ctypes.byref(big)) > 0
    assert fwd(big) == -2 and b'workspace' in lib.geotr_last_error()
    need = lib.geotr_diff_attn_backward_workspace_bytes(ctypes.byref(op()))
    assert need >= 3 * 5 * 4 * 4
    bwd = lambda o, g, ws: lib.geotr_diff_attn_backward(ctypes.byref(o), g, one, one, one, one, one, one, one if ws else None, ws, None)  # noqa: E731
    g = kernels.Heads(one, 4, 0, 128, 32)
    assert bwd(op(), ctypes.byref(g), need - 1) == -2 and bwd(op(), None, need) == -1
    assert bwd(op(), ctypes.byref(kernels.Heads(one, 3, 0, 128, 32)), need) == -1 and b'dout has 3 heads' in lib.geotr_last_error()


def test_modules_refuse_and_hold_their_parameters():
    with pytest.raises(ValueError, match='multiple of 16'):
        DifferentialMultiHeadAttention(72, 4)
    with pytest.raises(NotImplementedError):
        DifferentialMultiHeadAttention(64, 4, dropout=0.1)
    with pytest.raises(ValueError, match='Unsupported block type'):
        DifferentialConditionalTransformer(['self', 'both'], 64, 4)
    net = DifferentialConditionalTransformer(['self', 'cross', 'self'], 64, 4)
    assert [round(layer.attention.attention.lambda_init, 4) for layer in net.layers] == [0.2, 0.3555, 0.4707]
    keys = set(net.state_dict())
    assert 'layers.1.attention.attention.lambda_q2' in keys and not any('rotary' in k for k in keys)


@pytest.mark.parametrize('causal', [False, True])
def test_the_oracles_gradients_match_differences(causal):
    """Central differences in 64 bits, step 1e-5: truncation 1e-10, rounding 1e-16 / 1e-5 per unit; 1e-7 covers both by far."""
    q, k, v, lam = (t.double() for t in _qkv(rows=4, keys=6, heads=2, kv=1, d=8, dv=8))
    oracle.U[torch.float64], oracle.TINY[torch.float64] = 2.0 ** -53, 0.0
    masks = torch.tensor([False, True, False, False, False, False])
    dout = torch.randn(4, 2, 8, generator=torch.Generator().manual_seed(1)).double()
    f = lambda: float((oracle.differential_attention(q, k, v, lam, key_masks=masks, causal=causal)['out'][0] * dout).sum())  # noqa: E731
    grads = oracle.differential_attention(q, k, v, lam, key_masks=masks, causal=causal, dout=dout)
    for name, t in (('dq', q), ('dk', k), ('dv', v), ('dlam', lam)):
        flat = t.view(-1)
        for i in range(0, flat.numel(), 5):
            keep = float(flat[i])
            flat[i] = keep + 1e-5
            up = f()
            flat[i] = keep - 1e-5
            down = f()
            flat[i] = keep
            assert abs((up - down) / 2e-5 - float(grads[name][0].reshape(-1)[i])) < 1e-7, (name, i)


def test_the_oracle_catches_a_planted_mistake():
    """The bounds are tight enough to see one key too many: a causal limit off by one in the oracle is outside them."""
    q, k, v, lam = _qkv(rows=9, keys=9)
    good = oracle.differential_attention(q, k, v, lam, causal=True)['out']
    off = oracle.differential_attention(q[:8], k, v, lam, causal=True)['out'][0]  # every row sees one key more
    with pytest.raises(AssertionError, match='off by'):
        oracle.assert_within('out', off, good[0][:8], good[1][:8])
