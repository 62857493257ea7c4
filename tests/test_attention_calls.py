"""CPU: calls of the rotary positions and the differential attention that are refused, or have to be answered, away from the common forms."""
import pytest
import torch
from torch.autograd import forward_ad

from geotransformer_amd import kernels
from geotransformer_amd.modules.transformer import RotaryPositionalEmbedding, differential_attention


def _heads(rows=5, keys=7, heads=4, kv=2, d=16, dv=32, lead=()):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return r(*lead, rows, 2 * heads, d), r(*lead, keys, 2 * kv, d), r(*lead, keys, kv, dv), torch.rand(heads, generator=g)


@pytest.mark.parametrize('which', range(4))
@pytest.mark.parametrize('grad', [False, True])
def test_attention_refuses_tangents(monkeypatch, which, grad):
    """A dual tensor requires no grad: without the refusal the kernel call returns a result that has silently no tangent."""
    monkeypatch.setattr(kernels, 'diff_attention', lambda q, k, v, *a, **kw: q.new_zeros(5, 4, 32))
    inputs = list(_heads())
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        assert differential_attention(*inputs).shape == (5, 4, 32)  # no tangent: an ordinary call
        inputs[which] = forward_ad.make_dual(inputs[which], torch.ones_like(inputs[which]))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            differential_attention(*inputs)


@pytest.mark.parametrize('which', range(3))
@pytest.mark.parametrize('grad', [False, True])
def test_rotary_refuses_tangents(monkeypatch, which, grad):
    monkeypatch.setattr(kernels, 'rotary', lambda q, k, *a, **kw: (torch.zeros_like(q), k))
    q, k, _, _ = _heads(keys=5)
    inputs = [q, k, torch.arange(5, dtype=torch.float32)]
    rope = RotaryPositionalEmbedding(16)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        assert rope(*inputs)[0].shape == q.shape
        inputs[which] = forward_ad.make_dual(inputs[which], torch.ones_like(inputs[which]))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            rope(*inputs)


def test_a_stack_of_no_sequence_needs_no_lengths():
    """An empty tensor of lengths has no address: the entry point takes it (no rows here, so nothing is launched)."""
    import ctypes
    from geotransformer_amd import _lib
    lib, one = _lib.load(), 1 << 20  # a non-null, aligned address that is never read
    view = lambda heads, d: kernels.Heads(one, heads, 0, heads * d, d)  # noqa: E731
    op = kernels.DiffAttn(q=view(8, 16), k=view(4, 16), v=view(2, 32), dtype=0, stacked=1, batch=0, n=0, m=7, dim=16, v_dim=32, lam=one, scale=0.25)
    assert lib.geotr_diff_attn_forward(ctypes.byref(op), one, None, None, None, 0, None) == 0
    op.batch = 1
    assert lib.geotr_diff_attn_forward(ctypes.byref(op), one, None, None, None, 0, None) == -1 and b'both lengths' in lib.geotr_last_error()


def _state(q, v):
    lead, heads, kv = q.shape[:-2], q.shape[-2] // 2, v.shape[-2]
    return torch.zeros(*lead, heads, 2, v.shape[-1]), torch.zeros(kv, 4, *lead, heads // kv)


@pytest.mark.parametrize('change,error,text', [
    (dict(v=torch.zeros(6, 2, 32)), ValueError, 'do not fit'),            # a row less than k: rows behind v would be read
    (dict(k=torch.zeros(7, 4, 24)), ValueError, 'multiples of 8'),
    (dict(lam=torch.zeros(3)), ValueError, 'lam is'),
    (dict(q_lengths=torch.tensor([5], dtype=torch.int32), k_lengths=torch.tensor([7], dtype=torch.int32)), TypeError, 'int64'),
    (dict(q_lengths=torch.tensor([5])), ValueError, 'both lengths'),
    (dict(key_masks=torch.zeros(6, dtype=torch.bool)), ValueError, 'truth values'),
    (dict(scale=-1.0), ValueError, 'scale'),
    (dict(dout=torch.zeros(4, 4, 32)), ValueError, 'dout is'),
    (dict(state=(torch.zeros(4, 4, 2, 32), torch.zeros(2, 4, 5, 2))), ValueError, 'another call'),
    (dict(state=(torch.zeros(5, 4, 2, 32), torch.zeros(4, 4, 5, 1))), ValueError, 'another call'),   # the sums of other groups of heads
    (dict(state=(torch.zeros(5, 4, 2, 32), torch.zeros(2, 4, 4, 2))), ValueError, 'another call'),
    (dict(state=(torch.zeros(5, 4, 2, 32), torch.zeros(2, 4, 5, 2, dtype=torch.float16))), ValueError, 'as diff_attention left it'),
    (dict(state=(torch.zeros(5, 4, 32, 2).transpose(2, 3), torch.zeros(2, 4, 5, 2))), ValueError, 'as diff_attention left it'),
])
def test_the_gradient_entry_checks_its_arguments(change, error, text):
    """Also what reaches it without the function: shapes that do not fit would be read past their ends."""
    q, k, v, lam = _heads()
    args = dict(dout=torch.zeros(5, 4, 32), q=q, k=k, v=v, lam=lam, state=_state(q, v))
    args.update(change)
    with pytest.raises(error, match=text):
        kernels.diff_attention_backward(**args)


def test_strides_are_held_to_what_a_tile_reaches():
    """A cache laid out by heads, (heads, keys, channels) seen as (keys, heads, channels): heads may lie as far apart as the offsets of one tile
    allow, 1 GiB for the two maps of a key, any distance for values."""
    import ctypes
    from geotransformer_amd import _lib
    lib, one = _lib.load(), 1 << 20

    def call(**strides):
        view = lambda name, heads, d: kernels.Heads(one, heads, 0, *strides.get(name, (heads * d, d)))  # noqa: E731
        op = kernels.DiffAttn(q=view('q', 8, 16), k=view('k', 4, 16), v=view('v', 2, 32), dtype=0, batch=1, n=0, m=7, dim=16, v_dim=32, lam=one, scale=0.25)
        code = lib.geotr_diff_attn_forward(ctypes.byref(op), one, None, None, None, 0, None)
        return code, lib.geotr_last_error() if code else b''

    assert call(k=(16, 1 << 27), v=(32, 1 << 34), q=(16, 1 << 25)) == (0, b'')
    assert b'strides of k' in call(k=(16, 1 << 28))[1]
    assert b'strides of k' in call(k=(1 << 22, 16))[1] and b'strides of v' in call(v=(1 << 22, 32))[1]
    assert b'strides of v' in call(v=(32, 1 << 62))[1] and b'strides of v' in call(v=(1 << 62, 32))[1]  # their products would pass 64 bits


def test_a_scale_that_wants_a_gradient_is_refused():
    """It would be taken for a number, and its gradient would silently be missing."""
    scale = torch.tensor(0.25, requires_grad=True)
    with pytest.raises(NotImplementedError, match='scale'):
        differential_attention(*_heads(), scale=scale)
    kernels.check_diff_attention(*_heads(), scale=scale.detach())


def test_numbers_of_rows_that_pass_64_bits_are_refused():
    """Their products with the number of sequences came out small, and the call went on with them."""
    import ctypes
    from geotransformer_amd import _lib
    lib, one = _lib.load(), 1 << 20
    view = lambda heads, d: kernels.Heads(one, heads, 0, heads * d, d)  # noqa: E731
    for n, m in ((1 << 62, 7), (5, 1 << 62), ((1 << 62) + 1, 1 << 62), (1 << 31, 7), (5, 1 << 31)):
        op = kernels.DiffAttn(q=view(8, 16), k=view(4, 16), v=view(2, 32), dtype=0, batch=4, n=n, m=m, dim=16, v_dim=32, lam=one, scale=0.25)
        assert lib.geotr_diff_attn_forward(ctypes.byref(op), None, None, None, None, 0, None) == -1 and b'query rows' in lib.geotr_last_error(), (n, m)
        assert lib.geotr_diff_attn_workspace_bytes(ctypes.byref(op)) == lib.geotr_diff_attn_backward_workspace_bytes(ctypes.byref(op)) == 0
    for batch, rows in ((4, 1 << 62), (1 << 62, 4), (1 << 40, 1 << 40), (1 << 32, 1)):
        code = lib.geotr_rotary(ctypes.byref(view(4, 16)), ctypes.byref(view(4, 16)), None, None, 0, batch, rows, 16, 16, 0, one, 1, 0, 1, 0, one, one, 1.0, 0, None)
        assert code == -1 and b'tokens in one call' in lib.geotr_last_error(), (batch, rows)
