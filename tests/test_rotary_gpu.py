"""GPU: rotary positions through the C ABI against the 64-bit form.

Bound of an element: half a step of the type (the one rounding) + 2^-22 of the absolute products (cosine and sine each off by less than
2^-24 + the angle's 2^-25, three roundings of 32 bits) + half a subnormal step + 6 2^-53 of the angle times those products: the frequency
in turns (a quotient, 2 pi) and the product with the position are each rounded to 64 bits in the kernel, and again in the 64-bit form
(2^31 radians are off by 2^-22 in either)."""
import pytest
import torch

import attention_oracle as oracle

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def _want(rope, x, positions, inverse=False):
    pos = positions.cpu().double().reshape(-1, rope.num_axes)
    angles = pos[:, rope.axis.cpu().long()] * (rope.turn_bits.cpu().view(torch.float64) * 2 * torch.pi)
    y, b = oracle.rotary(x.detach().cpu().double().reshape(-1, *x.shape[-2:]), angles, rope.gain, rope.rotary_dim, rope.interleaved, inverse)
    u = oracle.U[x.dtype]
    b = b * (1 + 6 * 2.0 ** -53 * float(angles.abs().max()) / 2.0 ** -22) if angles.numel() else b
    return y.reshape(x.shape), (u * y.abs() + (1 + u) * 2.0 ** -22 * b + oracle.TINY[x.dtype]).reshape(x.shape)


def _check(rope, q, k, positions):
    q, k = q.requires_grad_(), None if k is None else k.requires_grad_()
    yq, yk = rope(q, k, positions)
    oracle.assert_within('q', yq, *_want(rope, q, positions))
    if k is not None:
        oracle.assert_within('k', yk, *_want(rope, k, positions))
    gq = torch.randn(yq.shape, device='cuda').to(q.dtype)
    if k is None:
        dq, = torch.autograd.grad(yq, q, gq)
    else:
        gk = torch.randn(yk.shape, device='cuda').to(q.dtype)
        dq, dk = torch.autograd.grad([yq, yk], [q, k], [gq, gk])
        oracle.assert_within('dk', dk, *_want(rope, gk, positions, inverse=True))
    oracle.assert_within('dq', dq, *_want(rope, gq, positions, inverse=True))


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('lead,heads,kv,dim,rot,axes', [
    ((1,), 8, 8, 64, 64, 1), ((7,), 3, 1, 32, 24, 3), ((2, 33), 4, 2, 96, 48, 1), ((5,), 2, 2, 30, 22, 1), ((3, 1), 1, 1, 128, 126, 3), ((1001,), 2, 1, 8, 2, 1),
    ((2, 17), 2, 1, 1024, 1024, 1), ((4,), 1, 5, 33, 32, 2), ((0,), 4, 2, 64, 64, 1)])
def test_values_and_gradients(dtype, interleaved, lead, heads, kv, dim, rot, axes):
    from geotransformer_amd.modules.transformer import RotaryPositionalEmbedding
    torch.manual_seed(0)
    rope = RotaryPositionalEmbedding(dim, rotary_dim=rot, interleaved=interleaved, num_axes=axes).cuda()
    q, k = (torch.randn(*lead, h, dim, device='cuda').to(DT[dtype]) for h in (heads, kv))
    pos = torch.randint(0, 5000, lead, device='cuda') if axes == 1 else (torch.rand(*lead, axes, device='cuda') - 0.5) * 60
    _check(rope, q, k, pos)


@pytest.mark.parametrize('kw', [dict(scaling='linear', scaling_factor=8.0), dict(scaling='ntk', scaling_factor=4.0),
                                dict(scaling='yarn', scaling_factor=16.0, original_length=4096)])
@pytest.mark.parametrize('start', [0, 10 ** 6, 2 ** 31 - 40])
def test_long_contexts(kw, start):
    """Far positions: an angle of 32 bits would be off by start 2^-24, i.e. by whole radians."""
    from geotransformer_amd.modules.transformer import RotaryPositionalEmbedding
    torch.manual_seed(1)
    rope = RotaryPositionalEmbedding(128, **kw).cuda()
    q, k = torch.randn(33, 4, 128, device='cuda'), torch.randn(33, 2, 128, device='cuda')
    pos = start + torch.arange(33, device='cuda')
    _check(rope, q, k, pos)
    _check(rope, q.detach(), None, pos.to(torch.int32))
    _check(rope, q.detach(), k.detach(), -pos.double())


def test_views_other_orders_and_k_none():
    from geotransformer_amd.modules.transformer import RotaryPositionalEmbedding
    torch.manual_seed(2)
    rope = RotaryPositionalEmbedding(32, rotary_dim=24, num_axes=3).cuda()
    fused = torch.randn(50, 24 * 32, device='cuda')
    q, k = fused[:, :512].unflatten(1, (16, 32)), fused[:, 512:].unflatten(1, (8, 32))  # row stride of the fused projection
    pos = torch.rand(50, 3, device='cuda').t().contiguous().t() * 20  # axes not contiguous
    plain = rope(q.contiguous(), k.contiguous(), pos.contiguous())
    for a, b in zip(rope(q, k, pos), plain):
        assert torch.equal(a, b)
    odd = torch.randn(50, 16, 33, device='cuda')[..., 1:]  # 4-byte alignment only
    assert torch.equal(rope(odd, None, pos)[0], rope(odd.contiguous(), None, pos)[0]) and rope(odd, None, pos)[1] is None
    turned = torch.randn(16, 32, 50, device='cuda').permute(2, 0, 1)  # channels not contiguous
    assert torch.equal(rope(turned, None, pos)[0], rope(turned.contiguous(), None, pos)[0])
    wide = q.expand(3, 50, 16, 32)  # batches that share memory, one position for all
    assert torch.equal(rope(wide, None, pos.expand(3, 50, 3))[0][2], plain[0])
    b16 = torch.randn(2, 9, 4, 32, device='cuda').bfloat16()
    assert torch.equal(rope(b16.transpose(0, 1).contiguous().transpose(0, 1), None, torch.ones(2, 9, 3, device='cuda'))[0],
                       rope(b16, None, torch.ones(2, 9, 3, device='cuda'))[0])


def test_only_one_gradient_and_a_second_derivative():
    from geotransformer_amd.modules.transformer import RotaryPositionalEmbedding
    torch.manual_seed(3)
    rope = RotaryPositionalEmbedding(16).cuda()
    q, k = (torch.randn(6, 2, 16, device='cuda', requires_grad=True) for _ in range(2))
    pos = torch.arange(6, device='cuda')
    yq, yk = rope(q, k, pos)
    g = torch.randn_like(yk, requires_grad=True)
    dk, = torch.autograd.grad(yk, k, g, create_graph=True)
    w = torch.randn_like(dk)
    ddg, = torch.autograd.grad(dk, g, w)
    oracle.assert_within('second', ddg, *_want(rope, w, pos))


def test_a_position_that_is_not_finite_spoils_its_row_only():
    from geotransformer_amd.modules.transformer import RotaryPositionalEmbedding
    rope = RotaryPositionalEmbedding(16).cuda()
    q = torch.randn(4, 2, 16, device='cuda')
    pos = torch.tensor([0.0, float('nan'), 2.0, float('inf')], device='cuda')
    y = rope(q, None, pos)[0]
    good = rope(q, None, torch.tensor([0.0, 1.0, 2.0, 3.0], device='cuda'))[0]
    assert bool(y[1].isnan().all()) and bool(y[3].isnan().all()) and torch.equal(y[0], good[0]) and torch.equal(y[2], good[2])
