"""GPU: the forms that the differential attention takes by its sizes (rows over a long axis dealt over blocks, query rows in one or two
groups, few rows), each against the 64-bit form, and what a call's neighbours in memory hold."""
import pytest
import torch

import attention_oracle as oracle
from test_diff_attention_gpu import _check, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('heads,kv,d,dv,causal', [(8, 8, 64, 64, False), (16, 8, 64, 128, True), (8, 8, 128, 128, False), (8, 8, 128, 256, True),
                                                  (40, 20, 32, 64, False), (20, 20, 24, 32, True)])
def test_many_blocks_of_keys(dtype, heads, kv, d, dv, causal):
    """More blocks of 128 keys than run at once: one group of query rows to a block; ragged lengths, rows that see nothing."""
    batch, n, m = 20, 37, 50
    q, k, v, lam, dout = _make(dtype, (batch, n), (batch, m), heads, kv, d, dv)
    ql, kl = [n - i for i in range(batch)], [(7 * i) % (m + 1) for i in range(batch)]
    with torch.no_grad():
        for b in range(batch):
            dout[b, ql[b]:] = 0.0
    _check(q, k, v, lam, dout, ql, kl, causal=causal)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('values', [[-0.5, -1.5, 0.0, 2.0], [0.0, 0.0, 0.0, 0.0], [1e-30, -1e-30, 1.0, -1.0]])
def test_any_lam(dtype, values):
    """Negative weights of the second map, none, and more than one."""
    for heads in ((4, 2), (4, 1)):
        q, k, v, _, dout = _make(dtype, (70,), (90,), *heads, 32, 64)
        _check(q, k, v, torch.tensor(values, device='cuda'), dout)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('heads,kv,d,dv', [(2, 1, 32, 32), (1, 1, 64, 128), (3, 1, 128, 256)])
def test_training_over_a_long_axis(dtype, heads, kv, d, dv):
    """Keys dealt over a few and over many blocks, joined for the gradients too; stacked clouds with rows behind the last."""
    _check(*_make(dtype, (3,), (2500,), heads, kv, d, dv))
    _check(*_make(dtype, (200,), (1100,), heads, kv, d, dv))
    q, k, v, lam, dout = _make(dtype, (50,), (2400,), heads, kv, d, dv)
    with torch.no_grad():
        q[45:], k[2300:], v[2300:], dout[45:] = float('nan'), float('nan'), float('inf'), 0.0
    from geotransformer_amd.modules.transformer import differential_attention
    ql, kl = [20, 25], [900, 1400]
    want = oracle.differential_attention(torch.nan_to_num(q, 0.0), torch.nan_to_num(k, 0.0), torch.nan_to_num(v, 0.0, 0.0, 0.0), lam, ql, kl, dout=dout)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
    y = differential_attention(*leaves, q_lengths=torch.tensor(ql, device='cuda'), k_lengths=torch.tensor(kl, device='cuda'))
    for name, got in zip(('out', 'dq', 'dk', 'dv', 'dlam'), (y,) + torch.autograd.grad(y, leaves, dout)):
        oracle.assert_within(name, got, *want[name])


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('heads,kv,d,dv', [(4, 4, 64, 128), (2, 1, 128, 128), (4, 2, 128, 256), (2, 2, 16, 24)])
@pytest.mark.parametrize('masked', [False, True])
def test_few_rows(dtype, heads, kv, d, dv, masked):
    """One to a few tokens: a wave streams keys of its own (narrow heads) or two groups share tiles of 64 (wide); odd ends, a masked tile."""
    for n, m in ((1, 1), (1, 63), (2, 97), (5, 700), (1, 1300)):
        q, k, v, lam, _ = _make(dtype, (2, n), (2, m), heads, kv, d, dv)
        masks = None
        if masked:
            masks = torch.rand(2, m, generator=torch.Generator('cuda').manual_seed(m), device='cuda') < 0.5
            masks[0, :64] = True  # a whole tile, and all of a short cache
        _check(q, k, v, lam, None, key_masks=masks, causal=n > 1 and n <= m, train=False)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_many_clouds_of_single_rows(dtype):
    """More clouds than a wave has lanes, each one row over keys that are dealt over blocks."""
    ql, kl = [1] * 70, [600 + (i % 7) for i in range(70)]
    q, k, v, lam, dout = _make(dtype, (70,), (sum(kl),), 1, 1, 32, 64)
    _check(q, k, v, lam, dout, ql, kl, train=False)
    _check(q, k, v, lam, dout, ql, kl)


def test_lengths_that_do_not_fit():
    """Lengths beyond the rows that exist are cut, negative ones are zero: nothing behind the arrays is read or written."""
    from geotransformer_amd.modules.transformer import differential_attention
    q, k, v, lam, dout = _make('bf16', (100,), (120,), 2, 1, 32, 64)
    got = differential_attention(q, k, v, lam, torch.tensor([30, -5, 2 ** 40], device='cuda'), torch.tensor([20, 7, 2 ** 40], device='cuda'))
    oracle.assert_within('out', got, *oracle.differential_attention(q, k, v, lam, [30, 0, 70], [20, 7, 93])['out'])
    q, k, v, lam, dout = _make('bf16', (2, 50), (2, 60), 2, 1, 32, 64)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
    y = differential_attention(*leaves, torch.tensor([50, 2 ** 40], device='cuda'), torch.tensor([-1, 2 ** 40], device='cuda'))
    want = oracle.differential_attention(q, k, v, lam, [50, 50], [0, 60], dout=dout)
    for name, g in zip(('out', 'dq', 'dk', 'dv', 'dlam'), (y,) + torch.autograd.grad(y, leaves, dout)):
        oracle.assert_within(name, g, *want[name])


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_hardly_any_difference_between_scores_beyond_2_20(dtype):
    """Scores whose size hides all differences: equal keys give equal weights, the gradients stay finite and those of q vanish."""
    from geotransformer_amd.modules.transformer import differential_attention
    q, k, v, lam, dout = _make(dtype, (40,), (70,), 2, 1, 32, 64)
    with torch.no_grad():
        q.fill_(200.0), k.fill_(-200.0)
        k[:, 1] = 200.0
    leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
    y = differential_attention(*leaves, scale=1.0)
    grads = torch.autograd.grad(y, leaves, dout)
    want = oracle.differential_attention(q * 0, k * 0, v, lam, dout=dout)  # weights 1 / 70
    oracle.assert_within('out', y, *want['out'])
    oracle.assert_within('dv', grads[2], *want['dv'])
    oracle.assert_within('dlam', grads[3], *want['dlam'])
    # dq = 200 sum dS: zero but for the roundings of dS, each |P (dP - del)| u
    u = oracle.U[q.dtype] + 90 * 2.0 ** -23
    dp = torch.einsum('nhv,mv->nhm', dout.double().cpu(), v[:, 0].double().cpu())
    top = 200.0 * 2 * u * (dp.abs() + dp.abs().mean(-1, keepdim=True)).mean(-1) * (1 + 2 * u) * max(1.0, float(lam.max())) + 200.0 * 70 * 2.0 ** -24
    assert bool((grads[0].double().cpu().unflatten(1, (2, 2)).abs().amax((-1, -2)) <= top).all())
    assert all(bool(torch.isfinite(g).all()) for g in grads)


def test_the_states_of_two_calls():
    """The gradient entry takes the state of its own call only, and dout of the output's shape and type."""
    from geotransformer_amd import kernels
    q, k, v, lam, dout = _make('bf16', (40,), (50,), 2, 1, 32, 64)
    _, state = kernels.diff_attention(q, k, v, lam, want_state=True)
    with pytest.raises(ValueError, match='dout is'):
        kernels.diff_attention_backward(dout[:39], q, k, v, lam, state)
    with pytest.raises(ValueError, match='dout is'):
        kernels.diff_attention_backward(dout.float(), q, k, v, lam, state)
    with pytest.raises(ValueError, match='another call'):
        kernels.diff_attention_backward(dout[:39], q[:39], k, v, lam, state)
    with pytest.raises(ValueError, match='one device'):
        kernels.diff_attention_backward(dout.cpu(), q, k, v, lam, state)


def test_nothing_around_the_results_changes():
    """Outputs and gradients of the entry points lie inside a larger allocation: its other bytes stay as they were."""
    import ctypes
    from geotransformer_amd import _lib, kernels
    q, k, v, lam, dout = _make('f16', (33,), (65,), 2, 1, 40, 72)
    lib, e = _lib.load(), 64
    sizes = dict(out=33 * 2 * 72, dq=q.numel(), dk=k.numel(), dv=v.numel())
    room = {n: torch.full((s + 2 * e,), 7.0, dtype=torch.float16, device='cuda') for n, s in sizes.items()}
    at = {n: ctypes.c_void_p(t.data_ptr() + 2 * e) for n, t in room.items()}
    maps, lse = (torch.full((s + 2 * e,), 7.0, device='cuda') for s in (33 * 2 * 2 * 72, 4 * 33 * 2))
    dlam = torch.full((2 + 2 * e,), 7.0, device='cuda')
    op, keep, _ = kernels._diff_attn(q, k, v, lam, None, None, None, False, None)
    need = lib.geotr_diff_attn_backward_workspace_bytes(op)
    ws = torch.full((need + 256,), 9, dtype=torch.uint8, device='cuda')
    stream = _lib.stream_ptr()
    ptr = lambda t, skip: ctypes.c_void_p(t.data_ptr() + skip)  # noqa: E731
    assert lib.geotr_diff_attn_workspace_bytes(op) == 0
    _lib.check(lib.geotr_diff_attn_forward(op, at['out'], ptr(maps, 4 * e), ptr(lse, 4 * e), None, 0, stream), 'forward')
    _lib.check(lib.geotr_diff_attn_backward(op, kernels._HEADS.pack(*kernels._heads(dout)), ptr(maps, 4 * e), ptr(lse, 4 * e), at['dq'], at['dk'], at['dv'],
                                            ptr(dlam, 4 * e), ptr(ws, 0), need, stream), 'backward')
    torch.cuda.synchronize()
    for t in list(room.values()) + [maps, lse, dlam]:
        assert bool((t[:e] == 7).all()) and bool((t[-e:] == 7).all())
    assert bool((ws[need:] == 9).all())
    want = oracle.differential_attention(q, k, v, lam, dout=dout)
    for n, shape in (('out', (33, 2, 72)), ('dq', q.shape), ('dk', k.shape), ('dv', v.shape)):
        oracle.assert_within(n, room[n][e:-e].view(shape), *want[n])
    del keep


@pytest.mark.parametrize('heads,kv,d,dv', [(2, 1, 32, 64), (2, 2, 64, 128), (4, 1, 128, 256)])
def test_large_values_and_lam_in_fp16(heads, kv, d, dv):
    """Gradients of 16-bit floats of narrow range: values up to the type's largest, outputs' gradients large and small, lam beyond 2^6.
    Results beyond the type's largest number are infinite, as their rounding is."""
    from geotransformer_amd.modules.transformer import differential_attention
    for size, grad, lam0, keys in ((10000.0, 1e-3, 1.0, 7), (10000.0, 1e-3, 1.0, 200), (1e-3, 1e-3, 1.0, 100), (1.0, 1.0, 300.0, 90), (1e-3, 1e4, -70.0, 40)):
        q, k, v, lam, dout = _make('f16', (50,), (keys,), heads, kv, d, dv)
        with torch.no_grad():
            v *= size
            dout *= grad
            lam *= lam0
        leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
        y = differential_attention(*leaves)
        want = oracle.differential_attention(q, k, v, lam, dout=dout)
        for name, got in zip(('out', 'dq', 'dk', 'dv', 'dlam'), (y,) + torch.autograd.grad(y, leaves, dout)):
            value, bound = want[name]
            got = got.detach().cpu().double()
            beyond = (value.abs() - bound >= 65520) if name != 'dlam' else torch.zeros_like(value, dtype=torch.bool)  # rounds to infinity
            near = (value.abs() + bound < 65520) | (name == 'dlam')
            assert torch.equal(got[beyond], torch.copysign(torch.full_like(value[beyond], float('inf')), value[beyond])), name
            oracle.assert_within(name, got[near], value[near], bound[near])


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('heads,kv,d,dv', [(4, 2, 32, 64), (2, 2, 64, 128), (2, 1, 128, 256)])
def test_clouds_of_very_different_sizes(dtype, heads, kv, d, dv):
    """Few rows on average, one cloud with many; rows behind the last; keys of one cloud are most of all keys."""
    ql, kl = [150] + [1] * 30, [3] * 30 + [1500]
    q, k, v, lam, _ = _make(dtype, (sum(ql) + 4,), (sum(kl) + 9,), heads, kv, d, dv)
    _check(q, k, v, lam, None, ql, kl, train=False)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_nothing_at_all(dtype):
    """No rows, no keys, no sequences: zeros of the right shapes."""
    from geotransformer_amd.modules.transformer import differential_attention
    for lead_q, lead_k in (((0,), (5,)), ((5,), (0,)), ((0,), (0,)), ((2, 0), (2, 5)), ((2, 5), (2, 0)), ((0, 4), (0, 5))):
        leaves = [t.requires_grad_() for t in _make(dtype, lead_q, lead_k, 4, 2, 32, 64)]
        dout = leaves.pop()
        with torch.no_grad():
            assert not differential_attention(*leaves).any()
        y = differential_attention(*leaves)
        assert y.shape == lead_q + (4, 64) and not y.any()
        for g, t in zip(torch.autograd.grad(y, leaves, dout.detach()), leaves):
            assert g.shape == t.shape and not g.any()


def test_the_same_tensor_in_several_places():
    """q, k and v as slices of one buffer, k as v, dout an expanded value: reads only, gradients add up."""
    from geotransformer_amd.modules.transformer import differential_attention
    x = torch.randn(60, 12, 64, device='cuda', generator=torch.Generator('cuda').manual_seed(2))
    lam = torch.rand(2, device='cuda')
    for q, k, v in ((x[:, :4], x[:, 4:8], x[:, 8:10]), (x[:, :4], x[:, :4], x[:, :2]), (x[:, 3:7], x[:, 4:8], x[:, 4:6])):
        one = differential_attention(q, k, v, lam)
        assert torch.equal(one, differential_attention(q.clone(), k.clone(), v.clone(), lam))
        oracle.assert_within('out', one, *oracle.differential_attention(q, k, v, lam)['out'])
    leaf = x.clone().requires_grad_()
    whole, = torch.autograd.grad(differential_attention(leaf[:, :4], leaf[:, :4], leaf[:, :2], lam).sum(), leaf)
    parts = [t.clone().requires_grad_() for t in (x[:, :4], x[:, :4], x[:, :2])]
    a, b, c = torch.autograd.grad(differential_attention(*parts, lam), parts, torch.ones(60, 2, 64, device='cuda'))
    want = torch.zeros_like(x)
    want[:, :4] += a + b
    want[:, :2] += c
    assert float((whole - want).abs().max()) <= 4 * 2.0 ** -24 * float((a.abs() + b.abs()).max() + c.abs().max())


@pytest.mark.parametrize('d,dv', [(8, 8), (32, 32), (24, 56), (64, 64), (40, 120), (128, 128), (128, 256)])
@pytest.mark.parametrize('heads,kv', [(2, 2), (3, 1), (4, 1)])
def test_one_to_four_rows_in_fp32(d, dv, heads, kv):
    """Rows by vector instructions: one to four packed rows, ends inside a step of a wave, keys dealt over blocks, a causal last row, masks."""
    for n, m, causal in ((1, 1, False), (1, 7, True), (1, 257, False), (2, 64, True), (1, 2600, False), (4 if kv == 2 else 1, 1029, True)):
        q, k, v, lam, _ = _make('f32', (2, n), (2, m), heads, kv, d, dv)
        _check(q, k, v, lam, None, None, [m, m // 2], causal=causal, train=False)
        masks = torch.rand(2, m, generator=torch.Generator('cuda').manual_seed(m), device='cuda') < 0.6
        with torch.no_grad():
            clean = (k.clone(), v.clone())
            k[masks], v[masks] = float('nan'), float('inf')
        from geotransformer_amd.modules.transformer import differential_attention
        got = differential_attention(q, k, v, lam, key_masks=masks, causal=causal)
        oracle.assert_within('out', got, *oracle.differential_attention(q, *clean, lam, key_masks=masks, causal=causal)['out'])
    ql, kl = [1, 0, 3, 1, 9] + [1] * 80, [300, 5, 0, 41, 64] + [3] * 80
    q, k, v, lam, _ = _make('f32', (sum(ql) + 2,), (sum(kl) + 2,), heads, kv, d, dv)
    _check(q, k, v, lam, None, ql, kl, train=False)
    with torch.no_grad():
        q, k = torch.full_like(q[:1], 200.0), torch.full_like(k[:70], -200.0)  # scores beyond 2^20, all the same: the mean of v
        mean = v[:70].double().mean(0).repeat_interleave(heads // kv, 0)
        got = differential_attention(q, k, v[:70], lam, scale=1.0)[0].double()
    assert float((got - (1 - lam.double())[:, None] * mean).abs().max()) <= 2 * 90 * 2.0 ** -23 * float(v[:70].abs().max())


def test_more_blocks_of_both_gradients_than_one_grid():
    """2.1 million rows and keys, all but 300 behind the last cloud: the gradients' blocks (64 rows each) take two launches."""
    from geotransformer_amd.modules.transformer import differential_attention
    clouds, rows = 33, 65024
    q, k, v, lam, dout = _make('f32', (clouds * rows,), (clouds * rows,), 1, 1, 8, 8)
    lens = torch.zeros(clouds, dtype=torch.int64, device='cuda')
    lens[0] = 300  # the rest lies behind the last cloud
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    y = differential_attention(*leaves, q_lengths=lens, k_lengths=lens)
    grads = torch.autograd.grad(y, leaves, dout)
    small = [t[:300].detach().requires_grad_() for t in (q, k, v)] + [lam.detach().requires_grad_()]
    want = oracle.differential_attention(*small, dout=dout[:300])
    for name, got in zip(('out', 'dq', 'dk', 'dv'), (y,) + grads):
        oracle.assert_within(name, got[:300], *want[name])
        assert not got[300:].any()
    oracle.assert_within('dlam', grads[3], *want['dlam'])
