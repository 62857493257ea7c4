"""GPU: the differential attention over more rows, tiles and sequences than an index of 32 bits or one grid holds."""
import pytest
import torch

import attention_oracle as oracle

pytestmark = pytest.mark.gpu


def _repeated(batch, n, m, heads=1, kv=1, d=8, dv=8, dtype=torch.bfloat16, seed=0):
    """`batch` times the same sequence, as views of one."""
    g = torch.Generator('cuda').manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device='cuda').to(dtype)  # noqa: E731
    one = [r(n, 2 * heads, d), r(m, 2 * kv, d), r(m, kv, dv), r(n, heads, dv)]
    return one, [t.expand(batch, *t.shape) for t in one], torch.rand(heads, generator=g, device='cuda')


def test_gradients_of_2_28_query_rows():
    """The rows' numbers take 2^33 bytes: every sequence has the gradients of the first, and these are within their bounds."""
    from geotransformer_amd import kernels
    batch, n, m = 65536, 4096, 8
    one, (q, k, v, dout), lam = _repeated(batch, n, m)
    out, state = kernels.diff_attention(q, k, v, lam, want_state=True)
    dq, dk, dv, dlam = kernels.diff_attention_backward(dout, q, k, v, lam, state)
    want = oracle.differential_attention(one[0], one[1], one[2], lam, dout=one[3])
    for name, got in (('out', out), ('dq', dq), ('dk', dk), ('dv', dv)):
        oracle.assert_within(name, got[0], *want[name])
        for b in range(0, batch, 4096):
            assert bool((got[b:b + 4096] == got[:1]).all()), (name, b)
    value, bound = want['dlam']
    assert float((dlam.cpu().double() / batch - value).abs().max()) <= float((bound + 2.0 ** -23 * value.abs()).max())
    del out, state, dq, dk, dv
    torch.cuda.empty_cache()


@pytest.mark.parametrize('train', [False, True])
@pytest.mark.parametrize('dtype,n,m,heads,kv,d,dv', [(torch.float32, 1, 5, 1, 1, 8, 8), (torch.float32, 3, 62, 1, 1, 8, 8), (torch.bfloat16, 3, 62, 2, 1, 64, 128),
                                                     (torch.bfloat16, 20, 9, 2, 1, 32, 64), (torch.float16, 20, 9, 1, 1, 128, 256),
                                                     (torch.float32, 20, 9, 2, 1, 64, 64)])
def test_stacks_of_more_sequences_than_a_grid_holds_tiles(dtype, n, m, heads, kv, d, dv, train):
    """70 000 times the same sequence, and rows behind the last: forward and both gradients, every form."""
    from geotransformer_amd import kernels
    batch = 70000
    one, _, lam = _repeated(1, n, m, heads, kv, d, dv, dtype)
    q, k, v, dout = (torch.cat([t.repeat(batch, 1, 1), t[:1]]) for t in one)
    lens = [torch.full((batch,), x, dtype=torch.int64, device='cuda') for x in (n, m)]
    want = oracle.differential_attention(one[0], one[1], one[2], lam, dout=one[3])
    if train:
        out, state = kernels.diff_attention(q, k, v, lam, *lens, want_state=True)
        dq, dk, dv_, _ = kernels.diff_attention_backward(dout, q, k, v, lam, state, *lens)
        results = (('out', out, n), ('dq', dq, n), ('dk', dk, m), ('dv', dv_, m))
    else:
        results = (('out', kernels.diff_attention(q, k, v, lam, *lens), n),)
    for name, got, rows in results:
        each = got[:batch * rows].unflatten(0, (batch, rows))
        oracle.assert_within(name, each[0], *want[name])
        assert bool((each == each[:1]).all()), name
        assert not got[batch * rows:].any(), name


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_more_tiles_of_a_head_than_a_grid_holds(dtype):
    """70 000 rows of 64 query heads to a key head in one sequence: 70 000 tiles of 64 packed rows."""
    from geotransformer_amd import kernels
    one, _, lam = _repeated(1, 70000, 5, 64, 1, 8, 8, dtype)
    q, k, v, dout = one
    out, state = kernels.diff_attention(q, k, v, lam, want_state=True)
    assert torch.equal(out, kernels.diff_attention(q, k, v, lam)) or dtype != torch.float32
    dq = kernels.diff_attention_backward(dout, q, k, v, lam, state)[0]
    some = torch.cat([torch.arange(40), torch.arange(65500, 65560), torch.arange(69960, 70000)]).cuda()  # rows do not depend on each other
    want = oracle.differential_attention(q[some], k, v, lam, dout=dout[some])
    oracle.assert_within('out', out[some], *want['out'])
    oracle.assert_within('dq', dq[some], *want['dq'])
    half = [kernels.diff_attention(q[a:b], k, v, lam, want_state=True) for a, b in ((0, 35000), (35000, 70000))]
    assert torch.equal(out, torch.cat([half[0][0], half[1][0]]))


@pytest.mark.parametrize('train', [False, True])
def test_more_heads_of_sequences_than_a_grid_holds(train):
    """2^20 sequences of 8 key heads: 2^23 blocks of 512 threads are 2^32 threads along one axis."""
    from geotransformer_amd import kernels
    batch = 1 << 20
    one, (q, k, v, dout), lam = _repeated(batch, 1, 2, 8, 8, 8, 8, torch.float32)
    want = oracle.differential_attention(one[0], one[1], one[2], lam, dout=one[3])
    if train:
        out, state = kernels.diff_attention(q, k, v, lam, want_state=True)
        results = (('out', out),) + tuple(zip(('dq', 'dk', 'dv'), kernels.diff_attention_backward(dout, q, k, v, lam, state)))
    else:
        results = (('out', kernels.diff_attention(q, k, v, lam)),)
    for name, got in results:
        oracle.assert_within(name, got[0], *want[name])
        assert bool((got == got[:1]).all()), name


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('d,dv', [(32, 64), (64, 128), (128, 256)])
@pytest.mark.parametrize('n,m', [(5, 7), (100, 600), (1, 3), (0, 4)])
def test_a_stack_of_no_sequence(dtype, d, dv, n, m):
    """Lengths of no cloud at all: every row lies behind the last one."""
    from geotransformer_amd.modules.transformer import differential_attention
    one, _, lam = _repeated(1, n, m, 2, 1, d, dv, dtype)
    none = torch.zeros(0, dtype=torch.int64, device='cuda')
    with torch.no_grad():
        assert not differential_attention(*one[:3], lam, none, none).any()
    leaves = [t.requires_grad_() for t in (*one[:3], lam)]
    y = differential_attention(*leaves, none, none)
    assert y.shape == (n, 2, dv) and not y.any()
    for g, t in zip(torch.autograd.grad(y, leaves, torch.full_like(y, float('nan'))), leaves):
        assert g.shape == t.shape and not g.any()


def test_rotary_of_more_sequences_than_a_grid_holds_blocks():
    """2^24 + 3 sequences of one token are 2^32 threads: the same as one sequence of as many tokens."""
    from geotransformer_amd.modules.transformer import RotaryPositionalEmbedding
    rows = (1 << 24) + 3
    rope = RotaryPositionalEmbedding(8).cuda()
    g = torch.Generator('cuda').manual_seed(0)
    q, pos = torch.randn(rows, 1, 8, generator=g, device='cuda').bfloat16(), torch.arange(rows, device='cuda')
    want = rope(q, None, pos)[0]
    got = rope(q[:, None], None, pos[:, None])[0]
    assert torch.equal(got[:, 0], want)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,heads,kv', [(1, 4, 2), (5, 4, 2), (90, 4, 2), (3, 64, 1)])
@pytest.mark.parametrize('d,dv', [(32, 64), (64, 128), (128, 256)])
def test_a_cache_laid_out_by_heads(dtype, n, heads, kv, d, dv):
    """(heads, keys, channels) seen as (keys, heads, channels), heads tens of megabytes apart: the same as contiguous tensors."""
    from geotransformer_amd.modules.transformer import differential_attention
    room, m = 140000 * 32 // d + 8, 333
    g = torch.Generator('cuda').manual_seed(0)
    by_heads = [torch.empty(h, room, c, dtype=dtype, device='cuda').transpose(0, 1) for h, c in ((2 * heads, d), (2 * kv, d), (kv, dv))]
    q, k, v = (t[:r].copy_(torch.randn(r, *t.shape[1:], generator=g, device='cuda')) for t, r in zip(by_heads, (n, m, m)))
    lam = torch.rand(heads, generator=g, device='cuda')
    assert q.stride(1) >= 2 ** 22 and torch.equal(differential_attention(q, k, v, lam), differential_attention(*(t.contiguous() for t in (q, k, v)), lam))
    dout = torch.empty(heads, room, dv, dtype=dtype, device='cuda').transpose(0, 1)[:n].copy_(torch.randn(n, heads, dv, generator=g, device='cuda'))
    grads = []
    for copy in (False, True):
        leaves = [(t.contiguous() if copy else t).detach().requires_grad_() for t in (q, k, v, lam)]
        grads.append(torch.autograd.grad(differential_attention(*leaves), leaves, dout.contiguous() if copy else dout))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_causal_gradients_of_many_more_keys_than_rows(dtype):
    """2 rows of 64 heads to a key head over 50 million equal keys: (keys - rows) x heads passes 2^31.  All scores of a row are the same, so that the
    weights are 1 / keys (sums of equal powers of two are exact) and dv is the same for all keys but the last, which row 0 does not see.
    Bound: each weight rounded to the type and its factors to 32 bits, products and sums in 32 bits, the result rounded once."""
    from geotransformer_amd import kernels
    n, m, heads = 2, 3 * 2 ** 24 + 64, 64
    one, _, lam = _repeated(1, n, 1, heads, 1, 8, 8, dtype)
    q, k, v, dout = one[0], one[1].expand(m, -1, -1), one[2].expand(m, -1, -1), one[3]
    out, state = kernels.diff_attention(q, k, v, lam, causal=True, want_state=True)
    dv = kernels.diff_attention_backward(dout, q, k, v, lam, state, causal=True)[2]
    seen = [torch.tensor([m - 1, m]).double(), torch.tensor([float('inf'), m]).double()]  # keys that the two rows see: of any key, of the last
    u = oracle.U[dtype]
    alike = bool((dv[:-1] == dv[:1]).all())
    assert alike
    for got, count in zip((dv[0], dv[-1]), seen):
        weights = (1 - lam.cpu().double())[None, :, None] / count[:, None, None]
        terms = weights.expand(n, heads, 8) * dout.cpu().double()
        size = ((1 + lam.cpu().double())[None, :, None] / count[:, None, None] * dout.cpu().double().abs()).sum((0, 1))
        value = terms.sum((0, 1))
        bound = u * terms.abs().sum((0, 1)) + 2.0 ** -24 * (n * heads + 16) * size
        oracle.assert_within('dv', got[0], value, bound + u * (value.abs() + bound))
