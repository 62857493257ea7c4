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
