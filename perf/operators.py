"""What is measured of the rotary positions and the differential attention: the cases, their inputs, their plain forms and their exact values.

Two operators (geotransformer_amd.modules.transformer):

* rotary positions: heads (..., H, D), one position per token (or one per token and axis, for points); frequency i turns the pair of
  channels (i, i + R/2) (half layout) or (2i, 2i + 1) (interleaved) of the first R channels by position * frequency;
* differential attention: heads in pairs of maps, out_h = (softmax(q_2h k_2h^T s) - lam_h softmax(q_2h+1 k_2h+1^T s)) v_h, for stacked
  clouds (rows, heads, D) with lengths, and for batches (B, rows, heads, D) such as a cache of keys and values.
"""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


# ---- cases ---------------------------------------------------------------------------------------------------------------------------
def _rotary(name, **kw):
    case = dict(kind='rotary', name=name, batch=1, rows=1, heads=8, kv_heads=8, dim=64, rotary_dim=64, interleaved=False, axes=1, dtype='bf16',
                scaling='none', factor=1.0, original=4096, start=0, train=False)
    case.update(kw)
    return case


def _attention(name, **kw):
    case = dict(kind='attention', name=name, stacked=False, batch=1, rows=1, keys=1, spread=0, heads=4, kv_heads=4, dim=32, v_dim=64, dtype='f32',
                causal=False, masked=0.0, ragged=False, train=False, rotary=False)
    case.update(kw)
    return case


def listed():
    return [
        # one new token of one sequence: what a step of serving turns, latency alone
        _rotary('rotary one token', start=1234),
        # a stack of 16 pairs: 32 clouds of some 300 superpoints, both maps of 4 heads of a 256-wide model, a third of the rotation for each axis
        _rotary('rotary stacked superpoints f32', rows=9583, heads=8, kv_heads=8, dim=32, rotary_dim=24, interleaved=True, axes=3, dtype='f32'),
        # a long prompt far beyond the trained length, shared key heads, frequencies stretched by parts
        _rotary('rotary long scaled', rows=32768, heads=32, kv_heads=8, dim=128, rotary_dim=128, scaling='yarn', factor=8.0, original=4096),
        # training: forward and the gradients, half of each head turned, an odd length
        _rotary('rotary train part of head f16', batch=4, rows=2047, heads=16, kv_heads=4, dim=96, rotary_dim=48, interleaved=True, dtype='f16',
                train=True),
        # one query row over a small memory: latency alone
        _attention('attention one row f32', rows=1, keys=257),
        # serving: one token for each of 8 sequences over a cache of up to 32768 keys, four query heads to a key head
        _attention('attention decode', batch=8, rows=1, keys=32768, heads=16, kv_heads=4, dim=64, v_dim=128, dtype='bf16', ragged=True),
        # the framework's own stack: 32 clouds of 250 to 340 superpoints, 4 heads of a 256-wide model, in the default arithmetic
        _attention('attention stacked superpoints f32', stacked=True, batch=32, rows=295, keys=295, spread=45),
        # the same stack in training, some superpoints masked as keys
        _attention('attention stacked train f32', stacked=True, batch=32, rows=295, keys=295, spread=45, masked=0.1, train=True),
        # positions and attention together, as a layer on points uses them, forward and gradients
        _attention('rotary and attention train f32', stacked=True, batch=16, rows=295, keys=295, spread=45, train=True, rotary=True),
        # a long prompt, causal, shared key heads
        _attention('attention long causal', rows=8192, keys=8192, heads=16, kv_heads=4, dim=64, v_dim=128, dtype='bf16', causal=True),
        # training on sequences, causal
        _attention('attention train causal', batch=2, rows=4096, keys=4096, heads=8, kv_heads=8, dim=64, v_dim=128, dtype='bf16', causal=True,
                   train=True),
        # wide heads, odd lengths, padded keys: a dense matching of two point sets
        _attention('attention wide odd f16', batch=2, rows=1531, keys=2777, heads=4, kv_heads=4, dim=128, v_dim=256, dtype='f16', masked=0.1),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.4:
        dim = rng.choice([32, 48, 64, 80, 96, 128])
        axes = rng.choice([1, 1, 3])
        half = dim // 2 // axes
        freqs = half if rng.random() < 0.5 else rng.randint(max(2, half // 2), half)
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4])
        batch = rng.choice([1, 1, 2, 5])
        rows = _log(rng, 1, 24000)
        train = rng.random() < 0.4
        most = 32768 * 40 * 128 // (2 if train else 1)  # elements of the largest listed case
        rows = max(1, min(rows, most // (2 * batch * (heads + kv) * dim)))
        scaling = rng.choice(['none', 'linear', 'ntk', 'yarn']) if axes == 1 else 'none'
        return {k: v for k, v in _rotary(
            '', batch=batch, rows=rows, heads=heads, kv_heads=kv, dim=dim, rotary_dim=2 * axes * freqs, interleaved=rng.random() < 0.5, axes=axes,
            dtype=rng.choice(['f32', 'bf16', 'f16']), scaling=scaling, factor=1.0 if scaling == 'none' else rng.choice([2.0, 4.0, 8.0]),
            original=rng.choice([512, 2048, 4096]), start=_log(rng, 1, 100000) if axes == 1 else 0, train=train).items() if k != 'name'}
    dtype = rng.choice(['f32', 'bf16', 'f16', 'bf16'])
    dim = rng.choice([16, 24, 32, 48, 64, 64, 80, 96, 128])
    v_dim = dim * rng.choice([1, 2, 2])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4])
    form = rng.choice(['stacked', 'stacked', 'one', 'batch'])
    train = form != 'one' and rng.random() < 0.4
    if form == 'stacked':
        batch, rows, keys = rng.randint(1, 32), _log(rng, 16, 700), _log(rng, 16, 700)
        more = dict(stacked=True, batch=batch, rows=rows, keys=keys, spread=min(rows, keys) // 4, masked=rng.choice([0.0, 0.1]))
    elif form == 'one':
        batch, rows, keys = rng.choice([1, 3, 8]), rng.choice([1, 1, 2, 5]), _log(rng, 64, 32768)
        more = dict(batch=batch, rows=rows, keys=keys, ragged=rng.random() < 0.5)
    else:
        batch, rows = rng.choice([1, 2]), _log(rng, 200, 5000)
        causal = rng.random() < 0.5
        keys = rows if causal else _log(rng, 200, 5000)
        more = dict(batch=batch, rows=rows, keys=keys, causal=causal, masked=0.0 if causal else rng.choice([0.0, 0.1]))
    # no more than the largest listed case: its products, and in 32 bits (a sixteenth of the rate) the training stack's some 60 times
    most = (8192 * 8192 // 2 * 16 * 512) / (3 if train else 1) / (8 if dtype == 'f32' else 1)
    while more['batch'] * more['rows'] * more['keys'] * heads * (4 * dim + 2 * v_dim) > most:
        more['rows'] = max(1, more['rows'] * 3 // 4)
        more['keys'] = more['rows'] if more.get('causal') else max(1, more['keys'] * 3 // 4)
        if 'spread' in more:
            more['spread'] = min(more['rows'], more['keys']) // 4
    return {k: v for k, v in _attention('', heads=heads, kv_heads=kv, dim=dim, v_dim=v_dim, dtype=dtype, train=train, **more).items()
            if k != 'name'}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------
def _frequencies(case):
    """Radians per unit of position, 64 bits, one for each turned pair, and the factor on cosine and sine."""
    per_axis = case['rotary_dim'] // 2 // case['axes']
    j = torch.arange(per_axis, dtype=torch.float64, device='cuda')
    base, factor, gain = 10000.0, case['factor'], 1.0
    if case['scaling'] == 'ntk':  # a larger base: the slowest pair slows down by the factor, the fastest keeps its rate
        base = base * factor ** (per_axis / (per_axis - 1.0)) if per_axis > 1 else base
    freq = base ** (-j / per_axis)
    if case['scaling'] == 'linear':
        freq = freq / factor
    if case['scaling'] == 'yarn':  # by parts: pairs that turn 32 times or more within the trained length keep their rate
        turns = case['original'] * freq / (2.0 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / factor)
        gain = 0.1 * math.log(factor) + 1.0
    return freq.repeat(case['axes']), gain


def _lengths(case, generator, mean, spread):
    """Ragged lengths about the mean whose sum is batch * mean."""
    off = torch.randint(-spread, spread + 1, (case['batch'] // 2,), generator=generator)
    off = torch.cat([off, -off, torch.zeros(case['batch'] % 2, dtype=torch.int64)])
    return mean + off[torch.randperm(case['batch'], generator=generator)]


def prepare(case, seed):
    g = torch.Generator('cuda').manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed))  # lengths: a user's program knows them on the host
    dtype = DTYPES[case['dtype']]

    def normal(*shape, scale=1.0):
        x = torch.randn(shape, generator=g, device='cuda', dtype=torch.float32)
        return x.mul_(scale).to(dtype)

    s = {'case': case}
    if case['kind'] == 'rotary':
        lead = (case['batch'], case['rows']) if case['batch'] > 1 else (case['rows'],)
        s['q'] = normal(*lead, case['heads'], case['dim'])
        s['k'] = normal(*lead, case['kv_heads'], case['dim'])
        if case['axes'] == 1:
            pos = case['start'] + torch.arange(case['rows'], device='cuda')
            s['positions'] = pos.expand(lead).contiguous() if case['batch'] > 1 else pos
        else:  # coordinates of superpoints in metres, in units of a coarse voxel
            s['positions'] = torch.rand(lead + (case['axes'],), generator=g, device='cuda') * 60.0 - 30.0
        s['freq'], s['gain'] = _frequencies(case)
        s['axis'] = torch.arange(case['axes'], device='cuda').repeat_interleave(case['rotary_dim'] // 2 // case['axes'])
        if case['train']:
            s['dq'], s['dk'] = normal(*s['q'].shape), normal(*s['k'].shape)
        s['rope'] = _own_rotary(case) if own else None
    else:
        h, hk, d, dv, b = case['heads'], case['kv_heads'], case['dim'], case['v_dim'], case['batch']
        if case['stacked']:
            ql = _lengths(case, host, case['rows'], case['spread'])
            kl = _lengths(case, host, case['keys'], case['spread']) if not case['rotary'] else ql.clone()
            nq, nk = int(ql.sum()), int(kl.sum())
            q_lead, k_lead = (nq,), (nk,)
            s['q_most'], s['k_most'] = int(ql.max()), int(kl.max())
            s['q_lengths'], s['k_lengths'] = ql.cuda(), kl.cuda()
        else:
            q_lead, k_lead = (b, case['rows']), (b, case['keys'])
            s['q_lengths'] = None
            s['k_lengths'] = None
            if case['ragged']:  # a cache filled to another length for each sequence
                s['k_lengths'] = torch.randint(max(1, case['keys'] // 2), case['keys'] + 1, (b,), generator=host).cuda()
        s['q'] = normal(*q_lead, 2 * h, d, scale=1.5)  # scores of a trained layer: a spread of some two units
        s['k'] = normal(*k_lead, 2 * hk, d, scale=1.5)
        s['v'] = normal(*k_lead, hk, dv)
        s['lam'] = torch.rand(h, generator=g, device='cuda') * 0.6 + 0.2
        s['masks'] = (torch.rand(k_lead, generator=g, device='cuda') < case['masked']) if case['masked'] else None
        s['positions'] = torch.rand(q_lead + (3,), generator=g, device='cuda') * 60.0 - 30.0 if case['rotary'] else None
        if case['rotary']:
            turn = _layer_rotary(case)
            s['freq'], s['gain'] = _frequencies(turn)
            s['axis'] = torch.arange(3, device='cuda').repeat_interleave(turn['rotary_dim'] // 6)
            s['rope'] = _own_rotary(turn) if own else None
        if case['train']:
            s['dout'] = normal(*q_lead, h, dv)
    if case['train']:
        for name in ('q', 'k', 'v', 'lam'):
            if name in s:
                s[name].requires_grad_(True)
    return s


def _layer_rotary(case):
    """The rotary part of the case that runs both: three axes, the largest multiple of 24 channels."""
    return _rotary('', heads=2 * case['heads'], kv_heads=2 * case['kv_heads'], dim=case['dim'], rotary_dim=case['dim'] // 24 * 24, axes=3)


def _own_rotary(case):
    from geotransformer_amd.modules.transformer import RotaryPositionalEmbedding
    return RotaryPositionalEmbedding(case['dim'], rotary_dim=case['rotary_dim'], interleaved=case['interleaved'], num_axes=case['axes'],
                                     scaling=None if case['scaling'] == 'none' else case['scaling'], scaling_factor=case['factor'],
                                     original_length=case['original']).cuda()


# ---- plain forms ---------------------------------------------------------------------------------------------------------------------
def _turn(x, cos, sin, rotary_dim, interleaved):
    """x (..., H, D) in 32 bits; cos, sin (..., R/2)."""
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    part, rest = x[..., :rotary_dim], x[..., rotary_dim:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = part[..., :rotary_dim // 2], part[..., rotary_dim // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _plain_rotary(q, k, positions, freq, gain, axis, rotary_dim, interleaved):
    pos = positions.double()
    angle = (pos.unsqueeze(-1) if positions.dim() == q.dim() - 2 else pos[..., axis]) * freq  # far positions: the angle needs 64 bits
    cos, sin = (torch.cos(angle) * gain).float(), (torch.sin(angle) * gain).float()
    return (_turn(q.float(), cos, sin, rotary_dim, interleaved).to(q.dtype), _turn(k.float(), cos, sin, rotary_dim, interleaved).to(k.dtype))


def _rows_of(lengths, most):
    """Row numbers (B, most) of stacked sequences and which of them exist."""
    start = torch.cumsum(lengths, 0) - lengths
    at = torch.arange(most, device=lengths.device)
    return start[:, None] + torch.minimum(at, (lengths[:, None] - 1).clamp(min=0)), at < lengths[:, None]


def _plain_attention(q, k, v, lam, heads, kv_heads, allowed):
    """q (B, n, 2H, D), k (B, m, 2 Hk, D), v (B, m, Hk, Dv); allowed: (B or 1, n or 1, m) truth values or None."""
    b, n, _, d = q.shape
    m, g = k.shape[1], heads // kv_heads
    q5 = q.float().reshape(b, n, kv_heads, g, 2, d).permute(0, 2, 4, 3, 1, 5).reshape(b, kv_heads, 2, g * n, d)
    k5 = k.float().reshape(b, m, kv_heads, 2, d).permute(0, 2, 3, 4, 1)
    v5 = v.float().permute(0, 2, 1, 3).unsqueeze(2)
    scores = torch.matmul(q5, k5).mul(1.0 / math.sqrt(d)).reshape(b, kv_heads, 2, g, n, m)
    if allowed is not None:
        scores = scores.masked_fill(~allowed[:, None, None, None], float('-inf'))
    top = scores.amax(dim=-1, keepdim=True).detach()
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    p = p / p.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(p.reshape(b, kv_heads, 2, g * n, m), v5).reshape(b, kv_heads, 2, g, n, -1)
    out = out[:, :, 0] - lam.reshape(1, kv_heads, g, 1, 1) * out[:, :, 1]
    return out.permute(0, 3, 1, 2, 4).reshape(b, n, heads, -1)


def _plain_layer(s):
    case = s['case']
    q, k, v, lam = s['q'], s['k'], s['v'], s['lam']
    if case['rotary']:
        turn = _layer_rotary(case)
        q, k = _plain_rotary(q, k, s['positions'], s['freq'], s['gain'], s['axis'], turn['rotary_dim'], False)
    if case['stacked']:
        q_at, q_in = _rows_of(s['q_lengths'], s['q_most'])
        k_at, k_in = _rows_of(s['k_lengths'], s['k_most'])
        allowed = k_in if s['masks'] is None else k_in & ~s['masks'][k_at]
        out = _plain_attention(q[q_at], k[k_at], v[k_at], lam, case['heads'], case['kv_heads'], allowed[:, None, :])
        return out[q_in].to(q.dtype)
    n, m = case['rows'], case['keys']
    allowed, keys = None, torch.arange(m, device='cuda')
    if case['causal']:
        allowed = (keys <= torch.arange(n, device='cuda')[:, None] + (m - n))[None]
    if s['k_lengths'] is not None:
        allowed = (keys < s['k_lengths'][:, None])[:, None]
    if s['masks'] is not None:
        allowed = ~s['masks'][:, None]
    return _plain_attention(q, k, v, lam, case['heads'], case['kv_heads'], allowed).to(q.dtype)


# ---- one pass ------------------------------------------------------------------------------------------------------------------------
def run(s):
    case = s['case']
    if case['kind'] == 'rotary':
        if own:
            q, k = s['rope'](s['q'], s['k'], s['positions'])
        else:
            q, k = _plain_rotary(s['q'], s['k'], s['positions'], s['freq'], s['gain'], s['axis'], case['rotary_dim'], case['interleaved'])
        if not case['train']:
            return {'q': q, 'k': k}
        dq, dk = torch.autograd.grad([q, k], [s['q'], s['k']], [s['dq'], s['dk']])
        return {'q': q.detach(), 'k': k.detach(), 'dq': dq, 'dk': dk}
    if own:
        from geotransformer_amd.modules.transformer import differential_attention
        q, k = (s['q'], s['k']) if not case['rotary'] else s['rope'](s['q'], s['k'], s['positions'])
        out = differential_attention(q, k, s['v'], s['lam'], q_lengths=s['q_lengths'], k_lengths=s['k_lengths'], key_masks=s['masks'],
                                     causal=case['causal'])
    else:
        out = _plain_layer(s)
    if not case['train']:
        return {'out': out}
    dq, dk, dv, dlam = torch.autograd.grad(out, [s['q'], s['k'], s['v'], s['lam']], s['dout'])
    return {'out': out.detach(), 'dq': dq, 'dk': dk, 'dv': dv, 'dlam': dlam}


def work(case):
    size = 4 if case['dtype'] == 'f32' else 2
    if case['kind'] == 'rotary':
        rows = case['batch'] * case['rows']
        elements = rows * (case['heads'] + case['kv_heads']) * case['dim']
        times = 2 if case['train'] else 1
        turned = rows * (case['heads'] + case['kv_heads']) * case['rotary_dim']
        return {'bytes': times * 2 * elements * size + rows * case['axes'] * (8 if case['axes'] == 1 else 4), 'flops': times * 3 * turned}
    b, n, m, h, hk, d, dv = (case[x] for x in ('batch', 'rows', 'keys', 'heads', 'kv_heads', 'dim', 'v_dim'))
    keys = m * 3 // 4 if case['ragged'] else m  # what a cache filled to between a half and the whole holds on average
    pairs = b * h * (n * (n + 1) // 2 if case['causal'] else n * keys)
    read = b * size * (n * 2 * h * d + keys * (2 * hk * d + hk * dv))
    out = b * size * n * h * dv
    if not case['train']:
        return {'bytes': read + out, 'flops': pairs * (4 * d + 2 * dv)}  # two products of scores, one of the joined weights with v
    return {'bytes': 2 * read + 2 * out, 'flops': pairs * (4 * d + 2 * dv + 8 * d + 4 * dv)}  # and dq, dk of both maps, dv, and dout v^T


# ---- exact values --------------------------------------------------------------------------------------------------------------------
def _exact_angles(case, positions):
    freq, gain = _frequencies(case)
    per_axis = freq.numel() // case['axes']
    pos = positions.double().reshape(-1, case['axes'])
    return torch.cat([pos[:, a:a + 1] * freq[a * per_axis:(a + 1) * per_axis] for a in range(case['axes'])], dim=1), gain


def _exact_turn(x, angles, gain, rotary_dim, interleaved):
    """Each pair as a complex number, times gain * exp(i angle)."""
    shape = x.shape
    x = x.detach().double().reshape(angles.shape[0], -1, shape[-1]).clone()
    half = rotary_dim // 2
    first, second = (slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)) if interleaved else (slice(0, half), slice(half, rotary_dim))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * torch.polar(torch.full_like(angles, gain), angles)[:, None]
    x[..., first], x[..., second] = z.real, z.imag
    return x.reshape(shape)


def _exact_head(q1, q2, k1, k2, v, lam, scale, allowed, dout):
    """One head of one sequence, 64 bits: the output and, for dout, (dq1, dq2, dk1, dk2, dv, dlam)."""
    def weights(q, k):
        x = (q @ k.t()) * scale
        if allowed is not None:
            x = torch.where(allowed, x, torch.full_like(x, -math.inf))
        w = torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0) if x.shape[1] else x
        return w
    a1, a2 = weights(q1, k1), weights(q2, k2)
    both = a1 - lam * a2
    out = both @ v
    if dout is None:
        return out, None
    dw = dout @ v.t()
    s1, s2 = (a1 * dw).sum(1, keepdim=True), (a2 * dw).sum(1, keepdim=True)
    x1, x2 = a1 * (dw - s1) * scale, a2 * (dw - s2) * (-lam * scale)
    return out, (x1 @ k1, x2 @ k2, x1.t() @ q1, x2.t() @ q2, both.t() @ dout, -s2.sum())


def exact(case, seed):
    s = prepare(case, seed)
    if case['kind'] == 'rotary':
        angles, gain = _exact_angles(case, s['positions'])
        res = {'q': _exact_turn(s['q'], angles, gain, case['rotary_dim'], case['interleaved']),
               'k': _exact_turn(s['k'], angles, gain, case['rotary_dim'], case['interleaved'])}
        if case['train']:
            res['dq'] = _exact_turn(s['dq'], -angles, gain, case['rotary_dim'], case['interleaved'])
            res['dk'] = _exact_turn(s['dk'], -angles, gain, case['rotary_dim'], case['interleaved'])
        return res
    q, k, v, lam = (s[x].detach().double() for x in ('q', 'k', 'v', 'lam'))
    turn = angles = gain = None
    if case['rotary']:
        turn = _layer_rotary(case)
        angles, gain = _exact_angles(turn, s['positions'])
        q, k = (_exact_turn(x, angles, gain, turn['rotary_dim'], False) for x in (q, k))
    lead_q, lead_k = q.shape[:-2], k.shape[:-2]
    q, k, v = q.reshape((-1,) + q.shape[-2:]), k.reshape((-1,) + k.shape[-2:]), v.reshape((-1,) + v.shape[-2:])
    b, g = case['batch'], case['heads'] // case['kv_heads']
    if case['stacked']:
        ql, kl = s['q_lengths'].tolist(), s['k_lengths'].tolist()
        q0 = [sum(ql[:i]) for i in range(b)]
        k0 = [sum(kl[:i]) for i in range(b)]
    else:
        ql, q0, k0 = [case['rows']] * b, [i * case['rows'] for i in range(b)], [i * case['keys'] for i in range(b)]
        kl = [case['keys']] * b if s['k_lengths'] is None else s['k_lengths'].tolist()
    masks = s['masks'].reshape(-1) if s['masks'] is not None else None
    dout = s['dout'].double().reshape(q.shape[0], case['heads'], -1) if case['train'] else None
    out = torch.zeros(q.shape[0], case['heads'], case['v_dim'], dtype=torch.float64, device='cuda')
    dq, dk, dv, dlam = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(lam)
    for i in range(b):
        qs, ks = slice(q0[i], q0[i] + ql[i]), slice(k0[i], k0[i] + kl[i])
        allowed = None
        if case['causal']:
            allowed = torch.ones(ql[i], kl[i], dtype=torch.bool, device='cuda').tril(kl[i] - ql[i])
        if masks is not None:
            allowed = (~masks[ks]).expand(ql[i], kl[i])
        for h in range(case['heads']):
            c = h // g
            out[qs, h], grads = _exact_head(q[qs, 2 * h], q[qs, 2 * h + 1], k[ks, 2 * c], k[ks, 2 * c + 1], v[ks, c], lam[h],
                                            1.0 / math.sqrt(case['dim']), allowed, None if dout is None else dout[qs, h])
            if grads is not None:
                dq[qs, 2 * h], dq[qs, 2 * h + 1] = grads[0], grads[1]
                dk[ks, 2 * c] += grads[2]
                dk[ks, 2 * c + 1] += grads[3]
                dv[ks, c] += grads[4]
                dlam[h] += grads[5]
    res = {'out': out.reshape(lead_q + out.shape[1:])}
    if case['train']:
        if case['rotary']:
            dq, dk = _exact_turn(dq, -angles, gain, turn['rotary_dim'], False), _exact_turn(dk, -angles, gain, turn['rotary_dim'], False)
        res.update(dq=dq.reshape(lead_q + dq.shape[1:]), dk=dk.reshape(lead_k + dk.shape[1:]), dv=dv.reshape(lead_k + dv.shape[1:]), dlam=dlam)
    return res
