"""Plain 64-bit forms of the rotary positions and the differential attention, with the bounds their kernels have to keep.

Bounds are worst cases of the roundings, u = half a step of the type: every P and dS is rounded once to the type before its product, every
result once, and for the gradients the outputs of the maps are summed from P in two parts of the type (u^2 is left) and kept in 32
bits; what is held in 32 bits is off by rho relative to the sum of absolute values, rho = 2 (d + 4) 2^-24 max|s||q||k| (a score
enters a weight and its sum) + (keys + 16) 2^-23 (sums, exponentials)."""
import math

import torch

U = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # half a step of the subnormal numbers


def rotary(x, angles, gain, rotary_dim, interleaved, inverse=False):
    """x (rows, H, D) float64 CPU, angles (rows, R/2) float64 -> (result, sum of absolute products)."""
    y, bound = x.clone(), torch.zeros_like(x)
    half = rotary_dim // 2
    a = slice(0, rotary_dim, 2) if interleaved else slice(0, half)
    b = slice(1, rotary_dim, 2) if interleaved else slice(half, rotary_dim)
    c, s = gain * torch.cos(angles)[:, None], gain * torch.sin(angles)[:, None] * (-1.0 if inverse else 1.0)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    bound[..., a] = bound[..., b] = gain * (x[..., a].abs() + x[..., b].abs())
    return y, bound


def sequences(q, k, q_lengths, k_lengths):
    """[(rows of q, rows of k)] as slices of the flattened rows."""
    if q.dim() == 4:
        n, m = q.shape[1], k.shape[1]
        return [(slice(b * n, b * n + (n if q_lengths is None else q_lengths[b])), slice(b * m, b * m + (m if k_lengths is None else k_lengths[b])))
                for b in range(q.shape[0])]
    if q_lengths is None:
        return [(slice(0, q.shape[0]), slice(0, k.shape[0]))]
    res, i, j = [], 0, 0
    for a, b in zip(q_lengths, k_lengths):
        res.append((slice(i, i + a), slice(j, j + b)))
        i, j = i + a, j + b
    return res


def differential_attention(q, k, v, lam, q_lengths=None, k_lengths=None, key_masks=None, causal=False, scale=None, dout=None):
    """Host lists for lengths; any float type.  Returns {'out': (value, bound), 'dq': ..., 'dk': ..., 'dv': ..., 'dlam': ...} in float64."""
    dtype = q.dtype
    u, tiny = U[dtype], TINY[dtype]
    q4, k4, v4 = (t.detach().cpu().double() for t in (q, k, v))
    lam = lam.detach().cpu().double().expand(q.shape[-2] // 2)
    qf, kf, vf = (t.reshape((-1,) + t.shape[-2:]) for t in (q4, k4, v4))
    masks = None if key_masks is None else key_masks.cpu().reshape(-1)
    heads, hk, d, dv = q.shape[-2] // 2, v.shape[-2], q.shape[-1], v.shape[-1]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    res = {'out': z(qf.shape[0], heads, dv), 'dq': torch.zeros_like(qf), 'dk': torch.zeros_like(kf), 'dv': torch.zeros_like(vf), 'dlam': z(heads)}
    far = {n: torch.zeros_like(t) for n, t in res.items()}
    gf = None if dout is None else dout.detach().cpu().double().reshape(-1, heads, dv)
    for qs, ks in sequences(q, k, q_lengths, k_lengths):
        n, m = qs.stop - qs.start, ks.stop - ks.start
        allowed = torch.ones(n, m, dtype=torch.bool)
        if causal:
            allowed = allowed.tril(m - n)
        if masks is not None:
            allowed &= ~masks[ks]
        used = allowed.any(0)
        for h in range(heads):
            c = h * hk // heads
            P, rho = [], 0.0
            for a in range(2):
                x, y = qf[qs, 2 * h + a], torch.where(used[:, None], kf[ks, 2 * c + a], torch.zeros(()).double())
                s = (x @ y.t()) * scale
                if n and m:
                    rho = max(rho, float((x.abs() @ y.abs().t()).max()) * scale * 2 * (d + 4) * 2.0 ** -24 + (m + 16) * 2.0 ** -23)
                s = torch.where(allowed, s, torch.full_like(s, -math.inf))
                top = s.amax(1, keepdim=True) if m else z(n, 1)
                p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
                P.append(p / p.sum(1, keepdim=True).clamp(min=1e-300))
            val = torch.where(used[:, None], vf[ks, c], torch.zeros(()).double())
            o1, o2 = P[0] @ val, P[1] @ val
            e1, e2 = ((u + rho) * (p @ val.abs()) + tiny * val.abs().sum(0) for p in P)
            out = o1 - lam[h] * o2
            res['out'][qs, h] = out
            e_out = e1 + lam[h].abs() * e2 + 2 * U[torch.float32] * (o1.abs() + lam[h].abs() * o2.abs())
            far['out'][qs, h] = e_out + u * (out.abs() + e_out) + tiny
            if gf is None:
                continue
            g = gf[qs, h]
            # fp16: dS is scaled by a power of two that keeps 2 Dv max|dout| max|v| (times |lam| beyond 1) between 2^14 and 2^15, P by 2^8
            # (less where |lam| > 2^6: 2^14 over the power of two above it) before they are rounded
            power = 2.0 ** max(0, math.ceil(math.log2(max(1.0, float(lam.abs().max())))))
            gs = tiny * 2.0 ** -14 * 2 * dv * float(gf.abs().max()) * float(vf[torch.isfinite(vf)].abs().max()) * power if tiny and m else 0.0
            dp = g @ val.t()
            e_dp = (dv + 2) * 2.0 ** -24 * (g.abs() @ val.abs().t())
            x1, x2 = ((u * u + rho) * (p @ val.abs()) + tiny * val.abs().sum(0) + U[torch.float32] * o.abs() for p, o in zip(P, (o1, o2)))
            d1, d2 = (g * o1).sum(1, keepdim=True), (g * o2).sum(1, keepdim=True)
            e_d1, e_d2 = ((g.abs() * (x + (dv + 4) * 2.0 ** -24 * o.abs())).sum(1, keepdim=True) for x, o in ((x1, o1), (x2, o2)))
            weights = P[0] - lam[h] * P[1]
            absw = P[0] + lam[h].abs() * P[1]
            x1, x2 = P[0] * (dp - d1), -lam[h] * P[1] * (dp - d2)
            f1 = (u + rho) * x1.abs() + (1 + u + rho) * P[0] * (e_dp + e_d1) + rho * P[0] * (dp.abs() + d1.abs()) + gs
            f2 = (u + rho) * x2.abs() + lam[h].abs() * ((1 + u + rho) * P[1] * (e_dp + e_d2) + rho * P[1] * (dp.abs() + d2.abs())) + gs
            k1, k2 = (torch.where(used[:, None], kf[ks, 2 * c + a], torch.zeros(()).double()) for a in range(2))
            acc = 1 + (max(n, m) + 2) * 2.0 ** -24
            for name, at, value, bound in (
                    ('dq', (qs, 2 * h), x1 @ k1, f1 @ k1.abs()), ('dq', (qs, 2 * h + 1), x2 @ k2, f2 @ k2.abs()),
                    ('dk', (ks, 2 * c), x1.t() @ qf[qs, 2 * h], f1.t() @ qf[qs, 2 * h].abs()),
                    ('dk', (ks, 2 * c + 1), x2.t() @ qf[qs, 2 * h + 1], f2.t() @ qf[qs, 2 * h + 1].abs())):
                res[name][at] += value * scale
                far[name][at] += bound * scale * acc + (max(n, m) + 2) * 2.0 ** -24 * bound * scale
            far['dq'][qs, 2 * h] += (m + 2) * 2.0 ** -24 * scale * (x1.abs() @ k1.abs())
            far['dq'][qs, 2 * h + 1] += (m + 2) * 2.0 ** -24 * scale * (x2.abs() @ k2.abs())
            far['dk'][ks, 2 * c] += (n + 2) * 2.0 ** -24 * scale * (x1.abs().t() @ qf[qs, 2 * h].abs())
            far['dk'][ks, 2 * c + 1] += (n + 2) * 2.0 ** -24 * scale * (x2.abs().t() @ qf[qs, 2 * h + 1].abs())
            res['dv'][ks, c] += weights.t() @ g
            # the difference of the two weights is rounded once, relative to itself; each weight is off by rho of its own
            far['dv'][ks, c] += (u * weights.abs() + (rho * (1 + u) + (n + 2) * 2.0 ** -24) * absw).t() @ g.abs() + tiny * max(2.0 ** -8, power * 2.0 ** -14) * g.abs().sum(0)
            res['dlam'][h] -= (P[1] * dp).sum()
            far['dlam'][h] += (P[1] * (e_dp + (rho + 2.0 ** -22 * (m + 2)) * dp.abs())).sum() * (1 + rho)
    for name in ('dq', 'dk', 'dv'):
        far[name] += u * (res[name].abs() + far[name]) + tiny
    far['dlam'] += 2.0 ** -24 * res['dlam'].abs()
    shapes = {'out': q.shape[:-2] + (heads, dv), 'dq': q.shape, 'dk': k.shape, 'dv': v.shape, 'dlam': (heads,)}
    return {n: (res[n].reshape(shapes[n]), far[n].reshape(shapes[n])) for n in res if n == 'out' or dout is not None}


def assert_within(name, got, value, bound):
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert bool(torch.isfinite(got).all()), f'{name}: not finite'
    over = (got - value).abs() - bound
    worst = int(over.argmax()) if over.numel() else 0
    assert over.numel() == 0 or float(over.max()) <= 0, \
        f'{name}: off by {float((got - value).abs().flatten()[worst]):.3e} at {worst}, bound {float(bound.flatten()[worst]):.3e}'
