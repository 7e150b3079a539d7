"""The transformer-block operators in float64, with bounds of the kernels' errors.

Each function returns the values and, beside each, an elementwise bound derived from the formula:
u |x| for the rounding of the result to its type, u for each rounding of an intermediate to that
type (the probabilities P and their gradient dS enter the matrix products in the operands'
type; the o of the backward pass is the rounded one), and float32 terms for the sums.
"""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
E_P = 2.0 ** -16      # a probability in float32: the score's sum and scaling, the exponential
E_F = 2.0 ** -18      # a float32 sum of products, of the sum of their magnitudes
TINY = {torch.bfloat16: 1e-30, torch.float16: 2.0 ** -24, torch.float32: 1e-30}   # float16's subnormal spacing


def attention(q, k, v, do, o_in, causal, scale, seqs, packed):
    """Per output (value, bound), sequence by sequence and head by head.  seqs: [(q rows, k rows)], slices
    of the packed rows, or (b, ql, kl).  o_in: the rounded o that the backward pass reads."""
    dt = q.dtype
    u = U[dt]
    Hq, Hkv = q.shape[-2], k.shape[-2]
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)     # noqa: E731
    out = {n: (z(t), z(t) + TINY[dt]) for n, t in (('o', q), ('dq', q), ('dk', k), ('dv', v))}
    lse = torch.full((Hq, q.shape[0]) if packed else (q.shape[0], Hq, q.shape[1]), -math.inf, dtype=torch.float64,
                     device=q.device)
    for where in seqs:
        for h in range(Hq):
            g = h // (Hq // Hkv)
            if packed:
                qi, ki, li = (where[0], h), (where[1], g), (h, where[0])
            else:
                b, ql, kl = where
                qi, ki, li = (b, slice(0, ql), h), (b, slice(0, kl), g), (b, h, slice(0, ql))
            Q, K, V = q[qi].double(), k[ki].double(), v[ki].double()
            n, m = len(Q), len(K)
            if n == 0 or m == 0:
                continue
            S = Q @ K.T * scale
            if causal:
                i, j = torch.arange(n, device=q.device)[:, None], torch.arange(m, device=q.device)[None]
                S = S.masked_fill(j > i + m - n, -math.inf)
            ls = torch.logsumexp(S, 1)
            P = torch.exp(S - torch.where(ls.isinf(), torch.zeros_like(ls), ls)[:, None])
            O = P @ V
            out['o'][0][qi], lse[li] = O, ls
            out['o'][1][qi] += u * O.abs() + (u + 2 * E_P) * (P @ V.abs())
            if do is None:
                continue
            G = do[qi].double()
            out['dv'][0][ki] += P.T @ G
            out['dv'][1][ki] += (u + E_P) * (P.T @ G.abs())
            dS = P * (G @ V.T - (G * O).sum(1, keepdim=True))
            err = (u + E_P) * dS.abs() + P * (E_F * (G.abs() @ V.abs().T) + (u + E_F) * (G.abs() * o_in[qi].double().abs()).sum(1, keepdim=True))
            out['dq'][0][qi] = dS @ K * scale
            out['dq'][1][qi] += scale * (err @ K.abs())
            out['dk'][0][ki] += dS.T @ Q * scale
            out['dk'][1][ki] += scale * (err.T @ Q.abs())
    for n in ('dq', 'dk', 'dv'):
        out[n][1].add_(u * out[n][0].abs())
    out['lse'] = (lse, 2 * E_P + E_F * torch.where(lse.isinf(), torch.zeros_like(lse), lse).abs())
    return out


def rotary(x, table, pos, interleaved, inverse):
    """(value, bound) of x (B, T, H, D) turned by positions (B, T, axes)."""
    half, axes = table.shape[1], pos.shape[-1]
    y = x.double().clone()
    mag = torch.zeros_like(y)
    cs = table.double()[pos.long()]
    c, s = cs[..., 0][:, :, None], cs[..., 1][:, :, None] * (-1 if inverse else 1)
    for a in range(axes):
        at = torch.arange(half, device=x.device)
        iu = a * 2 * half + (2 * at if interleaved else at)
        iw = iu + (1 if interleaved else half)
        u, w = x[..., iu].double(), x[..., iw].double()
        y[..., iu], y[..., iw] = u * c[..., a, :] - w * s[..., a, :], w * c[..., a, :] + u * s[..., a, :]
        mag[..., iu], mag[..., iw] = (u * c[..., a, :]).abs() + (w * s[..., a, :]).abs(), (w * c[..., a, :]).abs() + (u * s[..., a, :]).abs()
    return y, U[x.dtype] * y.abs() + 2.0 ** -22 * mag + TINY[x.dtype]


def norm(t, kind, eps, w, b):
    mu = t.mean(-1, keepdim=True) if kind == 'layer' else torch.zeros_like(t[..., :1])
    rstd = ((t - mu).square().mean(-1, keepdim=True) + eps).rsqrt()
    hat = (t - mu) * rstd
    return hat * w + b, hat, rstd, mu


def close(got, want, bound, what):
    got = got.double()
    fine = want.isfinite()
    assert torch.equal(fine, got.isfinite()) and torch.equal(want[~fine], got[~fine]), what
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, \
        f'{what}: off by {float((got - want).abs()[fine].max()):.3e}, {float(over.max()):.3e} over the bound'
