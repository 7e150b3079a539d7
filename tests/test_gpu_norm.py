"""The norms around a residual connection against their definition in float64, forward and backward."""
import pytest
import torch

from tests import block_reference as R

pytestmark = pytest.mark.gpu
DT = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
E = 2.0 ** -17     # a float32 row statistic and the few operations on it, of the terms' magnitudes


def _make(B, T, C, dtype, stream, kind, post, pre, gate, bias=True, wtype=None, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dt, sd, wt = DT[dtype], DT[stream], DT[wtype or dtype]
    n = lambda *s: torch.randn(*s, device='cuda', generator=g)       # noqa: E731
    pair = lambda: ((1 + 0.2 * n(C)).to(wt), (0.3 * n(C)).to(wt) if bias else None)   # noqa: E731
    kw = dict(kind=kind, eps=1e-5, residual_scale=0.75, post=pair() if post else None, pre=pair() if pre else None)
    shape = {None: None, 'channel': (C,), 'sample': (B, C), 'row1': (B, 1, C), 'token': (B, T, C)}[gate]
    kw['gate'] = None if shape is None else n(*shape).to(wt)
    return (n(B, T, C) + 0.5).to(dt), (2 * n(B, T, C)).to(sd), n(B, T, C).to(sd), n(B, T, C).to(dt), kw


def _gate_of(kw, y):
    g = kw['gate']
    if g is None:
        return torch.ones((), dtype=torch.float64, device=y.device)
    return g.double()[:, None] if g.dim() == 2 else g.double()


def _par(p, C, dev):
    one, zero = torch.ones(C, dtype=torch.float64, device=dev), torch.zeros(C, dtype=torch.float64, device=dev)
    if p is None or p is True:
        return one, zero
    return (one if p[0] is None else p[0].double()), (zero if p[1] is None else p[1].double())


def _norm_err(t, kind, eps, w):
    """Bound of a float32 norm's error: of |hat w|, and of the subtraction of a rounded mean."""
    _, hat, rstd, mu = R.norm(t, kind, eps, w, torch.zeros_like(w))
    return E * (hat.abs() + 1 + rstd * (mu.abs() + t.abs())) * w.abs()


def _forward(y, x, kw):
    C, dev, kind, eps = y.shape[-1], y.device, kw['kind'], kw['eps']
    n, en = y.double(), 0.0
    if kw['post'] is not None:
        w, b = _par(kw['post'], C, dev)
        en = _norm_err(n, kind, eps, w) + E * b.abs()
        n = R.norm(n, kind, eps, w, b)[0]
    g = _gate_of(kw, y)
    r = kw['residual_scale'] * x.double() + g * n
    er = E * (x.double().abs() + (g * n).abs()) + g.abs() * en
    out = {'r': (r, R.U[x.dtype] * r.abs() + er + R.TINY[x.dtype])}
    if kw['pre'] is not None:
        w, b = _par(kw['pre'], C, dev)
        h, hat, rstd, _ = R.norm(r, kind, eps, w, b)
        # an error of r reaches h through the norm, whose derivative is at most rstd (1 + 1 + hat^2 / C ...)
        spread = rstd * (er + er.mean(-1, keepdim=True) + hat.abs() * (er * hat.abs()).mean(-1, keepdim=True)) * w.abs()
        out['h'] = (h, R.U[y.dtype] * h.abs() + _norm_err(r, kind, eps, w) + E * b.abs() + spread + R.TINY[y.dtype])
    return out


def _backward(dr, dh, y, r, kw, gate_sum):
    """The formula's gradients and their bounds."""
    C, dev, kind, eps = y.shape[-1], y.device, kw['kind'], kw['eps']
    lay = kind == 'layer'
    wt = next((p[0].dtype for p in (kw['post'], kw['pre']) if p not in (None, True)), kw['gate'].dtype if kw['gate'] is not None else y.dtype)
    uw = R.U[wt]
    out = {}
    M = lambda t: t.mean(-1, keepdim=True)            # noqa: E731
    d = dr.double()
    ed = E * d.abs()
    rows = tuple(range(y.dim() - 1))

    def cols(name, terms, err):
        s = terms.sum(rows)
        out[name] = (s, uw * s.abs() + (E * terms.abs() + err).sum(rows) + R.TINY[wt])

    def through(z, ez, t, w):
        _, hat, rstd, mu = R.norm(t, kind, eps, w, torch.zeros_like(w))
        ehat = E * (hat.abs() + 1 + rstd * (mu.abs() + t.abs()))
        v = rstd * (z - (M(z) if lay else 0) - hat * M(z * hat))
        ez = ez + E * z.abs()
        e = rstd * (ez + M(ez) + hat.abs() * M(ez * hat.abs() + z.abs() * ehat) + ehat * M((z * hat).abs())
                    + E * (z.abs() + M(z.abs()) + hat.abs() * M((z * hat).abs())))
        return v, e, hat, ehat

    if kw['pre'] is not None:
        w, _ = _par(kw['pre'], C, dev)
        z = dh.double() * w
        v, e, hat, ehat = through(z, 0 * z, r.double(), w)
        cols('dw_pre', dh.double() * hat, dh.double().abs() * ehat)
        cols('db_pre', dh.double(), 0 * z)
        d, ed = d + v, ed + e + E * v.abs()
    dx = kw['residual_scale'] * d
    out['dx'] = (dx, R.U[r.dtype] * dx.abs() + ed + E * dx.abs() + R.TINY[r.dtype])
    w, b = _par(kw['post'], C, dev)
    n, en = y.double(), 0.0
    if kw['post'] is not None:
        n, hat, _, _ = R.norm(n, kind, eps, w, b)
        en = _norm_err(y.double(), kind, eps, w) + E * b.abs()
    if kw['gate'] is not None:
        t, et = d * n, ed * n.abs() + d.abs() * en
        s = gate_sum(t)
        out['dgate'] = (s, uw * s.abs() + gate_sum(E * t.abs() + et) + R.TINY[wt])
    g = _gate_of(kw, y)
    dn, edn = d * g, (ed + E * d.abs()) * g.abs()
    if kw['post'] is not None:
        ehat = E * (hat.abs() + 1 + R.norm(y.double(), kind, eps, w, b)[2] * (2 * y.double().abs()))
        cols('dw_post', dn * hat, edn * hat.abs() + dn.abs() * ehat)
        cols('db_post', dn, edn)
        dn, edn, _, _ = through(dn * w, edn * w.abs(), y.double(), w)
    out['dy'] = (dn, R.U[y.dtype] * dn.abs() + edn + E * dn.abs() + R.TINY[y.dtype])
    return out


def _sum_of(gate, B):
    return {'channel': lambda t: t.sum((0, 1)), 'sample': lambda t: t.sum(1), 'row1': lambda t: t.sum(1, keepdim=True),
            'token': lambda t: t, None: None}[gate]


CASES = [  # B, T, C, dtype, stream, kind, post, pre, gate
    (1, 1, 1024, 'bf16', 'bf16', 'rms', True, True, None),
    (1, 1, 1, 'f32', 'f32', 'layer', True, True, 'channel'),
    (2, 3, 7, 'bf16', 'f32', 'layer', True, True, 'sample'),
    (3, 50, 264, 'f16', 'f16', 'layer', True, True, 'sample'),
    (2, 400, 1000, 'bf16', 'f32', 'rms', False, True, 'channel'),
    (2, 333, 769, 'bf16', 'bf16', 'layer', True, False, 'token'),
    (5, 129, 1032, 'f16', 'f32', 'layer', False, True, 'token'),
    (7, 100, 2056, 'bf16', 'bf16', 'rms', True, True, 'row1'),
    (1, 700, 4096, 'bf16', 'bf16', 'layer', True, True, 'sample'),
    (2, 90, 8192, 'f32', 'f32', 'layer', True, True, 'channel'),
    (2, 9, 8191, 'bf16', 'bf16', 'rms', True, True, 'sample'),
    (4, 65, 96, 'f32', 'f32', 'rms', False, False, 'sample'),
    (1200, 1, 64, 'bf16', 'bf16', 'layer', True, True, 'sample'),
    (3, 5, 48, 'bf16', 'bf16', 'layer', False, False, None),
    (31, 90, 701, 'bf16', 'f32', 'layer', False, False, None),
    (3, 7, 2647, 'f16', 'f32', 'layer', False, True, 'sample'),
    (3, 70, 4097, 'bf16', 'bf16', 'rms', True, True, 'sample'),
    (2, 90, 5120, 'bf16', 'f32', 'layer', True, True, 'sample'),
    (3, 60, 5120, 'bf16', 'bf16', 'rms', True, True, 'channel'),
]


@pytest.mark.parametrize('case', CASES, ids=lambda c: '-'.join(map(str, c)))
def test_forward_and_backward(case):
    from blast3r_b200.norm import residual_norm_backward, residual_norm_forward
    B, T, C, dtype, stream, kind, post, pre, gate = case
    y, x, dr, dh, kw = _make(*case)
    r, h = residual_norm_forward(y, x, **kw)
    want = _forward(y, x, kw)
    R.close(r, *want['r'], 'r')
    if pre:
        R.close(h, *want['h'], 'h')
    else:
        assert h is None
    got = residual_norm_backward(dr, dh if pre else None, y, r, **kw)._asdict()
    want = _backward(dr, dh, y, r, kw, _sum_of(gate, B))
    for name, t in got.items():
        assert (t is None) == (name not in want), name
        if t is not None:
            R.close(t, *want[name], name)
    again = residual_norm_backward(dr, dh if pre else None, y, r, **kw)._asdict()
    assert all(t is None or torch.equal(t, got[n]) for n, t in again.items())     # the same sums every time


def test_float32_weights_no_bias_no_weight():
    from blast3r_b200.norm import residual_norm_backward, residual_norm_forward
    y, x, dr, dh, kw = _make(2, 40, 160, 'bf16', 'f32', 'layer', True, True, 'channel', bias=False, wtype='f32')
    for post, pre in ((kw['post'], kw['pre']), (True, kw['pre'][0]), (kw['post'], True)):
        k2 = dict(kw, post=post, pre=pre)
        norm = dict(k2, post=(None, None) if post is True else post, pre=(None, None) if pre is True else pre if isinstance(pre, tuple) else (pre, None))
        r, h = residual_norm_forward(y, x, **k2)
        want = _forward(y, x, norm)
        R.close(r, *want['r'], 'r'), R.close(h, *want['h'], 'h')
        got = residual_norm_backward(dr, dh, y, r, **k2)._asdict()
        want = _backward(dr, dh, y, r, dict(norm, post=norm['post'] if post is not True else (torch.ones(160, device='cuda'), None)),
                         _sum_of('channel', 2))
        for name in ('dx', 'dy', 'dgate'):
            R.close(got[name], *want[name], name)
        assert (got['dw_post'] is None) == (post is True) and got['db_post'] is None and (got['dw_pre'] is None) == (pre is True)


def test_strided_rows_and_offsets():
    from blast3r_b200.norm import residual_norm_forward
    y, x, _, _, kw = _make(3, 20, 128, 'bf16', 'bf16', 'layer', True, True, 'sample')
    want = residual_norm_forward(y, x, **kw)
    wide = torch.zeros(3, 20, 320, device='cuda', dtype=torch.bfloat16)
    wide[..., 64:192] = y
    odd = torch.zeros(3 * 20 * 128 + 5, device='cuda', dtype=torch.bfloat16)
    odd[5:] = x.flatten()
    cut = torch.zeros(3, 25, 128, device='cuda', dtype=torch.bfloat16)
    cut[:, :20] = x
    for a, b in ((wide[..., 64:192], x), (y, odd[5:].view(3, 20, 128)), (y, cut[:, :20]),
                 (y.transpose(0, 1).contiguous().transpose(0, 1), x)):
        got = residual_norm_forward(a, b, **kw)
        # another layout may add in another order: two roundings to bfloat16 apart at most
        assert all(float((p.double() - q.double()).abs().max()) <= 2 * R.U[torch.bfloat16] * float(q.abs().max()) for p, q in zip(got, want))


def test_zero_and_constant_rows():
    from blast3r_b200.norm import residual_norm_forward
    y = torch.zeros(4, 96, device='cuda')
    x = torch.zeros(4, 96, device='cuda')
    x[1], x[2] = 3.0, 1e4
    r, h = residual_norm_forward(y, x, kind='layer', post=True, pre=True)
    assert torch.equal(r, x) and bool(h.isfinite().all()) and float(h.abs().max()) < 1e-2
    r, h = residual_norm_forward(y, x, kind='rms', post=True, pre=True)
    assert float(h[0].abs().max()) == 0 and float((h[1:3] - 1).abs().max()) < 1e-5


def test_autograd_and_differences():
    """The whole function's gradient, and directional differences of the float64 definition."""
    from blast3r_b200.norm import residual_norm
    for kind in ('layer', 'rms'):
        y, x, dr, dh, kw = _make(3, 11, 40, 'f32', 'f32', kind, True, True, 'sample')
        ts = [y, x, kw['gate'], *kw['post'], *kw['pre']]
        for t in ts:
            t.requires_grad_()
        r, h = residual_norm(y, x, **kw)
        torch.autograd.backward((r, h), (dr, dh))

        def f(step, dirs):
            yy, xx, g, wp, bp, w, b = (t.detach().double() + step * v for t, v in zip(ts, dirs))
            n = R.norm(yy, kind, kw['eps'], wp, bp)[0]
            rr = kw['residual_scale'] * xx + g[:, None] * n
            return (rr * dr.double()).sum() + (R.norm(rr, kind, kw['eps'], w, b)[0] * dh.double()).sum()
        for t in range(7):
            dirs = [torch.randn(v.shape, device='cuda', dtype=torch.float64) if i == t else 0.0 for i, v in enumerate(ts)]
            diff = float(f(1e-5, dirs) - f(-1e-5, dirs)) / 2e-5
            mine = float((ts[t].grad.double() * dirs[t]).sum())
            size = float((ts[t].grad.double() * dirs[t]).abs().sum())
            assert abs(diff - mine) <= 1e-4 * size, (kind, t, diff, mine)


def test_empty_and_stream():
    from blast3r_b200.norm import residual_norm_backward, residual_norm_forward
    y, x, dr, dh, kw = _make(2, 300, 512, 'bf16', 'bf16', 'layer', True, True, 'channel')
    r, h = residual_norm_forward(y[:, :0], x[:, :0], **kw)
    assert r.shape == h.shape == (2, 0, 512)
    g = residual_norm_backward(dr[:, :0], dh[:, :0], y[:, :0], r, **kw)
    assert float(g.dw_post.abs().max()) == 0 and float(g.dgate.abs().max()) == 0
    want = residual_norm_forward(y, x, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = residual_norm_forward(y, x, **kw)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals():
    from blast3r_b200 import _lib as L
    from blast3r_b200.norm import residual_norm_backward, residual_norm_forward
    y, x, dr, dh, kw = _make(2, 6, 64, 'bf16', 'bf16', 'layer', True, True, 'sample')
    for bad in (lambda: residual_norm_forward(y.cpu(), x), lambda: residual_norm_forward(y, x[:1]),
                lambda: residual_norm_forward(y.double(), x), lambda: residual_norm_forward(y, x.half()),
                lambda: residual_norm_forward(y, x, kind='batch'), lambda: residual_norm_forward(y, x, gate=kw['gate'][:, :8]),
                lambda: residual_norm_forward(y, x, gate=y[:, :4]), lambda: residual_norm_forward(y, x, pre=kw['pre'][0][:8]),
                lambda: residual_norm_forward(y, x, pre=kw['pre'][0].half()),
                lambda: residual_norm_backward(dr.float(), dh, y, x, **kw), lambda: residual_norm_backward(dr, None, y, x, **kw)):
        with pytest.raises(RuntimeError):
            bad()
    big = torch.zeros(1, 8193, device='cuda')
    with pytest.raises(L.B3RError, match='channels'):
        residual_norm_forward(big, big)
