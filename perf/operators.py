"""The transformer-block operators that are measured: their cases, their plain forms and what they have to move.

Three operators that belong to one block's path, next to the bundle adjustment that refines what
the network answers with: rotary positions, attention (forward, and with its backward pass), and
the norms around a block's residual connection with its gate (forward and backward).

With ``own`` false, ``run`` computes the plain form with elementary torch operations in float32,
rounded once at the end; with ``own`` true it calls ``blast3r_b200``'s entry points.  ``exact``
computes the definition in float64, written apart from the plain form.
"""
import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
SIZE = {'bf16': 2, 'f16': 2, 'f32': 4}


def listed():
    return [
        # attention: serving one new query per sequence over caches of different lengths (latency)
        dict(name='attend one query', op='attention', train=False, form='lens', causal=False, B=6, Lq=1, Lk=2050,
             Hq=16, Hkv=4, D=64, dtype='bf16'),
        # one query over long caches: the work has to be split along the cache (bandwidth)
        dict(name='attend one query long', op='attention', train=False, form='lens', causal=True, B=16, Lq=1,
             Lk=32768, Hq=32, Hkv=8, D=128, dtype='bf16'),
        # the patch tokens (24 x 32, and one more) of a window of 64 frames: the network's forward pass
        dict(name='attend image tokens', op='attention', train=False, form='dense', causal=False, B=64, Lq=769, Lk=769,
             Hq=16, Hkv=16, D=64, dtype='f16'),
        # a long causal prefill with shared key/value heads
        dict(name='attend long causal', op='attention', train=False, form='dense', causal=True, B=1, Lq=16384, Lk=16384,
             Hq=16, Hkv=4, D=128, dtype='bf16'),
        # training on images of different sizes, packed one after the other
        dict(name='train packed images', op='attention', train=True, form='packed', causal=False, B=20, Lq=1025, Lk=1025,
             Hq=16, Hkv=16, D=64, dtype='bf16'),
        # training on long causal sequences with shared key/value heads
        dict(name='train long causal', op='attention', train=True, form='dense', causal=True, B=2, Lq=4096, Lk=4096,
             Hq=32, Hkv=8, D=128, dtype='bf16'),
        # rotary: one new token per sequence, deep in a long context (latency)
        dict(name='rotate one token', op='rotary', B=6, T=1, Hq=16, Hkv=4, D=64, axes=1, rot=64, interleaved=False,
             scaling='linear', inverse=False, n_pos=32768, dtype='bf16'),
        # the patch grid of 64 frames: two position axes over the whole head
        dict(name='rotate image grid', op='rotary', B=64, T=768, Hq=16, Hkv=16, D=64, axes=2, rot=64, interleaved=False,
             scaling='none', inverse=False, n_pos=64, dtype='f16'),
        # the gradient of a partial, interleaved rotation scaled for a long context
        dict(name='rotate long gradient', op='rotary', B=1, T=65536, Hq=32, Hkv=8, D=128, axes=1, rot=64,
             interleaved=True, scaling='yarn', inverse=True, n_pos=65536, dtype='bf16'),
        # norms: one token per sequence between two blocks (latency)
        dict(name='norm one token', op='norm', back=False, B=6, T=1, C=1024, kind='rms', post=True, pre=True,
             gate='none', alpha=1.0, stream='bf16', dtype='bf16'),
        # the patch tokens of 64 frames with a per-channel scale, a float32 residual stream
        dict(name='norm image tokens', op='norm', back=False, B=64, T=769, C=1024, kind='layer', post=False, pre=True,
             gate='channel', alpha=1.0, stream='f32', dtype='bf16'),
        # the backward pass of norms before and after a wide block with a gate per sequence
        dict(name='norm wide gradient', op='norm', back=True, B=8, T=4096, C=4096, kind='rms', post=True, pre=True,
             gate='sample', alpha=0.7, stream='bf16', dtype='bf16'),
    ]


def _loguniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_FLOPS = 1.15e12       # of a drawn attention case, by its full score matrix's share of the listed ones
_MOST_SCORES = 1.1e9        # values of its full score matrix, which the plain form holds
_MOST_BYTES = 1.3e9


def draw(rng):
    while True:
        c = _drawn(rng)
        if c is not None and 3072 not in c.values():
            return c


def _drawn(rng):
    """A case, or None where it would cost more than the listed ones."""
    op = rng.choice(['attention', 'attention', 'rotary', 'norm'])
    if op == 'attention':
        train = rng.random() < 0.5
        form = rng.choice(['dense', 'lens', 'packed'])
        causal = rng.random() < 0.5
        Hkv = rng.choice([1, 2, 3, 4, 8, 12, 16])
        Hq = Hkv * rng.choice([1, 1, 2, 3, 4, 8])
        Lk = _loguniform(rng, 1, 32768)
        Lq = Lk if train or form == 'packed' else rng.choice([1, Lk, _loguniform(rng, 1, Lk)])
        c = dict(op=op, train=train, form=form, causal=causal, B=_loguniform(rng, 1, 32), Lq=Lq, Lk=Lk, Hq=Hq, Hkv=Hkv,
                 D=rng.choice([32, 40, 64, 64, 72, 80, 96, 128, 128]), dtype=rng.choice(['bf16', 'f16']))
        if Hq <= 32 and work(c)['flops'] <= _MOST_FLOPS and work(c)['bytes'] <= _MOST_BYTES \
                and c['B'] * Hq * Lq * Lk <= _MOST_SCORES:
            return c
    elif op == 'rotary':
        axes = rng.choice([1, 1, 2, 3])
        D = rng.choice([48, 64, 96, 120, 128])
        rot = 2 * axes * rng.randint(4, D // (2 * axes))
        Hkv = rng.choice([1, 2, 4, 8, 16])
        c = dict(op=op, B=_loguniform(rng, 1, 64), T=_loguniform(rng, 1, 65536), Hq=Hkv * rng.choice([1, 2, 4]), Hkv=Hkv,
                 D=D, axes=axes, rot=rot, interleaved=rng.random() < 0.5,
                 scaling=rng.choice(['none', 'linear', 'ntk', 'yarn']), inverse=rng.random() < 0.5,
                 n_pos=_loguniform(rng, 64, 65536), dtype=rng.choice(['bf16', 'f16', 'f32']))
        if work(c)['bytes'] <= _MOST_BYTES:
            return c
    else:
        dtype = rng.choice(['bf16', 'f16', 'f32'])
        c = dict(op=op, back=rng.random() < 0.5, B=_loguniform(rng, 1, 64), T=_loguniform(rng, 1, 32768),
                 C=rng.choice([8 * _loguniform(rng, 8, 1024), _loguniform(rng, 33, 8192)]), kind=rng.choice(['layer', 'rms']),
                 post=rng.random() < 0.6, pre=rng.random() < 0.8, gate=rng.choice(['none', 'channel', 'sample', 'token']),
                 alpha=rng.choice([1.0, 0.5]), stream=rng.choice([dtype, 'f32']), dtype=dtype)
        if work(c)['bytes'] <= _MOST_BYTES:
            return c
    return None


# ------------------------------------------------------------------ lengths
def _lengths(case, n, most, empty):
    """Lengths of n sequences up to `most`, the first of them `most`; fixed by the case alone.
    With `empty`, the third of four or more has none (an idle slot of a serving batch)."""
    out = []
    for b in range(n):
        frac = ((b + 1) * 0.6180339887498949) % 1.0
        out.append(most if b == 0 else max(1, int(most * (0.25 + 0.75 * frac))))
    if empty and n >= 4:
        out[2] = 0
    return out


def _sequences(case):
    """Per sequence (queries, keys)."""
    B, Lq, Lk = case['B'], case['Lq'], case['Lk']
    if case['form'] == 'dense':
        return [Lq] * B, [Lk] * B
    kl = _lengths(case, B, Lk, True)
    if case['form'] == 'packed' or Lq == Lk:
        return kl, kl
    return [Lq] * B, kl


def _visible(case):
    """How many (query, key) pairs of one head are visible, over all sequences."""
    n = 0
    for ql, kl in zip(*_sequences(case)):
        if not case['causal']:
            n += ql * kl
        else:                       # query i sees keys j <= i + kl - ql
            lo = max(0, ql - kl)    # rows before it see nothing
            first = lo + kl - ql + 1
            n += (first + kl) * (ql - lo) // 2
    return n


def work(case):
    if case['op'] == 'attention':
        ql, kl = _sequences(case)
        e, D = SIZE[case['dtype']], case['D']
        rq, rk = sum(ql) * case['Hq'], sum(kl) * case['Hkv']
        byts = e * D * (2 * rq + 2 * rk) + 4 * rq
        flops = 4.0 * D * case['Hq'] * _visible(case)
        if case['train']:           # do in, dq, dk, dv out
            byts += e * D * (2 * rq + 2 * rk)
            flops += 10.0 * D * case['Hq'] * _visible(case)
        return {'bytes': float(byts), 'flops': flops}
    if case['op'] == 'rotary':
        n = case['B'] * case['T'] * (case['Hq'] + case['Hkv'])
        table = min(case['n_pos'], case['B'] * case['T']) * case['rot'] // (2 * case['axes']) * 8
        return {'bytes': float(2 * n * case['D'] * SIZE[case['dtype']] + table + 4 * case['B'] * case['T'] * case['axes']),
                'flops': 3.0 * n * case['rot']}
    n = case['B'] * case['T'] * case['C']
    s, e = SIZE[case['stream']], SIZE[case['dtype']]
    g = e * {'none': 0, 'channel': case['C'], 'sample': case['B'] * case['C'], 'token': n}[case['gate']]
    if not case['back']:
        byts = n * (2 * s + e + (e if case['pre'] else 0)) + g
    else:                           # dr, dh, y, r in (y only where something needs it), dx, dy out
        need_y = case['post'] or case['gate'] != 'none'
        byts = n * (s + s + (e if case['pre'] else 0) + (e if need_y else 0) + (s if case['pre'] else 0) + e) + 2 * g
    return {'bytes': float(byts), 'flops': 20.0 * n}


# ------------------------------------------------------------------ inputs
def _frequencies(case):
    """The rotary angles' frequencies, as a user gives them: (list of float, amplitude)."""
    half = case['rot'] // (2 * case['axes'])
    base, dim, factor, original = (100.0 if case['axes'] > 1 else 10000.0), 2 * half, 4.0, case['n_pos'] / 4.0
    if case['scaling'] == 'ntk':
        base *= factor ** (dim / max(dim - 2, 1))
    f = [base ** (-2.0 * k / dim) for k in range(half)]
    if case['scaling'] == 'linear':
        f = [v / factor for v in f]
    if case['scaling'] == 'yarn':   # frequencies that turn rarely within the trained context are interpolated
        lo, hi = (dim * math.log(original / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), dim - 1)
        ramp = [min(max((k - lo) / max(hi - lo, 0.001), 0.0), 1.0) for k in range(half)]
        f = [v / factor * r + v * (1 - r) for v, r in zip(f, ramp)]
        return f, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    dev = 'cuda'
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case['dtype']]

    def normal(*shape, dtype=dt, s=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * s).to(dtype)

    st = {'case': case}
    if case['op'] == 'attention':
        ql, kl = _sequences(case)
        B, D = case['B'], case['D']
        if case['form'] == 'packed':
            qs, ks = (sum(ql),), (sum(kl),)
            cu = [0]
            for n in ql:
                cu.append(cu[-1] + n)
            st['cu'] = torch.tensor(cu, dtype=torch.int32, device=dev)
        else:
            qs, ks = (B, case['Lq']), (B, case['Lk'])
            if case['form'] == 'lens':
                st['q_lens'] = torch.tensor(ql, dtype=torch.int32, device=dev) if case['Lq'] == case['Lk'] else None
                st['k_lens'] = torch.tensor(kl, dtype=torch.int32, device=dev)
        st['q'] = normal(*qs, case['Hq'], D, s=1.5)
        st['k'] = normal(*ks, case['Hkv'], D, s=1.5)
        st['v'] = normal(*ks, case['Hkv'], D)
        if case['train']:
            st['do'] = normal(*qs, case['Hq'], D)
        return st
    if case['op'] == 'rotary':
        B, T, D = case['B'], case['T'], case['D']
        st['q'], st['k'] = normal(B, T, case['Hq'], D), normal(B, T, case['Hkv'], D)
        f, amp = _frequencies(case)
        ang = torch.arange(case['n_pos'], dtype=torch.float64, device=dev)[:, None] * torch.tensor(f, dtype=torch.float64, device=dev)
        st['table'] = torch.stack([ang.cos() * amp, ang.sin() * amp], dim=-1).float().contiguous()   # (n_pos, half, 2)
        st['pos'] = torch.randint(0, case['n_pos'], (B, T, case['axes']), device=dev, generator=g, dtype=torch.int32)
        if case['axes'] == 1 and T > 1 and T <= case['n_pos']:      # running positions, as a sequence has them
            st['pos'] = torch.arange(T, device=dev, dtype=torch.int32).view(1, T, 1).expand(B, T, 1).contiguous()
        return st
    B, T, C = case['B'], case['T'], case['C']
    sd = DTYPES[case['stream']]
    st['y'] = normal(B, T, C)
    st['x'] = normal(B, T, C, dtype=sd, s=2.0)         # the stream: x forward, r backward
    for name, on in (('post', case['post']), ('pre', case['pre'])):
        w = (1 + 0.1 * torch.randn(C, device=dev, generator=g)).to(dt)
        b = (0.1 * torch.randn(C, device=dev, generator=g)).to(dt)
        st[name] = None if not on else (w, b if case['kind'] == 'layer' else None)
    shape = {'none': None, 'channel': (C,), 'sample': (B, C), 'token': (B, T, C)}[case['gate']]
    st['gate'] = None if shape is None else normal(*shape, s=0.5)
    if case['back']:
        st['dr'] = normal(B, T, C, dtype=sd)
        st['dh'] = normal(B, T, C) if case['pre'] else None
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    case = st['case']
    if own:
        return _run_own(st, case)
    return {'attention': _plain_attention, 'rotary': _plain_rotary,
            'norm': _plain_norm_back if case.get('back') else _plain_norm}[case['op']](st, case)


def _run_own(st, case):
    if case['op'] == 'attention':
        from blast3r_b200.attention import attention_backward, attention_forward
        kw = dict(causal=case['causal'])
        if case['form'] == 'packed':
            kw.update(cu_q=st['cu'], cu_k=st['cu'], max_q=case['Lq'], max_k=case['Lk'])
        elif case['form'] == 'lens':
            kw.update(q_lens=st['q_lens'], k_lens=st['k_lens'])
        o, lse = attention_forward(st['q'], st['k'], st['v'], **kw)
        if not case['train']:
            return {'o': o, 'lse': lse}
        dq, dk, dv = attention_backward(st['do'], st['q'], st['k'], st['v'], o, lse, **kw)
        return {'o': o, 'dq': dq, 'dk': dk, 'dv': dv}
    if case['op'] == 'rotary':
        from blast3r_b200.rotary import rotary
        q, k = rotary((st['q'], st['k']), st['table'], st['pos'], interleaved=case['interleaved'], inverse=case['inverse'])
        return {'q': q, 'k': k}
    from blast3r_b200.norm import residual_norm_backward, residual_norm_forward
    kw = dict(kind=case['kind'], post=st['post'], gate=st['gate'], residual_scale=case['alpha'], pre=st['pre'], eps=1e-6)
    if not case['back']:
        r, h = residual_norm_forward(st['y'], st['x'], **kw)
        return {'r': r, 'h': h}
    return dict(residual_norm_backward(st['dr'], st['dh'], st['y'], st['x'], **kw)._asdict())


def _padded(t, cu, L):
    """Packed rows as (B, L, ...), zeros after each sequence's end."""
    at = cu[:-1, None] + torch.arange(L, device=t.device)
    ok = at < cu[1:, None]
    rows = t[at.clamp(max=t.shape[0] - 1).long()]
    return torch.where(ok[:, :, None, None], rows, torch.zeros((), dtype=t.dtype, device=t.device))


def _plain_attention(st, case):
    B, Lq, Lk, Hq, Hkv, D = (case[n] for n in ('B', 'Lq', 'Lk', 'Hq', 'Hkv', 'D'))
    G, scale, dev, dt = Hq // Hkv, D ** -0.5, st['q'].device, st['q'].dtype
    q, k, v, do = st['q'], st['k'], st['v'], st.get('do')
    ql = kl = None
    if case['form'] == 'packed':
        cu = st['cu']
        ql = kl = cu[1:] - cu[:-1]
        q, k, v = _padded(q, cu, Lq), _padded(k, cu, Lk), _padded(v, cu, Lk)
        do = None if do is None else _padded(do, cu, Lq)
    elif case['form'] == 'lens':
        ql, kl = st['q_lens'], st['k_lens']
    ql = torch.full((B,), Lq, device=dev) if ql is None else ql
    kl = torch.full((B,), Lk, device=dev) if kl is None else kl
    i, j = torch.arange(Lq, device=dev)[:, None], torch.arange(Lk, device=dev)[None, :]
    seen = (i < ql[:, None, None]) & (j < kl[:, None, None])                 # (B, Lq, Lk)
    if case['causal']:
        seen = seen & (j <= i + (kl - ql)[:, None, None])
    hide = ~seen[:, None, None]                                              # (B, 1, 1, Lq, Lk)
    heads = lambda t, n: t.float().transpose(1, 2).reshape(B, Hkv, n, -1, D)  # noqa: E731
    qh, kh, vh = heads(q, G), heads(k, 1), heads(v, 1)
    flat = lambda t: t.reshape(B, Hkv, -1, t.shape[-1])                      # noqa: E731
    k2, v2 = kh[:, :, 0], vh[:, :, 0]
    p = (flat(qh * scale) @ k2.transpose(-1, -2)).view(B, Hkv, G, Lq, Lk)
    p.masked_fill_(hide, -math.inf)
    m = p.amax(-1, keepdim=True)
    safe = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p.sub_(safe).exp_()
    l = p.sum(-1, keepdim=True)
    lse = (m + l.log()).squeeze(-1)                                          # -inf where nothing is seen
    p.div_(torch.where(l == 0, torch.ones_like(l), l))
    o = (flat(p) @ v2).view(B, Hkv, G, Lq, D)

    def back(t):                                                             # (B, Hkv, n, L, D) -> the input's layout
        t = t.reshape(B, -1, t.shape[-2], D).transpose(1, 2).to(dt)
        if case['form'] == 'packed':
            at = torch.arange(st['q'].shape[0], device=dev)
            b = torch.bucketize(at, st['cu'][1:].long(), right=True)
            return t[b, at - st['cu'][b]].contiguous()
        return t.contiguous()

    if not case['train']:
        lse = lse.reshape(B, Hq, Lq)
        if case['form'] == 'packed':
            at = torch.arange(st['q'].shape[0], device=dev)
            b = torch.bucketize(at, st['cu'][1:].long(), right=True)
            lse = lse.transpose(1, 2)[b, at - st['cu'][b]].t().contiguous()
        return {'o': back(o), 'lse': lse}
    dh = heads(do, G)
    if case['form'] == 'lens':                                               # rows past a sequence's end give nothing
        dh = dh * (i < ql[:, None, None])[:, None, None]
    dv = (flat(p).transpose(-1, -2) @ flat(dh))[:, :, None]
    delta = (dh * o).sum(-1, keepdim=True)
    ds = (flat(dh) @ v2.transpose(-1, -2)).view(B, Hkv, G, Lq, Lk)
    ds.sub_(delta).mul_(p)
    del p
    dq = (flat(ds) @ k2).view(B, Hkv, G, Lq, D) * scale
    dk = (flat(ds).transpose(-1, -2) @ flat(qh))[:, :, None] * scale
    return {'o': back(o), 'dq': back(dq), 'dk': back(dk), 'dv': back(dv)}


def _plain_rotary(st, case):
    half, axes, rot = case['rot'] // (2 * case['axes']), case['axes'], case['rot']
    cs = st['table'][st['pos'].long()]                                       # (B, T, axes, half, 2)
    c, s = cs[..., 0][:, :, None], cs[..., 1][:, :, None]                    # (B, T, 1, axes, half)
    s = -s if case['inverse'] else s
    out = {}
    for name in ('q', 'k'):
        x = st[name]
        t = x[..., :rot].float().unflatten(-1, (axes, half, 2) if case['interleaved'] else (axes, 2, half))
        u, w = (t[..., 0], t[..., 1]) if case['interleaved'] else (t[..., 0, :], t[..., 1, :])
        z = torch.stack([u * c - w * s, w * c + u * s], dim=-1 if case['interleaved'] else -2).flatten(-3)
        out[name] = torch.cat([z.to(x.dtype), x[..., rot:]], dim=-1)
    return out


def _hat(t, kind, eps=1e-6):
    """(normalised rows, 1 / their scale)."""
    if kind == 'layer':
        t = t - t.mean(-1, keepdim=True)
    rstd = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    return t * rstd, rstd


def _gate(st, case):
    g = st['gate']
    return None if g is None else g.float().view(*({'channel': (1, 1), 'sample': (case['B'], 1)}.get(case['gate'], g.shape[:2])), case['C'])


def _affine(t, wb):
    t = t * wb[0].float()
    return t if wb[1] is None else t + wb[1].float()


def _plain_norm(st, case):
    n = st['y'].float()
    if st['post'] is not None:
        n = _affine(_hat(n, case['kind'])[0], st['post'])
    g = _gate(st, case)
    r = case['alpha'] * st['x'].float() + (n if g is None else g * n)
    h = None if st['pre'] is None else _affine(_hat(r, case['kind'])[0], st['pre']).to(st['y'].dtype)
    return {'r': r.to(st['x'].dtype), 'h': h}


def _hat_back(z, hat, rstd, kind):
    z = z - hat * (z * hat).mean(-1, keepdim=True) - (z.mean(-1, keepdim=True) if kind == 'layer' else 0.0)
    return z * rstd


def _plain_norm_back(st, case):
    out = dict(dx=None, dy=None, dgate=None, dw_post=None, db_post=None, dw_pre=None, db_pre=None)
    dt, kind = st['y'].dtype, case['kind']
    dr = st['dr'].float()
    if st['pre'] is not None:
        hat, rstd = _hat(st['x'].float(), kind)
        dh = st['dh'].float()
        out['dw_pre'] = (dh * hat).sum((0, 1)).to(dt)
        if st['pre'][1] is not None:
            out['db_pre'] = dh.sum((0, 1)).to(dt)
        dr = dr + _hat_back(dh * st['pre'][0].float(), hat, rstd, kind)
    out['dx'] = (case['alpha'] * dr).to(st['x'].dtype)
    n = y = st['y'].float()
    if st['post'] is not None:
        hat, rstd = _hat(y, kind)
        n = _affine(hat, st['post'])
    g = _gate(st, case)
    dn = dr
    if g is not None:
        dg = dr * n
        out['dgate'] = {'channel': lambda: dg.sum((0, 1)), 'sample': lambda: dg.sum(1), 'token': lambda: dg}[case['gate']]().to(dt)
        dn = dr * g
    if st['post'] is not None:
        out['dw_post'] = (dn * hat).sum((0, 1)).to(dt)
        if st['post'][1] is not None:
            out['db_post'] = dn.sum((0, 1)).to(dt)
        dn = _hat_back(dn * st['post'][0].float(), hat, rstd, kind)
    out['dy'] = dn.to(dt)
    return out


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {'attention': _exact_attention, 'rotary': _exact_rotary, 'norm': _exact_norm}[case['op']](st, case)


def _exact_attention(st, case):
    """Sequence by sequence and head by head, on the visible rows and columns only."""
    ql, kl = _sequences(case)
    q, k, v, do = st['q'], st['k'], st['v'], st.get('do')
    out = {n: torch.zeros(t.shape, dtype=torch.float64, device=t.device)
           for n, t in (('o', q), ('dq', q), ('dk', k), ('dv', v))}
    packed = case['form'] == 'packed'
    lse = torch.full((case['Hq'], q.shape[0]) if packed else (case['B'], case['Hq'], case['Lq']), -math.inf,
                     dtype=torch.float64, device=q.device)
    at = 0
    for b, (nq, nk) in enumerate(zip(ql, kl)):
        for h in range(case['Hq']):
            kv = h * case['Hkv'] // case['Hq']
            qi = (slice(at, at + nq), h) if packed else (b, slice(0, nq), h)
            ki = (slice(at, at + nk), kv) if packed else (b, slice(0, nk), kv)
            if nq == 0 or nk == 0:
                continue
            Q, K, V = q[qi].double(), k[ki].double(), v[ki].double()
            S = torch.einsum('id,jd->ij', Q, K) / math.sqrt(case['D'])
            if case['causal']:
                S = S + torch.full_like(S, -math.inf).triu(nk - nq + 1)
            ls = torch.logsumexp(S, dim=1)
            P = torch.exp(S - torch.where(ls.isinf(), torch.zeros_like(ls), ls)[:, None])
            O = P @ V
            out['o'][qi] = O
            lse[(h, slice(at, at + nq)) if packed else (b, h, slice(0, nq))] = ls
            if case['train']:
                dO = do[qi].double()
                out['dv'][ki] += P.T @ dO
                dS = P * (dO @ V.T - (dO * O).sum(1, keepdim=True))
                out['dq'][qi] = dS @ K / math.sqrt(case['D'])
                out['dk'][ki] += dS.T @ Q / math.sqrt(case['D'])
        at += nq
    return out if case['train'] else {'o': out['o'], 'lse': lse}


def _exact_rotary(st, case):
    """As complex numbers: each pair times the unit number of its angle."""
    f, amp = _frequencies(case)
    half, rot = len(f), case['rot']
    ang = st['pos'].double()[..., None] * torch.tensor(f, dtype=torch.float64, device=st['pos'].device)   # (B, T, axes, half)
    turn = torch.polar(torch.full_like(ang, amp), -ang if case['inverse'] else ang)[:, :, None]
    out = {}
    for name in ('q', 'k'):
        x = st[name].double()
        res = x.clone()
        for a in range(case['axes']):
            sec = x[..., a * 2 * half:(a + 1) * 2 * half]
            re, im = (sec[..., 0::2], sec[..., 1::2]) if case['interleaved'] else (sec[..., :half], sec[..., half:])
            z = torch.complex(re, im) * turn[..., a, :]
            sl = (slice(a * 2 * half, (a + 1) * 2 * half, 2), slice(a * 2 * half + 1, (a + 1) * 2 * half, 2)) if case['interleaved'] \
                else (slice(a * 2 * half, a * 2 * half + half), slice(a * 2 * half + half, (a + 1) * 2 * half))
            res[..., sl[0]], res[..., sl[1]] = z.real, z.imag
        out[name] = res
    return out


def _exact_norm(st, case):
    """The forward formula in 64 bits; the gradients by automatic differentiation of it.  The
    backward pass is given r, so x is what makes it: the formula is split at r."""
    def norm(t, wb):
        mu = t.mean(-1, keepdim=True) if case['kind'] == 'layer' else 0.0
        hat = (t - mu) / torch.sqrt(((t - mu) ** 2).mean(-1, keepdim=True) + 1e-6)
        return hat * wb[0] + (0.0 if wb[1] is None else wb[1])

    need = case['back']
    d = lambda t: None if t is None else t.double().requires_grad_(need)      # noqa: E731
    pair = lambda p: None if p is None else (d(p[0]), d(p[1]))                # noqa: E731
    y, x, gate, post, pre = d(st['y']), d(st['x']), d(st['gate']), pair(st['post']), pair(st['pre'])
    n = y if post is None else norm(y, post)
    g = 1.0 if gate is None else gate[:, None] if case['gate'] == 'sample' else gate
    if not need:
        r = case['alpha'] * x + g * n
        return {'r': r, 'h': None if pre is None else norm(r, pre)}
    dr = st['dr'].double()
    if pre is not None:                                                        # x holds r here
        h = norm(x, pre)
        want = [x] + [t for t in pre if t is not None]
        got = torch.autograd.grad(h, want, st['dh'].double())
        dr = dr + got[0]
    branch = g * n
    leaves = {'dy': y, 'dgate': gate, 'dw_post': post and post[0], 'db_post': post and post[1]}
    names = [k for k, t in leaves.items() if t is not None]
    res = dict(zip(names, torch.autograd.grad(branch, [leaves[k] for k in names], dr)))
    out = {k: res.get(k) for k in leaves}
    out.update(dx=case['alpha'] * dr, dw_pre=got[1] if pre is not None else None,
               db_pre=got[2] if pre is not None and pre[1] is not None else None)
    return out
