"""Attention and its backward pass against their definition in float64, within bounds derived from
the roundings, at the lengths, head sizes, layouts and masks where they can go wrong."""
import math

import pytest
import torch

from tests import block_reference as R

pytestmark = pytest.mark.gpu
DT = {'bf16': torch.bfloat16, 'f16': torch.float16}


def _rand(*shape, dtype, seed, s=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(*shape, device='cuda', generator=g) * s).to(dtype)


def _check(q, k, v, do, seqs, packed, causal, scale=None, **kw):
    """Both passes against the definition; returns the outputs."""
    from blast3r_b200.attention import attention_backward, attention_forward, check_attention
    kw.update(causal=causal, scale=scale)
    o, lse = attention_forward(q, k, v, **kw)
    dq, dk, dv = attention_backward(do, q, k, v, o, lse, **kw)
    check_attention()
    want = R.attention(q, k, v, do, o, causal, q.shape[-1] ** -0.5 if scale is None else scale, seqs, packed)
    got = dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv)
    for name in ('o', 'lse', 'dq', 'dk', 'dv'):
        R.close(got[name], *want[name], name)
    return got


def _dense(B, Lq, Lk, Hq, Hkv, D, dtype, seed=0):
    dt = DT[dtype]
    return (_rand(B, Lq, Hq, D, dtype=dt, seed=seed, s=1.5), _rand(B, Lk, Hkv, D, dtype=dt, seed=seed + 1, s=1.5),
            _rand(B, Lk, Hkv, D, dtype=dt, seed=seed + 2), _rand(B, Lq, Hq, D, dtype=dt, seed=seed + 3))


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('B,Lq,Lk,Hq,Hkv,D', [
    (1, 1, 1, 1, 1, 64),
    (2, 1, 300, 8, 2, 64),            # one query over a cache
    (1, 1, 5000, 4, 1, 128),          # a longer one: split along the keys
    (2, 3, 129, 6, 2, 128),           # a few queries, three heads to a group
    (1, 127, 128, 2, 2, 64),
    (1, 128, 128, 1, 1, 128),
    (1, 129, 257, 2, 1, 64),
    (2, 200, 200, 3, 3, 72),          # head sizes that fill no block of 64
    (1, 130, 70, 4, 4, 40),           # more queries than keys: causal leaves rows empty
    (1, 65, 300, 2, 2, 8),
    (1, 300, 300, 5, 1, 96),          # five heads share one
    (1, 513, 513, 2, 1, 128),
    (1, 700, 700, 1, 1, 64),
    (3, 33, 1, 2, 2, 64),             # one key
])
def test_dense(dtype, causal, B, Lq, Lk, Hq, Hkv, D):
    q, k, v, do = _dense(B, Lq, Lk, Hq, Hkv, D, dtype)
    _check(q, k, v, do, [(b, Lq, Lk) for b in range(B)], False, causal)


@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('D', [64, 128])
def test_padded_lengths_with_garbage_past_them(causal, D):
    """Rows past the lengths hold NaN and infinities, which reach nothing; sequences without
    keys, without queries, and with more queries than keys."""
    ql, kl = [200, 1, 0, 77, 130], [300, 0, 50, 129, 64]
    q, k, v, do = _dense(5, 200, 300, 4, 2, D, 'bf16')
    for b in range(5):
        for t, n in ((q, ql), (do, ql), (k, kl), (v, kl)):
            t[b, n[b]:] = math.nan
            t[b, n[b]::2] = math.inf
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device='cuda')       # noqa: E731
    got = _check(q, k, v, do, [(b, ql[b], kl[b]) for b in range(5)], False, causal, q_lens=i32(ql), k_lens=i32(kl))
    for b in range(5):
        assert float(got['o'][b, ql[b]:].abs().sum()) == 0 and bool((got['lse'][b, :, ql[b]:] == -math.inf).all())


@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('Lk', [257, 4000])
def test_one_query_over_padded_caches(causal, Lk):
    """A serving batch: idle slots, one-token caches, lengths that end inside a tile."""
    kl = [Lk, 0, 1, 128, 129, Lk - 1]
    q, k, v, do = _dense(6, 1, Lk, 8, 2, 64, 'bf16')
    for b in range(6):
        k[b, kl[b]:], v[b, kl[b]:] = math.nan, math.nan
    _check(q, k, v, do, [(b, 1, kl[b]) for b in range(6)], False, causal, k_lens=torch.tensor(kl, dtype=torch.int32, device='cuda'))


@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('D,Hq,Hkv', [(64, 2, 2), (128, 6, 2), (80, 2, 1)])
def test_packed(causal, D, Hq, Hkv):
    """Packed sequences, one of them full of NaN: it reaches no other."""
    ql, kl = [130, 0, 1, 257, 40, 90], [130, 33, 100, 257, 0, 200]
    cu = lambda n: torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32, device='cuda')   # noqa: E731
    q, k, v, do = (t[0] for t in _dense(1, sum(ql), sum(kl), Hq, Hkv, D, 'f16'))
    at = lambda n, i: slice(sum(n[:i]), sum(n[:i + 1]))                       # noqa: E731
    seqs = [(at(ql, i), at(kl, i)) for i in range(6)]
    kw = dict(cu_q=cu(ql), cu_k=cu(kl), max_q=257, max_k=257)
    clean = _check(q, k, v, do, seqs, True, causal, **kw)
    from blast3r_b200.attention import attention_backward, attention_forward
    for t, i in ((q, seqs[3][0]), (do, seqs[3][0]), (k, seqs[3][1]), (v, seqs[3][1])):
        t[i] = math.nan
    o, lse = attention_forward(q, k, v, causal=causal, **kw)
    dq, dk, dv = attention_backward(do, q, k, v, o, lse, causal=causal, **kw)
    for n in (0, 1, 2, 4, 5):
        a, b = seqs[n]
        assert torch.equal(o[a], clean['o'][a]) and torch.equal(dq[a], clean['dq'][a])
        assert torch.equal(dk[b], clean['dk'][b]) and torch.equal(dv[b], clean['dv'][b])


@pytest.mark.parametrize('Lq,Lk,causal', [(257, 257, False), (129, 300, True), (257, 100, True), (1, 700, False), (40, 513, False)])
@pytest.mark.parametrize('D', [64, 128])
def test_more_work_than_blocks(Lq, Lk, causal, D):
    """Many heads, so that a block gets several pieces of work one after the other, some of which
    leave half of it idle: last tiles of one row, causal tiles that see nothing, lengths of zero."""
    kl = [Lk, 0, Lk, 1, Lk // 2, Lk, Lk // 3, 130][:8]
    kl = [min(n, Lk) for n in kl]
    q, k, v, do = _dense(8, Lq, Lk, 42, 42, D, 'bf16')
    _check(q, k, v, do, [(b, Lq, kl[b]) for b in range(8)], False, causal, k_lens=torch.tensor(kl, dtype=torch.int32, device='cuda'))


@pytest.mark.parametrize('causal', [False, True])
def test_more_work_than_blocks_three_heads_to_a_group(causal):
    q, k, v, do = _dense(6, 130, 190, 90, 30, 64, 'f16')
    _check(q, k, v, do, [(b, 130, 190) for b in range(6)], False, causal)


def test_strides_and_scale():
    """The three parts of one projection, heads before rows, and a copy where D is not contiguous."""
    B, L, H, D = 2, 150, 3, 64
    qkv = _rand(B, L, 3, H, D, dtype=torch.bfloat16, seed=5)
    do = _rand(B, H, L, D, dtype=torch.bfloat16, seed=6).transpose(1, 2)
    q, k, v = qkv.unbind(2)
    seqs = [(b, L, L) for b in range(B)]
    first = _check(q, k, v, do, seqs, False, True, scale=0.3)
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    second = _check(*heads, do, seqs, False, True, scale=0.3)
    third = _check(q.transpose(1, 3).contiguous().transpose(1, 3), k, v, do, seqs, False, True, scale=0.3)
    off = torch.empty(B * L * H * D + 1, device='cuda', dtype=torch.bfloat16)[1:].view(B, L, H, D).copy_(q)
    fourth = _check(off, k, v, do.contiguous(), seqs, False, True, scale=0.3)
    for other in (second, third, fourth):
        assert all(torch.equal(first[n], other[n]) for n in first)


def test_large_scores():
    """Scores of hundreds, where one key takes everything, and equal scores."""
    q, k, v, do = _dense(1, 150, 260, 2, 1, 64, 'bf16')
    _check(q * 8, k * 8, v, do, [(0, 150, 260)], False, False)
    _check(torch.zeros_like(q), k, v, do, [(0, 150, 260)], False, True)
    q[:], k[:] = -3.0, 3.0                       # every score the same, far below zero
    _check(q, k, v, do, [(0, 150, 260)], False, False)


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('size,scale', [(64.0, None), (2.0 ** -6, None), (1.0, 1e-4), (1.0, 3.0)])
def test_sizes_of_gradients_and_scales(dtype, size, scale):
    """Large and small gradients, and scales far from D^-0.5 (many equal scores; one key that takes all)."""
    q, k, v, do = _dense(1, 200, 300, 4, 2, 64, dtype)
    _check(q, k, v, do * size, [(0, 200, 300)], False, True, scale=scale)


def test_many_sequences():
    """More sequences x heads than a grid's second dimension holds."""
    from blast3r_b200.attention import attention_backward, attention_forward
    B = 70000
    q, k, v, do = (_rand(B, 2, 1, 8, dtype=torch.float16, seed=s) for s in range(4))
    o, lse = attention_forward(q, k, v)
    dq, dk, dv = attention_backward(do, q, k, v, o, lse)
    at = torch.tensor([0, 1, 65535, 65536, B - 1], device='cuda')
    want = R.attention(q[at], k[at], v[at], do[at], o[at], False, 8 ** -0.5, [(b, 2, 2) for b in range(5)], False)
    for name, t in dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv).items():
        R.close(t[at], *want[name], name)


def test_same_results_every_time_and_on_another_stream():
    q, k, v, do = _dense(2, 300, 300, 8, 2, 128, 'bf16')
    from blast3r_b200.attention import attention_backward, attention_forward
    def both():
        o, lse = attention_forward(q, k, v, causal=True)
        return (o, lse, *attention_backward(do, q, k, v, o, lse, causal=True))
    first = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = both()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_autograd_and_differences():
    from blast3r_b200.attention import attention
    q, k, v, do = _dense(1, 40, 60, 4, 2, 32, 'f16')
    for t in (q, k, v):
        t.requires_grad_()
    o = attention(q, k, v, causal=True)
    o.backward(do)
    bound = R.attention(*(t.detach() for t in (q, k, v)), do, o.detach(), True, 32 ** -0.5, [(0, 40, 60)], False)

    def f(step, dirs):
        qq, kk, vv = (t.detach().double()[0].transpose(0, 1) + step * d for t, d in zip((q, k, v), dirs))
        kk, vv = kk.repeat_interleave(2, 0), vv.repeat_interleave(2, 0)
        S = (qq @ kk.transpose(1, 2)) * 32 ** -0.5
        S = S.masked_fill(torch.ones(40, 60, dtype=torch.bool, device='cuda').triu(60 - 40 + 1), -math.inf)
        return ((S.softmax(-1) @ vv) * do.double()[0].transpose(0, 1)).sum()
    for n, t in enumerate((q, k, v)):
        d = torch.randn(t.shape, device='cuda', dtype=torch.float64)
        dirs = [d[0].transpose(0, 1) if i == n else 0.0 for i in range(3)]
        diff = float(f(1e-5, dirs) - f(-1e-5, dirs)) / 2e-5
        mine = float((t.grad.double() * d).sum())
        slack = float((bound[('dq', 'dk', 'dv')[n]][1] * d.abs()).sum()) + 1e-6
        assert abs(diff - mine) <= slack, (n, diff, mine, slack)


def test_empty():
    from blast3r_b200.attention import attention_backward, attention_forward
    for Lq, Lk in ((0, 5), (5, 0), (0, 0)):
        q, k, v, do = _dense(2, Lq, Lk, 2, 2, 64, 'bf16')
        o, lse = attention_forward(q, k, v)
        dq, dk, dv = attention_backward(do, q, k, v, o, lse)
        assert float(sum(t.abs().sum() for t in (o, dq, dk, dv))) == 0 and bool((lse == -math.inf).all())


def test_lengths_outside_of_the_tensors_are_cut():
    from blast3r_b200.attention import attention_forward
    q, k, v, _ = _dense(2, 5, 70, 2, 2, 64, 'bf16')
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device='cuda')       # noqa: E731
    a, _ = attention_forward(q, k, v, k_lens=i32([1 << 30, -4]), q_lens=i32([1 << 30, 5]))
    b, _ = attention_forward(q, k, v, k_lens=i32([70, 0]))
    assert torch.equal(a, b)
    a, _ = attention_forward(q[0], k[0], v[0], cu_q=i32([0, 500]), cu_k=i32([-3, 500]), max_q=5, max_k=1000)
    assert torch.equal(a, attention_forward(q[:1], k[:1], v[:1])[0][0])


def test_refusals():
    from blast3r_b200.attention import attention_backward, attention_forward
    q, k, v, do = _dense(2, 5, 7, 4, 2, 64, 'bf16')
    o, lse = attention_forward(q, k, v)
    i32 = torch.zeros(3, dtype=torch.int32, device='cuda')
    for bad in (lambda: attention_forward(q.float(), k.float(), v.float()), lambda: attention_forward(q, k.half(), v),
                lambda: attention_forward(q.cpu(), k, v), lambda: attention_forward(q, k, v[:, :3]),
                lambda: attention_forward(q[..., :60], k[..., :60], v[..., :60]),
                lambda: attention_forward(q[:, :, :3], k, v), lambda: attention_forward(q[0], k[0], v[0]),
                lambda: attention_forward(q, k, v, k_lens=i32), lambda: attention_forward(q, k, v, k_lens=i32[:2].long()),
                lambda: attention_forward(q[0], k[0], v[0], cu_q=i32), lambda: attention_forward(q, k, v, max_q=3),
                lambda: attention_forward(q[0], k[0], v[0], cu_q=i32, cu_k=i32, max_q=5, max_k=-1),
                lambda: attention_backward(do[:, :2], q, k, v, o, lse), lambda: attention_backward(do, q, k, v, o, lse.double())):
        with pytest.raises(RuntimeError):
            bad()
