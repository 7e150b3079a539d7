"""Attention where blocks, layouts and values meet their edges, against the definition in float64 (the bounds of
``block_reference``)."""
import math

import pytest
import torch

from tests import block_reference as R
from tests.test_gpu_attention import DT, _check, _dense, _rand

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device='cuda')


def _cu(n):
    return _i32([sum(n[:i]) for i in range(len(n) + 1)])


def _seqs(ql, kl):
    at = lambda n, i: slice(sum(n[:i]), sum(n[:i + 1]))                       # noqa: E731
    return [(at(ql, i), at(kl, i)) for i in range(len(ql))]


# ---------------------------------------------------------------- heads to a group that do not divide 128
@pytest.mark.parametrize('G', [3, 5])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('causal', [False, True])
def test_idle_halves_where_the_groups_write_q(G, D, causal):
    """Many short packed sequences under a longer one: the second half of most blocks' rows is empty, for jobs in a row."""
    ql = [(7 * i) % 40 + 1 for i in range(300)]
    ql[17] = ql[211] = 400
    kl = [n + (11 * i) % 300 for i, n in enumerate(ql)]
    q, k, v, do = (t[0] for t in _dense(1, sum(ql), sum(kl), 2 * G, 2, D, 'bf16'))
    _check(q, k, v, do, _seqs(ql, kl), True, causal, cu_q=_cu(ql), cu_k=_cu(kl), max_q=max(ql), max_k=max(kl))


@pytest.mark.parametrize('G', [3, 5])
@pytest.mark.parametrize('D', [64, 128])
def test_idle_first_halves_where_the_groups_write_q(G, D):
    """Causal with more queries than keys: the first half of many blocks' rows sees nothing; and last tiles of few rows."""
    B, Lq, Lk = 40, 520 // G, 300
    kl = [(13 * b) % 60 + (200 if b % 5 == 0 else 1) for b in range(B)]
    q, k, v, do = _dense(B, Lq, Lk, 4 * G, 4, D, 'f16')
    _check(q, k, v, do, [(b, Lq, kl[b]) for b in range(B)], False, True, k_lens=_i32(kl))


# ---------------------------------------------------------------- values far from one
@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('size,scale', [(300.0, 1e-6), (3000.0, 2e-8), (0.5, 1e-9), (0.5, 1e-30)])
def test_statistics_of_any_size_in_raw_scores(dtype, size, scale):
    """lse / scale on both sides of 1.7e7, the end of 256 times a float16, with scores of ordinary size."""
    q, k, v, do = _dense(1, 200, 300, 4, 2, 128, dtype)
    q, k = q * (size / 1.5), k * (size / 1.5)
    _check(q, k, v, do, [(0, 200, 300)], False, True, scale=scale)


def test_large_deltas():
    """do . o above 1.7e7 in float16, beside queries of ordinary size and hidden ones."""
    q, k, v, do = _dense(2, 150, 260, 2, 1, 128, 'f16')
    sign = torch.where(_rand(128, dtype=torch.float32, seed=9) > 0, 1.0, -1.0)
    v = (20.0 * v + 200.0 * sign).half()
    do[:, ::3] = (30.0 * do[:, ::3] + 1000.0 * sign).half()
    q, k = q * 0.01, k * 0.01
    _check(q, k, v, do, [(0, 150, 260), (1, 90, 40)], False, True, q_lens=_i32([150, 90]), k_lens=_i32([260, 40]))


def test_raw_scores_past_float16_stay_finite():
    """Raw scores of 2e7 and more at the default scale: one key takes everything."""
    q, k, v, do = _dense(1, 130, 140, 1, 1, 128, 'f16')
    q, k = q.sign() * 500.0 + q, k.sign() * 500.0 + k
    k[:, ::7] = q[:, :20]
    from blast3r_b200.attention import attention_backward, attention_forward
    o, lse = attention_forward(q, k, v)
    assert float(lse.max()) > 1.7e7 * 128 ** -0.5
    assert all(bool(t.isfinite().all()) for t in (o, lse, *attention_backward(do, q, k, v, o, lse)))


def test_many_small_probabilities_beside_a_large_one():
    """One key takes nearly all, and many share the rest: their probabilities lie below float16's numbers."""
    for Lq, Lk in ((1, 30000), (140, 30000)):
        q = torch.zeros(1, Lq, 2, 64, device='cuda', dtype=torch.float16)
        k = torch.zeros(1, Lk, 1, 64, device='cuda', dtype=torch.float16)
        q[..., 0], k[:, 0, :, 0] = 8.0, 17.3 / 8.0
        v = torch.ones(1, Lk, 1, 64, device='cuda', dtype=torch.float16)
        v[:, 0] = 0.0
        _check(q, k, v, torch.ones_like(q), [(0, Lq, Lk)], False, False, scale=1.0)


# ---------------------------------------------------------------- NaN
@pytest.mark.parametrize('D', [64, 128])
def test_nan_of_a_split_row_stays(D):
    """A row of NaN scores is NaN, split along the keys or not; a NaN value or key reaches the rows that see it."""
    from blast3r_b200.attention import attention_forward
    q, k, v, _ = _dense(3, 1, 5000, 4, 2, D, 'bf16')
    q[0, 0, 1] = math.nan
    k[1, 3, 1] = math.nan
    kl = [5000, 60, 0]
    for n in (5000, 100):                       # split along the keys, and not
        o, lse = attention_forward(q, k[:, :n].contiguous(), v[:, :n].contiguous(), k_lens=_i32([min(n, x) for x in kl]))
        assert bool(o[0, 0, 1].isnan().all()) and bool(lse[0, 1].isnan())
        assert bool(o[1, 0, 2:].isnan().all()) and bool(lse[1, 2:].isnan().all())
        assert bool(o[0, 0, [0, 2, 3]].isfinite().all()) and bool(o[1, 0, :2].isfinite().all())
        assert float(o[2].abs().max()) == 0 and bool((lse[2] == -math.inf).all())


# ---------------------------------------------------------------- packed rows of no sequence
def _poison(n=64 << 20):
    """Leaves NaN in the memory that the next outputs are made of."""
    ts = [torch.full((n >> s,), math.nan, device='cuda') for s in range(0, 20, 2) for _ in range(2)]
    del ts


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('lens', [([130, 0, 1, 57], [60, 33, 0, 257]), ([3], [2]), ([0, 0], [0, 0])])
def test_packed_rows_of_no_sequence(dtype, lens):
    """Rows before the first sequence, past the last one, and past max_q / max_k: o = 0, lse = -inf, no gradients."""
    from blast3r_b200.attention import attention_backward, attention_forward
    ql, kl = lens
    most_q, most_k = max(max(ql) - 5, 1), max(max(kl) - 9, 1)
    cq, ck = [17 + sum(ql[:i]) for i in range(len(ql) + 1)], [5 + sum(kl[:i]) for i in range(len(kl) + 1)]
    q, k, v, do = (t[0] for t in _dense(1, cq[-1] + 300, ck[-1] + 131, 6, 2, 72, dtype))
    seqs = [(slice(cq[i], cq[i] + min(n, most_q)), slice(ck[i], ck[i] + min(m, most_k))) for i, (n, m) in enumerate(zip(ql, kl))]
    off_q, off_k = (torch.ones(n, dtype=torch.bool, device='cuda') for n in (len(q), len(k)))
    for a, b in seqs:
        off_q[a], off_k[b] = False, False
    for t, off in ((q, off_q), (do, off_q), (k, off_k), (v, off_k)):
        t[off] = math.nan
    kw = dict(cu_q=_i32(cq), cu_k=_i32(ck), max_q=most_q, max_k=most_k)
    _poison()
    o, lse = attention_forward(q, k, v, **kw)
    assert float(o[off_q].abs().max()) == 0 and bool((lse[:, off_q] == -math.inf).all())
    _poison()
    grads = attention_backward(do, q, k, v, o, lse, **kw)
    for g, off in zip(grads, (off_q, off_k, off_k)):
        assert float(g[off].abs().max()) == 0 and bool(g.isfinite().all())
    want = R.attention(q, k, v, do, o, False, 72 ** -0.5, seqs, True)
    for name, t in zip(('o', 'lse', 'dq', 'dk', 'dv'), (o, lse, *grads)):
        R.close(t, *want[name], name)


def test_packed_bounds_of_zero():
    """max_q or max_k of zero: nothing sees anything, and the outputs are still whole."""
    from blast3r_b200.attention import attention_backward, attention_forward
    q, k, v, do = (t[0] for t in _dense(1, 40, 50, 2, 2, 64, 'bf16'))
    for mq, mk in ((0, 50), (40, 0), (0, 0)):
        kw = dict(cu_q=_i32([0, 40]), cu_k=_i32([0, 50]), max_q=mq, max_k=mk)
        _poison()
        o, lse = attention_forward(q, k, v, **kw)
        _poison()
        grads = attention_backward(do, q, k, v, o, lse, **kw)
        assert all(float(t.abs().max()) == 0 for t in (o, *grads)) and bool((lse == -math.inf).all())


# ---------------------------------------------------------------- the status word
def test_a_raised_status_is_reported_once():
    from blast3r_b200 import _lib as L
    from blast3r_b200 import attention as A
    q, k, v, _ = _dense(1, 5, 7, 2, 2, 64, 'bf16')
    A.attention_forward(q, k, v)
    A.check_attention()
    for device in (None, 'cuda', 0, q.device):
        L.status_word('attention', q.get_device()).fill_(1)
        with pytest.raises(L.B3RError, match='ran out'):
            A.check_attention(device)
        A.check_attention(device)


def test_the_first_call_under_capture_has_a_status():
    """A graph captured by a process's first call reports failures as every other call."""
    import subprocess
    import sys
    code = '''
import torch
from blast3r_b200 import attention as A
q, k, v = (torch.randn(2, 300, 4, 64, device='cuda').bfloat16() for _ in range(3))
torch.cuda.synchronize()
seen = []
launch, A._launch = A._launch, lambda name, d, *a: (launch(name, d, *a), seen.append(d.status))
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    o, lse = A.attention_forward(q, k, v)
    grads = A.attention_backward(o, q, k, v, o, lse)
assert len(seen) == 2 and all(seen)
from blast3r_b200 import _lib as L
assert seen[0] == seen[1] == L.status_word('attention', 0).data_ptr()
g.replay()
A.check_attention()
want = A.attention_forward(q, k, v)
assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
assert all(torch.equal(a, b) for a, b in zip(grads, A.attention_backward(want[0], q, k, v, *want)))
q.mul_(0.5)
g.replay()
assert torch.equal(o, A.attention_forward(q, k, v)[0])
print('fine')
'''
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, '-c', code], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and 'fine' in out.stdout, out.stderr[-2000:]


# ---------------------------------------------------------------- arguments
def test_scales_out_of_range_are_refused():
    from blast3r_b200.attention import attention_forward
    q, k, v, _ = _dense(1, 5, 7, 2, 2, 64, 'bf16')
    for scale in (math.inf, 1e300, 1e-39, math.nan, 0.0, -1.0):
        with pytest.raises(RuntimeError, match='scale'):
            attention_forward(q, k, v, scale=scale)


def test_bounds_past_32_bits():
    """Bounds of any size bound the lengths; they do not wrap to others on their way to the library."""
    from blast3r_b200.attention import attention_forward
    q, k, v, _ = (t[0] for t in _dense(1, 50, 50, 2, 2, 64, 'bf16'))
    cu = dict(cu_q=_i32([0, 13, 50]), cu_k=_i32([0, 13, 50]))
    want = attention_forward(q, k, v, **cu, max_q=37, max_k=37)
    for most in (dict(max_q=2 ** 32 + 5, max_k=37), dict(max_q=37, max_k=2 ** 32 + 5), dict(max_q=2 ** 31, max_k=2 ** 40)):
        got = attention_forward(q, k, v, **cu, **most)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_what_is_no_tensor_is_refused():
    from blast3r_b200.attention import attention_backward, attention_forward
    q, k, v, do = _dense(1, 5, 7, 2, 2, 64, 'bf16')
    o, lse = attention_forward(q, k, v)
    cu = _i32([0, 5])
    for bad in (lambda: attention_forward(q, k, v, k_lens=[7]), lambda: attention_forward(q, k, v, q_lens=5),
                lambda: attention_forward(q[0], q[0], q[0], cu_q=[0, 5], cu_k=cu, max_q=5, max_k=5),
                lambda: attention_forward(q[0], q[0], q[0], cu_q=cu, cu_k=[0, 5], max_q=5, max_k=5),
                lambda: attention_backward(do, q, k, v, o, None), lambda: attention_backward(None, q, k, v, o, lse)):
        with pytest.raises(RuntimeError):
            bad()


def test_forward_mode_is_refused():
    """Nothing computes a tangent, so a dual tensor raises instead of losing its own."""
    import torch.autograd.forward_ad as fwd
    from blast3r_b200.attention import attention
    q, k, v, t = _dense(1, 5, 5, 2, 2, 64, 'bf16')
    with fwd.dual_level():
        for which in range(3):
            args = [fwd.make_dual(x, t) if i == which else x for i, x in enumerate((q, k, v))]
            with pytest.raises(RuntimeError):
                attention(*args)
            with torch.no_grad(), pytest.raises(RuntimeError):
                attention(*args)
        assert attention(q, k, v).shape == q.shape
    assert attention(q, k, v).shape == q.shape


def test_packed_without_sequences():
    """Offsets of no sequence at all: every row is of none."""
    from blast3r_b200.attention import attention_backward, attention_forward
    q, k, v, do = (t[0] for t in _dense(1, 40, 50, 2, 2, 64, 'f16'))
    kw = dict(cu_q=_i32([0]), cu_k=_i32([0]), max_q=40, max_k=50)
    _poison()
    o, lse = attention_forward(q, k, v, **kw)
    _poison()
    grads = attention_backward(do, q, k, v, o, lse, **kw)
    assert all(float(t.abs().max()) == 0 for t in (o, *grads)) and bool((lse == -math.inf).all())


# ---------------------------------------------------------------- a wait that runs out
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('G,Lq,Lk', [(2, 1, 900), (3, 1, 900), (2, 300, 700), (3, 300, 700)])
def test_a_lost_copy_is_reported(monkeypatch, D, G, Lq, Lk):
    """A tile that is never asked for: the wait for it runs out, the call ends, check_attention raises once, and the next
    call is right.  Both halves on one tile of rows or on their own, Q by TMA or written by them."""
    from blast3r_b200 import _lib as L
    from blast3r_b200 import attention as A
    q, k, v, do = _dense(40, Lq, Lk, 4 * G, 4, D, 'f16')
    o, lse = A.attention_forward(q, k, v)
    grads = A.attention_backward(do, q, k, v, o, lse)
    A.check_attention()
    call = L.call_on
    for f in (lambda: A.attention_forward(q, k, v), lambda: A.attention_backward(do, q, k, v, o, lse)):
        monkeypatch.setattr(L, 'call_on', lambda index, name, d: call(index, name + '_ex', d, 1))
        f()
        monkeypatch.undo()
        with pytest.raises(L.B3RError, match='ran out'):
            A.check_attention()
        A.check_attention()
    again = A.attention_forward(q, k, v)
    assert torch.equal(again[0], o) and torch.equal(again[1], lse)
    assert all(torch.equal(a, b) for a, b in zip(A.attention_backward(do, q, k, v, o, lse), grads))
