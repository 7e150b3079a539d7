"""The transformer-block operators where no GPU is needed: frequencies and tables, refusals, and the float64
definitions that the GPU tests compare with, against automatic differentiation."""
import ctypes as C
import math

import pytest
import torch

from blast3r_b200 import _lib as L
from blast3r_b200.attention import attention_forward
from blast3r_b200.norm import residual_norm_forward
from blast3r_b200.rotary import rotary, rotary_frequencies, rotary_table
from tests import block_reference as R


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 2, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match='GPU'):
        rotary(x, torch.zeros(4, 2, 2), torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match='GPU'):
        attention_forward(x, x, x)
    with pytest.raises(RuntimeError, match='GPU'):
        residual_norm_forward(x, x)


def test_frequencies_refuse_and_scale():
    with pytest.raises(ValueError):
        rotary_frequencies(7)
    with pytest.raises(ValueError):
        rotary_frequencies(8, scaling='other')
    with pytest.raises(ValueError, match='original'):
        rotary_frequencies(8, scaling='yarn', factor=2.0)
    f, amp = rotary_frequencies(8, base=16.0)
    assert amp == 1 and torch.allclose(f, torch.tensor([1, 0.5, 0.25, 0.125], dtype=torch.float64))
    t = rotary_table(3, 4, device='cpu', base=4.0)
    assert t.shape == (3, 2, 2) and abs(float(t[2, 1, 0]) - math.cos(1.0)) < 1e-7 and abs(float(t[1, 0, 1]) - math.sin(1.0)) < 1e-7


def _desc(**kw):
    d = L.AttentionDesc(B=1, Lq=4, Lk=4, Hq=2, Hkv=2, D=64, dtype=L.B3R_BF16, scale=0.1, Tq=4, Tk=4)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize('kw,what', [(dict(dtype=L.B3R_F32), 'dtype'), (dict(D=60), 'head size'), (dict(D=136), 'head size'),
                                     (dict(Hkv=3), 'evenly'), (dict(Lq=-1), 'negative'), (dict(scale=0.0), 'scale'),
                                     (dict(scale=-1.0), 'scale'), (dict(scale=math.nan), 'scale'), (dict(), 'NULL'),
                                     (dict(cu_q=16), 'cu_k'), (dict(B=1 << 30), 'too many')])
def test_c_abi_refuses_bad_attention_descriptors(kw, what):
    d = _desc(**kw)
    for f in ('b3r_attention_fwd', 'b3r_attention_bwd'):
        with pytest.raises(L.B3RError, match=what):
            L.call(f, C.byref(d), None)
    assert L.lib().b3r_attention_fwd_work_bytes(None) == -1


def test_c_abi_refuses_misaligned_attention_tensors():
    for name, t in (('q', (8, 0, 64, 64)), ('k', (16, 0, 60, 64)), ('v', (16, 0, 0, 64))):
        d = _desc()
        for n in ('q', 'k', 'v', 'o'):
            setattr(d, n, L.AttnTensor(16, 512, 128, 64))
        d.lse = L.AttnTensor(16, 8, 1, 4)
        setattr(d, name, L.AttnTensor(*t))
        with pytest.raises(L.B3RError, match='aligned' if name == 'q' else 'strides'):
            L.call('b3r_attention_fwd', C.byref(d), None)


def test_c_abi_refuses_bad_norms_and_rotations():
    d = L.ResidualNorm(rows=6, rows_per_gate=4, C=8, kind=0, dtype=L.B3R_BF16, stream_dtype=L.B3R_BF16,
                       weight_dtype=L.B3R_BF16, gate=16)
    for change, what in ((dict(), 'divide'), (dict(gate=None, stream_dtype=L.B3R_F16), 'stream'), (dict(gate=None, kind=7), 'kind'),
                         (dict(gate=None, C=0), 'channels'), (dict(gate=None, w_pre=16), 'switched off'), (dict(gate=None), 'NULL')):
        e = L.ResidualNorm.from_buffer_copy(d)
        for k, v in change.items():
            setattr(e, k, v)
        with pytest.raises(L.B3RError, match=what):
            L.call('b3r_residual_norm_fwd', C.byref(e), None, 8, None, 8, None, None, None)
    part = (L.RotaryPart * 1)(L.RotaryPart(None, None, 8, 8, 8, 8, 8, 8, 1, 0))
    for args, what in (((part, 1, 1, 1, 8, L.B3R_F64, 16, 4, 2, 1), 'dtype'), ((part, 1, 1, 1, 8, L.B3R_F32, 16, 4, 8, 1), 'exceeds'),
                       ((part, 3, 1, 1, 8, L.B3R_F32, 16, 4, 2, 1), 'parts'), ((part, 1, 1, 1, 8, L.B3R_F32, 16, 0, 2, 1), 'empty'),
                       ((part, 1, 1, 1, 8, L.B3R_F32, 16, 4, 2, 1), 'NULL tensor')):
        with pytest.raises(L.B3RError, match=what):
            L.call('b3r_rotary', *args, None, 0, 0, 0, 0, 0, None)


@pytest.mark.parametrize('causal,n,m', [(False, 5, 7), (True, 5, 7), (True, 6, 3)])
def test_the_definition_of_attention_is_differentiated_right(causal, n, m):
    g = torch.Generator().manual_seed(n)
    q, k, v, do = (torch.randn(s, generator=g, dtype=torch.float32) for s in ((1, n, 4, 8), (1, m, 2, 8), (1, m, 2, 8), (1, n, 4, 8)))
    qd, kd, vd = (t.double().requires_grad_() for t in (q, k, v))
    S = torch.einsum('bihd,bjhd->bhij', qd, kd.repeat_interleave(2, 2)) * 0.3
    if causal:
        S = S.masked_fill(torch.ones(n, m, dtype=torch.bool).triu(m - n + 1), -math.inf)
    P = torch.where(S.isinf().all(-1, keepdim=True), torch.zeros_like(S), S.softmax(-1).nan_to_num(0.0))
    o = torch.einsum('bhij,bjhd->bihd', P, vd.repeat_interleave(2, 2))
    want = torch.autograd.grad((torch.where(o.isnan(), torch.zeros_like(o), o) * do.double()).sum(), (qd, kd, vd))
    got = R.attention(q, k, v, do, o.detach().float(), causal, 0.3, [(0, n, m)], False)
    assert float((got['o'][0] - o.detach()).abs().max()) < 1e-12
    for name, w in zip(('dq', 'dk', 'dv'), want):
        assert float((got[name][0] - w.nan_to_num(0.0)).abs().max()) < 1e-12, name
