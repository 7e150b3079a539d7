"""Rotary positions and norms where tensors overlap, gradients go other ways and arguments do not fit."""
import math

import pytest
import torch

from tests import block_reference as R
from tests.test_gpu_norm import _backward, _forward, _make, _sum_of
from tests.test_gpu_rotary import _setup

pytestmark = pytest.mark.gpu


def test_rotary_in_place_counts_as_a_change():
    """A tensor that an earlier operator keeps for its backward pass: torch reports the change."""
    from blast3r_b200.rotary import rotary
    q, k, table, pos = _setup(1, 6, 2, 2, 16, 8, 1, 10, 'f32')
    w = torch.ones(16, device='cuda', requires_grad=True)
    y = (k * w).sum()
    before = k._version
    rotary(k, table, pos, inplace=True)
    assert k._version > before
    with pytest.raises(RuntimeError, match='inplace'):
        y.backward()
    with torch.inference_mode():
        x = q.clone()
        rotary(x, table, pos, inplace=True)
    assert torch.equal(x, rotary(q, table, pos))


def test_rotary_refuses_forward_mode():
    import torch.autograd.forward_ad as fwd
    from blast3r_b200.rotary import rotary
    q, k, table, pos = _setup(1, 6, 2, 2, 16, 8, 1, 10, 'f32')
    with fwd.dual_level():
        d = fwd.make_dual(q, torch.ones_like(q))
        for bad in (lambda: rotary(d, table, pos), lambda: rotary((k, d), table, pos), lambda: rotary(d, table, pos, inplace=True)):
            with pytest.raises(RuntimeError):
                bad()
        assert rotary(q, table, pos).shape == q.shape


def test_norm_refuses_forward_mode():
    import torch.autograd.forward_ad as fwd
    from blast3r_b200.norm import residual_norm
    y, x, _, _, kw = _make(2, 6, 64, 'f32', 'f32', 'layer', True, True, 'channel')
    with fwd.dual_level():
        for bad in (dict(y=fwd.make_dual(y, x)), dict(x=fwd.make_dual(x, y)), dict(gate=fwd.make_dual(kw['gate'], kw['gate']))):
            with pytest.raises(RuntimeError):
                residual_norm(**{'y': y, 'x': x, **kw, **bad})
        assert residual_norm(y, x, **kw)[0].shape == y.shape


def test_norm_refuses_what_is_no_tensor():
    from blast3r_b200.norm import residual_norm_forward
    y, x, _, _, kw = _make(2, 6, 64, 'bf16', 'bf16', 'layer', True, True, 'sample')
    for bad in (dict(gate=1.0), dict(pre=(1.0, None)), dict(post=(None, 0.5))):
        with pytest.raises(RuntimeError):
            residual_norm_forward(y, x, **{**kw, **bad})


@pytest.mark.parametrize('C,stream,gate', [(64, 'bf16', None), (1024, 'f32', 'token'), (1000, 'bf16', 'sample'), (1001, 'bf16', 'token'),
                                           (4096, 'bf16', 'channel'), (5120, 'bf16', None)])
@pytest.mark.parametrize('kind,weights', [('rms', False), ('layer', True)])
def test_a_lost_copy_is_reported(monkeypatch, C, stream, gate, kind, weights):
    """A wait for a row whose copies are never asked for runs out: the call ends, check_norm raises once, and the next
    call is right."""
    from blast3r_b200 import _lib as L
    from blast3r_b200.norm import check_norm, residual_norm_backward
    y, x, dr, dh, kw = _make(4, 175, C, 'bf16', stream, kind, True, True, gate)
    if not weights:
        kw.update(post=True, pre=True)
    want = residual_norm_backward(dr, dh, y, x, **kw)
    check_norm()
    call = L.call_on
    monkeypatch.setattr(L, 'call_on', lambda index, name, *a: call(index, name, *a[:-2], 100, 1))
    residual_norm_backward(dr, dh, y, x, **kw)
    monkeypatch.undo()
    with pytest.raises(L.B3RError, match='ran out'):
        check_norm()
    check_norm()
    again = residual_norm_backward(dr, dh, y, x, **kw)
    assert all(t is None or torch.equal(t, w) for t, w in zip(again, want))
