"""Rotary positions and norms where tensors overlap, gradients go other ways and arguments do not fit."""
import math

import pytest
import torch

from tests import block_reference as R
from tests.test_gpu_norm import _backward, _forward, _make, _sum_of
from tests.test_gpu_rotary import _setup

pytestmark = pytest.mark.gpu


class _Elsewhere(torch.Tensor):
    """A tensor that says it is on another GPU."""

    def get_device(self):
        return 1

    @property
    def device(self):
        return torch.device('cuda', 1)


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


def test_norm_backward_refuses_another_device():
    from blast3r_b200.norm import residual_norm_backward
    y, x, dr, dh, kw = _make(2, 6, 64, 'bf16', 'bf16', 'layer', True, True, 'sample')
    for a, b in ((dr.as_subclass(_Elsewhere), dh), (dr, dh.as_subclass(_Elsewhere))):
        with pytest.raises(RuntimeError, match='device'):
            residual_norm_backward(a, b, y, x, **kw)


def test_norm_refuses_what_is_no_tensor():
    from blast3r_b200.norm import residual_norm_forward
    y, x, _, _, kw = _make(2, 6, 64, 'bf16', 'bf16', 'layer', True, True, 'sample')
    for bad in (dict(gate=1.0), dict(pre=(1.0, None)), dict(post=(None, 0.5))):
        with pytest.raises(RuntimeError):
            residual_norm_forward(y, x, **{**kw, **bad})


@pytest.mark.parametrize('shape,gate', [((6, 1, 40), (1, 1, 40)), ((6, 2, 40), (1, 1, 40)), ((1, 5, 40), (1, 1, 40)),
                                        ((1, 1, 40), (1, 1, 40)), ((6, 1, 40), (6, 1, 40)), ((4, 1, 40), (1, 40))])
def test_gates_of_one_row(shape, gate):
    """A gate of one row for all fits a prompt and a single token alike."""
    from blast3r_b200.norm import residual_norm
    g = torch.Generator(device='cuda').manual_seed(0)
    y, x, gt, dr = (torch.randn(*s, device='cuda', generator=g).requires_grad_() for s in (shape, shape, gate, shape))
    r, _ = residual_norm(y, x, gate=gt)
    assert float((r - (x + gt * y)).abs().max()) <= 2.0 ** -21 * float((x.abs() + (gt * y).abs()).max())
    r.backward(dr)
    over = [i for i in range(3) if ((1,) * (3 - len(gate)) + gate)[i] == 1 and shape[i] > 1]
    want = dr.double() * y.double()
    want = (want.sum(over, keepdim=True) if over else want).reshape(gate)
    assert gt.grad.shape == gate and float((gt.grad - want).abs().max()) <= 2.0 ** -20 * shape[0] * shape[1] * 16


@pytest.mark.parametrize('dtype,stream', [('bf16', 'bf16'), ('f16', 'f16'), ('bf16', 'f32')])
@pytest.mark.parametrize('pre', [False, True])
def test_norm_under_autograd(dtype, stream, pre):
    """16-bit operands and calls without the second norm, through autograd."""
    from blast3r_b200.norm import residual_norm
    B, T, C = 3, 25, 96
    y, x, dr, dh, kw = _make(B, T, C, dtype, stream, 'layer', True, pre, 'sample')
    ts = [t for t in (y, x, kw['gate'], *kw['post'], *(kw['pre'] or ())) if t is not None]
    for t in ts:
        t.requires_grad_()
    r, h = residual_norm(y, x, **kw)
    assert (h is None) == (not pre)
    torch.autograd.backward((r, h) if pre else (r,), (dr, dh) if pre else (dr,))
    kw = {n: tuple(t.detach() for t in p) if isinstance(p, tuple) else p.detach() if isinstance(p, torch.Tensor) else p for n, p in kw.items()}
    want = _backward(dr, dh, y.detach(), r.detach(), kw, _sum_of('sample', B))
    names = ['dy', 'dx', 'dgate', 'dw_post', 'db_post'] + (['dw_pre', 'db_pre'] if pre else [])
    for name, t in zip(names, ts):
        R.close(t.grad, *want[name], name)


def test_capture():
    """Rotations and norms, both directions, in a graph."""
    from blast3r_b200.norm import residual_norm_backward, residual_norm_forward
    from blast3r_b200.rotary import rotary
    y, x, dr, dh, kw = _make(3, 50, 264, 'bf16', 'f32', 'layer', True, True, 'sample')
    q, k, table, pos = _setup(2, 40, 4, 2, 64, 16, 2, 50, 'bf16')

    def run():
        r, h = residual_norm_forward(y, x, **kw)
        return (*rotary((q, k), table, pos), r, h, *residual_norm_backward(dr, dh, y, r, **kw))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for t in (y, q, k, dh):
        t.mul_(0.75)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_widths_of_one_kernel_from_several_threads():
    """Calls of one kernel that need different amounts of shared memory, from six threads at once: none takes away what
    another's launch counts on."""
    import ctypes as C
    import threading
    from blast3r_b200 import _lib as L
    from blast3r_b200.norm import _describe
    lib, errors, made = L.lib(), [], []
    for width in (8191, 7999, 4096, 2048):
        y, x, dr, dh, _ = _make(1, 2, width, 'bf16', 'f32', 'rms', True, True, None)
        d, keep = _describe(y, x, 'rms', 1e-5, True, None, 1.0, True)
        outs = [torch.empty_like(t) for t in (x, y)]
        work = torch.empty(int(lib.b3r_residual_norm_work_bytes(C.byref(d))) + 256, dtype=torch.uint8, device='cuda')
        made.append((d, y, x, dr, dh, outs, work, keep))
    torch.cuda.synchronize()

    def forward(d, y, x, dr, dh, outs, work, keep, stream):
        return lib.b3r_residual_norm_fwd(C.byref(d), y.data_ptr(), d.C, x.data_ptr(), d.C, outs[0].data_ptr(), outs[1].data_ptr(), stream)

    def backward(d, y, x, dr, dh, outs, work, keep, stream):
        return lib.b3r_residual_norm_bwd(C.byref(d), dr.data_ptr(), d.C, dh.data_ptr(), d.C, y.data_ptr(), d.C, x.data_ptr(), d.C,
                                         outs[0].data_ptr(), outs[1].data_ptr(), None, None, None, None, None,
                                         work.data_ptr() + (-work.data_ptr()) % 256, stream)

    def work(f, args):
        stream = torch.cuda.Stream()
        for i in range(20000):
            if f(*args, stream.cuda_stream):
                errors.append(lib.b3r_last_error().decode())
            if i % 500 == 499:
                stream.synchronize()
    for f, (a, b) in ((forward, made[:2]), (backward, made[2:])):
        ts = [threading.Thread(target=work, args=(f, m)) for m in (a, b) * 3]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
    assert not errors, (len(errors), errors[0])


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


def _apart(D=16):
    """Pairs that share memory and no element, as projections are cut: (q, k)."""
    n = lambda *s: torch.randn(*s, device='cuda')                             # noqa: E731
    fused = n(2, 7, 3, 4, D)                                                  # token, part, head
    heads = n(2, 3, 4, 7, D).transpose(2, 3)                                  # part, head, token
    mixed = n(2, 7, 4, 2, D)                                                  # head, part
    uneven = n(2, 7, 6, D)                                                    # four query and two key heads
    thin = n(2, 1, 5, D)[:, :, :4].expand(2, 1, 4, D)
    yield fused[:, :, 0], fused[:, :, 1]
    yield heads[:, 0], heads[:, 1]
    yield mixed[:, :, :, 0], mixed[:, :, :, 1]
    yield uneven[:, :, :4], uneven[:, :, 4:]
    yield uneven[:, :, 4:], uneven[:, :, :4]
    yield thin[..., :], n(2, 1, 2, D)
    batch = n(4, 7, 2, D)
    yield batch[:2], batch[2:]                                                # halves of a batch
    yield batch[0::2], batch[1::2]
    time = n(2, 14, 2, D)
    yield time[:, :7], time[:, 7:]
    yield time[:, 0::2], time[:, 1::2]
    one = n(1, 1, 6, D)
    yield one[:, :, :3].as_strided((1, 1, 3, D), (1, 1, D, 1)), one[:, :, 3:]  # strides of dimensions of one do not matter


def test_rotary_in_place_on_parts_of_one_tensor():
    from blast3r_b200.rotary import rotary, rotary_table
    table = rotary_table(20, 16)
    for q, k in _apart():
        pos = torch.arange(q.shape[1], device='cuda', dtype=torch.int32)[:, None]
        want = rotary((q, k), table, pos)
        got = rotary((q, k), table, pos, inplace=True)
        assert got[0] is q and got[1] is k
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_rotary_in_place_refuses_overlaps():
    """An element that lies in two places would be turned twice, by threads that race for it."""
    from blast3r_b200.rotary import rotary, rotary_table
    table, pos = rotary_table(20, 16), torch.arange(6, device='cuda', dtype=torch.int32)[:, None]
    x = torch.randn(2, 6, 4, 16, device='cuda')
    flat = torch.randn(2000, device='cuda')
    one = x[:, :, :1]
    keep = x.clone(), flat.clone()
    for bad in (one.expand(2, 6, 4, 16), x[:1].expand(2, 6, 4, 16), x[:, :1].expand(2, 6, 4, 16),
                flat.as_strided((2, 6, 4, 16), (384, 64, 8, 1)), flat.as_strided((2, 6, 4, 16), (64, 16, 96, 1)),
                (x, x), (x, x[:, :, 1:3]), (x[:, :, :3], x[:, :, 2:]), (x[:, :, 0:3:2], x[:, :, 2:]),
                (flat.as_strided((2, 6, 1, 16), (192, 32, 32, 1)), flat.as_strided((2, 6, 1, 16), (192, 32, 32, 1), 8)),
                (one, one.expand(2, 6, 2, 16))):
        with pytest.raises(RuntimeError, match='overlap'):
            rotary(bad, table, pos, inplace=True)
    assert torch.equal(x, keep[0]) and torch.equal(flat, keep[1])
