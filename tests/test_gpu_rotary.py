"""Rotary positions against their definition in float64, at the layouts, sizes and strides where they can go wrong."""
import pytest
import torch

from tests import block_reference as R

pytestmark = pytest.mark.gpu
DT = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}


def _setup(B, T, Hq, Hk, D, half, axes, n_pos, dtype, seed=0):
    from blast3r_b200.rotary import rotary_table
    g = torch.Generator(device='cuda').manual_seed(seed)
    q = torch.randn(B, T, Hq, D, device='cuda', generator=g).to(DT[dtype])
    k = torch.randn(B, T, Hk, D, device='cuda', generator=g).to(DT[dtype])
    pos = torch.randint(0, n_pos, (B, T, axes), device='cuda', generator=g)
    return q, k, rotary_table(n_pos, 2 * half), pos


@pytest.mark.parametrize('dtype', ['bf16', 'f16', 'f32'])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('B,T,Hq,Hk,D,half,axes', [
    (1, 1, 16, 4, 64, 32, 1),        # one token, the whole head
    (2, 37, 5, 1, 128, 32, 1),       # half of the head; head counts that fill no group of four
    (3, 24, 16, 16, 64, 16, 2),      # patch grid
    (1, 130, 4, 2, 96, 16, 3),       # three axes
    (2, 19, 3, 3, 52, 13, 2),        # odd number of pairs: no vectors in the half layout
    (2, 19, 3, 2, 40, 6, 1),         # vectors that end inside a section
    (1, 3, 1, 1, 24, 1, 5),          # one pair to a section, more axes
    (1, 600, 2, 2, 6, 3, 1),
    (3, 700, 12, 4, 120, 17, 3),     # sections that no vector divides: whole tokens, several to a block
    (1, 5, 64, 2, 96, 5, 2),
    (700, 1, 2, 1, 64, 19, 1),       # a block's tokens lie in several batches
])
def test_turn_and_back(dtype, interleaved, B, T, Hq, Hk, D, half, axes):
    from blast3r_b200.rotary import rotary
    q, k, table, pos = _setup(B, T, Hq, Hk, D, half, axes, 50, dtype)
    for inverse in (False, True):
        got = rotary((q, k), table, pos, interleaved=interleaved, inverse=inverse)
        for name, x, y in (('q', q, got[0]), ('k', k, got[1])):
            want, bound = R.rotary(x, table, pos, interleaved, inverse)
            R.close(y, want, bound, f'{name} inverse={inverse}')
            assert torch.equal(y[..., axes * 2 * half:], x[..., axes * 2 * half:])
    # in place, int32 positions, one tensor
    mine = q.clone()
    assert rotary(mine, table, pos.int(), interleaved=interleaved, inplace=True) is mine
    assert torch.equal(mine, rotary(q, table, pos, interleaved=interleaved))


def test_strides_and_shared_positions():
    from blast3r_b200.rotary import rotary
    B, T, H, D = 2, 33, 4, 64
    g = torch.Generator(device='cuda').manual_seed(1)
    qkv = torch.randn(B, T, 3, H, D, device='cuda', generator=g).bfloat16()
    _, _, table, pos = _setup(B, T, 1, 1, D, 16, 2, 40, 'bf16')
    pos = pos[:1].int()
    q, k = qkv[:, :, 0], qkv[:, :, 1]
    want = [R.rotary(x, table, pos.expand(B, T, 2), False, False) for x in (q, k)]
    for y, (w, b) in zip(rotary((q, k), table, pos[0]), want):
        R.close(y, w, b, 'fused projection')
    for y, (w, b) in zip(rotary((q.transpose(1, 2).contiguous().transpose(1, 2), k[..., :]), table, pos), want):
        R.close(y, w, b, 'heads before tokens')
    v = qkv[:, :, 2].clone()
    rotary((q, k), table, pos, inplace=True)
    for y, (w, b) in zip((q, k), want):
        R.close(y, w, b, 'in place in the fused projection')
    assert torch.equal(qkv[:, :, 2], v)
    # a base that is not aligned to a vector
    flat = torch.randn(B * T * H * D + 3, device='cuda', generator=g).bfloat16()
    x = flat[3:].view(B, T, H, D)
    R.close(rotary(x, table, pos), *R.rotary(x, table, pos.expand(B, T, 2), False, False), 'odd base')


def test_positions_outside_of_the_table_are_nan_in_their_section():
    from blast3r_b200.rotary import rotary
    q, _, table, pos = _setup(1, 6, 2, 2, 40, 8, 2, 10, 'f32')
    pos[0, 2, 1], pos[0, 4, 0] = 10, -1
    y = rotary(q, table, pos)
    bad = torch.zeros(1, 6, 2, 40, dtype=torch.bool, device='cuda')
    bad[0, 2, :, 16:32] = True
    bad[0, 4, :, 0:16] = True
    assert torch.equal(y.isnan(), bad)


def test_gradient():
    from blast3r_b200.rotary import rotary
    q, k, table, pos = _setup(2, 9, 3, 1, 32, 6, 2, 30, 'f32')
    q.requires_grad_(), k.requires_grad_()
    y = rotary((q, k), table, pos, interleaved=True)
    gs = [torch.randn_like(t) for t in y]
    torch.autograd.backward(y, gs)
    for x, g in ((q, gs[0]), (k, gs[1])):
        R.close(x.grad, *R.rotary(g, table, pos, True, True), 'formula')
        # differences of the definition, which is linear: exact up to float64
        d = torch.randn_like(x)
        lin = (R.rotary(d, table, pos, True, False)[0] * g.double()).sum()
        slack = (R.rotary(g, table, pos, True, True)[1] * d.double().abs()).sum()
        assert abs(float(lin - (x.grad.double() * d.double()).sum())) <= float(slack)


def test_scalings():
    from blast3r_b200.rotary import rotary_frequencies, rotary_table
    f0, a0 = rotary_frequencies(64)
    assert a0 == 1 and f0[0] == 1
    f, a = rotary_frequencies(64, scaling='linear', factor=4.0)
    assert torch.equal(f, f0 / 4) and a == 1
    f, _ = rotary_frequencies(64, scaling='ntk', factor=4.0)
    assert f[0] == 1 and abs(float(f[-1] / (f0[-1] / 4)) - 1) < 1e-12
    f, a = rotary_frequencies(64, scaling='yarn', factor=4.0, original=1024)
    assert f[0] == f0[0] and f[-1] == f0[-1] / 4 and bool((f <= f0).all()) and bool((f >= f0 / 4).all()) and a > 1
    t = rotary_table(5, 64, scaling='yarn', factor=4.0, original=1024).double().cpu()
    want = torch.arange(5.).double()[:, None] * f
    assert float((t[..., 0] - a * want.cos()).abs().max()) < 2.0 ** -23
    assert float((t[..., 1] - a * want.sin()).abs().max()) < 2.0 ** -23


def test_another_stream_and_empty():
    from blast3r_b200.rotary import rotary
    q, k, table, pos = _setup(2, 300, 8, 2, 64, 16, 2, 50, 'bf16')
    want = rotary((q, k), table, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rotary((q, k), table, pos)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert rotary(q[:, :0], table, pos[:, :0]).shape == (2, 0, 8, 64)


def test_refusals():
    from blast3r_b200 import _lib as L
    from blast3r_b200.rotary import rotary
    q, k, table, pos = _setup(2, 5, 4, 2, 32, 8, 2, 50, 'bf16')
    for bad in (lambda: rotary(q.double(), table, pos), lambda: rotary((q, k.half()), table, pos),
                lambda: rotary(q[0], table, pos), lambda: rotary(q, table.double(), pos),
                lambda: rotary(q, table, pos.float()), lambda: rotary(q, table, pos[:, :4]),
                lambda: rotary(q, table, pos.repeat(1, 1, 2)), lambda: rotary(q.cpu(), table, pos),
                lambda: rotary(q.transpose(2, 3).contiguous().transpose(2, 3), table, pos, inplace=True),
                lambda: rotary(q.clone().requires_grad_(), table, pos, inplace=True)):
        with pytest.raises(RuntimeError):
            bad()
    flat = torch.zeros(2 * 5 * 4 * 33, device='cuda', dtype=torch.bfloat16)
    with pytest.raises(L.B3RError, match='aligned to a pair'):
        rotary(flat.view(2, 5, 4, 33), table, pos, interleaved=True)
