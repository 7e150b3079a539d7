"""Rotary positions on the B200 kernel ``b3r_rotary``.

The reference's networks turn queries and keys by their patch's position with a native extension
of their own (extensions/curope, 2 and 3 position axes, half layout, float or half tensors in
place).  ``rotary`` does this for any number of axes, the half and the interleaved layout,
rotations of a part of the head, and frequencies scaled for longer contexts, for queries and keys
in one launch; its gradient is the same call with the angles reversed.
"""
import ctypes as C
import math

import torch

from . import _lib as L

_PARTS = {n: L.RotaryPart * n for n in (1, 2)}
DTYPES = {torch.float32: L.B3R_F32, torch.bfloat16: L.B3R_BF16, torch.float16: L.B3R_F16}


def rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0):
    """(frequencies, amplitude) of a section of ``dim`` elements (dim / 2 pairs): pair k turns by
    base^(-2k/dim) per position, as float64.  scaling for contexts ``factor`` times longer:
    None; 'linear' (every frequency divided by factor); 'ntk' (a base under which the slowest
    frequency is divided by factor and the fastest stays); 'yarn' (pairs that turn more than
    ``fast`` times within the ``original`` context stay, pairs that turn less than ``slow`` times
    are divided by factor, with a linear ramp over the pairs between, and the amplitude is
    1 + 0.1 ln factor)."""
    if dim < 2 or dim % 2:
        raise ValueError(f'the section of a head must have an even number of elements, got {dim}')
    if scaling not in (None, 'linear', 'ntk', 'yarn'):
        raise ValueError(f'unknown scaling {scaling!r}')
    half = dim // 2
    if scaling == 'ntk':
        base = base * factor ** (dim / max(dim - 2, 1))
    f = torch.tensor([base ** (-2.0 * k / dim) for k in range(half)], dtype=torch.float64)
    if scaling == 'linear':
        return f / factor, 1.0
    if scaling == 'yarn':
        if original is None or original <= 0:
            raise ValueError("scaling='yarn' needs the original context's length")
        lo, hi = (dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (fast, slow))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), dim - 1)
        ramp = ((torch.arange(half, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return f, 1.0


def rotary_table(n_positions, dim, device='cuda', **kw):
    """float32 (n_positions, dim / 2, 2): the cosines and sines of positions 0..n_positions-1 for
    sections of ``dim`` elements, computed in float64 (``rotary_frequencies``'s arguments)."""
    f, amp = rotary_frequencies(dim, **kw)
    ang = torch.arange(n_positions, dtype=torch.float64)[:, None] * f
    return (torch.stack([ang.cos(), ang.sin()], dim=-1) * amp).float().to(device).contiguous()


def _bad(xs, table, positions):
    """Why the arguments cannot be used."""
    if not all(isinstance(x, torch.Tensor) and x.is_cuda for x in (*xs, table, positions)):
        return 'rotary runs on the GPU: pass CUDA tensors'
    if any(t.device != xs[0].device for t in (*xs, table, positions)):
        return 'rotary: all tensors must be on one device'
    if xs[0].dtype not in DTYPES or any(x.dtype != xs[0].dtype for x in xs):
        return f'rotary takes float32, bfloat16 or float16 tensors of one type, got {[x.dtype for x in xs]}'
    if any(x.dim() != 4 for x in xs) or any(x.shape[:2] != xs[0].shape[:2] or x.shape[3] != xs[0].shape[3] for x in xs):
        return f'rotary takes (B, T, heads, D) tensors of one B, T and D, got {[tuple(x.shape) for x in xs]}'
    if table.dtype != torch.float32 or table.dim() != 3 or table.shape[2] != 2 or not table.is_contiguous():
        return 'rotary: the table is a contiguous float32 (positions, pairs, 2) tensor (rotary_table)'
    return f'rotary: positions are int32 or int64, got {positions.dtype}'


def _rotate(xs, table, positions, interleaved, inverse, inplace):
    n = len(xs)
    if not 1 <= n <= 2:
        raise ValueError(f'one tensor or two (queries and keys), got {n}')
    x0 = xs[0]
    ok = isinstance(x0, torch.Tensor) and isinstance(table, torch.Tensor) and isinstance(positions, torch.Tensor) and x0.is_cuda
    if ok:
        dev, dt, shape0, tshape, pt = x0.get_device(), x0.dtype, x0.shape, table.shape, positions.dtype
        code, wide = DTYPES.get(dt), pt == torch.int64
        ok = (code is not None and len(shape0) == 4 and table.dtype == torch.float32 and len(tshape) == 3 and
              tshape[2] == 2 and table.is_contiguous() and table.get_device() == dev and positions.get_device() == dev and
              (wide or pt == torch.int32))
    if ok and n == 2:
        x1 = xs[1]
        ok = isinstance(x1, torch.Tensor) and x1.dtype == dt and x1.get_device() == dev
        if ok:
            s1 = x1.shape
            ok = len(s1) == 4 and s1[0] == shape0[0] and s1[1] == shape0[1] and s1[3] == shape0[3]
    if not ok:
        raise RuntimeError(_bad(xs, table, positions))
    B, T, _, D = shape0
    if positions.dim() == 2:                 # (T, axes), shared over the batch
        positions = positions.unsqueeze(0)
    shape = positions.shape
    if len(shape) != 3 or shape[0] not in (1, B) or shape[1] != T:
        raise RuntimeError(f'rotary: positions are (T, axes) or (B, T, axes), got {tuple(shape)} for B={B}, T={T}')
    axes, n_pos, half = shape[2], tshape[0], tshape[1]
    if axes < 1 or half < 1 or axes * 2 * half > D:
        raise RuntimeError(f'rotary: {axes} sections of {2 * half} elements exceed the head size {D}')
    ps = positions.stride()
    if ps[2] != 1:
        positions = positions.contiguous()
        ps = positions.stride()
    parts, outs, keep = _PARTS[n](), [], []
    for i, x in enumerate(xs):
        st = x.stride()
        if st[3] != 1 and D > 1:
            if inplace:
                raise RuntimeError('rotary in place needs tensors whose last dimension is contiguous')
            x = x.contiguous()
            st = x.stride()
        if inplace:
            out, so = x, st
        else:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
            so = out.stride()
        parts[i] = (x.data_ptr(), out.data_ptr(), st[0], st[1], st[2], so[0], so[1], so[2], x.shape[2], 0)
        outs.append(out)
        keep.append(x)
    L.call_on(dev, 'b3r_rotary', parts, n, B, T, D, code, table.data_ptr(), n_pos, half, axes, positions.data_ptr(), wide,
              0 if shape[0] == 1 else ps[0], ps[1], bool(interleaved), bool(inverse))
    if inplace:                              # what autograd keeps of them has changed
        torch.autograd.graph.increment_version([x for x in xs if not x.is_inference()])
    return outs


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, positions, interleaved, inverse, *xs):
        ctx.save_for_backward(table, positions)
        ctx.how = interleaved, inverse
        return tuple(_rotate(xs, table, positions, interleaved, inverse, False))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        table, positions = ctx.saved_tensors
        interleaved, inverse = ctx.how
        return (None, None, None, None, *_rotate(grads, table, positions, interleaved, not inverse, False))


def rotary(xs, table, positions, *, interleaved=False, inverse=False, inplace=False):
    """Turns ``xs``, a (B, T, heads, D) tensor or a pair of them (queries and keys, whose head
    counts may differ), by their tokens' positions.  positions: integers (T, axes) or (B, T, axes);
    table: ``rotary_table``, whose pairs give the size of a section; axis a turns the a-th section
    of the head, and elements past the sections pass through.  interleaved: pairs side by side
    instead of half a section apart.  inverse turns back.  inplace overwrites xs (not with
    gradients, nor where elements of xs overlap in memory).  A position outside of the table gives
    NaN.  Differentiable in xs."""
    pair = isinstance(xs, (tuple, list))
    ts = tuple(xs) if pair else (xs,)
    L.refuse_tangents('rotary', ts)
    if torch.is_grad_enabled() and any(isinstance(x, torch.Tensor) and x.requires_grad for x in ts):
        if inplace:
            raise RuntimeError('rotary: tensors that need gradients cannot be turned in place')
        outs = _Rotary.apply(table, positions, interleaved, inverse, *ts)
    else:
        outs = _rotate(ts, table, positions, interleaved, inverse, inplace)
    return tuple(outs) if pair else outs[0]
