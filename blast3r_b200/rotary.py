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


def _strides(t):
    """Strides of a (B, T, heads, D) tensor whose D is contiguous."""
    return t.stride(0), t.stride(1), t.stride(2)


def _rotate(xs, table, positions, interleaved, inverse, inplace):
    if not 1 <= len(xs) <= 2:
        raise ValueError(f'one tensor or two (queries and keys), got {len(xs)}')
    x0 = xs[0]
    if not all(isinstance(x, torch.Tensor) and x.is_cuda for x in (*xs, table, positions)):
        raise RuntimeError('rotary runs on the GPU: pass CUDA tensors')
    dev = x0.device
    if any(t.device != dev for t in (*xs, table, positions)):
        raise RuntimeError('rotary: all tensors must be on one device')
    if x0.dtype not in DTYPES or any(x.dtype != x0.dtype for x in xs):
        raise RuntimeError(f'rotary takes float32, bfloat16 or float16 tensors of one type, got {[x.dtype for x in xs]}')
    if any(x.dim() != 4 or x.shape[:2] != x0.shape[:2] or x.shape[3] != x0.shape[3] for x in xs):
        raise RuntimeError(f'rotary takes (B, T, heads, D) tensors of one B, T and D, got {[tuple(x.shape) for x in xs]}')
    B, T, _, D = x0.shape
    if table.dtype != torch.float32 or table.dim() != 3 or table.shape[2] != 2 or not table.is_contiguous():
        raise RuntimeError('rotary: the table is a contiguous float32 (positions, pairs, 2) tensor (rotary_table)')
    if positions.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f'rotary: positions are int32 or int64, got {positions.dtype}')
    if positions.dim() == 2:                 # (T, axes), shared over the batch
        positions = positions.unsqueeze(0)
    if positions.dim() != 3 or positions.shape[0] not in (1, B) or positions.shape[1] != T:
        raise RuntimeError(f'rotary: positions are (T, axes) or (B, T, axes), got {tuple(positions.shape)} for B={B}, T={T}')
    axes, half = positions.shape[2], table.shape[1]
    if axes < 1 or half < 1 or axes * 2 * half > D:
        raise RuntimeError(f'rotary: {axes} sections of {2 * half} elements exceed the head size {D}')
    if positions.stride(2) != 1:
        positions = positions.contiguous()
    parts = (L.RotaryPart * len(xs))()
    outs = []
    for i, x in enumerate(xs):
        if x.stride(3) != 1:
            if inplace:
                raise RuntimeError('rotary in place needs tensors whose last dimension is contiguous')
            x = x.contiguous()
        out = x if inplace else torch.empty(x.shape, dtype=x.dtype, device=dev)
        parts[i] = L.RotaryPart(x.data_ptr(), out.data_ptr(), *_strides(x), *_strides(out), x.shape[2], 0)
        outs.append(out)
    with torch.cuda.device(dev):
        L.call('b3r_rotary', parts, len(xs), B, T, D, DTYPES[x0.dtype], table.data_ptr(), table.shape[0], half, axes,
               positions.data_ptr(), int(positions.dtype == torch.int64),
               0 if positions.shape[0] == 1 else positions.stride(0), positions.stride(1), int(bool(interleaved)),
               int(bool(inverse)), torch.cuda.current_stream(dev).cuda_stream)
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
    gradients).  A position outside of the table gives NaN.  Differentiable in xs."""
    pair = isinstance(xs, (tuple, list))
    ts = tuple(xs) if pair else (xs,)
    if torch.is_grad_enabled() and any(isinstance(x, torch.Tensor) and x.requires_grad for x in ts):
        if inplace:
            raise RuntimeError('rotary: tensors that need gradients cannot be turned in place')
        outs = _Rotary.apply(table, positions, interleaved, inverse, *ts)
    else:
        outs = _rotate(ts, table, positions, interleaved, inverse, inplace)
    return tuple(outs) if pair else outs[0]
