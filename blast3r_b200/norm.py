"""The norms before and after a block with its gate and residual scale, on ``b3r_residual_norm_*``.

One call does what follows a block's output y in a residual network: the norm after the block, the
gate (or per-channel scale), the addition to the residual stream x, and the norm that the
next block begins with:

    n = N(y; post),   r = residual_scale * x + gate * n,   h = N(r; pre)

``residual_norm`` is differentiable; ``residual_norm_forward`` / ``residual_norm_backward`` are
the two passes on their own.
"""
import ctypes as C
from collections import namedtuple

import torch

from . import _lib as L
from .rotary import DTYPES

KINDS = {'layer': L.NORM_LAYER, 'rms': L.NORM_RMS}

NormGrads = namedtuple('NormGrads', 'dx, dy, dgate, dw_post, db_post, dw_pre, db_pre')


def check_norm(device=None):
    """Raises if a wait inside a ``residual_norm_backward`` of this process ran out on ``device`` (the
    current one by default), in a call or a graph's replay.  It waits for the work queued so far."""
    L.check_status('residual_norm', device)


def _rows(t):
    """t as (tensor, row stride) of rows of its last dimension, copied only where its strides
    have no single row stride."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.stride(-1) == 1 or t.shape[-1] == 1:
        lead = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
        if not lead:
            return t, t.shape[-1]
        if all(a[1] == b[0] * b[1] for a, b in zip(lead, lead[1:])) and lead[-1][1] >= t.shape[-1]:
            return t, lead[-1][1]
    return t.contiguous(), t.shape[-1]


def _pair(p, name):
    if p is None:
        return False, None, None
    if p is True:
        return True, None, None
    if isinstance(p, torch.Tensor):
        return True, p, None
    if not isinstance(p, (tuple, list)) or len(p) != 2:
        raise RuntimeError(f'residual_norm: {name} is None, True, a weight, or (weight or None, bias or None)')
    return True, p[0], p[1]


def _gate_rows(gate, shape):
    """Rows of y, of `shape`, to a row of the gate; None where the two do not fit."""
    if gate.shape[-1:] != shape[-1:]:
        return None
    g, lead = gate.shape[:-1], shape[:-1]
    rows = 1
    for n in lead:
        rows *= n
    k = len(g)
    if k > len(lead):
        return None
    while k > 0 and g[k - 1] == 1:
        k -= 1                                       # (B, 1, C): one row for each of the first dimensions
    if tuple(g[:k]) != tuple(lead[:k]):
        return None
    groups = 1
    for n in g[:k]:
        groups *= n
    return max(rows // groups, 1) if groups else 1


def _describe(y, x, kind, eps, post, gate, residual_scale, pre):
    """(descriptor, its tensors in order: w_post, b_post, gate, w_pre, b_pre) after the checks of every argument."""
    if not (isinstance(y, torch.Tensor) and isinstance(x, torch.Tensor) and y.is_cuda and x.is_cuda):
        raise RuntimeError('residual_norm runs on the GPU: pass CUDA tensors')
    shape, dt, sd, dev = y.shape, y.dtype, x.dtype, y.get_device()
    if y.dim() < 1 or shape != x.shape:
        raise RuntimeError(f'residual_norm: the block output {tuple(shape)} and the stream {tuple(x.shape)} differ in shape')
    if dt not in DTYPES or (sd != dt and sd != torch.float32):
        raise RuntimeError(f'residual_norm: float32, bfloat16 or float16 block outputs and a stream of that type or '
                           f'float32, got {dt} and {sd}')
    if kind not in KINDS:
        raise RuntimeError(f"residual_norm: kind is 'layer' or 'rms', got {kind!r}")
    Cn = shape[-1]
    has_post, w_post, b_post = _pair(post, 'post')
    has_pre, w_pre, b_pre = _pair(pre, 'pre')
    rows, per = (y.numel() // Cn if Cn else 0), 1
    if isinstance(gate, torch.Tensor):
        per = _gate_rows(gate, shape)
        if per is None:
            raise RuntimeError(f'residual_norm: the gate {tuple(gate.shape)} is (C,), (B, C), (B, 1, C) or the shape of '
                               f'the block output {tuple(shape)}')
    wt, keep, ptrs = None, [], []
    for t in (w_post, b_post, gate, w_pre, b_pre):
        if t is not None:
            if not isinstance(t, torch.Tensor):
                raise RuntimeError(f'residual_norm: weights, biases and the gate are tensors, got {t!r}')
            if t is not gate and (t.dim() != 1 or t.shape[0] != Cn):
                raise RuntimeError(f'residual_norm: weights and biases have {Cn} elements')
            if t.get_device() != dev:
                raise RuntimeError('residual_norm: all tensors must be on one CUDA device')
            if wt is None:
                wt = t.dtype
            if t.dtype != wt or (wt != dt and wt != torch.float32):
                raise RuntimeError(f'residual_norm: weights, biases and gate share one type, {dt} or float32')
            if not t.is_contiguous():
                t = t.contiguous()
            ptrs.append(t.data_ptr())
        else:
            ptrs.append(None)
        keep.append(t)
    if x.get_device() != dev:
        raise RuntimeError('residual_norm: all tensors must be on one CUDA device')
    d = L.ResidualNorm(rows, per, Cn, KINDS[kind], DTYPES[dt], DTYPES[sd], DTYPES[wt or dt], has_post, has_pre, eps,
                       residual_scale, *ptrs)
    return d, keep


def residual_norm_forward(y, x, *, kind='layer', eps=1e-6, post=None, gate=None, residual_scale=1.0, pre=None):
    """(r, h) for block output y and residual stream x, (..., C) each; h is None without ``pre``.

    post, pre: None (no such norm), True (no weights), a weight, or (weight or None, bias or
    None).  gate: None, or of shape (C,), (B, C), (B, 1, C) or y's
    (sizes of 1 at the end of its leading dimensions span y's).  x may be float32 beside
    bfloat16 or float16 blocks; r has x's type, h has y's.  1 to 8192 channels."""
    d, keep = _describe(y, x, kind, eps, post, gate, residual_scale, pre)
    (yt, ys), (xt, xs) = _rows(y), _rows(x)
    r = torch.empty_like(x, memory_format=torch.contiguous_format)
    h = torch.empty_like(y, memory_format=torch.contiguous_format) if d.pre else None
    L.call_on(y.get_device(), 'b3r_residual_norm_fwd', C.byref(d), yt.data_ptr(), ys, xt.data_ptr(), xs, r.data_ptr(),
              None if h is None else h.data_ptr())
    return r, h


def residual_norm_backward(dr, dh, y, r, *, kind='layer', eps=1e-6, post=None, gate=None, residual_scale=1.0, pre=None):
    """The gradients of ``residual_norm_forward`` with the same keywords, as a ``NormGrads`` (None
    for what is not there), from dr, the gradient that reaches r other than through h, dh
    (None without ``pre``), the block output y and the forward call's r."""
    d, keep = _describe(y, r, kind, eps, post, gate, residual_scale, pre)
    index = y.get_device()
    if not isinstance(dr, torch.Tensor) or dr.get_device() != index or dr.shape != r.shape or dr.dtype != r.dtype:
        raise RuntimeError('residual_norm backward: dr has the shape, type and device of r')
    if d.pre and (not isinstance(dh, torch.Tensor) or dh.get_device() != index or dh.shape != y.shape or dh.dtype != y.dtype):
        raise RuntimeError('residual_norm backward: dh has the shape, type and device of y')
    ts = [_rows(t) if t is not None else (None, 0) for t in (dr, dh if d.pre else None, y, r)]
    new = lambda t: None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)   # noqa: E731
    w_post, b_post, g, w_pre, b_pre = keep
    dx, dy = new(r), new(y)
    out = NormGrads(dx, dy, new(g), new(w_post), new(b_post), new(w_pre), new(b_pre))
    work = torch.empty(max(int(L.lib().b3r_residual_norm_work_bytes(C.byref(d))), 0) + 256, dtype=torch.uint8, device=y.device)
    wp = work.data_ptr()
    wp += (-wp) % 256
    if d.rows == 0 and out.dgate is not None:
        out.dgate.zero_()                # the library sees no rows and does not know the gate's
    ptr = lambda t: None if t is None else t.data_ptr()                                           # noqa: E731
    args = [a for t, s in ts for a in (ptr(t), s)]
    L.call_on(index, 'b3r_residual_norm_bwd_ex', C.byref(d), *args, *[ptr(t) for t in out], wp,
              L.status_word('residual_norm', index).data_ptr(), 0, 0)
    return out


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, w_post, b_post, gate, w_pre, b_pre, has_post, has_pre, kind, eps, residual_scale):
        kw = dict(kind=kind, eps=eps, residual_scale=residual_scale)
        r, h = residual_norm_forward(y, x, post=(w_post, b_post) if has_post else None, gate=gate,
                                     pre=(w_pre, b_pre) if has_pre else None, **kw)
        ctx.save_for_backward(y, r, w_post, b_post, gate, w_pre, b_pre)
        ctx.how = has_post, has_pre, kw
        ctx.set_materialize_grads(True)
        return r, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dr, dh):
        y, r, w_post, b_post, gate, w_pre, b_pre = ctx.saved_tensors
        has_post, has_pre, kw = ctx.how
        g = residual_norm_backward(dr, dh, y, r, post=(w_post, b_post) if has_post else None, gate=gate,
                                   pre=(w_pre, b_pre) if has_pre else None, **kw)
        return g.dy, g.dx, g.dw_post, g.db_post, g.dgate, g.dw_pre, g.db_pre, None, None, None, None, None


def residual_norm(y, x, *, kind='layer', eps=1e-6, post=None, gate=None, residual_scale=1.0, pre=None):
    """``residual_norm_forward``, differentiable in y, x, the gate, the weights and the biases."""
    has_post, w_post, b_post = _pair(post, 'post')
    has_pre, w_pre, b_pre = _pair(pre, 'pre')
    ts = (y, x, w_post, b_post, gate, w_pre, b_pre)
    L.refuse_tangents('residual_norm', ts)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in ts):
        return _ResidualNorm.apply(*ts, has_post, has_pre, kind, eps, residual_scale)
    return residual_norm_forward(y, x, kind=kind, eps=eps, post=post, gate=gate, residual_scale=residual_scale, pre=pre)
