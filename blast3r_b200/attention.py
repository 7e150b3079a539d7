"""Attention and its backward pass on the B200 kernels ``b3r_attention_fwd`` / ``_bwd``.

    S_ij = scale q_i . k_j,   lse_i = log sum_j exp S_ij,   o_i = sum_j exp(S_ij - lse_i) v_j

over the keys that a query sees.  The forward pass returns o and lse; the backward pass recomputes
the probabilities from lse instead of storing them.  Heads may be shared (grouped or single
key/value heads), sequences padded with lengths or packed one after the other, and a single
query may attend to a long cache.  ``attention`` is differentiable.
"""
import ctypes as C

import torch

from . import _lib as L

DTYPES = {torch.bfloat16: L.B3R_BF16, torch.float16: L.B3R_F16}


def check_attention(device=None):
    """Raises if a wait inside an attention kernel of this process ran out on ``device`` (the
    current one by default), in a call or a graph's replay.  It waits for the work queued so far."""
    L.check_status('attention', device)


def _tensor(t, packed):
    s = t.stride()
    return (t.data_ptr(), 0, s[0], s[1]) if packed else (t.data_ptr(), s[0], s[1], s[2])


def _lse_tensor(t, packed):
    s = t.stride()
    return (t.data_ptr(), 0, s[1], s[0]) if packed else (t.data_ptr(), s[0], s[2], s[1])


def _readable(t):
    """t itself where the kernels can read it: the head size contiguous, the other strides and the
    base multiples of 16 bytes; a copy otherwise."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        st = t.stride()
        if st[-1] == 1:
            for s, n in zip(st[:-1], t.shape):
                if n != 1 and (s <= 0 or s % 8):
                    break
            else:
                return t
    return t.clone(memory_format=torch.contiguous_format)


def _index(t, name, n, dev):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or t.get_device() != dev:
        raise RuntimeError(f'attention: {name} is an int32 tensor of {n} elements on the tensors\' device')
    return t.contiguous()


def _describe(q, k, v, causal, scale, q_lens, k_lens, cu_q, cu_k, max_q, max_k):
    if not (isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor) and
            q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError('attention runs on the GPU: pass CUDA tensors')
    dev = q.get_device()
    if k.get_device() != dev or v.get_device() != dev:
        raise RuntimeError('attention: all tensors must be on one device')
    if q.dtype not in DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError(f'attention takes bfloat16 or float16 tensors of one type, got {q.dtype}, {k.dtype}, {v.dtype}')
    packed = cu_q is not None or cu_k is not None
    nd = 3 if packed else 4
    what = '(rows, heads, D) with cu_q and cu_k' if packed else '(B, rows, heads, D)'
    if q.dim() != nd or k.dim() != nd or v.shape != k.shape or q.shape[-1] != k.shape[-1] or \
            (not packed and q.shape[0] != k.shape[0]):
        raise RuntimeError(f'attention takes {what}, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}')
    Hq, D = q.shape[-2:]
    Hkv = k.shape[-2]
    if D % 8 or not 8 <= D <= 128:
        raise RuntimeError(f'attention: the head size is a multiple of 8 up to 128, got {D}')
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise RuntimeError(f'attention: {Hq} query heads do not share {Hkv} key/value heads evenly')
    if scale is not None and not scale > 0:
        raise RuntimeError(f'attention: the scale must be positive, got {scale}')
    keep = []
    d = L.AttentionDesc(Hq=Hq, Hkv=Hkv, D=D, dtype=DTYPES[q.dtype], causal=int(bool(causal)),
                        scale=D ** -0.5 if scale is None else float(scale))
    if packed:
        if cu_q is None or cu_k is None or max_q is None or max_k is None:
            raise RuntimeError('attention: packed sequences need cu_q, cu_k, max_q and max_k')
        if q_lens is not None or k_lens is not None:
            raise RuntimeError('attention: packed sequences have no q_lens or k_lens')
        d.B = cu_q.shape[0] - 1 if isinstance(cu_q, torch.Tensor) and cu_q.dim() == 1 else -1
        if d.B < 0:
            raise RuntimeError('attention: cu_q has one element more than there are sequences')
        keep += [_index(cu_q, 'cu_q', d.B + 1, dev), _index(cu_k, 'cu_k', d.B + 1, dev)]
        d.cu_q, d.cu_k = keep[0].data_ptr(), keep[1].data_ptr()
        if max_q < 0 or max_k < 0:
            raise RuntimeError('attention: max_q and max_k must not be negative')
        d.Tq, d.Tk = q.shape[0], k.shape[0]
        d.Lq, d.Lk = min(int(max_q), d.Tq), min(int(max_k), d.Tk)      # (no sequence is longer than all rows)
    else:
        if max_q is not None or max_k is not None:
            raise RuntimeError('attention: max_q and max_k go with packed sequences')
        d.B, d.Lq, d.Lk = q.shape[0], q.shape[1], k.shape[1]
        d.Tq, d.Tk = d.Lq, d.Lk
        if q_lens is not None:
            keep.append(_index(q_lens, 'q_lens', d.B, dev))
            d.q_lens = keep[-1].data_ptr()
        if k_lens is not None:
            keep.append(_index(k_lens, 'k_lens', d.B, dev))
            d.k_lens = keep[-1].data_ptr()
    return d, packed, keep


def _launch(name, d, dev, index):
    d.status = L.status_word('attention', index).data_ptr()
    ref = C.byref(d)
    n = getattr(L.lib(), name + '_work_bytes')(ref)
    if n > 0:
        work = torch.empty(n + 256, dtype=torch.uint8, device=dev)
        p = work.data_ptr()
        d.work = p + (-p) % 256
    L.call_on(index, name, ref)


def attention_forward(q, k, v, *, causal=False, scale=None, q_lens=None, k_lens=None, cu_q=None, cu_k=None, max_q=None,
                      max_k=None):
    """(o, lse): o like q; lse float32 (B, Hq, Lq), or (Hq, Tq) for packed sequences.

    q (B, Lq, Hq, D), k and v (B, Lk, Hkv, D), Hq a multiple of Hkv, bfloat16 or float16, D a
    multiple of 8 up to 128; any strides (a copy is made where D is not contiguous or a row does
    not start on 16 bytes).  q_lens, k_lens: int32 (B,) lengths of padded sequences; what lies
    past them is not used.  Packed: q (Tq, Hq, D), k and v (Tk, Hkv, D), with cu_q, cu_k
    int32 (sequences + 1,), where each sequence begins and ends (they do not decrease), and max_q,
    max_k, bounds of their lengths: rows past them are not used.  Rows of no sequence have o = 0,
    lse = -inf and zero gradients.  causal: query i sees the keys j <= i + k_len - q_len, so the last query sees
    the last key.  A query that sees no key has o = 0 and lse = -inf.  scale: finite, 2**-100 at least,
    D**-0.5 by default.  Scores, their statistics and sums are float32; the probabilities are rounded to
    the inputs' type for their product with v, and o at the end."""
    d, packed, keep = _describe(q, k, v, causal, scale, q_lens, k_lens, cu_q, cu_k, max_q, max_k)
    q, k, v = _readable(q), _readable(k), _readable(v)
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((d.Hq, d.Tq) if packed else (d.B, d.Hq, d.Lq), dtype=torch.float32, device=q.device)
    d.q, d.k, d.v, d.o, d.lse = _tensor(q, packed), _tensor(k, packed), _tensor(v, packed), _tensor(o, packed), \
        _lse_tensor(lse, packed)
    _launch('b3r_attention_fwd', d, q.device, q.get_device())
    return o, lse


def attention_backward(do, q, k, v, o, lse, *, causal=False, scale=None, q_lens=None, k_lens=None, cu_q=None, cu_k=None,
                       max_q=None, max_k=None):
    """(dq, dk, dv) from do, the gradient of o, with the forward call's inputs, outputs and keywords.

    The probabilities are recomputed from lse in float32, and they and their gradient are rounded to the
    inputs' type for the matrix products (in float16 with powers of two that keep small ones out of
    its subnormal range); the rounded o gives delta."""
    d, packed, keep = _describe(q, k, v, causal, scale, q_lens, k_lens, cu_q, cu_k, max_q, max_k)
    for name, t in (('do', do), ('o', o)):
        if not isinstance(t, torch.Tensor) or t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise RuntimeError(f'attention backward: {name} has the shape, type and device of q')
    want = (d.Hq, d.Tq) if packed else (d.B, d.Hq, d.Lq)
    if not isinstance(lse, torch.Tensor) or tuple(lse.shape) != want or lse.dtype != torch.float32 or lse.device != q.device:
        raise RuntimeError(f'attention backward: lse is the forward call\'s, float32 {want}')
    do, q, k, v, o = (_readable(t) for t in (do, q, k, v, o))
    dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    for name, t in (('q', q), ('k', k), ('v', v), ('o', o), ('d_o', do), ('dq', dq), ('dk', dk), ('dv', dv)):
        setattr(d, name, _tensor(t, packed))
    d.lse = _lse_tensor(lse, packed)
    _launch('b3r_attention_bwd', d, q.device, q.get_device())
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_lens, k_lens, cu_q, cu_k, kw):
        o, lse = attention_forward(q, k, v, q_lens=q_lens, k_lens=k_lens, cu_q=cu_q, cu_k=cu_k, **kw)
        ctx.save_for_backward(q, k, v, o, lse, q_lens, k_lens, cu_q, cu_k)
        ctx.kw = kw
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, q_lens, k_lens, cu_q, cu_k = ctx.saved_tensors
        dq, dk, dv = attention_backward(do, q, k, v, o, lse, q_lens=q_lens, k_lens=k_lens, cu_q=cu_q, cu_k=cu_k, **ctx.kw)
        return dq, dk, dv, None, None, None, None, None


def attention(q, k, v, *, causal=False, scale=None, q_lens=None, k_lens=None, cu_q=None, cu_k=None, max_q=None, max_k=None):
    """o of ``attention_forward``, differentiable in q, k and v."""
    kw = dict(causal=causal, scale=scale, max_q=max_q, max_k=max_k)
    L.refuse_tangents('attention', (q, k, v))
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v)):
        return _Attention.apply(q, k, v, q_lens, k_lens, cu_q, cu_k, kw)
    return attention_forward(q, k, v, q_lens=q_lens, k_lens=k_lens, cu_q=cu_q, cu_k=cu_k, **kw)[0]
