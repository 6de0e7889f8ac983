"""Softmax attention of the transformer blocks (csrc/attention.hip): forward, and the backward that recomputes the probabilities."""
import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from .binding import AadgError, _check, _ptr, _stream, load

_ATTN_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_I64x3 = ctypes.c_int64 * 3


class _AttentionDesc(ctypes.Structure):
    """mirror of aadg_attention_desc (include/aadg_hip.h)"""
    _fields_ = ([(n, ctypes.c_int32) for n in ("dtype", "B", "H", "G", "Nq", "Nk", "d", "causal")] +
                [("scale", ctypes.c_float), ("reserved", ctypes.c_int32)] +
                [(n + "_stride", _I64x3) for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv")])


def _strides(t):
    """(batch, head, row) strides in elements; an axis of length 1 is never stepped over."""
    return _I64x3(*(st if n > 1 else 0 for n, st in zip(t.shape[:3], t.stride()[:3])))


def _rows16(t):
    """t itself if the kernels can read it in place (contiguous rows, every row on a 16-byte boundary), else a contiguous copy."""
    unit = 16 // t.element_size()
    if t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(st % unit == 0 or n <= 1 for n, st in zip(t.shape[:3], t.stride()[:3])):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _by_token(like):
    """[B, heads, n, d] tensor whose memory is [B, n, heads, d]: what the output projection reads and the input projections' gradients are."""
    B, h, n, d = like.shape
    return torch.empty((B, n, h, d), dtype=like.dtype, device=like.device).transpose(1, 2)


def _desc(q, k, scale, causal):
    de = _AttentionDesc()
    de.dtype = _ATTN_DTYPES[q.dtype]
    de.B, de.H, de.Nq, de.d = q.shape
    de.G, de.Nk = k.shape[1], k.shape[2]
    de.causal, de.scale = int(causal), scale
    return de


def _attention_forward(q, k, v, scale, causal, key_lengths, want_lse):
    lib = load()
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    o = _by_token(q)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if want_lse else None
    de = _desc(q, k, scale, causal)
    de.q_stride, de.k_stride, de.v_stride, de.o_stride = _strides(q), _strides(k), _strides(v), _strides(o)
    p = ctypes.byref(de)
    nbytes = lib.aadg_attention_forward_workspace_bytes(p)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _check(lib.aadg_attention_forward(p, q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(key_lengths), o.data_ptr(), _ptr(lse), _ptr(ws), nbytes,
                                      _stream()), "aadg_attention_forward")
    return q, k, v, o, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, key_lengths):
        ctx.scale, ctx.causal, ctx.shapes = scale, causal, (q.shape, k.shape)
        ctx.empty = q.numel() == 0 or k.numel() == 0
        if ctx.empty:
            return torch.zeros_like(q)
        with torch.cuda.device(q.device):
            q, k, v, o, lse = _attention_forward(q, k, v, scale, causal, key_lengths, True)
        ctx.save_for_backward(q, k, v, o, lse, key_lengths)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        need_q, need_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        if ctx.empty:
            sq, sk = ctx.shapes
            return (do.new_zeros(sq), do.new_zeros(sk), do.new_zeros(sk), None, None, None)
        q, k, v, o, lse, key_lengths = ctx.saved_tensors
        lib = load()
        with torch.cuda.device(q.device):
            do = _rows16(do)
            dq = _by_token(q) if need_q else None
            dk, dv = (_by_token(k), _by_token(v)) if need_kv else (None, None)
            de = _desc(q, k, ctx.scale, ctx.causal)
            for n, t in (("q", q), ("k", k), ("v", v), ("o", o), ("do", do), ("dq", dq), ("dk", dk), ("dv", dv)):
                if t is not None:
                    setattr(de, n + "_stride", _strides(t))
            p = ctypes.byref(de)
            nbytes = lib.aadg_attention_backward_workspace_bytes(p)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            _check(lib.aadg_attention_backward(p, q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(key_lengths), o.data_ptr(), lse.data_ptr(),
                                               do.data_ptr(), _ptr(dq), _ptr(dk), _ptr(dv), ws.data_ptr(), nbytes, _stream()),
                   "aadg_attention_backward")
        return dq, dk, dv, None, None, None


def attention_supported(q, k, v):
    """True where `attention` takes these tensors: GPU, float32 / bfloat16, [B, H, Nq, d] and [B, G, Nk, d] with H % G == 0, d % 8 == 0, d <= 128."""
    if not (q.is_cuda and q.dtype in _ATTN_DTYPES and q.dtype == k.dtype == v.dtype and q.device == k.device == v.device):
        return False
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        return False
    if k.shape[1] == 0 or q.shape[1] % k.shape[1] != 0 or q.shape[3] % 8 != 0 or not 0 < q.shape[3] <= 128:
        return False
    return q.numel() == 0 or k.numel() == 0 or bool(load().aadg_attention_supported(ctypes.byref(_desc(q, k, 1.0, False))))


def attention(q, k, v, scale=None, causal=False, key_lengths=None):
    """softmax(scale * q k^T) v on q [B, H, Nq, d] and k, v [B, G, Nk, d] (float32 or bfloat16, any strides; rows on 16-byte boundaries are
    read in place, others copied once).  H % G == 0: head h reads key head h // (H // G).  scale: default d ** -0.5.

    key_lengths: int32 [B] on the device, clamped to 0 ... Nk: keys and values behind a sequence's length are not used, whatever they hold.
    causal: query i of a sequence with L keys sees keys j <= i + L - Nq (the last query sees every key).  A query that sees no key
    gives zeros and takes no part in any gradient.  Inputs are expected finite (a key that only the causal rule hides included).

    Returns [B, H, Nq, d] over [B, Nq, H, d] memory: `.transpose(1, 2).reshape(B, Nq, H * d)` is free.  Differentiable once in q, k, v."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise AadgError("attention: expected q [B, H, Nq, d] and k, v [B, G, Nk, d]")
    for t in (q, k, v):
        if not t.is_cuda:
            raise AadgError("aadg_amd kernels need GPU tensors (got %s); there is no CPU path" % t.device)
    if not attention_supported(q, k, v):
        raise AadgError("attention: expected float32 / bfloat16 tensors of one type and device, q [B, H, Nq, d], k and v [B, G, Nk, d], H %% G == 0, "
                        "d %% 8 == 0, d <= 128; got %s %s %s" % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise AadgError("attention: scale must be positive and finite, got %r" % scale)
    if key_lengths is not None and (key_lengths.dtype != torch.int32 or key_lengths.shape != (q.shape[0],) or not key_lengths.is_contiguous() or
                                    key_lengths.device != q.device):
        raise AadgError("attention: key_lengths must be a contiguous int32 vector with one length per sequence (%d) on %s" % (q.shape[0], q.device))
    return _Attention.apply(q, k, v, scale, bool(causal), key_lengths)
