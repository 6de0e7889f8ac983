"""Softmax attention of the transformer blocks (csrc/attention.hip): forward, and the backward that recomputes the probabilities."""
import contextlib
import math
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .binding import AadgError, _check, _ptr, _stream, load

_ATTN_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_ATTN_DESC = struct.Struct("<8ifi24q")             # aadg_attention_desc (include/aadg_hip.h): 8 sizes, scale, a reserved word, 8 x (batch, head, row) strides
_NO_STRIDE = (0, 0, 0)


def _attn_desc(dtype, B, H, G, Nq, Nk, d, causal, scale, *strides):
    flat = [x for st in strides for x in st[:3]]
    try:
        return _ATTN_DESC.pack(dtype, B, H, G, Nq, Nk, d, causal, scale, 0, *flat, *(0,) * (24 - len(flat)))
    except (struct.error, OverflowError):                     # sizes past 32 bits, a scale past float32
        raise AadgError("attention: sizes (%d, %d, %d, %d, %d, %d) or scale %r out of range" % (B, H, G, Nq, Nk, d, scale)) from None


def _rows16(t):
    """t itself if the kernels can read it in place (contiguous rows, everything on 16-byte boundaries), else a contiguous copy."""
    a, b, c, e = t.stride()
    unit = 16 // t.element_size()
    if e == 1 and not (a | b | c) % unit and not t.data_ptr() % 16:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _by_token(like):
    """[B, heads, n, d] tensor whose memory is [B, n, heads, d]: what the output projection reads and the input projections' gradients are."""
    B, h, n, d = like.shape
    return like.new_empty_strided((B, h, n, d), (n * h * d, d, h * d, 1))


def _on(device):
    """the device the launches go to: nothing to do where it is the current one"""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _attention_forward(q, k, v, scale, causal, key_lengths, want_lse):
    lib = load()
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    o = _by_token(q)
    B, H, Nq, d = q.shape
    lse = torch.empty((B, H, Nq), dtype=torch.float32, device=q.device) if want_lse else None
    de = _attn_desc(_ATTN_DTYPES[q.dtype], B, H, k.shape[1], Nq, k.shape[2], d, causal, scale, q.stride(), k.stride(), v.stride(), o.stride())
    nbytes = lib.aadg_attention_forward_workspace_bytes(de)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _check(lib.aadg_attention_forward(de, q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(key_lengths), o.data_ptr(), _ptr(lse), _ptr(ws), nbytes,
                                      _stream()), "aadg_attention_forward")
    return q, k, v, o, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, key_lengths):
        ctx.scale, ctx.causal, ctx.shapes = scale, causal, (q.shape, k.shape)
        ctx.empty = q.numel() == 0 or k.numel() == 0
        if ctx.empty:
            return torch.zeros_like(q)
        with _on(q.device):
            q, k, v, o, lse = _attention_forward(q, k, v, scale, causal, key_lengths, True)
        ctx.save_for_backward(q, k, v, o, lse, key_lengths)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        if ctx.empty:
            sq, sk = ctx.shapes
            return (do.new_zeros(sq), do.new_zeros(sk), do.new_zeros(sk), None, None, None)
        q, k, v, o, lse, key_lengths = ctx.saved_tensors
        lib = load()
        with _on(q.device):
            do = _rows16(do)
            dq = _by_token(q) if need_q else None
            dk, dv = (_by_token(k), _by_token(v)) if need_k or need_v else (None, None)
            B, H, Nq, d = q.shape
            st = [_NO_STRIDE if t is None else t.stride() for t in (q, k, v, o, do, dq, dk, dv)]
            de = _attn_desc(_ATTN_DTYPES[q.dtype], B, H, k.shape[1], Nq, k.shape[2], d, ctx.causal, ctx.scale, *st)
            nbytes = lib.aadg_attention_backward_workspace_bytes(de)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            _check(lib.aadg_attention_backward(de, q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(key_lengths), o.data_ptr(), lse.data_ptr(),
                                               do.data_ptr(), _ptr(dq), _ptr(dk), _ptr(dv), ws.data_ptr(), nbytes, _stream()),
                   "aadg_attention_backward")
        return dq, dk if need_k else None, dv if need_v else None, None, None, None


def _fits(q, k, v):
    if not (q.is_cuda and q.dtype in _ATTN_DTYPES and q.dtype == k.dtype == v.dtype and q.device == k.device == v.device):
        return False
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        return False
    (B, H, Nq, d), (Bk, G, Nk, dk) = q.shape, k.shape
    return B == Bk and d == dk and G > 0 and H % G == 0 and d % 8 == 0 and 0 < d <= 128


def attention_supported(q, k, v):
    """True where `attention` takes these tensors: GPU, float32 / bfloat16, [B, H, Nq, d] and [B, G, Nk, d] with H % G == 0, d % 8 == 0, d <= 128."""
    if not _fits(q, k, v):
        return False
    (B, H, Nq, d), G, Nk = q.shape, k.shape[1], k.shape[2]
    if max(B, H, Nq, Nk) >= 1 << 31:
        return False
    return B * H * Nq * Nk == 0 or bool(load().aadg_attention_supported(_attn_desc(_ATTN_DTYPES[q.dtype], B, H, G, Nq, Nk, d, 0, 1.0)))


def attention(q, k, v, scale=None, causal=False, key_lengths=None):
    """softmax(scale * q k^T) v on q [B, H, Nq, d] and k, v [B, G, Nk, d] (float32 or bfloat16, any strides; rows on 16-byte boundaries are
    read in place, others copied once).  H % G == 0: head h reads key head h // (H // G).  scale: default d ** -0.5.

    key_lengths: int32 [B] on the device, clamped to 0 ... Nk: keys and values behind a sequence's length are not used, whatever they hold.
    causal: query i of a sequence with L keys sees keys j <= i + L - Nq (the last query sees every key).  A query that sees no key
    gives zeros and takes no part in any gradient, whatever it and its output's gradient hold.  Other inputs are expected finite (a key that
    only the causal rule hides included).

    Returns [B, H, Nq, d] over [B, Nq, H, d] memory: `.transpose(1, 2).reshape(B, Nq, H * d)` is free.  Differentiable once in q, k, v, in reverse mode (a
    forward-mode tangent raises NotImplementedError)."""
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise AadgError("aadg_amd kernels need GPU tensors (got %s, %s, %s); there is no CPU path" % (q.device, k.device, v.device))
    if not _fits(q, k, v):                                    # (sizes past the kernels' limits: the library refuses them)
        raise AadgError("attention: expected float32 / bfloat16 tensors of one type and device, q [B, H, Nq, d], k and v [B, G, Nk, d], H %% G == 0, "
                        "d %% 8 == 0, d <= 128; got %s %s %s" % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise AadgError("attention: scale must be positive and finite, got %r" % scale)
    if key_lengths is not None and (not torch.is_tensor(key_lengths) or key_lengths.dtype != torch.int32 or key_lengths.shape != (q.shape[0],) or
                                    not key_lengths.is_contiguous() or key_lengths.device != q.device):
        raise AadgError("attention: key_lengths must be a contiguous int32 vector with one length per sequence (%d) on %s" % (q.shape[0], q.device))
    # (inside a forward-mode level the call goes through autograd, which refuses tangents; the direct path would drop them)
    if (not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) and q.numel() > 0 and k.numel() > 0 and
            forward_ad._current_level < 0):
        with _on(q.device):
            return _attention_forward(q, k, v, scale, bool(causal), key_lengths, False)[3]
    return _Attention.apply(q, k, v, scale, bool(causal), key_lengths)
