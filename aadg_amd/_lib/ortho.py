"""Orthogonalised matrix updates by Newton-Schulz products (csrc/orthogonalize.hip), the operator of the Muon optimiser (aadg_amd/muon.py)."""
import ctypes

import torch

from .binding import AadgError, _check, _stream, load

NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)          # quintic of the Muon optimiser: singular values in (0, 1] end in about 0.7 ... 1.2 after five steps


class _Matrix(ctypes.Structure):
    """mirror of aadg_matrix (include/aadg_hip.h)"""
    _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p), ("rows", ctypes.c_int32), ("cols", ctypes.c_int32)]


def orthogonalize(mats, steps=5, eps=1e-7, coefficients=NEWTON_SCHULZ):
    """The orthogonalised form of every matrix of a list: U / (|U|_F + eps), then `steps` times X <- a X + (b A + c A A) X with A = X X^T
    (X^T X for a tall matrix).  float32 [rows, cols] tensors on one GPU, any sizes; products at float32 accuracy.  Five steps are 18 ... 22
    launches for all near-square matrices and as many for all wide ones, plus one for every further 26 of either.  Returns a list of new contiguous float32 tensors (not differentiable)."""
    mats = list(mats)
    for t in mats:
        if not (torch.is_tensor(t) and t.is_cuda):
            raise AadgError("aadg_amd kernels need GPU tensors; there is no CPU path")
        if t.dim() != 2 or t.dtype != torch.float32 or t.device != mats[0].device:
            raise AadgError("orthogonalize: expected 2-D float32 tensors on one device, got %s %s on %s" % (tuple(t.shape), t.dtype, t.device))
    if int(steps) != steps or not 1 <= steps <= 64 or not eps >= 0.0 or len(coefficients) != 3:
        raise AadgError("orthogonalize: steps must be 1 ... 64, eps not negative, three coefficients")
    src = [t.detach().contiguous() for t in mats]
    out = [torch.empty_like(t) for t in src]
    work = [(s, o) for s, o in zip(src, out) if s.numel() > 0]
    if not work:
        return out
    lib = load()
    with torch.cuda.device(src[0].device):
        arr = (_Matrix * len(work))(*((s.data_ptr(), o.data_ptr(), s.shape[0], s.shape[1]) for s, o in work))
        nbytes = lib.aadg_orthogonalize_workspace_bytes(arr, len(work))
        if nbytes == 0:
            raise AadgError("orthogonalize: unsupported size (at most 65536 a side, 2^28 elements, 4096 matrices)")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=src[0].device)
        _check(lib.aadg_orthogonalize_f32(arr, len(work), int(steps), *(float(c) for c in coefficients), float(eps), ws.data_ptr(), nbytes,
                                          _stream()), "aadg_orthogonalize_f32")
    return out
