"""CPU: the attention entry points check their arguments on the host, before anything touches a GPU."""
import ctypes

import pytest
import torch


class _Desc(ctypes.Structure):
    """aadg_attention_desc as include/aadg_hip.h declares it"""
    _fields_ = ([(n, ctypes.c_int32) for n in ("dtype", "B", "H", "G", "Nq", "Nk", "d", "causal")] + [("scale", ctypes.c_float), ("reserved", ctypes.c_int32)] +
                [(n + "_stride", ctypes.c_int64 * 3) for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv")])


def _desc(_lib, **kw):
    d = _Desc()
    for k, v in dict(dtype=1, B=2, H=4, G=2, Nq=8, Nk=16, d=64, causal=0, scale=0.125).items():
        setattr(d, k, kw.pop(k, v))
    for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
        setattr(d, n + "_stride", (ctypes.c_int64 * 3)(*kw.pop(n, (4096, 512, 64))))
    assert not kw
    return d


def test_descriptor_layout():
    from aadg_amd import _lib
    strides = [(100 * i + 1, 100 * i + 2, 100 * i + 3, 1) for i in range(8)]
    packed = _lib._attn_desc(1, 2, 4, 2, 8, 16, 64, True, 0.125, *strides)
    d = _Desc.from_buffer_copy(packed)
    assert len(packed) == ctypes.sizeof(_Desc)
    assert (d.dtype, d.B, d.H, d.G, d.Nq, d.Nk, d.d, d.causal, d.scale) == (1, 2, 4, 2, 8, 16, 64, 1, 0.125)
    assert [list(getattr(d, n + "_stride")) for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv")] == [list(s[:3]) for s in strides]


def test_attention_entry_points_validate_arguments():
    from aadg_amd import _lib
    lib = _lib.load()
    z, one, odd = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_void_p(24)
    ref = ctypes.byref
    ok = _desc(_lib)
    assert lib.aadg_attention_supported(ref(ok)) == 1 and lib.aadg_attention_supported(z) == 0
    for kw, rc in ((dict(dtype=2), -1), (dict(B=0), -1), (dict(Nq=0), -1), (dict(Nk=0), -1), (dict(G=3), -1), (dict(scale=0.0), -1), (dict(scale=-1.0), -1),
                   (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(d=60), -3), (dict(d=136), -3), (dict(Nk=1 << 31 - 1), -3),
                   (dict(B=1 << 20), -3)):
        d = _desc(_lib, **kw)
        assert lib.aadg_attention_supported(ref(d)) == 0, kw
        assert lib.aadg_attention_forward(ref(d), one, one, one, z, one, z, z, 0, z) == rc, kw
        assert lib.aadg_attention_backward(ref(d), one, one, one, z, one, one, one, one, one, one, one, 1 << 40, z) == rc, kw
        assert lib.aadg_attention_forward_workspace_bytes(ref(d)) == 0 and lib.aadg_attention_backward_workspace_bytes(ref(d)) == 0
    # pointers and strides: NULL, not on a 16-byte boundary
    for args in ((z, one, one, one), (one, z, one, one), (one, one, z, one), (one, one, one, z), (odd, one, one, one)):
        q, k, v, o = args
        assert lib.aadg_attention_forward(ref(ok), q, k, v, z, o, z, z, 0, z) == -1
        assert lib.aadg_attention_backward(ref(ok), q, k, v, z, o, one, one, one, one, one, one, 1 << 40, z) == -1
    assert lib.aadg_attention_forward(ref(_desc(_lib, k=(4096, 512, 60))), one, one, one, z, one, z, z, 0, z) == -1
    assert lib.aadg_attention_backward(ref(ok), one, one, one, z, one, z, one, one, one, one, one, 1 << 40, z) == -1          # no lse
    assert lib.aadg_attention_backward(ref(ok), one, one, one, z, one, one, one, one, one, z, one, 1 << 40, z) == -1          # dk without dv
    assert lib.aadg_attention_backward(ref(_desc(_lib, dv=(4096, 512, 4))), one, one, one, z, one, one, one, one, one, one, one, 1 << 40, z) == -1
    # workspaces
    assert lib.aadg_attention_backward(ref(ok), one, one, one, z, one, one, one, one, one, one, one, 16, z) == -2
    long = _desc(_lib, B=1, Nq=1, Nk=4096)
    need = lib.aadg_attention_forward_workspace_bytes(ref(long))
    assert need > 0
    assert lib.aadg_attention_forward(ref(long), one, one, one, z, one, z, one, need - 1, z) == -2
    assert lib.aadg_attention_forward(ref(long), one, one, one, z, one, z, z, need, z) == -2
    assert lib.aadg_attention_backward(ref(ok), one, one, one, z, one, one, one, z, z, z, z, 0, z) == 0                        # nothing asked for


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_attention_has_no_cpu_path():
    from aadg_amd import _lib
    q = torch.zeros(1, 1, 4, 64)
    assert not _lib.attention_supported(q, q, q)
    with pytest.raises(_lib.AadgError):
        _lib.attention(q, q, q)


@pytest.mark.parametrize("B,G,r,Nq,Nk,d", [(6, 1, 1, 3000, 3000, 128), (6, 1, 1, 3000, 3000, 64), (2, 2, 2, 700, 1500, 96), (1, 3, 1, 5000, 900, 72), (8, 2, 1, 1023, 517, 64)])
def test_float32_splits_count_the_bytes_that_the_join_moves(B, G, r, Nq, Nk, d):
    """The backward's workspace is D_i and the partials of dk, dv or of dq.  Splits, as at_plan states them: rounds of workgroups times the tiles of a
    split (D / 20 + 1 us each), and for a join 4 us and the partials at 4.7 TB/s, written and read once: Nk keys, whatever number of waves owns them."""
    from aadg_amd import _lib
    D = 32 if d <= 32 else 64 if d <= 64 else 128

    def splits(own, count, other, tile, small, tensors):
        nw = small if own <= 32 * small else 4
        waves, n = B * G * (-(-own // (32 * nw))) * nw, -(-other // tile)
        part = 8.0 * tensors * B * G * count * d / 4.7e6
        costs = [((waves * x + 1023) // 1024 * -(-n // x)) * (D / 20.0 + 1.0) + (4.0 + part * x if x > 1 else 0.0) for x in range(1, min(64, n) + 1)]
        per = -(-n // (costs.index(min(costs)) + 1))
        return -(-n // per)
    f = 2 if d > 64 else 1
    sk, sq = splits(f * Nk, Nk, r * Nq, 32, f, 2), splits(r * Nq, r * Nq, Nk, 64, 1, 1)
    want = -(-B * G * r * Nq * 4 // 256) * 256 + max(sk * 2 * B * G * Nk * d * 4 if sk > 1 else 0, sq * B * G * r * Nq * d * 4 if sq > 1 else 0)
    desc = _desc(_lib, dtype=0, B=B, H=G * r, G=G, Nq=Nq, Nk=Nk, d=d)
    assert _lib.load().aadg_attention_backward_workspace_bytes(ctypes.byref(desc)) == want


@pytest.mark.parametrize("change", [dict(scale=1e39), dict(Nq=1 << 31), dict(B=1 << 33)])
def test_descriptor_refuses_what_it_cannot_hold(change):
    from aadg_amd import _lib
    a = {**dict(dtype=0, B=1, H=1, G=1, Nq=8, Nk=8, d=8, causal=False, scale=1.0), **change}
    with pytest.raises(_lib.AadgError):
        _lib._attn_desc(*a.values())
