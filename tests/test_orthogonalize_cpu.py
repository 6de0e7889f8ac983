"""CPU: the orthogonalisation entry point checks its arguments on the host, before anything touches a GPU."""
import ctypes

import pytest
import torch


def test_orthogonalize_validates_arguments():
    from aadg_amd import _lib
    lib = _lib.load()
    z, ws = ctypes.c_void_p(0), ctypes.c_void_p(256)
    mk = lambda *m: (_lib._Matrix * len(m))(*m)                                                 # noqa: E731
    ok = mk((16, 16, 64, 100))
    f = ctypes.c_float
    call = lambda m, n=1, steps=5, eps=1e-7, w=ws, nb=1 << 40: lib.aadg_orthogonalize_f32(m, n, steps, f(3.0), f(-3.0), f(1.0), f(eps), w, nb, z)      # noqa: E731
    need = lib.aadg_orthogonalize_workspace_bytes(ok, 1)
    assert need >= 2 * 3 * 2 * 64 * 100
    assert lib.aadg_orthogonalize_workspace_bytes(z, 1) == 0 and lib.aadg_orthogonalize_workspace_bytes(ok, 0) == 0
    assert call(z) == -1 and call(ok, n=0) == -1 and call(ok, n=5000) == -1 and call(ok, steps=0) == -1 and call(ok, steps=65) == -1
    assert call(ok, eps=-1.0) == -1 and call(ok, eps=float("nan")) == -1
    assert call(mk((0, 16, 64, 100))) == -1 and call(mk((16, 0, 64, 100))) == -1 and call(mk((18, 16, 64, 100))) == -1
    assert call(mk((16, 16, 0, 100))) == -1 and call(mk((16, 16, 65537, 1))) == -3 and call(mk((16, 16, 1 << 15, (1 << 13) + 1))) == -3
    assert call(ok, nb=need - 1) == -2 and call(ok, w=z) == -2 and call(ok, w=ctypes.c_void_p(128)) == -2


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_orthogonalize_has_no_cpu_path():
    from aadg_amd import _lib
    with pytest.raises(_lib.AadgError):
        _lib.orthogonalize([torch.zeros(3, 4)])
