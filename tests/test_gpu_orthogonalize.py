"""GPU: orthogonalised updates (csrc/orthogonalize.hip) against the definition in 64 bits.

The kernels' products are float32-grade, like those of the float32 form written with torch: the same number of float32 roundings, in another
order.  The iteration magnifies both by the same singular-value map, so the bound is set by the float32 form's own distance from the
definition on the same matrix: three times it (two independent samples of one error, of matrices down to one element), plus 2^-21 of the
result's size where that distance happens to be zero."""
import pytest
import torch

pytestmark = pytest.mark.gpu
COEF = (3.4445, -4.7750, 2.0315)


def form(u, dtype, steps=5, eps=1e-7, coef=COEF):
    a, b, c = coef
    x = u.to(dtype)
    x = x.t() if u.shape[0] > u.shape[1] else x
    x = x / (x.double().square().sum().sqrt().to(dtype) + eps)
    for _ in range(steps):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return (x.t() if u.shape[0] > u.shape[1] else x).contiguous()


def check(got, u, **kw):
    want, plain = form(u, torch.float64, **kw), form(u, torch.float32, **kw)
    assert got.shape == u.shape and got.dtype == torch.float32 and got.is_contiguous() and torch.isfinite(got).all()
    size = want.square().mean().sqrt().item()
    rms = lambda x: (x.double() - want).square().mean().sqrt().item()                          # noqa: E731
    worst = lambda x: (x.double() - want).abs().max().item()                                   # noqa: E731
    assert rms(got) <= 3 * rms(plain) + 2.0 ** -21 * size, (u.shape, rms(got), rms(plain))
    assert worst(got) <= 3 * worst(plain) + 2.0 ** -19 * want.abs().max().item(), (u.shape, worst(got), worst(plain))


def matrix(r, c, kind="noise", seed=0):
    torch.manual_seed(seed * 131 + r * 7 + c)
    u = torch.randn(r, c, device="cuda")
    if kind == "low rank":
        u = torch.randn(r, 3, device="cuda") @ torch.randn(3, c, device="cuda") + 0.01 * u
    return u * 1e-3


@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (2, 768), (7, 5), (31, 33), (64, 64), (65, 64), (37, 301), (301, 37), (64, 4096), (320, 1280),
                                   (130, 257), (512, 512), (768, 100), (257, 2304)])
@pytest.mark.parametrize("kind", ["noise", "low rank"])
def test_one_matrix(hip, shape, kind):
    u = matrix(*shape, kind)
    keep = u.clone()
    check(hip.orthogonalize([u])[0], u)
    assert torch.equal(u, keep)


def test_lists(hip):
    """sizes mixed in one call, more than one table launch, wide tiles; equal inputs give equal bits wherever they stand in the list"""
    shapes = [(320, 320), (640, 320), (1280, 320), (320, 1280), (5, 3), (64, 147), (512, 2048), (1, 1), (256, 2304), (768, 320)] * 4 + [(1024, 512)] * 3
    mats = [matrix(r, c, "low rank" if i % 3 == 0 else "noise", seed=i) for i, (r, c) in enumerate(shapes)]
    out = hip.orthogonalize(mats)
    for u, o in list(zip(mats, out))[::3]:
        check(o, u)
    again = hip.orthogonalize(mats[::-1])[::-1]
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    # mats[1] is noise, 640 x 320: singular values of U / |U|_F between (sqrt 640 -+ sqrt 320) / sqrt(640 320) = 0.016 and 0.095; five steps take
    # 0.016 through 0.056, 0.19, 0.63 into the band of the quintic, 0.68 ... 1.21 (mats[0] is of rank 3 over 1 % noise: its small ones stay small)
    sv = torch.linalg.svdvals(out[1].double())
    assert sv.max() < 1.25 and sv.min() > 0.6


def test_extremes(hip):
    zero = torch.zeros(20, 30, device="cuda")
    assert not hip.orthogonalize([zero])[0].any()
    for s in (1e30, 1e-30):                                             # squares outside float32
        u = matrix(40, 50) * s
        check(hip.orthogonalize([u], eps=0.0)[0], u, eps=0.0)
    u = matrix(40, 50)
    bad = u.clone()
    bad[3, 4] = float("nan")
    inf = u.clone()
    inf[3, 4] = float("inf")
    out = hip.orthogonalize([u, bad, u, inf, u])                        # a broken matrix stays its own
    assert torch.isnan(out[1]).all() and torch.isnan(out[3]).any()
    assert torch.equal(out[0], out[2]) and torch.equal(out[0], out[4]) and torch.isfinite(out[0]).all()
    assert hip.orthogonalize([]) == []
    e = hip.orthogonalize([torch.empty(0, 5, device="cuda"), u])
    assert e[0].shape == (0, 5) and torch.equal(e[1], out[0])
    check(hip.orthogonalize([u], steps=1, coefficients=(1.5, -0.5, 0.0))[0], u, steps=1, coef=(1.5, -0.5, 0.0))
    check(hip.orthogonalize([u], steps=2)[0], u, steps=2)


def test_strided_and_unaligned(hip):
    u = matrix(60, 90)
    check(hip.orthogonalize([u.t()])[0], u.t())
    buf = torch.cat([torch.zeros(1, device="cuda"), u.flatten()])
    v = buf[1:].view(60, 90)                                            # 4-byte alignment, as a slice of a gradient bucket
    assert torch.equal(hip.orthogonalize([v])[0], hip.orthogonalize([u])[0])


def test_in_place_through_the_library(hip):
    """aadg_orthogonalize_f32 with dst == src (aadg_hip.h allows it), and the same matrix twice in a list"""
    import ctypes
    u, v = matrix(70, 130), matrix(90, 20)
    want = hip.orthogonalize([u, v, u])
    assert torch.equal(want[0], want[2])
    a, b = u.clone(), v.clone()
    arr = (hip._Matrix * 2)((a.data_ptr(), a.data_ptr(), 70, 130), (b.data_ptr(), b.data_ptr(), 90, 20))
    lib = hip.load()
    need = lib.aadg_orthogonalize_workspace_bytes(arr, 2)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    f = ctypes.c_float
    assert lib.aadg_orthogonalize_f32(arr, 2, 5, f(COEF[0]), f(COEF[1]), f(COEF[2]), f(1e-7), ws.data_ptr(), need, hip._stream()) == 0
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_stream_and_graph(hip):
    mats = [matrix(64, 200), matrix(300, 40), matrix(128, 128)]
    want = hip.orthogonalize(mats)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = hip.orthogonalize(mats)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    bufs = [m.clone() for m in mats]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = hip.orthogonalize(bufs)
    for n in range(3):
        fresh = [matrix(*m.shape, seed=n + 5) for m in mats]
        for b, f in zip(bufs, fresh):
            b.copy_(f)
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, hip.orthogonalize(fresh)))


def test_refusals(hip):
    u = matrix(8, 9)
    for bad in ([u.double()], [u.bfloat16()], [u[0]], [u.cpu()], [u, u.cpu()], [u[None]]):
        with pytest.raises(hip.AadgError):
            hip.orthogonalize(bad)
    for kw in (dict(steps=0), dict(steps=65), dict(eps=-1.0), dict(eps=float("nan")), dict(coefficients=(1.0, 2.0))):
        with pytest.raises(hip.AadgError):
            hip.orthogonalize([u], **kw)
    with pytest.raises(hip.AadgError):
        hip.orthogonalize([torch.zeros(1, 65537, device="cuda")])
