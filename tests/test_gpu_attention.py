"""GPU: softmax attention (csrc/attention.hip, the transformer blocks: mix_transformer.py:86-100) against its definition in 64 bits,
forward and gradients.

Tolerances are bounds, element by element.  With u = 2^-24, t = half a step of the tensors' type, P the probabilities, |.| elementwise:
  scores      d + 4 roundings of sum |q||k|: relative error of p   e = u ((d + 4) max(scale |Q||K|^T) + Nk + 32)
  o           t |o| (store) + (t + e + u Nk) P |V|                 (p is rounded to the tensors' type for the product)
  dP, D       u (d + 2) |dO||V|^T;   |dO| . o_err + u (d + 2) |dO| . |o|
  dS          P (e (|dP| + |D|) + dP_err + D_err + 4 u (|dP| + |D|)) + t |dS|
  dq, dk, dv  the products of these with |K|, |Q|, |dO|, + u n of the accumulation, + t of the store
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def definition(q, k, v, scale, causal, lengths, do=None, few_keys=False):
    """o, (dq, dk, dv) and their error bounds, in float64."""
    dt = q.dtype
    t, u = torch.finfo(dt).eps / 2, 2.0 ** -24
    B, H, Nq, d = q.shape
    G, Nk = k.shape[1], k.shape[2]
    r = H // G
    Q, K, V = q.double(), k.double().repeat_interleave(r, 1), v.double().repeat_interleave(r, 1)
    L = torch.full((B,), Nk, device=q.device) if lengths is None else lengths.long().clamp(0, Nk)
    j, i = torch.arange(Nk, device=q.device), torch.arange(Nq, device=q.device)
    ok = (j.view(1, 1, 1, Nk) < L.view(B, 1, 1, 1)).expand(B, 1, Nq, Nk)
    if causal:
        ok = ok & (j.view(1, 1, 1, Nk) <= i.view(1, 1, Nq, 1) + (L - Nq).view(B, 1, 1, 1))
    used = j.view(1, 1, Nk, 1) < L.view(B, 1, 1, 1)
    K, V = torch.where(used, K, 0.0), torch.where(used, V, 0.0)
    KT, VT = K.transpose(2, 3).contiguous(), V.transpose(2, 3).contiguous()
    S = (scale * torch.matmul(Q, KT)).masked_fill(~ok, -math.inf)
    m = S.amax(3, keepdim=True)
    P = torch.exp(S - torch.where(m == -math.inf, 0.0, m))
    l = P.sum(3, keepdim=True)
    P = P / torch.where(l == 0, 1.0, l)
    o = torch.matmul(P, V)
    A = (scale * torch.matmul(Q.abs(), KT.abs())).masked_fill(~ok, 0.0).max().item()
    e = u * ((d + 4) * A + Nk + 32)
    o_err = t * o.abs() + (t + e + u * Nk) * torch.matmul(P, V.abs())
    if do is None:
        return o, o_err
    g = do.double()
    dP, D = torch.matmul(g, VT), (g * o).sum(3, keepdim=True)
    mag = dP.abs() + D.abs()
    dS = P * (dP - D)
    D_err = (g.abs() * o_err).sum(3, keepdim=True) + u * (d + 2) * (g.abs() * o.abs()).sum(3, keepdim=True)
    ts = t
    if few_keys:                                                            # D_i = sum_j p_ij dp_ij, none of o's rounding in it; dS in two terms
        ts = t if 32 < Nk <= 256 and 32 < d <= 64 else t * t
        D_err = (P * ((e + u * (Nk + 8)) * mag + u * (d + 2) * torch.matmul(g.abs(), VT.abs()))).sum(3, keepdim=True)
    dS_err = P * (e * mag + u * (d + 2) * torch.matmul(g.abs(), VT.abs()) + D_err + 4 * u * mag) + ts * dS.abs()
    fold = lambda x: x.view(B, G, r, Nk, d).sum(2)                                              # noqa: E731  heads that share a key head
    tr = lambda x: x.transpose(2, 3).contiguous()                                               # noqa: E731
    dq, dk, dv = scale * torch.matmul(dS, K), fold(scale * torch.matmul(tr(dS), Q)), fold(torch.matmul(tr(P), g))
    n = r * Nq
    dq_err = scale * torch.matmul(dS_err + u * Nk * dS.abs(), K.abs()) + t * dq.abs()
    dk_err = fold(scale * torch.matmul(tr(dS_err + u * n * dS.abs()), Q.abs())) + t * dk.abs()
    dv_err = fold((t + e + u * n) * torch.matmul(tr(P), g.abs())) + t * dv.abs()
    return (o, o_err), (dq, dq_err), (dk, dk_err), (dv, dv_err)


def check(got, want_err, name):
    want, err = want_err
    bad = (got.double() - want).abs() - (1.01 * err + 1e-30)
    assert torch.isfinite(got).all(), name
    assert bad.max().item() <= 0, "%s: worst excess %.3e at bound %.3e" % (name, bad.max().item(), err.flatten()[bad.argmax()].item())


def inputs(dtype, B, H, G, Nq, Nk, d, seed=0, std=1.0):
    torch.manual_seed(seed * 7919 + B * 1000 + Nq * 31 + Nk * 7 + d)
    mk = lambda *s: (torch.randn(*s, device="cuda") * std).to(dtype)                             # noqa: E731
    return mk(B, H, Nq, d), mk(B, G, Nk, d), mk(B, G, Nk, d), mk(B, H, Nq, d)


SHAPES = [
    # B, H, G, Nq, Nk, d, causal, lengths
    (1, 1, 1, 1, 1, 8, False, None),
    (1, 1, 1, 1, 1, 128, True, None),
    (2, 2, 2, 33, 31, 32, False, None),
    (3, 4, 2, 1, 300, 64, False, [300, 0, 7]),              # single tokens against a cache, one of them empty
    (2, 8, 1, 1, 2050, 128, True, [2050, 1999]),            # split over the keys
    (1, 6, 2, 5, 1000, 40, True, None),                     # rows of shared heads in one tile, causal
    (2, 1, 1, 130, 256, 64, False, None),
    (2, 3, 3, 257, 129, 64, True, None),                    # more queries than keys: the first rows are empty
    (2, 4, 2, 65, 65, 96, True, [65, 13]),
    (3, 2, 1, 200, 77, 24, False, [0, 77, 64]),
    (1, 2, 2, 64, 64, 64, True, None),
    (1, 4, 1, 100, 333, 128, True, None),
    (1, 2, 1, 2000, 40, 64, False, None),                   # many rows, few keys: split over the rows
    (1, 1, 1, 3, 3, 16, True, [2]),
    (1, 1, 1, 513, 700, 104, True, None),
    # bfloat16, 33 ... 256 keys, widths 33 ... 64: every key in one workgroup
    (2, 4, 2, 150, 200, 48, True, [200, 0]),
    (1, 1, 1, 1100, 256, 64, False, None),
    (2, 2, 1, 600, 100, 64, True, [100, 37]),
    (3, 1, 1, 31, 33, 40, False, None),
    (2, 2, 2, 1030, 250, 56, False, [250, 129]),
    (300, 1, 1, 40, 129, 64, False, None),
    # causal: more row tiles than places, tiles that do not divide by the shared heads; rows in long pieces
    (130, 3, 1, 200, 150, 32, True, None),
    (70, 6, 2, 300, 310, 72, True, None),
    (128, 8, 2, 1540, 70, 24, True, None),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_and_gradients_match_the_definition(hip, dtype, shape):
    B, H, G, Nq, Nk, d, causal, lens = shape
    q, k, v, do = inputs(dtype, B, H, G, Nq, Nk, d)
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    scale = d ** -0.5
    want = definition(q, k, v, scale, causal, lengths, do)
    with torch.no_grad():
        check(hip.attention(q, k, v, causal=causal, key_lengths=lengths), want[0], "o (no grad)")
    for t in (q, k, v):
        t.requires_grad_(True)
    o = hip.attention(q, k, v, causal=causal, key_lengths=lengths)
    grads = torch.autograd.grad(o, (q, k, v), do)
    assert o.dtype == dtype and o.shape == q.shape and o.transpose(1, 2).is_contiguous()
    check(o.detach(), want[0], "o")
    for name, g, w in zip(("dq", "dk", "dv"), grads, want[1:]):
        check(g, w, name)
    if lens is not None:                                                    # keys behind the length: exactly zero
        for b in range(B):
            assert not grads[1][b, :, lens[b]:].any() and not grads[2][b, :, lens[b]:].any()


@pytest.mark.parametrize("shape", [
    (1, 1, 1, 1, 1, 8, False, None),                        # one key: dq = dk = 0 but for float32's roundings
    (2, 4, 2, 17, 2, 24, True, None),
    (1, 5, 5, 400, 3, 16, False, None),
    (2, 4, 1, 130, 9, 128, False, [9, 2]),
    (3, 2, 2, 31, 32, 64, True, [32, 5, 0]),
    (2, 2, 2, 200, 32, 32, False, [32, 3]),
    (3, 2, 2, 70, 200, 64, False, [4, 1, 32]),              # every key in one workgroup, few of them in use
    (2, 4, 2, 32, 100, 48, True, [32, 17]),
    (2, 2, 1, 50, 900, 40, False, [2, 30]),                 # a long cache, few of its keys in use: split over the keys
])
def test_gradients_of_few_keys_do_not_carry_the_rounding_of_the_output(hip, shape):
    B, H, G, Nq, Nk, d, causal, lens = shape
    q, k, v, do = inputs(torch.bfloat16, B, H, G, Nq, Nk, d, seed=11)
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = definition(q, k, v, d ** -0.5, causal, lengths, do, few_keys=True)
    for t in (q, k, v):
        t.requires_grad_(True)
    o = hip.attention(q, k, v, causal=causal, key_lengths=lengths)
    for name, g, w in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do), want[1:]):
        check(g, w, name)
    o = hip.attention(q.detach(), k, v, causal=causal, key_lengths=lengths)
    for name, g, w in zip(("dk", "dv"), torch.autograd.grad(o, (k, v), do), want[2:]):          # without dq
        check(g, w, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Nq,Nk", [(96, 100), (1, 5000), (300, 20)])
def test_large_scores_and_scales(hip, dtype, Nq, Nk):
    """scores far beyond exp's range, a scale other than the default"""
    q, k, v, do = inputs(dtype, 1, 2, 2, Nq, Nk, 64, seed=3, std=4.0)
    want = definition(q, k, v, 0.7, False, None, do)
    for t in (q, k, v):
        t.requires_grad_(True)
    o = hip.attention(q, k, v, scale=0.7)
    check(o.detach(), want[0], "o")
    for name, g, w in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do), want[1:]):
        check(g, w, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_behind_the_length_are_never_used(hip, dtype):
    B, H, Nq, Nk, d = 2, 2, 70, 150, 64
    q, k, v, do = inputs(dtype, B, H, H, Nq, Nk, d)
    lengths = torch.tensor([90, 0], dtype=torch.int32, device="cuda")

    def run(k, v):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        o = hip.attention(*leaves, key_lengths=lengths)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]
    want = run(k, v)
    for poison in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min):
        kp, vp = k.clone(), v.clone()
        kp[0, :, 90:] = poison
        vp[0, :, 90:] = poison
        kp[1], vp[1] = poison, poison
        for a, b in zip(run(kp, vp), want):
            assert torch.equal(a, b)
    assert not want[0][1].any() and not any(g[1].any() for g in want[1:])               # a sequence without keys
    big = torch.tensor([10 ** 9, -5], dtype=torch.int32, device="cuda")                 # clamped to 0 ... Nk
    full = torch.tensor([Nk, 0], dtype=torch.int32, device="cuda")
    assert torch.equal(hip.attention(q, k, v, key_lengths=big), hip.attention(q, k, v, key_lengths=full))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_broadcast_and_misaligned_inputs(hip, dtype):
    """The projections' own layouts are read in place, a broadcast batch gets its summed gradient, and a row that does not start on a 16-byte
    boundary is copied first."""
    B, H, Nq, Nk, d = 3, 2, 50, 40, 64
    torch.manual_seed(5)
    x = torch.randn(B, Nq, H * d, device="cuda").to(dtype).requires_grad_(True)
    kv = torch.randn(B, Nk, 2 * H * d, device="cuda").to(dtype).requires_grad_(True)
    do = torch.randn(B, H, Nq, d, device="cuda").to(dtype)
    q = x.view(B, Nq, H, d).transpose(1, 2)
    k, v = kv.view(B, Nk, 2, H, d).permute(2, 0, 3, 1, 4).unbind(0)
    gx, gkv = torch.autograd.grad(hip.attention(q, k, v), (x, kv), do)
    want = definition(q.detach(), k.detach(), v.detach(), d ** -0.5, False, None, do)
    check(gx.view(B, Nq, H, d).transpose(1, 2), want[1], "dq")
    gk, gv = gkv.view(B, Nk, 2, H, d).permute(2, 0, 3, 1, 4).unbind(0)
    check(gk, want[2], "dk")
    check(gv, want[3], "dv")
    # one key set for the whole batch
    k1 = k.detach()[:1].clone().requires_grad_(True)
    o = hip.attention(q.detach(), k1.expand(B, -1, -1, -1), v.detach())
    want = definition(q.detach(), k1.detach().expand(B, -1, -1, -1), v.detach(), d ** -0.5, False, None, do)
    check(o.detach(), want[0], "o")
    g = torch.autograd.grad(o, k1, do)[0]
    t = torch.finfo(dtype).eps / 2
    check(g, (want[2][0].sum(0, keepdim=True), want[2][1].sum(0, keepdim=True) + 3 * t * want[2][0].abs().sum(0, keepdim=True)), "dk of the broadcast")
    # rows one element off a 16-byte boundary; a gradient without contiguous rows
    buf = torch.randn(B * H * Nq * d + 1, device="cuda").to(dtype)
    qm = buf[1:].view(B, H, Nq, d).requires_grad_(True)
    om = hip.attention(qm, k.detach(), v.detach())
    want = definition(qm.detach(), k.detach(), v.detach(), d ** -0.5, False, None, torch.ones_like(do))
    check(om.detach(), want[0], "o")
    check(torch.autograd.grad(om.sum(), qm)[0], want[1], "dq")


def test_gradients_match_differences(hip):
    """float32: directional central differences of a scalar of the output, in 64 bits over the kernel's float32 outputs.  Step 2^-7: the
    rounding of the outputs (~1e-6 relative) gives ~1e-4 of the slope, the third-order term ~1e-4."""
    q, k, v, do = inputs(torch.float32, 2, 4, 2, 37, 53, 32, seed=9)
    lengths = torch.tensor([53, 20], dtype=torch.int32, device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    f = lambda a: (hip.attention(*a, causal=True, key_lengths=lengths).double() * do.double()).sum()         # noqa: E731
    grads = torch.autograd.grad(f(leaves), leaves)
    eps = 2.0 ** -7
    with torch.no_grad():
        for i in range(3):
            torch.manual_seed(i)
            w = torch.randn_like(leaves[i])
            w = w / w.norm() * 8
            at = lambda s: f([t + s * eps * w if n == i else t for n, t in enumerate((q, k, v))]).item()         # noqa: E731
            slope = (grads[i].double() * w.double()).sum().item()
            assert abs((at(1) - at(-1)) / (2 * eps) - slope) <= 2e-3 * max(1.0, grads[i].norm().item())


def test_selected_gradients_and_repeatability(hip):
    q, k, v, do = inputs(torch.bfloat16, 2, 4, 2, 300, 700, 64)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    all_ = torch.autograd.grad(hip.attention(*leaves, causal=True), leaves, do)
    again = torch.autograd.grad(hip.attention(*leaves, causal=True), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(all_, again))                          # fixed order of every sum
    only_q = torch.autograd.grad(hip.attention(leaves[0], k, v, causal=True), leaves[0], do)[0]
    only_v = torch.autograd.grad(hip.attention(q, k, leaves[2], causal=True), leaves[2], do)[0]
    assert torch.equal(only_q, all_[0]) and torch.equal(only_v, all_[2])


def test_empty_inputs(hip):
    q, k = torch.randn(2, 2, 0, 64, device="cuda", requires_grad=True), torch.randn(2, 2, 5, 64, device="cuda", requires_grad=True)
    o = hip.attention(q, k, k)
    assert o.shape == (2, 2, 0, 64) and not torch.autograd.grad(o.sum(), k)[0].any()
    q2, k2 = torch.randn(2, 2, 3, 64, device="cuda", requires_grad=True), torch.randn(2, 2, 0, 64, device="cuda")
    o = hip.attention(q2, k2, k2)
    assert o.shape == q2.shape and not o.any() and not torch.autograd.grad(o.sum(), q2)[0].any()


def test_offsets_past_32_bits(hip):
    """rows 2^24 elements apart: the last of 200 lies 6.7 GB into the buffer"""
    n, d = 200, 64
    buf = torch.empty(n << 24, dtype=torch.bfloat16, device="cuda")
    q, k, v, do = inputs(torch.bfloat16, 1, 1, 1, 40, n, d, seed=2)
    far = [buf[64 * i:].as_strided((1, 1, n, d), (0, 0, 1 << 24, 1)) for i in range(2)]
    far[0].copy_(k)
    far[1].copy_(v)
    got = hip.attention(q, *far)
    assert torch.equal(got, hip.attention(q, k, v))
    leaves, near = [t.detach().requires_grad_(True) for t in far], [t.clone().requires_grad_(True) for t in (k, v)]
    for a, b in zip(torch.autograd.grad(hip.attention(q, *leaves), leaves, do), torch.autograd.grad(hip.attention(q, *near), near, do)):
        assert torch.equal(a, b)


def test_other_stream_and_captured_graph(hip):
    """A captured forward + backward replays on new inputs to the eager bits; two graphs and eager work keep apart."""
    shape = (2, 2, 1, 40, 1200, 64)
    cur = torch.cuda.current_stream()
    side = torch.cuda.Stream()
    lengths = torch.tensor([1200, 700], dtype=torch.int32, device="cuda")

    def step(q, k, v, do):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = hip.attention(*leaves, key_lengths=lengths)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]
    first = inputs(torch.bfloat16, *shape, seed=1)
    want = step(*first)
    side.wait_stream(cur)
    with torch.cuda.stream(side):
        got = step(*first)
    cur.wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got, want
    bufs = [[t.clone() for t in first], [t.clone() for t in first]]
    graphs, outs = [], []
    for b in bufs:
        side.wait_stream(cur)
        with torch.cuda.stream(side):
            step(*b)
        cur.wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*b))
        graphs.append(g)
    for n in range(3):
        fresh = [inputs(torch.bfloat16, *shape, seed=10 * n + w) for w in range(2)]
        for b, f in zip(bufs, fresh):
            for x, y in zip(b, f):
                x.copy_(y)
        for g in graphs:
            g.replay()
        for f, o in zip(fresh, outs):
            assert all(torch.equal(x, y) for x, y in zip(o, step(*f)))


def test_refusals(hip):
    q, k, v, _ = inputs(torch.float32, 2, 4, 2, 8, 8, 64)
    lens = torch.tensor([8, 8], dtype=torch.int32, device="cuda")
    bad = [dict(q=q.bfloat16()), dict(q=q.half(), k=k.half(), v=v.half()), dict(q=q[..., :60], k=k[..., :60], v=v[..., :60]), dict(v=v[:, :, :7]), dict(k=k[:1], v=v[:1]),
           dict(q=q[:, :3]), dict(q=q[0]), dict(q=torch.randn(2, 4, 8, 136, device="cuda"), k=torch.randn(2, 2, 8, 136, device="cuda"),
                                                v=torch.randn(2, 2, 8, 136, device="cuda")),
           dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(key_lengths=lens.long()), dict(key_lengths=lens[:1]),
           dict(key_lengths=lens.cpu()), dict(q=q.cpu()), dict(key_lengths=torch.stack([lens, lens], 1)[:, 0])]
    for kw in bad:
        with pytest.raises(hip.AadgError):
            hip.attention(**{**dict(q=q, k=k, v=v), **kw})
    x = q.clone().requires_grad_(True)
    g = torch.autograd.grad(hip.attention(x, k, v).sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()                                                              # differentiable once


@pytest.mark.parametrize("shape", [
    # bfloat16, sequences of up to 32 keys in a batch padded to 33 ... 256: the gradients of the same sequences in a batch padded to 32
    (3, 2, 2, 70, 200, 64, False, [4, 1, 32]),
    (2, 4, 2, 90, 100, 48, True, [32, 17]),
    (2, 1, 1, 1500, 256, 64, False, [31, 9]),               # rows split over workgroups
    (40, 2, 1, 33, 33, 40, False, [1 + i % 32 for i in range(40)]),
])
def test_gradients_of_few_keys_do_not_depend_on_the_padding(hip, shape):
    B, H, G, Nq, Nk, d, causal, lens = shape
    q, k, v, do = inputs(torch.bfloat16, B, H, G, Nq, Nk, d, seed=17)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    n = max(lens)
    want = definition(q, k[:, :, :n], v[:, :, :n], d ** -0.5, causal, lengths, do, few_keys=True)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(hip.attention(*leaves, causal=causal, key_lengths=lengths), leaves, do)
    check(grads[0], want[1], "dq")
    for name, g, w in zip(("dk", "dv"), grads[1:], want[2:]):
        check(g[:, :, :n], w, name)
        assert not g[:, :, n:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [
    # sequences without a key, causal sequences with more queries than keys: every backward kernel
    (3, 2, 1, 70, 200, 64, False, [200, 0, 64]),
    (2, 2, 2, 257, 129, 64, True, None),
    (2, 2, 1, 90, 100, 48, True, [100, 30]),
    (2, 4, 2, 400, 300, 32, True, [300, 7]),
    (2, 2, 1, 150, 100, 128, True, [100, 0]),
    (1, 2, 1, 40, 9, 96, True, None),
    (1, 2, 1, 40, 9, 16, True, None),
    (2, 1, 1, 900, 500, 64, True, [500, 420]),
])
def test_queries_that_see_no_key_take_no_part_whatever_they_hold(hip, dtype, shape):
    B, H, G, Nq, Nk, d, causal, lens = shape
    q, k, v, do = inputs(dtype, B, H, G, Nq, Nk, d, seed=23)
    L = [Nk] * B if lens is None else lens
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    rows = [Nq if n == 0 else max(0, Nq - n) if causal else 0 for n in L]              # the first rows of a sequence see nothing

    def run(fill, ask):
        leaves = [t.clone() for t in (q, k, v)]
        g = do.clone()
        for b, n in enumerate(rows):
            leaves[0][b, :, :n] = fill
            g[b, :, :n] = fill
        for i in ask:
            leaves[i].requires_grad_(True)
        o = hip.attention(*leaves, causal=causal, key_lengths=lengths)
        return [o.detach(), *torch.autograd.grad(o, [leaves[i] for i in ask], g)]
    assert any(rows)
    for ask in ((0, 1, 2), (1, 2), (0,)):
        want = run(0.0, ask)
        for fill in (float("nan"), float("inf")):
            got = run(fill, ask)
            assert all(torch.isfinite(a).all() and torch.equal(a, b) for a, b in zip(got, want)), (ask, fill)


def test_more_rows_than_one_launch_of_16_lanes_a_row_has_threads(hip):
    """2^28 + 192 rows, gradients of keys and values only: 16 threads a row would be past the 2^32 threads of a launch.  All rows but the first and
    the last 128 are zero in q and dO and add nothing."""
    n, d, Nk = (1 << 28) + 192, 8, 40
    q, k, v, do = inputs(torch.bfloat16, 1, 1, 1, 256, Nk, d, seed=4)
    far = [torch.zeros(1, 1, n, d, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for f, t in zip(far, (q, do)):
        f[:, :, :128] = t[:, :, :128]
        f[:, :, n - 128:] = t[:, :, 128:]
    want = definition(q, k, v, d ** -0.5, False, None, do)
    leaves = [t.requires_grad_(True) for t in (k, v)]
    o = hip.attention(far[0], *leaves)
    check(torch.cat([o.detach()[:, :, :128], o.detach()[:, :, n - 128:]], 2), want[0], "o")
    for name, g, w in zip(("dk", "dv"), torch.autograd.grad(o, leaves, far[1]), want[2:]):
        check(g, w, name)


def test_forward_mode_derivatives_are_refused(hip):
    """a tangent is not dropped"""
    from torch.autograd import forward_ad
    q, k, v, _ = inputs(torch.float32, 1, 2, 2, 9, 12, 64)
    want = hip.attention(q, k, v)
    with forward_ad.dual_level():
        assert torch.equal(hip.attention(q, k, v), want)                                # no tangent anywhere
        for i in range(3):
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if n == i else t for n, t in enumerate((q, k, v))]
            with pytest.raises(NotImplementedError):
                hip.attention(*args)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                hip.attention(*args)


def test_sizes_and_scales_past_the_descriptor_are_refused(hip):
    q, k, v, _ = inputs(torch.float32, 1, 1, 1, 8, 8, 8)
    for kw in (dict(scale=1e39), dict(scale=1e-60), dict(key_lengths=[8]), dict(key_lengths=8)):
        with pytest.raises(hip.AadgError):
            hip.attention(q, k, v, **kw)
    wide = k[:, :, :1].expand(1, 1, 1 << 31, 8)
    assert not hip.attention_supported(q, wide, wide)
    with pytest.raises(hip.AadgError):
        hip.attention(q, wide, wide)
