"""Cases, plain forms and 64-bit definitions of the transformer-training operators: attention forward, attention forward + backward, and
the orthogonalised update of a list of weight matrices.

own = False: elementary torch operations in float32.  own = True: the calls a user of the package makes.
"""
import math

import torch

own = False

_COEF = (3.4445, -4.7750, 2.0315)          # the quintic a x + b x^3 + c x^5 of the orthogonalised update
_EPS = 1e-7


# ------------------------------------------------------------------------------------------------ cases
def _attn(name, kind, dtype, B, H, G, Nq, Nk, d, causal=False, ragged=False):
    return dict(name=name, op=kind, dtype=dtype, B=B, H=H, G=G, Nq=Nq, Nk=Nk, d=d, causal=causal, ragged=ragged)


def _orth(name, shapes):
    return dict(name=name, op="orthogonalize", shapes=";".join("%dx%d" % s for s in shapes))


def _encoder_matrices(dims, depths, sr):
    """The weight matrices of encoder stages after the one of width dims[0] (convolutions as [out, in * kh * kw])."""
    out = []
    for below, c, n, s in zip(dims, dims[1:], depths, sr):
        out.append((c, below * 9))                                                 # overlapping patch embedding
        for _ in range(n):
            out += [(c, c), (2 * c, c), (c, c), (4 * c, c), (c, 4 * c)]            # q, kv, proj, fc1, fc2
            if s > 1:
                out.append((c, c * s * s))                                         # key / value reduction
    return out


def listed():
    return [
        # one new token per sequence against a long cache, few shared key heads: latency and the cache's bytes
        _attn("attend_token", "attend", "bfloat16", 8, 8, 2, 1, 4096, 64, ragged=True),
        # first encoder stage, 512 x 512 crops, the 48 rows of one rank: many queries, 256 reduced keys
        _attn("attend_stage1", "attend", "bfloat16", 48, 1, 1, 16384, 256, 64),
        # long causal sequence, shared key heads: the largest
        _attn("attend_causal_8k", "attend", "bfloat16", 2, 16, 4, 8192, 8192, 128, causal=True),
        # third stage in float32
        _attn("attend_stage3_f32", "attend", "float32", 48, 5, 5, 1024, 256, 64),
        # a padded batch, odd sizes, a head width between the tiles, one sequence without any key
        _attn("attend_padded", "attend", "bfloat16", 7, 5, 5, 333, 259, 40, ragged=True),
        # training: first stage
        _attn("train_stage1", "train", "bfloat16", 48, 1, 1, 16384, 256, 64),
        # training: last stage of a small batch, launch-bound
        _attn("train_stage4", "train", "bfloat16", 6, 8, 8, 256, 256, 64),
        # training: causal, shared key heads
        _attn("train_causal_4k", "train", "bfloat16", 2, 8, 2, 4096, 4096, 128, causal=True),
        # training in float32, padded batch, odd lengths
        _attn("train_padded_f32", "train", "float32", 8, 2, 2, 1023, 517, 64, ragged=True),
        # one small matrix: fifteen dependent small products
        _orth("orth_one", [(64, 64)]),
        # every matrix of the last two stages of the B2 encoder (most of its parameters)
        _orth("orth_encoder", _encoder_matrices((128, 320, 512), (6, 3), (2, 1))),
        # wide and tall convolution matrices of the residual backbone and its pyramid head, an odd one among them
        _orth("orth_convs", [(512, 4608), (512, 2048), (2048, 1024), (256, 18432), (1024, 256), (37, 301)]),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "train", "orthogonalize"])
    if op == "orthogonalize":
        shapes, budget = [], 1.4e11
        for _ in range(_log(rng, 1, 40)):
            s = (_log(rng, 2, 2048), _log(rng, 2, 4608))
            f = _orth_flops([s])
            if f <= budget:
                budget -= f
                shapes.append(s)
        return dict(op=op, shapes=";".join("%dx%d" % s for s in (shapes or [(48, 65)])))
    dtype = rng.choice(["bfloat16", "float32"])
    G = rng.choice([1, 1, 2, 3, 4, 5])
    H = G * rng.choice([1, 1, 1, 2, 4])
    d = 8 * rng.randint(1, 16)
    limit = 4.0e8 if op == "attend" else 1.2e8                                     # score-matrix elements of the plain form
    while True:
        B, Nq, Nk = _log(rng, 1, 48), _log(rng, 1, 16384), _log(rng, 1, 8192)
        if B * H * Nq * Nk <= limit and B * H * max(Nq, Nk) * d <= 1.0e8:
            break
    return dict(op=op, dtype=dtype, B=B, H=H, G=G, Nq=Nq, Nk=Nk, d=d, causal=rng.random() < 0.4, ragged=rng.random() < 0.4)


def _lengths(case):
    """Keys of each sequence: 0 ... Nk in even steps (one sequence: all but a quarter)."""
    B, Nk = case["B"], case["Nk"]
    if not case["ragged"]:
        return [Nk] * B
    return [Nk * b // (B - 1) for b in range(B)] if B > 1 else [Nk - Nk // 4]


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(";")]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "orthogonalize":
        # gradients: a few strong directions over noise, small values
        mats = []
        for r, c in _shapes(case):
            low = torch.randn(r, 4, device="cuda", generator=gen) @ torch.randn(4, c, device="cuda", generator=gen)
            mats.append((torch.randn(r, c, device="cuda", generator=gen) + 0.5 * low) * 1e-3)
        return dict(case=case, mats=mats)
    dt = getattr(torch, case["dtype"])
    B, H, G, Nq, Nk, d = (case[k] for k in ("B", "H", "G", "Nq", "Nk", "d"))
    # as the projections leave them: queries [B, Nq, H, d], keys and values together [B, Nk, 2, G, d]
    q = torch.randn(B, Nq, H, d, device="cuda", generator=gen).to(dt).transpose(1, 2)
    kv = torch.randn(B, Nk, 2, G, d, device="cuda", generator=gen).to(dt).permute(2, 0, 3, 1, 4)
    st = dict(case=case, q=q, k=kv[0], v=kv[1], lengths=None, scale=d ** -0.5)
    if case["ragged"]:
        st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    if case["op"] == "train":
        st["do"] = (torch.randn(B, Nq, H, d, device="cuda", generator=gen) * 0.1).to(dt).transpose(1, 2)
        if own:
            for n in "qkv":
                st[n].requires_grad_(True)
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if state["case"]["op"] == "orthogonalize":
        if own:
            from aadg_amd import _lib
            return _lib.orthogonalize(state["mats"])
        return [_orthogonalize_plain(u) for u in state["mats"]]
    q, k, v, causal = state["q"], state["k"], state["v"], state["case"]["causal"]
    if own:
        from aadg_amd import _lib
        o = _lib.attention(q, k, v, scale=state["scale"], causal=causal, key_lengths=state["lengths"])
        if "do" not in state:
            return o
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), state["do"])]
    return _attention_plain(q, k, v, state.get("do"), state["scale"], causal, state["lengths"])


def _allowed(B, Nq, Nk, causal, lengths, device):
    """[B or 1, 1, Nq or 1, Nk] truth values, None where every query sees every key."""
    if not causal and lengths is None:
        return None
    j = torch.arange(Nk, device=device).view(1, 1, 1, Nk)
    L = torch.full((1, 1, 1, 1), Nk, device=device) if lengths is None else lengths.long().view(B, 1, 1, 1)
    ok = j < L
    if causal:
        ok = ok & (j <= torch.arange(Nq, device=device).view(1, 1, Nq, 1) + L - Nq)
    return ok


def _attention_plain(q, k, v, do, scale, causal, lengths):
    dt, (B, H, Nq, d), G, Nk = q.dtype, q.shape, k.shape[1], k.shape[2]
    r = H // G
    qf = q.float().reshape(B, G, r * Nq, d)
    kf, vf = k.float().contiguous(), v.float().contiguous()
    s = torch.matmul(qf, kf.transpose(2, 3)).view(B, H, Nq, Nk) * scale
    ok = _allowed(B, Nq, Nk, causal, lengths, q.device)
    if ok is not None:
        s = s.masked_fill(~ok, -math.inf)
    m = s.amax(dim=3, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    del s
    l = p.sum(dim=3, keepdim=True)
    p = p / torch.where(l == 0, torch.ones_like(l), l)
    pg = p.view(B, G, r * Nq, Nk)
    of = torch.matmul(pg, vf)
    o = of.view(B, H, Nq, d).to(dt)
    if do is None:
        return o
    dof = do.float().reshape(B, G, r * Nq, d)
    dv = torch.matmul(pg.transpose(2, 3), dof)
    ds = pg * (torch.matmul(dof, vf.transpose(2, 3)) - (dof * of).sum(dim=3, keepdim=True))
    dq = torch.matmul(ds, kf).view(B, H, Nq, d) * scale
    dk = torch.matmul(ds.transpose(2, 3), qf) * scale
    return [o, dq.to(dt), dk.to(dt), dv.to(dt)]


def _orthogonalize_plain(u):
    a, b, c = _COEF
    tall = u.shape[0] > u.shape[1]
    x = u.t() if tall else u
    x = x / (torch.sqrt((x * x).sum()) + _EPS)
    for _ in range(5):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if tall else x


# ------------------------------------------------------------------------------------------------ counts and definition
def _pairs(case):
    """(query, key) pairs the definition has, all heads."""
    n, Nq = 0, case["Nq"]
    for L in _lengths(case):
        if not case["causal"]:
            n += Nq * L
        else:
            # query i sees max(0, i + L - Nq + 1) keys
            first = max(0, Nq - L)
            n += sum((first + L - Nq + 1, L)) * (Nq - first) // 2 if first < Nq else 0
    return n * case["H"]


def _orth_flops(shapes):
    t = 0.0
    for r, c in shapes:
        m, n = min(r, c), max(r, c)
        t += 5.0 * (3.0 * m * m * n + m * m * m)                                   # two symmetric products at half, one full
    return t


def work(case):
    if case["op"] == "orthogonalize":
        shapes = _shapes(case)
        return dict(bytes=float(sum(8 * r * c for r, c in shapes)), flops=_orth_flops(shapes))
    size = 2 if case["dtype"] == "bfloat16" else 4
    q = case["B"] * case["H"] * case["Nq"] * case["d"] * size
    kv = 2 * sum(_lengths(case)) * case["G"] * case["d"] * size
    train = case["op"] == "train"
    full = 2 * case["B"] * case["Nk"] * case["G"] * case["d"] * size
    return dict(bytes=float(2 * q + kv + ((2 * q + full) if train else 0)), flops=float(_pairs(case) * case["d"] * (14 if train else 4)))


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "orthogonalize":
        out = []
        for u in st["mats"]:
            # the same odd polynomial, applied from the other side: X <- X (a + b X'X + c (X'X)^2) on the narrow orientation
            w = u.double()
            y = w if w.shape[0] >= w.shape[1] else w.t()
            y = y / (torch.linalg.vector_norm(y) + _EPS)
            eye = torch.eye(y.shape[1], dtype=torch.float64, device=y.device)
            for _ in range(5):
                h = y.t() @ y
                y = y @ (_COEF[0] * eye + h @ (_COEF[1] * eye + _COEF[2] * h))
            out.append(y if w.shape[0] >= w.shape[1] else y.t())
        return out
    train, scale = case["op"] == "train", case["d"] ** -0.5
    B, H, G, Nq, Nk, d = (case[k] for k in ("B", "H", "G", "Nq", "Nk", "d"))
    lens = _lengths(case)
    f64 = dict(dtype=torch.float64, device="cuda")
    o = torch.zeros(B, H, Nq, d, **f64)
    dq, dk, dv = torch.zeros_like(o), torch.zeros(B, G, Nk, d, **f64), torch.zeros(B, G, Nk, d, **f64)
    step = max(1, (1 << 26) // Nk)
    for b in range(B):
        L = lens[b]
        for h in range(H):
            g = h // (H // G)
            kb, vb = st["k"][b, g, :L].detach().double(), st["v"][b, g, :L].detach().double()
            for i0 in range(0, Nq, step):
                i1 = min(Nq, i0 + step)
                qb = st["q"][b, h, i0:i1].detach().double()
                first = 0                                                          # rows in front of it see no key
                if case["causal"]:
                    first = min(max(0, Nq - L - i0), i1 - i0)
                if L == 0 or first == i1 - i0:
                    continue
                qb = qb[first:]
                s = scale * (qb @ kb.t())
                if case["causal"]:
                    rows = torch.arange(i0 + first, i1, device="cuda")
                    s = s.masked_fill(torch.arange(L, device="cuda")[None, :] > (rows + (L - Nq))[:, None], -math.inf)
                p = torch.softmax(s, dim=1)
                ob = p @ vb
                o[b, h, i0 + first:i1] = ob
                if train:
                    gb = st["do"][b, h, i0 + first:i1].double()
                    dv[b, g, :L] += p.t() @ gb
                    t = gb @ vb.t()
                    t = p * (t - (t * p).sum(dim=1, keepdim=True))
                    dq[b, h, i0 + first:i1] = scale * (t @ kb)
                    dk[b, g, :L] += scale * (t.t() @ qb)
    return [o, dq, dk, dv] if train else o
