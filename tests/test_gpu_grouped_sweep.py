"""Seeded random calls of the grouped products and the adapters over sizes, alignment, strides, lists and epilogues: against
64-bit products, with NaN wherever a call has nothing to read, and captured after one eager call."""
import random

import pytest
import torch

from test_gpu_grouped import F16, F32, ints, vedic

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F64 = torch.float64
GELU_C = 0.7978845608028654
NAN = float("nan")


def gelu(x):
    return 0.5 * x * (1 + torch.tanh(GELU_C * (x + 0.044715 * x ** 3)))


def gelu_grad(x):
    t = torch.tanh(GELU_C * (x + 0.044715 * x ** 3))
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * GELU_C * (1 + 3 * 0.044715 * x * x)


def log(r, lo, hi):
    return int(round(lo * (hi / lo) ** r.random()))


def width(r, lo, hi):
    w, p = log(r, lo, hi), r.random()
    return max(lo, w // 64 * 64) if p < 0.35 else max(8, w // 8 * 8) if p < 0.6 else w


def laid(x, r):
    """x with padding (NaN) behind its rows and its base off by some elements, or as it is; the view and its buffer."""
    pad, shift = r.choice([(0, 0), (0, 0), (8, 0), (3, 0), (8, 1), (0, 1), (5, 3)])
    *lead, a, b = x.shape
    buf = torch.full((x.numel() // b * (b + pad) + shift,), NAN, dtype=x.dtype, device="cuda")
    view = buf[shift:].view(*lead, a, b + pad)[..., :b]
    view.copy_(x)
    return view, buf


def close(got, want, mag, K, dtype, extra=0.0):
    """K sums of the magnitudes' size and four more roundings; the output's own; a GELU's (extra)."""
    half = 2.0 ** -11 if dtype == F16 else U
    tol = (K + 4) * U * mag + 2 * half * want.abs() + extra + (2.0 ** -24 if dtype == F16 else 2.0 ** -140)
    return bool(((got.double() - want).abs() <= tol).all())


def grouped(v, r, g):
    """One call of vedic_gemm_grouped: the call, and the check of what it wrote."""
    op = r.choice([v.OP_NN, v.OP_NT, v.OP_TN])
    tn = op == v.OP_TN
    dt = r.choice([F16, F16, F32])
    ot = F16 if dt == F16 and not tn and r.random() < 0.5 else F32
    G, R = (log(r, 1, 80) if r.random() < 0.95 else 1024), log(r, 1, 4000)
    K, N = width(r, 1, 2600), width(r, 1, 1200)
    while R * K * N > 1e9 or G * K * N > 3e7:
        K, N, R = max(1, K // 2), max(1, N // 2), max(1, R - R // 4)
    sizes = [int(R / G * 2 * r.random() ** 2) if r.random() > 0.25 else 0 for _ in range(G)]
    off = [0]
    for n in sizes:
        off.append(off[-1] + n)
    used = off[-1]
    R = max(used, R)
    listed = r.random() < 0.5
    T = max(1, r.choice([R // 2, R + 1, 3 * R])) if listed else R
    mk = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=g) * std).to(dt)
    A, B = mk(T, K), mk(R, N) if tn else mk(G, *((K, N) if op == v.OP_NN else (N, K)), std=K ** -0.5)
    a, b = A.double(), B.double()
    live = torch.zeros(T, dtype=torch.bool, device="cuda")
    rows = None
    if listed:
        rows = torch.randint(0, T, (R,), device="cuda", generator=g, dtype=torch.int32)
        if r.random() < 0.3:
            rows[torch.rand(R, device="cuda", generator=g) < 0.1] = r.choice([-1, T, 2 ** 31 - 1, -2 ** 31])
        ok = (rows >= 0) & (rows < T)
        a = torch.where(ok[:, None], a[rows.clamp(0, T - 1).long()], torch.zeros((), dtype=F64, device="cuda"))
        live[rows[:used][ok[:used]].long()] = True
    else:
        live[:used] = True
    A, _ = laid(A, r)
    B, _ = laid(B, r)
    A[~live] = NAN
    if tn:
        B[used:] = NAN
    else:
        for i in range(G):
            if sizes[i] == 0:
                B[i] = NAN
    text = f"op {op} {dt} -> {ot} G {G} R {R} used {used} T {T} K {K} N {N} list {listed} A {A.stride()} B {B.stride()}"
    o = ints(off)
    if tn:
        beta = r.choice([0.0, 0.0, 1.0, -0.5])
        c0, db0 = torch.randn(G, K, N, device="cuda", generator=g), torch.randn(G, N, device="cuda", generator=g)
        C, buf = laid(c0, r)
        db = db0.clone()

        def call():
            C.copy_(c0)
            db.copy_(db0)
            return v.gemm_grouped(op, A, B, o, C, rows=rows, beta=beta, db=db, db_beta=beta), db

        def check():
            for i in range(G):
                s, n = slice(off[i], off[i + 1]), max(1, sizes[i])
                if not close(C[i], a[s].t() @ b[s] + beta * c0[i].double(), a[s].abs().t() @ b[s].abs() + abs(beta) * c0[i].abs(),
                             n, F32):
                    return False
                if not close(db[i], b[s].sum(0) + beta * db0[i].double(), b[s].abs().sum(0) + abs(beta) * db0[i].abs(), n, F32):
                    return False
            return int(torch.isnan(buf).sum()) == buf.numel() - G * K * N

        return text, call, check
    epi = r.choice(["none", "bias", "gelu", "gelu and preact"] if op == v.OP_NN else ["none", "gelu backward"])
    C, buf = laid(torch.empty(R, N, dtype=ot, device="cuda"), r)
    kw, P = dict(rows=rows), None
    if op == v.OP_NN and epi != "none":
        bias = torch.randn(G, N, device="cuda", generator=g)
        kw.update(bias=bias, epilogue=v.EPI_BIAS if epi == "bias" else v.EPI_BIAS_GELU)
    if epi == "gelu and preact":
        kw["preact"] = P = laid(torch.empty(R, N, dtype=ot, device="cuda"), r)[0]
    if epi == "gelu backward":
        P, _ = laid((torch.randn(R, N, device="cuda", generator=g) * 2).to(ot), r)
        kw.update(preact=P, epilogue=v.EPI_GELU_BWD)

    def call():
        C.fill_(7.0)
        if epi == "gelu and preact":
            P.fill_(7.0)
        out = v.gemm_grouped(op, A, B, o, C, **kw)
        return (out, P) if epi == "gelu and preact" else (out,)

    def check():
        t, m = torch.zeros(used, N, dtype=F64, device="cuda"), torch.zeros(used, N, dtype=F64, device="cuda")
        for i in range(G):
            if sizes[i]:
                s, w = slice(off[i], off[i + 1]), b[i] if op == v.OP_NN else b[i].t()
                t[s], m[s] = a[s] @ w, a[s].abs() @ w.abs()
                if op == v.OP_NN and epi != "none":
                    t[s] += bias[i].double()
                    m[s] += bias[i].double().abs()
        good = bool((C[used:] == 7.0).all()) and int(torch.isnan(buf).sum()) == buf.numel() - R * N
        if epi.startswith("gelu and") or epi == "gelu":
            good &= close(C[:used], gelu(t), 1.13 * m, K, ot, 16 * U * gelu(t).abs())
            if P is not None:
                good &= close(P[:used], t, m, K, ot) and bool((P[used:] == 7.0).all())
        elif epi == "gelu backward":
            good &= close(C[:used], t * gelu_grad(P[:used].double()), 1.13 * m, K, ot, 20 * U * t.abs())
        else:
            good &= close(C[:used], t, m, K, ot)
        return good

    return text + " " + epi, call, check


def adapters(v, r, g):
    """One call of vedic_gemm_lora or vedic_lora_add."""
    dt = r.choice([F16, F16, F32])
    M, K, N = log(r, 1, 2000), width(r, 1, 1500), width(r, 1, 1500)
    rank, G = r.choice([1, 3, 4, 8, 12, 16, 20, 32, 48, 64, 100, 128]), log(r, 1, 100)
    while G * max(K, N) * rank > 2e7:
        G = max(1, G // 2)
    mk = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=g) * std).to(dt)
    X, W = mk(M, K), mk(K, N, std=K ** -0.5)
    A, B = mk(G, K, rank, std=K ** -0.5), mk(G, rank, N, std=rank ** -0.5)
    ids = torch.randint(-1, G, (M,), device="cuda", generator=g, dtype=torch.int32)
    if r.random() < 0.5:
        ids = ids.sort().values.contiguous()
    off, rows, _ = v.group_rows(ids, G)
    scales = torch.rand(G, device="cuda", generator=g) * 2 if r.random() < 0.7 else None
    base = r.random() < 0.5
    c0 = torch.randn(M, N, device="cuda", generator=g)
    x, w = X.double(), W.double()
    want, mag = (x @ w, x.abs() @ w.abs()) if base else (c0.double(), c0.double().abs())
    for i in range(G):
        at = (ids == i).nonzero()[:, 0]
        if at.numel():
            s = 1.0 if scales is None else scales[i].double()
            want[at] += s * (x[at] @ A[i].double() @ B[i].double())
            mag[at] += s * (x[at].abs() @ A[i].double().abs() @ B[i].double().abs())
        else:
            A[i], B[i] = NAN, NAN
    X, _ = laid(X, r)
    W, _ = laid(W, r)
    C, _ = laid(c0, r)
    if not base:
        X[ids < 0] = NAN

    def call():
        C.copy_(c0)
        if base:
            return (v.gemm_lora(X, W, A, B, off, rows, scales=scales, out=C),)
        return (v.lora_add(C, X, A, B, off, rows, scales),)

    text = f"adapters {dt} M {M} K {K} N {N} rank {rank} G {G} base {base} X {X.stride()} W {W.stride()} C {C.stride()}"
    return text, call, lambda: close(C, want, mag, K + rank, F32)


@pytest.mark.parametrize("block", range(12))
def test_random_calls(block):
    v = vedic()
    for seed in range(30 * block, 30 * block + 30):
        r, g = random.Random(seed), torch.Generator(device="cuda")
        g.manual_seed(seed)
        text, call, check = r.choice([grouped, grouped, adapters])(v, r, g)
        call()
        assert check(), f"seed {seed}: {text}"


@pytest.mark.parametrize("block", range(4))
def test_random_calls_captured(block):
    """Each on a stream of its own: one eager call, a capture, two replays with the eager call between."""
    from logos_amd import _lib

    v = vedic()
    for seed in range(10000 + 15 * block, 10015 + 15 * block):
        r, g = random.Random(seed), torch.Generator(device="cuda")
        g.manual_seed(seed)
        text, call, _ = r.choice([grouped, adapters])(v, r, g)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            eager = [t.clone() for t in call()]
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            recorded = call()
        for _ in range(2):
            for t in recorded:
                t.fill_(NAN)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(recorded, eager)), f"seed {seed}: {text}"
            with torch.cuda.stream(s):
                call()
            s.synchronize()
        del graph
        assert _lib.load().vedic_workspace_release(s.cuda_stream) == _lib.STATUS_OK
