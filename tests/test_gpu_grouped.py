"""Products grouped by expert against 64-bit products of each group: every op, type and epilogue, ragged and empty groups,
row lists, strides, unaligned operands, and rows that have to stay as they were."""
import numpy as np
import pytest
import torch

from _expert_helpers import gelu, gelu_grad, sizes_to_offsets
from _gpu_helpers import GELU_SLOPE, assert_componentwise
from oracle import oracle as o

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def vedic():
    from logos_amd import vedic as v

    return v


def make(rng, shape, dtype, std=1.0):
    x = torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(dtype)
    return x.cuda(), x.double().numpy()


def pitched(x, pad, shift=0):
    """The same 2-D or 3-D values with `pad` columns behind each row (NaN there) and a base `shift` elements in."""
    r, c = x.shape[-2:]
    lead = x.shape[:-2]
    n = int(np.prod(lead, dtype=int)) * r * (c + pad) + shift
    buf = torch.full((n,), float("nan"), dtype=x.dtype, device=x.device)
    view = buf[shift:].view(*lead, r, c + pad)[..., :c]
    view.copy_(x)
    return view


def ints(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def unit_of(dtype):
    return o.U16 if dtype == F16 else o.U32


SIZES = [
    ([5], 40, 24),                          # one group, a tile's corner
    ([0, 3, 0, 0, 130, 1, 0], 96, 72),      # empty groups first, between and last
    ([257, 64, 300], 264, 320),             # past one and two tiles each way
    ([1] * 70, 64, 64),                     # more groups than a wave has lanes
    ([700, 20], 1024, 136),
    ([33, 12], 1, 8),                       # contractions of one and two
    ([33, 12], 2, 8),
    ([12, 31], 17, 33),                     # nothing aligned
    ([150, 90], 131, 259),
    ([2100, 1, 3000], 40, 56),              # few tiles and long groups: the contraction is shared (TN)
    ([130, 0, 5, 111], 2056, 104),          # and a long one of few rows (NN, NT)
    ([60, 1], 2051, 67),
]
COMBOS = [(F16, F16), (F16, F32), (F32, F32)]


def check_rows(got, want, absdot, K, dtype, label, slope=1.0, terms=None, extra=0.0):
    assert_componentwise(got, want, slope * absdot, K, rounded=terms, unit=unit_of(dtype), extra_rel=extra, label=label)


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("dtypes", COMBOS)
@pytest.mark.parametrize("case", SIZES, ids=str)
def test_nn(case, dtypes, listed):
    v = vedic()
    sizes, K, N = case
    dt, ot = dtypes
    rng = np.random.default_rng(hash((tuple(sizes), K, N, listed)) % 2 ** 32)
    G, R = len(sizes), sum(sizes)
    off = sizes_to_offsets(sizes)
    T = R // 2 + 1 if listed else R
    X, x = make(rng, (T, K), dt)
    W, w = make(rng, (G, K, N), dt, K ** -0.5)
    b, bv = make(rng, (G, N), F32)
    rows = rng.integers(0, T, R).astype(np.int32) if listed else np.arange(R)
    g = np.repeat(np.arange(G), sizes)
    a = x[rows]
    dot = np.einsum("rk,rkn->rn", a, w[g]) if R * K * N < 5e7 else np.concatenate(
        [a[off[i]:off[i + 1]] @ w[i] for i in range(G)])
    absdot = np.concatenate([np.abs(a[off[i]:off[i + 1]]) @ np.abs(w[i]) for i in range(G)])
    kw = dict(rows=ints(rows) if listed else None, out_dtype=ot)
    offs = ints(off)
    plain = v.gemm_grouped(v.OP_NN, X, W, offs, **kw)
    assert plain.dtype == ot
    check_rows(plain.double().cpu().numpy(), dot, absdot, K, ot, "plain")
    biased = v.gemm_grouped(v.OP_NN, X, W, offs, bias=b, epilogue=v.EPI_BIAS, **kw)
    t = dot + bv[g]
    check_rows(biased.double().cpu().numpy(), t, absdot, K, ot, "bias", terms=np.abs(dot) + np.abs(bv[g]))
    P = torch.empty(R, N, dtype=ot, device="cuda")
    H = v.gemm_grouped(v.OP_NN, X, W, offs, bias=b, epilogue=v.EPI_BIAS_GELU, preact=P, **kw)
    check_rows(P.double().cpu().numpy(), t, absdot, K, ot, "preact", terms=np.abs(dot) + np.abs(bv[g]))
    # err(H) <= slope (err of t) + the GELU's own few ulp
    check_rows(H.double().cpu().numpy(), gelu(t), absdot, K, ot, "gelu", slope=GELU_SLOPE,
               terms=GELU_SLOPE * (np.abs(dot) + np.abs(bv[g])) + 4 * np.abs(gelu(t)))
    again = v.gemm_grouped(v.OP_NN, X, W, offs, bias=b, epilogue=v.EPI_BIAS_GELU, **kw)
    assert torch.equal(again, H)  # with and without the pre-activation, and from call to call


@pytest.mark.parametrize("dtypes", COMBOS)
@pytest.mark.parametrize("case", SIZES, ids=str)
def test_nt(case, dtypes):
    v = vedic()
    sizes, K, N = case
    dt, ot = dtypes
    rng = np.random.default_rng(hash((tuple(sizes), K, N, 7)) % 2 ** 32)
    G, R = len(sizes), sum(sizes)
    off = sizes_to_offsets(sizes)
    dY, a = make(rng, (R, K), dt)
    W, w = make(rng, (G, N, K), dt, K ** -0.5)
    P, p = make(rng, (R, N), ot, 2.0)
    dot = np.concatenate([a[off[i]:off[i + 1]] @ w[i].T for i in range(G)])
    absdot = np.concatenate([np.abs(a[off[i]:off[i + 1]]) @ np.abs(w[i]).T for i in range(G)])
    plain = v.gemm_grouped(v.OP_NT, dY, W, ints(off), out_dtype=ot)
    check_rows(plain.double().cpu().numpy(), dot, absdot, K, ot, "plain")
    dH = v.gemm_grouped(v.OP_NT, dY, W, ints(off), epilogue=v.EPI_GELU_BWD, preact=P, out_dtype=ot)
    # the derivative's own error: exp2, rcp and a handful of products, at most 16 u on a value of at most 1.13
    check_rows(dH.double().cpu().numpy(), dot * gelu_grad(p), absdot, K, ot, "gelu backward", slope=GELU_SLOPE,
               terms=np.abs(dot * gelu_grad(p)) + (8 * np.abs(dot) * (o.U32 / unit_of(ot))))


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("case", SIZES, ids=str)
def test_tn(case, dt, listed):
    v = vedic()
    sizes, M, N = case
    rng = np.random.default_rng(hash((tuple(sizes), M, N, 11, listed)) % 2 ** 32)
    G, R = len(sizes), sum(sizes)
    off = sizes_to_offsets(sizes)
    T = R // 2 + 1 if listed else R
    X, x = make(rng, (T, M), dt)
    dY, dy = make(rng, (R, N), dt)
    rows = rng.integers(0, T, R).astype(np.int32) if listed else np.arange(R)
    a = x[rows]
    seg = [slice(off[i], off[i + 1]) for i in range(G)]
    dot = np.stack([a[s].T @ dy[s] for s in seg])
    absdot = np.stack([np.abs(a[s]).T @ np.abs(dy[s]) for s in seg])
    rl = ints(rows) if listed else None
    db = torch.empty(G, N, device="cuda")
    dW = v.gemm_grouped(v.OP_TN, X, dY, ints(off), rows=rl, db=db)
    got = dW.double().cpu().numpy()
    for i in range(G):
        n = max(1, sizes[i])
        check_rows(got[i], dot[i], absdot[i], n, F32, f"group {i} of {n}")
        check_rows(db[i].double().cpu().numpy(), dy[seg[i]].sum(0), np.abs(dy[seg[i]]).sum(0), n, F32, f"db {i}")
    # accumulated onto what is there, as micro-batches are
    C0, c0 = make(rng, (G, M, N), F32)
    db0, b0 = make(rng, (G, N), F32)
    acc = v.gemm_grouped(v.OP_TN, X, dY, ints(off), C0, rows=rl, beta=0.5, db=db0, db_beta=1.0)
    assert acc is C0
    for i in range(G):
        n = max(1, sizes[i])
        check_rows(acc[i].double().cpu().numpy(), dot[i] + 0.5 * c0[i], absdot[i], n, F32, f"beta {i}",
                   terms=np.abs(dot[i]) + np.abs(c0[i]))
        check_rows(db0[i].double().cpu().numpy(), dy[seg[i]].sum(0) + b0[i], np.abs(dy[seg[i]]).sum(0), n, F32, f"db beta {i}",
                   terms=np.abs(dy[seg[i]].sum(0)) + np.abs(b0[i]))
    # alone: another fixed order of the same n terms, which the same bound of n u sum |dY| holds for
    alone = v.bias_grad_grouped(dY, ints(off))
    for i in range(G):
        check_rows(alone[i].double().cpu().numpy(), dy[seg[i]].sum(0), np.abs(dy[seg[i]]).sum(0), max(1, sizes[i]), F32,
                   f"db alone {i}")
    assert torch.equal(alone, v.bias_grad_grouped(dY, ints(off)))
    db2 = torch.empty_like(db)
    assert torch.equal(dW, v.gemm_grouped(v.OP_TN, X, dY, ints(off), rows=rl, db=db2)) and torch.equal(db, db2)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (8, 1)])
def test_strides_and_rows_behind(dt, pad, shift):
    """Pitched operands (NaN between their rows), bases off 16 bytes, and C's rows behind the last group."""
    v = vedic()
    sizes, K, N = [70, 0, 41], 72, 104
    rng = np.random.default_rng(pad + shift)
    off, R, extra = sizes_to_offsets(sizes), sum(sizes), 9
    X, _ = make(rng, (R + extra, K), dt)
    W, _ = make(rng, (3, K, N), dt, K ** -0.5)
    Wt = W.transpose(1, 2).contiguous()
    X[R:] = float("nan")
    for op, B in ((v.OP_NN, W), (v.OP_NT, Wt)):
        want = v.gemm_grouped(op, X[:R].contiguous(), B, ints(off))
        C = pitched(torch.full((R + extra, N), 7.0, device="cuda"), pad, shift)
        got = v.gemm_grouped(op, pitched(X, pad, shift), pitched(B, pad, shift), ints(off), C)
        if dt == F32 or (pad % 8 == 0 and shift == 0):
            assert torch.equal(got[:R], want)  # the same kernel, or one of the same arithmetic
        else:
            torch.testing.assert_close(got[:R], want, rtol=0, atol=72 * 2.0 ** -20)  # 2 K u sum |ab|, the sum below 8
        assert torch.all(got[R:] == 7.0)
        base = C._base[shift:].view(R + extra, N + pad) if C._base is not None else None
        if base is not None:
            assert torch.isnan(base[:, N:]).all()  # between C's rows
    # TN: pitched C, and gradient rows behind the last group that count for none
    dY, _ = make(rng, (R + extra, N), dt)
    dY[R:] = float("nan")
    want = v.gemm_grouped(v.OP_TN, X[:R].contiguous(), dY[:R].contiguous(), ints(off))
    C = pitched(torch.full((3, K, N), 7.0, device="cuda"), pad, shift)
    got = v.gemm_grouped(v.OP_TN, pitched(X, pad, shift), pitched(dY, pad, shift), ints(off), C)
    torch.testing.assert_close(got, want, rtol=0, atol=70 * 2.0 ** -16)  # 2 n u sum |ab|, the sum below 128
    assert torch.all(got[1] == 0)


@pytest.mark.parametrize("dt", [F16, F32])
def test_bad_plan_stays_inside(dt):
    """Offsets out of order or range and rows outside A: clamped, read as zeros, nothing else touched."""
    v = vedic()
    rng = np.random.default_rng(3)
    X, x = make(rng, (50, 64), dt)
    W, w = make(rng, (3, 64, 72), dt, 0.125)
    rows = rng.integers(0, 50, 40).astype(np.int32)
    rows[[3, 17]] = [-1, 50]
    a = np.where(((rows >= 0) & (rows < 50))[:, None], x[np.clip(rows, 0, 49)], 0.0)
    C = torch.full((40, 72), 7.0, device="cuda")
    got = v.gemm_grouped(v.OP_NN, X, W, ints([-5, 20, 10, 900]), C, rows=ints(rows)).double().cpu().numpy()
    # group 0: 0..19; group 1: 20..10, empty; group 2: 10..39, written over group 0's end
    for g, s in ((0, slice(0, 10)), (2, slice(20, 40))):
        check_rows(got[s], a[s] @ w[g], np.abs(a[s]) @ np.abs(w[g]), 64, F32, f"group {g}")
    assert not np.isnan(got).any()
    dW = v.gemm_grouped(v.OP_TN, X, X, ints([60, 10, 2, -1]))
    assert torch.all(dW == 0)


@pytest.mark.parametrize("dt", [F16, F32])
def test_values_that_are_not_finite(dt):
    """An infinity or a NaN of one row reaches that row alone, and another group's weight none."""
    v = vedic()
    rng = np.random.default_rng(5)
    X, _ = make(rng, (96, 64), dt)
    W, _ = make(rng, (2, 64, 64), dt, 0.125)
    clean = v.gemm_grouped(v.OP_NN, X, W, ints([0, 48, 96]))
    X2, W2 = X.clone(), W.clone()
    X2[5, 3] = float("nan")
    X2[70, 9] = float("inf")
    W2[0, 2, 7] = float("nan")
    got = v.gemm_grouped(v.OP_NN, X2, W2, ints([0, 48, 96]))
    assert torch.isnan(got[5]).all() and torch.isnan(got[:48, 7]).all()
    assert not torch.isfinite(got[70]).any()
    keep = torch.ones(96, 64, dtype=torch.bool, device="cuda")
    keep[5] = keep[70] = False
    keep[:48, 7] = False
    torch.testing.assert_close(got[keep], clean[keep], rtol=0, atol=64 * 2.0 ** -19)  # 2 K u sum |ab|, the sum below 16


@pytest.mark.parametrize("out", [F16, F32])
@pytest.mark.parametrize("dt,K", [(F16, 2056), (F16, 2051), (F32, 2050)])
def test_shared_contraction(dt, K, out):
    """A long contraction of few rows: values that are not finite in each part of it, pitched rows, rows behind the last
    group and between C's rows."""
    if out == F16 and dt == F32:
        pytest.skip("float32 operands give float32")
    v = vedic()
    rng = np.random.default_rng(K)
    sizes, N, extra = [40, 0, 24], 72, 5
    off, R = sizes_to_offsets(sizes), 64
    X, x = make(rng, (R + extra, K), dt)
    W, w = make(rng, (3, K, N), dt, K ** -0.5)
    bad = {3: (7, float("inf")), 11: (K // 2, float("nan")), 50: (K - 1, float("-inf"))}
    for r, (k, value) in bad.items():
        X[r, k] = value
    X[R:] = float("nan")
    b, bv = make(rng, (3, N), F32)
    g = np.repeat(np.arange(3), sizes)
    dot = np.einsum("rk,rkn->rn", x[:R], w[g])
    absdot = np.einsum("rk,rkn->rn", np.abs(x[:R]), np.abs(w[g]))
    keep = np.array([r not in bad for r in range(R)])
    for op, B in ((v.OP_NN, W), (v.OP_NT, W.transpose(1, 2).contiguous())):
        kw, t = (dict(bias=b, epilogue=v.EPI_BIAS), bv[g]) if op == v.OP_NN else ({}, np.zeros((R, N)))
        C = pitched(torch.full((R + extra, N), 7.0, device="cuda", dtype=out), 8)
        got = v.gemm_grouped(op, pitched(X, 8), B, ints(off), C, **kw)
        check_rows(got[:R].double().cpu().numpy()[keep], (dot + t)[keep], absdot[keep], K, out, "shared",
                   terms=(np.abs(dot) + np.abs(t))[keep])
        assert not torch.isfinite(got[:R].float()[torch.from_numpy(~keep).cuda()]).any()
        assert torch.all(got[R:] == 7.0)
        assert torch.isnan(C._base.view(R + extra, N + 8)[:, N:]).all()


@pytest.mark.parametrize("op", ["NN", "TN"])
def test_no_rows(op):
    v = vedic()
    off = ints([0, 0, 0])
    if op == "NN":
        C = v.gemm_grouped(v.OP_NN, torch.empty(0, 64, device="cuda"), torch.randn(2, 64, 32, device="cuda"), off)
        assert C.shape == (0, 32)
    else:
        C = torch.ones(2, 64, 32, device="cuda")
        db = torch.ones(2, 32, device="cuda")
        v.gemm_grouped(v.OP_TN, torch.empty(0, 64, device="cuda"), torch.empty(0, 32, device="cuda"), off, C, db=db)
        assert torch.all(C == 0) and torch.all(db == 0)


def test_gelu_backward_at_large_values():
    """gelu' of infinities, of values whose cube overflows, and of a NaN."""
    v = vedic()
    p = [float("inf"), float("-inf"), 3e38, -3e38, 1e13, -1e13, 60.0, -60.0, 0.0, float("nan")]
    P = torch.tensor(p, device="cuda").expand(4, 10).contiguous()
    got = v.gemm_grouped(v.OP_NT, torch.full((4, 1), 2.0, device="cuda"), torch.ones(1, 10, 1, device="cuda"), ints([0, 4]),
                         epilogue=v.EPI_GELU_BWD, preact=P)
    assert got[2].tolist()[:1] == [2.0] and got[1, 2].item() == got[1, 4].item() == got[1, 6].item() == 2.0
    assert torch.all(got[:, [1, 3, 5, 7]].abs() < 1e-30) and torch.all(got[:, 8] == 1.0) and torch.isnan(got[:, 9]).all()


def test_gradient_against_differences():
    """d<H, G>/dX and /dW of the grouped up product against central differences in 64 bits of the same plain form."""
    v = vedic()
    rng = np.random.default_rng(9)
    sizes, K, N = [6, 0, 11], 24, 40
    off = sizes_to_offsets(sizes)
    g = np.repeat(np.arange(3), sizes)
    X, x = make(rng, (17, K), F32)
    W, w = make(rng, (3, K, N), F32, K ** -0.5)
    b, bv = make(rng, (3, N), F32)
    Gm, gv = make(rng, (17, N), F32)

    def loss(x, w):
        return (gelu(np.einsum("rk,rkn->rn", x, w[g]) + bv[g]) * gv).sum()

    P = torch.empty(17, N, device="cuda")
    v.gemm_grouped(v.OP_NN, X, W, ints(off), bias=b, epilogue=v.EPI_BIAS_GELU, preact=P)
    # dP = G * gelu'(P): the backward product of an identity weight
    eye = torch.eye(N, device="cuda").expand(3, N, N).contiguous()
    dP = v.gemm_grouped(v.OP_NT, Gm, eye, ints(off), epilogue=v.EPI_GELU_BWD, preact=P)
    dX = v.gemm_grouped(v.OP_NT, dP, W, ints(off)).cpu().numpy()
    dW = v.gemm_grouped(v.OP_TN, X, dP, ints(off)).cpu().numpy()
    h = 1e-5
    for _ in range(20):
        i, j = rng.integers(17), rng.integers(K)
        d = np.zeros_like(x)
        d[i, j] = h
        # central differences: h^2 of a third derivative of order 10, and rounding 1e-16 |loss| / h
        assert abs((loss(x + d, w) - loss(x - d, w)) / (2 * h) - dX[i, j]) < 1e-4
        e, i, j = rng.choice([0, 2]), rng.integers(K), rng.integers(N)
        d = np.zeros_like(w)
        d[e, i, j] = h
        assert abs((loss(x, w + d) - loss(x, w - d)) / (2 * h) - dW[e, i, j]) < 1e-4
    assert np.all(dW[1] == 0)
