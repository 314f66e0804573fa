"""Row lists into operands with more rows than the list (a share of the tokens): the listed rows at every alignment, against
64-bit products of them."""
import numpy as np
import pytest
import torch

from _expert_helpers import gelu, sizes_to_offsets
from _gpu_helpers import GELU_SLOPE
from test_gpu_grouped import F16, F32, check_rows, ints, make, pitched, vedic

pytestmark = pytest.mark.gpu

CASES = [  # group sizes, rows of A, contraction (TN: rows of C), columns, padding behind a row, base off by
    ([3, 0, 2], 12, 41, 67, 0, 0),
    ([3, 0, 2], 12, 64, 72, 0, 0),
    ([3, 0, 2], 12, 64, 72, 3, 0),        # a pitch off 16 bytes
    ([3, 0, 2], 12, 64, 72, 8, 1),        # a base off 16 bytes
    ([1], 5000, 41, 64, 0, 0),
    ([40, 1, 90], 132, 72, 41, 0, 0),     # one row more than the list
    ([300, 17, 260], 4001, 131, 259, 0, 0),
    ([30, 34], 999, 2051, 67, 0, 0),      # a long contraction, shared (NN, NT)
    ([1500, 1700], 9001, 41, 56, 0, 0),   # long groups, shared (TN)
]


def listing(rng, sizes, T, outside):
    """Rows of A, most of them past the list's length, the first and last among them, and some outside A."""
    R = sum(sizes)
    rows = rng.integers(min(R, T - 1), T, R).astype(np.int32)
    rows[0] = T - 1
    if R > 4:
        rows[1] = 0
        rows[[2, 4]] = [-1, T] if outside else rows[[2, 4]]
    return rows


def read(x, rows):
    return np.where(((rows >= 0) & (rows < len(x)))[:, None], x[np.clip(rows, 0, len(x) - 1)], 0.0)


@pytest.mark.parametrize("outside", [False, True])
@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_nn_and_nt(case, dt, outside):
    v = vedic()
    sizes, T, K, N, pad, shift = case
    rng = np.random.default_rng(T + K + N)
    off, R, G = sizes_to_offsets(sizes), sum(sizes), len(sizes)
    X, x = make(rng, (T, K), dt)
    W, w = make(rng, (G, K, N), dt, K ** -0.5)
    b, bv = make(rng, (G, N), F32)
    rows = listing(rng, sizes, T, outside)
    a, g = read(x, rows), np.repeat(np.arange(G), sizes)
    dot = np.concatenate([a[off[i]:off[i + 1]] @ w[i] for i in range(G)])
    absdot = np.concatenate([np.abs(a[off[i]:off[i + 1]]) @ np.abs(w[i]) for i in range(G)])
    X, W, Wt = pitched(X, pad, shift), pitched(W, pad, shift), pitched(W.transpose(1, 2).contiguous(), pad, shift)
    kw = dict(rows=ints(rows))
    nn = v.gemm_grouped(v.OP_NN, X, W, ints(off), **kw)
    check_rows(nn.double().cpu().numpy(), dot, absdot, K, F32, "NN")
    nt = v.gemm_grouped(v.OP_NT, X, Wt, ints(off), **kw)
    check_rows(nt.double().cpu().numpy(), dot, absdot, K, F32, "NT")
    H = v.gemm_grouped(v.OP_NN, X, W, ints(off), bias=b, epilogue=v.EPI_BIAS_GELU, **kw)
    t = dot + bv[g]
    check_rows(H.double().cpu().numpy(), gelu(t), absdot, K, F32, "gelu", slope=GELU_SLOPE,
               terms=GELU_SLOPE * (np.abs(dot) + np.abs(bv[g])) + 4 * np.abs(gelu(t)))


@pytest.mark.parametrize("outside", [False, True])
@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_tn(case, dt, outside):
    v = vedic()
    sizes, T, M, N, pad, shift = case
    rng = np.random.default_rng(T + M + N + 1)
    off, R, G = sizes_to_offsets(sizes), sum(sizes), len(sizes)
    X, x = make(rng, (T, M), dt)
    dY, dy = make(rng, (R, N), dt)
    rows = listing(rng, sizes, T, outside)
    a = read(x, rows)
    db = torch.empty(G, N, device="cuda")
    dW = v.gemm_grouped(v.OP_TN, pitched(X, pad, shift), pitched(dY, pad, shift), ints(off), rows=ints(rows), db=db)
    for i in range(G):
        s, n = slice(off[i], off[i + 1]), max(1, sizes[i])
        check_rows(dW[i].double().cpu().numpy(), a[s].T @ dy[s], np.abs(a[s]).T @ np.abs(dy[s]), n, F32, f"group {i}")
        check_rows(db[i].double().cpu().numpy(), dy[s].sum(0), np.abs(dy[s]).sum(0), n, F32, f"db {i}")


def test_eager_and_captured_rows():
    """A capture on a stream without a workspace block takes the general kernel: the same rows."""
    v = vedic()
    X, W = torch.randn(60, 41, device="cuda").half(), torch.randn(2, 41, 24, device="cuda").half()
    off, rows = ints([0, 3, 9]), ints([59, 8, 30, 31, 9, 0, 58, 57, 12])
    eager = v.gemm_grouped(v.OP_NN, X, W, off, rows=rows)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        recorded = v.gemm_grouped(v.OP_NN, X, W, off, rows=rows)
    for _ in range(2):
        recorded.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        torch.testing.assert_close(recorded, eager, rtol=0, atol=41 * 2.0 ** -17)  # 2 K u sum |ab|, the sum below 64


@pytest.mark.parametrize("K", [41, 48])
@pytest.mark.parametrize("R", [5, 700])
def test_column_slice_past_two_gibibytes(K, R):
    """A few columns of a matrix whose pitch takes its rows past 2 GiB, and a workspace that held NaN before."""
    v = vedic()
    T, N, sizes = 600, 72, [R // 2, R - R // 2]
    rng = np.random.default_rng(K + R)
    off = sizes_to_offsets(sizes)
    wide = torch.empty(T, 1 << 21, dtype=F16, device="cuda")
    X, x = make(rng, (T, K), F16)
    wide[:, 7:7 + K] = X
    W, w = make(rng, (2, K, N), F16, K ** -0.5)
    dY, dy = make(rng, (R, N), F16)
    rows = rng.integers(0, T, R).astype(np.int32)
    rows[0] = T - 1
    a = x[rows]
    spoil = pitched(torch.full((20000, 48), float("nan"), dtype=F16, device="cuda"), 0, 1)
    for _ in range(2):  # (the block grows with the first call and is written by the second)
        v.gemm_grouped(v.OP_NN, spoil, torch.ones(1, 48, 8, dtype=F16, device="cuda"), ints([0, 20000]))
    dot = np.concatenate([a[off[i]:off[i + 1]] @ w[i] for i in range(2)])
    absdot = np.concatenate([np.abs(a[off[i]:off[i + 1]]) @ np.abs(w[i]) for i in range(2)])
    A = wide[:, 7:7 + K]
    nn = v.gemm_grouped(v.OP_NN, A, W, ints(off), rows=ints(rows))
    check_rows(nn.double().cpu().numpy(), dot, absdot, K, F32, "NN")
    nt = v.gemm_grouped(v.OP_NT, A, W.transpose(1, 2).contiguous(), ints(off), rows=ints(rows))
    check_rows(nt.double().cpu().numpy(), dot, absdot, K, F32, "NT")
    dW = v.gemm_grouped(v.OP_TN, A, dY, ints(off), rows=ints(rows))
    for i in range(2):
        s = slice(off[i], off[i + 1])
        check_rows(dW[i].double().cpu().numpy(), a[s].T @ dy[s], np.abs(a[s]).T @ np.abs(dy[s]), sizes[i], F32, f"group {i}")


def test_one_call_before_a_capture():
    """A stream whose block holds a call's first and last piece but not the middle one: after that one call the block fits all
    three, so the captured call shares its contraction as the eager one does."""
    from logos_amd import _lib

    v = vedic()
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    X, W = (torch.randn(*s, device="cuda", generator=g).half() for s in ((64, 2051), (3, 2051, 67)))
    off = ints([0, 40, 40, 64])
    first = pitched(torch.ones(4700, 64, dtype=F16, device="cuda"), 0, 1)  # 601,600 bytes of padded rows
    w1 = torch.ones(1, 64, 64, dtype=F16, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        v.gemm_grouped(v.OP_NN, first, w1, ints([0, 4700]))
        eager = v.gemm_grouped(v.OP_NN, X, W, off)  # copies of 263,168 and 886,032 bytes, slabs of 68,608
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        recorded = v.gemm_grouped(v.OP_NN, X, W, off)
    for _ in range(2):
        recorded.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(recorded, eager)
    del graph
    assert _lib.load().vedic_workspace_release(s.cuda_stream) == _lib.STATUS_OK
