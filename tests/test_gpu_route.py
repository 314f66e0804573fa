"""The router against its 64-bit plain form: choices and plans exactly, weights and gradients in fp32."""
import numpy as np
import pytest
import torch

from _expert_helpers import choose, plan, weights

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def vedic():
    from logos_amd import vedic as v

    return v


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def check(logits, k, renorm, got):
    ids = choose(logits, k)
    off, rows, slots = plan(ids, logits.shape[1], k)
    np.testing.assert_array_equal(got.ids.cpu().numpy(), ids)
    np.testing.assert_array_equal(got.offsets.cpu().numpy(), off)
    np.testing.assert_array_equal(got.rows.cpu().numpy(), rows)
    np.testing.assert_array_equal(got.slots.cpu().numpy(), slots)
    want = weights(logits, ids, renorm)
    # w = e_j / sum: the difference of two logits is off by u |x_j - max|, the exponential and the division by 2 ulp
    # each, the sum of n positive terms by log2(n) + n / 64 roundings; the exponent's error counts against w itself
    x = np.where(np.isfinite(logits), logits, 0).astype(np.float64)
    spread = np.abs(x).max(1, initial=0) * 2
    n = k if renorm else logits.shape[1]
    tol = (spread[:, None] + 8 + 6 + n / 64 + 2) * U * 2
    err = np.abs(got.weights.double().cpu().numpy() - want)
    ok = np.isfinite(want)
    assert np.all(err[ok] <= (tol * want + 2.0 ** -149)[ok])
    assert np.all(np.isnan(got.weights.cpu().numpy()[~ok]))


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k", [(0, 8, 2), (1, 1, 1), (1, 8, 2), (3, 7, 7), (63, 64, 6), (64, 60, 4), (65, 65, 3),
                                   (200, 128, 8), (1500, 16, 1), (513, 129, 9), (70, 257, 33), (67, 1000, 64), (10, 1024, 5)])
def test_route(T, E, k, renorm):
    rng = np.random.default_rng(T * 1000 + E)
    logits = (rng.standard_normal((T, E)) * 3).astype(np.float32)
    check(logits, k, renorm, vedic().route_topk(cuda(logits), k, renorm))


@pytest.mark.parametrize("T", [9, 300])
def test_ties_masks_and_infinities(T):
    rng = np.random.default_rng(T)
    E, k = 20, 4
    logits = rng.integers(-2, 3, (T, E)).astype(np.float32)  # ties everywhere
    logits[0] = 0.0
    logits[0, ::2] = -0.0                            # equal to +0
    logits[1] = -np.inf                              # nothing left
    logits[2] = -np.inf
    logits[2, [3, 17]] = [1.0, 2.0]                  # fewer than k
    logits[3] = np.finfo(np.float32).min             # the type's lowest value is a value
    logits[4] = np.finfo(np.float32).min
    logits[4, 5] = 1.0
    logits[5, 7] = np.nan
    logits[6, 2] = np.inf
    logits[7, :10] = -np.inf
    logits[8] = np.float32(1e-40) * np.arange(E)     # subnormal
    check(logits, k, True, vedic().route_topk(cuda(logits), k, True))
    with np.errstate(invalid="ignore"):
        check(logits, k, False, vedic().route_topk(cuda(logits), k, False))


def test_strided_logits_and_many_tokens():
    rng = np.random.default_rng(2)
    wide = (rng.standard_normal((3001, 77))).astype(np.float32)
    v = vedic()
    t = cuda(wide)[:, 5:38]
    check(wide[:, 5:38], 5, True, v.route_topk(t, 5))
    # a long batch of one favoured expert: every pair in one group
    logits = np.zeros((70000, 8), np.float32)
    logits[:, 6] = 1
    r = v.route_topk(cuda(logits), 2)
    assert r.offsets.tolist() == [0, 70000, 70000, 70000, 70000, 70000, 70000, 140000, 140000]
    assert torch.equal(r.slots[:, 0], torch.arange(70000, 140000, dtype=torch.int32, device="cuda"))
    assert torch.equal(r.rows, torch.arange(140000, dtype=torch.int32, device="cuda") % 70000)


@pytest.mark.parametrize("n,groups", [(0, 3), (1, 1), (1000, 5), (1024, 1024), (1025, 3), (9000, 300), (300001, 17)])
def test_group_rows(n, groups):
    rng = np.random.default_rng(n)
    ids = rng.integers(-2, groups + 2, n).astype(np.int32)
    off, rows, slots = vedic().group_rows(cuda(ids), groups)
    w = plan(ids, groups, 1)
    np.testing.assert_array_equal(off.cpu().numpy(), w[0])
    np.testing.assert_array_equal(rows.cpu().numpy(), w[1])
    np.testing.assert_array_equal(slots.cpu().numpy(), w[2])


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k", [(0, 4, 1), (1, 8, 2), (130, 60, 4), (33, 300, 9), (50, 5, 5)])
def test_route_backward(T, E, k, renorm):
    rng = np.random.default_rng(E)
    logits = (rng.standard_normal((T, E)) * 2).astype(np.float32)
    if T > 20:
        logits[3] = -np.inf
        logits[4, 2:] = -np.inf
    v = vedic()
    r = v.route_topk(cuda(logits), k, renorm)
    dw = rng.standard_normal((T, k)).astype(np.float32)
    ids, w = choose(logits, k), weights(logits, choose(logits, k), renorm)
    want = np.zeros((T, E))
    x = logits.astype(np.float64)
    for t in range(T):
        sel = [j for j in range(k) if ids[t, j] >= 0]
        inner = sum(w[t, j] * dw[t, j] for j in sel)
        if not renorm and sel:
            e = np.exp(x[t] - x[t, ids[t, 0]])
            want[t] = -e / e.sum() * inner
        for j in sel:
            want[t, ids[t, j]] += w[t, j] * dw[t, j] - (w[t, j] * inner if renorm else 0)
    got = v.route_topk_bwd(cuda(logits), r.ids, r.weights, cuda(dw), renorm)
    # p (g - inner): p as in the forward (spread <= 32, n <= 300 terms), inner k products, one subtraction, one product
    scale = np.abs(dw).max(initial=0) * (1 + k)
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= 64 * U * scale)


@pytest.mark.parametrize("renorm", [True, False])
def test_route_backward_against_differences(renorm):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 9)).astype(np.float32)
    dw = rng.standard_normal((6, 3)).astype(np.float32)
    ids = choose(x, 3)
    v = vedic()
    r = v.route_topk(cuda(x), 3, renorm)
    got = v.route_topk_bwd(cuda(x), r.ids, r.weights, cuda(dw), renorm).cpu().numpy()
    h = 1e-5
    for t in range(6):
        for e in range(9):
            d = np.zeros((6, 9))
            d[t, e] = h
            up, dn = weights(x + d, ids, renorm), weights(x - d, ids, renorm)
            assert abs(((up - dn) * dw).sum() / (2 * h) - got[t, e]) < 1e-5  # fp32 logits' 3e-7 dominate h^2


@pytest.mark.parametrize("T,E,k,pad", [(70001, 32, 2, 4), (200000, 4, 1, 0), (30011, 260, 3, 1), (40000, 64, 8, 0)])
def test_many_tokens(T, E, k, pad):
    """More tokens than one pass of the workgroups; pitched logits.  Distinct integers choose; torch sorts them."""
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    noise = torch.rand(T, E, device="cuda", generator=g)
    logits = torch.full((T, E + pad), 1e9, device="cuda")
    logits[:, :E] = noise.argsort(1).float() / 8  # a permutation of 0 .. E - 1 in each row: no ties
    v = vedic()
    got = v.route_topk(logits[:, :E], k)
    top = logits[:, :E].topk(k, 1)
    assert torch.equal(got.ids.long(), top.indices)
    torch.testing.assert_close(got.weights.double(), top.values.double().softmax(1), rtol=64 * U, atol=0)
    flat = top.indices.reshape(-1)
    order = flat.argsort(stable=True)
    assert torch.equal(got.rows.long(), order // k)
    assert torch.equal(got.offsets[1:].long(), torch.bincount(flat, minlength=E).cumsum(0)) and got.offsets[0] == 0
    assert torch.equal(got.slots.reshape(-1)[order].long(), torch.arange(T * k, device="cuda"))


def test_smallest_calls_of_the_set():
    """No tokens at all, and tokens of which none has an expert or an adapter."""
    v = vedic()
    rt = v.route_topk(torch.empty(0, 4, device="cuda"), 2)
    assert rt.offsets.tolist() == [0] * 5
    Y = v.gemm_grouped(v.OP_NN, torch.empty(0, 8, device="cuda"), torch.ones(4, 8, 16, device="cuda"), rt.offsets, rows=rt.rows)
    assert Y.shape == (0, 16) and v.combine_rows(Y, rt.slots, rt.weights).shape == (0, 16)
    dY, dw = v.combine_rows_bwd(torch.empty(0, 16, device="cuda"), Y, rt.slots, rt.weights)
    assert dY.shape == (0, 16) and dw.shape == (0, 2)
    rt = v.route_topk(torch.full((3, 4), -float("inf"), device="cuda"), 2)
    assert rt.ids.eq(-1).all() and rt.slots.eq(-1).all() and rt.weights.eq(0).all() and rt.offsets.eq(0).all()
    C = torch.full((6, 16), 7.0, device="cuda")
    X = torch.ones(3, 8, device="cuda")
    v.gemm_grouped(v.OP_NN, X, torch.ones(4, 8, 16, device="cuda"), rt.offsets, C, rows=rt.rows)
    assert C.eq(7.0).all()
    res = torch.randn(3, 16, device="cuda")
    assert torch.equal(v.combine_rows(C, rt.slots, rt.weights, residual=res), res)
    off, rows, _ = v.group_rows(torch.full((3,), -1, dtype=torch.int32, device="cuda"), 2)
    W = torch.randn(8, 16, device="cuda")
    got = v.gemm_lora(X, W, torch.ones(2, 8, 4, device="cuda"), torch.ones(2, 4, 16, device="cuda"), off, rows)
    assert torch.equal(got, v.gemm(v.OP_NN, X, W))
