"""Sorted rows back in token order, and the backward, against 64-bit sums."""
import numpy as np
import pytest
import torch

from _expert_helpers import plan

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F16, F32 = torch.float16, torch.float32


def vedic():
    from logos_amd import vedic as v

    return v


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def case(T, k, D, E, seed, drop=True):
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32) if T else np.empty((0, k), np.int32)
    if drop and T > 2:
        ids[1] = -1          # a token without an expert
        ids[2, 0] = E + 3    # a pair without one
    off, rows, slots = plan(ids, E, k)
    return rng, ids, off, rows, slots


SHAPES = [(0, 2, 64), (1, 1, 1), (1, 2, 64), (5, 3, 7), (17, 8, 1000), (40, 9, 257), (300, 2, 1024), (3, 11, 4100)]


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("T,k,D", SHAPES)
def test_combine(T, k, D, dt):
    rng, ids, off, rows, slots = case(T, k, D, 12, T + k + D)
    v = vedic()
    Y = torch.from_numpy(rng.standard_normal((T * k, D)).astype(np.float32)).to(dt).cuda()
    Y[off[-1]:] = float("nan")  # rows of no pair are not read
    w = rng.random((T, k)).astype(np.float32)
    res = rng.standard_normal((T, D)).astype(np.float32)
    y = np.where((slots >= 0)[:, :, None], np.nan_to_num(Y.double().cpu().numpy())[np.maximum(slots, 0)], 0) if T * k else \
        np.zeros((T, k, D))
    for weights in (w, None):
        for residual in (res, None):
            ww = np.ones((T, k)) if weights is None else w.astype(np.float64)
            want = (ww[:, :, None] * y).sum(1) + (0 if residual is None else res)
            mag = (np.abs(ww)[:, :, None] * np.abs(y)).sum(1) + (0 if residual is None else np.abs(res))
            got = v.combine_rows(Y, cuda(slots), None if weights is None else cuda(w),
                                 residual=None if residual is None else cuda(res))
            # k fused multiply-adds and one addition
            assert np.all(np.abs(got.double().cpu().numpy() - want) <= (k + 1) * U * mag)
    inplace = cuda(res)
    out = v.combine_rows(Y, cuda(slots), cuda(w), residual=inplace, out=inplace)
    assert torch.equal(out, v.combine_rows(Y, cuda(slots), cuda(w), residual=cuda(res)))


@pytest.mark.parametrize("dt,ot", [(F32, F16), (F32, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("T,k,D", SHAPES)
def test_combine_backward(T, k, D, dt, ot):
    rng, ids, off, rows, slots = case(T, k, D, 12, T + k + D + 1)
    v = vedic()
    Y = torch.from_numpy(rng.standard_normal((T * k, D)).astype(np.float32)).to(dt).cuda()
    w = rng.random((T, k)).astype(np.float32)
    dout = rng.standard_normal((T, D)).astype(np.float32)
    dY0 = torch.full((T * k, D), 7.0, dtype=ot, device="cuda")
    dY, dw = v.combine_rows_bwd(cuda(dout), Y, cuda(slots), cuda(w), dY=dY0)
    y, g = Y.double().cpu().numpy(), dout.astype(np.float64)
    want = np.full((T * k, D), 7.0)
    wdw, mag = np.zeros((T, k)), np.zeros((T, k))
    for t in range(T):
        for j in range(k):
            s = slots[t, j]
            if s >= 0:
                want[s] = float(w[t, j]) * g[t]
                wdw[t, j] = (g[t] * y[s]).sum()
                mag[t, j] = (np.abs(g[t]) * np.abs(y[s])).sum()
    half = torch.finfo(ot).eps / 2
    tiny = 2.0 ** -25 if ot == F16 else 2.0 ** -150
    # the product rounds to fp32 and then to the type
    assert np.all(np.abs(dY.double().cpu().numpy() - want) <= (half + U) * np.abs(want) + tiny)
    # a lane adds D / 64 terms, then 2 + 6 levels
    assert np.all(np.abs(dw.double().cpu().numpy() - wdw) <= (D / 64 + 10) * U * mag)


@pytest.mark.parametrize("shift", [0, 1])
def test_strides(shift):
    """Pitched Y, residual and output, on and off 16 bytes, and slots outside Y."""
    v = vedic()
    rng, ids, off, rows, slots = case(20, 2, 96, 5, 3)
    base = torch.from_numpy(rng.standard_normal((40, 112)).astype(np.float32)).cuda()
    Y = base[:, shift:shift + 96]
    res = torch.randn(20, 104, device="cuda")[:, shift:shift + 96]
    out = torch.full((20, 104), 7.0, device="cuda")
    w = cuda(rng.random((20, 2)).astype(np.float32))
    s = cuda(slots)
    got = v.combine_rows(Y, s, w, residual=res, out=out[:, shift:shift + 96])
    assert torch.equal(got, v.combine_rows(Y.contiguous(), s, w, residual=res.contiguous()))
    mask = torch.ones(104, dtype=torch.bool)
    mask[shift:shift + 96] = False
    assert torch.all(out[:, mask.cuda()] == 7.0)
    bad = s.clone()
    bad[0] = torch.tensor([40, -7], dtype=torch.int32)
    assert torch.all(v.combine_rows(Y, bad, w)[0] == 0)


def test_gradient_against_differences():
    v = vedic()
    rng, ids, off, rows, slots = case(7, 2, 10, 4, 8)
    Y = rng.standard_normal((14, 10)).astype(np.float32)
    w = rng.random((7, 2)).astype(np.float32)
    dout = rng.standard_normal((7, 10)).astype(np.float32)

    def loss(Y, w):
        y = np.where((slots >= 0)[:, :, None], Y[np.maximum(slots, 0)], 0)
        return ((w[:, :, None] * y).sum(1) * dout).sum()

    dY, dw = v.combine_rows_bwd(cuda(dout), cuda(Y), cuda(slots), cuda(w), dY=torch.zeros(14, 10, device="cuda"))
    dY, dw = dY.cpu().numpy(), dw.cpu().numpy()
    h = 1e-3  # (the loss is linear in each: the differences are exact but for 64-bit rounding)
    Yd, wd = Y.astype(np.float64), w.astype(np.float64)
    for t in range(7):
        for j in range(2):
            d = np.zeros((7, 2))
            d[t, j] = h
            assert abs((loss(Yd, wd + d) - loss(Yd, wd - d)) / (2 * h) - dw[t, j]) < 1e-5
    for i in range(14):
        d = np.zeros((14, 10))
        d[i, i % 10] = h
        assert abs((loss(Yd + d, wd) - loss(Yd - d, wd)) / (2 * h) - dY[i, i % 10]) < 1e-5
