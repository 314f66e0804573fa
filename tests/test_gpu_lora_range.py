"""Adapters whose inner product has columns of very different size: each keeps its fp32 precision."""
import numpy as np
import pytest
import torch

from _gpu_helpers import assert_componentwise

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def vedic():
    from logos_amd import vedic as v

    return v


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("r", [2, 4, 8, 16, 24, 32, 40, 64, 100, 128])
@pytest.mark.parametrize("N,top", [(8, 128), (272, 128), (520, 128), (272, 4096), (104, 2.0 ** 14)])
def test_columns_of_different_size(N, top, r, dt):
    """One column of X A near 10^3 to 10^5, the others near 2^-20, and columns of B that leave the first out: their sums of r
    products are as exact as the others'."""
    v = vedic()
    rng = np.random.default_rng(r + N)
    M, K, G = 37, 64, 3
    X = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).to(dt).cuda()
    a = rng.integers(-8, 9, (G, K, r)) * 2.0 ** -24
    a[:, :, 0] = np.clip(rng.standard_normal((G, K)), -3, 3) * top
    A = torch.from_numpy(a.astype(np.float32)).to(dt).cuda()
    b = rng.standard_normal((G, r, N))
    b[:, 0, : N // 2] = 0.0
    B = torch.from_numpy(b.astype(np.float32)).to(dt).cuda()
    off = torch.tensor([0, 5, 5, M], dtype=torch.int32, device="cuda")
    order = rng.permutation(M)
    rows = torch.from_numpy(order.astype(np.int32)).cuda()
    g = np.empty(M, int)
    g[order] = np.repeat([0, 2], [5, M - 5])
    x, a, b = (t.double().cpu().numpy() for t in (X, A, B))
    h = np.einsum("mk,mkr->mr", x, a[g])
    want = np.einsum("mr,mrn->mn", h, b[g])
    mag = np.einsum("mr,mrn->mn", np.einsum("mk,mkr->mr", np.abs(x), np.abs(a[g])), np.abs(b[g]))
    got = v.lora_add(torch.zeros(M, N, device="cuda"), X, A, B, off, rows).double().cpu().numpy()
    # the sums of K, then r products; one rounding of the scale's product
    assert_componentwise(got, want, mag, K + r, label=f"rank {r}")
    got = v.gemm_lora(X, torch.zeros(K, N, dtype=dt, device="cuda"), A, B, off, rows).double().cpu().numpy()
    assert_componentwise(got, want, mag, K + r, label=f"rank {r}, beside the projection")


@pytest.mark.parametrize("r", [4, 16, 40, 128])
@pytest.mark.parametrize("down", [0, 10, 20, 27, 31, 36, 40, 44, 48])
def test_parts_of_the_inner_product(down, r):
    """One column of X A of 2^25, the others 2^down below: each is held to 2^-24 of itself down to 2^-28 of the row's largest,
    to 2^-22 down to 2^-40, to 2^-51 of the largest below.  (The largest is scaled to 2^14 at least: 2^-14, the smallest
    normal binary16, is 2^-28 of it, and 2^-26, of which 2^12 times is that, 2^-40.)"""
    v = vedic()
    rng = np.random.default_rng(down + r)
    M, K, N = 33, 8, 264
    # X A = x0 A[0] + x1 A[1] + x2 A[2], the first only in column 0, x and A normal binary16 numbers throughout
    x = np.zeros((M, K))
    x[:, 0] = 2.0 ** 10
    half = min(down, 20) // 2
    x[:, 1:3] = rng.uniform(1, 2, (M, 2)) * 2.0 ** (10 - half)
    a = np.zeros((1, K, r))
    a[0, 0, 0] = 2.0 ** 15
    a[0, 1:3, 1:] = rng.uniform(1, 2, (2, r - 1)) * 2.0 ** (14 - (down - half)) * rng.choice([-1, 1], (2, r - 1))
    b = rng.standard_normal((1, r, N))
    b[0, 0] = 0.0
    X, A, B = (torch.from_numpy(t.astype(np.float32)).half().cuda() for t in (x, a, b))
    x, a, b = (t.double().cpu().numpy() for t in (X, A, B))
    h, hmag = x @ a[0], np.abs(x) @ np.abs(a[0])
    top = 2.0 ** 25
    held = np.where(np.abs(h) >= top * 2.0 ** -28, 2.0 ** -24 * np.abs(h),
                    np.where(np.abs(h) >= top * 2.0 ** -40, 2.0 ** -22 * np.abs(h), 2.0 ** -51 * top))
    off = torch.tensor([0, M], dtype=torch.int32, device="cuda")
    rows = torch.arange(M, dtype=torch.int32, device="cuda")
    got = v.lora_add(torch.zeros(M, N, device="cuda"), X, A, B, off, rows).double().cpu().numpy()
    # two products summed in fp32; what the parts hold; r products, each sum and its alignment a unit; the parts' sums
    bound = (2 * 2.0 ** -24 * hmag + held) @ np.abs(b[0]) + (2 * r + 4) * 2.0 ** -24 * (np.abs(h) @ np.abs(b[0]))
    assert np.all(np.abs(got - h @ b[0]) <= bound), (np.abs(got - h @ b[0]) / bound).max()
