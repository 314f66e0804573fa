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
@pytest.mark.parametrize("N", [8, 272, 520])
def test_columns_of_different_size(N, r, dt):
    """One column of X A near 10^3, the others near 2^-20, and columns of B that leave the first out: their sums of r products
    are as exact as the others'."""
    v = vedic()
    rng = np.random.default_rng(r + N)
    M, K, G = 37, 64, 3
    X = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).to(dt).cuda()
    a = rng.integers(-8, 9, (G, K, r)) * 2.0 ** -24
    a[:, :, 0] = rng.standard_normal((G, K)) * 128
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
