"""Low-rank adapters of many requests beside a shared projection, against 64-bit products."""
import numpy as np
import pytest
import torch

from _expert_helpers import plan
from _gpu_helpers import assert_componentwise

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def vedic():
    from logos_amd import vedic as v

    return v


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


CASES = [  # rows, K, N, rank, adapters, how rows choose
    (1, 64, 64, 8, 1, "one"), (1, 1024, 4096, 16, 5, "each"), (7, 100, 33, 3, 4, "each"), (16, 1024, 520, 16, 32, "each"),
    (64, 256, 256, 1, 3, "runs"), (70, 130, 258, 128, 3, "runs"), (300, 512, 384, 64, 7, "runs"), (513, 72, 1000, 24, 100, "each"),
    (600, 264, 136, 40, 2, "one"), (50, 64, 128, 8, 3, "none"),
]


def ids_of(rng, M, G, how):
    if how == "none":
        return np.full(M, -1, np.int32)
    if how == "one":
        return np.full(M, G - 1, np.int32)
    if how == "each":
        return rng.integers(-1, G, M).astype(np.int32)
    return np.repeat(rng.integers(-1, G, M // 13 + 1), 13)[:M].astype(np.int32)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_lora(case, dt):
    v = vedic()
    M, K, N, r, G, how = case
    rng = np.random.default_rng(M + K + N)
    mk = lambda shape, std: torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(dt).cuda()
    X, W, A, B = mk((M, K), 1), mk((K, N), K ** -0.5), mk((G, K, r), K ** -0.5), mk((G, r, N), r ** -0.5)
    b = cuda(rng.standard_normal(N).astype(np.float32))
    sc = (rng.random(G) + 0.5).astype(np.float32)
    ids = ids_of(rng, M, G, how)
    off, rows, _ = v.group_rows(cuda(ids), G)
    x, w, a, bb = (t.double().cpu().numpy() for t in (X, W, A, B))
    base = x @ w + b.double().cpu().numpy()
    want, mag = base.copy(), np.abs(x) @ np.abs(w) + np.abs(b.double().cpu().numpy())
    for i in range(M):
        if ids[i] >= 0:
            want[i] += sc[ids[i]] * (x[i] @ a[ids[i]] @ bb[ids[i]])
            mag[i] += sc[ids[i]] * (np.abs(x[i]) @ np.abs(a[ids[i]]) @ np.abs(bb[ids[i]]))
    got = v.gemm_lora(X, W, A, B, off, rows, bias=b, scales=cuda(sc))
    # the sums of K, then r, then the base's K products: K + r + a few roundings of their magnitudes
    assert_componentwise(got.double().cpu().numpy(), want, mag, K + r, label="gemm_lora")
    # in place, and rows without an adapter untouched
    C0 = torch.randn(M, N, device="cuda")
    C = C0.clone()
    out = v.lora_add(C, X, A, B, off, rows)
    assert out is C
    none = cuda(ids < 0)
    assert torch.equal(C[none], C0[none])
    low = np.zeros((M, N))
    lmag = np.zeros((M, N))
    for i in range(M):
        if ids[i] >= 0:
            low[i] = x[i] @ a[ids[i]] @ bb[ids[i]]
            lmag[i] = np.abs(x[i]) @ np.abs(a[ids[i]]) @ np.abs(bb[ids[i]])
    c0 = C0.double().cpu().numpy()
    assert_componentwise(C.double().cpu().numpy(), c0 + low, lmag, K + r, rounded=np.abs(c0) + np.abs(low), label="lora_add")
    C2 = v.lora_add(C0.clone(), X, A, B, off, rows)
    assert torch.equal(C, C2)


@pytest.mark.parametrize("dt", [F16, F32])
def test_strides_and_bad_rows(dt):
    v = vedic()
    rng = np.random.default_rng(1)
    X = torch.randn(30, 75, device="cuda").to(dt)[:, 3:67]
    A, B = (torch.randn(2, 64, 8, device="cuda") * 0.1).to(dt), (torch.randn(2, 8, 96, device="cuda") * 0.1).to(dt)
    wide = torch.full((30, 101), 7.0, device="cuda")
    C = wide[:, 2:98]
    C.zero_()
    rows = torch.arange(30, dtype=torch.int32, device="cuda").flip(0).contiguous()
    off = cuda(np.array([0, 11, 30], np.int32))
    v.lora_add(C, X, A, B, off, rows)
    want = v.lora_add(torch.zeros(30, 96, device="cuda"), X.contiguous(), A, B, off, rows)
    torch.testing.assert_close(C, want, rtol=0, atol=72 * 2.0 ** -20)
    assert torch.all(wide[:, :2] == 7.0) and torch.all(wide[:, 98:] == 7.0)
    rows[4], rows[20] = -3, 30  # outside: no row
    C3 = torch.zeros(30, 96, device="cuda")
    v.lora_add(C3, X, A, B, cuda(np.array([-2, 11, 99], np.int32)), rows)
    gone = torch.zeros(30, dtype=torch.bool, device="cuda")
    gone[29 - 4] = gone[29 - 20] = True
    assert torch.all(C3[gone] == 0)
    torch.testing.assert_close(C3[~gone], want[~gone], rtol=0, atol=72 * 2.0 ** -20)
