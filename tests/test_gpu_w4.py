"""Four-bit weights: the format bit for bit, and products against 64 bits."""
import numpy as np
import pytest
import torch

import _cache_helpers as plain
from _expert_helpers import gelu
from logos_amd import vedic

pytestmark = pytest.mark.gpu


def weight(seed, K, N, group):
    """A weight and its values [K, N]."""
    rng = np.random.default_rng(seed)
    G, Kp = -(-K // group), -(-K // 32) * 32
    n = rng.integers(0, 16, (N, G * group)).astype(np.uint32)
    n[:, K:] = 9  # behind the end: nobody's
    s = (rng.random((N, G)) * 0.02).astype(np.float16)
    m = (-rng.random((N, G)) * 0.15).astype(np.float16)
    v = plain.values(n.reshape(N, G, group), s, m).reshape(N, -1)[:, :K].T
    codes = plain.words(n)[:, :Kp // 8].astype(np.uint32).view(np.int32)
    return vedic.W4(torch.from_numpy(np.ascontiguousarray(codes)).cuda(), torch.from_numpy(np.stack([s, m], -1)).cuda(), K, group), v


def check(seed, M, K, N, group, epilogue=None, out_dtype=torch.float32, x32=False, ldx=None, align=0):
    w, v = weight(seed, K, N, group)
    rng = np.random.default_rng(seed + 1)
    x = rng.standard_normal((M, K)).astype(np.float32 if x32 else np.float16)
    ld = ldx or K
    flat = torch.full((M * ld + align,), float("nan"), dtype=torch.float32 if x32 else torch.float16, device="cuda")
    X = flat[align:].view(M, ld)[:, :K]
    X.copy_(torch.from_numpy(x))
    b = rng.standard_normal(N).astype(np.float32)
    old = rng.standard_normal((M, N)).astype(np.float32)
    epilogue = vedic.EPI_NONE if epilogue is None else epilogue
    bias = torch.from_numpy(b).cuda() if epilogue in (vedic.EPI_BIAS, vedic.EPI_BIAS_GELU, vedic.EPI_BIAS_RESIDUAL) else None
    resid = epilogue in (vedic.EPI_RESIDUAL, vedic.EPI_BIAS_RESIDUAL)
    wide = torch.full((M, N + 3), 7.0, dtype=out_dtype, device="cuda")
    out = wide[:, :N]
    if resid:
        out.copy_(torch.from_numpy(old))
    got = vedic.gemm_w4(X, w, bias=bias, epilogue=epilogue, out=out).double().cpu().numpy()
    assert (wide[:, N:] == 7).all()
    x64, v64 = x.astype(np.float16).astype(np.float64), v.astype(np.float64)
    y = x64 @ v64
    # K roundings of the partial sums, the bias and the old value one each; GELU's slope is at most 1.13, its own error a few steps
    tol = (K + 4) * 2.0 ** -24 * (np.abs(x64) @ np.abs(v64) + 4 + np.abs(old))
    if bias is not None:
        y = y + b
    if epilogue == vedic.EPI_BIAS_GELU:
        y = gelu(y)
        tol = 1.13 * tol + 2.0 ** -20 * np.abs(y) + 2.0 ** -22
    if resid:
        y = y + old
    if out_dtype == torch.float16:
        tol = tol + 2.0 ** -11 * np.abs(y) + 2.0 ** -25
    err = np.abs(got - y)
    assert bool((err <= tol).all()), (float(err.max()), float(tol.max()))


@pytest.mark.parametrize("M", [1, 2, 5, 16, 17, 32, 33, 63, 64, 65, 128, 200])
@pytest.mark.parametrize("K,N,group", [(64, 16, 32), (1024, 512, 64), (8, 1, 128), (1999, 301, 32), (200, 130, 128), (4096, 96, 128),
                                       (33, 17, 64)])
def test_rows_and_widths(M, K, N, group):
    check(M * 7 + K, M, K, N, group)


@pytest.mark.parametrize("M", [1, 20, 150])
@pytest.mark.parametrize("x32", [False, True])
@pytest.mark.parametrize("epilogue,out", [(vedic.EPI_NONE, torch.float16), (vedic.EPI_BIAS, torch.float32), (vedic.EPI_BIAS, torch.float16),
                                          (vedic.EPI_BIAS_GELU, torch.float32), (vedic.EPI_BIAS_GELU, torch.float16),
                                          (vedic.EPI_RESIDUAL, torch.float32), (vedic.EPI_BIAS_RESIDUAL, torch.float32)])
def test_epilogues(M, x32, epilogue, out):
    check(M, M, 320, 257, 64, epilogue, out, x32)


@pytest.mark.parametrize("M", [3, 40, 100])
@pytest.mark.parametrize("x32", [False, True])
@pytest.mark.parametrize("ldx,align", [(264, 0), (256, 1), (257, 0), (259, 3)])
def test_strides_and_alignment(M, x32, ldx, align):
    check(M, M, 256, 64, 32, x32=x32, ldx=ldx, align=align)


def test_slabs():
    """A weight whose expanded columns take several slabs."""
    check(3, 70, 16384, 2500, 128)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("K,N,group", [(64, 64, 32), (1000, 70, 64), (31, 5, 128), (257, 129, 32)])
def test_quantize_and_unpack(dtype, K, N, group):
    rng = np.random.default_rng(K)
    x = (rng.standard_normal((K, N)) * 0.3).astype(np.float16 if dtype == torch.float16 else np.float32)
    x[:, 0] = 0.25
    x[K // 2, N - 1] = np.nan
    x[1, N - 2] = np.inf
    if dtype == torch.float32:
        x[2, 1] = 1e6  # clamped
    buf = torch.zeros(K, N + 3, dtype=dtype, device="cuda")
    buf[:, :N] = torch.from_numpy(x)
    w = vedic.w4_quantize(buf[:, :N], group)
    h = np.where(np.isfinite(x), np.clip(x, -65504, 65504), x).astype(np.float16).T
    G = -(-K // group)
    full = np.concatenate([h, np.repeat(h[:, -1:], G * group - K, 1)], 1)  # (the last value again changes neither least nor largest)
    n, s, m = plain.quantize(full.reshape(N, G, group))
    v = plain.values(n, s, m).reshape(N, -1)[:, :K].T
    got = vedic.w4_unpack(w).cpu().numpy()
    assert ((got == v) | (np.isnan(got) & np.isnan(v))).all()
    sc = w.scales.cpu().numpy()
    assert ((sc[..., 0] == s) | np.isnan(s)).all() and (np.isnan(sc) == np.isnan(np.stack([s, m], -1))).all()
    out = torch.full((K, N + 1), 3.0, dtype=torch.float16, device="cuda")
    vedic.w4_unpack(w, out[:, :N])
    assert (out[:, N] == 3).all()


def test_captured():
    """With a block from an eager call the same bits as eager; without one, rows 64 at a time."""
    w, v = weight(5, 512, 384, 64)
    for M in (1, 40, 300):
        X = torch.randn(M, 512, device="cuda").half()
        want = vedic.gemm_w4(X, w)
        for warm in (True, False):
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            out = torch.zeros_like(want)
            with torch.cuda.stream(s):
                if warm:
                    vedic.gemm_w4(X, w, out=out)
                s.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    vedic.gemm_w4(X, w, out=out)
            for _ in range(4):
                out.fill_(9)
                g.replay()
                torch.cuda.synchronize()
                if warm:
                    assert torch.equal(out, want)
                assert (out - want).abs().max() <= 1024 * 2.0 ** -24 * 512 * 0.3 * 5
                torch.randn(1000, device="cuda").sum().item()
            with torch.cuda.stream(s):
                del g
                vedic._lib.load().vedic_workspace_release(s.cuda_stream)
            torch.cuda.synchronize()


def test_codes_behind_the_last_value():
    """Codes behind K may be any; with their column's scale they overflow binary16 here, and do not count."""
    for M, N in ((1, 32), (40, 32), (300, 1000)):
        K, rng = 40, np.random.default_rng(M)
        n = rng.integers(0, 10, (N, 64)).astype(np.uint32)
        n[:, K:] = 15
        s, m = np.full((N, 2), 6000, np.float16), np.zeros((N, 2), np.float16)
        v = plain.values(n.reshape(N, 2, 32), s, m).reshape(N, -1)[:, :K].T
        w = vedic.W4(torch.from_numpy(plain.words(n).view(np.int32)).cuda(), torch.from_numpy(np.stack([s, m], -1)).cuda(), K, 32)
        x = rng.standard_normal((M, K)).astype(np.float16)
        got = vedic.gemm_w4(torch.from_numpy(x).cuda(), w).double().cpu().numpy()
        x64, v64 = x.astype(np.float64), v.astype(np.float64)
        assert (np.abs(got - x64 @ v64) <= K * 2.0 ** -24 * (np.abs(x64) @ np.abs(v64))).all()


@pytest.mark.parametrize("M,K,N,group", [(300, 200, 900, 32), (257, 1024, 1300, 64), (700, 40, 700, 128), (700, 1999, 515, 64), (1000, 96, 1000, 32),
                                         (2100, 136, 2100, 128), (2049, 640, 2070, 32), (2100, 2056, 3700, 64), (300, 2100, 900, 64),
                                         (200, 4096, 1500, 128), (385, 64, 1025, 64), (500, 72, 777, 32)])
def test_many_rows(M, K, N, group):
    """Tiles of both heights, whole and ragged in rows, columns, steps and words of K; and weights expanded first."""
    check(M + K, M, K, N, group)


@pytest.mark.parametrize("x32", [False, True])
def test_slabs_of_many_rows(x32):
    """Expanded columns in two slabs, with a bias and the rows' copy beside them."""
    check(3, 130, 16384, 2500, 128, vedic.EPI_BIAS, x32=x32)


@pytest.mark.parametrize("x32", [False, True])
@pytest.mark.parametrize("epilogue,out", [(vedic.EPI_NONE, torch.float16), (vedic.EPI_BIAS, torch.float32), (vedic.EPI_BIAS_GELU, torch.float16),
                                          (vedic.EPI_RESIDUAL, torch.float32), (vedic.EPI_BIAS_RESIDUAL, torch.float32)])
@pytest.mark.parametrize("N", [1301, 1280])
def test_many_rows_epilogues(x32, epilogue, out, N):
    check(1, 333, 320, N, 64, epilogue, out, x32)


@pytest.mark.parametrize("x32", [False, True])
@pytest.mark.parametrize("ldx,align", [(264, 0), (256, 1), (257, 0), (259, 3)])
def test_many_rows_strides(x32, ldx, align):
    check(2, 333, 256, 1000, 32, x32=x32, ldx=ldx, align=align)


def test_whole_rows_of_out():
    """Rows of C that are whole 16-byte pieces, which the tiles store as such; what is behind them stays."""
    w, _ = weight(3, 256, 1024, 64)
    X = torch.randn(400, 256, device="cuda").half()
    wide = vedic.gemm_w4(X, w)
    for dt in (torch.float32, torch.float16):
        out = torch.full((400, 1032), 7.0, dtype=dt, device="cuda")
        vedic.gemm_w4(X, w, out=out[:, :1024])
        assert torch.equal(out[:, :1024], wide.to(dt)) and (out[:, 1024:] == 7).all()


def test_many_rows_captured():
    """fp32 rows, which the tiles take as binary16 from the workspace: with a block the eager bits, without one 64 rows at a time."""
    w, v = weight(6, 256, 700, 64)
    X = torch.randn(700, 256, device="cuda")
    want = vedic.gemm_w4(X, w)
    tol = 260 * 2.0 ** -23 * (X.half().double().abs().cpu() @ torch.from_numpy(np.abs(v.astype(np.float64))))
    for warm in (True, False):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        out = torch.zeros_like(want)
        with torch.cuda.stream(s):
            if warm:
                vedic.gemm_w4(X, w, out=out)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                vedic.gemm_w4(X, w, out=out)
        for _ in range(4):
            out.fill_(9)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) if warm else bool(((out - want).double().cpu().abs() <= tol).all())
            torch.randn(1000, device="cuda").sum().item()
        with torch.cuda.stream(s):
            del g
            vedic._lib.load().vedic_workspace_release(s.cuda_stream)
        torch.cuda.synchronize()


@pytest.mark.parametrize("M,K,N", [(20000, 64, 17), (17000, 33, 5), (4000, 264, 129)])
def test_narrow_weights_of_many_rows(M, K, N):
    check(M + N, M, K, N, 32, vedic.EPI_BIAS)


def test_more_rows_than_one_launch_takes_captured():
    """fp32 rows past 64 * 65535, without a workspace block: whole numbers, exact in any order."""
    M, K, N = 64 * 65535 + 200, 8, 3
    n = torch.randint(0, 16, (N, 32), generator=torch.Generator().manual_seed(1))
    codes = plain.words(n.numpy().astype(np.uint32)).view(np.int32)
    w = vedic.W4(torch.from_numpy(codes).cuda(), torch.tensor([[[1.0, -8.0]]] * N, dtype=torch.float16, device="cuda"), K, 32)
    X = torch.randint(-9, 10, (M, K), device="cuda").float()
    out = torch.full((M, N), 7.0, dtype=torch.float16, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            vedic.gemm_w4(X, w, out=out)
        g.replay()
    torch.cuda.synchronize()
    want = (X.double().cpu() @ (n[:, :K].double().t() - 8)).half()
    assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("x32", [False, True])
@pytest.mark.parametrize("epilogue,out", [(vedic.EPI_NONE, torch.float32), (vedic.EPI_BIAS_GELU, torch.float16), (vedic.EPI_BIAS_RESIDUAL, torch.float32)])
@pytest.mark.parametrize("M,K,N,group", [(2048, 2048, 4096, 128), (2040, 2112, 4100, 64), (2048, 2176, 4224, 32)])
def test_tall_tiles(M, K, N, group, epilogue, out, x32):
    """Tiles of 256 rows: K in whole steps, an even and an odd number of them, whole and ragged rows and columns."""
    check(M + K, M, K, N, group, epilogue, out, x32)


def test_captured_without_a_block_to_fp32():
    """Rows that go 64 at a time in a graph whose stream has no workspace block, against 64 bits."""
    w, v = weight(5, 512, 384, 64)
    v = v.astype(np.float64)
    for M in (1, 40, 300):
        X = torch.randn(M, 512, device="cuda").half()
        x64 = X.double().cpu().numpy()
        want, tol = x64 @ v, 516 * 2.0 ** -24 * (np.abs(x64) @ np.abs(v))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        out = torch.zeros(M, 384, device="cuda")
        with torch.cuda.stream(s):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                vedic.gemm_w4(X, w, out=out)
        for _ in range(3):
            out.fill_(9)
            g.replay()
            torch.cuda.synchronize()
            assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
            torch.randn(1000, device="cuda").sum().item()
        del g
