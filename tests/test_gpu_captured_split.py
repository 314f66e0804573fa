"""Products whose contraction is shared among workgroups, captured after one call on their stream: the eager call's bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("M,N,K", [(90, 52, 2240), (441, 8, 1432), (74, 176, 1344), (64, 64, 4096), (300, 40, 9000), (128, 128, 5064)])
def test_captured_product(M, N, K, dt):
    """Contractions that do not divide into as many slices as the CUs would take (2240: 16 slices asked for, 14 of 160)."""
    from logos_amd import _lib, vedic as v

    g = torch.Generator(device="cuda")
    g.manual_seed(K)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)
    X, W, A, B, Xt = r(M, K), r(K, N), r(3, K, 8), r(3, 8, N), r(K, M)
    off, rows, _ = v.group_rows(torch.randint(-1, 3, (M,), device="cuda", dtype=torch.int32), 3)
    sums = torch.zeros(N, device="cuda")

    def work():
        return [v.gemm(v.OP_NN, X, W), v.gemm(v.OP_TN, Xt, W), v.gemm_lora(X, W, A, B, off, rows),
                v.gemm(v.OP_NN, X, W, colsum=sums, colsum_beta=0.0), sums.clone()]

    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        eager = work()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        recorded = work()
    for _ in range(2):
        for t in recorded:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(recorded, eager)):
            assert torch.equal(a, b), i
    del graph
    assert _lib.load().vedic_workspace_release(s.cuda_stream) == _lib.STATUS_OK
