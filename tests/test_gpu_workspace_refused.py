"""A call whose temporaries no GPU has room for fails alone: what follows on its stream, and torch's own launches, run."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_after_a_refused_allocation():
    from logos_amd import _lib, vedic as v

    X, W = torch.randn(70, 41, device="cuda").half(), torch.randn(2, 41, 24, device="cuda").half()
    off = torch.tensor([0, 30, 70], dtype=torch.int32, device="cuda")
    # listed fp32 rows are copied: 2^24 of 8192 values, 512 GiB
    R, M = 1 << 24, 8192
    wide, rows = torch.ones(2, M, device="cuda"), torch.zeros(R, dtype=torch.int32, device="cuda")
    dY, ends = torch.ones(R, 1, device="cuda"), torch.tensor([0, R], dtype=torch.int32, device="cuda")
    want = v.gemm_grouped(v.OP_NN, X, W, off)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        first = v.gemm_grouped(v.OP_NN, X, W, off)
        C = torch.full((1, M, 1), 7.0, device="cuda")
        for _ in range(2):
            with pytest.raises(RuntimeError):
                v.gemm_grouped(v.OP_TN, wide, dY, ends, C, rows=rows)
            y = X + 1  # (no error left for torch's next launch)
            again = v.gemm_grouped(v.OP_NN, X, W, off)
        s.synchronize()
    assert torch.equal(first, want) and torch.equal(again, want)
    assert torch.all(C == 7.0) and torch.equal(y, X + 1)
    # (and the stream's block is still there: a captured call has its padded copies)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        recorded = v.gemm_grouped(v.OP_NN, X, W, off)
    recorded.fill_(float("nan"))
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(recorded, want)
    del g
    assert _lib.load().vedic_workspace_release(s.cuda_stream) == _lib.STATUS_OK
