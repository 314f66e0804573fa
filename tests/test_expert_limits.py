"""Sizes that the expert and adapter operators refuse because a launch cannot have them (CPU)."""
import pytest

from logos_amd import _lib
from test_expert_refusals import P, grouped

N22 = (1 << 22) - 1


@pytest.mark.parametrize("kw", [
    # one row in each of 1024 groups, as many columns as a row can have: 1032 x 32768 tiles
    dict(in_dtype=0, groups=1024, rows=1024, K=1, N=N22, lda=1, ldb=N22, ldc=N22, stride_b=0),
    dict(op=1, in_dtype=0, groups=1024, rows=1024, K=1, N=N22, lda=1, ldb=1, ldc=N22, stride_b=0),
    dict(op=2, in_dtype=0, groups=1024, rows=1024, M=1, N=N22, lda=1, ldb=N22, ldc=N22, stride_c=N22),
])
def test_grouped_tiles(kw):
    assert grouped(**kw) == _lib.STATUS_TOO_LARGE


@pytest.mark.parametrize("dtype,N", [(0, N22), (1, N22), (1, N22 - 7)])
def test_adapter_tiles(dtype, N):
    args = (P, dtype, 8, 1024, P, P, 1024, 4, P, P, 1024, None, P, N if N % 8 else N + 4, 8, N, None)
    assert _lib.load().vedic_lora_add(*args) == _lib.STATUS_TOO_LARGE


@pytest.mark.parametrize("R,N", [(1 << 30, 1), ((1 << 31) - 1, 1), (4, 1 << 30)])
def test_bias_gradient_counts(R, N):
    assert _lib.load().vedic_bias_grad_grouped(P, 1, N, R, N, P, 2, 0.0, P, None) == _lib.STATUS_TOO_LARGE
