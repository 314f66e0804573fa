"""More rows, tokens or pairs than one launch has threads for."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
MANY = (1 << 26) + 5  # 64 threads each pass 2^32


def vedic():
    from logos_amd import vedic as v

    return v


def test_combine():
    v = vedic()
    Y = torch.randn(7, 2, device="cuda").half()
    slots = torch.randint(-1, 8, (MANY, 1), device="cuda", dtype=torch.int32)
    slots[-1] = 6
    got = v.combine_rows(Y, slots)
    table = torch.cat([torch.zeros(1, 2, device="cuda"), Y.float(), torch.zeros(1, 2, device="cuda")])
    assert torch.equal(got, table[(slots[:, 0] + 1).long()])


def test_combine_backward():
    v = vedic()
    Y = torch.randn(MANY, 1, device="cuda")
    dout = torch.randn(MANY, 1, device="cuda")
    w = torch.rand(MANY, 1, device="cuda")
    slots = torch.arange(MANY - 1, -1, -1, device="cuda", dtype=torch.int32)[:, None].contiguous()
    dY, dw = v.combine_rows_bwd(dout, Y, slots, w)
    assert torch.equal(dY, (w * dout).flip(0))
    assert torch.equal(dw, dout * Y.flip(0))


def test_route_and_its_backward():
    v = vedic()
    logits = torch.randn(MANY, 2, device="cuda")
    dw = torch.randn(MANY, 1, device="cuda")
    r = v.route_topk(logits, 1, renorm=False)
    second = logits[:, 1] > logits[:, 0]
    assert torch.equal(r.ids[:, 0], second.int())
    assert r.offsets.tolist() == [0, MANY - int(second.sum()), MANY]
    assert torch.equal(r.rows[r.slots[:, 0].long()].long(), torch.arange(MANY, device="cuda"))
    got = v.route_topk_bwd(logits, r.ids, r.weights, dw, renorm=False)
    for part in (slice(0, 1 << 25), slice(1 << 25, 1 << 26), slice(1 << 26, MANY)):
        want = v.route_topk_bwd(logits[part], r.ids[part], r.weights[part], dw[part], renorm=False)
        assert torch.equal(got[part], want)


def test_listed_rows():
    """The copy of a list of 2^24 rows and more, 256 threads each."""
    v = vedic()
    R = (1 << 24) + 9
    X = torch.tensor([[1.0], [2.0], [4.0]], device="cuda")
    rows = torch.randint(0, 3, (R,), device="cuda", dtype=torch.int32)
    rows[-1] = 2
    dY = torch.zeros(R, 1, device="cuda")
    dY[[0, 5, R // 2, R - 3, R - 1]] = torch.tensor([[1.0], [3.0], [16.0], [32.0], [0.5]], device="cuda")
    off = torch.tensor([0, R], dtype=torch.int32, device="cuda")
    got = v.gemm_grouped(v.OP_TN, X, dY, off, rows=rows)
    assert got.item() == (X[rows.long()] * dY).sum().item()


@pytest.mark.parametrize("op", ["NN", "NT"])
def test_few_rows_of_many_columns(op):
    """One row in each of 1024 groups: more tiles of the few-row kernel than a launch has."""
    v = vedic()
    G, K, N = 1024, 8, 1 << 20
    X = torch.randn(G, K, device="cuda").half()
    W = torch.randn(N, K, device="cuda").half()
    off = torch.arange(G + 1, dtype=torch.int32, device="cuda")
    if op == "NN":
        got = v.gemm_grouped(v.OP_NN, X, W.t().contiguous().expand(G, K, N), off, out_dtype=F16)
    else:
        got = v.gemm_grouped(v.OP_NT, X, W.expand(G, N, K), off, out_dtype=F16)
    for g in (0, 1, 500, G - 1):
        want = X[g].double() @ W.double().t()
        mag = X[g].double().abs() @ W.double().abs().t()
        # K products and sums in fp32, one rounding to binary16
        err = (got[g].double() - want).abs()
        assert (err <= (K * 2.0 ** -24) * mag + 2.0 ** -11 * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -25).all()
    assert torch.isfinite(got[:, -1]).all()


@pytest.mark.parametrize("rows,d", [((1 << 24) + 7, 3), (MANY, 4)])
def test_layer_normalisation(rows, d):
    v = vedic()
    X = torch.randn(rows, d, device="cuda")
    gamma, beta = torch.randn(d, device="cuda"), torch.randn(d, device="cuda")
    Y, Y16 = v.layernorm(X, gamma, beta, fp16=True)
    step = 1 << 22
    for at in (0, step, rows // step // 2 * step, rows // step * step):
        y, y16 = v.layernorm(X[at:at + step], gamma, beta, fp16=True)
        assert torch.equal(Y[at:at + step], y) and torch.equal(Y16[at:at + step], y16)
    h = torch.empty(rows, d, dtype=F16, device="cuda")
    h.copy_(X)
    Y16 = v.layernorm_fp16(h, gamma, beta)
    at = rows // step * step
    assert torch.equal(Y16[at:], v.layernorm_fp16(h[at:], gamma, beta))
