"""A whole expert layer, forward and backward, as a training step uses the operators: against 64 bits, recorded into a graph,
and on other streams and threads at once."""
import threading

import numpy as np
import pytest
import torch

from _expert_helpers import choose, gelu, gelu_grad, plan, weights

pytestmark = pytest.mark.gpu

F16 = torch.float16


def vedic():
    from logos_amd import vedic as v

    return v


class Layer:
    """E experts of D -> F -> D with k chosen per token, binary16 operands."""

    def __init__(self, T, E, k, D, F, seed, dtype=F16):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        r = lambda *s, std=1.0, dt=torch.float32: (torch.randn(*s, device="cuda", generator=g) * std).to(dt)
        self.T, self.E, self.k, self.D, self.F, self.dt = T, E, k, D, F, dtype
        self.x = r(T, D, dt=dtype)
        self.res = r(T, D)
        self.Wr = r(D, E, std=D ** -0.5, dt=dtype)
        self.W1, self.W2 = r(E, D, F, std=D ** -0.5, dt=dtype), r(E, F, D, std=F ** -0.5, dt=dtype)
        self.b1, self.b2 = r(E, F, std=0.1), r(E, D, std=0.1)
        self.dout = r(T, D, std=0.1)

    def step(self):
        v = vedic()
        logits = v.gemm(v.OP_NN, self.x, self.Wr)
        rt = v.route_topk(logits, self.k)
        R = self.T * self.k
        P = torch.empty(R, self.F, dtype=self.dt, device="cuda")
        H = v.gemm_grouped(v.OP_NN, self.x, self.W1, rt.offsets, rows=rt.rows, bias=self.b1, epilogue=v.EPI_BIAS_GELU, preact=P,
                           out_dtype=self.dt)
        Y = v.gemm_grouped(v.OP_NN, H, self.W2, rt.offsets, bias=self.b2, epilogue=v.EPI_BIAS)
        out = v.combine_rows(Y, rt.slots, rt.weights, residual=self.res)
        dY, dw = v.combine_rows_bwd(self.dout, Y, rt.slots, rt.weights, out_dtype=self.dt)
        db1, db2 = (torch.empty(self.E, n, device="cuda") for n in (self.F, self.D))
        dW2 = v.gemm_grouped(v.OP_TN, H, dY, rt.offsets, db=db2)
        dH = v.gemm_grouped(v.OP_NT, dY, self.W2, rt.offsets, epilogue=v.EPI_GELU_BWD, preact=P, out_dtype=self.dt)
        dW1 = v.gemm_grouped(v.OP_TN, self.x, dH, rt.offsets, rows=rt.rows, db=db1)
        dXr = v.gemm_grouped(v.OP_NT, dH, self.W1, rt.offsets)
        dlog = v.route_topk_bwd(logits, rt.ids, rt.weights, dw)
        dx = v.combine_rows(dXr, rt.slots, residual=None)
        return dict(logits=logits, ids=rt.ids, weights=rt.weights, offsets=rt.offsets, rows=rt.rows, slots=rt.slots, P=P, H=H,
                    Y=Y, out=out, dY=dY, dw=dw, dW2=dW2, db2=db2, dH=dH, dW1=dW1, db1=db1, dx=dx, dlog=dlog)


def rel(got, want):
    return np.linalg.norm(got.double().cpu().numpy() - want) / max(np.linalg.norm(want), 1e-30)


@pytest.mark.parametrize("T,E,k,D,F,dtype", [(37, 5, 2, 64, 96, F16), (300, 8, 2, 128, 256, F16), (50, 6, 3, 41, 67, F16),
                                             (90, 4, 1, 72, 88, torch.float32), (1, 3, 2, 64, 64, F16)])
def test_layer(T, E, k, D, F, dtype):
    L = Layer(T, E, k, D, F, T + E, dtype)
    o = L.step()
    n = lambda t: t.double().cpu().numpy()
    # the choice and the plan exactly, from the logits as computed
    ids = choose(o["logits"].cpu().numpy(), k)
    off, rows, slots = plan(ids, E, k)
    for name, want in (("ids", ids), ("offsets", off), ("rows", rows), ("slots", slots)):
        np.testing.assert_array_equal(o[name].cpu().numpy(), want)
    w = weights(o["logits"].cpu().numpy(), ids, True)
    x, W1, W2 = n(L.x), n(L.W1), n(L.W2)
    g = np.repeat(np.arange(E), np.diff(off))
    A = x[rows]
    P = np.concatenate([A[off[e]:off[e + 1]] @ W1[e] for e in range(E)]) + n(L.b1)[g]
    H = gelu(P)
    Y = np.concatenate([H[off[e]:off[e + 1]] @ W2[e] for e in range(E)]) + n(L.b2)[g]
    out = n(L.res) + (w[:, :, None] * Y[slots]).sum(1)
    dout = n(L.dout)
    dY = np.empty_like(Y)
    dY[slots.reshape(-1)] = (w[:, :, None] * dout[:, None]).reshape(-1, D)
    dw = (Y[slots] * dout[:, None]).sum(2)
    dH = np.concatenate([dY[off[e]:off[e + 1]] @ W2[e].T for e in range(E)]) * gelu_grad(P)
    dXr = np.concatenate([dH[off[e]:off[e + 1]] @ W1[e].T for e in range(E)])
    seg = [slice(off[e], off[e + 1]) for e in range(E)]
    want = dict(out=out, P=P, H=H, Y=Y, dY=dY, dw=dw, dH=dH, dx=dXr[slots].sum(1),
                dW1=np.stack([A[s].T @ dH[s] for s in seg]), dW2=np.stack([H[s].T @ dY[s] for s in seg]),
                db1=np.stack([dH[s].sum(0) for s in seg]), db2=np.stack([dY[s].sum(0) for s in seg]))
    inner = (w * dw).sum(1, keepdims=True)
    dl = np.zeros((T, E))
    np.put_along_axis(dl, ids.astype(np.int64), w * (dw - inner), 1)
    want["dlog"] = dl
    # Each value passes at most three roundings to the operands' type (P and H; dY; dH), half a unit each and, as they are
    # independent, no more than their number together in the 2-norm; sums of up to 512 products in fp32 add 2^-24 sqrt(512)
    # of their magnitude, for which 32 is more than these data's cancellation gives.
    half = torch.finfo(dtype).eps / 2
    tol = 4 * half + 32 * 23 * 2.0 ** -24
    for name, wv in want.items():
        assert rel(o[name], wv) < tol, (name, rel(o[name], wv), tol)


def test_layer_in_a_graph():
    """Forward and backward recorded once and replayed on new inputs, other work of the program between the replays."""
    v = vedic()
    L = Layer(200, 8, 2, 128, 256, 1)
    odd = Layer(40, 4, 2, 41, 67, 2)     # unaligned: padded copies in the workspace
    M = Layer(70, 3, 1, 64, 64, 3)
    la = dict(X=torch.randn(24, 64, device="cuda").half(), W=torch.randn(64, 80, device="cuda").half(),
              A=torch.randn(3, 64, 8, device="cuda").half(), B=torch.randn(3, 8, 80, device="cuda").half())
    off, rows, _ = v.group_rows(torch.randint(-1, 3, (24,), device="cuda", dtype=torch.int32), 3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    long = torch.randn(64, 2048, device="cuda")
    Wl = torch.randn(2, 2048, 96, device="cuda")
    tall, dt = torch.randn(8192, 64, device="cuda").half(), torch.randn(8192, 128, device="cuda").half()
    ends = {n: torch.tensor([0, n // 3, n], dtype=torch.int32, device="cuda") for n in (64, 8192)}

    def work():
        # (a long contraction shared by several workgroups, fp32 NN and binary16 TN)
        shared = dict(nn=v.gemm_grouped(v.OP_NN, long, Wl, ends[64]), tn=v.gemm_grouped(v.OP_TN, tall, dt, ends[8192]))
        return [L.step(), odd.step(), shared, dict(lora=v.gemm_lora(la["X"], la["W"], la["A"], la["B"], off, rows))]

    with torch.cuda.stream(s):
        work()  # the stream's workspace block
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        recorded = work()
    for i in range(3):
        torch.manual_seed(i)
        for layer in (L, odd):
            layer.x.copy_(torch.randn_like(layer.x))
            layer.dout.copy_(torch.randn_like(layer.dout))
        la["X"].copy_(torch.randn_like(la["X"]))
        long.copy_(torch.randn_like(long))
        tall.copy_(torch.randn_like(tall))
        g.replay()
        torch.cuda.synchronize()
        eager = work()
        M.step()
        torch.cuda.synchronize()
        for a, b in zip(recorded, eager):
            for name in a:
                assert torch.equal(a[name], b[name]), (i, name)
    s.synchronize()
    del g
    from logos_amd import _lib

    assert _lib.load().vedic_workspace_release(s.cuda_stream) == _lib.STATUS_OK


def test_capture_without_a_block_is_refused():
    """A captured call that needs temporaries on a stream without any records nothing and says so."""
    v = vedic()
    X, W = torch.randn(24, 41, device="cuda").half(), torch.randn(41, 80, device="cuda").half()
    A, B = torch.randn(3, 41, 8, device="cuda").half(), torch.randn(3, 8, 80, device="cuda").half()
    off, rows, _ = v.group_rows(torch.zeros(24, dtype=torch.int32, device="cuda"), 3)
    C = torch.full((24, 80), 7.0, device="cuda")
    want = v.gemm_grouped(v.OP_NN, X, W[None], torch.tensor([0, 24], dtype=torch.int32, device="cuda"))
    one = torch.tensor([0, 24], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        with pytest.raises(RuntimeError):
            v.gemm_lora(X, W, A, B, off, rows, out=C)
        D = v.gemm_grouped(v.OP_NN, X, W[None], one)  # needs none: the general kernel
    g.replay()
    torch.cuda.synchronize()
    assert torch.all(C == 7.0)
    torch.testing.assert_close(D, want, rtol=0, atol=41 * 2.0 ** -17)  # 2 K u sum |ab|, the sum below 64


def test_rows_past_two_gibibytes():
    """Row lists into operands whose offsets pass 32 bits, and outputs that do."""
    v = vedic()
    rows = torch.tensor([0, 1_099_999, 7, 600_123, 1_048_577], dtype=torch.int32, device="cuda")
    for dt, T in ((F16, 1_100_000), (torch.float32, 1_100_000)):
        X = torch.empty(T, 1024, dtype=dt, device="cuda")
        x = torch.randn(5, 1024, device="cuda").to(dt)
        X[rows.long()] = x
        W = (torch.randn(2, 1024, 64, device="cuda") / 32).to(dt)
        off = torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
        assert torch.equal(v.gemm_grouped(v.OP_NN, X, W, off, rows=rows), v.gemm_grouped(v.OP_NN, x, W, off))
        dY = torch.randn(5, 64, device="cuda").to(dt)
        assert torch.equal(v.gemm_grouped(v.OP_TN, X, dY, off, rows=rows), v.gemm_grouped(v.OP_TN, x, dY, off))
        A, B = (torch.randn(2, 1024, 8, device="cuda") / 32).to(dt), torch.randn(2, 8, 1024, device="cuda").to(dt)
        C = torch.empty(T, 1024, device="cuda")
        C[rows.long()] = 0.0
        want = torch.zeros(5, 1024, device="cuda")
        v.lora_add(want, x, A, B, off, torch.arange(5, dtype=torch.int32, device="cuda"))
        got = v.lora_add(C, X, A, B, off, rows)
        assert torch.equal(got[rows.long()], want)
        # (slots that far into Y, and dY)
        w = torch.tensor([[0.5, 2.0]], device="cuda")
        slots = torch.tensor([[1_099_999, 600_123]], dtype=torch.int32, device="cuda")
        out = v.combine_rows(X, slots, w)
        torch.testing.assert_close(out[0], 0.5 * x[1].float() + 2.0 * x[3].float(), rtol=2.0 ** -22, atol=2.0 ** -20)
        g = torch.randn(1, 1024, device="cuda")
        dYf, dw = v.combine_rows_bwd(g, X, slots, w, dY=C)
        assert torch.equal(dYf[1_099_999], 0.5 * g[0]) and torch.equal(dYf[600_123], 2.0 * g[0])
        torch.testing.assert_close(dw[0].double(), x[[1, 3]].double() @ g[0].double(), rtol=0, atol=1024 * 2.0 ** -20)
        del X, C, dYf


@pytest.mark.parametrize("shared", [False, True])
def test_streams_and_threads(shared):
    """Four threads on streams of their own, or on one, all operators at once: the bits of the calls made alone."""
    layers = [Layer(60 + 31 * i, 4 + i, 2, 64 + 8 * i, 128, 10 + i) for i in range(4)]
    alone = [layer.step() for layer in layers]
    torch.cuda.synchronize()
    bad = []
    one = torch.cuda.Stream()

    def run(i):
        s = one if shared else torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                o = layers[i].step()
                s.synchronize()
                bad.extend((i, name) for name in o if not torch.equal(o[name], alone[i][name]))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
