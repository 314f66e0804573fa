"""A layer of a decoder over the paged cache: four-bit projection, append, attention, four-bit projection added to the input;
a prompt, pieces of prompts beside single tokens, and single tokens; eager, recorded, on several streams and threads."""
import threading

import numpy as np
import pytest
import torch

import _cache_helpers as plain
from logos_amd import vedic
from test_gpu_w4 import weight

pytestmark = pytest.mark.gpu


class Layer:
    def __init__(self, seed, four_bit, Hq=4, H=2, dh=64, width=192, sequences=3, ps=16, longest=400):
        self.Hq, self.H, self.dh, self.four = Hq, H, dh, four_bit
        self.w_in, self.v_in = weight(seed, width, (Hq + 2 * H) * dh, 64)
        self.w_out, self.v_out = weight(seed + 1, Hq * dh, width, 32)
        most = -(-longest // ps)
        self.cache = vedic.kv_cache(sequences * most, ps, H, dh, four_bit)
        self.table = torch.randperm(sequences * most, generator=torch.Generator().manual_seed(seed)).to(torch.int32).view(sequences, most).cuda()
        self.rope = torch.from_numpy(plain.rope_table(longest, dh)).cuda()

    def step(self, x, lens, starts=None, keep=None):
        """x float32 [tokens, width] -> x + the layer's, the steps' results in keep."""
        h, g, d = self.Hq, self.H, self.dh
        y = vedic.gemm_w4(x, self.w_in, out_dtype=torch.float16).view(-1, h + 2 * g, d)
        q = vedic.kv_append(y[:, :h], y[:, h:h + g], y[:, h + g:], *self.cache, self.table, lens, starts, self.rope)
        a = vedic.paged_attention(q, *self.cache, self.table, lens, starts)
        out = vedic.gemm_w4(a.view(-1, h * d), self.w_out, epilogue=vedic.EPI_RESIDUAL, out=x.clone())
        if keep is not None:
            keep.append((x, y, q, a, out))
        return out


def product(x, v):
    x = x.double().cpu().numpy().astype(np.float16).astype(np.float64)
    v = v.astype(np.float64)
    return x @ v, (x.shape[1] + 4) * 2.0 ** -24 * (np.abs(x) @ np.abs(v))


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


STEPS = [([100, 1, 37], [100, 1, 37]), ([1, 90, 1], [101, 91, 38]), ([1, 1, 1], [102, 92, 39]), ([3, 0, 120], [105, 92, 159])]


@pytest.mark.parametrize("four_bit", [False, True])
def test_steps(four_bit):
    """Each result against the formulas of the results it is made of (the operators' own tolerances), the keys of all steps."""
    la = Layer(5, four_bit)
    gen = torch.Generator().manual_seed(1)
    keys = [np.zeros((2, 0, la.H, la.dh), np.float16) for _ in range(3)]
    for new, lens in STEPS:
        x = torch.randn(sum(new), 192, generator=gen).cuda()
        starts = np.concatenate([[0], np.cumsum(new)])
        kept = []
        la.step(x, ints(lens), ints(starts), kept)
        _, y, q, a, out = kept[0]
        want, tol = product(x, la.v_in)
        got = y.double().cpu().numpy().reshape(want.shape)
        assert (np.abs(got - want) <= tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25).all()
        yn, rope = y.cpu().numpy(), la.rope.cpu().numpy()
        pos = np.concatenate([np.arange(L - n, L) for n, L in zip(new, lens)]).astype(int)
        assert (plain.rotate(yn[:, :la.Hq], pos, rope, False) == q.cpu().numpy()).all()
        k, v = plain.rotate(yn[:, la.Hq:la.Hq + la.H], pos, rope, False), yn[:, la.Hq + la.H:]
        for b in range(3):
            r = slice(starts[b], starts[b + 1])
            if new[b] == 0:
                continue
            both = plain.values_of(plain.rows_of(np.stack([k[r], v[r]]), four_bit), four_bit)
            keys[b] = np.concatenate([keys[b], both], 1)
            want, _, tol = plain.attention(q[r].cpu().numpy(), *keys[b], pos[r], la.dh ** -0.5)
            assert (np.abs(a[r].double().cpu().numpy() - want) <= tol).all()
        want, tol = product(a.view(len(x), -1), la.v_out)
        old = x.double().cpu().numpy()
        assert (np.abs(out.double().cpu().numpy() - want - old) <= tol + 8 * 2.0 ** -24 * (np.abs(old) + np.abs(want))).all()


@pytest.mark.parametrize("four_bit", [False, True])
def test_recorded(four_bit):
    """One graph of a step of single tokens, replayed while the lengths grow: the eager steps' bits."""
    def start():
        la = Layer(9, four_bit)
        x0 = torch.randn(3, 192, generator=torch.Generator().manual_seed(2)).cuda()
        prompt = torch.randn(60, 192, generator=torch.Generator().manual_seed(3)).cuda()
        la.step(prompt, ints([30, 20, 10]), ints([0, 30, 50, 60]))
        return la, x0, ints([30, 20, 10])

    la, x, lens = start()
    want = []
    for _ in range(6):
        lens += 1
        x = la.step(x, lens)
        want.append(x.clone())
    la, x, lens = start()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first, count = x.clone(), lens.clone()
        lens += 1
        la.step(x, lens)  # (the stream's workspace)
        s.synchronize()
        x.copy_(first)
        lens.copy_(count)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            lens += 1
            x.copy_(la.step(x, lens))
        for w in want:
            graph.replay()
            s.synchronize()
            assert torch.equal(x, w)
            torch.randn(1000, device="cuda").sum().item()
        del graph
    torch.cuda.synchronize()


def test_streams_and_threads():
    """Four threads, a stream and a cache each, one set of weights' values: each the bits of a run by itself."""
    layers = [Layer(20, i % 2 == 1) for i in range(4)]
    torch.cuda.synchronize()

    def run(la, seed):
        gen = torch.Generator().manual_seed(seed)
        return [la.step(torch.randn(sum(new), 192, generator=gen).cuda(), ints(lens), ints([0, *np.cumsum(new)])) for new, lens in STEPS]

    want = [run(la, i) for i, la in enumerate(layers)]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(3):
                    got[i] = run(layers[i], i)
                s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            assert torch.equal(a, b)
