"""Attention over a paged cache against 64 bits: formats, head layouts, lengths, pages, masks, strides, what masks hide."""
import numpy as np
import pytest
import torch

import _cache_helpers as plain
from logos_amd import vedic

pytestmark = pytest.mark.gpu


class Batch:
    """Sequences with new[b] new rows and lens[b] tokens in a cache with its pages in a random order."""

    def __init__(self, seed, Hq, H, D, four_bit, ps, new, lens, before=0, after=0, spare=2, token_major=False):
        rng = np.random.default_rng(seed)
        self.Hq, self.H, self.D, self.new, self.lens, self.four = Hq, H, D, new, lens, four_bit
        most = [-(-n // ps) for n in lens]
        pages = sum(most) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(lens), max(1, max(most)) + 1), -7, np.int32)
        at = 0
        for b, m in enumerate(most):
            self.table[b, :m] = order[at:at + m]
            at += m
        self.x = [rng.standard_normal((pages, H, ps, D)).astype(np.float16) for _ in range(2)]
        self.T = before + sum(new) + after
        self.q = rng.standard_normal((self.T, Hq, D)).astype(np.float16)
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) + before
        self.rows = [plain.rows_of(x, four_bit) for x in self.x]
        self.ps, self.token_major = ps, token_major

    def device(self):
        caches = []
        for r in self.rows:
            t = torch.from_numpy(np.ascontiguousarray(r.transpose(0, 2, 1, 3) if self.token_major else r)).cuda()
            caches.append(t.transpose(1, 2) if self.token_major else t)
        return (torch.from_numpy(self.q).cuda(), *caches, torch.from_numpy(self.table).cuda(),
                torch.tensor(self.lens, dtype=torch.int32, device="cuda"), torch.from_numpy(self.starts).cuda())

    def sequence(self, b):
        """k and v [L, H, D] of sequence b, as the cache's rows stand for them."""
        L, ps = self.lens[b], self.ps
        pages = self.table[b, :-(-L // ps)] if L else np.zeros(0, int)
        return [plain.values_of(r[pages].swapaxes(1, 2).reshape(-1, self.H, r.shape[-1])[:L], self.four) for r in self.rows]

    def check(self, got, lse=None, scale=None, causal=True, window=0, stride=0, skip=()):
        got = got.float().cpu().numpy()
        scale = self.D ** -0.5 if scale is None else scale
        for b in range(len(self.lens)):
            r0, r1 = self.starts[b], self.starts[b + 1]
            pos = np.arange(self.lens[b] - self.new[b], self.lens[b])
            k, v = self.sequence(b)
            out, want_lse, tol = plain.attention(self.q[r0:r1], k, v, pos, scale, causal, window, stride)
            for i in range(r1 - r0):
                if (b, i) in skip:
                    continue
                err = np.abs(got[r0 + i] - out[i])
                assert bool((err <= tol[i]).all()), (b, i, float(err.max()), float(tol[i].max()))
                if lse is not None:
                    g = lse[r0 + i].cpu().numpy()
                    fin = np.isfinite(want_lse[i])
                    assert (np.isinf(g) & (g > 0) == ~fin).all()
                    # the scores' fp32 sums (|q||k| of a few tens, D roundings) and the logarithm's
                    assert np.abs(g[fin] - want_lse[i][fin]).max(initial=0) <= 2.0 ** -24 * (self.D + 32) * 64


def run(b, one_each=False, **kw):
    q, k, v, table, lens, starts = b.device()
    return vedic.paged_attention(q, k, v, table, lens, q_start=None if one_each else starts, **kw)


@pytest.mark.parametrize("four_bit,D", [(False, d) for d in (8, 40, 64, 72, 96, 128, 160, 192, 200, 256)] +
                         [(True, d) for d in (32, 64, 96, 128, 160, 192, 224, 256)])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 150, 70]])
def test_head_sizes(four_bit, D, new):
    b = Batch(D + four_bit, 6, 2, D, four_bit, 24, new, [n + p for n, p in zip(new, (40, 77, 0))])
    b.check(run(b))


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("Hq,H", [(1, 1), (3, 3), (6, 2), (16, 1), (20, 1), (34, 2), (72, 1), (130, 1)])
def test_shared_heads_one_token(four_bit, Hq, H):
    lens = [1, 31, 64, 129, 200]
    b = Batch(Hq, Hq, H, 64, four_bit, 16, [1] * 5, lens)
    b.check(run(b, one_each=True))


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("ps", [1, 7, 16, 33, 64, 100, 256, 1000])
def test_pages(four_bit, ps):
    b = Batch(ps, 4, 2, 64, four_bit, ps, [1, 2, 90, 1], [1, 63, 130, 257])
    b.check(run(b))
    b = Batch(ps, 4, 2, 64, four_bit, ps, [1, 2, 90, 1], [1, 63, 130, 257], token_major=True)
    b.check(run(b))


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("lens", [[5000], [9, 4097, 2, 1500, 800], [1] * 70 + [3000] + [2] * 70])
def test_long_and_ragged_decoding(four_bit, lens):
    """Long sequences are shared out over workgroups, more than one wave of sequences."""
    b = Batch(len(lens), 4, 1, 64, four_bit, 64, [1] * len(lens), lens)
    lse = torch.full((b.T, 4), -5.0, device="cuda")
    b.check(run(b, one_each=True, lse=lse), lse)


@pytest.mark.parametrize("new,lens", [
    ([300], [300]), ([200, 1, 129, 64], [200, 900, 2000, 64]), ([70, 65, 0, 5], [4000, 70, 33, 5]), ([33], [3001])])
@pytest.mark.parametrize("four_bit", [False, True])
def test_prompts_and_pieces(new, lens, four_bit):
    b = Batch(sum(new), 4, 2, 64, four_bit, 48, new, lens)
    lse = torch.full((b.T, 4), -5.0, device="cuda")
    b.check(run(b, lse=lse), lse)


@pytest.mark.parametrize("window,stride", [(1, 0), (30, 0), (64, 7), (100, 16), (5, 1), (1 << 30, 0), (50, 100000)])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 140, 33]])
def test_masks(window, stride, new):
    b = Batch(window % 1000 + stride % 1000, 4, 2, 64, False, 32, new, [n + p for n, p in zip(new, (0, 300, 77))])
    lse = torch.full((b.T, 4), -5.0, device="cuda")
    b.check(run(b, window=window, stride=stride, lse=lse), lse, window=window, stride=stride)


@pytest.mark.parametrize("new", [[2, 9, 1], [80, 140, 0]])
def test_not_causal(new):
    b = Batch(11, 4, 2, 64, False, 32, new, [n + p for n, p in zip(new, (0, 300, 77))])
    b.check(run(b, causal=False, scale=0.2), causal=False, scale=0.2)


@pytest.mark.parametrize("n", [3, 100])
def test_rows_without_keys_and_rows_of_no_sequence(n):
    """Rows before the first position see nothing (zeros, lse +inf); rows outside the sequences are left as they are."""
    b = Batch(n, 4, 2, 64, False, 16, [n, 0, n, n], [n - 2, 9, 0, n + 20], before=3, after=5)
    q, k, v, table, lens, starts = b.device()
    out = torch.full((b.T, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    lse = torch.full((b.T, 4), 7.0, device="cuda")
    vedic.paged_attention(q, k, v, table, lens, q_start=starts, out=out, lse=lse)
    b.check(out, lse)
    for t in (out, lse):
        assert (t[:3] == 7).all() and (t[-5:] == 7).all()
    assert (out[3:5] == 0).all() and torch.isinf(lse[3:5]).all()
    assert (out[3 + n:3 + 2 * n] == 0).all()


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("new,past", [([1, 1], 90), ([9, 3], 40), ([100, 150], 30), ([90, 140], 700)])
def test_what_is_hidden_does_not_count(four_bit, bad, new, past):
    """NaN and infinities in unused rows of pages, in keys behind a row's own position, and in keys a window leaves out."""
    lens = [past + n for n in new]
    b = Batch(past, 4, 2, 64, four_bit, 32, new, lens)
    filled = [np.full_like(x, bad) for x in b.x]
    for s in range(2):
        for p in range(lens[s]):
            page, at = b.table[s, p // 32], p % 32
            for f, x in zip(filled, b.x):
                f[page, :, at] = x[page, :, at]
    # sequence 0's last key and value, which only its last row sees; sequence 1's first, which no window reaches
    for f in filled:
        f[b.table[0, (lens[0] - 1) // 32], :, (lens[0] - 1) % 32, 5] = bad
        f[b.table[1, 0], :, 0, 5] = bad
    b.rows = [plain.rows_of(f, four_bit) for f in filled]
    got = run(b, window=past - 3)
    with np.errstate(invalid="ignore"):
        b.check(got, window=past - 3, skip={(0, new[0] - 1)})
    assert not torch.isfinite(got[new[0] - 1]).all()


def test_large_scores():
    """Weights far apart: the largest score's key has all but 2^-20 of the weight, a long tail the rest."""
    b = Batch(5, 2, 1, 64, False, 64, [1, 70], [3000, 3000])
    b.q *= np.float16(6)
    b.check(run(b, scale=1.0), scale=1.0)


def test_a_tail_of_small_weights_counts():
    """One key 20 above 16383 others that are alike: they have 16383 e^-20 / (1 + ..) = 3.4e-5 of it, each weight below binary16's
    smallest normal; their value is 2^14 times the first's, so that a third of the sum is theirs."""
    L, D = 16384, 64
    k, v = np.zeros((L, 1, D), np.float16), np.full((L, 1, D), 16384.0, np.float16)
    k[0, 0, 0] = 20.0
    v[0] = 1.0
    q = np.zeros((1, 1, D), np.float16)
    q[0, 0, 0] = 1.0
    table = torch.arange(L // 64, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([L], dtype=torch.int32, device="cuda")
    kc, vc = (torch.from_numpy(np.ascontiguousarray(x.reshape(L // 64, 64, 1, D).transpose(0, 2, 1, 3))).cuda() for x in (k, v))
    got = vedic.paged_attention(torch.from_numpy(q).cuda(), kc, vc, table, lens, scale=1.0).float().cpu().numpy()
    out, _, tol = plain.attention(q, k, v, [L - 1], 1.0)
    assert (np.abs(got - out) <= tol + 2.0 ** -11 * np.abs(out)).all(), (got[0, 0, 0], out[0, 0, 0])


def test_strided_q_and_out():
    """q a view of a packed projection, out a view of a wider buffer."""
    b = Batch(3, 4, 2, 64, False, 16, [1, 80, 3], [50, 80, 40])
    q, k, v, table, lens, starts = b.device()
    packed = torch.randn(b.T, 8, 64, device="cuda").half()
    packed[:, 2:6] = q
    wide = torch.full((b.T, 6, 72), 3.0, dtype=torch.float16, device="cuda")
    vedic.paged_attention(packed[:, 2:6], k, v, table, lens, q_start=starts, out=wide[:, 1:5, :64])
    b.check(wide[:, 1:5, :64])
    assert (wide[:, 0] == 3).all() and (wide[:, 5] == 3).all() and (wide[:, :, 64:] == 3).all()
    # heads before tokens
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    b.check(vedic.paged_attention(qt, k, v, table, lens, q_start=starts))


@pytest.mark.parametrize("new", [1, 100])
def test_cache_past_four_gib(new):
    """Pages whose offsets pass 32 bits."""
    pages, H, ps, D = 5200, 4, 1024, 128  # 5.2 GiB each
    free = torch.cuda.mem_get_info()[0]
    if free < 16 << 30:
        pytest.skip("needs 16 GiB")
    b = Batch(9, 8, H, D, False, ps, [new], [new + 1500], spare=0)
    k, v = (torch.empty(pages, H, ps, D, dtype=torch.float16, device="cuda") for _ in range(2))
    at = torch.tensor([pages - 1, 4200, 5000][:b.rows[0].shape[0]], device="cuda")
    for c, r in zip((k, v), b.rows):
        c[at] = torch.from_numpy(r).cuda()
    q, _, _, table, lens, starts = b.device()
    n = b.rows[0].shape[0]
    table[0, :n] = at[table[0, :n].long()].int()
    b.check(vedic.paged_attention(q, k, v, table, lens, q_start=starts))


def test_bad_lists_stay_in_range():
    """Lengths past the table, pages that are none, starts that do not ascend: values are wrong, accesses are not."""
    b = Batch(4, 4, 2, 64, False, 16, [4, 90, 2], [40, 120, 33])
    q, k, v, table, lens, starts = b.device()
    wild = torch.tensor([[1 << 30, -5, 2], [3, 1 << 20, -1], [0, 0, 0]], dtype=torch.int32, device="cuda")
    for ln in ([1 << 31 - 1, 500, -4], [0, 48, 7]):
        for st in ([0, 90, 20, 96], [-5, 10, 1 << 30, 3], [96, 0, 96, 0]):
            got = vedic.paged_attention(q, k, v, wild, torch.tensor(ln, dtype=torch.int64).clamp(-2 ** 31, 2 ** 31 - 1).int().cuda(),
                                        q_start=torch.tensor(st, dtype=torch.int32, device="cuda"))
            torch.cuda.synchronize()
            assert got.shape == (96, 4, 64)


def test_empty_calls():
    b = Batch(4, 4, 2, 64, False, 16, [4], [40])
    q, k, v, table, lens, starts = b.device()
    assert vedic.paged_attention(q[:0], k, v, table[:0], lens[:0]).shape == (0, 4, 64)
    out = torch.full_like(q, 2.0)
    vedic.paged_attention(q, k, v, table[:0], lens[:0], q_start=starts[:1], out=out)
    assert (out == 2).all()


@pytest.mark.parametrize("new,lens", [([1] * 6, [3000, 5, 700, 1, 64, 2000]), ([1, 300, 2, 90], [2500, 300, 50, 4000])])
def test_captured(new, lens):
    """Recorded into a graph: with a block from an eager call the same bits on every replay, also with other lengths in the
    same tensors; and without a block (a stream the library has not seen), unsplit."""
    b = Batch(21, 8, 2, 64, True, 32, new, lens)
    q, k, v, table, ln, starts = b.device()
    kw = dict(q_start=None if set(new) == {1} else starts)
    for warm in (True, False):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        out = torch.zeros_like(q)
        with torch.cuda.stream(s):
            if warm:
                vedic.paged_attention(q, k, v, table, ln, out=out, **kw)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                vedic.paged_attention(q, k, v, table, ln, out=out, **kw)
        torch.cuda.synchronize()
        want = vedic.paged_attention(q, k, v, table, ln, **kw)
        for _ in range(4):
            out.fill_(9)
            g.replay()
            torch.cuda.synchronize()
            if warm:
                assert torch.equal(out, want)
            b.check(out)
            torch.randn(1000, device="cuda").sum().item()
        if warm:
            short = torch.tensor([max(n, L - 37) for n, L in zip(new, lens)], dtype=torch.int32, device="cuda")
            keep = ln.clone()
            ln.copy_(short)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, vedic.paged_attention(q, k, v, table, short, **kw))
            ln.copy_(keep)
        with torch.cuda.stream(s):
            del g
            vedic._lib.load().vedic_workspace_release(s.cuda_stream)
        torch.cuda.synchronize()


def test_repeated_calls_give_the_same_bits():
    b = Batch(2, 8, 2, 128, False, 64, [1, 1, 100], [6000, 2000, 4000])
    args = b.device()
    first = vedic.paged_attention(*args[:5], q_start=args[5])
    for _ in range(5):
        assert torch.equal(first, vedic.paged_attention(*args[:5], q_start=args[5]))


def test_many_sequences_of_which_two_are_split():
    """More rows that might have parts than workgroups to give each one: a wave joins a row."""
    b = Batch(33, 4, 2, 64, False, 16, [1] * 300, [5000, 1200] + [3] * 298)
    b.check(run(b))


@pytest.mark.parametrize("new", [1, 20, 500])
@pytest.mark.parametrize("where,bad", [(0, np.nan), (0, np.inf), (1, np.nan), (1, -np.inf)])
def test_infinities_and_nan_that_are_seen(new, where, bad):
    """A key or value of position 350: what the formula gives for the rows that see it (few and many rows, split and not), and
    for the others what it gives without."""
    b = Batch(31, 4, 2, 64, False, 16, [new, 1], [700, 3000])
    page, row = b.table[0, 350 // 16], 350 % 16
    b.rows[where][page, 1, row, 5] = bad
    lse = torch.empty(b.T, 4, device="cuda")
    got = run(b, lse=lse).double().cpu().numpy()
    for s in range(2):
        r = slice(b.starts[s], b.starts[s + 1])
        k, v = b.sequence(s)
        with np.errstate(invalid="ignore"):
            want, want_lse, tol = plain.attention(b.q[r], k, v, np.arange(b.lens[s] - b.new[s], b.lens[s]), 64 ** -0.5)
        fin = np.isfinite(want)
        assert (np.isnan(got[r]) == np.isnan(want)).all() and (got[r][np.isinf(want)] == want[np.isinf(want)]).all()
        assert (np.abs(got[r][fin] - want[fin]) <= tol[fin]).all()
        assert (np.isnan(lse[r].cpu().numpy()) == np.isnan(want_lse)).all()


@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.004, 1.5])
@pytest.mark.parametrize("new", [2, 200])
def test_scales(scale, new):
    b = Batch(41, 4, 2, 64, False, 16, [new], [600])
    lse = torch.empty(b.T, 4, device="cuda")
    b.check(run(b, scale=scale, lse=lse), lse, scale=scale)


@pytest.mark.parametrize("new", [[1, 1], [300, 3]])
def test_sequences_that_share_pages(new):
    """Two sequences with one beginning: the same pages in both rows of the table."""
    b = Batch(43, 4, 2, 64, True, 32, new, [800, 640])
    b.table[1, :15] = b.table[0, :15]
    b.check(run(b))


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("one_each", [True, False])
@pytest.mark.parametrize("sequences", [1, 2, 5])
@pytest.mark.parametrize("group", [63, 64, 65, 128])
def test_query_heads_around_the_few_rows(group, sequences, one_each, four_bit):
    """As many query heads a key head as the kernel of few rows takes of one token, one fewer and more."""
    b = Batch(group, group, 1, 64, four_bit, 16, [1] * sequences, [200, 1, 129, 64, 31][:sequences])
    out = torch.full((b.T, group, 64), float("nan"), dtype=torch.float16, device="cuda")
    lse = torch.full((b.T, group), float("nan"), device="cuda")
    run(b, one_each=one_each, out=out, lse=lse)
    b.check(out, lse)


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("D", [224, 256])
def test_single_tokens_of_wide_heads_beside_a_long_piece(four_bit, D):
    """They are the few-row kernel's: the bits of a call without the piece (no key is shared out in either, so that the order of
    the sums is the same)."""
    b = Batch(47, 8, 2, D, four_bit, 32, [1] * 9 + [700], [128, 1, 90, 31, 64, 127, 5, 100, 77, 900])
    q, k, v, table, lens, starts = b.device()
    got = vedic.paged_attention(q, k, v, table, lens, q_start=starts)
    b.check(got)
    assert torch.equal(got[:9], vedic.paged_attention(q[:9], k, v, table[:9, :4], lens[:9]))


@pytest.mark.parametrize("four_bit,D", [(False, 64), (True, 128), (False, 160)])
def test_single_tokens_beside_a_long_piece(four_bit, D):
    b = Batch(48, 8, 2, D, four_bit, 32, [1] * 9 + [700], [128, 1, 90, 31, 64, 1270, 5, 100, 77, 900])
    b.check(run(b))


@pytest.mark.parametrize("new", [1, 20, 500])
@pytest.mark.parametrize("four_bit,D,bad", [(False, d, s * np.inf) for d in (8, 40, 64, 96, 104, 160, 200, 224, 256) for s in (1, -1)] +
                         [(True, d, np.inf) for d in (32, 64, 96, 160, 224)])
def test_infinities_at_the_end_of_a_row(four_bit, D, bad, new):
    """A seen key with an infinity among its last eight values (in four bits: a group whose last code stands for more than binary16's
    largest): weight 0 where the score is -infinity, for heads that fill the kernels' widths and for narrower ones."""
    b = Batch(53 + D, 4, 2, D, four_bit, 16, [new, 1], [700, 3000])
    page, row = b.table[0, 350 // 16], 350 % 16
    x = b.x[0][page, 1, row].copy()
    x[D - 3] = bad
    if four_bit:
        x[D - 32:] = -65504
        x[D - 3] = 65504
    b.rows[0][page, 1, row] = plain.rows_of(x, four_bit)
    assert np.isinf(plain.values_of(b.rows[0][page, 1, row], four_bit)).nonzero()[0].tolist() == [D - 3]
    lse = torch.empty(b.T, 4, device="cuda")
    got = run(b, lse=lse).double().cpu().numpy()
    for s in range(2):
        r = slice(b.starts[s], b.starts[s + 1])
        k, v = b.sequence(s)
        at = (b.q[r], k, v, np.arange(b.lens[s] - b.new[s], b.lens[s]), D ** -0.5)
        with np.errstate(invalid="ignore"):
            want, want_lse, _ = plain.attention(*at)
        k0 = k.copy()
        k0[~np.isfinite(k).all(-1)] = 0  # (that key's score has no error: the tolerance is the other keys')
        tol = plain.attention(at[0], k0, *at[2:])[2]
        fin = np.isfinite(want)
        assert (np.isnan(got[r]) == np.isnan(want)).all() and (np.isnan(lse[r].cpu().numpy()) == np.isnan(want_lse)).all()
        assert (np.abs(got[r][fin] - want[fin]) <= tol[fin]).all()


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("size", [100.0, 4000.0, 60000.0])
@pytest.mark.parametrize("new,lens", [([1, 1], [1, 300]), ([1, 3], [5000, 3]), ([200, 90], [200, 2000])])
def test_scores_far_from_zero(new, lens, size, four_bit):
    """Finite scores of up to 2^38, whose fp32 step is far above 1: a row is the value of its largest score (all of some rows' are
    below zero), wherever the next one is further away than the rounding of the sums."""
    b = Batch(59, 4, 2, 64, four_bit, 32, new, lens)
    rng = np.random.default_rng(7)
    b.x[0][:] = (0.5 + 0.5 * rng.random(b.x[0].shape)) * size
    b.rows = [plain.rows_of(x, four_bit) for x in b.x]
    b.q[:] = (0.5 + 0.5 * rng.random(b.q.shape)) * size * np.where(rng.random((b.T, 4, 1)) < 0.5, -1, 1)
    lse = torch.empty(b.T, 4, device="cuda")
    got = run(b, lse=lse).double().cpu().numpy()
    lse, clear = lse.double().cpu().numpy(), 0
    for s in range(2):
        k, v = (x.astype(np.float64) for x in b.sequence(s))
        for i in range(new[s]):
            r, p = b.starts[s] + i, lens[s] - new[s] + i
            for h in range(4):
                x = k[:p + 1, h // 2] @ b.q[r, h].astype(np.float64) / 8
                top = x.argmax()
                step = 67 * 2.0 ** -24 * np.abs(x[top])  # (64 products' sum, the scale and log2(e), each half a step)
                assert abs(lse[r, h] - x[top]) <= step + 10
                if (np.delete(x, top) < x[top] - 2 * step - 30).all():
                    clear += 1
                    want = v[top, h // 2]
                    assert (np.abs(got[r, h] - want) <= 2.0 ** -10 * np.abs(want) + 2.0 ** -11).all(), (s, i, h)
    assert clear > b.T


@pytest.mark.parametrize("new", [1, 30, 300])
def test_rows_whose_scores_are_all_minus_infinity(new):
    """Undefined by the formula (nothing over nothing), unlike a row that sees no key; the rows beside them are not touched."""
    b = Batch(61, 4, 2, 64, False, 16, [new, 2], [new + 3, 1])
    for p in range(4):
        b.rows[0][b.table[0, p // 16], :, p % 16, 7] = -np.inf
    b.q[:, :, 7] = np.abs(b.q[:, :, 7]) + np.float16(0.5)
    b.q[0, 1, 7] = -1.0
    lse = torch.empty(b.T, 4, device="cuda")
    got = run(b, lse=lse, window=2).float().cpu().numpy()
    lse = lse.cpu().numpy()
    for i in range(new + 2):
        for h in range(4):
            if i == 0:  # position 3 sees 1 .. 3 only, of -infinity, or +infinity for the head whose value is below zero
                assert np.isnan(got[0, h]).all() and np.isnan(lse[0, h])
            elif i == new:  # before the first position of a sequence with one token
                assert (got[i, h] == 0).all() and lse[i, h] == np.inf
            else:
                assert np.isfinite(got[i, h]).all() and np.isfinite(lse[i, h])


@pytest.mark.parametrize("D", [8, 40, 64, 128, 160, 256])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [700, 3, 6000]), ([3, 9, 16], [40, 9, 3000])])
def test_weights_of_few_rows_over_binary16(D, new, lens):
    """In two binary16 parts, 2^-22 of a weight instead of 2^-11: the output's own rounding and the scores' are what is left."""
    b = Batch(67 + D, 4, 2, D, False, 32, new, lens)
    got = run(b).double().cpu().numpy()
    for s in range(3):
        r = slice(b.starts[s], b.starts[s + 1])
        k, v = b.sequence(s)
        at = (np.arange(lens[s] - new[s], lens[s]), D ** -0.5)
        out, _, tol = plain.attention(b.q[r], k, v, *at)
        size = plain.attention(b.q[r], k, np.abs(v), *at)[0]  # the weights' sum of |v|
        assert (np.abs(got[r] - out) <= tol - (2.0 ** -11 - 2.0 ** -22) * size).all()


def many_sequences(seed, count, long, four_bit=False, one_each=True):
    """Short sequences and, at the places of `long`, (new rows, tokens) of others."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(int(four_bit), 12, count).tolist()
    new = [1] * count if one_each else [min(n, int(rng.integers(0, 3))) for n in lens]
    for at, (n, L) in long.items():
        lens[at], new[at] = L, 1 if one_each else n
    return Batch(seed, 4, 2, 64, four_bit, 16, new, lens)


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("one_each", [True, False])
@pytest.mark.parametrize("count,long", [(65, {64: (300, 900)}), (200, {0: (1, 1200), 128: (70, 3000)}), (4161, {4160: (90, 700), 63: (5, 2000)}),
                                        (9000, {4100: (200, 1500)})])
def test_many_sequences(count, long, one_each, four_bit):
    """More than a wave's lanes, and more blocks of 64 than that; first and last ones long, parts among them."""
    b = many_sequences(count, count, long, four_bit, one_each)
    lse = torch.full((b.T, 4), -5.0, device="cuda")
    out = run(b, one_each=one_each, lse=lse)
    b.check(out, lse)
    assert torch.equal(out, run(b, one_each=one_each))


def test_many_sequences_captured():
    """Recorded with a block and without, replayed after the lengths have changed in place."""
    b = many_sequences(3, 300, {7: (1, 2000), 299: (1, 900)})
    q, k, v, table, ln, _ = b.device()
    keep, other = ln.clone(), ln.clone()
    other[7], other[0], other[299] = 20, 3, 0
    want = [vedic.paged_attention(q, k, v, table, x) for x in (keep, other)]
    for warm in (True, False):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        out = torch.zeros_like(q)
        with torch.cuda.stream(s):
            if warm:
                vedic.paged_attention(q, k, v, table, ln, out=out)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                vedic.paged_attention(q, k, v, table, ln, out=out)
        torch.cuda.synchronize()
        for i in (0, 1, 0, 1):
            ln.copy_((keep, other)[i])
            out.fill_(9)
            g.replay()
            torch.cuda.synchronize()
            if warm:
                assert torch.equal(out, want[i])
            assert (out - want[i]).abs().max() <= 2.0 ** -9 * 4
            torch.randn(1000, device="cuda").sum().item()
        ln.copy_(keep)
        with torch.cuda.stream(s):
            del g
            vedic._lib.load().vedic_workspace_release(s.cuda_stream)
        torch.cuda.synchronize()


def test_bad_lists_of_many_sequences_stay_in_range():
    b = many_sequences(5, 300, {5: (60, 500)}, one_each=False)
    q, k, v, table, ln, starts = b.device()
    table[::3, 0] = 1 << 30
    for st in (starts.flip(0).contiguous(), starts * 0 + b.T, torch.randint(-5, b.T + 9, (301,), dtype=torch.int32, device="cuda")):
        for lens in (ln, ln * 0 + 2 ** 31 - 1, -ln):
            vedic.paged_attention(q, k, v, table, lens, q_start=st)
            torch.cuda.synchronize()


def test_more_sequences_than_a_captured_call_walks():
    """Refused without a workspace block, where every workgroup would walk all of them; the capture goes on."""
    n = 16385
    k_cache, v_cache = vedic.kv_cache(1, 1, 1, 8)
    q, table = torch.zeros(n, 1, 8, dtype=torch.float16, device="cuda"), torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    lens, out = torch.ones(n, dtype=torch.int32, device="cuda"), torch.ones_like(q)
    v_cache.fill_(3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            with pytest.raises(RuntimeError):
                vedic.paged_attention(q, k_cache, v_cache, table, lens, out=out)
            vedic.paged_attention(q[:100], k_cache, v_cache, table[:100], lens[:100], out=out[:100])
        g.replay()
    torch.cuda.synchronize()
    assert (out[:100] == 3).all() and (out[100:] == 1).all()
    assert (vedic.paged_attention(q, k_cache, v_cache, table, lens) == 3).all()


@pytest.mark.parametrize("four_bit", [False, True])
def test_scores_of_some_thousands(four_bit):
    """Rows whose scores rise from key to key, all near -2^12 or 2^12 times the scale's unit, so that every block brings a new largest
    one: weights of different blocks against each other, at the scores' own rounding."""
    b = Batch(71, 4, 2, 64, four_bit, 32, [200, 90], [900, 3000])
    for x in b.x:
        x[:] = 0
    for s in range(2):
        for t in range(b.lens[s]):
            page, at = b.table[s, t // 32], t % 32
            b.x[0][page, :, at, :2] = 64 * t / b.lens[s], 64.0
            b.x[1][page, :, at] = np.float16(np.random.default_rng(t).standard_normal(64))
    b.rows = [plain.rows_of(x, four_bit) for x in b.x]
    b.q[:] = 0
    b.q[:, :, 0], b.q[:, ::2, 1], b.q[:, 1::2, 1] = 0.125, 48.0, -48.0
    got = run(b, scale=1.0).double().cpu().numpy()
    for s in range(2):
        r = slice(b.starts[s], b.starts[s + 1])
        k, v = b.sequence(s)
        at = (np.arange(b.lens[s] - b.new[s], b.lens[s]), 1.0)
        out = plain.attention(b.q[r], k, v, *at)[0]
        size = plain.attention(b.q[r], k, np.abs(v), *at)[0]
        # (two products of a score that are not 0, both exact, and a sum below 2^12: 2^-13 off, above and below the division; the
        # weights' half step, 2^-11; c times the differences, exponentials and sums, 2^-13)
        assert (np.abs(got[r] - out) <= 2.0 ** -11 * np.abs(out) + (2.0 ** -11 + 2.0 ** -12 + 2.0 ** -13) * size + 2.0 ** -25).all()


@pytest.mark.parametrize("four_bit,D,ps", [(True, 64, 16), (True, 128, 48), (True, 160, 7), (True, 256, 33), (False, 40, 5), (False, 128, 100),
                                           (False, 160, 7), (False, 256, 32)])
@pytest.mark.parametrize("window,stride", [(40, 0), (33, 100), (64, 16), (200, 3), (7, 1)])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 140, 33]])
def test_masks_of_other_shapes(four_bit, D, ps, window, stride, new):
    """Lists of 0 to some hundred far keys, that end within a block of 32 or 64, over pages of any size and both formats."""
    b = Batch(window + stride + D, 4, 2, D, four_bit, ps, new, [n + p for n, p in zip(new, (1, 1700, 380))])
    lse = torch.full((b.T, 4), -5.0, device="cuda")
    b.check(run(b, window=window, stride=stride, lse=lse), lse, window=window, stride=stride)


@pytest.mark.parametrize("four_bit", [False, True])
def test_the_largest_lengths_and_rows_stay_in_range(four_bit):
    """INT_MAX and INT_MIN in the lists, far keys of a window among them."""
    b = Batch(4, 4, 2, 64, four_bit, 16, [4, 90, 2], [40, 120, 33])
    q, k, v, table, _, _ = b.device()
    top, low = 2 ** 31 - 1, -2 ** 31
    wild = torch.tensor([[top, low, 2], [3, low, -1], [0, top, 0]], dtype=torch.int32, device="cuda")
    for ln in ([top, 500, low], [top, top, top]):
        for st in ([0, 90, 20, 96], [low, 10, top, 3], [0, 4, 94, top]):
            for mask in (dict(), dict(window=20, stride=3), dict(causal=False)):
                got = vedic.paged_attention(q, k, v, wild, torch.tensor(ln, dtype=torch.int32, device="cuda"),
                                            q_start=torch.tensor(st, dtype=torch.int32, device="cuda"), **mask)
                torch.cuda.synchronize()
                assert got.shape == (96, 4, 64)
