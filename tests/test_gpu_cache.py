"""New tokens into a paged cache and rows back from it, bit for bit against the formats' definitions."""
import numpy as np
import pytest
import torch

import _cache_helpers as plain
from logos_amd import vedic

pytestmark = pytest.mark.gpu


def bits(t):
    return t.view(torch.int16) if t.dtype == torch.float16 else t


def same(got, want):
    """Equal, NaN where NaN."""
    g = got.cpu().numpy()
    if g.dtype == np.float16:
        return (np.isnan(g) == np.isnan(want)).all() and (g[~np.isnan(g)] == want[~np.isnan(g)]).all()
    return (g == want).all()


def batch(seed, new, lens, ps, spare=2):
    rng = np.random.default_rng(seed)
    most = [-(-n // ps) for n in lens]
    order = rng.permutation(sum(most) + spare)
    table = np.full((len(lens), max(1, max(most))), -3, np.int32)
    at = 0
    for b, m in enumerate(most):
        table[b, :m] = order[at:at + m]
        at += m
    return rng, table, np.concatenate([[0], np.cumsum(new)]).astype(np.int32), len(order)


def append_and_check(seed, Hq, H, D, four_bit, ps, new, lens, rot, inter, dtype, x=None, one_each=False, make=None):
    rng, table, starts, pages = batch(seed, new, lens, ps)
    T = int(starts[-1])
    x = rng.standard_normal((T, Hq + 2 * H, D)) * 3 if x is None else x
    x = x.astype(np.float16 if dtype == torch.float16 else np.float32)
    rope = plain.rope_table(max(max(lens), 1), rot) if rot else None
    k_cache, v_cache = vedic.kv_cache(pages, ps, H, D, four_bit) if make is None else make(pages)
    for c in (k_cache, v_cache):
        bits(c).fill_(77)
    t = torch.from_numpy(x).cuda()
    q, k, v = t[:, :Hq], t[:, Hq:Hq + H], t[:, Hq + H:]
    tb, ln, st = torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.from_numpy(starts).cuda()
    kw = dict(q_start=None if one_each else st)
    out = torch.full((T, Hq, D), 5.0, dtype=torch.float16, device="cuda")
    got = vedic.kv_append(q if Hq else None, k, v, k_cache, v_cache, tb, ln, rope=None if rope is None else torch.from_numpy(rope).cuda(),
                          interleaved=inter, out=out if Hq else None, **kw)
    pos = np.concatenate([np.arange(L - n, L) for n, L in zip(new, lens)]).astype(int)
    seq = np.repeat(np.arange(len(new)), new)
    there = pos >= 0
    want_q = plain.rotate(x[:, :Hq], np.maximum(pos, 0), rope, inter)
    want_q[~there] = 5.0
    if Hq:
        assert same(got, want_q)
    kk = plain.rotate(x[:, Hq:Hq + H], np.maximum(pos, 0), rope, inter)
    with np.errstate(over="ignore"):
        vv = x[:, Hq + H:].astype(np.float16)
    for c, y in ((k_cache, kk), (v_cache, vv)):
        want = np.zeros(tuple(c.shape), np.uint8 if four_bit else np.float16)
        (want if four_bit else want.view(np.int16))[:] = 77
        rows = plain.rows_of(y, four_bit)
        for r in np.nonzero(there)[0]:
            want[table[seq[r], pos[r] // ps], :, pos[r] % ps] = rows[r]
        if four_bit:  # (a NaN pair's codes are nobody's business)
            g = plain.values_of(c.cpu().numpy(), True)
            w = plain.values_of(want, True)
            assert ((g == w) | (np.isnan(g) & np.isnan(w))).all()
            if np.isfinite(x).all():
                assert same(c, want)
        else:
            assert same(c, want)
    kr, vr = vedic.kv_read(k_cache, v_cache, tb, ln, tokens=T, **kw)
    for g, y in ((kr, kk), (vr, vv)):
        w = plain.values_of(plain.rows_of(y, four_bit), four_bit)
        assert same(g[torch.from_numpy(there).cuda()], w[there])


@pytest.mark.parametrize("four_bit,D", [(False, 8), (False, 40), (False, 64), (False, 96), (False, 128), (False, 256),
                                        (True, 32), (True, 64), (True, 96), (True, 128), (True, 256)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
def test_head_sizes(four_bit, D, dtype, inter):
    for rot in (0, 2, D // 8 * 4, D):
        append_and_check(D, 6, 2, D, four_bit, 16, [3, 1, 20], [3, 40, 33], rot, inter, dtype)


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("ps", [1, 5, 16, 100])
def test_pages_and_counts(four_bit, ps):
    append_and_check(1, 4, 4, 64, four_bit, ps, [0, 7, 0, 64, 1], [4, 7, 0, 1000, 1], 64, False, torch.float16)
    append_and_check(2, 0, 3, 64, four_bit, ps, [1] * 200, list(range(1, 201)), 32, True, torch.float32, one_each=True)
    append_and_check(3, 2, 1, 64, four_bit, ps, [9, 5], [6, 0], 64, False, torch.float16)  # rows before the first position


def test_a_prompt():
    append_and_check(4, 16, 16, 64, False, 64, [4000, 1, 333], [4000, 900, 1333], 64, False, torch.float32)
    append_and_check(5, 8, 2, 128, True, 48, [1, 4000], [77, 5000], 128, True, torch.float16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_values_at_the_formats_edges(dtype):
    """Equal values, zeros, subnormals, the largest, infinities and NaN in one group of 32 and not in its neighbours."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((8, 3, 64))
    x[0], x[1] = 0, 1.5
    x[2] *= 1e-6
    x[3, :, :32] = np.where(rng.random((3, 32)) < 0.5, 65504, -65504)
    x[4, :, 3], x[5, :, 40], x[6, :, 63] = np.nan, np.inf, -np.inf
    x[7, :, 0] = 1e5 if dtype == torch.float32 else 3
    for four_bit in (False, True):
        append_and_check(0, 1, 1, 64, four_bit, 4, [8], [8], 0, False, dtype, x=x)


def test_other_layouts():
    """Rows of a token's heads side by side, pages of k and v in one tensor; fp32 rows that are not 16-byte aligned."""
    for four_bit in (False, True):
        row = 40 if four_bit else 64

        def make(pages):
            dt = torch.uint8 if four_bit else torch.float16
            both = torch.empty(pages, 2, 16, 3, row, dtype=dt, device="cuda")
            return both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
        append_and_check(7, 3, 3, 64, four_bit, 16, [5, 1, 50], [20, 7, 90], 64, False, torch.float16, make=make)
    x = torch.randn(40 * 6 * 64 + 1, device="cuda")[1:].view(40, 6, 64)
    k_cache, v_cache = vedic.kv_cache(8, 16, 2, 64)
    table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    lens, starts = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([40], [0, 40]))
    rope = torch.from_numpy(plain.rope_table(40, 64)).cuda()
    args = (k_cache, v_cache, table, lens, starts, rope)
    got = vedic.kv_append(x[:, :2], x[:, 2:4], x[:, 4:], *args)
    want = plain.rotate(x.cpu().numpy(), np.arange(40), rope.cpu().numpy(), False)
    assert same(got, want[:, :2])
    assert same(vedic.kv_read(k_cache, v_cache, table, lens, starts, 40)[0], want[:, 2:4])
    # rows shared by the heads (a stride of 0)
    one = x[:, :1].expand(40, 2, 64)
    vedic.kv_append(None, one, one, *args)
    assert same(vedic.kv_read(k_cache, v_cache, table, lens, starts, 40)[0], np.repeat(want[:, :1], 2, 1))


def test_bad_lists_stay_in_range():
    q = torch.randn(12, 4, 64, device="cuda").half()
    for four_bit in (False, True):
        k_cache, v_cache = vedic.kv_cache(4, 16, 4, 64, four_bit)
        wild = torch.tensor([[1 << 30, -5], [3, 1 << 20]], dtype=torch.int32, device="cuda")
        rope = torch.ones(3, 64, device="cuda")
        for ln in ([2 ** 31 - 1, 20], [-9, 40]):
            for st in ([0, 30, 4], [-4, 5, 2 ** 31 - 1], [12, 0, 12]):
                args = (torch.tensor(ln, dtype=torch.int32, device="cuda"), torch.tensor(st, dtype=torch.int32, device="cuda"))
                vedic.kv_append(q, q, q, k_cache, v_cache, wild, *args, rope=rope)
                vedic.kv_read(k_cache, v_cache, wild, *args, tokens=12)
                torch.cuda.synchronize()


def test_pages_past_four_gib():
    pages, H, ps, D = 5200, 4, 1024, 128
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GiB")
    k, v = (torch.empty(pages, H, ps, D, dtype=torch.float16, device="cuda") for _ in range(2))
    x = torch.randn(1500, H, D, device="cuda").half()
    table = torch.tensor([[4100, pages - 1]], dtype=torch.int32, device="cuda")
    lens, starts = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([1500], [0, 1500]))
    vedic.kv_append(None, x, x, k, v, table, lens, starts)
    assert torch.equal(k[4100], x[:1024].transpose(0, 1)) and torch.equal(v[pages - 1, :, :476], x[1024:].transpose(0, 1))
    a, b = vedic.kv_read(k, v, table, lens, starts, 1500)
    assert torch.equal(a, x) and torch.equal(b, x)


@pytest.mark.parametrize("four_bit", [False, True])
def test_a_padded_batch(four_bit):
    """Rows before the first sequence and behind the last one write nothing: not the cache, not q's output, not what is read back."""
    k_cache, v_cache = vedic.kv_cache(6, 8, 2, 64, four_bit)
    for c in (k_cache, v_cache):
        bits(c).fill_(77)
    x = torch.randn(12, 6, 64, device="cuda").half()
    table = torch.tensor([[4, 1], [2, 0]], dtype=torch.int32, device="cuda")
    lens, starts = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([9, 3], [2, 6, 9]))
    out = torch.full((12, 2, 64), 5.0, dtype=torch.float16, device="cuda")
    vedic.kv_append(x[:, :2], x[:, 2:4], x[:, 4:], k_cache, v_cache, table, lens, starts, out=out)
    assert torch.equal(out[2:9], x[2:9, :2]) and (out[:2] == 5).all() and (out[9:] == 5).all()
    there = torch.zeros(6, 8, dtype=torch.bool)
    there[4, 5:], there[1, 0], there[2, :3] = True, True, True  # positions 5 .. 8 and 0 .. 2
    for c in (k_cache, v_cache):
        touched = (bits(c) != 77).any(-1).any(1).cpu()
        assert (touched == there).all()
    kr, vr = vedic.kv_read(k_cache, v_cache, table, lens, starts, 12)
    want = [torch.from_numpy(plain.values_of(plain.rows_of(x[2:9, i:i + 2].cpu().numpy(), four_bit), four_bit)).cuda() for i in (2, 4)]
    assert torch.equal(kr[2:9], want[0]) and torch.equal(vr[2:9], want[1])


def test_recorded_beside_another_stream():
    """An append recorded on one stream, replayed while lengths grow in place, with eager appends to another cache on a second one."""
    caches = [vedic.kv_cache(4, 16, 2, 64) for _ in range(2)]
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    lens = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2)]
    x = torch.randn(40, 1, 2, 64, device="cuda").half()
    step = torch.empty(1, 2, 64, dtype=torch.float16, device="cuda")
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            lens[0] += 1
            vedic.kv_append(None, step, step, *caches[0], table, lens[0])
    for i in range(40):
        with torch.cuda.stream(s):
            step.copy_(x[i])
            graph.replay()
        with torch.cuda.stream(other):
            lens[1] += 1
            vedic.kv_append(None, x[i], x[i], *caches[1], table, lens[1])
    torch.cuda.synchronize()
    for c in caches:
        assert torch.equal(c[0].transpose(1, 2).reshape(64, 2, 64)[:40], x[:, 0])
    assert torch.equal(caches[0][1], caches[1][1])


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("count", [64, 65, 300, 4160])
def test_many_sequences(count, four_bit):
    """Empty ones among them, at both ends too, more than a wave's lanes and more blocks of 64 than that."""
    rng = np.random.default_rng(count)
    lens = rng.integers(0, 9, count)
    new = np.minimum(lens, rng.integers(0, 4, count))
    new[0] = new[-1] = new[count // 2:count // 2 + 20] = 0
    append_and_check(count, 1, 1, 32, four_bit, 4, new.tolist(), lens.tolist(), 32, False, torch.float16)


def test_a_padded_batch_of_many_sequences():
    """Rows before the first of 200 sequences and behind the last one belong to none."""
    n = 200
    k_cache, v_cache = vedic.kv_cache(n, 4, 1, 8)
    x = torch.randn(n + 9, 1, 8, device="cuda").half()
    table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None]
    lens, starts = torch.full((n,), 2, dtype=torch.int32, device="cuda"), torch.arange(n + 1, dtype=torch.int32, device="cuda") + 5
    out = torch.full((n + 9, 1, 8), 5.0, dtype=torch.float16, device="cuda")
    vedic.kv_append(x, x, x, k_cache, v_cache, table, lens, starts, out=out)
    assert torch.equal(out[5:-4], x[5:-4]) and (out[:5] == 5).all() and (out[-4:] == 5).all()
    assert torch.equal(k_cache[:, 0, 1], x[5:-4, 0]) and (k_cache[:, 0, [0, 2, 3]] == 0).all()
    for st in (starts.flip(0).contiguous(), torch.randint(-9, n + 30, (n + 1,), dtype=torch.int32, device="cuda")):
        vedic.kv_append(x, x, x, k_cache, v_cache, table, lens, st)
        vedic.kv_read(k_cache, v_cache, table, lens, st, tokens=n + 9)
        torch.cuda.synchronize()
