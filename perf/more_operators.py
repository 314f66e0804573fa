"""Measured cases of decoding with a paged cache and 4-bit weights: append, attention over the cache, products.

A sequence's keys and values lie in pages; `table[b]` lists sequence b's pages, `lens[b]` how many tokens it has, the new
ones included, and `q_start[b] .. q_start[b + 1] - 1` are the rows of its new tokens (its last ones).

  append  q and k rotated by their positions, q rounded to binary16, k and v written into the cache
  attend  each new row against the cached tokens up to its own position, heads of q sharing heads of k in groups; with a
          window w the keys from w tokens back on, and further back those whose position is a multiple of the stride
  w4      Y = epi(X W + b), W held in 4 bits with a scale and a minimum per group of values along K

Four bits: a 32-bit word holds eight consecutive values, value 2i in bits 4i .. 4i + 3, value 2i + 1 in bits 16 + 4i ..
19 + 4i; code n of a group with (s, m) stands for binary16(s n + m).  A cache row (one token, one head) is D binary16
values, or D / 8 words followed by D / 32 pairs (s, m); a weight is N columns of K / 8 words, and [N, groups, 2] pairs.
Sizes are the repository's (width 1024 in 16 heads of 64, FFN width 4096, 8192 tokens) or generic (shared heads of 128).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
GELU_C = 0.7978845608028654


def listed() -> list[dict]:
    return [
        # one decoded token of the repository's width: the smallest append, bound by latency
        dict(name="append_1", kind="append", B=1, T=1, Hq=16, H=16, D=64, fmt="f16", ps=64, past=4095, rot=64, inter=False,
             dtype="f16"),
        # a whole prompt, straight from the fp32 output of the packed projection
        dict(name="append_prompt_8192", kind="append", B=1, T=8192, Hq=16, H=16, D=64, fmt="f16", ps=64, past=0, rot=64,
             inter=False, dtype="f32"),
        # prompts of many requests in one ragged batch into a 4-bit cache, pages of an odd size, half of each head rotated
        dict(name="append_i4_ragged", kind="append", B=37, T=3001, Hq=32, H=8, D=128, fmt="i4", ps=48, past=2000, rot=64,
             inter=True, dtype="f16"),
        # one sequence's next token: few workgroups unless its keys are shared out
        dict(name="attend_1x4100", kind="attend", B=1, T=1, Hq=16, H=16, D=64, fmt="f16", ps=64, past=4099, window=0, stride=0),
        # a batch of sequences of unequal length decoded together, four heads of q to each of k: the cache is read once
        dict(name="attend_decode_32", kind="attend", B=32, T=32, Hq=32, H=8, D=128, fmt="f16", ps=64, past=16383, window=0,
             stride=0),
        # twice as many from a 4-bit cache, small pages
        dict(name="attend_decode_i4_64", kind="attend", B=64, T=64, Hq=32, H=8, D=128, fmt="i4", ps=16, past=16383, window=0,
             stride=0),
        # a whole prompt in one pass, bound by the matrix cores
        dict(name="attend_prompt_8192", kind="attend", B=1, T=8192, Hq=16, H=16, D=64, fmt="f16", ps=64, past=0, window=0,
             stride=0),
        # the next pieces of three long prompts from a 4-bit cache, a sparse mask far back
        dict(name="attend_chunk_i4", kind="attend", B=3, T=1500, Hq=32, H=8, D=128, fmt="i4", ps=48, past=12000, window=4000,
             stride=16),
        # one decoded row through the FFN's first product: the smallest product
        dict(name="w4_1", kind="w4", M=1, K=1024, N=4096, group=64, epi="gelu", out="f16"),
        # sixteen decoded rows against a large weight
        dict(name="w4_16", kind="w4", M=16, K=4096, N=16384, group=128, epi="none", out="f32"),
        # five rows at widths that are no multiple of anything
        dict(name="w4_odd_5", kind="w4", M=5, K=1999, N=3001, group=32, epi="bias", out="f32"),
        # a prompt's rows through the same weights
        dict(name="w4_prompt_2048", kind="w4", M=2048, K=1024, N=4096, group=64, epi="gelu", out="f16"),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo: int, hi: int) -> int:
    """A layer width: mostly multiples of 64, some multiples of 8, some odd."""
    w = _log(rng, lo, hi)
    p = rng.random()
    return max(64, w // 64 * 64) if p < 0.7 else max(8, w // 8 * 8) if p < 0.85 else w | 1


def draw(rng) -> dict:
    """One more case of the ranges above; none needs more work than the largest listed one of its operator."""
    kind = rng.choice(["append", "attend", "attend", "attend", "w4", "w4"])
    if kind == "w4":
        M = _log(rng, 1, 64) if rng.random() < 0.7 else _log(rng, 65, 2048)
        top = 16384 if M <= 64 else 4096
        return dict(kind="w4", M=M, K=_width(rng, 256, 4096 if M <= 64 else 1024), N=_width(rng, 256, top),
                    group=rng.choice([32, 64, 128]), epi=rng.choice(["none", "bias", "gelu"]), out=rng.choice(["f16", "f32"]))
    fmt = rng.choice(["f16", "i4"])
    Hq, H, D = rng.choice([(16, 16, 64), (32, 8, 128), (8, 1, 256), (12, 4, 96), (5, 5, 32), (24, 3, 160), (16, 2, 64)])
    if fmt == "f16" and rng.random() < 0.2:
        D = rng.choice([40, 72, 104])
    ps = rng.choice([16, 48, 64, 128, 200])
    B = _log(rng, 1, 64)
    if kind == "append":
        T = B if rng.random() < 0.4 else max(B, _log(rng, 1, 8192))
        while T * (Hq + 2 * H) * D > 8192 * 48 * 64:
            T = max(1, T // 2)
        B = min(B, T)
        return dict(kind="append", B=B, T=T, Hq=Hq, H=H, D=D, fmt=fmt, ps=ps, past=_log(rng, 1, 4096),
                    rot=rng.choice([D, D // 8 * 4, 0]), inter=rng.random() < 0.5, dtype=rng.choice(["f16", "f32"]))
    past = _log(rng, 1, 16383)
    T = B if rng.random() < 0.6 else max(B, _log(rng, 1, 8192))
    while B * (past + T) * H * D > 32 * 16384 * 8 * 128:  # the largest listed caches
        B, T = B // 2, T // 2
        past = past if B > 8 else past // 2
        B, T = max(B, 1), max(T, 1)
    # (rows of one sequence are at most T - B + 1)
    while B * (T - B + 1) * Hq * (past + T) > 16 * 8192 * 8192 or T * Hq * D * (past + T // 2) > 16 * 64 * 8192 * 4096:
        T = max(B, T // 2)
        past = max(1, past * 3 // 4)
    window = 0 if rng.random() < 0.6 else _log(rng, 16, 4096)
    return dict(kind="attend", B=B, T=T, Hq=Hq, H=H, D=D, fmt=fmt, ps=ps, past=past, window=window,
                stride=0 if not window or rng.random() < 0.5 else rng.choice([7, 16, 100]))


# ---------------------------------------------------------------- inputs


def _lengths(c):
    """(new rows, tokens) of each sequence: the batch's shape, the same for every seed."""
    rng = random.Random(c["B"] * 1000003 + c["T"] * 101 + c["past"])
    B, T, past = c["B"], c["T"], c["past"]
    cuts = sorted(rng.sample(range(1, T), B - 1)) if B > 1 else []
    new = [b - a for a, b in zip([0] + cuts, cuts + [T])]
    old = [past] + [rng.randint(past // 8, past) for _ in range(B - 1)]
    return new, [n + p for n, p in zip(new, old)]


def _quantize(x):
    """Codes and (s, m) of groups of values [..., group] (binary16 values, held in any type)."""
    h = x.to(torch.float16).to(torch.float32)
    lo, hi = h.amin(-1, keepdim=True), h.amax(-1, keepdim=True)
    s = ((hi - lo) / 15.0).to(torch.float16).to(torch.float32)
    n = torch.where(s > 0, torch.round((h - lo) / s), torch.zeros_like(h)).clamp(0, 15)
    return n.to(torch.int32), torch.cat([s, lo], -1).to(torch.float16)


def _words(n):
    """Codes [..., 8 k] in words [..., k]."""
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=n.device)
    w = (n.reshape(*n.shape[:-1], -1, 8).to(torch.int64) << shift).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _codes(w):
    """The codes [..., 8 k] of words [..., k]."""
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=w.device)
    return ((w[..., None] >> shift) & 15).reshape(*w.shape[:-1], -1)


def _rows_of(x, fmt):
    """Cache rows of values [..., D]."""
    if fmt == "f16":
        return x.to(torch.float16)
    n, sm = _quantize(x.reshape(*x.shape[:-1], -1, 32))
    w = _words(n.reshape(x.shape)).contiguous().view(torch.uint8)
    return torch.cat([w, sm.reshape(*x.shape[:-1], -1).contiguous().view(torch.uint8)], -1)


def _values_of(rows, fmt, D):
    """The values [..., D] that cache rows stand for, fp32."""
    if fmt == "f16":
        return rows.to(torch.float32)
    n = _codes(rows[..., :D // 2].contiguous().view(torch.int32)).to(torch.float32)
    sm = rows[..., D // 2:].contiguous().view(torch.float16).to(torch.float32).reshape(*rows.shape[:-1], D // 32, 2)
    v = n.reshape(*rows.shape[:-1], D // 32, 32) * sm[..., :1] + sm[..., 1:]
    return v.to(torch.float16).to(torch.float32).reshape(*rows.shape[:-1], D)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    c = case

    def rnd(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)

    if c["kind"] == "w4":
        M, K, N, group = c["M"], c["K"], c["N"], c["group"]
        G = -(-K // group)
        w = torch.zeros(N, G * group, device=DEV)
        w[:, :K] = rnd(N, K, std=K ** -0.5)
        n, sm = _quantize(w.reshape(N, G, group))
        Kw = -(-K // 32) * 4  # words of a column: whole 16 bytes
        return dict(case=c, X=rnd(M, K, dtype=torch.float16), codes=_words(n.reshape(N, -1))[:, :Kw].contiguous(), sm=sm,
                    bias=rnd(N, std=0.1))
    new, lens = _lengths(c)
    B, T, Hq, H, D, ps = c["B"], c["T"], c["Hq"], c["H"], c["D"], c["ps"]
    most = [-(-n // ps) for n in lens]
    pages = sum(most) + 3
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    table = torch.full((B, max(most) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b in range(B):
        table[b, :most[b]] = order[at:at + most[b]]
        at += most[b]
    s = dict(case=c, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV), longest=max(lens), rows=max(new),
             q_start=torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV))
    shape = (pages, H, ps, D)
    if c["kind"] == "append":
        row = D if c["fmt"] == "f16" else D * 5 // 8
        s["k_cache"], s["v_cache"] = (torch.zeros(*shape[:3], row, device=DEV, dtype=torch.float16 if c["fmt"] == "f16" else
                                                  torch.uint8) for _ in range(2))
        dt = torch.float16 if c["dtype"] == "f16" else torch.float32
        s["qkv"] = rnd(T, Hq + 2 * H, D, dtype=dt)  # the packed projection's output
        if c["rot"]:
            angle = torch.arange(max(lens), device=DEV, dtype=torch.float64)[:, None] * \
                10000.0 ** (-torch.arange(0, c["rot"], 2, device=DEV, dtype=torch.float64) / c["rot"])
            s["rope"] = torch.cat([angle.cos(), angle.sin()], 1).to(torch.float32)
        else:
            s["rope"] = None
        return s
    # (page by page: what a page holds does not depend on the others)
    s["k_cache"], s["v_cache"] = (torch.cat([_rows_of(rnd(min(256, pages - i), *shape[1:]), c["fmt"])
                                             for i in range(0, pages, 256)]) for _ in range(2))
    s["q"] = rnd(T, Hq, D, dtype=torch.float16)
    return s


# ---------------------------------------------------------------- the operators


def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s: dict):
    from logos_amd import vedic

    c = s["case"]
    if c["kind"] == "w4":
        epi = {"none": vedic.EPI_NONE, "bias": vedic.EPI_BIAS, "gelu": vedic.EPI_BIAS_GELU}[c["epi"]]
        w = vedic.W4(s["codes"], s["sm"], c["K"], c["group"])
        return vedic.gemm_w4(s["X"], w, bias=None if c["epi"] == "none" else s["bias"], epilogue=epi,
                             out_dtype=torch.float16 if c["out"] == "f16" else torch.float32)
    q_start = None if c["T"] == c["B"] else s["q_start"]
    if c["kind"] == "attend":
        return vedic.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], q_start=q_start,
                                     window=c["window"], stride=c["stride"])
    Hq, H = c["Hq"], c["H"]
    q, k, v = s["qkv"][:, :Hq], s["qkv"][:, Hq:Hq + H], s["qkv"][:, Hq + H:]
    q16 = vedic.kv_append(q, k, v, s["k_cache"], s["v_cache"], s["table"], s["lens"], q_start=q_start, rope=s["rope"],
                          interleaved=c["inter"])
    if c["fmt"] == "f16":
        return q16, s["k_cache"], s["v_cache"]
    return (q16, *vedic.kv_read(s["k_cache"], s["v_cache"], s["table"], s["lens"], q_start=q_start, tokens=c["T"]))


def _rotate(x, pos, rope, inter):
    """Rows [T, heads, D] in fp32 turned by the angles of their positions."""
    x = x.to(torch.float32)
    if rope is None:
        return x
    rot = rope.shape[1]
    cos, sin = rope[pos][:, None, :rot // 2], rope[pos][:, None, rot // 2:]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    y = x.clone()
    if inter:
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    return y


def _gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(GELU_C * (x + 0.044715 * x * x * x)))


def _run_plain(s: dict):
    c = s["case"]
    f32 = torch.float32
    if c["kind"] == "w4":
        n = _codes(s["codes"])[:, :c["K"]].to(f32)
        group = torch.arange(c["K"], device=DEV) // c["group"]
        w = (n * s["sm"][:, group, 0].to(f32) + s["sm"][:, group, 1].to(f32)).to(torch.float16).to(f32)
        y = s["X"].to(f32) @ w.t()
        if c["epi"] != "none":
            y = y + s["bias"]
        y = _gelu(y) if c["epi"] == "gelu" else y
        return y.to(torch.float16) if c["out"] == "f16" else y
    Hq, H, D, ps, T = c["Hq"], c["H"], c["D"], c["ps"], c["T"]
    table, lens, q_start = s["table"].long(), s["lens"].long(), s["q_start"].long()
    k_cache, v_cache = s["k_cache"], s["v_cache"]
    if c["kind"] == "append":
        row = torch.arange(T, device=DEV)
        b = (q_start[None, 1:] <= row[:, None]).sum(1)
        pos = lens[b] - q_start[b + 1] + row
        x = s["qkv"]
        q = _rotate(x[:, :Hq], pos, s["rope"], c["inter"]).to(torch.float16)
        k = _rotate(x[:, Hq:Hq + H], pos, s["rope"], c["inter"]).to(torch.float16)
        v = x[:, Hq + H:].to(torch.float16)
        page, inside = table[b, pos // ps], pos % ps
        k_cache[page, :, inside] = _rows_of(k, c["fmt"])
        v_cache[page, :, inside] = _rows_of(v, c["fmt"])
        if c["fmt"] == "f16":
            return q, k_cache, v_cache
        return (q, _values_of(k_cache[page, :, inside], "i4", D).to(torch.float16),
                _values_of(v_cache[page, :, inside], "i4", D).to(torch.float16))
    # every sequence padded to the longest: keys and values [B, H, L, D], rows of q [B, H, G n, D]
    B, G, n, L = c["B"], Hq // H, s["rows"], s["longest"]
    t = torch.arange(L, device=DEV)
    page, inside = table[:, t // ps].clamp(min=0), (t % ps).expand(B, L)
    there = (t < lens[:, None])[:, None, :, None]
    k = _values_of(k_cache[page, :, inside], c["fmt"], D).transpose(1, 2)
    v = torch.where(there, _values_of(v_cache[page, :, inside], c["fmt"], D).transpose(1, 2), 0.0)
    i = torch.arange(n, device=DEV)
    count = q_start[1:] - q_start[:-1]
    at = (q_start[:-1, None] + i).clamp(max=T - 1)
    q = s["q"].to(f32)[at].reshape(B, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    x = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    pos = (lens - count)[:, None] + i
    seen = t <= pos[:, :, None]
    if c["window"]:
        near = t >= pos[:, :, None] - c["window"]
        seen &= near | (t % c["stride"] == 0) if c["stride"] else near
    x = x.reshape(B, H, G, n, L).masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    x = (x / x.sum(-1, keepdim=True)).reshape(B, H, G * n, L)
    o = (x @ v).reshape(B, H, G, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)
    return o[i < count[:, None]].to(torch.float16)


# ---------------------------------------------------------------- cost and exact values


def _seen(c, pos):
    """Keys that the row at position `pos` sees."""
    w, stride = c["window"], c["stride"]
    if not w or pos <= w:
        return pos + 1
    far = pos - w  # keys 0 .. far - 1 lie outside the window
    return w + 1 + ((far + stride - 1) // stride if stride else 0)


def work(case: dict) -> dict:
    c = case
    if c["kind"] == "w4":
        M, K, N, G = c["M"], c["K"], c["N"], -(-c["K"] // c["group"])
        return {"bytes": N * (K / 2 + 4 * G) + 2 * M * K + M * N * (2 if c["out"] == "f16" else 4) +
                (0 if c["epi"] == "none" else 4 * N), "flops": 2 * M * N * K}
    T, Hq, H, D = c["T"], c["Hq"], c["H"], c["D"]
    row = 2 * D if c["fmt"] == "f16" else D * 5 // 8
    new, lens = _lengths(c)
    if c["kind"] == "append":
        b = 2 if c["dtype"] == "f16" else 4
        return {"bytes": T * (Hq + 2 * H) * D * b + T * Hq * D * 2 + 2 * T * H * row + 4 * T * c["rot"],
                "flops": 3 * T * (Hq + H) * c["rot"]}
    pairs = sum(_seen(c, n - m + i) for m, n in zip(new, lens) for i in range(m))
    keys = sum(n if not c["window"] else min(n, _seen(c, n - 1) + (m - 1)) for m, n in zip(new, lens))
    return {"bytes": 2 * keys * H * row + 4 * T * Hq * D, "flops": 4 * pairs * Hq * D}


def exact(case: dict, seed: int):
    """The outputs by their definitions in 64 bits, for the inputs of this seed."""
    s = prepare(case, seed)
    c = case
    f64 = torch.float64
    if c["kind"] == "w4":
        K, N = c["K"], c["N"]
        w = torch.empty(N, K, dtype=f64, device=DEV)
        for k in range(8):  # value k of every word
            bit = 16 * (k % 2) + 4 * (k // 2)
            cols = torch.arange(k, K, 8, device=DEV)
            sm = s["sm"][:, cols // c["group"]].to(f64)
            n = (s["codes"][:, :cols.numel()] >> bit) % 16
            w[:, cols] = (sm[..., 0] * n.to(f64) + sm[..., 1]).to(torch.float16).to(f64)
        y = torch.matmul(w, s["X"].to(f64).t()).t()
        if c["epi"] != "none":
            y = y + s["bias"].to(f64)
        return y * torch.sigmoid(2.0 * GELU_C * (y + 0.044715 * y ** 3)) if c["epi"] == "gelu" else y

    def four_bits(x):
        """Values [..., D] as 4-bit rows give them back, with the format's roundings to binary16."""
        h = x.to(torch.float16).to(f64).unflatten(-1, (-1, 32))
        m = h.min(-1, keepdim=True).values
        step = ((h.max(-1, keepdim=True).values - m) / 15).to(torch.float16).to(f64)
        n = ((h - m) / step.masked_fill(step == 0, 1.0)).round().clamp(0, 15)
        return (step * n + m).to(torch.float16).to(f64).flatten(-2)

    Hq, H, D, ps = c["Hq"], c["H"], c["D"], c["ps"]
    new, lens = _lengths(c)
    table = s["table"].tolist()
    ends = s["q_start"].tolist()
    if c["kind"] == "append":
        out = s["qkv"].to(f64)
        pos = torch.tensor([n - m + i for m, n in zip(new, lens) for i in range(m)], device=DEV)
        if c["rot"]:
            half = c["rot"] // 2
            z = torch.complex(s["rope"][pos, :half].to(f64), s["rope"][pos, half:].to(f64))[:, None]
            part = out[:, :Hq + H]
            if c["inter"]:
                turned = torch.view_as_real(torch.view_as_complex(part[..., :c["rot"]].unflatten(-1, (half, 2)).contiguous()) * z)
                part[..., :c["rot"]] = turned.flatten(-2)
            else:
                turned = torch.complex(part[..., :half], part[..., half:c["rot"]]) * z
                part[..., :half], part[..., half:c["rot"]] = turned.real, turned.imag
        q, k, v = out[:, :Hq], out[:, Hq:Hq + H], out[:, Hq + H:]
        if c["fmt"] == "i4":
            return q, four_bits(k.to(torch.float32)), four_bits(v)
        caches = []
        for x, cache in ((k, s["k_cache"]), (v, s["v_cache"])):
            cache = cache.to(f64)
            for b in range(c["B"]):
                p = pos[ends[b]:ends[b + 1]]
                pages = s["table"][b].long()[torch.div(p, ps, rounding_mode="floor")]
                cache[pages, :, p % ps] = x[ends[b]:ends[b + 1]]
            caches.append(cache)
        return (q, *caches)
    out = torch.empty(c["T"], Hq, D, dtype=f64, device=DEV)
    G = Hq // H
    for b in range(c["B"]):
        pages = torch.tensor(table[b][:-(-lens[b] // ps)], device=DEV)
        kv = []
        for cache in (s["k_cache"], s["v_cache"]):
            rows = cache[pages].transpose(1, 2).flatten(0, 1)[:lens[b]]  # [tokens, H, row]
            kv.append(_values_of(rows, c["fmt"], D).to(f64))
        p = torch.arange(lens[b] - new[b], lens[b], device=DEV)[:, None]
        t = torch.arange(lens[b], device=DEV)[None]
        hidden = t > p
        if c["window"]:
            away = p - t > c["window"]
            hidden = hidden | (away & (t.remainder(c["stride"]) != 0) if c["stride"] else away)
        for h in range(Hq):
            x = s["q"][ends[b]:ends[b + 1], h].to(f64) @ kv[0][:, h // G].t() / D ** 0.5
            out[ends[b]:ends[b + 1], h] = torch.softmax(x.masked_fill(hidden, -math.inf), 1) @ kv[1][:, h // G]
    return out
