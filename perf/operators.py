"""Measured cases of the operators whose rows choose their weights: routed experts and per-request low-rank adapters.

A feed-forward layer of E experts sends each token to k of them.  Its steps, forward and backward, and the adapters of
many requests beside one shared projection, are the four operators here (sizes: the repository's model width 1024, FFN
width 4096, 8192 tokens, down to one decoded token, and odd ones):

  route     the k largest of a token's E logits (a tie goes to the lower expert), their softmax weights, and the token
            lists by expert that the products need (offsets, rows, slots); backward: the logits' gradient
  experts   products whose R = tokens x k rows, sorted by expert, each take their expert's weight:
              up   H = gelu(X[rows] W1[e] + b1[e]), with the pre-activation P that the backward reads
              down Y = H W2[e] + b2[e]
              dh   dH = (dY W2[e]^T) * gelu'(P)        dx   dXr = dH W1[e]^T
              dw1  dW1[e] = X[rows_e]^T dH_e, db1[e]   dw2  dW2[e] = H_e^T dY_e, db2[e]
  combine   out[t] = residual[t] + sum over j of w[t, j] Y[slot[t, j]]; backward: dY[slot] = w dout, dw = <dout, Y>
  adapters  Y = X W + b, and for the rows of adapter g  Y += s[g] (X A[g]) B[g]

The GELU is the tanh form.  Binary16 operands accumulate in fp32.  `rows` is the token of each sorted row, `offsets`
the first sorted row of each expert (and the end), `slots` the sorted row of each (token, j).
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
GELU_C = 0.7978845608028654


def listed() -> list[dict]:
    return [
        # one decoded token's choice of 2 experts of 8: the smallest call, bound by latency
        dict(name="route_1x8", kind="route", T=1, E=8, k=2, renorm=True, bwd=False),
        # a long prompt over many small experts: 8 of 128, renormalised weights
        dict(name="route_8192x128", kind="route", T=8192, E=128, k=8, renorm=True, bwd=False),
        # the router's backward of an odd batch over 60 experts, weights from the softmax over all of them
        dict(name="route_bwd_4099x60", kind="route", T=4099, E=60, k=4, renorm=False, bwd=True),
        # four sequences decoded together: every chosen expert's weight is read for a row or two
        dict(name="experts_up_decode_4", kind="experts", op="up", T=4, E=8, k=2, D=1024, F=4096, dtype="f16"),
        # the layer's first product over a full training batch, binary16, the pre-activation kept
        dict(name="experts_up_8192", kind="experts", op="up", T=8192, E=8, k=2, D=1024, F=4096, dtype="f16"),
        # the backward through the activation for many smaller experts, few rows each
        dict(name="experts_dh_2048x32", kind="experts", op="dh", T=2048, E=32, k=4, D=1024, F=1024, dtype="f16"),
        # weight gradients of the first product over a full batch: ragged contractions, tokens gathered
        dict(name="experts_dw1_8192", kind="experts", op="dw1", T=8192, E=8, k=2, D=1024, F=4096, dtype="f16"),
        # the second product in strict fp32 at widths that are no multiple of anything (rows not 16-byte aligned)
        dict(name="experts_down_fp32_odd", kind="experts", op="down", T=1003, E=7, k=2, D=1001, F=1999, dtype="f32"),
        # the experts' outputs back in token order onto the residual stream
        dict(name="combine_8192", kind="combine", T=8192, E=8, k=2, D=1024, residual=True, bwd=False),
        # its backward: rows of gradient in binary16 for the products, and the weights' gradients
        dict(name="combine_bwd_4099", kind="combine", T=4099, E=60, k=4, D=1000, residual=False, bwd=True),
        # sixteen sequences decoded together, each with an adapter of its own beside the shared projection
        dict(name="adapters_decode_16", kind="adapters", M=16, K=1024, N=4096, r=16, G=32, dtype="f16"),
        # prompts of a dozen requests in one batch, adapters of rank 64, some rows without one
        dict(name="adapters_prompt_4096", kind="adapters", M=4096, K=1024, N=4096, r=64, G=12, dtype="f16"),
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
    kind = rng.choice(["route", "experts", "experts", "experts", "combine", "adapters"])
    if kind == "route":
        E = _log(rng, 4, 256)
        return dict(kind="route", T=_log(rng, 1, 8192 if E <= 128 else 4096), E=E, k=rng.randint(1, min(E, 8)),
                    renorm=rng.random() < 0.5, bwd=rng.random() < 0.4)
    if kind == "combine":
        k = rng.randint(1, 8)
        return dict(kind="combine", T=_log(rng, 1, 16384 // k), E=_log(rng, max(4, k), 64), k=k, D=_width(rng, 64, 1024),
                    residual=rng.random() < 0.5, bwd=rng.random() < 0.5)
    dtype = "f16" if rng.random() < 0.75 else "f32"
    if kind == "adapters":
        return dict(kind="adapters", M=_log(rng, 1, 4096), K=_width(rng, 256, 1024), N=_width(rng, 256, 4096),
                    r=rng.choice([4, 8, 16, 24, 32, 64]), G=_log(rng, 2, 64), dtype=dtype)
    E = _log(rng, 2, 64)
    k = rng.randint(1, min(E, 4))
    T = _log(rng, 1, 16384 // k)
    D, F = _width(rng, 256, 1024), _width(rng, 256, 4096)
    while E * D * F > 8 * 1024 * 4096:  # as many weights as the listed layers have at most
        E = max(k, E // 2)
        F = max(256, F // 2)
    return dict(kind="experts", op=rng.choice(["up", "down", "dh", "dx", "dw1", "dw2"]), T=T, E=E, k=k, D=D, F=F,
                dtype=dtype)


# ---------------------------------------------------------------- inputs


def _logits(g, T, E):
    """Router logits with some experts in more demand than others, as a trained router has them."""
    return torch.randn(T, E, device=DEV, generator=g) + 0.5 * torch.randn(E, device=DEV, generator=g)


def _choose(logits, k):
    """The k largest logits of each row, the lower index first among equals."""
    order = torch.argsort(logits, dim=1, descending=True, stable=True)
    return order[:, :k].to(torch.int32).contiguous()


def _group(ids, groups, per_row):
    """(offsets, rows, slots): the entries of `ids` sorted by group, in their order within each."""
    flat = ids.reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    edges = torch.arange(groups + 1, device=ids.device)
    offsets = (flat[None, :] < edges[:, None]).sum(1).to(torch.int32)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(flat.numel(), device=ids.device)
    return offsets, (order // per_row).to(torch.int32), slots.to(torch.int32).reshape(ids.shape)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def rnd(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)

    kind = case["kind"]
    if kind == "route":
        T, E, k = case["T"], case["E"], case["k"]
        s = dict(case=case, logits=_logits(g, T, E))
        if case["bwd"]:
            s["ids"] = _choose(s["logits"], k)
            s["weights"] = _weights(s["logits"], s["ids"], case["renorm"], torch.float32)
            s["dw"] = rnd(T, k)
        return s
    if kind == "combine":
        T, E, k, D = case["T"], case["E"], case["k"], case["D"]
        logits = _logits(g, T, E)
        ids = _choose(logits, k)
        _, _, slots = _group(ids, E, k)
        s = dict(case=case, slots=slots, weights=_weights(logits, ids, True, torch.float32), Y=rnd(T * k, D))
        s["residual"] = rnd(T, D) if case["residual"] else None
        if case["bwd"]:
            s["dout"] = rnd(T, D, std=0.1)
        return s
    dt = torch.float16 if case["dtype"] == "f16" else torch.float32
    if kind == "experts":
        T, E, k, D, F, op = case["T"], case["E"], case["k"], case["D"], case["F"], case["op"]
        offsets, rows, _ = _group(_choose(_logits(g, T, E), k), E, k)
        s = dict(case=case, offsets=offsets, rows=rows, ends=offsets.tolist())
        R = T * k
        if op in ("up", "dw1"):
            s["X"] = rnd(T, D, dtype=dt)
        if op in ("up", "dx"):
            s["W1"] = rnd(E, D, F, std=D ** -0.5, dtype=dt)
        if op in ("down", "dh"):
            s["W2"] = rnd(E, F, D, std=F ** -0.5, dtype=dt)
        if op == "up":
            s["b1"] = rnd(E, F, std=0.1)
        if op == "down":
            s["b2"] = rnd(E, D, std=0.1)
        if op in ("down", "dw2"):
            s["H"] = rnd(R, F, std=0.5, dtype=dt)
        if op == "dh":
            s["P"] = rnd(R, F, dtype=dt)
        if op in ("dh", "dw2"):
            s["dY"] = rnd(R, D, std=0.1, dtype=dt)
        if op in ("dx", "dw1"):
            s["dH"] = rnd(R, F, std=0.1, dtype=dt)
        return s
    M, K, N, r, G = case["M"], case["K"], case["N"], case["r"], case["G"]
    # the rows of one request lie together (about G requests; decoded rows: one each), one request in eight has no adapter
    cuts = torch.rand(M, device=DEV, generator=g) < max(min(1.0, 2.0 * G / M), 1e-3) if M > 64 else \
        torch.ones(M, dtype=torch.bool, device=DEV)
    request = torch.cumsum(cuts.long(), 0)
    of_request = torch.randint(0, G, (M + 1,), device=DEV, generator=g)
    of_request[torch.rand(M + 1, device=DEV, generator=g) < 0.125] = G
    ids = of_request[request]
    offsets, rows, _ = _group(ids, G, 1)
    ends = offsets.tolist()
    return dict(case=case, offsets=offsets, rows=rows, ends=ends, X=rnd(M, K, dtype=dt), W=rnd(K, N, std=K ** -0.5, dtype=dt),
                b=rnd(N, std=0.1), A=rnd(G, K, r, std=K ** -0.5, dtype=dt), B=rnd(G, r, N, std=r ** -0.5, dtype=dt),
                scales=torch.rand(G, device=DEV, generator=g) + 0.5)


# ---------------------------------------------------------------- the operators


def _weights(logits, ids, renorm, dt):
    """The chosen experts' weights: their softmax among themselves (renorm) or within all experts."""
    x = logits.to(dt)
    sel = x.gather(1, ids.long())
    top = sel.amax(1, keepdim=True)
    e = torch.exp(sel - top)
    return e / (e if renorm else torch.exp(x - top)).sum(1, keepdim=True)


def _gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(GELU_C * (x + 0.044715 * x * x * x)))


def _gelu_grad(x):
    t = torch.tanh(GELU_C * (x + 0.044715 * x * x * x))
    return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * GELU_C * (1.0 + 3.0 * 0.044715 * x * x)


def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s: dict):
    from logos_amd import vedic

    c = s["case"]
    if c["kind"] == "route":
        if c["bwd"]:
            return vedic.route_topk_bwd(s["logits"], s["ids"], s["weights"], s["dw"], renorm=c["renorm"])
        r = vedic.route_topk(s["logits"], c["k"], renorm=c["renorm"])
        return r.ids, r.weights, r.offsets, r.rows, r.slots
    if c["kind"] == "combine":
        if c["bwd"]:
            return vedic.combine_rows_bwd(s["dout"], s["Y"], s["slots"], s["weights"], out_dtype=torch.float16)
        return vedic.combine_rows(s["Y"], s["slots"], s["weights"], residual=s["residual"])
    if c["kind"] == "adapters":
        return vedic.gemm_lora(s["X"], s["W"], s["A"], s["B"], s["offsets"], s["rows"], bias=s["b"], scales=s["scales"])
    op, off = c["op"], s["offsets"]
    if op == "up":
        P = torch.empty(c["T"] * c["k"], c["F"], dtype=s["X"].dtype, device=DEV)
        H = vedic.gemm_grouped(vedic.OP_NN, s["X"], s["W1"], off, rows=s["rows"], bias=s["b1"], preact=P,
                               epilogue=vedic.EPI_BIAS_GELU, out_dtype=s["X"].dtype)
        return H, P
    if op == "down":
        return vedic.gemm_grouped(vedic.OP_NN, s["H"], s["W2"], off, bias=s["b2"], epilogue=vedic.EPI_BIAS)
    if op == "dh":
        return vedic.gemm_grouped(vedic.OP_NT, s["dY"], s["W2"], off, preact=s["P"], epilogue=vedic.EPI_GELU_BWD,
                                  out_dtype=s["dY"].dtype)
    if op == "dx":
        return vedic.gemm_grouped(vedic.OP_NT, s["dH"], s["W1"], off)
    A, B, rows = (s["X"], s["dH"], s["rows"]) if op == "dw1" else (s["H"], s["dY"], None)
    db = torch.empty(c["E"], B.shape[1], device=DEV)
    return vedic.gemm_grouped(vedic.OP_TN, A, B, off, rows=rows, db=db), db


def _run_plain(s: dict):
    c = s["case"]
    f32 = torch.float32
    if c["kind"] == "route":
        logits = s["logits"]
        if c["bwd"]:
            w, dw, ids = s["weights"], s["dw"], s["ids"].long()
            inner = (w * dw).sum(1, keepdim=True)
            if c["renorm"]:
                return torch.zeros_like(logits).scatter(1, ids, w * (dw - inner))
            p = torch.exp(logits - logits.amax(1, keepdim=True))
            p = p / p.sum(1, keepdim=True)
            return p * (torch.zeros_like(p).scatter(1, ids, dw) - inner)
        ids = _choose(logits, c["k"])
        return (ids, _weights(logits, ids, c["renorm"], f32), *_group(ids, c["E"], c["k"]))
    if c["kind"] == "combine":
        slots = s["slots"].long()
        w, Y = s["weights"], s["Y"].to(f32)
        if c["bwd"]:
            dout = s["dout"].to(f32)
            dY = torch.empty_like(Y)
            dY[slots.reshape(-1)] = (w[:, :, None] * dout[:, None, :]).reshape(-1, Y.shape[1])
            return dY.to(torch.float16), (Y[slots] * dout[:, None, :]).sum(2)
        out = (w[:, :, None] * Y[slots]).sum(1)
        return out if s["residual"] is None else s["residual"] + out
    ends = s["ends"]
    if c["kind"] == "adapters":
        X = s["X"].to(f32)
        Y = X @ s["W"].to(f32) + s["b"]
        for g in range(c["G"]):
            if ends[g] < ends[g + 1]:
                i = s["rows"][ends[g]:ends[g + 1]].long()
                Y[i] += s["scales"][g] * ((X[i] @ s["A"][g].to(f32)) @ s["B"][g].to(f32))
        return Y
    op, E = c["op"], c["E"]
    groups = [(e, ends[e], ends[e + 1]) for e in range(E)]
    rows = s["rows"].long()
    if op in ("up", "down", "dh", "dx"):
        src = {"up": "X", "down": "H", "dh": "dY", "dx": "dH"}[op]
        A, W = s[src].to(f32), s["W1" if op in ("up", "dx") else "W2"]
        out = torch.empty(rows.numel(), W.shape[2] if op in ("up", "down") else W.shape[1], device=DEV)
        for e, i0, i1 in groups:
            if i0 < i1:
                a = A[rows[i0:i1]] if op == "up" else A[i0:i1]
                w = W[e].to(f32)
                out[i0:i1] = a @ w if op in ("up", "down") else a @ w.t()
                if op in ("up", "down"):
                    out[i0:i1] += s["b1" if op == "up" else "b2"][e]
        if op == "up":
            return _gelu(out).to(s["X"].dtype), out.to(s["X"].dtype)
        if op == "dh":
            return (out * _gelu_grad(s["P"].to(f32))).to(s["dY"].dtype)
        return out
    A, B = (s["X"].to(f32), s["dH"].to(f32)) if op == "dw1" else (s["H"].to(f32), s["dY"].to(f32))
    dW = torch.zeros(E, A.shape[1], B.shape[1], device=DEV)
    db = torch.zeros(E, B.shape[1], device=DEV)
    for e, i0, i1 in groups:
        if i0 < i1:
            a = A[rows[i0:i1]] if op == "dw1" else A[i0:i1]
            dW[e] = a.t() @ B[i0:i1]
            db[e] = B[i0:i1].sum(0)
    return dW, db


# ---------------------------------------------------------------- cost and exact values


def _experts_widths(c):
    """(contraction, output width) of the row products; (M, N) of the weight gradients."""
    D, F = c["D"], c["F"]
    return {"up": (D, F), "down": (F, D), "dh": (D, F), "dx": (F, D), "dw1": (D, F), "dw2": (F, D)}[c["op"]]


def work(case: dict) -> dict:
    c = case
    if c["kind"] == "route":
        T, E, k = c["T"], c["E"], c["k"]
        if c["bwd"]:  # ids, weights and their gradients in (the logits where all of them count), the gradient out
            return {"bytes": 4 * T * (3 * k + E * (1 if c["renorm"] else 2)), "flops": 4 * T * (k if c["renorm"] else E)}
        return {"bytes": 4 * (T * E + 4 * T * k + E + 1), "flops": 3 * T * (k if c["renorm"] else E)}
    if c["kind"] == "combine":
        T, k, D = c["T"], c["k"], c["D"]
        if c["bwd"]:
            return {"bytes": T * D * 4 + T * k * (D * 6 + 12), "flops": 3 * T * k * D}
        return {"bytes": T * D * (8 if c["residual"] else 4) + T * k * (D * 4 + 8), "flops": 2 * T * k * D}
    b = 2 if c["dtype"] == "f16" else 4
    if c["kind"] == "adapters":
        M, K, N, r = c["M"], c["K"], c["N"], c["r"]
        used = min(c["G"], M)
        return {"bytes": b * (M * K + K * N + used * r * (K + N)) + 4 * (M * N + N),
                "flops": 2 * M * K * N + 2 * M * r * (K + N)}
    T, E, R = c["T"], c["E"], c["T"] * c["k"]
    used = min(E, R)
    K, N = _experts_widths(c)
    op = c["op"]
    flops = 2 * R * K * N
    if op == "up":
        return {"bytes": b * (T * K + used * K * N + 2 * R * N) + 4 * (R + used * N), "flops": flops}
    if op == "down":
        return {"bytes": b * (R * K + used * K * N) + 4 * (R * N + used * N), "flops": flops}
    if op == "dh":
        return {"bytes": b * (R * K + used * K * N + 2 * R * N), "flops": flops}
    if op == "dx":
        return {"bytes": b * (R * K + used * K * N) + 4 * R * N, "flops": flops}
    rows_in = T * K if op == "dw1" else R * K
    return {"bytes": b * (rows_in + R * N) + 4 * (E * K * N + E * N), "flops": flops}


def exact(case: dict, seed: int):
    """The outputs by their definitions in 64 bits, for the inputs of this seed."""
    s = prepare(case, seed)
    c = case
    f64 = torch.float64
    if c["kind"] == "route":
        x = s["logits"].to(f64)
        if c["bwd"]:
            # d/dx of sum_j dw_j w_j(x) through the definition of w, with the weights recomputed in 64 bits
            ids, dw = s["ids"].long(), s["dw"].to(f64)
            p = torch.softmax(x, 1)
            q = p.gather(1, ids)
            grad = torch.zeros_like(x)
            if c["renorm"]:
                z = q.sum(1, keepdim=True)
                q = q / z
                mean = torch.einsum("tj,tj->t", q, dw)
                for j in range(c["k"]):
                    grad[torch.arange(c["T"], device=DEV), ids[:, j]] = q[:, j] * (dw[:, j] - mean)
                return grad
            mean = torch.einsum("tj,tj->t", q, dw)
            grad = -p * mean[:, None]
            for j in range(c["k"]):
                grad[torch.arange(c["T"], device=DEV), ids[:, j]] += q[:, j] * dw[:, j]
            return grad
        T, E, k = c["T"], c["E"], c["k"]
        left = x.clone()
        ids = torch.empty(T, k, dtype=torch.int64, device=DEV)
        for j in range(k):
            best = left.amax(1, keepdim=True)
            at = torch.where(left == best, torch.arange(E, device=DEV)[None, :], E).amin(1)
            ids[:, j] = at
            left[torch.arange(T, device=DEV), at] = -math.inf
        p = torch.softmax(x, 1).gather(1, ids)
        if c["renorm"]:
            p = p / p.sum(1, keepdim=True)
        counts = torch.bincount(ids.reshape(-1), minlength=E)
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), counts.cumsum(0)])
        key = ids.reshape(-1) * (T * k) + torch.arange(T * k, device=DEV)
        pairs = key.sort().values % (T * k)
        slots = torch.empty_like(pairs)
        slots[pairs] = torch.arange(T * k, device=DEV)
        i32 = torch.int32
        return ids.to(i32), p, offsets.to(i32), (pairs // k).to(i32), slots.reshape(T, k).to(i32)
    if c["kind"] == "combine":
        slots, w, Y = s["slots"].long(), s["weights"].to(f64), s["Y"].to(f64)
        if c["bwd"]:
            dout = s["dout"].to(f64)
            dY = torch.empty_like(Y)
            dw = torch.empty_like(w)
            for j in range(c["k"]):
                dY[slots[:, j]] = w[:, j, None] * dout
                dw[:, j] = (dout * Y[slots[:, j]]).sum(1)
            return dY, dw
        out = torch.zeros(c["T"], c["D"], dtype=f64, device=DEV) if s["residual"] is None else s["residual"].to(f64)
        for j in range(c["k"]):
            out = out + w[:, j, None] * Y[slots[:, j]]
        return out
    if c["kind"] == "adapters":
        X = s["X"].to(f64)
        Y = X @ s["W"].to(f64) + s["b"].to(f64)
        for g in range(c["G"]):
            i = s["rows"][s["ends"][g]:s["ends"][g + 1]].long()
            if i.numel():
                Y[i] += s["scales"][g].to(f64) * (X[i] @ s["A"][g].to(f64) @ s["B"][g].to(f64))
        return Y
    op, ends = c["op"], s["ends"]
    out, sums = [], []
    for e in range(c["E"]):
        at = slice(ends[e], ends[e + 1])
        token = s["rows"][at].long()
        if op == "up":
            out.append(s["X"][token].to(f64) @ s["W1"][e].to(f64) + s["b1"][e].to(f64))
        elif op == "down":
            out.append(s["H"][at].to(f64) @ s["W2"][e].to(f64) + s["b2"][e].to(f64))
        elif op == "dh":
            out.append(s["dY"][at].to(f64) @ s["W2"][e].to(f64).t())
        elif op == "dx":
            out.append(s["dH"][at].to(f64) @ s["W1"][e].to(f64).t())
        else:
            a = s["X"][token] if op == "dw1" else s["H"][at]
            b = (s["dH"] if op == "dw1" else s["dY"])[at].to(f64)
            out.append(a.to(f64).t() @ b)
            sums.append(b.sum(0))
    if op in ("dw1", "dw2"):
        return torch.stack(out), torch.stack(sums)
    C = torch.cat(out)
    if op == "up":
        return C * torch.sigmoid(2.0 * GELU_C * (C + 0.044715 * C ** 3)), C
    if op == "dh":
        P = s["P"].to(f64)
        sg = torch.sigmoid(2.0 * GELU_C * (P + 0.044715 * P ** 3))
        return C * (sg + P * sg * (1.0 - sg) * 2.0 * GELU_C * (1.0 + 0.134145 * P ** 2))
    return C
