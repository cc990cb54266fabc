"""The feed-forward half of a layer, operator by operator: the residual addition and
RMS norm with an 8-bit output, the int8 matrix product that takes it, and the
mixture-of-experts layer for a few tokens.  A case is a dict of plain values;
`prepare` makes what a caller holds before the call, `run` is one pass (by elementary
torch operations, or by this library where `own` is true), `exact` the same result
in 64 bits.

Kinds (the "kind" of a case):
  norm   h = x + delta, y = rmsnorm(h) * w; h, and y in 8 bits: one scale a row
         ("row") or planar Q8_1 blocks of 32 ("planar")
  gemm   int8 rows times int8 weight rows, a scale a token and a channel
  moe    router, choice of k experts, their Q4_0 gate/up/down products, weighted sum
"""
import math
import os
import sys

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = float(torch.tensor(1e-5, dtype=torch.float32))     # the fp32 constant, as a C caller passes it
_TINY = 2.0 ** -120


def _lib():
    pkg = os.path.join(os.getcwd(), "lfm2-ampere_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import lk_attn
    return lk_attn


def listed():
    return [
        # one decode token between the attention projection and the feed-forward half: latency
        {"name": "norm_1x2048_f32", "kind": "norm", "rows": 1, "n": 2048, "type": "f32", "form": "row", "pad": 0},
        # a short prompt's rows on their way into a Q4_0 product
        {"name": "norm_333x2048_f32_q81", "kind": "norm", "rows": 333, "n": 2048, "type": "f32", "form": "planar",
         "pad": 0},
        # a whole prefill chunk, residual stream in 16 bits
        {"name": "norm_4096x2048_bf16", "kind": "norm", "rows": 4096, "n": 2048, "type": "bf16", "form": "row",
         "pad": 0},
        # one decode token through a wide projection: the weights' bytes
        {"name": "gemm_1x8192x2048_f16", "kind": "gemm", "M": 1, "N": 8192, "K": 2048, "type": "f16", "res": False,
         "pad": 0},
        # a few sequences decoded together, sizes that no tile divides
        {"name": "gemm_19x5003x1111_bf16", "kind": "gemm", "M": 19, "N": 5003, "K": 1111, "type": "bf16",
         "res": False, "pad": 0},
        # a short prompt's square projection, added to the residual rows
        {"name": "gemm_333x2048x2048_f32_res", "kind": "gemm", "M": 333, "N": 2048, "K": 2048, "type": "f32",
         "res": True, "pad": 0},
        # a prefill chunk through a wide projection
        {"name": "gemm_4096x8192x2048_bf16", "kind": "gemm", "M": 4096, "N": 8192, "K": 2048, "type": "bf16",
         "res": False, "pad": 0},
        # the largest chunk through the largest weights: the matrix cores' rate
        {"name": "gemm_8192x8192x8192_bf16", "kind": "gemm", "M": 8192, "N": 8192, "K": 8192, "type": "bf16",
         "res": False, "pad": 0},
        # one decode token's experts, added to the fp32 residual stream
        {"name": "moe_1_f32", "kind": "moe", "T": 1, "hidden": 2048, "ffn": 1536, "E": 64, "k": 4,
         "score": "sigmoid", "type": "f32", "res": True},
        # a few sequences, softmax routing over fewer, wider experts
        {"name": "moe_5_f16", "kind": "moe", "T": 5, "hidden": 2048, "ffn": 1792, "E": 32, "k": 2,
         "score": "softmax", "type": "f16", "res": False},
        # a batch of sequences, or the tokens of a draft that are checked at once
        {"name": "moe_19_bf16", "kind": "moe", "T": 19, "hidden": 2048, "ffn": 1536, "E": 64, "k": 4,
         "score": "sigmoid", "type": "bf16", "res": True},
        # the largest batch: nearly every expert has a token
        {"name": "moe_64_bf16", "kind": "moe", "T": 64, "hidden": 2048, "ffn": 1536, "E": 64, "k": 4,
         "score": "sigmoid", "type": "bf16", "res": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "gemm", "moe"])
    t = rng.choice(["f32", "f16", "bf16"])
    if kind == "norm":
        form = rng.choice(["row", "row", "planar"])
        n = 32 * _log(rng, 2, 256) if form == "planar" else _log(rng, 33, 16384)
        return {"kind": kind, "rows": _log(rng, 1, max(2, min(16384, (1 << 25) // n))), "n": n, "type": t,
                "form": form, "pad": rng.choice([0, 0, 8, 64])}
    if kind == "gemm":
        while True:
            M, N, K = _log(rng, 1, 8192), _log(rng, 16, 8192), _log(rng, 32, 8192)
            if rng.random() < 0.5:                           # half of them as most layers are
                N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
            if M * N * K <= 8192 ** 3 // 2:
                return {"kind": kind, "M": M, "N": N, "K": K, "type": t, "res": rng.random() < 0.4,
                        "pad": rng.choice([0, 0, 16, 64])}
    while True:
        c = {"kind": kind, "T": _log(rng, 1, 64), "hidden": 32 * rng.choice([16, 33, 40, 64, 64, 80, 128]),
             "ffn": 32 * rng.choice([8, 24, 37, 48, 56, 64]), "E": rng.choice([8, 16, 32, 60, 64, 128]),
             "k": rng.choice([1, 2, 4, 4, 6, 8]), "score": rng.choice(["sigmoid", "softmax"]), "type": t,
             "res": rng.random() < 0.6}
        # the weights of a state, and the gathered copies of the plain form, within the largest listed case's
        if c["E"] * c["ffn"] * c["hidden"] <= 64 * 1536 * 2048 and \
                c["T"] * c["k"] * c["ffn"] * c["hidden"] <= 256 * 1536 * 2048:
            return c


# ---- inputs -----------------------------------------------------------------------
def _gen(seed, tag):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + tag) & 0x7FFFFFFFFFFF)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rand(g, lo, hi, *shape):
    return lo + (hi - lo) * torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rows(x, pad):
    """x as rows of a buffer that is `pad` values wider (16-byte-aligned int8 rows in any case)."""
    n = x.shape[1]
    ld = n + pad
    if x.dtype == torch.int8:
        ld = (ld + 15) // 16 * 16
    if ld == n:
        return x.contiguous()
    buf = torch.zeros(x.shape[0], ld, dtype=x.dtype, device=x.device)
    buf[:, :n] = x
    return buf[:, :n]


def _norm_inputs(case, seed):
    g = _gen(seed, 1)
    rows, n, dt = case["rows"], case["n"], DT[case["type"]]
    # a residual stream: channels of unequal size, a few of them large
    chan = torch.exp(0.5 * _randn(g, n))
    chan[torch.randint(0, n, (max(1, n // 512),), generator=g, device="cuda")] *= 20.0
    x = (_randn(g, rows, n) * chan * 2.0).to(dt)
    delta = _randn(g, rows, n).to(dt)
    return _rows(x, case["pad"]), _rows(delta, case["pad"]), _rand(g, 0.5, 1.5, n)


def _gemm_inputs(case, seed):
    g = _gen(seed, 2)
    M, N, K = case["M"], case["N"], case["K"]
    # quantised rows and channels: near-normal values whose largest is 127
    def quant(rows):
        v = _randn(g, rows, K)
        a = v.abs().amax(1, keepdim=True)
        return torch.round(v * (127.0 / a)).to(torch.int8), (a / 127.0).reshape(-1).contiguous()
    x, sx = quant(M)
    w, sw = quant(N)
    res = _randn(g, M, N).to(DT[case["type"]]) * 8 if case["res"] else None
    return _rows(x, case["pad"]), sx, _rows(w, 0), (sw * K ** -0.5).contiguous(), res


def _q4(g, *rows_bpr):
    qs = torch.randint(0, 256, (*rows_bpr, 16), generator=g, device="cuda", dtype=torch.uint8)
    return qs, _rand(g, 0.002, 0.02, *rows_bpr).half()


def _moe_inputs(case, seed):
    g = _gen(seed, 3)
    T, H, F, E = case["T"], case["hidden"], case["ffn"], case["E"]
    x = (_randn(g, T, H) * _rand(g, 0.5, 1.5, H)).to(DT[case["type"]])
    return {"x": x, "router": _randn(g, E, H) * H ** -0.5,
            "bias": _randn(g, E) * 0.1 if case["score"] == "sigmoid" else None,
            "gate": _q4(g, E, F, H // 32), "up": _q4(g, E, F, H // 32), "down": _q4(g, E, H, F // 32),
            "res": (_randn(g, T, H) * 8).to(DT[case["type"]]) if case["res"] else None}


def prepare(case, seed):
    s = {"case": case}
    if own:
        s["lk"] = _lib()
    dt = DT[case["type"]]
    if case["kind"] == "norm":
        rows, n = case["rows"], case["n"]
        s["x"], s["delta"], s["w"] = _norm_inputs(case, seed)
        s["h"] = torch.empty(rows, n, dtype=dt, device="cuda")
        ld = (n + 15) // 16 * 16 if case["form"] == "row" else n
        s["q"] = torch.empty(rows, ld, dtype=torch.int8, device="cuda")[:, :n]
        s["sc"] = torch.empty((rows,) if case["form"] == "row" else (rows, n // 32, 2), device="cuda")
        s["values"] = torch.empty(rows, n, dtype=torch.float16 if dt == torch.float32 else dt, device="cuda")
    elif case["kind"] == "gemm":
        s["x"], s["sx"], s["w"], s["sw"], s["res"] = _gemm_inputs(case, seed)
        s["out"] = torch.empty(case["M"], case["N"], dtype=dt, device="cuda")
    else:
        s.update(_moe_inputs(case, seed))
        s["out"] = torch.empty_like(s["x"])
        s["ids"] = torch.empty(case["T"], case["k"], dtype=torch.int32, device="cuda")
        s["weights"] = torch.empty(case["T"], case["k"], device="cuda")
        if own:                                              # the layer's handle: its weights and workspace
            s["layer"] = s["lk"].MoeQ4_0(s["router"], s["gate"], s["up"], s["down"], case["k"],
                                         score=case["score"], bias=s["bias"], max_tokens=case["T"])
    return s


# ---- one pass -----------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        return {"norm": _own_norm, "gemm": _own_gemm, "moe": _own_moe}[case["kind"]](s, case)
    return {"norm": _plain_norm, "gemm": _plain_gemm, "moe": _plain_moe}[case["kind"]](s, case)


def _own_norm(s, case):
    s["lk"].norm_q8(s["x"], s["w"], s["q"], s["sc"], delta=s["delta"], res=s["h"], eps=_EPS)
    # the values that the 8 bits stand for
    if case["form"] == "row":
        torch.mul(s["q"], s["sc"].unsqueeze(1), out=s["values"])
    else:
        blocks = (case["rows"], case["n"] // 32, 32)
        torch.mul(s["q"].view(blocks), s["sc"][:, :, :1], out=s["values"].view(blocks))
    return {"h": s["h"], "scales": s["sc"], "values": s["values"]}


def _own_gemm(s, case):
    s["lk"].gemm_i8(s["x"], s["sx"], s["w"], s["sw"], s["out"], res=s["res"])
    return {"out": s["out"]}


def _own_moe(s, case):
    s["layer"](s["x"], s["out"], res=s["res"], ids=s["ids"], weights=s["weights"])
    return {"out": s["out"], "ids": s["ids"], "weights": s["weights"]}


def _plain_norm(s, case):
    rows, n = case["rows"], case["n"]
    h = s["x"].float() + s["delta"].float()
    # the mean square in 64 bits: the 8-bit values next to a rounding border follow from it
    r = (1.0 / torch.sqrt(h.double().square().sum(-1, keepdim=True) / n + _EPS)).float()
    y = (h * r) * s["w"]
    if case["form"] == "row":
        amax = y.abs().amax(-1, keepdim=True)
        some = amax >= _TINY
        scale = torch.where(some, amax / 127.0, torch.zeros_like(amax))
        q = torch.round(y * torch.where(some, 127.0 / amax, torch.zeros_like(amax)))
        values, scales = q * scale, scale.reshape(-1)
    else:
        y = y.view(rows, n // 32, 32)
        d = y.abs().amax(-1, keepdim=True) / 127.0
        v = torch.where(d > 0, y / d, torch.zeros_like(y))
        t = torch.trunc(v)
        q = t + torch.sign(v) * ((v - t).abs() >= 0.5)       # halves away from zero
        b = y
        for half in (16, 8, 4, 2, 1):                        # the format's own order of the 32 additions
            b = b[..., :half] + b[..., half:]
        d16 = d.half().float()
        values, scales = (q * d16).view(rows, n), torch.cat([d16, 8.0 * b.half().float()], -1)
    return {"h": h.to(s["h"].dtype), "scales": scales, "values": values.to(s["values"].dtype)}


def _plain_gemm(s, case):
    out = torch.mm(s["x"].float(), s["w"].float().t()) * s["sx"].unsqueeze(1) * s["sw"]
    if s["res"] is not None:
        out = s["res"].float() + out
    return {"out": out.to(s["out"].dtype)}


def _dense(q4, ids):
    """The Q4_0 rows of the chosen experts in fp32: byte j of a block holds element j
    in its low bits and element 16 + j in its high bits, 8 stands for zero."""
    qs, d = q4[0][ids], q4[1][ids]
    w = (torch.cat([qs & 15, qs >> 4], -1).float() - 8.0) * d.float().unsqueeze(-1)
    return w.flatten(-2)


def _plain_moe(s, case):
    T, k = case["T"], case["k"]
    x = s["x"].float()
    # the scores in 64 bits: which experts are chosen depends on their order
    logits = torch.mm(x.double(), s["router"].double().t())
    score = torch.sigmoid(logits) if case["score"] == "sigmoid" else torch.softmax(logits, -1)
    rank = score if s["bias"] is None else score + s["bias"].double()
    ids = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :k]
    wt = torch.gather(score, 1, ids)
    wt = (wt / (wt.sum(-1, keepdim=True) + 1e-20)).float()
    flat = ids.reshape(-1)
    xa = x.repeat_interleave(k, 0).unsqueeze(-1)
    g = torch.bmm(_dense(s["gate"], flat), xa)
    u = torch.bmm(_dense(s["up"], flat), xa)
    y = torch.bmm(_dense(s["down"], flat), g / (1.0 + torch.exp(-g)) * u).view(T, k, -1)
    out = (y * wt.unsqueeze(-1)).sum(1)
    if s["res"] is not None:
        out = s["res"].float() + out
    return {"out": out.to(s["out"].dtype), "ids": ids.to(torch.int32), "weights": wt}


# ---- what a pass cannot do without ---------------------------------------------------
def work(case):
    b = SIZE[case["type"]]
    if case["kind"] == "norm":
        rows, n = case["rows"], case["n"]
        scales = rows * 4 if case["form"] == "row" else rows * n // 4
        return {"bytes": rows * n * (3 * b + 1) + scales + 4 * n, "flops": 7 * rows * n}
    if case["kind"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": (M + N) * (K + 4) + M * N * b * (2 if case["res"] else 1), "flops": 2 * M * N * K}
    T, H, F, E, k = (case[c] for c in ("T", "hidden", "ffn", "E", "k"))
    # the experts that T tokens of independent choice meet, on average
    met = E * (1.0 - (1.0 - k / E) ** T)
    return {"bytes": met * 3 * F * H * 18 / 32 + E * H * 4 + T * H * b * (3 if case["res"] else 2) + 8 * T * k,
            "flops": 2 * T * (3 * k * F * H + E * H)}


# ---- the same in 64 bits ----------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "norm":
        x, delta, w = (t.double() for t in _norm_inputs(case, seed))
        h = x + delta
        y = h / torch.sqrt((h * h).mean(1, keepdim=True) + _EPS) * w
        if case["form"] == "row":
            sc = y.abs().max(1, keepdim=True).values / 127
            return {"h": h, "scales": sc[:, 0], "values": torch.round(y / sc) * sc}
        y = y.reshape(case["rows"], -1, 32)
        d = y.abs().max(2, keepdim=True).values / 127
        q = torch.floor((y / d).abs() + 0.5) * torch.sign(y)
        # the scales are 16-bit numbers, one of them of a sum taken in a given order in 32 bits
        return {"h": h, "scales": None, "values": (q * d.half().double()).reshape(h.shape)}
    if case["kind"] == "gemm":
        x, sx, w, sw, res = _gemm_inputs(case, seed)
        out = torch.empty(case["M"], case["N"], dtype=torch.float64, device="cuda")
        wt = (w.double() * sw.double().unsqueeze(1)).t().contiguous()
        for i in range(0, case["M"], 2048):
            out[i:i + 2048] = (x[i:i + 2048].double() * sx[i:i + 2048].double().unsqueeze(1)) @ wt
        return {"out": out if res is None else out + res.double()}
    s = _moe_inputs(case, seed)
    x, E, k = s["x"].double(), case["E"], case["k"]
    logits = x @ s["router"].double().t().contiguous()
    if case["score"] == "sigmoid":
        p = 1 / (1 + torch.exp(-logits))
    else:
        p = torch.exp(logits - logits.max(1, keepdim=True).values)
        p = p / p.sum(1, keepdim=True)
    rank = p + (s["bias"].double() if s["bias"] is not None else 0)
    out = torch.zeros_like(x) if s["res"] is None else s["res"].double()
    order = []
    for _ in range(k):                                       # the largest that is left, the lowest index of equals
        best = torch.argmax((rank == rank.max(1, keepdim=True).values).to(torch.int32), 1)
        order.append(best)
        rank = rank.scatter(1, best.unsqueeze(1), -math.inf)
    ids = torch.stack(order, 1)
    wt = torch.gather(p, 1, ids)
    wt = wt / wt.sum(1, keepdim=True)

    def weights(q4, e):
        q, d = q4[0][e].long(), q4[1][e].double()
        return torch.stack([(q % 16) - 8, (q // 16) - 8], 2).double().mul(d[:, :, None, None]).reshape(q.shape[0], -1)

    for e in range(E):
        here = ids == e
        if here.any():
            t = here.any(1).nonzero()[:, 0]
            g, u = x[t] @ weights(s["gate"], e).t().contiguous(), x[t] @ weights(s["up"], e).t().contiguous()
            y = (g * torch.sigmoid(g) * u) @ weights(s["down"], e).t().contiguous()
            out[t] += y * (wt * here).sum(1)[t].unsqueeze(1)
    return {"out": out, "ids": None, "weights": wt}
