"""Serving over a paged cache, operator by operator: the append of a step's keys and
values with the head norms and the position rotation, the attention of each sequence's
new tokens over its pages (single tokens, drafted trees, prompts), and the commit of a
tree's accepted path.  A case is a dict of plain values; `prepare` makes what a caller
holds before the call, `run` is one pass (by elementary torch operations, or by this
library where `own` is true), `exact` the same result in 64 bits.

Kinds (the "kind" of a case):
  append  q and k normed and rotated, k and v written to their sequences' pages
  attend  softmax attention of the new tokens; "form" says what those are: "one" token a
          sequence, a "tree" of drafted tokens (a row sees its ancestors), or a "run"
          (causal: a prompt, or a plain draft)
  commit  the accepted tokens of each tree moved behind their sequence's end

Every sequence b of a batch has lens[b] positions in its pages and n_b new tokens, whose
rows are first[b] .. first[b + 1] and which take the slots from lens[b] on.
"""
import math
import os
import random
import sys

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = float(torch.tensor(1e-5, dtype=torch.float32))     # the fp32 constant, as a C caller passes it
CAP = 20.0


def _lib():
    pkg = os.path.join(os.getcwd(), "lfm2-ampere_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import lk_attn
    return lk_attn


def _cache_type(case):
    return torch.bfloat16 if case["type"] == "bf16" else torch.float16


def _heads(hq, hkv, d):
    return {"Hq": hq, "Hkv": hkv, "D": d}


def listed():
    lfm = _heads(32, 8, 64)
    return [
        # one decoded token's producers: latency
        {"name": "append_1_f32", "kind": "append", "B": 1, "n": 1, "len": 389, "type": "f32", "page": 64, **lfm},
        # a batch of drafts on its way into the cache, wide heads
        {"name": "append_61x7_bf16", "kind": "append", "B": 61, "n": 7, "len": 500, "type": "bf16", "page": 16,
         **_heads(32, 8, 128)},
        # a prompt's largest chunk
        {"name": "append_2x4096_f16", "kind": "append", "B": 2, "n": 4096, "len": 512, "type": "f16", "page": 64, **lfm},
        # one sequence's token over a short context: latency
        {"name": "one_1x389_f32", "kind": "attend", "form": "one", "B": 1, "n": 1, "len": 389, "type": "f32", "page": 64,
         "cap": False, "bias": False, **lfm},
        # one sequence's token over the longest context: the cache's bytes
        {"name": "one_1x131072_f16", "kind": "attend", "form": "one", "B": 1, "n": 1, "len": 131071, "type": "f16",
         "page": 64, "cap": False, "bias": False, **lfm},
        # a server's batch, sequences of unequal length, wide heads
        {"name": "one_64x8192_bf16", "kind": "attend", "form": "one", "B": 64, "n": 1, "len": 8192, "type": "bf16",
         "page": 16, "cap": False, "bias": False, **_heads(32, 8, 128)},
        # the same with capped scores and a bias by distance, few key heads
        {"name": "one_19x5003_f16_cap_bias", "kind": "attend", "form": "one", "B": 19, "n": 1, "len": 5003,
         "type": "f16", "page": 32, "cap": True, "bias": True, **_heads(16, 2, 64)},
        # a draft of 16 tokens in a tree, checked at once
        {"name": "tree_1x16x32768_f16", "kind": "attend", "form": "tree", "B": 1, "n": 16, "len": 32768, "type": "f16",
         "page": 64, "cap": False, "bias": False, **lfm},
        # the largest trees, several sequences
        {"name": "tree_13x64x4096_bf16", "kind": "attend", "form": "tree", "B": 13, "n": 64, "len": 4096,
         "type": "bf16", "page": 64, "cap": False, "bias": False, **lfm},
        # two prompts' chunks behind a short prefix
        {"name": "run_2x4096_f16", "kind": "attend", "form": "run", "B": 2, "n": 4096, "len": 333, "type": "f16",
         "page": 64, "cap": False, "bias": False, **lfm},
        # one sequence's accepted path
        {"name": "commit_1_f16", "kind": "commit", "B": 1, "n": 16, "len": 2500, "type": "f16", "page": 64, **lfm},
        # a batch's accepted paths
        {"name": "commit_128_bf16", "kind": "commit", "B": 128, "n": 64, "len": 256, "type": "bf16", "page": 16,
         **_heads(32, 8, 128)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_LAYOUTS = [(32, 8, 64), (32, 8, 64), (32, 8, 128), (16, 16, 64), (8, 1, 128), (12, 4, 128), (20, 4, 64), (24, 6, 64),
            (7, 7, 128), (14, 2, 64), (40, 5, 128), (64, 8, 64)]


def draw(rng):
    while True:
        kind = rng.choice(["append", "attend", "attend", "attend", "commit"])
        c = {"kind": kind, "type": rng.choice(["f32", "f16", "bf16"]), "page": rng.choice([16, 16, 32, 64, 128, 256]),
             **_heads(*rng.choice(_LAYOUTS))}
        row = c["Hkv"] * c["D"] * 4                          # bytes of a position
        if kind == "append":
            c.update(B=_log(rng, 1, 128), n=_log(rng, 1, 8192), len=_log(rng, 1, 16384))
            if c["B"] * c["n"] * (c["Hq"] + 2 * c["Hkv"]) * c["D"] > 8192 * 48 * 64:
                continue
        elif kind == "commit":
            c.update(B=_log(rng, 1, 128), n=_log(rng, 2, 64), len=_log(rng, 1, 4096))
        else:
            form = rng.choice(["one", "one", "tree", "tree", "run"])
            c.update(form=form, B=_log(rng, 1, 64), n={"one": 1, "tree": _log(rng, 2, 64), "run": _log(rng, 2, 4096)}[form],
                     len=_log(rng, 1, 131072), cap=rng.random() < 0.25, bias=rng.random() < 0.25)
            # both the scores that the plain form holds and the products within the largest listed case's
            if c["B"] * c["n"] * c["Hq"] * c["D"] * (c["len"] + c["n"]) > 2 * 4096 * 2048 * 4429:
                continue
        if c["B"] * (c["len"] + c["n"]) * row <= (1 << 30 if kind == "attend" else 1 << 27):
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


def _lengths(case):
    """Positions before the step and new tokens of each sequence: the first has the most of
    both, the others from a quarter up (of a case, not of a seed: the work is the case's)."""
    rng = random.Random(case["B"] * 1000003 + case["len"] * 101 + case["n"])
    lens, news = [case["len"]], [case["n"]]
    for _ in range(case["B"] - 1):
        lens.append(rng.randint((case["len"] + 3) // 4, case["len"]))
        news.append(case["n"] if case.get("form") == "one" else rng.randint((case["n"] + 3) // 4, case["n"]))
    return lens, news


def _signed(word):
    return word - (1 << 64) if word >> 63 else word


def _batch(case, seed):
    """The step's tables on the device, and what of them a caller knows on the host: parents of
    the trees' tokens, the accepted paths."""
    rng = random.Random(seed * 7919 + 11)
    lens, news = _lengths(case)
    B, page = case["B"], case["page"]
    need = [-(-(a + n) // page) for a, n in zip(lens, news)]
    width, n_pages = max(need), sum(need) + 1
    order = list(range(n_pages))
    rng.shuffle(order)
    table, at = [[-1] * width for _ in range(B)], 0
    for b in range(B):
        table[b][:need[b]] = order[at:at + need[b]]
        at += need[b]
    first = [0]
    for n in news:
        first.append(first[-1] + n)
    parents, masks, depth, paths = [], [], [], []
    for b in range(B):
        # a tree: every token under one of those before it, more often under a late one
        par = [-1] + [max(rng.randrange(j), rng.randrange(j)) for j in range(1, news[b])]
        word, dep = [], []
        for j, p in enumerate(par):
            word.append((word[p] if p >= 0 else 0) | 1 << j if news[b] <= 64 else 0)
            dep.append(dep[p] + 1 if p >= 0 else 0)
        parents.append(par)
        masks += [_signed(w) for w in word]
        depth += [lens[b] + (d if case.get("form") == "tree" else j) for j, d in enumerate(dep)]
        # accepted: the root, then tokens of later branches (or of a plain draft's beginning)
        k = rng.randint(1, min(8, news[b]))
        later = range(k, news[b])
        paths.append(list(range(k)) if k - 1 > len(later) or rng.random() < 0.2 else [0] + sorted(rng.sample(later, k - 1)))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"lens_h": lens, "news_h": news, "first_h": first, "table_h": table, "parents": parents, "paths": paths,
            "n_pages": n_pages, "rows": first[-1], "lens": ints(lens), "first": ints(first), "table": ints(table),
            "pos": ints(depth), "mask": torch.tensor(masks, dtype=torch.int64, device="cuda"),
            "path": ints([p + [-1] * (8 - len(p)) for p in paths]), "count": ints([len(p) for p in paths])}


def _pools(case, g, n_pages, scale=1.0):
    shape = (n_pages, case["page"], case["Hkv"], case["D"])
    k = (_randn(g, *shape) * scale).to(_cache_type(case))
    return k, _randn(g, *shape).to(_cache_type(case))


def _append_inputs(case, seed):
    g = _gen(seed, 1)
    s = _batch(case, seed)
    hq, hkv, d, rows = case["Hq"], case["Hkv"], case["D"], s["rows"]
    # the projection's rows, q | k | v side by side, channels of unequal size
    qkv = _randn(g, rows, (hq + 2 * hkv) * d) * torch.exp(0.5 * _randn(g, (hq + 2 * hkv) * d))
    s["qkv"] = qkv.to(DT[case["type"]])
    s["qn"], s["kn"] = _rand(g, 0.5, 1.5, d), _rand(g, 0.5, 1.5, d)
    s["freq"] = torch.tensor([1e7 ** (-2 * i / d) for i in range(d // 2)], dtype=torch.float64).float().cuda()
    s["k"], s["v"] = _pools(case, g, s["n_pages"])
    return s


def _attend_inputs(case, seed):
    g = _gen(seed, 2)
    s = _batch(case, seed)
    # normed and rotated queries and keys: values near 1, some keys matched well
    s["q"] = (_randn(g, s["rows"], case["Hq"] * case["D"]) * 1.5).to(DT[case["type"]])
    s["k"], s["v"] = _pools(case, g, s["n_pages"])
    s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / case["Hq"]) for h in range(case["Hq"])],
                               device="cuda") if case["bias"] else None
    return s


def _commit_inputs(case, seed):
    g = _gen(seed, 3)
    s = _batch(case, seed)
    s["k"], s["v"] = _pools(case, g, s["n_pages"])
    return s


_INPUTS = {"append": _append_inputs, "attend": _attend_inputs, "commit": _commit_inputs}


def prepare(case, seed):
    s = _INPUTS[case["kind"]](case, seed)
    s["case"] = case
    if case["kind"] == "append":
        s["q_out"] = torch.empty(s["rows"], case["Hq"] * case["D"], dtype=DT[case["type"]], device="cuda")
    elif case["kind"] == "attend":
        s["out"] = torch.empty_like(s["q"])
    else:
        s["new_lens"] = torch.empty_like(s["lens"])
    if own:                                                  # the cache's handle, and the step's tables
        lk = _lib()
        s["cache"] = lk.PagedCache(s["k"], s["v"], case["Hq"])
        tree = case["kind"] == "attend" and case["form"] == "tree"
        s["step"] = lk.PagedStep(s["first"], s["lens"], s["table"], s["rows"], pos=s["pos"] if tree else None,
                                 mask=s["mask"] if tree else None, max_new=case["n"])
    return s


# ---- one pass -----------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "commit": _own_commit}[case["kind"]](s, case)
    return {"append": _plain_append, "attend": _plain_attend, "commit": _plain_commit}[case["kind"]](s, case)


def _split(s, case):
    a, b = case["Hq"] * case["D"], (case["Hq"] + case["Hkv"]) * case["D"]
    return s["qkv"][:, :a], s["qkv"][:, a:b], s["qkv"][:, b:]


def _own_append(s, case):
    q, k, v = _split(s, case)
    s["cache"].append(s["step"], k, v, q=q, q_out=s["q_out"], qn=s["qn"], kn=s["kn"], freq=s["freq"], eps=_EPS)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _own_attend(s, case):
    s["cache"].attend(s["step"], s["q"], s["out"], cap=CAP if case["cap"] else 0.0, slopes=s["slopes"])
    return {"out": s["out"]}


def _own_commit(s, case):
    s["cache"].commit(s["step"], s["path"], s["count"], s["new_lens"])
    return {"k": s["k"], "v": s["v"], "lens": s["new_lens"]}


def _slots(s, case, seq, pos):
    """Row of the pool (positions of all pages in a line) of a position of a sequence."""
    page = case["page"]
    return s["table"][seq, torch.div(pos, page, rounding_mode="floor")].long() * page + pos % page


def _plain_append(s, case):
    rows, d = s["rows"], case["D"]
    row = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["first"], row, right=True) - 1
    pos = s["lens"][seq] + row - s["first"][seq]
    angle = pos.double()[:, None, None] * s["freq"].double()
    c, sn = torch.cos(angle).float(), torch.sin(angle).float()

    def turn(x, w):
        x = x.float().view(rows, -1, d)
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * w
        a, b = y[..., :d // 2], y[..., d // 2:]
        return torch.cat([a * c - b * sn, a * sn + b * c], -1)

    q, k, v = _split(s, case)
    slot = _slots(s, case, seq, pos)
    s["k"].view(-1, case["Hkv"], d)[slot] = turn(k, s["kn"]).to(s["k"].dtype)
    s["v"].view(-1, case["Hkv"], d)[slot] = v.float().view(rows, -1, d).to(s["v"].dtype)
    s["q_out"].copy_(turn(q, s["qn"]).view(rows, -1))
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _plain_attend(s, case):
    hq, hkv, d, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    g = hq // hkv
    bit = torch.arange(64, device="cuda")
    for b in range(case["B"]):
        n, have, r0 = s["news_h"][b], s["lens_h"][b], s["first_h"][b]
        end = have + n
        pages = s["table"][b, :-(-end // page)]
        k = s["k"][pages].view(-1, hkv, d)[:end].float().permute(1, 0, 2).contiguous()
        v = s["v"][pages].view(-1, hkv, d)[:end].float().permute(1, 0, 2).contiguous()
        pos = s["pos"][r0:r0 + n]
        kpos = torch.cat([torch.arange(have, device="cuda", dtype=torch.int32), pos])
        if case["form"] == "tree":
            sees = (s["mask"][r0:r0 + n, None] >> bit[:n]) & 1 != 0
        else:
            sees = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        some = max(1, (1 << 26) // (hkv * g * end))          # rows at a time
        for i in range(0, n, some):
            m = min(some, n - i)
            q = s["q"][r0 + i:r0 + i + m].float().view(m, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * m, d)
            x = torch.bmm(q, k.transpose(1, 2).contiguous()).view(hkv, g, m, end) * d ** -0.5
            if case["cap"]:
                x = CAP * torch.tanh(x / CAP)
            if case["bias"]:
                dist = (kpos[None, :] - pos[i:i + m, None]).float()
                x = x + s["slopes"].view(hkv, g, 1, 1) * dist
            x[..., have:].masked_fill_(~sees[i:i + m], -math.inf)
            p = torch.exp(x - x.amax(-1, keepdim=True))
            o = torch.bmm(p.view(hkv, g * m, end), v).view(hkv, g, m, d) / p.sum(-1, keepdim=True)
            s["out"][r0 + i:r0 + i + m] = o.permute(2, 0, 1, 3).reshape(m, hq * d)
    return {"out": s["out"]}


def _plain_commit(s, case):
    B = case["B"]
    seq = torch.arange(B, device="cuda")[:, None].expand(B, 8)
    j = torch.arange(8, device="cuda", dtype=torch.int32).expand(B, 8)
    live = j < s["count"][:, None]
    # a place that is not accepted moves the last accepted row onto itself once more
    j = torch.minimum(j, s["count"][:, None] - 1)
    src = _slots(s, case, seq, s["lens"][:, None] + torch.gather(s["path"], 1, j.long()))
    dst = _slots(s, case, seq, s["lens"][:, None] + j)
    for pool in (s["k"], s["v"]):
        flat = pool.view(-1, case["Hkv"], case["D"])
        flat[dst] = flat[src]
    torch.add(s["lens"], live.sum(1, dtype=torch.int32), out=s["new_lens"])
    return {"k": s["k"], "v": s["v"], "lens": s["new_lens"]}


# ---- what a pass cannot do without ---------------------------------------------------
def work(case):
    lens, news = _lengths(case)
    hq, hkv, d, b = case["Hq"], case["Hkv"], case["D"], SIZE[case["type"]]
    rows = sum(news)
    if case["kind"] == "append":
        return {"bytes": rows * d * (b * (2 * hq + 2 * hkv) + 4 * hkv), "flops": rows * (hq + hkv) * d * 8}
    if case["kind"] == "attend":
        pairs = 0
        for a, n in zip(lens, news):
            # rows of a tree see some of its tokens; a run's rows half of them
            pairs += a * n + (n if case["form"] == "one" else n * (n + 1) // 2)
        kv = sum(a + n for a, n in zip(lens, news)) * hkv * d * 4
        return {"bytes": kv + 2 * rows * hq * d * b, "flops": 4 * hq * d * pairs}
    # about three of the accepted rows of a sequence change their place
    return {"bytes": case["B"] * (3 * hkv * d * 8 + 48), "flops": 0}


# ---- the same in 64 bits ----------------------------------------------------------------
def _places(s, case, b, lo, hi):
    """Rows of the pool of the positions lo .. hi of sequence b."""
    page = case["page"]
    return torch.tensor([s["table_h"][b][p // page] * page + p % page for p in range(lo, hi)], device="cuda")


def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    hq, hkv, d = case["Hq"], case["Hkv"], case["D"]
    x = s["qkv"].double().reshape(s["rows"], hq + 2 * hkv, d)
    k, v = s["k"].double().reshape(-1, hkv, d), s["v"].double().reshape(-1, hkv, d)
    out = torch.empty(s["rows"], hq, d, dtype=torch.float64, device="cuda")
    for b in range(case["B"]):
        r0, r1, at = s["first_h"][b], s["first_h"][b + 1], s["lens_h"][b]
        head = x[r0:r1, :hq + hkv]
        head = head * torch.rsqrt(head.square().sum(-1, keepdim=True) / d + _EPS)
        head = torch.cat([head[:, :hq] * s["qn"].double(), head[:, hq:] * s["kn"].double()], 1)
        # pairs (i, i + d / 2) as complex numbers, turned by their angle
        z = torch.complex(head[..., :d // 2].contiguous(), head[..., d // 2:].contiguous())
        p = torch.arange(at, at + r1 - r0, dtype=torch.float64, device="cuda")
        a = torch.outer(p, s["freq"].double())
        z = torch.view_as_real(z * torch.polar(torch.ones_like(a), a).unsqueeze(1))
        head = torch.cat([z[..., 0], z[..., 1]], -1)
        out[r0:r1] = head[:, :hq]
        to = _places(s, case, b, at, at + r1 - r0)
        k[to], v[to] = head[:, hq:], x[r0:r1, hq + hkv:]
    return {"q": out.reshape(s["rows"], -1), "k": k.reshape(s["k"].shape), "v": v.reshape(s["v"].shape)}


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    hq, hkv, d = case["Hq"], case["Hkv"], case["D"]
    out = torch.empty(s["rows"], hq, d, dtype=torch.float64, device="cuda")
    for b in range(case["B"]):
        n, have, r0 = s["news_h"][b], s["lens_h"][b], s["first_h"][b]
        at = _places(s, case, b, 0, have + n)
        where = list(range(have)) + s["pos"][r0:r0 + n].tolist()
        where = torch.tensor(where, dtype=torch.float64, device="cuda")
        if case["form"] == "tree":
            sees = torch.zeros(n, n, dtype=torch.bool)
            for i in range(n):
                j = i
                while j >= 0:
                    sees[i, j] = True
                    j = s["parents"][b][j]
            sees = sees.cuda()
        else:
            sees = torch.arange(n, device="cuda")[:, None] >= torch.arange(n, device="cuda")
        hidden = torch.cat([torch.zeros(n, have, dtype=torch.bool, device="cuda"), ~sees], 1)
        for h in range(hq):
            k = s["k"].view(-1, hkv, d)[at, h // (hq // hkv)].double()
            v = s["v"].view(-1, hkv, d)[at, h // (hq // hkv)].double()
            x = s["q"][r0:r0 + n, h * d:(h + 1) * d].double() @ k.t().contiguous() / math.sqrt(d)
            if case["cap"]:
                x = torch.tanh(x / CAP) * CAP
            if case["bias"]:
                x = x - s["slopes"][h].double() * (where[have:, None] - where[None, :])
            out[r0:r0 + n, h] = torch.softmax(x.masked_fill(hidden, -math.inf), 1) @ v
    return {"out": out.reshape(s["rows"], -1)}


def _exact_commit(case, seed):
    s = _commit_inputs(case, seed)
    k, v = s["k"].double(), s["v"].double()
    for b in range(case["B"]):
        at, path = s["lens_h"][b], s["paths"][b]
        to = _places(s, case, b, at, at + len(path))
        for pool in (k, v):
            flat = pool.view(-1, case["Hkv"], case["D"])
            rows = [flat[_places(s, case, b, at + j, at + j + 1)[0]].clone() for j in path]
            flat[to] = torch.stack(rows)
    return {"k": k, "v": v, "lens": None}


def exact(case, seed):
    if case["kind"] == "attend" and case["B"] * case["n"] * case["Hq"] * case["D"] * (case["len"] + case["n"]) > 2e11:
        return None
    return {"append": _exact_append, "attend": _exact_attend, "commit": _exact_commit}[case["kind"]](case, seed)
