"""References of the paged-cache tests in 64 bits, with the errors that the definitions
allow, and batches of sequences over scattered pages."""
import math
import random

import torch

from ffn_util import HALF_STEP, TYPES

U = 2.0 ** -24                                  # half a step of fp32


class Batch:
    """Sequences of given lengths and new tokens over pages in random order.  Tables on the
    CPU; `width` pages a sequence at least, unneeded entries -1."""

    def __init__(self, seed, lens, news, page, width=0, spare=2, pad=0):
        rng = random.Random(seed)
        self.lens, self.news, self.page = list(lens), list(news), page
        need = [-(-(a + n) // page) for a, n in zip(lens, news)]
        self.width = max(need + [width, 1])
        self.n_pages = sum(need) + spare
        order = list(range(self.n_pages))
        rng.shuffle(order)
        self.table, at = [], 0
        for k in need:
            self.table.append(order[at:at + k] + [-1] * (self.width - k))
            at += k
        self.first = [0]
        for n in news:
            self.first.append(self.first[-1] + n)
        self.rows = self.first[-1] + pad        # rows behind the last sequence: padding

    def slot(self, b, s):
        """Row of the pools (positions of all pages in a line) of slot s of sequence b."""
        return self.table[b][s // self.page] * self.page + s % self.page

    def slots(self, b, lo, hi):
        return torch.tensor([self.slot(b, s) for s in range(lo, hi)], dtype=torch.long)

    def step(self, lk, pos=None, mask=None, max_new=0, work=None):
        i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        m = None if mask is None else torch.tensor([signed(w) for w in mask], dtype=torch.int64, device="cuda")
        return lk.PagedStep(i(self.first), i(self.lens), i(self.table).view(len(self.lens), self.width), self.rows,
                            pos=None if pos is None else i(pos), mask=m, max_new=max_new, work=work)


def signed(w):
    return w - (1 << 64) if w >> 63 else w


def tree(rng, n):
    """(parents, masks): a random tree of n tokens, each under an earlier one."""
    par = [-1] + [rng.randrange(j) for j in range(1, n)]
    masks = []
    for j, p in enumerate(par):
        masks.append((masks[p] if p >= 0 else 0) | 1 << j)
    return par, masks


def depths(par):
    d = []
    for p in par:
        d.append(d[p] + 1 if p >= 0 else 0)
    return d


def pool_type(t):
    return torch.bfloat16 if t == "bf16" else torch.float16


def pools(seed, batch, hkv, d, t, fill=None):
    """K and V pools; `fill`: value of every position that no sequence uses."""
    g = torch.Generator().manual_seed(seed)
    shape = (batch.n_pages, batch.page, hkv, d)
    k, v = (torch.randn(shape, generator=g).to(pool_type(t)) for _ in range(2))
    if fill is not None:
        used = torch.zeros(batch.n_pages * batch.page, dtype=torch.bool)
        for b, (a, n) in enumerate(zip(batch.lens, batch.news)):
            used[batch.slots(b, 0, a + n)] = True
        for x in (k, v):
            x.view(-1, hkv, d)[~used] = fill
    return k, v


# ---- append ---------------------------------------------------------------------------
def append_ref(x, w, pos, freq, rot, pairs, eps, dtype):
    """Normed and rotated heads x [rows][heads][d] in 64 bits, and how far fp32 arithmetic and
    the one rounding may be off.  The sum of squares: 16 steps and 3 additions, each off by
    half a step, so 10 steps of 1/sqrt; its estimate 1, two products, sine and cosine one
    each, the rotation's products and sum 2: below 16 half steps of |u| + |v|."""
    x = x.double()
    d = x.shape[-1]
    y = x
    if w is not None:
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    out, size = y.clone(), y.abs()
    if rot:
        a = pos.double()[:, None, None] * freq.double()
        c, s = torch.cos(a), torch.sin(a)
        lo, hi = (torch.arange(0, rot, 2), torch.arange(1, rot, 2)) if pairs else \
            (torch.arange(rot // 2), torch.arange(rot // 2, rot))
        u, v = y[..., lo], y[..., hi]
        out[..., lo], out[..., hi] = u * c - v * s, u * s + v * c
        size = size.clone()
        size[..., lo] = size[..., hi] = u.abs() + v.abs()
    tol = 16 * U * size + HALF_STEP[dtype] * out.abs() * (1 + 2.0 ** -8) + (2.0 ** -25 if dtype == torch.float16 else 0)
    return out, tol


# ---- attention ----------------------------------------------------------------------------
def attend_ref(q, k, v, sees, t, scale, cap=0.0, slopes=None, qpos=None, kpos=None):
    """One sequence's rows q [n][hq][d] over keys k, v [N][hkv][d] with sees bool [n][N]: the
    result in 64 bits, and how far the kernel's may be off.

    With weights p_j (1 + e_j) in numerator and denominator alike the result moves by
    sum p_j e_j (v_j - o) / sum p_j, at most max|e| * (A + |o|), A = sum p |v| / sum p.  e holds:
    the weight's rounding (half a step of the type; for fp32 rows, q and weights in two fp16
    parts, 2^-22 each), and what moves the exponent: the dot product's additions (32 in a
    product of the matrix cores, their sums chained: below 42 half steps of S = sum |q k| scale),
    the argument's roundings (4 half steps of the score's size, cap and bias included, and of its
    distance from the maximum) and the exponential's own (2).  The sums over keys add 16 keys a
    product, and the products and joins in order: N / 16 + 48 half steps of A.  fp16 weights below
    2^-14 of the largest have steps of 2^-24."""
    n, hq, d = q.shape
    N, hkv = k.shape[:2]
    g = hq // hkv
    qd = q.double().permute(1, 0, 2)
    kd, vd = (x.double().permute(1, 0, 2).repeat_interleave(g, 0) for x in (k, v))
    # what no row sees does not enter at all
    hid = ~sees.any(0)
    kd[:, hid], vd[:, hid] = 0, 0
    out, tol = torch.zeros(hq, n, d, dtype=torch.float64), torch.zeros(hq, n, d, dtype=torch.float64)
    for i in range(n):
        j = sees[i].nonzero()[:, 0]
        if len(j) == 0:
            continue
        prod = qd[:, i:i + 1] * kd[:, j].reshape(hq, len(j), d)
        raw = prod.sum(-1) * scale
        S = (prod.abs().sum(-1) * scale).amax(-1)
        x = cap * torch.tanh(raw / cap) if cap else raw
        size = x.abs()
        if slopes is not None:
            bias = slopes.double()[:, None] * (kpos[j] - qpos[i]).double()[None]
            x, size = x + bias, size + bias.abs()
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - top)
        z = p.sum(-1, keepdim=True)
        vj = vd[:, j]
        o = (p.unsqueeze(-1) * vj).sum(1) / z
        A = (p.unsqueeze(-1) * vj.abs()).sum(1) / z
        e = (2.0 ** -21 if t == torch.float32 else HALF_STEP[t]) + \
            U * (42 * S + 4 * size.amax(-1) + 2 * (x - top).abs().amax(-1) + 2) + (2.0 ** -22 * S if t == torch.float32 else 0)
        e = e.unsqueeze(-1)
        w = e * (A + o.abs()) + (len(j) / 16 + 48) * U * A
        if t == torch.float16:
            w = w + (2.0 ** -25 * (p < 2.0 ** -14).sum(-1, keepdim=True) / z) * vj.abs().amax(1)
        out[:, i], tol[:, i] = o, w + HALF_STEP[t] * (o.abs() + w) + (2.0 ** -25 if t == torch.float16 else 0)
    return out.permute(1, 0, 2), tol.permute(1, 0, 2)


def causal(n, have):
    s = torch.ones(n, have + n, dtype=torch.bool)
    s[:, have:] = torch.ones(n, n, dtype=torch.bool).tril()
    return s


def by_mask(masks, have):
    """Rows of words over blocks of 64 tokens: earlier blocks whole, the own one by its bits."""
    n = len(masks)
    s = torch.ones(n, have + n, dtype=torch.bool)
    for i, w in enumerate(masks):
        for j in range(n):
            s[i, have + j] = j < i // 64 * 64 or (j // 64 == i // 64 and bool(w >> (j % 64) & 1))
    return s


def layout(hq, hkv, d):
    return {"hq": hq, "hkv": hkv, "d": d}


__all__ = ["Batch", "HALF_STEP", "TYPES", "append_ref", "attend_ref", "by_mask", "causal", "depths", "layout", "math",
           "pool_type", "pools", "signed", "tree"]
