"""References of the norm, int8 product and mixture-of-experts tests, in torch on
the CPU, and views inside guarded buffers."""
import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half a step of rounding to nearest, relative to the value
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in TYPES.values()}


def guarded(rows, n, dtype, pad=0, fill=None, device="cuda"):
    """(buffer, view): a [rows][n] view with `pad` more columns and two rows around
    it in a buffer of a sentinel value."""
    if fill is None:
        fill = 77
    buf = torch.full((rows + 2, n + pad), fill, dtype=dtype, device=device)
    return buf, buf[1:rows + 1, :n]


def untouched(buf, rows, n, fill=77) -> bool:
    b = buf.cpu().clone()
    b[1:rows + 1, :n] = fill
    return bool((b == fill).all())


def bits(t: torch.Tensor) -> np.ndarray:
    t = t.detach().cpu().contiguous()
    return t.view({4: torch.int32, 2: torch.int16, 1: torch.int8}[t.element_size()]).numpy()


def same(a, b) -> bool:
    """Equal bits, every NaN like every other."""
    a, b = a.detach().cpu(), b.detach().cpu()
    n = torch.isnan(a) & torch.isnan(b)
    return bool(((a == b) | n).all())


def norm_ref(x, delta, w, eps):
    """(h, y) in fp32 with the definition's roundings, the mean square in fp64."""
    h = x.float() if delta is None else x.float() + delta.float()
    ms = h.double().square().sum(-1, keepdim=True) / h.shape[1]
    r = (1.0 / torch.sqrt(ms + float(np.float32(eps)))).float()
    r[~torch.isfinite(ms)] = float("nan")
    return h, (h * r) * w


def q8_row_ref(y):
    a = y.abs().amax(-1, keepdim=True)
    fin = torch.isfinite(a)
    some = fin & (a >= 2.0 ** -120)
    sc = torch.where(some, a / 127.0, torch.where(fin, 0.0, float("nan")))
    # a tensor over a tensor: a number over one is its reciprocal, rounded, times the number
    q = torch.where(some, torch.round(y * (torch.full_like(a, 127.0) / a)), torch.zeros_like(y))
    return q.to(torch.int8), sc[:, 0]


def gemm_ref(x, sx, w, sw, dtype, res=None):
    """The exact sum (below 2^53 in fp64), then the roundings of the definition.  An integer
    zero is +0; the product of one column in fp64 may make it -0."""
    s = (x.double() @ w.double().t()).float() + 0.0
    v = (s * sx[:, None]) * sw[None, :]
    if res is not None:
        v = res.float() + v
    return v.to(dtype)


# ---- mixture of experts -----------------------------------------------------------
def q4_planes(g, E, rows, cols, lo=0.002, hi=0.02):
    """Random Q4_0 planes (qs uint8 [E][rows][cols/32][16], d fp16 [E][rows][cols/32])."""
    qs = torch.randint(0, 256, (E, rows, cols // 32, 16), generator=g, dtype=torch.uint8)
    return qs, (lo + (hi - lo) * torch.rand(E, rows, cols // 32, generator=g)).half()


def q4_pack(w):
    """Quant bytes of integer weights -8..7, [..., cols]: element i of a block in the
    low bits of byte i, element 16 + i in its high bits."""
    n = (w + 8).reshape(*w.shape[:-1], -1, 32).to(torch.uint8)
    return n[..., :16] | (n[..., 16:] << 4)


def q4_dense(p, e):
    """One expert's weights in fp64, [rows][cols]."""
    qs, d = p[0][e], p[1][e].double()
    n = torch.cat([qs & 15, qs >> 4], -1).double() - 8
    return (n * d[..., None]).flatten(-2)


def moe_ref(x, router, bias, gate, up, down, k, score, renorm=True, scale=1.0, res=None):
    """(out, ids, weights) in fp64: choice by the score plus bias, of equals the
    lowest index, NaN last."""
    x, E = x.double(), router.shape[0]
    logit = x @ router.double().t()
    s = torch.sigmoid(logit) if score == "sigmoid" else torch.softmax(logit, -1)
    rank = logit if bias is None else s + bias.double()
    order = [sorted(range(E), key=lambda e: (not (r[e] == r[e]), -r[e] if r[e] == r[e] else 0.0, e)) for r in rank.tolist()]
    ids = torch.tensor([o[:k] for o in order])
    w = torch.gather(s, 1, ids)
    if renorm:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    w = w * scale
    out = torch.zeros_like(x) if res is None else res.double().clone()
    for e in sorted(set(ids.flatten().tolist())):
        G, U, D = (q4_dense(p, e) for p in (gate, up, down))
        for t, j in (ids == e).nonzero().tolist():
            g, u = G @ x[t], U @ x[t]
            out[t] += w[t, j] * (D @ (g * torch.sigmoid(g) * u))
    return out, ids, w
