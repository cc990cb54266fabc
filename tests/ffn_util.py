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
    q = torch.where(some, torch.round(y * (127.0 / a)), torch.zeros_like(y))
    return q.to(torch.int8), sc[:, 0]


def gemm_ref(x, sx, w, sw, dtype, res=None):
    """The exact sum (below 2^53 in fp64), then the roundings of the definition."""
    s = (x.double() @ w.double().t()).float()
    v = (s * sx[:, None]) * sw[None, :]
    if res is not None:
        v = res.float() + v
    return v.to(dtype)
