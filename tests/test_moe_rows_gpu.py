"""Rows of the mixture-of-experts layer (lk_moe_q4_0) that are not like normal ones, on
the GPU: large channels, rows that are not numbers, values at the ends of the range.

Tolerances are those of test_moe_gpu.py where nothing else is said.
"""
import pytest
import torch

from ffn_util import TYPES, moe_ref, q4_planes
from gpu_util import note
from test_moe_gpu import _close, _layer, _make, _run, _x

pytestmark = pytest.mark.gpu


def _without(plane, cols):
    """The plane with weights of zero in the given columns."""
    qs, d = plane
    qs = qs.clone()
    for c in cols:
        b, i = c // 32, c % 32
        old = qs[:, :, b, i % 16]
        qs[:, :, b, i % 16] = old & 0xF0 | 8 if i < 16 else old & 0x0F | 0x80
    return qs, d


def _louder(plane, rows, times):
    d = plane[1].clone()
    d[:, rows] = (d[:, rows].float() * times).half()
    return plane[0], d


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T", [1, 5, 9, 64])
def test_large_channels(lk, T, t):
    """Residual streams have a few channels far above the rest, and so have activations: four
    channels of x, and four of h, about 1000 times the others, whose weights in the
    product that follows are zero, so that all that counts is what is left of their
    neighbours.

    Tolerance: a block's values are held as whole numbers whose largest is between 2^22 and
    2^23 (16-bit rows) or 2^30 and 2^31 (fp32 rows).  4 of the 16 blocks of x have a value 1000
    times the others: their 31 neighbours are off by 0.29 / 2^22.5 of it, all in all
    sqrt(4 / 16) * 1000 * 0.29 / 2^22.5 = 2.4e-5 of the row, twice as much where the four are
    twice as large; silu(g) u by up to three times that, and the down product adds as much
    again as x, for 4 of 8 blocks: 2e-4 at the most, as allowed for 16-bit rows; fp32 rows 256 times less,
    of the 1e-5."""
    hidden, ffn, E, k, dt = 512, 256, 6, 2, TYPES[t]
    L = _layer(70 + T, E, hidden, ffn)
    chan, rows = [3, 100, 317, 511], [0, 77, 140, 223]
    L["router"][:, chan] = 0.0
    L["gate"], L["up"] = (_louder(_without(L[w], chan), rows, 32.0) for w in ("gate", "up"))
    L["down"] = _without(L["down"], rows)
    x = _x(71 + T, T, hidden, torch.float32)
    x[:, chan] = 1500.0 * torch.sign(x[:, chan])
    x = x.to(dt)
    note(f"moe large channels T={T} {t}")
    out, ids, _ = _run(lk, _make(lk, L, k, max_tokens=T), x, hidden, dt, k)
    want, ids1, _ = moe_ref(x, k=k, score="sigmoid", **L)
    assert torch.equal(ids.long(), ids1)
    _close(out, want, dt, (T, t))
