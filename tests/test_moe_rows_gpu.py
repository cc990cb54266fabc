"""Rows of the mixture-of-experts layer (lk_moe_q4_0) that are not like normal ones, on
the GPU: large channels, rows that are not numbers, values at the ends of the range.

Tolerances are those of test_moe_gpu.py where nothing else is said.
"""
import pytest
import torch

from ffn_util import HALF_STEP, TYPES, moe_ref, q4_pack
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


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T", [3, 5, 10, 64])
@pytest.mark.parametrize("t", TYPES)
def test_rows_that_are_not_numbers_stay_alone(lk, t, T, score):
    """A NaN or an infinity in a token makes its own row NaN; the others, which share all their
    experts with it (3 of 3 are chosen), keep their bytes, in all kinds of launch."""
    hidden, ffn, E, dt = 96, 64, 3, TYPES[t]
    x = _x(80 + T, T, hidden, dt)
    layer = _make(lk, _layer(81, E, hidden, ffn), 3, score=score, max_tokens=T)
    clean, ids0, w0 = _run(lk, layer, x, hidden, dt, 3)
    for at, value in ((0, float("nan")), (T // 2, float("inf")), (T - 1, -float("inf"))):
        bad = x.clone()
        bad[at, (at * 31) % hidden] = value
        note(f"moe row {at} of {T} with {value} {score} {t}")
        out, ids, w = _run(lk, layer, bad, hidden, dt, 3)
        rows = [i for i in range(T) if i != at]
        assert torch.equal(out[rows], clean[rows]) and torch.equal(ids[rows], ids0[rows]) and torch.equal(w[rows], w0[rows])
        assert torch.isnan(out[at]).all() and sorted(ids[at].tolist()) == [0, 1, 2]


@pytest.mark.parametrize("tokens", [1, 5, 40, 64])
def test_every_gate_and_up_weight(lk, tokens):
    """Unit vectors for every column of gate and up, as many tokens at a time: one or five and
    forty tokens that each have an expert of their own (dot products in both kinds of launch), 64
    of one expert (matrix instructions)."""
    hidden, ffn = 160, 96
    E = 1 if tokens == 64 else 40
    L = _layer(84, E, hidden, ffn)
    if E > 1:                                            # column c chooses expert c / 4
        L["router"] = (torch.arange(hidden)[None, :] // 4 == torch.arange(E)[:, None]).float()
    layer = _make(lk, L, 1, max_tokens=tokens)
    cols = torch.arange(hidden).view(40, 4).t().flatten()                # neighbours have different experts
    for c in cols.split(tokens):
        x = torch.zeros(len(c), hidden)
        x[torch.arange(len(c)), c] = 100.0
        note(f"moe unit vectors {len(c)} from {int(c[0])}")
        out, ids, _ = _run(lk, layer, x, hidden, torch.float32, 1)
        want, ids1, _ = moe_ref(x, k=1, score="sigmoid", **L)
        assert torch.equal(ids.long(), ids1)
        _close(out, want, torch.float32, (tokens, int(c[0])))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tokens,each", [(1, 1), (5, 1), (8, 2), (64, 1), (64, 2), (64, 7)])
def test_every_down_weight(lk, tokens, each, t):
    """Expert j has one row of up that is not zero, row j, and its tokens are unit vectors: h has a
    single value, and the layer's output is column j of its down weights times that, compared
    value by value.

    Tolerance: g and u are single products of 15 bits, exact.  silu takes 3 units of 2^-23 for
    the exponential and the reciprocal and 3 roundings, h times u one, h's whole number is off by
    at most 2^-23 of it, the product, its scale and the sum round 4 times: 24 of 2^-24, and the
    output's half step (outputs are 2e-4 and more, normal in fp16)."""
    hidden, ffn, dt = 96, 64, TYPES[t]
    E, e = ffn, torch.arange(ffn)
    L = _layer(90, E, hidden, ffn)
    for w in ("gate", "up"):                             # the weight that counts: 7 (of 8 zero would be left)
        qs, b, i = L[w][0], e // 32, e % 32
        qs[e, e, b, i % 16] = torch.where(i < 16, qs[e, e, b, i % 16] | 0x0F, qs[e, e, b, i % 16] | 0xF0)
    d = torch.zeros_like(L["up"][1])
    d[e, e] = L["up"][1][e, e]
    L["up"] = (L["up"][0], d)
    L["router"] = torch.zeros(E, hidden)
    L["router"][e, e] = 1.0
    layer = _make(lk, L, 1, max_tokens=tokens)
    for some in e.repeat_interleave(each).split(tokens):
        x = torch.zeros(len(some), hidden)
        x[torch.arange(len(some)), some] = 32.0
        note(f"moe down columns {int(some[0])}..{int(some[-1])}, {each} tokens each, {tokens} at a time {t}")
        out, ids, _ = _run(lk, layer, x.to(dt), hidden, dt, 1)
        want, _, _ = moe_ref(x, k=1, score="sigmoid", **L)
        assert torch.equal(ids[:, 0].long(), some) and bool((want != 0).any(1).all())
        off = (out.cpu().double() - want).abs()
        assert bool((off <= (24 * 2.0 ** -24 + (0 if t == "f32" else HALF_STEP[dt])) * want.abs()).all())


@pytest.mark.parametrize("T", [1, 5, 10, 64])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_activations_beyond_fp32(lk, t, T):
    """silu(gate . x) * (up . x) beyond fp32's range makes the token's row NaN (the formula's would be
    infinities of both signs and NaN), and no other row."""
    hidden, ffn, E, dt = 96, 64, 3, TYPES[t]
    L = _layer(82, E, hidden, ffn)
    L["router"] *= 1e-20
    layer = _make(lk, L, 3, max_tokens=T)
    x = _x(83 + T, T, hidden, dt)
    clean, ids0, _ = _run(lk, layer, x, hidden, dt, 3)
    big = x.clone()
    big[T // 2] = big[T // 2] * 1e25                     # h of 1e48
    note(f"moe activations beyond fp32 T={T} {t}")
    out, ids, w = _run(lk, layer, big, hidden, dt, 3)
    rows = [i for i in range(T) if i != T // 2]
    assert torch.isnan(out[T // 2]).all() and torch.isfinite(w).all() and sorted(ids[T // 2].tolist()) == [0, 1, 2]
    assert torch.equal(out[rows], clean[rows]) and torch.equal(ids[rows], ids0[rows])


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 12])
def test_small_activations(lk, T, t):
    """Down to 2^-100 a block of h counts: x of 2^-p, 32 weights of one each, make g and u 2^(5 - p) and
    h half their product, 2^(9 - 2 p); the output is 32 of it, exact (silu's half is off by 2^-50
    of itself)."""
    hidden = ffn = 32
    one = torch.ones(1, 32, 32, dtype=torch.int64)
    plane = (q4_pack(one), torch.ones(1, 32, 1).half())
    layer = _make(lk, {"router": torch.zeros(1, hidden), "bias": None, "gate": plane, "up": plane, "down": plane}, 1, max_tokens=T)
    for p in (50, 52, 53, 54, 55):
        note(f"moe activations of 2^{9 - 2 * p} T={T} {t}")
        out, _, _ = _run(lk, layer, torch.full((T, hidden), 2.0 ** -p).to(TYPES[t]), hidden, TYPES[t], 1)
        want = 2.0 ** (14 - 2 * p) if 9 - 2 * p >= -100 else 0.0
        assert bool((out.double().cpu() == want).all()), (p, out[0, 0].item())
