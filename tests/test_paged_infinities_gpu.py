"""Infinities and NaN among the keys, values and queries that a row of lk_paged_attn does see, in earlier
and in new positions, against the definition in 64 bits: softmax(x) . v, in which a score of -inf has the
weight 0, one of +inf or NaN makes the row NaN, and the weight of a finite score, however small, is
above 0.  (0 times an infinity is NaN.)"""
import math

import pytest
import torch

from gpu_util import note
from paged_util import HALF_STEP, TYPES, U, Batch, causal, pools

pytestmark = pytest.mark.gpu
INF = math.inf
LOST = {"f32": 2.0 ** -21, "f16": 2.0 ** -21, "bf16": 2.0 ** -16}      # of a weight in two parts (fp32 rows: and of q)


def _row(x, S, v, t):
    """softmax(x) . v for visible scores x [N] and values v [N][d] in 64 bits, with how far finite results may be
    off: as paged_util.attend_ref, the weight's own part by LOST.  S: largest sum of |q k|, scaled."""
    d = v.shape[1]
    if len(x) == 0:
        return torch.zeros(d, dtype=torch.float64), torch.zeros(d, dtype=torch.float64)
    top = x.max()
    if bool(torch.isnan(x).any()) or not bool(torch.isfinite(top)):
        return torch.full((d,), math.nan, dtype=torch.float64), torch.zeros(d, dtype=torch.float64)
    p = torch.exp(x - top)
    fin = torch.isfinite(v)
    vf = torch.where(fin, v, 0.0)
    z = p.sum()
    o, A = (p[:, None] * vf).sum(0) / z, (p[:, None] * vf.abs()).sum(0) / z
    # nothing finite is left beside an infinity
    odd = torch.where(fin, 0.0, torch.where((x > -INF)[:, None], v, math.nan)).sum(0)
    ends = torch.isfinite(x)
    e = LOST[t] + U * (42 * S + 4 * x[ends].abs().max() + 2 * (x[ends] - top).abs().max() + 2) + 2.0 ** -22 * S
    w = e * (A + o.abs()) + (len(x) / 16 + 48) * U * A
    return torch.where(fin.all(0), o, odd), w + HALF_STEP[TYPES[t]] * (o.abs() + w) + (2.0 ** -25 if t == "f16" else 0)


def _defined(b, q, k, v, t, scale, cap=0.0, masks=None):
    hkv, d = k.shape[2:]
    hq = q.shape[1] // d
    want, tol = [], []
    for s, (a, n) in enumerate(zip(b.lens, b.news)):
        at = b.slots(s, 0, a + n)
        ks, vs = (x.view(-1, hkv, d)[at].double() for x in (k, v))
        sees = causal(n, a)
        if masks is not None:
            sees[:, a:] = torch.tensor([[bool(masks[b.first[s] + i] >> j & 1) for j in range(n)] for i in range(n)]).view(n, n)
        for i in range(n):
            for h in range(hq):
                kv = h * hkv // hq
                prod = q[b.first[s] + i].view(hq, d)[h].double() * ks[sees[i], kv]
                x = prod.sum(-1) * scale
                x = cap * torch.tanh(x / cap) if cap else x
                S = float((torch.where(torch.isfinite(prod), prod, 0.0).abs().sum(-1) * scale).max()) if len(x) else 0.0
                w, e = _row(x, S, vs[sees[i], kv], t)
                want.append(w)
                tol.append(e)
    return torch.stack(want).view(-1, hq, d), torch.stack(tol).view(-1, hq, d)


def _check(lk, what, b, q, k, v, t, hints, scale=0.25, cap=0.0, masks=None):
    """Compares finite outputs by the bound, infinities and NaN as such.  Returns the expected rows."""
    hkv, d = k.shape[2:]
    hq = q.shape[1] // d
    want, tol = _defined(b, q, k, v, t, scale, cap, masks)
    cache, qd = lk.PagedCache(k.cuda(), v.cuda(), hq), q.cuda()
    for hint in hints:
        out = torch.full((b.rows, hq * d), 77.0, dtype=TYPES[t], device="cuda")
        note(f"{what}, {t}, {hq}/{hkv}/{d}, lens {b.lens}, hint {hint}")
        cache.attend(b.step(lk, mask=masks, max_new=hint), qd, out, scale=scale, cap=cap)
        torch.cuda.synchronize()
        got = out.cpu().double().view(-1, hq, d)
        good = (torch.isnan(got) & torch.isnan(want)) | (got == want) | \
            (torch.isfinite(got) & torch.isfinite(want) & ((got - want).abs() <= tol))
        bad = (~good).nonzero()
        assert len(bad) == 0, (hint, len(bad), [(r.tolist(), got[tuple(r)].item(), want[tuple(r)].item()) for r in bad[:4]])
    return want


def _rows(seed, n, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, generator=g) * scale).to(dtype)


SHAPES = [(4, 2, 64), (4, 2, 128), (33, 1, 64)]
TINY = {"f32": 1e-30, "f16": 2.0 ** -20, "bf16": 2.0 ** -100}


def _batches():
    """(batch, hints): one token behind few and many keys, a run, a run of many chunks."""
    return ((Batch(1, [50, 900], [1, 1], 16), (1, 16, 64)), (Batch(2, [50, 300], [20, 3], 32), (1, 16, 64, 300)))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("value", [INF, -INF])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_infinite_keys(lk, hq, hkv, d, t, value, cap):
    """A key whose score is -inf counts as none, one of +inf, or a 0 against the infinity, makes the row NaN; capped
    scores are plus or minus the cap.  The query's value may be as small as the type has any."""
    for b, hints in _batches():
        for where in ("first", "late", "new"):
            k, v = pools(3, b, hkv, d, t)
            for s in range(2):
                at = {"first": 7, "late": b.lens[s] - 2, "new": b.lens[s]}[where]
                k.view(-1, hkv, d)[b.slot(s, at), 0, 3] = value
            q = _rows(4, b.rows * hq * d, TYPES[t]).view(b.rows, hq * d)
            heads = q.view(b.rows, hq, d)
            heads[:, :, 3] = torch.where(heads[:, :, 3] >= 0, 0.5, -0.5)
            heads[0, 1, 3], heads[-1, 0, 3], heads[-1, -1, 3] = 0.0, TINY[t], -TINY[t]
            want = _check(lk, f"a {where} key of {value}, cap {cap}", b, q, k, v, t, hints, cap=cap)
            assert bool(torch.isfinite(want).all(-1).any()) and bool(torch.isnan(want).any())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("value", [INF, -INF, math.nan])
def test_queries_that_are_not_finite(lk, hq, hkv, d, t, value):
    """The row and head are NaN, or, capped, see every score at plus or minus the cap; no other row changes."""
    for b, hints in _batches():
        for cap in (0.0, 5.0):
            k, v = pools(5, b, hkv, d, t)
            q = _rows(6, b.rows * hq * d, TYPES[t]).view(b.rows, hq * d)
            q.view(b.rows, hq, d)[0, 0, 9] = value
            q.view(b.rows, hq, d)[0, 0, 10] = 6e4 if t == "f16" else 1e30
            if cap:
                k.view(-1, hkv, d)[:, :, 9] = torch.where(k.view(-1, hkv, d)[:, :, 9] >= 0, 0.5, -0.5).to(k.dtype)
            _check(lk, f"a query of {value}, cap {cap}", b, q, k, v, t, hints, cap=cap)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_rows_whose_scores_are_all_minus_infinity(lk, hq, hkv, d, t):
    """No number, as the quotient of two sums of 0 is, however the keys are divided among workgroups; beside
    it a row that sees nothing is zeros."""
    for lens, news, hints in (([50, 900], [1, 1], (1, 64)), ([40000], [1], (1, 64)), ([0, 300], [20, 3], (1, 16, 64, 300))):
        b = Batch(7, lens, news, 16)
        k, v = pools(8, b, hkv, d, t)
        k.view(-1, hkv, d)[:, :, 3] = -INF
        q = _rows(9, b.rows * hq * d, TYPES[t]).view(b.rows, hq * d)
        heads = q.view(b.rows, hq, d)
        heads[:, :, 3] = heads[:, :, 3].abs() + 0.5
        heads[0, 0, 3] = -1.0                                   # scores of +inf
        # of the run of 20 rows, 4 see nothing and one a key that is finite
        masks = [0 if i % 5 == 0 else 1 << i for i in range(b.rows)] if lens[0] == 0 else None
        if masks:
            k.view(-1, hkv, d)[b.slot(0, 6), :, 3] = 1.0
        want = _check(lk, "scores of -inf", b, q, k, v, t, hints, masks=masks)
        if masks:
            assert bool((want[[0, 5, 10, 15]] == 0).all()) and bool(torch.isfinite(want[6]).all())
            assert bool(torch.isnan(want[[1, 2, 3, 4, 7]]).all())
        else:
            assert bool(torch.isnan(want).all())


def _spoiled(b, v, s, at, dims, value):
    v.view(-1, *v.shape[2:])[b.slot(s, at), 0, dims] = value


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("lens,news,hints", [([50, 900], [1, 1], (1, 64)), ([50, 300], [20, 3], (1, 16, 64, 300)), ([40000], [1], (1, 64)),
                                             ([200] * 40, [1] * 40, (1,)), ([60] * 30, [9] * 30, (16,)), ([5000], [130], (130,))])
def test_infinite_values(lk, hq, hkv, d, t, lens, news, hints):
    """Each dim of the output is the sum of the infinities and NaN that the row sees there, in earlier and in new
    positions, alone or several; the other dims, heads and rows do not notice."""
    if sum(lens) * hq > 400000:
        hq, hkv = 2, 1
    b = Batch(11, lens, news, 16)
    k, v = pools(12, b, hkv, d, t)
    for s in range(0, len(lens), 3):
        a, n = lens[s], news[s]
        _spoiled(b, v, s, 7, 5, INF)
        _spoiled(b, v, s, a - 1, 6, -INF)
        _spoiled(b, v, s, a, 17, INF)                           # a new token
        _spoiled(b, v, s, a + n - 1, 18, -INF)                  # the last one: of a run its own row alone sees it
        _spoiled(b, v, s, 20, 33, math.nan)
        _spoiled(b, v, s, a // 2, 34, INF)                      # two of one sign, two of both
        _spoiled(b, v, s, a // 2 + 9, 34, INF)
        _spoiled(b, v, s, a // 2, 63, INF)
        _spoiled(b, v, s, a // 2 + 9, 63, -INF)
        _spoiled(b, v, s, 30, [0, d - 1], 1e30 if t == "bf16" else 6e4)
    q = _rows(13, b.rows * hq * d, TYPES[t]).view(b.rows, hq * d)
    want = _check(lk, "infinite values", b, q, k, v, t, hints)
    assert bool((want[0, 0, [5, 34]] == INF).all()) and float(want[0, 0, 6]) == -INF and math.isnan(float(want[0, 0, 33]))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("gap", [12.0, 80.0, 400.0])
def test_infinite_values_of_small_weights(lk, hq, hkv, d, t, gap):
    """A weight e^-gap of the largest, far below what its type or fp32 holds, is above 0: its infinity counts.  One of a
    score of -inf makes the dim NaN."""
    for lens, news, hints in (([50, 900], [1, 1], (1, 64)), ([50, 300], [20, 3], (1, 16, 64, 300)), ([9000], [1], (1, 64))):
        b = Batch(14, lens, news, 16)
        k, v = pools(15, b, hkv, d, t)
        flat = k.view(-1, hkv, d)
        for s in range(len(lens)):
            a, n = lens[s], news[s]
            for at, dim in ((3, 40), (a - 1, 41), (a, 42), (a // 2, 43)):
                flat[b.slot(s, at), 0, 0] = -gap
                _spoiled(b, v, s, at, dim, INF)
            if gap > 100:
                flat[b.slot(s, 30), 0, 1] = -INF
                _spoiled(b, v, s, 30, 50, -INF)
        q = _rows(16, b.rows * hq * d, TYPES[t], 0.1).view(b.rows, hq * d)
        q.view(b.rows, hq, d)[:, :, 0] = 4.0
        q.view(b.rows, hq, d)[:, :, 1] = 0.5
        want = _check(lk, f"weights of e^-{gap}", b, q, k, v, t, hints)
        assert bool((want[:, 0, [40, 41, 43]] == INF).all())
        assert gap < 100 or bool(torch.isnan(want[:, 0, 50]).all())


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_values_near_the_end_of_the_type(lk, hq, hkv, d):
    """bf16 values up to 2^125, whose weighted sums are finite: no weight is above 1."""
    for b, hints in _batches():
        k, v = pools(17, b, hkv, d, "bf16")
        v = v.float().clamp(-4, 4).mul(2.0 ** 123).bfloat16()
        q = _rows(18, b.rows * hq * d, TYPES["bf16"]).view(b.rows, hq * d)
        want = _check(lk, "large values", b, q, k, v, "bf16", hints, scale=0.25)
        assert bool(torch.isfinite(want).all())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,d", [(1, 64), (2, 64), (2, 128), (4, 64)])
def test_rows_of_nan_beside_others(lk, t, hq, d):
    """Half of the rows a wave holds are NaN; the scores of the others grow along the keys."""
    for lens, n in (([300], 64), ([2000], 130)):
        b = Batch(19, lens, [n], 16)
        k, v = pools(20, b, 1, d, t)
        at = b.slots(0, 0, lens[0] + n)
        k.view(-1, 1, d)[at, :, 0] = torch.linspace(0.0, 40.0, lens[0] + n)[:, None].to(k.dtype)
        q = _rows(21, n * hq * d, TYPES[t], 0.1).view(n, hq, d)
        q[:, :, 0] = 4.0
        for nan in (slice(0, 8), slice(8, 16), slice(0, 16), slice(0, n, 2)):
            spoiled = q.clone()
            spoiled[nan, :, 7] = math.nan
            want = _check(lk, f"NaN in rows {nan}", b, spoiled.view(n, -1), k, v, t, (1, 64, 300))
            assert int(torch.isnan(want[:, 0, 0]).sum()) == len(range(n)[nan])


@pytest.mark.parametrize("shift", [-120, -70, 100, 125])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_fp32_queries_to_the_ends_of_the_type(lk, hq, hkv, d, shift):
    """A power of two moved from the scale to the queries leaves every bit as it was, beyond 2^60 either way, and with
    an infinite key.  (By 2^-120 queries below 2^-6, by 2^125 the scale 2^-127 and its product with log2(e), are below the
    normal numbers of fp32 and have bits fewer: there the bound alone holds.)"""
    for b, hints in _batches():
        k, v = pools(22, b, hkv, d, "f32")
        q = _rows(23, b.rows * hq * d, TYPES["f32"]).clamp(-3.9, 3.9).view(b.rows, hq * d)
        for value in (1.0, -INF):
            k.view(-1, hkv, d)[b.slot(0, 9), 0, 3] = value
            _check(lk, f"queries by 2^{shift}", b, q * 2.0 ** shift, k, v, "f32", hints, scale=0.25 * 2.0 ** -shift)
            if shift in (-120, 125):
                continue
            cache, outs = lk.PagedCache(k.cuda(), v.cuda(), hq), []
            for f in (0, shift):
                outs.append(torch.empty(b.rows, hq * d, device="cuda"))
                cache.attend(b.step(lk, max_new=16), (q * 2.0 ** f).cuda(), outs[-1], scale=0.25 * 2.0 ** -f)
            torch.cuda.synchronize()
            assert torch.equal(outs[0].view(torch.int32), outs[1].view(torch.int32))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_rows_of_nan_that_see_infinite_values(lk, hq, hkv, d, t):
    """A row whose scores make it NaN stays so in every dim, the infinite values' among them; its neighbours get those."""
    for lens, news, hints in (([50, 900], [1, 1], (1, 64)), ([60] * 30, [9] * 30, (1, 16)), ([0, 300], [20, 150], (1, 16, 64, 300)),
                              ([9000], [2], (1, 64))):
        b = Batch(24, lens, news, 16)
        k, v = pools(25, b, hkv, d, t)
        q = _rows(26, b.rows * hq * d, TYPES[t]).view(b.rows, hq, d)
        for s, (a, n) in enumerate(zip(lens, news)):
            for at in {a // 2, a, a + n - 1}:
                _spoiled(b, v, s, at, [2, d - 2], INF if s % 2 else -INF)
            _spoiled(b, v, s, a + n // 2, slice(None), INF)     # all dims of one token
            q[b.first[s]:b.first[s + 1]:2, s % hq, 4] = (math.nan, INF)[s % 2]
            if s % 3 == 1:
                k.view(-1, hkv, d)[b.slot(s, a), -1, 5] = math.nan
        _check(lk, "NaN rows and infinite values", b, q.view(b.rows, -1), k, v, t, hints)
