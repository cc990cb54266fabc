"""lk_paged_attn on the GPU against 64 bits: single tokens, trees, causal runs, every head
layout and type, and the places where it can go wrong.  The bound of every comparison is
derived in paged_util.attend_ref."""
import math
import random

import pytest
import torch

from gpu_util import note
from paged_util import TYPES, Batch, attend_ref, by_mask, causal, depths, pools, tree

pytestmark = pytest.mark.gpu
LAYOUTS = [(32, 8, 64), (16, 2, 64), (7, 7, 128), (8, 1, 128), (64, 8, 64), (12, 4, 128), (40, 5, 128), (33, 1, 64), (64, 1, 64),
           (96, 32, 64), (20, 4, 64), (32, 8, 128), (6, 3, 128)]


def _q(seed, rows, n, dtype, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, n, generator=g) * scale).to(dtype)


def _slopes(hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)])


def _want(batch, q, k, v, hq, t, masks, pos, scale, cap, slopes):
    """(result, bound) of the rows in 64 bits, sequence after sequence."""
    hkv, d = k.shape[2:]
    want, tol = [], []
    for b, (a, n) in enumerate(zip(batch.lens, batch.news)):
        if n == 0:
            continue
        at = batch.slots(b, 0, a + n)
        r0 = batch.first[b]
        own = torch.arange(a, a + n) if pos is None else torch.tensor(pos[r0:r0 + n])
        sees = causal(n, a) if masks is None else by_mask(masks[r0:r0 + n], a)
        w, e = attend_ref(q[r0:r0 + n].view(n, hq, d), k.view(-1, hkv, d)[at], v.view(-1, hkv, d)[at], sees, TYPES[t],
                          scale, cap, slopes, own, torch.cat([torch.arange(a), own]))
        want.append(w)
        tol.append(e)
    return torch.cat(want), torch.cat(tol)


def _check(lk, seed, batch, hq, hkv, d, t, masks=None, pos=None, cap=0.0, bias=False, scale=None, q=None, kv=None, max_new=0, fill=None,
           step=None):
    dt, rows = TYPES[t], batch.rows
    q = _q(seed, rows, hq * d, dt) if q is None else q
    k, v = pools(seed + 1, batch, hkv, d, t, fill=fill) if kv is None else kv
    slopes = _slopes(hq) if bias else None
    scale = d ** -0.5 if scale is None else scale
    qd = torch.zeros(rows, hq * d + 24, dtype=dt, device="cuda")[:, 8:hq * d + 8]
    qd.copy_(q)
    out = torch.full((rows + 2, hq * d + 16), 77.0, dtype=dt, device="cuda")
    o = out[1:rows + 1, 8:hq * d + 8]
    cache = lk.PagedCache(k.cuda(), v.cuda(), hq)
    step = batch.step(lk, pos=pos, mask=masks, max_new=max_new) if step is None else step
    note(f"attend {hq}/{hkv}/{d} {t} lens {batch.lens[:6]} news {batch.news[:6]} page {batch.page} cap {cap} bias {bias} hint {max_new}")
    cache.attend(step, qd, o, scale=scale, cap=cap, slopes=None if slopes is None else slopes.cuda())
    torch.cuda.synchronize()
    used = batch.first[-1]
    got = o[:used].cpu().double().view(used, hq, d)
    want, tol = _want(batch, q, k, v, hq, t, masks, pos, float(torch.tensor(scale, dtype=torch.float32)),
                      float(torch.tensor(cap, dtype=torch.float32)), slopes)
    off = (got - want).abs()
    bad = ~(off <= tol) & ~(torch.isnan(got) & torch.isnan(want)) & ~(got == want)
    assert not bool(bad.any()), (bad.nonzero()[:4].tolist(), (off / tol)[bad].max().item())
    assert bool((o[used:] == 77).all())
    guard = out.clone()
    guard[1:rows + 1, 8:hq * d + 8] = 77
    assert bool((guard == 77).all())
    return o[:used].clone()


def _trees(seed, news, lens):
    rng, masks, pos = random.Random(seed), [], []
    for n, a in zip(news, lens):
        par, m = tree(rng, n) if n else ([], [])
        masks += m
        pos += [a + x for x in depths(par)]
    return masks, pos


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
def test_single_tokens(lk, hq, hkv, d, t):
    _check(lk, hq + d, Batch(hq, [389, 0, 16, 700, 1], [1] * 5, 16, pad=2), hq, hkv, d, t, max_new=1)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
def test_trees(lk, hq, hkv, d, t):
    news, lens = [64, 1, 17, 0, 40], [100, 3, 0, 50, 333]
    masks, pos = _trees(hq, news, lens)
    _check(lk, hq + d, Batch(d, lens, news, 32, pad=3), hq, hkv, d, t, masks=masks + [0] * 3, pos=pos + [0] * 3, max_new=64)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
def test_runs(lk, hq, hkv, d, t):
    _check(lk, hq + d, Batch(d, [0, 37, 64], [130, 65, 5], 64, pad=1), hq, hkv, d, t, max_new=130)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9, 13, 16, 21, 32, 33, 63, 64])
@pytest.mark.parametrize("hq,hkv,d,t", [(32, 8, 64, "f16"), (15, 3, 128, "bf16"), (14, 2, 64, "f32")])
def test_every_number_of_new_tokens(lk, hq, hkv, d, t, n):
    """All shapes of workgroups."""
    lens = [250, 31, 90]
    masks, pos = _trees(n, [n] * 3, lens)
    _check(lk, n, Batch(n, lens, [n] * 3, 16), hq, hkv, d, t, masks=masks, pos=pos, max_new=n)
    _check(lk, n, Batch(n, lens, [n] * 3, 16), hq, hkv, d, t, max_new=n)


@pytest.mark.parametrize("hq,hkv,d,t", [(2, 2, 64, "f16"), (2, 2, 64, "f32"), (2, 2, 128, "bf16"), (8, 1, 64, "f32")])
def test_runs_of_many_chunks(lk, hq, hkv, d, t):
    """Beyond a thousand new tokens a wave holds more columns."""
    _check(lk, hq + d, Batch(d, [30, 0], [1030, 9], 64), hq, hkv, d, t, max_new=1030)


@pytest.mark.parametrize("cap,bias", [(20.0, False), (0.0, True), (5.0, True), (0.25, False)])
@pytest.mark.parametrize("hq,hkv,d,t", [(32, 8, 64, "f16"), (12, 4, 128, "bf16"), (16, 2, 64, "f32"), (8, 1, 128, "f32")])
def test_capped_and_biased_scores(lk, hq, hkv, d, t, cap, bias):
    lens, news = [300, 0, 77], [20, 64, 1]
    masks, pos = _trees(3, news, lens)
    _check(lk, 1, Batch(1, lens, news, 16), hq, hkv, d, t, masks=masks, pos=pos, cap=cap, bias=bias, max_new=64)
    _check(lk, 2, Batch(2, [500, 40], [1, 1], 16), hq, hkv, d, t, cap=cap, bias=bias, max_new=1)
    _check(lk, 3, Batch(3, [5, 40], [150, 70], 16), hq, hkv, d, t, cap=cap, bias=bias, max_new=150)


def test_biased_scores_at_given_positions_of_long_runs(lk):
    """Positions of new tokens beyond the first 64 come from the step too."""
    news = [150, 3]
    pos = [1000 + 3 * i for i in range(150)] + [7, 900, 8]
    _check(lk, 4, Batch(4, [33, 20], news, 16), 8, 2, 64, "f32", pos=pos, bias=True, max_new=150)


@pytest.mark.parametrize("hint", [0, 1, 3, 16, 64, 5000])
def test_the_hint_changes_no_result(lk, hint):
    """max_new chooses a kernel; any value is right."""
    lens, news = [100, 0, 9], [70, 1, 33]
    for t in ("f32", "bf16"):
        _check(lk, 5, Batch(5, lens, news, 16), 12, 4, 64, t, max_new=hint)
        masks, pos = _trees(5, [64, 1, 33], lens)
        _check(lk, 6, Batch(6, lens, [64, 1, 33], 16), 12, 4, 64, t, masks=masks, pos=pos, max_new=hint)


@pytest.mark.parametrize("B", [63, 64, 65, 200, 1000])
def test_many_sequences(lk, B):
    rng = random.Random(B)
    lens = [rng.choice([0, 1, 15, 16, 17, 40, 100]) for _ in range(B)]
    news = [rng.choice([0, 1, 1, 2]) for _ in range(B)]
    news[-1] = 1
    _check(lk, B, Batch(B, lens, news, 16, width=9, pad=5), 4, 2, 64, "f16", max_new=2)


@pytest.mark.parametrize("page", [16, 64, 256, 65536])
def test_page_sizes(lk, page):
    _check(lk, page, Batch(page, [300, 17], [1, 40], page, spare=1), 8, 2, 64, "f16")


def test_masks_over_blocks_of_64(lk):
    """More than 64 rows with words: earlier blocks are seen whole, the own one by its bits."""
    rng, n = random.Random(9), 150
    masks = [rng.getrandbits(64) | 1 << (i % 64) for i in range(n)]
    for t in ("f16", "f32"):
        _check(lk, 9, Batch(9, [45], [n], 16), 8, 2, 64, t, masks=masks, max_new=64)


def test_rows_that_see_nothing_are_zero(lk):
    """No positions before and an empty word; with positions before, those alone."""
    masks = [0, 1, 0, 1 << 3 | 1, 0, 2]
    b = Batch(10, [0, 20], [4, 2], 16)
    for t in ("f32", "f16", "bf16"):
        for d, hq, hkv in ((64, 8, 2), (128, 3, 1)):
            for hint in (1, 64):
                o = _check(lk, 10, b, hq, hkv, d, t, masks=masks, max_new=hint)
                assert bool((o[0] == 0).all()) and bool((o[2] == 0).all()) and not bool((o[1] == 0).all())


def test_bits_past_the_tokens_do_not_count(lk):
    """Words with all bits set, among them those of tokens that the sequence does not have."""
    masks = [(1 << 64) - 1] * 7
    b = Batch(11, [10, 3], [5, 2], 16, spare=4)
    k, v = pools(11, b, 2, 64, "f16", fill=float("nan"))
    _check(lk, 11, b, 8, 2, 64, "f16", masks=masks, kv=(k, v), max_new=64)
    _check(lk, 11, b, 8, 2, 64, "f16", masks=masks, kv=(k, v), max_new=1)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), 6e4])
def test_stale_positions_do_not_count(lk, t, fill):
    """Whatever lies behind the last token, in its page and in pages nobody has."""
    for d, hq, hkv in ((64, 32, 8), (128, 8, 4)):
        _check(lk, 12, Batch(12, [0, 1, 15, 16, 100, 250], [1, 1, 1, 1, 1, 1], 64), hq, hkv, d, t, fill=fill, max_new=1)
        _check(lk, 13, Batch(13, [0, 13, 100], [70, 5, 20], 64), hq, hkv, d, t, fill=fill, max_new=64)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_what_a_row_does_not_see_does_not_touch_it(lk, t, value):
    """A token whose key, or one value, is not a number spoils its own descendants and no other row."""
    n, lens = 40, [20, 77]
    masks, pos = _trees(20, [n, n], lens)
    for d, hq, hkv in ((64, 8, 2), (128, 4, 2)):
        b = Batch(20, lens, [n, n], 16)
        for which in ("key", "value"):
            k, v = pools(21, b, hkv, d, t)
            at, hit = b.slot(0, lens[0] + 7), 7
            if which == "key":
                k.view(-1, hkv, d)[at, 0] = value
            else:
                v.view(-1, hkv, d)[at, :, 5] = value
            q = _q(22, 2 * n, hq * d, TYPES[t])
            for hint in (4, 64):
                step = b.step(lk, pos=pos, mask=masks, max_new=hint)
                out = torch.empty(2 * n, hq * d, dtype=TYPES[t], device="cuda")
                note(f"a {which} of {value}, {t}, {hq}/{hkv}/{d}, hint {hint}")
                lk.PagedCache(k.cuda(), v.cuda(), hq).attend(step, q.cuda(), out)
                torch.cuda.synchronize()
                got = out.cpu().double().view(2 * n, hq, d)
                clean_k, clean_v = k.clone(), v.clone()
                clean_k.view(-1, hkv, d)[at], clean_v.view(-1, hkv, d)[at] = 0, 0
                want, tol = _want(b, q, clean_k, clean_v, hq, t, masks, None, d ** -0.5, 0.0, None)
                sees = torch.tensor([i < n and bool(masks[i] >> hit & 1) for i in range(2 * n)])
                assert bool(((got - want).abs() <= tol)[~sees].all())
                assert sees.any()
                if which == "value":
                    assert not bool(torch.isfinite(got[sees][:, :, 5]).any())
                    other = [c for c in range(d) if c != 5]
                    assert bool(torch.isfinite(got[sees][:, :, other]).all())
                elif value != value:
                    assert not bool(torch.isfinite(got[sees][:, :hq // hkv]).any())


def test_pages_that_are_not_there_count_as_zeros(lk):
    """Entries of the table outside the pool are not read; the other sequences do not notice."""
    b = Batch(30, [100, 40, 90], [1, 17, 1], 16)
    k, v = pools(31, b, 2, 64, "f16")
    q = _q(32, b.rows, 8 * 64, torch.float16)
    b.table[0][2], b.table[0][4], b.table[2][0] = -1, b.n_pages, 2 ** 31 - 1
    for hint in (1, 64):
        step = b.step(lk, max_new=hint)
        out = torch.empty(b.rows, 512, dtype=torch.float16, device="cuda")
        note(f"pages outside the pool, hint {hint}")
        lk.PagedCache(k.cuda(), v.cuda(), 8).attend(step, q.cuda(), out)
        torch.cuda.synchronize()
        good = Batch(30, [100, 40, 90], [1, 17, 1], 16)
        zero_k, zero_v = (torch.cat([x, torch.zeros(1, 16, 2, 64, dtype=x.dtype)]) for x in (k, v))
        good.table[0][2] = good.table[0][4] = good.table[2][0] = good.n_pages
        want, tol = _want(good, q, zero_k, zero_v, 8, "f16", None, None, 0.125, 0.0, None)
        assert bool(((out.cpu().double().view(-1, 8, 64) - want).abs() <= tol).all())


def test_lengths_and_bounds_out_of_range(lk):
    """A length past the table counts as the table's, one below zero as none; a sequence whose bounds
    decrease has no rows."""
    b = Batch(33, [64, 64], [0, 0], 16)
    k, v = pools(34, b, 2, 64, "f16")
    q = _q(35, 6, 256, torch.float16)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for lens, first, who in (([2 ** 31 - 1, -5], [0, 3, 3], 0), ([64, 2 ** 31 - 1], [3, 1, 4], 1)):
        step = lk.PagedStep(i(first), i(lens), i(b.table), 6)
        out = torch.full((6, 256), 77.0, dtype=torch.float16, device="cuda")
        note(f"lens {lens}, first {first}")
        lk.PagedCache(k.cuda(), v.cuda(), 4).attend(step, q.cuda(), out)
        torch.cuda.synchronize()
        r0, n = (0, 3) if who == 0 else (1, 3)
        at = b.slots(who, 0, 64)                              # the new tokens have no slots: the 64 positions alone
        want, tol = attend_ref(q[r0:r0 + n].view(n, 4, 64), k.view(-1, 2, 64)[at], v.view(-1, 2, 64)[at],
                               torch.ones(n, 64, dtype=torch.bool), torch.float16, 0.125)
        got = out.cpu().double().view(6, 4, 64)
        assert bool(((got[r0:r0 + n] - want).abs() <= tol).all())
        rest = [r for r in range(6) if not r0 <= r < r0 + n]
        assert bool((got[rest] == 77).all())


def test_queries_past_the_range_of_fp16(lk):
    """fp32 rows: a head of large queries is scaled and its scores scaled back."""
    b = Batch(40, [50, 200], [3, 1], 16)
    for d, hq, hkv in ((64, 8, 2), (128, 4, 4)):
        q = _q(41, b.rows, hq * d, torch.float32)
        q[0, :d] *= 1e6
        q[1, d:2 * d] *= 4e4
        q[2, :d] *= 1e-6
        k, v = pools(42, b, hkv, d, "f32")
        k = k * 1e-3
        for hint in (1, 64):
            _check(lk, 43, b, hq, hkv, d, "f32", q=q, kv=(k.half(), v), max_new=hint)


@pytest.mark.parametrize("shift", [-50, -20, 20])
def test_fp32_queries_of_any_size(lk, shift):
    """A power of two moved from the scale to the queries leaves every bit as it was."""
    b = Batch(46, [50, 200, 700], [3, 20, 1], 16)
    for d, hq, hkv in ((64, 8, 2), (128, 4, 4)):
        q, kv = _q(47, b.rows, hq * d, torch.float32), pools(48, b, hkv, d, "f32")
        for hint in (1, 64):
            for cap in (0.0, 8.0):
                want = _check(lk, 49, b, hq, hkv, d, "f32", q=q, kv=kv, max_new=hint, scale=0.25, cap=cap)
                got = _check(lk, 49, b, hq, hkv, d, "f32", q=q * 2.0 ** shift, kv=kv, max_new=hint, scale=0.25 * 2.0 ** -shift, cap=cap)
                assert torch.equal(got, want)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_many_small_weights_beside_a_large_one(lk, d, t):
    """3000 keys of weight 2^-14 of the first one's, whose values lie on the other side."""
    b = Batch(50, [3000], [1], 16)
    k, v = torch.zeros(b.n_pages, 16, 2, d, dtype=pools(1, b, 2, d, t)[0].dtype), None
    v = torch.full_like(k, -1.0)
    at = b.slots(0, 0, 3001)
    k.view(-1, 2, d)[at[0], :, 0] = 14 * math.log(2.0)
    v.view(-1, 2, d)[at[0]] = 1.0
    q = torch.zeros(b.rows, 4 * d, dtype=TYPES[t])
    q.view(-1, 4, d)[:, :, 0] = 1.0
    k.view(-1, 2, d)[at[1:], :, 1] = torch.linspace(-0.2, 0.2, 3000)[:, None].to(k.dtype)
    q.view(-1, 4, d)[:, :, 1] = 1.0
    for hint in (1, 64):
        _check(lk, 51, b, 4, 2, d, t, q=q, kv=(k, v), scale=1.0, max_new=hint)


@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_scores_of_many_millions(lk, t, up):
    """The key of the largest score is all of the row: the next one is 2^18 below."""
    for d, page in ((64, 16), (128, 64)):
        b = Batch(55, [1500, 900], [1, 20], page)
        k, v = pools(56, b, 2, d, t)
        k.zero_()
        for s, n in enumerate((1501, 920)):
            at = b.slots(s, 0, n)
            steps = torch.arange(n)[:, None] % 250
            k.view(-1, 2, d)[at, :, 0] = (128.0 * (steps if up else 250 - steps)).to(k.dtype)
        q = torch.zeros(b.rows, 4, d, dtype=TYPES[t])
        q[:, :, 0] = 2048.0
        for hint in (1, 64):
            out = torch.empty(b.rows, 4 * d, dtype=TYPES[t], device="cuda")
            note(f"scores to 2^26 {t} {d} up {up} hint {hint}")
            lk.PagedCache(k.cuda(), v.cuda(), 4).attend(b.step(lk, max_new=hint), q.cuda().view(b.rows, -1), out, scale=1.0)
            torch.cuda.synchronize()
            got = out.cpu().double().view(-1, 4, d)
            assert bool(torch.isfinite(got).all())
            for r in range(21):
                s, n = (0, 1501) if r == 0 else (1, 901 + r - 1)
                at = b.slots(s, 0, n)
                top = k.view(-1, 2, d)[at, 0, 0].double()
                rows = v.view(-1, 2, d)[at[top == top.max()]].double().repeat_interleave(2, 1)
                # equal weights: their common rounding cancels, the sums and the one rounding stay
                assert bool(((got[r] - rows.mean(0)).abs() <= 2.0 ** -18 * rows.abs().amax(0) +
                             torch.finfo(TYPES[t]).eps * rows.mean(0).abs()).all())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_outputs_over_the_queries(lk, t):
    for lens, news in (([300, 0, 5000], [1, 1, 1]), ([40, 0, 900], [20, 3, 64]), ([0, 30], [200, 65])):
        b = Batch(52, lens, news, 16)
        k, v = pools(53, b, 2, 64, t)
        q = _q(54, b.rows, 512, TYPES[t]).cuda()
        cache, step, out = lk.PagedCache(k.cuda(), v.cuda(), 8), b.step(lk, max_new=max(news)), torch.empty_like(q)
        cache.attend(step, q, out)
        cache.attend(step, q, q)
        torch.cuda.synchronize()
        assert torch.equal(q, out)


def test_scores_that_grow_along_the_keys(lk):
    """The running maximum is raised again and again, in every piece."""
    for t in ("f32", "f16", "bf16"):
        b = Batch(44, [900], [40], 16)
        k, v = pools(45, b, 2, 64, t)
        at = b.slots(0, 0, 940)
        ramp = torch.linspace(0.0, 6.0, 940)[:, None, None]
        flat = k.view(-1, 2, 64)
        flat[at] = (flat[at].float() * 0.2 + ramp).to(k.dtype)
        q = (_q(46, 40, 8 * 64, TYPES[t], 0.3).float() + 0.4).to(TYPES[t])
        for hint in (1, 64):
            _check(lk, 47, b, 8, 2, 64, t, q=q, kv=(k, v), max_new=hint)


@pytest.mark.parametrize("lens,news,hq,hkv,d,t", [([20000], [1], 32, 8, 64, "f16"), ([9000, 3000], [1, 1], 16, 4, 128, "bf16"),
                                                  ([7000], [16], 32, 8, 64, "f16"), ([2500], [64], 8, 2, 128, "f16"),
                                                  ([3000], [200], 4, 1, 64, "bf16"), ([6000, 1, 5], [1, 1, 1], 8, 8, 64, "f32")])
def test_long_contexts(lk, lens, news, hq, hkv, d, t):
    """Items in many pieces."""
    b = Batch(50, lens, news, 64)
    _check(lk, 51, b, hq, hkv, d, t, max_new=max(news))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_rows_at_any_alignment_and_wide_tables(lk, t):
    """Rows that begin at odd elements and lie an odd number apart; a table that is a part of a wider one."""
    b = Batch(55, [100, 33], [1, 20], 16, pad=2)
    dt = TYPES[t]
    k, v = pools(56, b, 2, 64, t)
    q = _q(57, b.rows, 512, dt)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    wide = torch.full((2, b.width + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:b.width + 2] = i(b.table)
    for hint in (1, 64):
        step = lk.PagedStep(i(b.first), i(b.lens), wide[:, 2:b.width + 2], b.rows, max_new=hint)
        qd = torch.zeros(b.rows, 517, dtype=dt, device="cuda")[:, 1:513]
        qd.copy_(q)
        out = torch.full((b.rows, 519), 77.0, dtype=dt, device="cuda")
        note(f"odd rows {t}, hint {hint}")
        lk.PagedCache(k.cuda(), v.cuda(), 8).attend(step, qd, out[:, 3:515])
        torch.cuda.synchronize()
        want, tol = _want(b, q, k, v, 8, t, None, None, 0.125, 0.0, None)
        got = out.cpu().double()
        assert bool(((got[:21, 3:515].view(21, 8, 64) - want).abs() <= tol).all())
        got[:21, 3:515] = 77
        assert bool((got == 77).all())


def test_a_workspace_that_grows(lk):
    """One step with caches of different needs: the larger workspace replaces the smaller, whose memory
    a captured call may still use."""
    b = Batch(58, [700, 33], [1, 1], 16)
    step = b.step(lk, max_new=1)
    outs = []
    for hq, hkv, d in ((8, 8, 64), (64, 8, 64), (8, 8, 64)):
        k, v = (x.cuda() for x in pools(59, b, hkv, d, "f16"))
        q = _q(60, 2, hq * d, torch.float16).cuda()
        out = torch.empty_like(q)
        note(f"workspace of {hq} heads")
        lk.PagedCache(k, v, hq).attend(step, q, out)
        outs.append(out)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[2]) and len(step._old) <= 2


def test_runs_are_the_same_bits(lk):
    """No atomics: every call gives the same bits, whatever the workspace held before."""
    b = Batch(60, [3000, 100, 700], [1, 30, 5], 16)
    k, v = (x.cuda() for x in pools(61, b, 8, 64, "f16"))
    q = _q(62, b.rows, 32 * 64, torch.float16).cuda()
    cache = lk.PagedCache(k, v, 32)
    for hint in (1, 64):
        work = torch.full((cache.work_bytes(torch.float16, hint),), 255, dtype=torch.uint8, device="cuda")     # NaN everywhere
        step = b.step(lk, max_new=hint, work=work)
        first = torch.empty_like(q)
        note(f"the same bits, hint {hint}")
        cache.attend(step, q, first)
        for _ in range(3):
            out = torch.empty_like(q)
            cache.attend(step, q, out)
            assert torch.equal(out.view(torch.int16), first.view(torch.int16))


def test_the_mirror_refuses(lk):
    b = Batch(63, [10], [2], 16)
    k, v = (x.cuda() for x in pools(64, b, 2, 64, "f16"))
    cache, step = lk.PagedCache(k, v, 4), b.step(lk)
    q = torch.zeros(2, 256, dtype=torch.float16, device="cuda")
    for call, word in ((lambda: cache.attend(step, q[:, :255], q), "q"), (lambda: cache.attend(step, q, q.float()), "out"),
                       (lambda: cache.attend(step, q[:1], q[:1]), "q"), (lambda: cache.attend(step, q, q, slopes=torch.ones(4)), "slopes"),
                       (lambda: cache.append(step, q[:, :128], q[:, :64]), "v"), (lambda: cache.attend(step, q.cpu(), q), "device"),
                       (lambda: cache.append(step, q[:, :128], q[:, 128:], kn=torch.ones(32, device="cuda")), "kn"),
                       (lambda: cache.commit(step, None, torch.zeros(2, dtype=torch.int32, device="cuda"), step._keep[1]), "count"),
                       (lambda: b.step(lk, work=torch.zeros(4, device="cuda")), "work"),
                       (lambda: lk.PagedCache(k, v[:-1], 4), "v"), (lambda: lk.PagedCache(k.permute(0, 2, 1, 3), v, 4), "k")):
        with pytest.raises(ValueError, match=word):
            call()
    for call in (lambda: cache.attend(step, q.bfloat16(), q.bfloat16()), lambda: lk.PagedCache(k, v, 5).attend(step, q, q),
                 lambda: cache.attend(b.step(lk, work=torch.zeros(16, dtype=torch.uint8, device="cuda")), q, q.clone()),
                 lambda: cache.attend(step, q, q, cap=-1.0), lambda: cache.append(step, q[:, :128], q[:, 128:], q=q)):
        with pytest.raises((lk.LkError, ValueError)):
            call()
