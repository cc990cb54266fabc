"""lk_paged_append and lk_paged_commit on the GPU: against 64 bits, every page order, style and
stride, and what they leave alone."""
import random

import pytest
import torch

from gpu_util import note
from paged_util import HALF_STEP, TYPES, Batch, append_ref, pool_type, pools

pytestmark = pytest.mark.gpu
EPS = float(torch.tensor(1e-5, dtype=torch.float32))
LAYOUTS = [(32, 8, 64), (16, 2, 64), (7, 7, 128), (8, 1, 128), (64, 8, 64), (24, 3, 128), (256, 32, 64)]


def _rows(seed, rows, n, dtype):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, n, generator=g) * torch.exp(0.5 * torch.randn(n, generator=g))).to(dtype)


def _freq(rot, theta=1e7):
    return torch.tensor([theta ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float64).float()


def _check(lk, seed, batch, hq, hkv, d, t, rot=None, pairs=False, norm=True, q=True, pos=None, inplace=False, extra=8, bad=()):
    """One call and its reference.  The rows are parts of wider ones; `bad`: (sequence, page index, entry)
    of the table that are not pages of the pool."""
    dt, rows = TYPES[t], batch.rows
    rot = d if rot is None else rot
    wide = _rows(seed, rows, (hq + 2 * hkv) * d + extra, dt)
    g = torch.Generator().manual_seed(seed + 1)
    qn, kn = (0.5 + torch.rand(d, generator=g) for _ in range(2))
    kp, vp = pools(seed + 2, batch, hkv, d, t)
    for b, i, e in bad:
        batch.table[b][i] = e
    step = batch.step(lk, pos=pos)
    k, v, dev = kp.cuda(), vp.cuda(), wide.cuda()
    cache = lk.PagedCache(k, v, hq)
    a, b = hq * d, (hq + hkv) * d
    part = (dev[:, :a], dev[:, a:b], dev[:, b:b + hkv * d])
    out = part[0] if inplace else torch.full((rows + 2, a + 16), 77.0, dtype=dt, device="cuda")[1:rows + 1, 8:a + 8]
    kw = dict(freq=_freq(rot).cuda() if rot else None, pairs=pairs, eps=EPS)
    if norm:
        kw.update(qn=qn.cuda(), kn=kn.cuda())
    if q:
        kw.update(q=part[0], q_out=out)
    note(f"append {hq}/{hkv}/{d} {t} rows {rows} rot {rot} pairs {pairs} norm {norm} q {q}")
    cache.append(step, part[1], part[2], **kw)
    torch.cuda.synchronize()
    seq = [(b, i) for b in range(len(batch.news)) for i in range(batch.news[b])]
    used = len(seq)
    slot = [batch.lens[b] + i for b, i in seq]
    at = torch.tensor(slot if pos is None else pos[:used], dtype=torch.int64)
    x = wide[:used, :b].view(used, hq + hkv, d)
    f = _freq(rot) if rot else None
    want_q, tol_q = append_ref(x[:, :hq], qn if norm else None, at, f, rot, pairs, EPS, dt)
    want_k, tol_k = append_ref(x[:, hq:], kn if norm else None, at, f, rot, pairs, EPS, pool_type(t))
    if q:
        got = out[:used].cpu().double().view(used, hq, d)
        assert bool(((got - want_q).abs() <= tol_q).all()), ((got - want_q).abs() / tol_q).max().item()
        if inplace:
            assert torch.equal(out[used:].cpu(), wide[used:, :a])
        else:
            assert bool((out[used:] == 77).all())
            whole = torch.as_strided(out, (rows + 2, a + 16), (a + 16, 1), out.storage_offset() - (a + 16) - 8)
            whole[1:rows + 1, 8:a + 8] = 77
            assert bool((whole == 77).all())
    # the pools: the new rows, and not a bit elsewhere
    flat_k, flat_v = kp.view(-1, hkv, d), vp.view(-1, hkv, d)
    keep = torch.ones(len(flat_k), dtype=torch.bool)
    gk, gv = k.cpu().view(-1, hkv, d), v.cpu().view(-1, hkv, d)
    for r, ((b, i), s) in enumerate(zip(seq, slot)):
        if s >= batch.width * batch.page or not 0 <= batch.table[b][s // batch.page] < batch.n_pages:
            continue
        p = batch.slot(b, s)
        keep[p] = False
        off = (gk[p].double() - want_k[r]).abs()
        assert bool((off <= tol_k[r]).all()), (r, (off / tol_k[r]).max().item())
        assert torch.equal(gv[p], wide[r, (hq + hkv) * d:(hq + 2 * hkv) * d].view(hkv, d).to(pool_type(t))), r
    assert torch.equal(gk[keep], flat_k[keep]) and torch.equal(gv[keep], flat_v[keep])


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
def test_append_layouts(lk, hq, hkv, d, t):
    _check(lk, 100 + hq, Batch(hq + d, [389, 0, 15, 16, 1000], [1, 3, 1, 17, 0], 16, pad=3), hq, hkv, d, t)


@pytest.mark.parametrize("rot,pairs,norm", [(64, True, True), (32, False, True), (32, True, False), (16, False, False), (48, True, True),
                                            (0, False, True), (0, False, False), (64, False, False)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_append_styles(lk, rot, pairs, norm, t):
    _check(lk, 200 + rot, Batch(rot, [5, 100], [9, 2], 32), 12, 4, 64, t, rot=rot, pairs=pairs, norm=norm)


@pytest.mark.parametrize("rot,pairs", [(128, True), (64, False), (112, True), (96, False)])
def test_append_styles_wide(lk, rot, pairs):
    _check(lk, 220 + rot, Batch(rot, [5, 100], [9, 2], 32), 6, 2, 128, "f16", rot=rot, pairs=pairs)


@pytest.mark.parametrize("lens,news", [([0], [1]), ([70000], [5]), ([0], [4100]), ([31, 32, 33], [700, 1, 1400]),
                                       (list(range(0, 300)), [b % 3 for b in range(300)]), ([64] * 1025, [2] * 1025)])
def test_append_batches(lk, lens, news):
    """Few rows and many (two kernels), batches of more sequences than a workgroup has lanes."""
    _check(lk, 300 + len(lens), Batch(len(lens), lens, news, 64, pad=1), 4, 2, 64, "f16", extra=0)


def test_append_rows_without_queries_and_in_place(lk):
    b = Batch(7, [10, 20], [4, 30], 16, pad=2)
    _check(lk, 400, b, 8, 2, 64, "bf16", q=False)
    _check(lk, 401, b, 8, 2, 64, "bf16", inplace=True)
    _check(lk, 402, b, 8, 2, 128, "f32", inplace=True)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_append_rows_at_any_alignment(lk, t):
    """Rows an odd number of elements apart."""
    _check(lk, 450, Batch(15, [10, 3], [4, 3000], 16, pad=1), 5, 1, 64, t, extra=7)
    _check(lk, 451, Batch(15, [10, 3], [4, 3], 16, pad=1), 5, 1, 128, t, extra=1)


def test_append_far_and_given_positions(lk):
    """Angles in 64 bits: positions far past 2^24, negative ones, and not those of the slots."""
    b = Batch(8, [10, 20], [4, 30], 16)
    _check(lk, 500, b, 8, 2, 64, "f32", pos=[2 ** 24 + 1 + 977 * i for i in range(34)])
    _check(lk, 501, b, 8, 2, 128, "f32", pos=[2 ** 30 - 3 - i for i in range(34)])
    _check(lk, 502, b, 8, 2, 64, "f16", pos=[-i for i in range(34)])


def test_append_leaves_what_the_table_does_not_name(lk):
    """Entries that are no pages of the pool, and slots past the table: not written."""
    b = Batch(9, [14, 30, 3], [20, 5, 40], 16)
    _check(lk, 600, b, 8, 2, 64, "f16", bad=[(0, 1, -1), (1, 2, b.n_pages), (2, 0, 2 ** 31 - 1), (2, 2, -2 ** 31)])
    b = Batch(10, [14, 3], [4, 4], 16)
    b.news, b.first, b.rows = [40, 4], [0, 40, 44], 44           # more tokens than the table has slots for
    _check(lk, 601, b, 8, 2, 64, "f16")


def test_append_bounds_out_of_range(lk):
    """Row bounds and lengths out of range count as the nearest in it."""
    b = Batch(11, [0, 0], [4, 4], 16)
    k, v = (x.cuda() for x in pools(1, b, 2, 64, "f16"))
    cache = lk.PagedCache(k, v, 4)
    rows = _rows(2, 8, 256, torch.float16).cuda()
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    step = lk.PagedStep(i([-5, 4, 99]), i([-7, 2 ** 31 - 1]), i(b.table), 8)
    before = k.cpu().clone()
    note("append with bounds out of range")
    cache.append(step, rows[:, :128], rows[:, 128:])
    torch.cuda.synchronize()
    got, at = k.cpu().view(-1, 2, 64), b.slots(0, 0, 4)
    assert torch.equal(got[at], rows[:4, :128].cpu().view(4, 2, 64))       # from slot 0 on
    keep = torch.ones(len(got), dtype=torch.bool)
    keep[at] = False
    assert torch.equal(got[keep], before.view(-1, 2, 64)[keep])            # the second has no slot left


# ---- commit -----------------------------------------------------------------------------
def _commit(lk, seed, batch, paths, count=None, hkv=2, d=64, t="f16", ldp=None, inplace=False, bad=()):
    kp, vp = pools(seed, batch, hkv, d, t)
    for b, i, e in bad:
        batch.table[b][i] = e
    k, v = kp.cuda(), vp.cuda()
    step = batch.step(lk)
    ldp = ldp or max([1] + [len(p) for p in paths])
    count = [len(p) for p in paths] if count is None else count
    path = torch.tensor([p + [-1] * (ldp - len(p)) for p in paths], dtype=torch.int32, device="cuda")
    lens = step._keep[1]
    new = lens if inplace else torch.full((len(paths),), -5, dtype=torch.int32, device="cuda")
    note(f"commit {len(paths)} sequences, lists of {ldp}, inplace {inplace}")
    lk.PagedCache(k, v, hkv).commit(step, path, torch.tensor(count, dtype=torch.int32, device="cuda"), new)
    torch.cuda.synchronize()
    want_k, want_v, want_len = kp.clone().view(-1, hkv, d), vp.clone().view(-1, hkv, d), []
    have = lambda b, s: s < batch.width * batch.page and 0 <= batch.table[b][s // batch.page] < batch.n_pages  # noqa: E731
    for b, p in enumerate(paths):
        took = 0
        at = batch.lens[b]
        for j in range(max(0, min(count[b], ldp))):
            i = p[j] if j < len(p) else -1
            if not 0 <= i < batch.news[b] or (j and i <= p[j - 1]) or not have(b, at + i) or not have(b, at + j):
                break
            took += 1
        src = [batch.slot(b, at + i) for i in p[:took]]
        dst = [batch.slot(b, at + j) for j in range(took)]
        for w, o in ((want_k, kp), (want_v, vp)):
            if took:
                w[dst] = o.view(-1, hkv, d)[src]
        want_len.append(at + took)
    assert new.cpu().tolist() == want_len
    assert torch.equal(k.cpu().view(-1, hkv, d), want_k) and torch.equal(v.cpu().view(-1, hkv, d), want_v)


@pytest.mark.parametrize("hkv,d,t", [(2, 64, "f16"), (8, 64, "f16"), (8, 128, "bf16"), (1, 128, "f32"), (3, 64, "bf16"), (32, 128, "f16")])
@pytest.mark.parametrize("inplace", [False, True])
def test_commit_paths(lk, hkv, d, t, inplace):
    rng = random.Random(hkv * d)
    news = [64, 1, 17, 30, 0, 64, 2]
    paths = [sorted(rng.sample(range(n), rng.randint(0, n))) for n in news]
    paths[0], paths[5] = list(range(64)), [0, 63]
    _commit(lk, 700 + hkv, Batch(hkv, [0, 5, 15, 33, 4, 100, 16], news, 16), paths, hkv=hkv, d=d, t=t, inplace=inplace)


def test_commit_lists_that_end_early(lk):
    """Not increasing, out of range, the same place twice, a count past the list or below zero."""
    b = Batch(12, [3, 14, 15, 16, 0, 7, 9], [8] * 7, 16)
    _commit(lk, 720, b, [[0, 2, 1, 5], [0, 3, 3], [4, 8], [-1, 2], [2, 5, 6], [1, 2], [0, 1]], count=[4, 3, 2, 2, 9, -3, 2 ** 31 - 1])


def test_commit_pages_that_are_missing(lk):
    b = Batch(13, [14, 30, 3], [20, 5, 40], 16)
    _commit(lk, 730, b, [[0, 1, 5, 19], [1, 3], [2, 13, 39]], bad=[(0, 1, -1), (2, 2, b.n_pages)])


@pytest.mark.parametrize("n", [1, 1000])
def test_commit_a_plain_draft(lk, n):
    """No list: the first tokens as they lie, counts up to what there is."""
    b = Batch(14, [5] * n, [7] * n, 32)
    k, v = (x.cuda() for x in pools(1, b, 2, 64, "f16"))
    old = k.clone(), v.clone()
    step, new = b.step(lk), torch.empty(n, dtype=torch.int32, device="cuda")
    count = torch.tensor([(3, -1, 9)[i % 3] for i in range(n)], dtype=torch.int32, device="cuda")
    note(f"commit without lists, {n} sequences")
    lk.PagedCache(k, v, 2).commit(step, None, count, new)
    torch.cuda.synchronize()
    assert new.cpu().tolist() == [5 + (3, 0, 7)[i % 3] for i in range(n)]
    assert torch.equal(k, old[0]) and torch.equal(v, old[1])


def test_half_steps_are_those_of_the_types():
    assert HALF_STEP[torch.float16] == 2.0 ** -11 and HALF_STEP[torch.bfloat16] == 2.0 ** -8
