"""The paged cache as a server uses it, on the GPU: prompts, single tokens and drafted trees of
several sequences, append -> attend -> commit step after step; the same captured and replayed;
on streams of its own; past 4 GiB.

Each step's attention is compared with the definition over the bytes that the pools hold
(paged_util.attend_ref), the appends and commits with a model of the pools on the host."""
import random

import pytest
import torch

from gpu_util import d_pos_for, note
from paged_util import TYPES, Batch, append_ref, attend_ref, by_mask, causal, depths, pool_type, tree, signed

pytestmark = pytest.mark.gpu
EPS = float(torch.tensor(1e-5, dtype=torch.float32))


def _i(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class _Server:
    """Sequences that grow over pages handed out as they are needed."""

    def __init__(self, lk, seed, hq, hkv, d, t, page, n_seqs, n_pages, width):
        self.lk, self.rng, self.t, self.page, self.width = lk, random.Random(seed), t, page, width
        self.hq, self.hkv, self.d = hq, hkv, d
        g = torch.Generator().manual_seed(seed)
        shape = (n_pages, page, hkv, d)
        self.k, self.v = (torch.full(shape, float("nan"), dtype=pool_type(t), device="cuda") for _ in range(2))
        self.free = list(range(n_pages))
        self.rng.shuffle(self.free)
        self.table = [[-1] * width for _ in range(n_seqs)]
        self.lens = [0] * n_seqs
        self.qn, self.kn = (0.5 + torch.rand(d, generator=g) for _ in range(2))
        self.freq = torch.tensor([1e4 ** (-2 * i / d) for i in range(d // 2)], dtype=torch.float64).float()
        self.cache = lk.PagedCache(self.k, self.v, hq)
        self.dev = {"qn": self.qn.cuda(), "kn": self.kn.cuda(), "freq": self.freq.cuda()}
        self.g = g

    def flat(self, x):
        return x.cpu().view(-1, self.hkv, self.d)

    def slots(self, b, lo, hi):
        return torch.tensor([self.table[b][s // self.page] * self.page + s % self.page for s in range(lo, hi)], dtype=torch.long)

    def step(self, news, trees=None, stream=None):
        """One step; `trees`: per sequence (parents, masks) or None for causal runs.  Returns the outputs."""
        dt, hq, hkv, d = TYPES[self.t], self.hq, self.hkv, self.d
        for b, n in enumerate(news):
            for p in range(-(-(self.lens[b] + n) // self.page)):
                if self.table[b][p] < 0:
                    self.table[b][p] = self.free.pop()
        first = [0]
        for n in news:
            first.append(first[-1] + n)
        rows = first[-1]
        masks = pos = None
        if trees:
            masks = [w for _, m in trees for w in m]
            pos = [a + x for a, (par, _) in zip(self.lens, trees) for x in depths(par)]
        step = self.lk.PagedStep(_i(first), _i(self.lens), _i(self.table), rows, pos=None if pos is None else _i(pos),
                                 mask=None if masks is None else torch.tensor([signed(w) for w in masks], device="cuda"),
                                 max_new=max(news))
        wide = torch.randn(rows, (hq + 2 * hkv) * d, generator=self.g).to(dt)
        dev = wide.cuda()
        a, e = hq * d, (hq + hkv) * d
        q = torch.empty(rows, a, dtype=dt, device="cuda")
        out = torch.empty_like(q)
        before_k, before_v = self.flat(self.k).clone(), self.flat(self.v).clone()
        torch.cuda.synchronize()
        self.cache.append(step, dev[:, a:e], dev[:, e:], q=dev[:, :a], q_out=q, eps=EPS, stream=stream, **self.dev)
        self.cache.attend(step, q, out, stream=stream)
        torch.cuda.synchronize()
        # the pools: the new rows alone
        x = wide[:, :e].view(rows, hq + hkv, d)
        at = torch.tensor(pos if pos else [s + i for s, n in zip(self.lens, news) for i in range(n)])
        want, tol = append_ref(x[:, hq:], self.kn, at, self.freq, d, False, EPS, pool_type(self.t))
        keep = torch.ones(len(before_k), dtype=torch.bool)
        k, v = self.flat(self.k), self.flat(self.v)
        for b, n in enumerate(news):
            p = self.slots(b, self.lens[b], self.lens[b] + n)
            keep[p] = False
            r = slice(first[b], first[b + 1])
            assert bool(((k[p].double() - want[r]).abs() <= tol[r]).all())
            assert torch.equal(v[p], wide[r, e:].view(n, hkv, d).to(pool_type(self.t)))
        same = lambda x, y: bool(((x == y) | (torch.isnan(x) & torch.isnan(y))).all())  # noqa: E731
        assert same(k[keep], before_k[keep]) and same(v[keep], before_v[keep])
        # the attention over what the pools hold now
        got = out.cpu().double().view(rows, hq, d)
        for b, n in enumerate(news):
            if n == 0:
                continue
            p = self.slots(b, 0, self.lens[b] + n)
            sees = by_mask(trees[b][1], self.lens[b]) if trees else causal(n, self.lens[b])
            w, e2 = attend_ref(q[first[b]:first[b + 1]].cpu().view(n, hq, d), k[p], v[p], sees, dt, d ** -0.5)
            assert bool(((got[first[b]:first[b + 1]] - w).abs() <= e2).all()), b
        return step, out

    def commit(self, step, paths, stream=None):
        n = max(1, max(len(p) for p in paths))
        count = _i([len(p) for p in paths])
        new = torch.empty(len(paths), dtype=torch.int32, device="cuda")
        before_k, before_v = self.flat(self.k).clone(), self.flat(self.v).clone()
        path = _i([p + [-1] * (n - len(p)) for p in paths])
        torch.cuda.synchronize()
        self.cache.commit(step, path, count, new, stream=stream)
        torch.cuda.synchronize()
        k, v = self.flat(self.k), self.flat(self.v)
        for b, p in enumerate(paths):
            if p:
                src = self.slots(b, 0, self.lens[b] + p[-1] + 1)[[self.lens[b] + j for j in p]]
                dst = self.slots(b, self.lens[b], self.lens[b] + len(p))
                assert torch.equal(k[dst], before_k[src]) and torch.equal(v[dst], before_v[src])
            self.lens[b] += len(p)
        assert new.cpu().tolist() == self.lens


@pytest.mark.parametrize("hq,hkv,d,t,page", [(8, 2, 64, "f16", 16), (6, 3, 128, "bf16", 32), (12, 4, 64, "f32", 16)])
@pytest.mark.parametrize("side", [False, True])
def test_a_server_run(lk, hq, hkv, d, t, page, side):
    """Prompts, then rounds of single tokens and of drafted trees with some of each accepted."""
    note(f"server run {hq}/{hkv}/{d} {t}, side stream {side}")
    s = _Server(lk, hq, hq, hkv, d, t, page, 4, 80, 20)
    stream = torch.cuda.Stream() if side else None
    step, _ = s.step([70, 3, 0, 130], stream=stream)
    s.commit(step, [list(range(64)), [0, 1, 2], [], list(range(64))], stream=stream)    # (lists of at most 64)
    s.lens[0], s.lens[3] = 70, 130
    for turn in range(3):
        step, _ = s.step([1, 1, 1, 1], stream=stream)
        s.commit(step, [[0]] * 4, stream=stream)
        news = [s.rng.randint(1, 20) for _ in range(4)]
        trees = [tree(s.rng, n) for n in news]
        step, _ = s.step(news, trees, stream=stream)
        paths = []
        for par, masks in trees:                         # a path from the root to a random token
            j, p = s.rng.randrange(len(par)), []
            while j >= 0:
                p.append(j)
                j = par[j]
            paths.append(p[::-1])
        s.commit(step, paths, stream=stream)


def test_a_captured_step(lk):
    """A step captured once and replayed: lengths move on the device, each replay against the same calls
    made eagerly on a copy, with other work between the replays."""
    hq, hkv, d, page, B, n = 8, 2, 64, 16, 3, 4
    g = torch.Generator().manual_seed(5)
    width = 12
    tab = torch.randperm(B * width, generator=g).view(B, width)
    start = [5, 0, 31]
    par, masks = tree(random.Random(1), n)
    freq = torch.tensor([1e4 ** (-2 * i / d) for i in range(d // 2)], dtype=torch.float64).float().cuda()

    class Side:
        def __init__(self):
            self.k, self.v = (torch.zeros(B * width, page, hkv, d, dtype=torch.float16, device="cuda") for _ in range(2))
            for x in (self.k, self.v):
                x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(6)))
            self.lens = _i(start)
            self.pos = torch.empty(B * n, dtype=torch.int32, device="cuda")
            self.deep = _i(depths(par)).repeat(B)
            self.wide = torch.zeros(B * n, (hq + 2 * hkv) * d, dtype=torch.float16, device="cuda")
            self.q = torch.empty(B * n, hq * d, dtype=torch.float16, device="cuda")
            self.out = torch.empty_like(self.q)
            self.path, self.count = _i([[0, -1]] * B), _i([1] * B)
            mask = torch.tensor(masks * B, device="cuda")
            self.step = lk.PagedStep(_i([0, n, 2 * n, 3 * n]), self.lens, tab.int().cuda(), B * n, pos=self.pos, mask=mask, max_new=n)
            self.cache = lk.PagedCache(self.k, self.v, hq)

        def once(self):
            torch.add(self.lens.repeat_interleave(n, output_size=B * n), self.deep, out=self.pos)
            a, e = hq * d, (hq + hkv) * d
            self.cache.append(self.step, self.wide[:, a:e], self.wide[:, e:], q=self.wide[:, :a], q_out=self.q, freq=freq)
            self.cache.attend(self.step, self.q, self.out)
            self.cache.commit(self.step, self.path, self.count, self.lens)

    eager, captured = Side(), Side()
    note("a captured step")
    captured.once()
    eager.once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.once()
    for turn in range(6):
        new = torch.randn(B * n, (hq + 2 * hkv) * d, generator=g).half().cuda()
        path = [[0, 1 + turn % 3], [0, -1], [1, 3]]
        count = [2, 1 + turn % 2, 2]
        for s in (eager, captured):
            s.wide.copy_(new)
            s.path.copy_(_i(path))
            s.count.copy_(_i(count))
        graph.replay()
        eager.once()
        junk = torch.randn(1 << 20, device="cuda").sum()
        torch.cuda.synchronize()
        assert junk == junk
        assert eager.lens.tolist() == captured.lens.tolist()
        for x, y in ((eager.out, captured.out), (eager.k, captured.k), (eager.v, captured.v)):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16)), turn
    assert eager.lens.tolist()[0] == start[0] + 1 + 12


def test_a_step_dropped_while_a_stream_works_on_it(lk):
    """The step's workspace is not handed to the next allocation while a side stream has still to use it."""
    b = Batch(3, [3000, 50], [1, 1], 16)
    k, v = (torch.randn(b.n_pages, 16, 8, 64, device="cuda").half() for _ in range(2))
    q = torch.randn(2, 2048, device="cuda").half()
    cache = lk.PagedCache(k, v, 32)
    want = torch.empty_like(q)
    step = b.step(lk, max_new=1)
    cache.attend(step, q, want)
    a = torch.ones(8192, 8192, device="cuda", dtype=torch.bfloat16)
    c = torch.empty_like(a)
    side, out = torch.cuda.Stream(), torch.empty_like(q)
    step = b.step(lk, max_new=1)
    tables = step._keep                                   # the tables are the caller's tensors
    torch.cuda.synchronize()
    note("a step dropped while a side stream works")
    with torch.cuda.stream(side):
        for _ in range(20):
            torch.mm(a, a, out=c)
    cache.attend(step, q, out, stream=side)
    at, n = step._work.data_ptr(), step._work.numel()
    del step
    new = torch.empty(n, dtype=torch.uint8, device="cuda")
    early, other = not side.query(), new.data_ptr() != at
    new.fill_(255)
    torch.cuda.synchronize()
    assert early and other and torch.equal(out, want)
    del tables


def test_two_streams_with_a_step_each(lk):
    b = Batch(4, [2000, 700], [1, 9], 16)
    k, v = (torch.randn(b.n_pages, 16, 8, 64, device="cuda").half() for _ in range(2))
    q = torch.randn(10, 2048, device="cuda").half()
    cache = lk.PagedCache(k, v, 32)
    want, outs = torch.empty_like(q), [torch.empty_like(q) for _ in range(2)]
    cache.attend(b.step(lk, max_new=9), q, want)
    streams, steps = [torch.cuda.Stream() for _ in range(2)], [b.step(lk, max_new=9) for _ in range(2)]
    torch.cuda.synchronize()
    note("two streams")
    for _ in range(20):
        for s, st, o in zip(streams, steps, outs):
            cache.attend(st, q, o, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


class _Elsewhere:
    """A stream of a device that the tensors are not on."""
    device_index, cuda_stream = 1, 0x1000


def test_a_stream_of_another_device_is_refused(lk):
    b = Batch(5, [20], [1], 16)
    k, v = (torch.randn(b.n_pages, 16, 2, 64, device="cuda").half() for _ in range(2))
    q = torch.randn(1, 512, device="cuda").half()
    cache, step = lk.PagedCache(k, v, 8), b.step(lk, max_new=1)
    note("a stream of another device")
    for call in (lambda: cache.append(step, q[:, :128], q[:, 128:256], stream=_Elsewhere()),
                 lambda: cache.attend(step, q, q.clone(), stream=_Elsewhere()),
                 lambda: cache.commit(step, None, _i([1]), step._keep[1], stream=_Elsewhere())):
        with pytest.raises(ValueError, match="another device"):
            call()


def test_the_decode_path_over_one_contiguous_cache(lk):
    """A contiguous cache is a pool whose pages lie in order: lk_attn_decode's result."""
    seq, page = 1000, 8 * 16
    g = torch.Generator().manual_seed(9)
    n = -(-seq // page)
    kc, vc = (torch.randn(n * page, 8, 64, generator=g).half().cuda() for _ in range(2))
    q = torch.randn(32, 64, generator=g).cuda()
    part, want = torch.empty(lk.part_bytes() // 4, device="cuda"), torch.empty(32, 64, device="cuda")
    note("decode over one contiguous cache")
    lk.attn_decode(q, kc, vc, d_pos_for(seq), part, want)
    out = torch.empty(1, 2048, device="cuda")
    step = lk.PagedStep(_i([0, 1]), _i([seq - 1]), _i([list(range(n))]), 1, max_new=1)
    lk.PagedCache(kc.view(n, page, 8, 64), vc.view(n, page, 8, 64), 32).attend(step, q.view(1, 2048), out)
    torch.cuda.synchronize()
    ref, tol = attend_ref(q.cpu().view(1, 32, 64), kc[:seq].cpu(), vc[:seq].cpu(), torch.ones(1, seq, dtype=torch.bool), torch.float32,
                          0.125)
    assert bool(((out.cpu().double().view(1, 32, 64) - ref).abs() <= tol).all())
    assert bool(((want.cpu().double().view(1, 32, 64) - ref).abs() <= tol).all())


def test_pools_past_4_gib(lk):
    """Pages whose bytes lie past 2^32 and past 2^31 rows of values."""
    page, hkv, d, hq = 64, 8, 128, 16
    n_pages = 36000                                      # 4.7 GB a pool
    k, v = (torch.empty(n_pages, page, hkv, d, dtype=torch.float16, device="cuda") for _ in range(2))
    lens, news = [200, 64], [20, 3]
    b = Batch(6, lens, news, page)
    high = [n_pages - 1 - 3 * i for i in range(8)]
    b.table, b.n_pages = [high[:4], high[4:8]], n_pages
    b.width = 4
    g = torch.Generator().manual_seed(7)
    for x in (k, v):
        for p in high:
            x[p] = torch.randn(page, hkv, d, generator=g).half().cuda()
    step = b.step(lk, max_new=20)
    rows = torch.randn(23, (hq + 2 * hkv) * d, generator=g).half().cuda()
    q, out = torch.empty(23, hq * d, dtype=torch.float16, device="cuda"), torch.empty(23, hq * d, dtype=torch.float16, device="cuda")
    cache = lk.PagedCache(k, v, hq)
    note("pools past 4 GiB")
    cache.append(step, rows[:, hq * d:(hq + hkv) * d], rows[:, (hq + hkv) * d:], q=rows[:, :hq * d], q_out=q)
    cache.attend(step, q, out)
    new = torch.empty(2, dtype=torch.int32, device="cuda")
    hold = {p: (k[p].cpu(), v[p].cpu()) for p in high}
    cache.commit(step, _i([[2, 7, 19], [0, 2, -1]]), _i([3, 2]), new)
    torch.cuda.synchronize()
    assert new.tolist() == [203, 66]
    row = lambda which, p, s: hold[p[s // page]][which][s % page]  # noqa: E731
    for i, (a, n) in enumerate(zip(lens, news)):
        tab = b.table[i]
        r = slice(b.first[i], b.first[i + 1])
        ks, vs = (torch.stack([row(w, tab, s) for s in range(a + n)]) for w in (0, 1))
        assert torch.equal(ks[a:], rows[r, hq * d:(hq + hkv) * d].cpu().view(n, hkv, d))
        want, tol = attend_ref(q[r].cpu().view(n, hq, d), ks, vs, causal(n, a), torch.float16, d ** -0.5)
        assert bool(((out[r].cpu().double().view(n, hq, d) - want).abs() <= tol).all())
        for j, src in enumerate(([2, 7, 19], [0, 2])[i]):
            p, o = tab[(a + j) // page], (a + j) % page
            assert torch.equal(k[p, o].cpu(), ks[a + src]) and torch.equal(v[p, o].cpu(), vs[a + src])
