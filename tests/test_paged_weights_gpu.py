"""How far the softmax weights of lk_paged_attn may be off, apart from the output's rounding: values
that cancel leave a small output, on which the weights' own errors show.  Two parts of the pools'
type hold a weight to 2^-22 (fp16) and 2^-16 (bf16), in every kernel that max_new chooses."""
import pytest
import torch

from gpu_util import note
from paged_util import HALF_STEP, TYPES, U, Batch, pool_type

LOST = {"f32": 2.0 ** -22, "f16": 2.0 ** -22, "bf16": 2.0 ** -16}


def _inputs(seed, n_keys, hkv, d, t):
    """Keys of one component and values whose weighted sum nearly vanishes, in the pools' type."""
    g = torch.Generator().manual_seed(seed)
    k = torch.zeros(n_keys, hkv, d)
    k[:, :, 0] = 2 * torch.rand(n_keys, hkv, generator=g) - 1
    k = k.to(pool_type(t))
    p = torch.softmax(k[:, :, 0].double(), 0).unsqueeze(-1)
    v = torch.randn(n_keys, hkv, d, generator=g).double()
    return k, (v - (p * v).sum(0)).to(pool_type(t)), p


def _bound(p, v, t):
    """(result [hkv][d], bound).  Scores q.k are one exact product, between -1 and 1.  A weight 2^a is off by
    LOST, by a's rounding (a is below 16: 2^-21, times ln 2), by the factor log2(e) of the scores
    (two half steps of 1.44) and by the exponential's own step 2^-23, together below LOST + 2^-20; in numerator
    and denominator alike that moves the result by at most this times A + |o|, A = sum p |v|.  The sums over keys
    add 16 keys a product, and the products and joins in order: n / 16 + 48 half steps of A."""
    o, A = (p * v.double()).sum(0), (p * v.double().abs()).sum(0)
    w = (LOST[t] + 2.0 ** -20) * (A + o.abs()) + (len(p) / 16 + 48) * U * A
    return o, w + HALF_STEP[TYPES[t]] * (o.abs() + w) + (2.0 ** -25 if t == "f16" else 0)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("n_keys", [40, 96])
@pytest.mark.parametrize("d", [64, 128])
def test_one_part_would_be_seen(t, n_keys, d):
    """Weights rounded once to the type leave the bound (CPU)."""
    _, v, p = _inputs(n_keys + d, n_keys, 2, d, t)
    o, tol = _bound(p, v, t)
    once = (p / p.amax(0) * 128).to(pool_type(t)).double()
    off = (once * v.double()).sum(0) / once.sum(0) - o
    assert float((off.abs() / tol).max()) > 3


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_keys", [40, 96])
@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 64), (8, 2, 64), (2, 2, 128), (8, 2, 128), (64, 2, 64)])
def test_weights_in_two_parts(lk, hq, hkv, d, t, n_keys):
    """One token, and 40 rows that all see the earlier positions alone, by every kind of workgroup."""
    k, v, p = _inputs(n_keys + d, n_keys, hkv, d, t)
    o, tol = _bound(p, v, t)
    for n, hints in ((1, (1, 2, 16, 64, 300)), (40, (1, 8, 40, 300, 2000))):
        b = Batch(n_keys, [n_keys], [n], 16)
        pools = [torch.zeros(b.n_pages, 16, hkv, d, dtype=pool_type(t)) for _ in range(2)]
        for pool, x in zip(pools, (k, v)):
            pool.view(-1, hkv, d)[b.slots(0, 0, n_keys)] = x
        q = torch.zeros(n, hq, d, dtype=TYPES[t])
        q[:, :, 0] = 1.0
        for hint in hints:
            out = torch.empty(n, hq * d, dtype=TYPES[t], device="cuda")
            note(f"weights {hq}/{hkv}/{d} {t}, {n_keys} keys, {n} rows, hint {hint}")
            lk.PagedCache(pools[0].cuda(), pools[1].cuda(), hq).attend(b.step(lk, mask=[0] * n, max_new=hint), q.view(n, -1).cuda(), out,
                                                                       scale=1.0)
            torch.cuda.synchronize()
            got = out.cpu().double().view(n, hkv, hq // hkv, d)
            off = (got - o[None, :, None]).abs() / tol[None, :, None]
            assert float(off.max()) <= 1, (n, hint, float(off.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_an_unknown_number_of_new_tokens(lk, t):
    """max_new 0 is the mean, rounded up, where the workspace has room for that, and 1 where not: the same bits as
    of those."""
    hq, hkv, d = 8, 2, 64
    for news in ([130, 65], [1, 1, 1], [40, 0, 0, 3], [1]):
        b = Batch(1, [37, 200, 9, 0][:len(news)], news, 16, pad=1)
        g = torch.Generator().manual_seed(2)
        k, v = (torch.randn(b.n_pages, 16, hkv, d, generator=g).to(pool_type(t)).cuda() for _ in range(2))
        q = torch.randn(b.rows, hq * d, generator=g).to(TYPES[t]).cuda()
        cache, mean = lk.PagedCache(k, v, hq), -(-b.rows // len(news))
        small, large = (cache.work_bytes(TYPES[t], n) for n in (1, mean))
        works = {"own": None, "small": torch.empty(small, dtype=torch.uint8, device="cuda"),
                 "large": torch.empty(large, dtype=torch.uint8, device="cuda")}
        outs = {}
        for name, hint, work in (("one", 1, None), ("mean", mean, None), *(("0 " + w, 0, works[w]) for w in works)):
            outs[name] = torch.zeros_like(q)
            note(f"max_new {hint}, {name}, {t}, news {news}")
            step = b.step(lk, max_new=hint, work=work)
            cache.attend(step, q, outs[name])
            torch.cuda.synchronize()
            if work is None:
                assert step._work.numel() == (small if hint == 1 else large)
        same = lambda x, y: torch.equal(outs[x].view(torch.int16), outs[y].view(torch.int16))  # noqa: E731
        assert same("0 own", "mean") and same("0 large", "mean") and same("0 small", "mean" if small >= large else "one")
