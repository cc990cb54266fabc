"""The mixture-of-experts layer for a few tokens (lk_moe_q4_0) on the GPU.

Tolerance.  A block of 32 values of x, and of h, becomes whole numbers whose largest is at
least 2^14 (16-bit rows) or 2^22 (fp32 rows): an rms error of 0.29 / 2^14 = 1.8e-5 of the
block's largest value, which is 2.2 times the rms of 32 normal values and about 4 times
that of products h.  g and u are off by 4e-5 of themselves then, silu(g) u by up to
three times as much, the down product adds 7e-5: 2e-4 of a row's norm, and 256 times
less, 8e-7, for fp32 rows.  Everything else is exact or rounds in fp32: a block's sum and its
scaling (4 roundings), the chain over a wave's blocks and the sum of 8 waves, about 4e-7
of a row's norm in each product.  2e-4 is allowed for 16-bit rows, and half a step
of every output, 1e-5 for fp32 rows and besides.  Where all values are
small integers nothing rounds, and the results are compared exactly.
"""
import numpy as np
import pytest
import torch

from ffn_util import HALF_STEP, TYPES, guarded, moe_ref, q4_pack, q4_planes, untouched
from gpu_util import note

pytestmark = pytest.mark.gpu


def _layer(seed, E, hidden, ffn, bias=False):
    g = torch.Generator().manual_seed(seed)
    return {"router": torch.randn(E, hidden, generator=g) * hidden ** -0.5, "bias": 0.2 * torch.randn(E, generator=g) if bias else None,
            "gate": q4_planes(g, E, ffn, hidden), "up": q4_planes(g, E, ffn, hidden), "down": q4_planes(g, E, hidden, ffn)}


def _dev(L):
    return {k: None if v is None else tuple(t.cuda() for t in v) if isinstance(v, tuple) else v.cuda() for k, v in L.items()}


def _make(lk, L, k, **kw):
    D = _dev(L)
    return lk.MoeQ4_0(D["router"], D["gate"], D["up"], D["down"], k, bias=D["bias"], **kw)


def _x(seed, T, hidden, dt):
    return (torch.randn(T, hidden, generator=torch.Generator().manual_seed(seed)) * 1.5).to(dt)


def _close(out, want, dt, what):
    off = (out.cpu().double() - want).norm(dim=1)
    norm = want.norm(dim=1)
    tol = 1e-5 + (0 if dt == torch.float32 else 2e-4 + HALF_STEP[dt])
    assert bool((off <= tol * norm).all()), (what, (off / norm).max().item(), tol)


def _run(lk, layer, x, hidden, dt, k, res=None, pad=0):
    T = x.shape[0]
    ob, out = guarded(T, hidden, dt, pad)
    xb, xv = guarded(T, hidden, dt, pad)
    xv.copy_(x)
    ids = torch.full((T, k), -5, dtype=torch.int32, device="cuda")
    w = torch.empty(T, k, device="cuda")
    layer(xv, out, res=None if res is None else res.cuda(), ids=ids, weights=w)
    torch.cuda.synchronize()
    assert untouched(ob, T, hidden)
    return out, ids.cpu(), w.cpu()


# T, hidden, ffn, E, k, score: one block and one token; block counts off the groups
# of four; a tile of tokens, one more and several; all experts met and few; the
# limits of tokens, experts and choices
CASES = [(1, 32, 32, 1, 1, "sigmoid"), (1, 64, 32, 3, 2, "softmax"), (2, 96, 160, 8, 4, "sigmoid"),
         (3, 160, 224, 60, 6, "softmax"), (4, 512, 256, 64, 8, "sigmoid"), (5, 256, 96, 16, 3, "softmax"),
         (9, 1056, 288, 32, 2, "sigmoid"), (17, 128, 512, 8, 8, "softmax"), (64, 256, 128, 64, 4, "sigmoid"),
         (64, 64, 64, 256, 8, "softmax"), (33, 96, 64, 2, 1, "sigmoid"), (1, 2048, 1536, 8, 4, "sigmoid")]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,hidden,ffn,E,k,score", CASES)
def test_layer(lk, T, hidden, ffn, E, k, score, t):
    dt = TYPES[t]
    L = _layer(T + hidden + ffn, E, hidden, ffn, bias=score == "sigmoid" and E > 1)
    x = _x(T + E, T, hidden, dt)
    res = (torch.randn(T, hidden, generator=torch.Generator().manual_seed(9)) * 3).to(dt) if T % 2 else None
    note(f"moe T={T} hidden={hidden} ffn={ffn} E={E} k={k} {score} {t}")
    layer = _make(lk, L, k, score=score, renorm=k != 3, scale=1.0 if k != 2 else 2.5, max_tokens=T)
    out, ids, w = _run(lk, layer, x, hidden, dt, k, res, pad=T % 3)
    want, ids1, w1 = moe_ref(x, k=k, score=score, renorm=k != 3, scale=1.0 if k != 2 else 2.5, res=res, **L)
    assert torch.equal(ids.long(), ids1)
    # a logit: 32 fp32 roundings in a lane's chain and 6 in the tree at most, of |x||r| about
    # 3 for these rows; exp and the divisions a few more
    assert bool(((w.double() - w1).abs() <= 60 * 2.0 ** -24 * 3 * w1.abs() + 1e-30).all())
    _close(out, want, dt, (T, hidden, ffn, E, k, score, t))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hidden,ffn,T", [(64, 64, 1), (64, 96, 7), (32, 160, 6), (128, 32, 33)])
def test_exact_integers(lk, hidden, ffn, T, t):
    """x of ones, gate and up weights 1 or 2, down -1, 0 or 1, block scales 1: g is at
    least 32, where silu(g) = g in fp32.  With hidden 32 and 64 h is at most 2^14 and
    its whole numbers are exact, a block's sums stay below 2^24: nothing rounds.  With
    hidden 128 h reaches 2^16, beyond the 2^15 of two digits: each h is off by at most 2, a sum
    of its one block of 32 by 64 (99 * 4 is allowed)."""
    dt = TYPES[t]
    E = 5
    g = torch.Generator().manual_seed(hidden + ffn)

    def ints(lo, hi, rows, cols):
        w = torch.randint(lo, hi + 1, (E, rows, cols), generator=g)
        return w, (q4_pack(w), torch.ones(E, rows, cols // 32).half())
    G, gate = ints(1, 2, ffn, hidden)
    U, up = ints(1, 2, ffn, hidden)
    D, down = ints(-1, 1, hidden, ffn)
    router = torch.randn(E, hidden, generator=g)
    x = torch.ones(T, hidden).to(dt)
    note(f"moe exact integers {hidden} {ffn} T={T} {t}")
    layer = _make(lk, {"router": router, "bias": None, "gate": gate, "up": up, "down": down}, 1, max_tokens=T)
    out, ids, w = _run(lk, layer, x, hidden, dt, 1)
    e = int(torch.argmax(router.double().sum(1)))
    assert (ids == e).all() and (w == 1).all()
    want = (D[e] @ (G[e].sum(1) * U[e].sum(1))).float().to(dt)
    if hidden < 128:
        assert torch.equal(out.cpu(), want.expand(T, hidden))
    else:
        exact = (D[e] @ (G[e].sum(1) * U[e].sum(1))).double().expand(T, hidden)
        off, top = (out.cpu().double() - exact).abs(), torch.finfo(dt).max
        near = exact.abs() < top - 2 * 99 * 4
        assert bool((off <= 99 * 4 + 2 * HALF_STEP[dt] * exact.abs())[near].all())
        assert torch.isinf(out.cpu()[exact.abs() > top + 2 * 99 * 4]).all()      # fp16's range ends


def test_every_weight_counts(lk):
    """Each single element of a gate, up or down row reaches the place it should: unit
    vectors through weights that name their own row, column and matrix."""
    hidden, ffn = 160, 96
    g = torch.Generator().manual_seed(4)
    L = _layer(4, 1, hidden, ffn)
    x = torch.zeros(64, hidden)
    cols = torch.randperm(hidden, generator=g)[:64]
    x[torch.arange(64), cols] = 100.0
    note("moe unit vectors")
    out, _, _ = _run(lk, _make(lk, L, 1, max_tokens=64), x, hidden, torch.float32, 1)
    want, _, _ = moe_ref(x, k=1, score="sigmoid", **L)
    _close(out, want, torch.float32, "unit vectors")


def test_ties_go_to_the_lowest_index(lk):
    """Equal router rows, and rows that differ in the sign of zero; biases that tie
    scores; and scores that saturate, which without a bias still follow the logits."""
    hidden, ffn, E = 64, 32, 40
    L = _layer(1, E, hidden, ffn)
    L["router"][:] = L["router"][0]
    x = _x(3, 6, hidden, torch.float32)
    note("moe ties")
    for score in ("sigmoid", "softmax"):
        _, ids, w = _run(lk, _make(lk, L, 8, score=score), x, hidden, torch.float32, 8)
        assert torch.equal(ids.long(), torch.arange(8).expand(6, 8)) and bool((w - 0.125).abs().max() < 1e-6)
    L["router"][:] = 0.0
    L["router"][::2] = -0.0
    L["bias"] = torch.zeros(E)
    L["bias"][[7, 19, 33]] = 0.25
    _, ids, _ = _run(lk, _make(lk, L, 5), x, hidden, torch.float32, 5)
    assert torch.equal(ids.long(), torch.tensor([7, 19, 33, 0, 1]).expand(6, 5))
    L["bias"] = None
    L["router"] = torch.arange(E).float()[:, None].expand(E, hidden).contiguous()
    _, ids, w = _run(lk, _make(lk, L, 4), torch.ones(2, hidden), hidden, torch.float32, 4)
    assert torch.equal(ids.long(), torch.tensor([39, 38, 37, 36]).expand(2, 4)) and torch.equal(w, torch.full((2, 4), 0.25))


def test_all_tokens_choose_the_same(lk):
    """One expert takes all 64 tokens (a bias), another half of them."""
    hidden, ffn, E = 128, 64, 12
    L = _layer(2, E, hidden, ffn)
    L["bias"] = torch.zeros(E)
    L["bias"][5] = 10.0
    for t, dt in TYPES.items():
        x = _x(6, 64, hidden, dt)
        note(f"moe one expert for all {t}")
        out, ids, _ = _run(lk, _make(lk, L, 2), x, hidden, dt, 2)
        want, ids1, _ = moe_ref(x, k=2, score="sigmoid", **L)
        assert torch.equal(ids.long(), ids1) and (ids[:, 0] == 5).all()
        _close(out, want, dt, "one expert")


def test_tokens_that_are_not_numbers(lk):
    """A NaN or an infinity in a token makes its own row NaN, and no other row differs
    by a bit; NaN and infinite biases order as documented and stay in range."""
    hidden, ffn, E = 96, 64, 9
    L = _layer(3, E, hidden, ffn)
    x = _x(7, 10, hidden, torch.float32)
    layer = _make(lk, L, 3)
    note("moe rows that are not numbers")
    clean, ids0, _ = _run(lk, layer, x, hidden, torch.float32, 3)
    bad = x.clone()
    bad[2, 5], bad[3, 95], bad[8, 0] = float("nan"), float("inf"), -float("inf")
    out, ids, _ = _run(lk, layer, bad, hidden, torch.float32, 3)
    rows = [i for i in range(10) if i not in (2, 3, 8)]
    assert torch.equal(out[rows], clean[rows]) and torch.equal(ids[rows], ids0[rows])
    assert torch.isnan(out[[2, 3, 8]]).all()
    assert bool(((ids >= 0) & (ids < E)).all()) and all(len(set(r)) == 3 for r in ids.tolist())
    L["bias"] = torch.zeros(E)
    L["bias"][[0, 1, 2, 3, 4, 5]] = float("nan")
    L["bias"][6] = -float("inf")
    _, ids, _ = _run(lk, _make(lk, L, 5), x, hidden, torch.float32, 5)
    assert bool((ids[:, 2] == 6).all()) and torch.equal(ids[:, 3:].long(), torch.tensor([0, 1]).expand(10, 2))
    assert bool((ids[:, :2].sort(1).values == torch.tensor([7, 8])).all())


def test_small_and_large_values(lk):
    """fp32 rows far beyond what fp16 holds, and far below."""
    hidden, ffn = 64, 64
    L = _layer(5, 4, hidden, ffn)
    L["router"] *= 1e-3
    for scale in (1e-12, 1e-4, 1e4, 1e9):
        x = _x(5, 3, hidden, torch.float32) * scale
        L1 = {**L, "router": L["router"] / scale}
        note(f"moe values of about {scale}")
        out, ids, _ = _run(lk, _make(lk, L1, 2), x, hidden, torch.float32, 2)
        want, ids1, _ = moe_ref(x, k=2, score="sigmoid", **L1)
        assert torch.equal(ids.long(), ids1)
        _close(out, want, torch.float32, scale)


def test_in_place_stream_graph_and_workspaces(lk):
    """out over x and over res; a side stream; two graphs with workspaces of their own
    replayed together, one layer's weights."""
    hidden, ffn, E, k = 256, 128, 16, 4
    L = _layer(8, E, hidden, ffn)
    layer = _make(lk, L, k, max_tokens=20)
    x, res = _x(1, 20, hidden, torch.bfloat16), _x(2, 20, hidden, torch.bfloat16)
    want, _, _ = _run(lk, layer, x, hidden, torch.bfloat16, k, res)
    note("moe in place, streams and graphs")
    a, r = x.cuda(), res.cuda()
    layer(a, a, res=r)
    assert torch.equal(a, want)
    a = x.cuda()
    layer(a, r, res=r)
    assert torch.equal(r, want)
    st = torch.cuda.Stream()
    o = torch.empty_like(a)
    r = res.cuda()
    st.wait_stream(torch.cuda.current_stream())
    layer(a, o, res=r, stream=st)
    st.synchronize()
    assert torch.equal(o, want)
    sides = []
    for i in range(2):
        xs, os, ws = torch.empty_like(a), torch.empty_like(a), torch.empty(layer.work_bytes(), dtype=torch.uint8, device="cuda")
        gr = torch.cuda.CUDAGraph()
        s = torch.cuda.Stream()
        xs.copy_(x)
        torch.cuda.synchronize()
        with torch.cuda.graph(gr, stream=s):
            layer(xs, os, res=r, work=ws)
        sides.append((xs, os, gr, s, ws))                  # the graph's buffers live as long as it
    for rep in range(3):
        xx = [_x(30 + 2 * rep + i, 20, hidden, torch.bfloat16) for i in range(2)]
        wants = [_run(lk, layer, v, hidden, torch.bfloat16, k, res)[0] for v in xx]
        for v, (xs, os, gr, s, _) in zip(xx, sides):
            xs.copy_(v)
            os.zero_()
        torch.cuda.synchronize()
        for xs, os, gr, s, _ in sides:
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for w, (xs, os, gr, s, _) in zip(wants, sides):
            assert torch.equal(os, w)


def test_fewer_tokens_than_made_for(lk):
    """One workspace for calls of other sizes in turn; no tokens at all."""
    hidden, ffn = 128, 64
    L = _layer(6, 8, hidden, ffn)
    layer = _make(lk, L, 2, max_tokens=64)
    for T in (64, 1, 13, 0, 4):
        x = _x(T, T, hidden, torch.float32)
        note(f"moe T={T} of 64")
        if T == 0:
            e = torch.empty(0, hidden, device="cuda")
            layer(e, e)
            continue
        out, _, _ = _run(lk, layer, x, hidden, torch.float32, 2)
        _close(out, moe_ref(x, k=2, score="sigmoid", **L)[0], torch.float32, T)


@pytest.mark.parametrize("t", TYPES)
def test_a_token_does_not_depend_on_the_others(lk, t):
    """Above eight tokens a row's bytes are the same alone with few at its experts and among
    many: experts met once take one kind of product, the others another."""
    hidden, ffn, E, k = 544, 352, 12, 3                  # 17 and 11 blocks: last steps of one and three
    dt = TYPES[t]
    layer = _make(lk, _layer(41, E, hidden, ffn), k)
    x = _x(42, 64, hidden, dt)
    note(f"moe rows in batches of 64, 32, 16 and 9 {t}")
    whole, _, _ = _run(lk, layer, x, hidden, dt, k)
    for T in (32, 16, 9):
        for at in range(0, 64 - T + 1, T):
            assert torch.equal(_run(lk, layer, x[at:at + T], hidden, dt, k)[0], whole[at:at + T]), (T, at)


@pytest.mark.parametrize("T", [1, 7, 9, 64])
@pytest.mark.parametrize("hidden,ffn", [(32768, 32), (32, 32768)])
def test_longest_rows(lk, hidden, ffn, T):
    """The largest dimensions, in both kinds of launch."""
    dt = TYPES["f32"] if T % 2 else TYPES["bf16"]
    L = _layer(T, 3, hidden, ffn, bias=True)
    x = _x(50 + T, T, hidden, dt)
    note(f"moe hidden={hidden} ffn={ffn} T={T}")
    out, ids, _ = _run(lk, _make(lk, L, 2), x, hidden, dt, 2)
    want, ids1, _ = moe_ref(x, k=2, score="sigmoid", **L)
    assert torch.equal(ids.long(), ids1)
    _close(out, want, dt, (hidden, ffn, T))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,k", [(5, 8), (6, 2), (6, 3), (8, 2), (8, 1), (7, 3), (7, 4), (8, 4), (8, 8)])
def test_both_sides_of_the_line_between_launches(lk, T, k, t):
    """Up to 5 tokens, or 8 of 28 choices in all (fp32 rows: 16), in three launches, more in five."""
    hidden, ffn, E, dt = 288, 160, 9, TYPES[t]
    L = _layer(60 + T, E, hidden, ffn, bias=k > 2)
    x, res = _x(T, T, hidden, dt), _x(T + 1, T, hidden, dt)
    note(f"moe T={T} k={k} {t}")
    out, ids, _ = _run(lk, _make(lk, L, k), x, hidden, dt, k, res)
    want, ids1, _ = moe_ref(x, k=k, score="sigmoid", res=res, **L)
    assert torch.equal(ids.long(), ids1)
    _close(out, want, dt, (T, k))
