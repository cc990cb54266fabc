"""The operators of a layer's second half as they are used together, on the GPU:
attention -> its output projection -> lk_norm_q8 -> lk_gemv_q4_0 / lk_pf_gemm_q4_0 /
lk_gemm_i8 / lk_moe_q4_0 -> the next norm -> the head, with the residual stream kept by
the norm.

Each step is compared with its reference on the bytes the GPU itself handed to it (so no
step's rounding is another's error): the norm, the quants and the products bit for bit,
the mixture of experts within 1e-5 of a row's norm for fp32 rows and 2e-4 and half a step
for bf16 rows (the derivation stands in test_moe_gpu.py; gate and up scales are those of
its layers).
"""
import numpy as np
import pytest
import torch

from ffn_util import HALF_STEP, bits, gemm_ref, moe_ref, norm_ref, q4_planes, q8_row_ref, same
from gpu_util import d_pos_for, dev, dev_h, host, note

pytestmark = pytest.mark.gpu

H, F, E, K, V = 2048, 256, 16, 4, 1000        # hidden, ffn, experts, choices, rows of the head


def _cuda(x):
    return None if x is None else tuple(t.cuda() for t in x) if isinstance(x, tuple) else x.cuda()


class _Weights:
    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.wo = q4_planes(g, 1, H, H)
        self.w1, self.w2 = torch.rand(H, generator=g) + 0.5, torch.rand(H, generator=g) + 0.5
        self.dense = q4_planes(g, 1, 128, H)                             # a dense Q4_0 product beside the experts
        self.moe = {"router": torch.randn(E, H, generator=g) * H ** -0.5, "bias": 0.2 * torch.randn(E, generator=g),
                    "gate": q4_planes(g, E, F, H), "up": q4_planes(g, E, F, H), "down": q4_planes(g, E, H, F)}
        self.head = torch.randint(-127, 128, (V, H), generator=g, dtype=torch.int8)
        self.head_s = (0.5 + torch.rand(V, generator=g)) / 127 / H ** 0.5

    def device(self, lk):
        d = {k: _cuda(v) for k, v in vars(self).items() if k != "moe"}
        m = {k: _cuda(v) for k, v in self.moe.items()}
        d["layer"] = lk.MoeQ4_0(m["router"], m["gate"], m["up"], m["down"], K, bias=m["bias"], max_tokens=64)
        return d


def _q4(p):
    """(qs, d) of a single plane as the oracle and the dense products take them."""
    return p[0][0].numpy(), p[1][0].numpy().view(np.uint16)


def _check_moe(W, y, h, out, dt):
    want, _, _ = moe_ref(y.cpu(), k=K, score="sigmoid", res=h.cpu(), **W.moe)
    off, norm = (out.cpu().double() - want).norm(dim=1), (want - h.cpu().double()).norm(dim=1)
    tol = 1e-5 if dt == torch.float32 else 2e-4 + 1e-5
    # the sum with the residual rounds once, relative to the sum
    assert bool((off <= tol * norm + HALF_STEP[dt] * want.norm(dim=1)).all()), (off / norm).max().item()


class _Decode:
    """One decoded token's buffers and the calls on them."""

    def __init__(self, lk, D, kc, vc, seq):
        f = lambda *s: torch.zeros(*s, device="cuda")
        self.lk, self.D, self.kc, self.vc, self.pos = lk, D, kc, vc, d_pos_for(seq)
        self.q, self.x = f(32, 64), f(1, H)
        self.part, self.att = f(lk.part_bytes() // 4), f(32, 64)
        self.yq8 = torch.zeros(64 * 36, dtype=torch.uint8, device="cuda")
        self.delta, self.h, self.y, self.dense = f(1, H), f(1, H), f(1, H), f(128)
        self.blk = torch.zeros(1, 64 * 36, dtype=torch.uint8, device="cuda")
        self.q8, self.sc, self.q8b, self.scb = lk.i8_rows(1, H), f(1), lk.i8_rows(1, H), f(1)
        self.out, self.h2, self.logits = f(1, H), f(1, H), f(1, V)
        self.work = torch.empty(D["layer"].work_bytes(), dtype=torch.uint8, device="cuda")

    def run(self):
        lk, D = self.lk, self.D
        lk.attn_decode(self.q, self.kc, self.vc, self.pos, self.part, self.att, self.yq8)
        lk.gemv_q4_0(D["wo"][0], D["wo"][1], self.yq8, H, 64, self.delta)
        # h = x + delta; its norm for the dense product, and the fp32 rows for the experts
        lk.norm_q8(self.x, D["w1"], self.blk, delta=self.delta, res=self.h, y=self.y)
        lk.gemv_q4_0(D["dense"][0], D["dense"][1], self.blk, 128, 64, self.dense)
        D["layer"](self.y, self.out, res=self.h, work=self.work)
        lk.norm_q8(self.out, D["w2"], self.q8, self.sc, res=self.h2)
        lk.gemm_i8(self.q8, self.sc, D["head"], D["head_s"], self.logits)


def _decode(lk, seed, seq):
    rng = np.random.default_rng(seed)
    kc, vc = (dev_h(rng.standard_normal((seq, 8, 64)).astype(np.float16).view(np.uint16)) for _ in range(2))
    W = _Weights(seed)
    return W, _Decode(lk, W.device(lk), kc, vc, seq), rng


def _fill(s, rng):
    s.q.copy_(torch.from_numpy(rng.standard_normal((32, 64)).astype(np.float32)))
    s.x.copy_(torch.from_numpy(rng.standard_normal((1, H)).astype(np.float32)))


def test_decode_chain(lk, oracle):
    W, s, rng = _decode(lk, 5, 700)
    _fill(s, rng)
    note("decode attention -> projection -> norm -> dense and experts -> norm -> int8 head")
    s.run()
    torch.cuda.synchronize()
    qs, d = _q4(W.wo)
    assert np.array_equal(host(s.delta)[0].view(np.uint32), oracle.gemv_q4_0(qs, d, host(s.yq8).reshape(64, 36), H, 64).view(np.uint32))
    h, y = norm_ref(s.x.cpu(), s.delta.cpu(), W.w1, 1e-5)
    assert same(s.h, h) and same(s.y, y)
    # the blocks: the quants of the planar form (the scale in fp16 here)
    q1, _ = oracle.pf_quant_rows(y.numpy(), 1, H, 64)
    assert np.array_equal(host(s.blk).reshape(64, 36)[:, 4:].view(np.int8).reshape(-1), np.asarray(q1).reshape(-1))
    qs, d = _q4(W.dense)
    assert np.array_equal(host(s.dense).view(np.uint32), oracle.gemv_q4_0(qs, d, host(s.blk).reshape(64, 36), 128, 64).view(np.uint32))
    _check_moe(W, s.y, s.h, s.out, torch.float32)
    h2, y2 = norm_ref(s.out.cpu(), None, W.w2, 1e-5)
    q2, sc2 = q8_row_ref(y2)
    assert same(s.h2, h2) and torch.equal(s.q8.cpu(), q2) and same(s.sc, sc2)
    assert np.array_equal(bits(s.logits), bits(gemm_ref(q2, sc2, W.head, W.head_s, torch.float32)))


def test_decode_chain_in_a_graph(lk):
    """Captured once, replayed with other inputs between eager runs of the same chain on
    other buffers: every replay's bytes are the eager run's."""
    W, s, rng = _decode(lk, 6, 300)
    e = _Decode(lk, s.D, s.kc, s.vc, 300)
    _fill(s, rng)
    note("the decode chain captured and replayed")
    s.run()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        s.run()
    for rep in range(4):
        _fill(e, rng)
        s.q.copy_(e.q)
        s.x.copy_(e.x)
        gr.replay()
        e.run()
        torch.cuda.synchronize()
        for n in ("delta", "h", "y", "blk", "dense", "out", "h2", "q8", "sc", "logits"):
            assert torch.equal(getattr(s, n), getattr(e, n)), (rep, n)


def test_two_chains_on_two_streams(lk):
    """The same layer on two streams at once, a workspace to each."""
    W, a, rng = _decode(lk, 7, 260)
    b = _Decode(lk, a.D, a.kc, a.vc, 260)
    _fill(a, rng)
    _fill(b, rng)
    note("two decode chains on two streams")
    a.run()
    b.run()
    torch.cuda.synchronize()
    want = [(s.out.clone(), s.logits.clone()) for s in (a, b)]
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, t in zip((a, b), st):
            with torch.cuda.stream(t):
                s.out.zero_()
                s.run()
    torch.cuda.synchronize()
    for s, (o, l) in zip((a, b), want):
        assert torch.equal(s.out, o) and torch.equal(s.logits, l)


@pytest.mark.parametrize("m", [1, 37, 64])
def test_prefill_chain(lk, oracle, m):
    """A chunk's rows: planar Q8_1 through the Q4_0 GEMM, the residual and norm in bf16 and
    planar again, the experts over the chunk, and the int8 product with its residual."""
    W = _Weights(20 + m)
    D = W.device(lk)
    g = torch.Generator().manual_seed(m)
    att = torch.randn(m, H, generator=g)
    f = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")
    x = torch.randn(m, H, generator=g).bfloat16()
    aqs, asc = f(m, H, dt=torch.int8), f(m, 64, 2)
    note(f"prefill chain m={m}")
    lk.pf_quant_rows(att.cuda(), m, H, 64, aqs, asc)
    delta32 = f(m, H)
    lk.pf_gemm_q4_0(D["wo"][0], D["wo"][1], H, 64, aqs, asc, m, delta32)
    delta = delta32.bfloat16()
    h, y, q, sc = f(m, H, dt=torch.bfloat16), f(m, H, dt=torch.bfloat16), f(m, H, dt=torch.int8), f(m, 64, 2)
    lk.norm_q8(x.cuda(), D["w1"], q, sc, delta=delta, res=h, y=y)
    dense = f(m, 128)
    lk.pf_gemm_q4_0(D["dense"][0], D["dense"][1], 128, 64, q, sc, m, dense)
    out = f(m, H, dt=torch.bfloat16)
    D["layer"](y, out, res=h)
    q8, s8 = lk.i8_rows(m, H), f(m)
    lk.norm_q8(out, D["w2"], q8, s8)
    up = f(m, V, dt=torch.bfloat16)
    lk.gemm_i8(q8, s8, D["head"], D["head_s"], up, res=up)
    torch.cuda.synchronize()
    hr, yr = norm_ref(x, delta.cpu(), W.w1, 1e-5)
    assert same(h, hr.bfloat16()) and same(y, yr.bfloat16())
    q1, sc1 = oracle.pf_quant_rows(yr.numpy(), m, H, 64)
    assert np.array_equal(host(q).reshape(-1), np.asarray(q1).reshape(-1)) and \
        np.array_equal(host(sc).view(np.uint32).reshape(-1), np.asarray(sc1, np.float32).view(np.uint32).reshape(-1))
    qs, d = _q4(W.dense)
    want = oracle.pf_gemm_q4_0(qs, d, 128, 64, host(q), host(sc), m, out=np.zeros((m, 128), np.float32), out_ld=128)
    assert np.array_equal(host(dense).view(np.uint32), want.view(np.uint32))
    _check_moe(W, y, h, out, torch.bfloat16)
    _, y2 = norm_ref(out.cpu(), None, W.w2, 1e-5)
    q2, sc2 = q8_row_ref(y2)
    assert torch.equal(q8.cpu(), q2) and same(s8, sc2)
    assert np.array_equal(bits(up), bits(gemm_ref(q2, sc2, W.head, W.head_s, torch.bfloat16, torch.zeros(m, V).bfloat16())))
