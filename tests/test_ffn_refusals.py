"""What lk_norm_q8, lk_gemm_i8 and lk_moe_q4_0 refuse, through the C ABI and through the Python
mirror.  CPU only: every call here fails its checks, or has nothing to do, before
anything is launched."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(0x1000)      # never dereferenced
O = ctypes.c_void_p(0x1001)
F = ctypes.c_float(1e-5)


def test_norm_c_refusals(lk_host):
    f = lk_host.load().lk_norm_q8
    ok = dict(type=0, x=P, ldx=64, delta=None, ldd=0, w=P, eps=F, rows=4, n=64, res=None, ldr=0, y=None, ldy=0, form=0, q=P,
              ldq=64, sc=P, stream=None)

    def rc(**kw):
        return f(*{**ok, **kw}.values())
    for bad in (dict(type=3), dict(type=-1), dict(form=3), dict(form=-1), dict(rows=-1), dict(n=0), dict(n=32769, ldx=40000, ldq=40000),
                dict(eps=ctypes.c_float(-1.0)), dict(eps=ctypes.c_float(float("nan"))), dict(x=None), dict(w=None), dict(q=None),
                dict(sc=None), dict(ldx=63), dict(delta=P, ldd=63), dict(res=P, ldr=63), dict(y=P, ldy=63), dict(ldq=63),
                dict(form=1, ldq=80), dict(form=2, ldq=80), dict(form=1, n=48, ldq=48), dict(form=2, n=48, ldq=48),
                dict(x=O), dict(delta=O, ldd=64), dict(res=O, ldr=64), dict(y=O, ldy=64), dict(w=O), dict(sc=O),
                dict(form=1, sc=ctypes.c_void_p(0x1004)), dict(form=2, q=O, sc=None), dict(type=1, x=O),
                dict(rows=2 ** 26), dict(rows=2 ** 22, n=5000, ldx=5000, ldq=5000)):
        assert rc(**bad) == 1, bad
        assert b"lk_norm_q8" in lk_host.load().lk_last_error(), bad
    assert rc(rows=0, x=None, w=None, q=None, sc=None) == 0


def test_gemm_c_refusals(lk_host):
    f = lk_host.load().lk_gemm_i8
    ok = dict(x=P, ldx=64, sx=P, w=P, ldw=64, sw=P, M=4, N=4, K=64, type=0, res=None, ldr=0, out=P, ldo=4, stream=None)

    def rc(**kw):
        return f(*{**ok, **kw}.values())
    for bad in (dict(type=3), dict(M=-1), dict(N=-1), dict(K=0), dict(K=131072, ldx=131072, ldw=131072), dict(x=None), dict(sx=None),
                dict(w=None), dict(sw=None), dict(out=None), dict(ldx=48), dict(ldx=72), dict(ldw=48), dict(ldw=65), dict(ldo=3),
                dict(res=P, ldr=3), dict(ldx=8388624), dict(ldw=8388624), dict(x=ctypes.c_void_p(0x1008)),
                dict(w=ctypes.c_void_p(0x1008)), dict(sx=O), dict(sw=O), dict(out=O), dict(res=O, ldr=4),
                dict(M=2 ** 31 - 1), dict(N=2 ** 31 - 1, ldo=2 ** 31 - 1), dict(M=2 ** 31 - 1, N=2 ** 31 - 1, ldo=2 ** 31 - 1)):
        assert rc(**bad) == 1, bad
        assert b"lk_gemm_i8" in lk_host.load().lk_last_error(), bad
    assert rc(M=0, x=None) == 0 and rc(N=0, w=None) == 0


def test_mirror_refusals(lk_host):
    """Host tensors of every kind are refused, wrong types and shapes before that."""
    lk = lk_host
    x, w = torch.zeros(3, 64), torch.ones(64)
    q, sc = torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3)
    with pytest.raises(ValueError, match="device memory"):
        lk.norm_q8(x, w, q, sc)
    for kw, word in ((dict(x=x.double()), "fp32, fp16 or bf16"), (dict(x=x[0]), "x must be"), (dict(w=w.half()), "w"), (dict(w=w[:63]), "w"),
                     (dict(q=q.float()), "q"), (dict(q=q[:, :63]), "q"), (dict(sc=sc[:2]), "sc"), (dict(sc=torch.zeros(3, 1, 2)), "sc"),
                     (dict(delta=x.half()), "delta"), (dict(delta=x[:2]), "delta"), (dict(res=x.t()), "res"), (dict(y=x[:, :32]), "y"),
                     (dict(x=x.t().contiguous().t()), "contiguous"), (dict(x=x[:1].expand(3, 64)), "overlap"), (dict(sc=None), "q")):
        with pytest.raises(ValueError, match=word):
            lk.norm_q8(**{**dict(x=x, w=w, q=q, sc=sc), **kw})
    a, b, o = lk.i8_rows(3, 50, device="cpu"), lk.i8_rows(5, 50, device="cpu"), torch.zeros(3, 5)
    sa, sb = torch.ones(3), torch.ones(5)
    assert a.shape == (3, 50) and a.stride(0) == 64
    with pytest.raises(ValueError, match="device memory"):
        lk.gemm_i8(a, sa, b, sb, o)
    for kw, word in ((dict(x=a.float()), "x"), (dict(x=a[:, :49]), "w"), (dict(sx=sa[:2]), "sx"), (dict(sw=sb.double()), "sw"),
                     (dict(out=o.double()), "fp32"), (dict(out=o.t()), "out"), (dict(res=o.half()), "res"), (dict(x=a[0]), "must be"),
                     (dict(x=torch.zeros(3, 50, dtype=torch.int8)), "storage"), (dict(w=b.t().contiguous().t()), "contiguous")):
        with pytest.raises(ValueError, match=word):
            lk.gemm_i8(**{**dict(x=a, sx=sa, w=b, sw=sb, out=o), **kw})


def test_mirror_refuses_what_an_int_cannot_count(lk_host):
    """Strides and counts past 2^31 - 1, which the C entry points take as int (meta tensors:
    shapes without memory)."""
    lk, big = lk_host, 2 ** 31
    m = lambda shape, dt=torch.float32, stride=None: torch.empty_strided(  # noqa: E731
        shape, stride or (shape[-1], 1)[-len(shape):], dtype=dt, device="meta")
    for x, q, sc in ((m((2, 8), stride=(big, 1)), m((2, 8), torch.int8), m((2,))), (m((big, 8)), m((big, 8), torch.int8), m((big,)))):
        with pytest.raises(ValueError, match="beyond"):
            lk.norm_q8(x, m((8,)), q, sc)
    with pytest.raises(ValueError, match="beyond"):
        lk.gemm_i8(m((2, 16), torch.int8, (2 * big, 1)), m((2,)), m((3, 16), torch.int8), m((3,)), m((2, 3)))


def _desc(lk, **kw):
    d = dict(n_experts=8, top_k=2, hidden=64, ffn=32, score=0, renorm=1, scale=1.0, router=0x1000, bias=None, gate_qs=0x1000,
             gate_d=0x1000, up_qs=0x1000, up_d=0x1000, down_qs=0x1000, down_d=0x1000)
    return lk.MoeDesc(**{**d, **kw})


def test_moe_c_refusals(lk_host):
    lib = lk_host.load()
    need = lib.lk_moe_work_bytes(ctypes.byref(_desc(lk_host)), 4)
    assert need > 0 and need % 16 == 0
    assert need < lib.lk_moe_work_bytes(ctypes.byref(_desc(lk_host)), 5)
    ok = dict(type=0, x=P, ldx=64, T=4, res=None, ldr=0, out=P, ldo=64, ids=None, weights=None, work=P, work_bytes=need, stream=None)

    def rc(desc={}, **kw):
        return lib.lk_moe_q4_0(ctypes.byref(_desc(lk_host, **desc)), *{**ok, **kw}.values())
    for bad in (dict(n_experts=0), dict(n_experts=257), dict(top_k=0), dict(top_k=9), dict(n_experts=1), dict(hidden=0), dict(hidden=48),
                dict(hidden=32800), dict(ffn=0), dict(ffn=40), dict(ffn=32800), dict(score=2), dict(score=-1)):
        assert rc(bad) == 1 and b"lk_moe" in lib.lk_last_error(), bad
        assert lib.lk_moe_work_bytes(ctypes.byref(_desc(lk_host, **bad)), 4) == 0, bad
    for bad in (dict(router=None), dict(gate_qs=None), dict(gate_d=None), dict(up_qs=None), dict(up_d=None), dict(down_qs=None),
                dict(down_d=None), dict(gate_qs=0x1008), dict(up_qs=0x1008), dict(down_qs=0x1008), dict(gate_d=0x1001),
                dict(router=0x1002), dict(bias=0x1002)):
        assert rc(bad) == 1 and b"lk_moe_q4_0" in lib.lk_last_error(), bad
    for bad in (dict(type=3), dict(T=-1), dict(T=65), dict(x=None), dict(out=None), dict(work=None), dict(work_bytes=need - 1),
                dict(work=ctypes.c_void_p(0x1008)), dict(ldx=63), dict(ldo=63), dict(res=P, ldr=63), dict(x=O), dict(out=O),
                dict(res=O, ldr=64), dict(ids=O), dict(weights=O)):
        assert rc(**bad) == 1 and b"lk_moe_q4_0" in lib.lk_last_error(), bad
    assert lib.lk_moe_q4_0(None, *ok.values()) == 1
    assert rc(T=0, x=None, out=None, work=None, work_bytes=0) == 0
    assert lib.lk_moe_work_bytes(None, 4) == 0 and lib.lk_moe_work_bytes(ctypes.byref(_desc(lk_host)), 65) == 0


def test_moe_mirror_refusals(lk_host):
    lk = lk_host
    q = lambda r, c: (torch.zeros(4, r, c // 32, 16, dtype=torch.uint8), torch.zeros(4, r, c // 32).half())  # noqa: E731
    ok = dict(router=torch.zeros(4, 64), gate=q(32, 64), up=q(32, 64), down=q(64, 32), top_k=2)
    with pytest.raises(ValueError, match="device memory"):
        lk.MoeQ4_0(**ok)
    for kw, word in ((dict(score="tanh"), "score"), (dict(router=torch.zeros(4)), "router"), (dict(router=torch.zeros(5, 64)), "gate"),
                     (dict(router=torch.zeros(4, 48)), "multiples"), (dict(gate=q(64, 32)), "gate"), (dict(up=q(32, 96)), "up"),
                     (dict(down=q(32, 64)), "down"), (dict(bias=torch.zeros(3)), "bias"), (dict(bias=torch.zeros(4).half()), "bias"),
                     (dict(gate=(ok["gate"][0], ok["gate"][1].float())), "gate scales")):
        with pytest.raises(ValueError, match=word):
            lk.MoeQ4_0(**{**ok, **kw})
    for kw, word in ((dict(top_k=0), "top_k"), (dict(top_k=5), "top_k"), (dict(max_tokens=65), "65 tokens")):
        with pytest.raises(lk.LkError, match=word):
            lk.MoeQ4_0(**{**ok, **kw})
