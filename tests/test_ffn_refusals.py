"""What lk_norm_q8 and lk_gemm_i8 refuse, through the C ABI and through the Python
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
                dict(form=1, sc=ctypes.c_void_p(0x1004)), dict(form=2, q=O, sc=None), dict(type=1, x=O)):
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
                dict(w=ctypes.c_void_p(0x1008)), dict(sx=O), dict(sw=O), dict(out=O), dict(res=O, ldr=4)):
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
