"""What lk_paged_append, lk_paged_attn and lk_paged_commit refuse, through the C ABI and
through the Python mirror.  CPU only: every call here fails its checks, or has nothing to do,
before anything is launched."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(0x1000)      # never dereferenced
O = ctypes.c_void_p(0x1001)
F = ctypes.c_float


def _pages(lk, **kw):
    return lk.Pages(**{**dict(type=1, n_heads=32, n_kv_heads=8, head_dim=64, page=64, n_pages=10, k=0x1000, v=0x1000), **kw})


def _step(lk, **kw):
    return lk.Step(**{**dict(n_seqs=2, rows=3, first=0x1000, lens=0x1000, table=0x1000, ldt=8, width=8, pos=None, mask=None,
                             max_new=0), **kw})


BAD_PAGES = (dict(type=0), dict(type=3), dict(head_dim=0), dict(head_dim=96), dict(head_dim=256), dict(n_heads=0), dict(n_kv_heads=0),
             dict(n_heads=31), dict(n_heads=4), dict(n_heads=264), dict(n_heads=130, n_kv_heads=2), dict(page=0), dict(page=8),
             dict(page=48), dict(page=131072))
BAD_POOLS = (dict(n_pages=0), dict(k=None), dict(v=None), dict(k=0x1008), dict(v=0x1002))
BAD_STEP = (dict(n_seqs=-1), dict(rows=-1), dict(max_new=-1), dict(n_seqs=2 ** 20 + 1), dict(rows=2 ** 24 + 1), dict(width=0),
            dict(ldt=7), dict(width=2 ** 24 + 1, ldt=2 ** 24 + 1), dict(first=None), dict(lens=None), dict(table=None),
            dict(first=0x1002), dict(lens=0x1001), dict(table=0x1002), dict(pos=0x1002), dict(mask=0x1004))


def _descriptions(lk, rc, word):
    lib = lk.load()
    for bad in BAD_PAGES + BAD_POOLS:
        assert rc(pages=_pages(lk, **bad)) == 1 and word in lib.lk_last_error(), bad
    for bad in BAD_STEP:
        assert rc(step=_step(lk, **bad)) == 1 and word in lib.lk_last_error(), bad
    assert rc(pages=None) == 1 and rc(step=None) == 1
    empty = dict(first=None, lens=None, table=None)
    assert rc(step=_step(lk, n_seqs=0, **empty)) == 0


def test_append_c_refusals(lk_host):
    lk = lk_host
    f = lk.load().lk_paged_append
    ok = dict(pages=_pages(lk), step=_step(lk), type=1, q=P, ldq=2048, k=P, ldk=512, v=P, ldv=512, qn=P, kn=P, eps=F(1e-5),
              freq=P, rot=64, style=0, qo=P, ldqo=2048, stream=None)

    def rc(**kw):
        a = {**ok, **kw}
        for n in ("pages", "step"):
            a[n] = None if a[n] is None else ctypes.byref(a[n])
        return f(*a.values())
    _descriptions(lk, rc, b"lk_paged_append")
    for bad in (dict(type=2), dict(type=3), dict(type=-1), dict(style=2), dict(style=-1), dict(rot=8), dict(rot=80), dict(rot=-16),
                dict(rot=0), dict(freq=None), dict(eps=F(-1.0)), dict(eps=F(float("nan"))), dict(k=None), dict(v=None), dict(qo=None),
                dict(q=None), dict(ldq=2047), dict(ldk=511), dict(ldv=511), dict(ldqo=2047), dict(q=O), dict(k=O), dict(v=O), dict(qo=O),
                dict(type=0, k=ctypes.c_void_p(0x1002)), dict(qn=ctypes.c_void_p(0x1004)), dict(kn=O), dict(freq=ctypes.c_void_p(0x1008))):
        assert rc(**bad) == 1 and b"lk_paged_append" in lk.load().lk_last_error(), bad
    assert rc(pages=_pages(lk, type=2)) == 1                # fp16 rows with bf16 pools
    assert rc(step=_step(lk, rows=0), k=None) == 0


def test_attn_c_refusals(lk_host):
    lk = lk_host
    lib = lk.load()
    need = lib.lk_paged_attn_work_bytes(ctypes.byref(_pages(lk)), 1, 0)
    assert need > 0 and need % 16 == 0
    ok = dict(pages=_pages(lk), step=_step(lk), type=1, q=P, ldq=2048, scale=F(0.125), cap=F(0.0), slopes=None, out=P, ldo=2048,
              work=P, work_bytes=need, stream=None)

    def rc(**kw):
        a = {**ok, **kw}
        for n in ("pages", "step"):
            a[n] = None if a[n] is None else ctypes.byref(a[n])
        return lib.lk_paged_attn(*a.values())
    _descriptions(lk, rc, b"lk_paged_attn")
    inf, nan = float("inf"), float("nan")
    for bad in (dict(type=2), dict(type=3), dict(scale=F(0.0)), dict(scale=F(-1.0)), dict(scale=F(inf)), dict(scale=F(nan)), dict(cap=F(-1.0)), dict(cap=F(1e-31)),
                dict(cap=F(inf)), dict(cap=F(nan)), dict(q=None), dict(out=None), dict(work=None), dict(work_bytes=need - 1),
                dict(work=ctypes.c_void_p(0x1008)), dict(ldq=2047), dict(ldo=2047), dict(q=O), dict(out=O),
                dict(slopes=ctypes.c_void_p(0x1002)), dict(type=0, q=ctypes.c_void_p(0x1002)),
                dict(step=_step(lk, max_new=64))):          # a larger workspace is needed for trees
        assert rc(**bad) == 1 and b"lk_paged_attn" in lib.lk_last_error(), bad
    assert rc(step=_step(lk, rows=0), q=None, work=None, work_bytes=0) == 0
    for bad in BAD_PAGES:
        assert lib.lk_paged_attn_work_bytes(ctypes.byref(_pages(lk, **bad)), 1, 0) == 0, bad
    assert lib.lk_paged_attn_work_bytes(None, 1, 0) == 0
    assert lib.lk_paged_attn_work_bytes(ctypes.byref(_pages(lk)), 2, 0) == 0
    assert lib.lk_paged_attn_work_bytes(ctypes.byref(_pages(lk)), 1, -1) == 0


@pytest.mark.parametrize("d", [64, 128])
def test_workspace_of_every_shape(lk_host, d):
    """Every layout and hint has a workspace; it does not depend on the batch or on the pools."""
    lk, lib = lk_host, lk_host.load()
    for ty, pool in ((0, 1), (1, 1), (2, 2)):
        for hkv in (1, 2, 3, 4, 8, 12, 64):
            for g in (1, 2, 3, 4, 7, 16, 33, 64):
                if hkv * g > 256:
                    continue
                p = _pages(lk, type=pool, n_heads=hkv * g, n_kv_heads=hkv, head_dim=d, n_pages=0, k=None, v=None)
                for n in (0, 1, 2, 5, 16, 64, 65, 100000):
                    w = lib.lk_paged_attn_work_bytes(ctypes.byref(p), ty, n)
                    assert 0 < w <= 160 << 20 and w % 16 == 0, (ty, hkv, g, n, w)


def test_commit_c_refusals(lk_host):
    lk, lib = lk_host, lk_host.load()
    ok = dict(pages=_pages(lk), step=_step(lk), path=P, ldp=8, count=P, new_lens=P, stream=None)

    def rc(**kw):
        a = {**ok, **kw}
        for n in ("pages", "step"):
            a[n] = None if a[n] is None else ctypes.byref(a[n])
        return lib.lk_paged_commit(*a.values())
    _descriptions(lk, rc, b"lk_paged_commit")
    for bad in (dict(ldp=0), dict(ldp=65), dict(count=None), dict(new_lens=None), dict(path=O), dict(count=O), dict(new_lens=O)):
        assert rc(**bad) == 1 and b"lk_paged_commit" in lib.lk_last_error(), bad


def test_mirror_refusals(lk_host):
    lk = lk_host
    k = torch.zeros(3, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="device memory"):
        lk.PagedCache(k, k, 4)
    for a, b, word in ((k.double(), k, "fp32, fp16 or bf16"), (k[0], k[0], "pools must be")):
        with pytest.raises(ValueError, match=word):
            lk.PagedCache(a, b, 4)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="device memory"):
        lk.PagedStep(i(3), i(2), i(2, 4), 5)
    for a in ((i(3), i(2, 1), i(2, 4), 5), (i(3), i(2), i(4), 5)):
        with pytest.raises(ValueError, match="lens must be"):
            lk.PagedStep(*a)
