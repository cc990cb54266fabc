"""Outputs over the queries in rows of another stride: a row would be written over queries that are still to
be read.  lk_paged_append and lk_paged_attn refuse it.  CPU only: nothing is launched."""
import ctypes

import pytest

P = ctypes.c_void_p(0x1000)      # never dereferenced
F = ctypes.c_float


@pytest.mark.parametrize("other", [2052, 4096])
def test_output_over_queries_of_another_stride(lk_host, other):
    lk, lib = lk_host, lk_host.load()
    pages = lk.Pages(type=1, n_heads=32, n_kv_heads=8, head_dim=64, page=64, n_pages=10, k=0x1000, v=0x1000)
    step = lk.Step(n_seqs=2, rows=3, first=0x1000, lens=0x1000, table=0x1000, ldt=8, width=8, pos=None, mask=None, max_new=0)
    p, s = ctypes.byref(pages), ctypes.byref(step)
    need = lib.lk_paged_attn_work_bytes(p, 1, 0)
    for ldq, ldo in ((2048, other), (other, 2048)):
        assert lib.lk_paged_attn(p, s, 1, P, ldq, F(0.125), F(0.0), None, P, ldo, P, need, None) == 1
        assert b"over queries" in lib.lk_last_error()
        assert lib.lk_paged_append(p, s, 1, P, ldq, P, 512, P, 512, P, P, F(1e-5), P, 64, 0, P, ldo, None) == 1
        assert b"over queries" in lib.lk_last_error()
