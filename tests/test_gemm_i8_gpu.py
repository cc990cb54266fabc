"""The int8 product with scales for each token and channel (lk_gemm_i8) on the GPU.

The sums are exact and the steps behind them round as written, so every case is
compared bit for bit with the same steps on the CPU (the sum in fp64, exact below
2^53).  The bytes between K and a row's next multiple of 16 hold garbage.
"""
import numpy as np
import pytest
import torch

from ffn_util import TYPES, bits, gemm_ref, guarded, untouched
from gpu_util import host, note

pytestmark = pytest.mark.gpu


def _rows(g, rows, K, pad=0):
    """(the int8 rows, a device view of them with garbage around and between)"""
    q = torch.randint(-128, 128, (rows, K), generator=g, dtype=torch.int8)
    buf = torch.full((rows, (K + 15) // 16 * 16 + pad), 99, dtype=torch.int8)
    buf[:, :K] = q
    return q, buf.cuda()[:, :K]


def _case(lk, M, N, K, dt, res, pad, seed):
    g = torch.Generator().manual_seed(seed)
    x, xd = _rows(g, M, K, pad)
    w, wd = _rows(g, N, K)
    sx, sw = 0.01 + torch.rand(M, generator=g), (0.01 + torch.rand(N, generator=g)) / 64 / K
    r = (torch.randn(M, N, generator=g) * 30).to(dt) if res else None
    ob, out = guarded(M, N, dt, pad % 5)
    lk.gemm_i8(xd, sx.cuda(), wd, sw.cuda(), out, res=None if r is None else r.cuda())
    torch.cuda.synchronize()
    want = gemm_ref(x, sx, w, sw, dt, r)
    assert np.array_equal(bits(out), bits(want))
    assert untouched(ob, M, N)


# token counts on both sides of every launch shape's line, sizes off every tile, K
# of one byte, one short of and past 16, 64 and 128 bytes
MS = [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 100, 257]
NKS = [(1, 1), (16, 64), (17, 63), (5, 65), (100, 15), (64, 127), (129, 128), (300, 129), (48, 1111), (33, 2048)]


@pytest.mark.parametrize("M", MS)
@pytest.mark.parametrize("N,K", NKS)
def test_small_shapes_bit_exact(lk, M, N, K):
    dt = list(TYPES.values())[(M + N + K) % 3]
    note(f"gemm_i8 M={M} N={N} K={K} {dt}")
    _case(lk, M, N, K, dt, (M + K) % 2 == 0, (0, 16, 48)[(M + N) % 3], M * 1000 + N + K)


@pytest.mark.parametrize("M,N,K", [(2100, 2000, 100), (2048, 2048, 256), (4097, 4100, 80), (4096, 4096, 448),
                                   (1, 5000, 4100), (24, 2048, 8192), (333, 2048, 2048), (512, 1030, 640),
                                   (700, 130, 1040)])
@pytest.mark.parametrize("res", [False, True])
def test_large_shapes_bit_exact(lk, M, N, K, res):
    dt = TYPES["f32"] if res else TYPES["bf16"]
    note(f"gemm_i8 M={M} N={N} K={K} {dt} res={res}")
    _case(lk, M, N, K, dt, res, 0, M + N + K)


# tile counts on both sides of every line between the tiles: 32x32 / 64x32 / 64x64 /
# 128x64 / 128x128 (one and two workgroups a unit) / 256x256; ragged in every direction
@pytest.mark.parametrize("M,N,K", [(16, 4096, 300), (16, 4097, 300), (130, 1650, 515), (250, 2040, 260), (257, 2050, 1025),
                                   (500, 2040, 130), (513, 2049, 129), (1000, 1030, 385), (1020, 2047, 641), (1030, 2050, 300),
                                   (2000, 2020, 257), (2060, 2049, 129), (4090, 2040, 200), (3000, 4090, 400)])
def test_lines_between_tiles_bit_exact(lk, M, N, K):
    dt = list(TYPES.values())[(M + N) % 3]
    note(f"gemm_i8 M={M} N={N} K={K} {dt}")
    _case(lk, M, N, K, dt, (M + N + K) % 2 == 1, 16, M + N + K)


@pytest.mark.parametrize("M,N,K", [(1, 16385, 70), (17, 16500, 260), (32, 20001, 515), (33, 16390, 130)])
def test_few_tokens_and_many_rows_bit_exact(lk, M, N, K):
    dt = list(TYPES.values())[M % 3]
    note(f"gemm_i8 M={M} N={N} K={K} {dt}")
    _case(lk, M, N, K, dt, M % 2 == 1, 16, M + N + K)


# more tiles than the units hold at once, so that a workgroup goes on to a second and third, with one,
# two and three stages of K (the ring's place changes from tile to tile, or not)
@pytest.mark.parametrize("M,N,K", [(4100, 8200, 100), (4100, 8200, 130), (4100, 8200, 300), (2600, 8190, 300), (2600, 8190, 128)])
def test_workgroups_of_several_tiles_bit_exact(lk, M, N, K):
    dt = TYPES["bf16"] if K != 130 else TYPES["f32"]
    note(f"gemm_i8 M={M} N={N} K={K} {dt}")
    _case(lk, M, N, K, dt, K == 130, 0, M + N + K)


@pytest.mark.parametrize("M", [1, 40])
def test_largest_sums(lk, M):
    """-128 * -128 over the longest K: 2^31 - 2^14, the int32 range's end; and its
    negative with 127."""
    K = 131071
    x = torch.full((M, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    w = torch.full((3, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    w[1] = 127
    w[2, 1:] = 0
    out = torch.empty(M, 3, device="cuda")
    one = torch.ones(M, device="cuda"), torch.ones(3, device="cuda")
    note(f"gemm_i8 largest sums M={M}")
    lk.gemm_i8(x, one[0], w, one[1], out)
    want = torch.tensor([K * 16384, -K * 128 * 127, 16384], dtype=torch.float64).float()
    assert torch.equal(out.cpu(), want.expand(M, 3))


def test_scales_that_are_not_numbers(lk):
    """A row's NaN scale makes its outputs NaN and no others."""
    g = torch.Generator().manual_seed(1)
    for M in (5, 70):
        _, x = _rows(g, M, 200)
        _, w = _rows(g, 90, 200)
        sx, sw = torch.ones(M), torch.ones(90)
        sx[3] = float("nan")
        sw[11] = float("inf")
        out = torch.empty(M, 90, device="cuda")
        note(f"gemm_i8 NaN scales M={M}")
        lk.gemm_i8(x, sx.cuda(), w, sw.cuda(), out)
        o = out.cpu()
        fine = torch.ones(M, 90, dtype=torch.bool)
        fine[3], fine[:, 11] = False, False
        assert torch.isnan(o[3]).all() and torch.isfinite(o[fine]).all()
        assert not torch.isfinite(o[[i for i in range(M) if i != 3], 11]).any()


def test_residual_in_place_and_no_rows(lk):
    g = torch.Generator().manual_seed(2)
    for M in (3, 50):
        x, xd = _rows(g, M, 96)
        w, wd = _rows(g, 70, 96)
        sx, sw = torch.rand(M, generator=g), torch.rand(70, generator=g)
        r = torch.randn(M, 70, generator=g) * 1000
        out = r.cuda()
        note(f"gemm_i8 residual in place M={M}")
        lk.gemm_i8(xd, sx.cuda(), wd, sw.cuda(), out, res=out)
        assert np.array_equal(bits(out), bits(gemm_ref(x, sx, w, sw, torch.float32, r)))
    e = torch.empty(0, 70, device="cuda")
    lk.gemm_i8(xd[:0], sx[:0].cuda(), wd, sw.cuda(), e)


def test_side_stream_and_graph(lk):
    g = torch.Generator().manual_seed(4)
    w, wd = _rows(g, 500, 320)
    sw = torch.rand(500, generator=g)
    for M in (9, 300):
        x, xd = _rows(g, M, 320)
        sx = torch.rand(M, generator=g)
        sxd, swd, out = sx.cuda(), sw.cuda(), torch.zeros(M, 500, device="cuda")
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        note(f"gemm_i8 on a side stream and in a graph M={M}")
        lk.gemm_i8(xd, sxd, wd, swd, out, stream=st)
        st.synchronize()
        assert np.array_equal(bits(out), bits(gemm_ref(x, sx, w, sw, torch.float32)))
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            lk.gemm_i8(xd, sxd, wd, swd, out)
        for _ in range(3):
            x = torch.randint(-128, 128, (M, 320), generator=g, dtype=torch.int8)
            xd.copy_(x)
            out.zero_()
            gr.replay()
            torch.cuda.synchronize()
            assert np.array_equal(bits(out), bits(gemm_ref(x, sx, w, sw, torch.float32)))
