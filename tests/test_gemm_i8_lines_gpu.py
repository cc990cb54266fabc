"""The int8 product at both sides of the line between the kernel for few tokens and the smallest
tiles, on the GPU, bit for bit (see test_gemm_i8_gpu.py)."""
import pytest

from ffn_util import TYPES
from gpu_util import note
from test_gemm_i8_gpu import _case

pytestmark = pytest.mark.gpu


# M K up to 16384 with up to 4096 rows (any M up to 16 where K is up to 2048), up to 8192 with 8192
@pytest.mark.parametrize("M,N,K", [(16, 4096, 2048), (16, 4096, 2049), (8, 4096, 2048), (8, 300, 2049), (7, 300, 2340), (7, 300, 2341),
                                   (2, 1000, 8192), (2, 1000, 8193), (1, 500, 16384), (1, 500, 16385), (16, 17, 130), (4, 8192, 2048),
                                   (5, 8192, 1638), (5, 8192, 1639), (16, 5000, 512), (16, 5000, 513), (17, 4096, 64), (1, 8193, 2048)])
def test_few_tokens_or_tiles_bit_exact(lk, M, N, K):
    dt = list(TYPES.values())[(M + N + K) % 3]
    note(f"gemm_i8 M={M} N={N} K={K} {dt}")
    _case(lk, M, N, K, dt, K % 2 == 1, (0, 16)[M % 2], M * 7 + N + K)
