"""lk_norm_q8 where y, or 1 / sqrt, leaves fp32's range, on the GPU: bit for bit the
definition's steps, as in test_norm_q8_gpu.py."""
import numpy as np
import pytest
import torch

from ffn_util import TYPES, bits, norm_ref, q8_row_ref, same
from gpu_util import host, note

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES)
def test_weights_that_take_y_out_of_range(lk, t):
    """Finite rows, a weight that makes one value of y infinite: scale NaN and quants 0, y as
    computed, the other values finite; in the Q8_1 forms the block alone, with the bytes of
    lk_pf_quant_rows."""
    rows, n, dt = 5, 224, TYPES[t]
    x = torch.randn(rows, n, generator=torch.Generator().manual_seed(3)).to(dt)
    x[:, 70] = 8.0
    x[3, 70] = 0.0                                       # this row stays finite
    w = torch.ones(n)
    w[70] = torch.finfo(torch.float32).max
    note(f"norm_q8 weights out of range {t}")
    q, sc = torch.empty(rows, n, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    res, y = torch.empty(rows, n, dtype=dt, device="cuda"), torch.empty(rows, n, dtype=dt, device="cuda")
    lk.norm_q8(x.cuda(), w.cuda(), q, sc, res=res, y=y)
    pq, psc = torch.empty_like(q), torch.empty(rows, n // 32, 2, device="cuda")
    lk.norm_q8(x.cuda(), w.cuda(), pq, psc)
    h1, y1 = norm_ref(x, None, w, 1e-5)
    q1, s1 = q8_row_ref(y1)
    q2, sc2 = torch.empty_like(q), torch.empty_like(psc)
    lk.pf_quant_rows(y1.cuda(), rows, n, n // 32, q2, sc2)
    torch.cuda.synchronize()
    assert torch.isnan(sc[[0, 1, 2, 4]]).all() and torch.isfinite(sc[3]) and not q[[0, 1, 2, 4]].any()
    assert same(sc, s1) and np.array_equal(host(q), q1.numpy())
    assert np.array_equal(bits(y), bits(y1.to(dt))) and np.array_equal(bits(res), bits(h1.to(dt)))
    assert bool((torch.isinf(y[[0, 1, 2, 4]]).sum(1) == 1).all())
    assert torch.equal(pq, q2) and same(psc, sc2) and torch.isfinite(psc[:, [0, 1, 3, 4, 5, 6]]).all()


def test_eps_of_zero(lk):
    """With eps 0 a row of zeros has 1 / sqrt(0): NaN, like 0 times infinity; other rows are as
    with any eps."""
    n = 300
    x = torch.randn(4, n, generator=torch.Generator().manual_seed(4))
    x[1] = 0
    w = torch.ones(n)
    note("norm_q8 eps 0")
    q, sc, y = torch.empty(4, n, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda"), torch.empty(4, n, device="cuda")
    lk.norm_q8(x.cuda(), w.cuda(), q, sc, y=y, eps=0.0)
    torch.cuda.synchronize()
    assert torch.isnan(sc[1]) and not q[1].any() and torch.isnan(y[1]).all()
    rows = [0, 2, 3]
    _, y1 = norm_ref(x[rows], None, w, 0.0)
    q1, s1 = q8_row_ref(y1)
    assert same(y[rows], y1) and same(sc[rows], s1) and np.array_equal(host(q[rows]), q1.numpy())
