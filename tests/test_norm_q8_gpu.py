"""The residual addition, RMS norm and 8-bit output in one kernel (lk_norm_q8) on
the GPU, through the Python mirror of the C ABI.

Every fp32 step of the definition rounds as written and the mean square is taken
in fp64, so h, y, quants and scales are compared bit for bit with the same steps on
the CPU (a different fp64 summation order moves the mean by about 2^-50, which
reaches the rounded 1/sqrt in about one row of 10^8).  Apart from that the values
that the quants stand for are held to the fp64 formula: y has at most 5 roundings
of fp32 (h, r, two products, a's division), the quantiser half a step.
"""
import numpy as np
import pytest
import torch

from ffn_util import TYPES, bits, guarded, norm_ref, q8_row_ref, same, untouched
from gpu_util import dev, host, note

pytestmark = pytest.mark.gpu


def _inputs(rows, n, dtype, seed, delta=True):
    g = torch.Generator().manual_seed(seed)
    chan = torch.exp(0.7 * torch.randn(n, generator=g))
    x = (torch.randn(rows, n, generator=g) * chan * 3).to(dtype)
    d = torch.randn(rows, n, generator=g).to(dtype) if delta else None
    return x, d, 0.5 + torch.rand(n, generator=g)


def _view(t, pad):
    buf, v = guarded(t.shape[0], t.shape[1], t.dtype, pad)
    v.copy_(t)
    return v


# rows, n: a single value, one side and the other of every launch shape (512, 2048,
# 8192 values), tails of one to seven values, the longest row
SHAPES = [(1, 1), (3, 7), (1, 33), (6, 511), (5, 512), (9, 513), (4, 1000), (3, 2048), (7, 2049), (2, 8191), (2, 8192),
          (3, 8193), (1, 32768), (130, 96)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,n", SHAPES)
def test_row_form(lk, rows, n, t):
    dt = TYPES[t]
    pad = (0, 1, 16)[(rows + n) % 3]
    x, d, w = _inputs(rows, n, dt, rows * 7 + n, delta=n % 2 == 0 or rows == 1)
    note(f"norm_q8 row form {rows}x{n} {t} pad {pad}")
    rb, r = guarded(rows, n, dt, pad)
    yb, y = guarded(rows, n, dt, pad + 1)
    qb, q = guarded(rows, n, torch.int8, 3)
    sc = torch.full((rows + 1,), 77.0, device="cuda")
    lk.norm_q8(_view(x, pad), w.cuda(), q, sc[:rows], delta=None if d is None else _view(d, pad + 2), res=r, y=y, eps=1e-5)
    torch.cuda.synchronize()
    h1, y1 = norm_ref(x, d, w, 1e-5)
    q1, s1 = q8_row_ref(y1)
    assert np.array_equal(bits(r), bits(h1.to(dt))) and np.array_equal(bits(y), bits(y1.to(dt)))
    assert np.array_equal(host(q), q1.numpy()) and np.array_equal(bits(sc[:rows]), bits(s1))
    assert untouched(rb, rows, n) and untouched(yb, rows, n) and untouched(qb, rows, n) and sc[rows].item() == 77.0
    # against the formula in 64 bits
    h = x.double() + (0 if d is None else d.double())
    ref = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5) * w.double()
    step = sc[:rows].cpu().double()[:, None]
    off = (q.cpu().double() * step - ref).abs()
    # eps is 1e-5 rounded to fp32 (2^-24 of it, at most as much of r): one more rounding
    assert bool((off <= step / 2 + 8 * 2.0 ** -24 * ref.abs().amax(-1, keepdim=True)).all())


@pytest.mark.parametrize("rows,n", [(9, 512), (3, 513), (5, 1024), (3, 1025), (2, 4096), (3, 4097), (2, 8192), (2, 8193), (1, 16384),
                                    (2, 16385)])
def test_row_form_at_the_lines_between_launch_shapes(lk, rows, n):
    """One value more or less than the lanes of a launch shape hold."""
    test_row_form(lk, rows, n, list(TYPES)[(rows + n) % 3])


@pytest.mark.parametrize("t", TYPES)
def test_many_rows(lk, t):
    """Eight million values: those next to a rounding border among them."""
    test_row_form(lk, 4096, 2048, t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 32), (5, 64), (3, 2048), (2, 2080), (3, 4128), (1, 8224), (67, 256)])
def test_q81_forms_are_the_quantisers_bytes(lk, rows, n, t):
    """Planar Q8_1 byte for byte what lk_pf_quant_rows makes of the normed fp32 row,
    and the blocks the same quants with the raw sum."""
    dt = TYPES[t]
    x, d, w = _inputs(rows, n, dt, 3 * rows + n)
    x[0, :32] = 0                                        # a block of zeros
    if d is not None:
        d[0, :32] = 0
    note(f"norm_q8 Q8_1 forms {rows}x{n} {t}")
    q = torch.empty(rows, n, dtype=torch.int8, device="cuda")
    sc = torch.empty(rows, n // 32, 2, device="cuda")
    blk = torch.empty(rows, n // 32 * 36, dtype=torch.uint8, device="cuda")
    lk.norm_q8(_view(x, 8), w.cuda(), q, sc, delta=_view(d, 0))
    lk.norm_q8(_view(x, 8), w.cuda(), blk, delta=_view(d, 0))
    _, y = norm_ref(x, d, w, 1e-5)
    q1, sc1 = torch.empty_like(q), torch.empty_like(sc)
    lk.pf_quant_rows(y.cuda(), rows, n, n // 32, q1, sc1)
    torch.cuda.synchronize()
    assert torch.equal(q, q1) and np.array_equal(bits(sc), bits(sc1))
    b = host(blk).reshape(rows, n // 32, 36)
    assert np.array_equal(b[..., 4:].view(np.int8).reshape(rows, n), host(q))
    ds = b[..., :4].copy().view(np.float16).astype(np.float32)
    assert np.array_equal(ds[..., 0], host(sc)[..., 0]) and np.array_equal(8 * ds[..., 1], host(sc)[..., 1])


def test_in_place(lk):
    """res in x's own rows, and in delta's; y over x."""
    for t, dt in TYPES.items():
        x, d, w = _inputs(5, 1001, dt, 11)
        note(f"norm_q8 in place {t}")
        h1, y1 = norm_ref(x, d, w, 1e-5)
        q1, s1 = q8_row_ref(y1)
        q, sc = torch.empty(5, 1001, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
        a, b = x.cuda(), d.cuda()
        lk.norm_q8(a, w.cuda(), q, sc, delta=b, res=a)
        assert np.array_equal(bits(a), bits(h1.to(dt))) and np.array_equal(host(q), q1.numpy())
        a, b = x.cuda(), d.cuda()
        lk.norm_q8(a, w.cuda(), q, sc, delta=b, res=b, y=a)
        assert np.array_equal(bits(b), bits(h1.to(dt))) and np.array_equal(bits(a), bits(y1.to(dt)))


def test_rows_that_are_not_numbers(lk):
    """An infinity or a NaN makes its own row NaN with zero quants, and no other; rows
    of zeros and of the smallest values give zeros; the largest finite values do not
    overflow the sum of squares."""
    n = 700
    for t, dt in TYPES.items():
        x, _, w = _inputs(8, n, dt, 5, delta=False)
        x[1, 13], x[2, 699], x[3, 0] = float("inf"), float("nan"), -float("inf")
        x[4] = 0
        x[5] = torch.finfo(dt).smallest_normal
        x[6] = torch.finfo(dt).max * torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)
        note(f"norm_q8 rows that are not numbers {t}")
        q, sc = torch.empty(8, n, dtype=torch.int8, device="cuda"), torch.empty(8, device="cuda")
        y = torch.empty(8, n, dtype=dt, device="cuda")
        lk.norm_q8(x.cuda(), w.cuda(), q, sc, y=y, eps=1e-5)
        _, y1 = norm_ref(x, None, w, 1e-5)
        q1, s1 = q8_row_ref(y1)
        assert same(sc, s1) and np.array_equal(host(q), q1.numpy()) and same(y, y1.to(dt))
        assert torch.isnan(sc[1:4]).all() and torch.isfinite(sc[4:]).all() and not q[1:5].any()
        # eps 0: a row of zeros has no norm
        lk.norm_q8(x.cuda(), w.cuda(), q, sc, eps=0.0)
        assert torch.isnan(sc[4]).item() and torch.isfinite(sc[0]).item()


def test_small_scales(lk):
    """Weights that bring a row's largest value to both sides of 2^-120."""
    x = torch.randn(2, 64, generator=torch.Generator().manual_seed(3))
    for e in (-100, -118, -119, -121, -122, -140):
        w = torch.full((64,), 2.0 ** e)
        q, sc = torch.empty(2, 64, dtype=torch.int8, device="cuda"), torch.empty(2, device="cuda")
        lk.norm_q8(x.cuda(), w.cuda(), q, sc)
        _, y = norm_ref(x, None, w, 1e-5)
        q1, s1 = q8_row_ref(y)
        assert np.array_equal(host(q), q1.numpy()) and np.array_equal(bits(sc), bits(s1)), e
    assert not q.any() and not sc.any()


def test_no_rows(lk):
    e = torch.empty(0, 64, device="cuda")
    lk.norm_q8(e, torch.ones(64, device="cuda"), torch.empty(0, 64, dtype=torch.int8, device="cuda"),
               torch.empty(0, device="cuda"), res=e, y=e)


def test_side_stream_and_graph(lk):
    """On a stream of its own, and captured once and replayed over new inputs."""
    x, d, w = _inputs(37, 2048, torch.bfloat16, 8)
    xd, dd, wd = x.cuda(), d.cuda(), w.cuda()
    q, sc = torch.empty(37, 2048, dtype=torch.int8, device="cuda"), torch.empty(37, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    note("norm_q8 on a side stream and in a graph")
    lk.norm_q8(xd, wd, q, sc, delta=dd, res=xd, stream=st)
    st.synchronize()
    h1, y1 = norm_ref(x, d, w, 1e-5)
    assert np.array_equal(host(q), q8_row_ref(y1)[0].numpy())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lk.norm_q8(xd, wd, q, sc, delta=dd, res=xd)
    for k in range(3):
        x, d, _ = _inputs(37, 2048, torch.bfloat16, 20 + k)
        xd.copy_(x)
        dd.copy_(d)
        g.replay()
        torch.cuda.synchronize()
        h1, y1 = norm_ref(x, d, w, 1e-5)
        q1, s1 = q8_row_ref(y1)
        assert np.array_equal(host(q), q1.numpy()) and np.array_equal(bits(sc), bits(s1))
        assert np.array_equal(bits(xd), bits(h1.bfloat16()))
