"""lk_paged_append without eps: heads of small values are normed as long as the mean of their squares is a
normal number of fp32, and are NaN below."""
import pytest
import torch

from gpu_util import note
from paged_util import Batch, append_ref, pool_type

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,dtype", [("f32", torch.float32), ("bf16", torch.bfloat16)])
@pytest.mark.parametrize("d", [64, 128])
def test_small_heads_without_eps(lk, t, dtype, d):
    b = Batch(1, [0], [5], 16)
    g = torch.Generator().manual_seed(d)
    # between 1 and 2, by a power of two a row
    x = (1 + torch.rand(5, d, generator=g)) * torch.tensor([1.0, 2.0 ** -40, 2.0 ** -62, 2.0 ** -66, 0.0])[:, None]
    x = x.to(dtype)
    w = torch.ones(d)
    k, v = (torch.zeros(b.n_pages, 16, 1, d, dtype=pool_type(t), device="cuda") for _ in range(2))
    out, cache = torch.empty(5, d, dtype=dtype, device="cuda"), lk.PagedCache(k, v, 1)
    note(f"small heads {t} {d}")
    cache.append(b.step(lk, max_new=5), x.cuda(), x.cuda(), q=x.cuda(), q_out=out, qn=w.cuda(), kn=w.cuda(), eps=0.0)
    torch.cuda.synchronize()
    want, tol = append_ref(x[:3].view(3, 1, d), w, torch.arange(3), None, 0, False, 0.0, dtype)
    got = out.cpu().double()
    assert bool(((got[:3] - want[:, 0]).abs() <= tol[:, 0]).all())
    assert bool(torch.isnan(got[3:]).all())
    kept = k.view(-1, d)[b.slots(0, 0, 5).cuda()].cpu()
    assert bool(torch.isfinite(kept[:3]).all()) and bool(torch.isnan(kept[3:]).all())
