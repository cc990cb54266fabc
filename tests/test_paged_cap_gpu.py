"""The tanh of capped scores, below 1/2 a series: what it leaves out is of one sign, so that it shows in
the mean over many scores, where roundings cancel."""
import math
import random

import pytest
import torch

from gpu_util import note
from paged_util import Batch

CAP, ROWS, HEADS, SEQS = 1024.0, 64, 64, 4


@pytest.mark.gpu
def test_the_series_of_tanh_leaves_out_less_than_a_rounding(lk):
    """Rows that see two keys each: one of score CAP tanh(t), t just below 1/2, and one whose score, t about 1/4, a bias by
    distance lifts to nearly the same.  Output: the first one's weight, a logistic function of the
    scores' difference, which is so measured to 1e-6.  The series leaves out 2^-26 of a score below 474, 7e-6;
    each of the 16384 differences is off by at most ten half steps of 512 (2^-15: the argument, series, two
    factors and sum of each score), of either sign: their mean by six times 10 * 2^-15 / sqrt(3 * 16384), 9e-6."""
    rng = random.Random(1)
    b = Batch(1, [0] * SEQS, [ROWS] * SEQS, 64)
    # pairs of tokens 2i, 2i + 1, so many positions apart
    apart = [rng.randrange(150, 250) for _ in range(ROWS // 2)]
    pos = [x for a in apart for x in (0, a)] * SEQS
    masks = [3 << (r // 2 * 2) for r in range(ROWS)] * SEQS
    q, want = torch.zeros(SEQS * ROWS, HEADS, 64, dtype=torch.float64), torch.empty(SEQS * ROWS, HEADS, dtype=torch.float64)
    for r in range(SEQS * ROWS):
        for h in range(HEADS):
            t = rng.uniform(0.47, 0.4995)
            d = apart[r % ROWS // 2]
            x = round(t * CAP * 256) / 256                      # both exact in two fp16 parts
            y = round(math.atanh(math.tanh(x / CAP) - (d + rng.uniform(-1, 1)) / CAP) * CAP * 256) / 256
            q[r, h, 0], q[r, h, 1] = x, y
            want[r, h] = CAP * (math.tanh(x / CAP) - math.tanh(y / CAP)) - d
    k, v = torch.zeros(b.n_pages, 64, 1, 64, dtype=torch.float16), torch.zeros(b.n_pages, 64, 1, 64, dtype=torch.float16)
    for s in range(SEQS):
        for i in range(ROWS):
            k.view(-1, 64)[b.slot(s, i), i % 2] = 1.0
            v.view(-1, 64)[b.slot(s, i)] = 1.0 - i % 2
    for hint in (1, 64):
        out = torch.empty(b.rows, HEADS * 64, device="cuda")
        note(f"capped scores, hint {hint}")
        lk.PagedCache(k.cuda(), v.cuda(), HEADS).attend(b.step(lk, pos=pos, mask=masks, max_new=hint), q.float().view(b.rows, -1).cuda(),
                                                        out, scale=1.0, cap=CAP, slopes=torch.ones(HEADS, device="cuda"))
        torch.cuda.synchronize()
        w = out.cpu().double().view(b.rows, HEADS, 64)[:, :, 0]
        off = torch.log(w / (1 - w)) - want
        assert float(off.abs().max()) <= 20 * 2.0 ** -15
        assert abs(float(off.mean())) <= 7e-6 + 9e-6, float(off.mean())
