"""The choice of experts of lk_moe_q4_0 where a lane holds more than one of them (more than 64
experts), on the GPU, in every kind of launch: up to 5 tokens, 8, up to 16, 32 and 64.

Tokens are unit vectors and router rows multiples of 1/32, so that a logit is a
product by one and sums of zeros: exact in fp32, as is the order of the logits.  Scores next to
each other differ by at least 1/32 of sigmoid's slope, 5e-4 at the ends (-4 and 4); biases
are 0 or 2, and the sum rounds by 2^-23.
"""
import pytest
import torch

from ffn_util import TYPES, moe_ref
from gpu_util import note
from test_moe_gpu import _close, _layer, _make, _run

pytestmark = pytest.mark.gpu

H, F = 64, 32


def _exact(seed, E, T, bias):
    """(layer, rows): every column of the router a permutation of E multiples of 1/32."""
    g = torch.Generator().manual_seed(seed)
    L = _layer(seed, E, H, F)
    for c in range(H):
        L["router"][:, c] = (torch.randperm(E, generator=g) - E // 2) / 32.0
    if bias:
        L["bias"] = torch.zeros(E)
        L["bias"][torch.randperm(E, generator=g)[:3]] = 2.0
    x = torch.zeros(T, H)
    x[torch.arange(T), torch.randperm(H, generator=g)[:T]] = 1.0
    return L, x


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T", [1, 5, 8, 12, 24, 33, 64])
@pytest.mark.parametrize("E", [64, 65, 100, 128, 129, 200, 256])
def test_many_experts(lk, E, T, score):
    k, t = 8 if E != 100 else 5, list(TYPES)[(E + T) % 3]
    L, x = _exact(E + T, E, T, score == "sigmoid")
    x = x.to(TYPES[t])
    note(f"moe choice E={E} T={T} k={k} {score} {t}")
    out, ids, w = _run(lk, _make(lk, L, k, score=score, max_tokens=T), x, H, TYPES[t], k)
    want, ids1, w1 = moe_ref(x, k=k, score=score, **L)
    assert torch.equal(ids.long(), ids1)
    # exp and the divisions: a few roundings of 2^-24; the softmax' sum of 256 terms by a tree: 10 more
    assert bool(((w.double() - w1).abs() <= 24 * 2.0 ** -24 * w1).all())
    _close(out, want, TYPES[t], (E, T, score))
    if T == 64:
        assert set((ids // 64).flatten().tolist()) == set(range((E + 63) // 64))    # from every register


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T", [1, 5, 8, 12, 24, 64])
@pytest.mark.parametrize("E", [65, 128, 130, 256])
def test_ties_across_a_lanes_experts(lk, E, T, score):
    """Equal logits at both sides of 64, 128 and 192, and at the last: the lowest index first."""
    L, x = _exact(3 * E + T, E, T, False)
    top = [e for e in (191, 62, 64, 127, 63, 128, 192, E - 1, 0, 129) if e < E]
    L["router"][top] = 5.0
    if score == "sigmoid":
        L["bias"] = torch.full((E,), 0.5)                # the sums tie as well
    note(f"moe ties E={E} T={T} {score}")
    k = min(8, len(set(top)))
    _, ids, w = _run(lk, _make(lk, L, k, score=score, max_tokens=T), x, H, torch.float32, k)
    assert torch.equal(ids, torch.tensor(sorted(set(top))[:k], dtype=torch.int32).expand(T, k))
    assert bool((w - 1.0 / k).abs().max() <= 4 * 2.0 ** -24)


@pytest.mark.parametrize("T", [1, 8, 12, 64])
def test_all_scores_masked_but_some(lk, T):
    """Biases of minus infinity and of the type's lowest value leave fewer experts than are chosen:
    first those that are left, then by bias, then by index."""
    E, k, lowest = 200, 6, torch.finfo(torch.float32).min
    L, x = _exact(77, E, T, False)
    L["bias"] = torch.full((E,), -float("inf"))
    L["bias"][[70, 150]] = 0.0
    L["bias"][[199, 66]] = lowest
    note(f"moe masked experts T={T}")
    _, ids, w = _run(lk, _make(lk, L, k, max_tokens=T), x, H, torch.float32, k)
    assert bool((ids[:, :2].sort(1).values == torch.tensor([70, 150])).all())
    assert torch.equal(ids[:, 2:], torch.tensor([66, 199, 0, 1], dtype=torch.int32).expand(T, 4))
    assert bool(torch.isfinite(w).all())
