"""ops.sample_logits at the ends of what it accepts, against the definition in 64 bits (tests/test_gpu_sample.py: check, with
its tolerances).  Row lengths reach each way that a row is worked on: whole in a list, by one block, cut over many blocks."""
import sys

import pytest
import torch

from generative_recommenders_amd import ops
from test_gpu_sample import DEV, check, rows

pytestmark = pytest.mark.gpu

LENGTHS = [1500, 3000, 65537, 140001]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", LENGTHS)
def test_smallest_temperatures(V, dtype):
    """Down to the least positive double: the scores equal to the maximum share the draws, whatever else is set."""
    logits, u = rows(3, V, 8, dtype, seed=V)
    logits[1, ::V // 7] = logits[1].max()                 # 8 of them (or one less)
    logits[2] = 0.0                                       # the smallest differences there are
    logits[2, ::V // 5] = 1e-45 if dtype == torch.float32 else 1e-40
    for t in (1e-50, 1e-300, sys.float_info.min, 1e-310, 5e-324):
        for setting in (dict(), dict(k=3), dict(k=30), dict(p=0.7303), dict(k=2501, p=0.7303), dict(mp=0.5)):
            ids, probs = check(logits, u, t=t, **setting)
            assert bool((ids >= 0).all()) and bool((ids < V).all())
            assert int((logits[0] == logits[0].max()).sum()) > 1 or bool((probs[0] == 1).all())
            assert bool((logits.gather(1, ids) == logits.max(1, keepdim=True).values).all())
    assert int(check(logits, u, t=5e-324)[0][1].unique().numel()) > 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", LENGTHS)
def test_scores_further_apart_than_the_largest_number(V, dtype):
    """All but one score 6.6e38 below it: at a temperature of 2.9e38 each of them weighs a tenth, and their mass counts."""
    logits, u = rows(3, V, 8, dtype, seed=V + 2)
    logits = (logits * 1e33 - 3.3e38).to(dtype)
    logits[0, V // 3] = 3.3e38
    logits[1, ::V // 7] = 3.3e38
    logits[2, V - 1] = float("inf")
    for t in (2.9e38, 1e38, 1e37):
        for setting in (dict(), dict(k=30), dict(p=0.7303), dict(k=2501, p=0.7303), dict(mp=0.05)):
            check(logits, u, t=t, **setting)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", LENGTHS)
def test_largest_temperatures(V, dtype):
    """Every finite one is a temperature: all scores weigh the same, also where a row has float32's largest as its own."""
    logits, u = rows(5, V, 8, dtype, seed=V + 3)
    logits[1] = (logits[1] * 1e38).nan_to_num(0.0, 3e38, -3e38)
    logits[2, V // 2] = float("inf")
    logits[3, ::3] = float("-inf")
    for t in (3.2e38, 1e39, 1e45, 1e59, 1e61, 1e300, sys.float_info.max):
        for setting in (dict(), dict(k=30), dict(p=0.7303), dict(k=2501, p=0.7303), dict(mp=0.01)):
            check(logits, u, t=t, **setting)
    own = torch.tensor([3.1e38, 3.4028234e38, 1.0, 1e-45, float("inf")], device=DEV)
    for setting in (dict(), dict(k=30), dict(p=0.7303)):
        ids, probs = ops.sample_logits(logits, u, own, setting.get("k", 0), setting.get("p", 1.0))
        want = check(logits, u, torch.where(torch.isfinite(own), own, torch.zeros_like(own)), **setting)
        assert torch.equal(ids, want[0]) and torch.equal(probs, want[1])
    assert int(ops.sample_logits(logits, u, own)[0][0].unique().numel()) > 4


@pytest.mark.parametrize("V", [6000, 80001])
def test_the_same_scores_elsewhere_in_the_row(V):
    """bfloat16 scores without a counter (below 2^-22, from 1024 on) are listed in the order that atomics give: rows that hold
    the same scores in the same order, between other gaps, draw the same ones with the same probabilities."""
    n, B = 3000, 8
    g = torch.Generator(device=DEV).manual_seed(V)
    scores = torch.cat([1024 + 8 * torch.randint(0, 3, (n // 2,), generator=g, device=DEV),
                        1016 - 4 * torch.randint(0, 3, (n - n // 2,), generator=g, device=DEV)])
    scores = scores[torch.randperm(n, generator=g, device=DEV)].bfloat16()
    logits = torch.full((B, V), float("-inf"), dtype=torch.bfloat16, device=DEV)
    at = torch.stack([torch.randperm(V, generator=g, device=DEV)[:n].sort().values for _ in range(B)])
    logits.scatter_(1, at, scores.expand(B, n))
    u = torch.rand(1, 500, generator=g, device=DEV, dtype=torch.float64).expand(B, 500)
    for setting in (dict(t=7.0), dict(t=7.0, p=0.9), dict(t=7.0, k=2000), dict(t=30.0, k=2000, p=0.8, mp=0.1)):
        ids, probs = ops.sample_logits(logits, u, setting["t"], setting.get("k", 0), setting.get("p", 1.0), setting.get("mp", 0.0))
        rank = torch.searchsorted(at, ids)
        assert torch.equal(at.gather(1, rank), ids)
        assert torch.equal(rank, rank[:1].expand_as(rank)) and torch.equal(probs, probs[:1].expand_as(probs))
        check(logits[:2], u[:2], **setting)


@pytest.mark.parametrize("V", [1500, 70001])
def test_top_k_past_64_bits(V):
    logits, u = rows(2, V, 50, seed=V)
    want = ops.sample_logits(logits, u)
    for k in (V, V + 1, 2 ** 63 - 1, 2 ** 63, 2 ** 64 + 5, 10 ** 30):
        got = ops.sample_logits(logits, u, top_k=k)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k


def kinds(B):
    """Settings of B rows, neighbours of different kinds: greedy, a small top_k, one above 2000, top_p, min_p, all of them, and
    none; with those, a row worked on by maxima, by bins, by narrowing and by tiles stand side by side."""
    t = torch.tensor([0.0, 1.0, 0.7, 1.0, 1.3, 1.0, 1.0, float("inf")], device=DEV).repeat(-(-B // 8))[:B]
    k = torch.tensor([0, 20, 2500, 0, 0, 300, 0, 5], dtype=torch.int32, device=DEV).repeat(-(-B // 8))[:B]
    p = torch.tensor([1.0, 1.0, 0.93, 0.87, 1.0, 0.8, 1.0, 1.0], device=DEV).repeat(-(-B // 8))[:B]
    mp = torch.tensor([0.0, 0.0, 0.001, 0.0, 0.03, 0.01, 0.0, 0.0], device=DEV).repeat(-(-B // 8))[:B]
    return t, k, p, mp


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V", [(10, 9001), (10, 70001), (10, 300001), (64, 65536), (3, 1_000_003)])
def test_rows_of_every_kind_beside_each_other(B, V, dtype):
    """Each row's draws are those of its own settings, also where one launch cuts rows of different kinds over many blocks."""
    logits, u = rows(B, V, 7, dtype, seed=V + B)
    if B >= 10:
        logits[9] = float("-inf")                         # nothing to draw
        logits[4, ::2] = float("nan")
        logits[6] = 0.25                                  # one score for the whole row
        logits[3, 1::2] = logits[3, 0]                    # a border among equal scores
    t, k, p, mp = kinds(B)
    got = ops.sample_logits(logits, u, t, k, p, mp)
    plain_t = torch.where(torch.isfinite(t), t, torch.zeros_like(t))
    some = torch.arange(min(B, 10), device=DEV)
    want = check(logits[some], u[some], plain_t[some], k[some], p[some], mp[some])
    for a, b in zip(got, want):
        assert torch.equal(a[some], b)
    for i in range(B):                                    # alone, with numbers for settings
        one = ops.sample_logits(logits[i], u[i], plain_t[i].item(), int(k[i]), p[i].item(), mp[i].item())
        assert torch.equal(one[0], got[0][i])
        # by its length and the number of rows a row is worked on in ways whose scales differ: a rounding of a weight, 2^-24 of probs
        assert bool(((one[1] - got[1][i]).abs() <= 2.0 ** -23 * got[1][i]).all())


def test_probabilities_are_the_shares():
    logits, u = rows(3, 700, 2000, seed=12)
    ids, probs = ops.sample_logits(logits, u, top_k=40)
    kept = torch.topk(logits, 40).values[:, -1:]
    w = torch.where(logits >= kept, torch.exp(logits.double() - logits.double().max(1, keepdim=True).values), torch.zeros_like(logits).double())
    want = (w / w.sum(1, keepdim=True)).gather(1, ids)
    assert bool(((probs.double() - want).abs() <= (2.0 ** -24 + 1e-9) * want).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_longest_rows(dtype):
    """2^31 - 1 scores, the most there may be: equal ones (each index its share, the lowest kept), and three among -infinity."""
    V = 2 ** 31 - 1
    logits = torch.ones(1, V, dtype=dtype, device=DEV)
    at = torch.tensor([0, 1, 12345, 2 ** 30 + 5, 2 ** 31 - 2 - 4096, V - 1], device=DEV)
    u = ((at.double() + 0.5) / V).view(1, -1)
    ids, probs = ops.sample_logits(logits, u)
    assert torch.equal(ids[0], at) and bool(((probs.double() * V - 1).abs() <= 2.0 ** -23).all())
    if dtype == torch.bfloat16:                           # (equal fp32 scores are counted in one place: seconds at this length)
        half = u / 2                                          # top_p 0.5 keeps the first 2^30 (of 2^31 - 1 equal shares)
        ids, probs = ops.sample_logits(logits, half, top_p=0.5)
        assert torch.equal(ids[0], (half[0] * 2 ** 30).floor().long()) and bool(((probs.double() * 2 ** 30 - 1).abs() <= 2.0 ** -23).all())
        ids, probs = ops.sample_logits(logits, u, top_k=5)
        assert torch.equal(ids[0], (u[0] * 5).floor().long()) and bool(((probs.double() * 5 - 1).abs() <= 2.0 ** -23).all())
    logits.fill_(float("-inf"))
    three = torch.tensor([7, V - 2 ** 20, V - 1], device=DEV)
    logits[0, three] = 2.0
    for setting in (dict(), dict(top_k=100), dict(top_p=0.9), dict(temperature=0.1, min_p=0.5)):
        ids, probs = ops.sample_logits(logits, u, **setting)
        assert torch.equal(ids[0], three[(u[0] * 3).floor().long()]) and bool(((probs.double() * 3 - 1).abs() <= 2.0 ** -23).all()), setting
