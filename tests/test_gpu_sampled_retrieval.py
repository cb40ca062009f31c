"""retrieval.SampledRetriever: the last norm in 8 bits, 4-bit scores and the draw, run together as a user runs them, against
the formulas in 64 bits.  Scores of d products are off by at most (d + 16) 2^-24 of the sum of their magnitudes; the draw is
compared on the scores it was made from (tests/test_gpu_sample.py: check)."""
import pytest
import torch

from generative_recommenders_amd import enc_ops, hmx, mx_ops, ops
from generative_recommenders_amd.retrieval import SampledRetriever
from test_gpu_sample import check, rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def setup(n=5, items=30001, d=64, draws=4, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    table = torch.randn(items, d, generator=g, device=DEV)
    table[0] = 0
    return (table, torch.randn(n, d, generator=g, device=DEV), torch.randn(n, d, generator=g, device=DEV),
            1 + 0.1 * torch.randn(d, generator=g, device=DEV), torch.rand(n, draws, generator=g, device=DEV, dtype=torch.float64))


@pytest.mark.parametrize("d", [60, 64, 128, 200])
def test_norm_scores_and_draws(d):
    table, h, res, scale, u = setup(d=d)
    rt = SampledRetriever(table)
    sc = rt.scores(h, scale, res)
    codes, xs, s = mx_ops.add_rmsnorm_mx8(h, res, scale)
    x64 = mx_ops.dequantize_mx8(codes, xs, d, torch.float32).double()
    w64 = mx_ops.dequantize_mx4(rt.codes, rt.scales, d, torch.float32).double()
    err = (sc.double() - x64 @ w64.t()).abs()
    assert bool((err <= (d + 16) * U * (x64.abs() @ w64.abs().t())).all())
    # the 8-bit values stand next to the norm that training uses: half a step of e4m3, or of the block's smallest step
    y, s2 = enc_ops.add_rmsnorm(h, res, scale)
    unit = torch.exp2(xs.double() - 127).repeat_interleave(32, 1)[:, :d]
    assert torch.equal(s, s2)
    assert bool(((x64 - y.double()).abs() <= torch.maximum(2.0 ** -4 * y.abs().double(), 2.0 ** -10 * unit) + 64 * U * y.abs()).all())
    for setting in (dict(), dict(top_k=50), dict(top_p=0.9, temperature=0.7), dict(top_k=200, top_p=0.8, min_p=0.01, temperature=1.5)):
        ids, probs = rt.sample(h, u, **setting, norm_scale=scale, residual=res)
        names = dict(temperature="t", top_k="k", top_p="p", min_p="mp")
        want = check(sc, u, **{names[k]: v for k, v in setting.items()})
        assert torch.equal(ids, want[0]) and torch.equal(probs, want[1])


def test_greedy_draw_is_the_best_item_of_the_values_stored():
    table, h, _, _, u = setup(n=40, d=64)
    rt = SampledRetriever(table)
    ids, probs = rt.sample(h, u, temperature=0.0)
    stored = mx_ops.dequantize_mx4(rt.codes, rt.scales, 64, torch.float32)
    best = ops.score_topk_exact(h, stored, 2)
    clear = best[1][:, 0] - best[1][:, 1] > 1e-4 * best[1][:, 0].abs()      # beyond what two orders of 64 products differ by
    assert int(clear.sum()) >= 30
    assert torch.equal(ids[clear], best[0][clear, :1].expand(-1, 4)) and bool((probs == 1).all())


def test_chunks_offsets_settings_per_state_and_refresh():
    table, h, res, scale, u = setup(n=11, items=5003, seed=3)
    k = torch.arange(1, 12, dtype=torch.int32, device=DEV) * 7
    t = torch.linspace(0.0, 1.5, 11, device=DEV)
    whole = SampledRetriever(table).sample(h, u, temperature=t, top_k=k, top_p=0.95)
    cut = SampledRetriever(table, id_offset=1000, score_bytes=5003 * 4 * 3).sample(h, u, temperature=t, top_k=k, top_p=0.95)
    assert torch.equal(whole[0] + 1000, cut[0]) and torch.equal(whole[1], cut[1])
    rt = SampledRetriever(torch.zeros_like(table))
    assert bool((rt.sample(h, u, top_k=1)[0] == 0).all())            # all scores equal: the lowest index
    rt.refresh(table)
    got = rt.sample(h, u, temperature=t, top_k=k, top_p=0.95)
    assert torch.equal(got[0], whole[0])
    one = rt.sample(h, u[:, 0], temperature=t, top_k=k, top_p=0.95)
    assert one[0].shape == (11,) and torch.equal(one[0], whole[0][:, 0])
    assert rt.sample(h[:0], u[:0])[0].shape == (0, 4)


def test_exclude():
    table, h, _, _, u = setup(n=6, items=700, draws=50, seed=5)
    rt = SampledRetriever(table, id_offset=10)
    free = rt.sample(h, u, temperature=3.0)[0]
    ex = free[:, ::3].clone()
    ex[:, 0] = -1                                                    # padding and foreign ids are no items
    ex[:, 1] = 5
    ex[:, 2] = 10 ** 6
    got, probs = rt.sample(h, u, temperature=3.0, exclude=ex)
    assert not bool((got.unsqueeze(2) == ex.unsqueeze(1)).any()) and bool((got >= 10).all()) and bool((probs > 0).all())
    sc = rt.scores(h)
    for i in range(6):
        for v in ex[i].tolist():
            if 10 <= v < 710:
                sc[i, v - 10] = float("-inf")
    want = check(sc, u, t=3.0)
    assert torch.equal(got, want[0] + 10)
    every = torch.arange(10, 710, device=DEV).expand(6, -1)
    ids, probs = rt.sample(h, u, exclude=every)
    assert bool((ids == -1).all()) and bool((probs == 0).all())


def test_graph_of_the_whole_path():
    table, h, res, scale, u = setup(n=3, items=200003, seed=7)
    rt = SampledRetriever(table)
    hs = h.clone()
    settings = dict(temperature=0.8, top_k=100, top_p=0.9, norm_scale=scale, residual=res)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rt.sample(hs, u, **settings)
    for k in range(3):
        hs.copy_(h * (1 - 0.5 * k))
        graph.replay()
        torch.cuda.synchronize()
        want = rt.sample(hs, u, **settings)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refresh_reaches_a_captured_graph():
    table, h, res, scale, u = setup(n=3, items=70001, seed=8)
    rt = SampledRetriever(table)
    settings = dict(temperature=0.8, top_p=0.9, norm_scale=scale)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rt.sample(h, u, **settings)
    for k in range(3):
        new = table.roll(1000 * (k + 1), 0) * (1 + k)
        rt.refresh(new)
        graph.replay()
        want = SampledRetriever(new).sample(h, u, **settings)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    rt.refresh(table[:500])                      # another shape: memory of its own
    assert rt.sample(h, u)[0].max() < 500


def test_refusals():
    table, h, res, scale, u = setup()
    rt = SampledRetriever(table)
    for call in (lambda: rt.sample(h[:, :10], u), lambda: rt.sample(h, u[:3]), lambda: rt.sample(h, u, residual=res),
                 lambda: rt.sample(h.cpu(), u), lambda: SampledRetriever(table.half()), lambda: rt.sample(h, u.unsqueeze(2)),
                 lambda: rt.sample(h, u, norm_scale=scale[:5])):
        with pytest.raises(hmx.HmxError):
            call()
