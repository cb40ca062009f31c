"""retrieval.SampledRetriever: what a call holds in memory, what it refuses."""
import pytest
import torch

from generative_recommenders_amd import hmx
from generative_recommenders_amd.retrieval import SampledRetriever
from test_gpu_sampled_retrieval import setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("excluded", [False, True])
def test_scores_of_one_chunk_are_held_at_a_time(excluded):
    """The outputs, the sampling's workspace (0.13 MB for each of 4 rows) and the index tensors take less than a MB."""
    table, h, res, scale, u = setup(n=12, items=500003, seed=2)
    rt = SampledRetriever(table, score_bytes=4 * 4 * 500003)
    ex = torch.arange(12, device="cuda").view(12, 1) if excluded else None
    want = rt.sample(h, u, top_p=0.9, exclude=ex, norm_scale=scale, residual=res)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = rt.sample(h, u, top_p=0.9, exclude=ex, norm_scale=scale, residual=res)
    assert torch.cuda.max_memory_allocated() - held <= rt.score_bytes + (1 << 20)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("score_bytes", [1 << 30, 4 * 5003 * 2])
def test_operands_of_another_number_of_states_are_refused(score_bytes):
    table, h, res, scale, u = setup(n=5, items=5003, seed=4)
    rt = SampledRetriever(table, score_bytes=score_bytes)
    seven = torch.ones(7, device="cuda")
    ex = torch.zeros(7, 3, dtype=torch.int64, device="cuda")
    for bad in (dict(temperature=seven), dict(top_k=seven.int()), dict(top_p=seven), dict(min_p=0 * seven), dict(temperature=seven[:4]),
                dict(temperature=seven[0]), dict(temperature=seven[:5].view(5, 1)), dict(exclude=ex), dict(exclude=ex[:4]),
                dict(exclude=ex[0]), dict(exclude=ex[:5].int()), dict(norm_scale=scale, residual=torch.cat([res, res])),
                dict(norm_scale=scale, residual=res[:4]), dict(norm_scale=scale, residual=res[:1])):
        with pytest.raises(hmx.HmxError):
            rt.sample(h, u, **bad)
    for states in (h[0], h[:, :10], h[:0, :10]):
        with pytest.raises(hmx.HmxError):
            rt.sample(states, u[:states.shape[0]])
    got = rt.sample(h, u, temperature=seven[:5], top_k=seven[:5].int(), exclude=ex[:5, :0])
    assert torch.equal(got[0], rt.sample(h, u, top_k=1)[0])


def test_a_refused_table_leaves_the_old_one():
    table, h, res, scale, u = setup(n=5, items=5003, seed=6)
    rt = SampledRetriever(table)
    want = rt.sample(h, u, top_p=0.9)
    for bad in (table[:, :60].half(), table[:, :40].cpu(), table[:, :0], table[0]):
        with pytest.raises(hmx.HmxError):
            rt.refresh(bad)
        got = rt.sample(h, u, top_p=0.9)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        with pytest.raises(hmx.HmxError):
            rt.sample(h[:, :60], u)
    rt.refresh(table[:, :60])
    assert rt.sample(h[:, :60], u)[0].shape == u.shape
