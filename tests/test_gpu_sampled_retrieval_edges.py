"""retrieval.SampledRetriever: what a call holds in memory."""
import pytest
import torch

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
