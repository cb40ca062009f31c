"""ops.sample_logits against the definition in 64 bits (sorted row, running sums, search).

ids are compared for equality.  The two sides' running sums differ by rounding: u is kept (by the test) away from every
border of the kept set's running sums by 1e-9 of the mass, top_p away from its border by 1e-9, so that no rounding of either
side (2^-51 of the largest weight per element, 2^-53 per addition) can move a draw.  probs: one fp32 rounding (2^-24) and
1e-9 for the sums."""
import pytest
import torch

from generative_recommenders_amd import hmx, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
SLACK = 1e-9


def kept_row(l, t, k, p, mp):
    """-> weights of a row (0: not kept) in 64 bits, how near top_p comes to its border, on l's device."""
    l = l.double()
    ok = l > float("-inf")
    if not bool(ok.any()):
        return torch.zeros_like(l), 1.0
    if not t > 0:
        t, k = 1.0, 1
    top = l[ok].max()
    z = torch.where(l == top, torch.zeros_like(l), (l - top) / t)
    w = torch.where(ok, torch.exp(z), torch.zeros_like(l))
    order = torch.sort(torch.where(ok, l, torch.full_like(l, -float("inf"))), descending=True, stable=True).indices
    order = order[:int(ok.sum())]
    if k > 0:
        order = order[:k]
    gap = 1.0
    if p < 1:
        upto = torch.cumsum(w[order], 0)
        share = upto / upto[-1]
        gap = float((share - p).abs().min())
        order = order[:int((share < p).sum()) + 1]
    keep = torch.zeros_like(l)
    keep[order] = 1
    return torch.where(z >= (torch.log(torch.tensor(float(mp), dtype=torch.float64)) if mp > 0 else -float("inf")), w * keep,
                       torch.zeros_like(l)), gap


def check(logits, u, t=1.0, k=0, p=1.0, mp=0.0, allow=0.01):
    """Runs the draw for (B, V) logits and (B, S) u and compares; numbers or per-row tensors.  allow: the part of the draws
    that may lie too near to a border to be compared."""
    B = logits.shape[0]

    def at(x, i):
        return x[i].item() if isinstance(x, torch.Tensor) else x
    u = u.clone()
    want_ids, want_probs, close = [], [], []
    for i in range(B):
        w, gap = kept_row(logits[i], at(t, i), int(at(k, i)), at(p, i), at(mp, i))
        upto = torch.cumsum(w, 0)
        total = upto[-1]
        if total == 0:
            want_ids.append(torch.full_like(u[i], -1, dtype=torch.int64))
            want_probs.append(torch.zeros_like(u[i], dtype=torch.float64))
            close.append(torch.zeros_like(u[i], dtype=torch.bool))
            continue
        at_ = (u[i].double() * total).contiguous()
        ids = torch.searchsorted(upto, at_, right=True).clamp_max(w.numel() - 1)
        last = int(w.nonzero().max())
        ids = ids.clamp_max(last)
        before = torch.where(ids > 0, upto[(ids - 1).clamp_min(0)], torch.zeros_like(at_))
        # an id is only compared where u is clear of the borders next to it
        near = (torch.minimum((upto[ids] - at_).abs(), torch.where(before > 0, (at_ - before).abs(), total)) < SLACK * total) | (gap < SLACK)
        want_ids.append(ids)
        want_probs.append(w[ids] / total)
        close.append(near)
    ids, probs = ops.sample_logits(logits, u, t, k, p, mp)
    want_ids, want_probs, close = torch.stack(want_ids), torch.stack(want_probs), torch.stack(close)
    assert ids.dtype == torch.int64 and probs.dtype == torch.float32 and ids.shape == u.shape
    assert float(close.float().mean()) <= allow
    wrong = (ids != want_ids) & ~close
    assert not bool(wrong.any()), (ids[wrong][:5], want_ids[wrong][:5], int(wrong.sum()))
    err = (probs.double() - want_probs).abs()
    assert not bool(((err > (2.0 ** -24 + SLACK) * want_probs) & ~close).any())
    return ids, probs


def rows(B, V, S, dtype=torch.float32, spread=3.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (spread * torch.randn(B, V, generator=g, device=DEV)).to(dtype), torch.rand(B, S, generator=g, device=DEV, dtype=torch.float64)


SETTINGS = [dict(), dict(t=0.7), dict(k=1), dict(k=50), dict(p=0.9), dict(mp=0.05), dict(t=1.3, k=40, p=0.8),
            dict(t=0.9, k=700, p=0.95, mp=0.01), dict(p=0.05), dict(p=0.999, mp=0.0005), dict(t=0.0)]


@pytest.mark.parametrize("setting", SETTINGS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 4096, 4097, 20000, 131073])
def test_settings(V, dtype, setting):
    logits, u = rows(3, V, 9, dtype, seed=V)
    check(logits, u, **setting)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread,setting", [(1e-3, dict(p=0.7)), (1e-3, dict(k=9000)), (0.0, dict(p=0.37)), (0.0, dict(k=10001)),
                                            (0.05, dict(k=15000, p=0.6)), (1.0, dict(k=12000, p=0.9)), (1e-8, dict(p=0.5)),
                                            (40.0, dict(k=8000)), (1.0, dict(t=1e-3, k=6000)), (1.0, dict(t=100.0, p=0.99)),
                                            (0.5, dict(k=29999)), (200.0, dict(k=20000, p=0.999999))])
def test_large_kept_sets_and_ties(spread, setting, dtype):
    """Kept sets that fit no list: borders inside one bin of close values, one value for the whole row, and far below the
    maximum."""
    logits, u = rows(2, 30001, 8, dtype, spread, seed=5)
    check(logits + 1.0, u, **setting)


def test_per_row_settings():
    B = 12
    logits, u = rows(B, 9001, 5, seed=3)
    t = torch.tensor([0.0, 0.5, 1.0, 2.0, -1.0, float("inf"), float("nan"), 1.0, 1.0, 1.0, 1.0, 1.0], device=DEV)
    k = torch.tensor([0, 5, 0, 100, 3, 7, 9, 1 << 30, -4, 1, 5000, 9000], dtype=torch.int32, device=DEV)
    p = torch.tensor([1, 1, .5, .9, 1, 1, 1, 2.0, 0.0, 1, .99, .999], device=DEV)
    mp = torch.tensor([0, 0, 0, 0, 0, 0, 0, -1.0, 0, 0, .001, 0], device=DEV)
    plain_t = torch.where(torch.isfinite(t) & (t > 0), t, torch.zeros_like(t))
    ids, probs = ops.sample_logits(logits, u, t, k, p, mp)
    want = check(logits, u, plain_t, k.clamp_min(0), p.clamp(max=1.0), mp.clamp_min(0))
    assert torch.equal(ids, want[0]) and torch.equal(probs, want[1])
    for i in (0, 4, 5, 6):
        assert bool((ids[i] == logits[i].argmax()).all()) and bool((probs[i] == 1).all())


@pytest.mark.parametrize("V", [100, 6000, 200003])
def test_special_values(V):
    logits, u = rows(9, V, 6, seed=7)
    logits[0] = float("-inf")
    logits[1] = float("nan")
    logits[2, :] = torch.finfo(torch.float32).min
    logits[3, ::3] = float("-inf")
    logits[3, 1::3] = float("nan")
    logits[4, [3, 50, 77]] = float("inf")
    logits[5] = float("-inf")
    logits[5, V - 1] = -5.0
    logits[6, ::2] = torch.finfo(torch.float32).min
    logits[7] = 0.0
    logits[7, ::2] = -0.0
    logits[8] *= 1e4
    for setting in (dict(), dict(k=7), dict(p=0.6), dict(mp=0.2), dict(t=0.0), dict(k=V, p=0.9)):
        # rows 2 and 7 hold equal scores only: a share of 60 of 100 of them is a border itself
        ids, probs = check(logits, u, **setting, allow=0.25)
        assert bool((ids[:2] == -1).all()) and bool((probs[:2] == 0).all()) and bool((ids[5] == V - 1).all())
        assert bool(torch.isin(ids[4], torch.tensor([3, 50, 77], device=DEV)).all())
        # equal scores, -0 among them: the lowest indices are kept
        if setting.get("k") == 7:
            assert int(ids[7].max()) <= 6 and int(ids[2].max()) <= 6


def test_u_at_its_borders():
    logits = torch.tensor([[0.0, float("-inf"), 0.0, 0.0, float("-inf")]], device=DEV)
    for dt in (torch.float32, torch.float64):
        u = torch.tensor([[0.0, 0.3, 0.34, 0.66, 0.67, 0.999, 1.0, 2.0, -1.0, float("nan"), float("inf")]], dtype=dt, device=DEV)
        ids, probs = ops.sample_logits(logits, u)
        assert ids.tolist() == [[0, 0, 2, 2, 3, 3, 3, 3, 0, 0, 3]]
        assert bool((probs - 1 / 3).abs().max() <= 2.0 ** -24)


def test_frequencies():
    """Equal parts of [0, 1) as u: every item is drawn its share of them, give or take one."""
    logits, _ = rows(1, 50, 1, seed=2)
    n = 100000
    u = (torch.arange(n, dtype=torch.float64, device=DEV) + 0.5).view(1, n) / n
    ids, probs = ops.sample_logits(logits, u, top_k=20)
    count = torch.bincount(ids[0], minlength=50).double()
    w, _ = kept_row(logits[0], 1.0, 20, 1.0, 0.0)
    assert float((count - n * w / w.sum()).abs().max()) <= 1.0
    assert torch.equal(probs[0], probs[0].clone()) and int((count > 0).sum()) <= 20


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes_strides_and_offsets(dtype):
    logits, u = rows(12, 5003, 4, dtype, seed=9)
    want = check(logits, u, k=300, p=0.9)
    wide = torch.full((12, 5100), float("inf"), device=DEV, dtype=dtype)
    wide[:, 13:5016] = logits
    for v, uu in ((wide[:, 13:5016], u), (logits.t().contiguous().t(), u), (logits.view(3, 4, 5003), u.view(3, 4, 4)),
                  (logits, u.t().contiguous().t())):
        got = ops.sample_logits(v, uu, top_k=300, top_p=0.9)
        assert torch.equal(got[0].view(12, 4), want[0]) and torch.equal(got[1].view(12, 4), want[1])
    got = ops.sample_logits(logits, u[:, 0], top_k=300, top_p=0.9)
    assert got[0].shape == (12,) and torch.equal(got[0], want[0][:, 0])
    got = ops.sample_logits(logits[0], u[0], top_k=300, top_p=0.9)
    assert torch.equal(got[0], want[0][0])
    got = ops.sample_logits(logits[:1].expand(12, 5003), u, top_k=300, top_p=0.9)
    assert torch.equal(got[0][0], want[0][0])
    assert ops.sample_logits(logits[:0], u[:0])[0].shape == (0, 4)
    assert ops.sample_logits(logits, u[:, :0])[0].shape == (12, 0)
    single = u.float()
    assert torch.equal(ops.sample_logits(logits, single)[0], ops.sample_logits(logits, single.double())[0])
    g = torch.Generator(device=DEV).manual_seed(4)
    big = torch.empty(2, (1 << 31) // (1 if dtype == torch.bfloat16 else 2), dtype=dtype, device=DEV)[:, :300000]
    big.copy_(torch.randn(2, 300000, generator=g, device=DEV))
    check(big, u[:2], p=0.9)                              # the second row starts past 2^31 bytes


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("setting", [dict(), dict(k=1000, p=0.95, mp=0.001), dict(p=0.9), dict(p=0.5, t=0.8), dict(mp=0.01),
                                     dict(k=100000), dict(k=100000, p=0.8), dict(t=0.0)])
def test_item_table_rows(setting, dtype):
    logits, u = rows(2, 2_000_003, 16, dtype, 2.0, seed=21)
    check(logits, u, **setting)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [3000, 65537, 140001])
def test_temperatures_at_the_ends(V, dtype):
    """Almost the highest score alone, almost equal weights, and a spread of scores near the type's range.  (Shares that no
    whole number of equal weights makes: 21 of 30 equal ones are 0.7 itself.)"""
    logits, u = rows(3, V, 6, dtype, seed=V + 1)
    for t in (1e-30, 1e-3, 1e30):
        for setting in (dict(), dict(k=30), dict(p=0.7303), dict(k=2501, p=0.7303), dict(mp=0.5)):
            check(logits, u, t=t, **setting)
    check(logits * 1e37, u, t=3e37, p=0.9)
    check(logits * 1e-37, u, t=1e-37, k=40, p=0.9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V", [(70, 66000), (2, 65535), (2, 65536), (5, 131071), (64, 70001)])
def test_rows_about_where_they_are_cut(B, V, dtype):
    logits, u = rows(B, V, 2, dtype, seed=B)
    for setting in (dict(), dict(k=50), dict(p=0.9), dict(k=3000, p=0.9), dict(mp=0.02)):
        ids, probs = ops.sample_logits(logits, u, setting.get("t", 1.0), setting.get("k", 0), setting.get("p", 1.0), setting.get("mp", 0.0))
        some = slice(0, B, max(1, B // 3))
        want = check(logits[some], u[some], **setting)
        assert torch.equal(ids[some], want[0]) and torch.equal(probs[some], want[1])


def test_scores_in_order():
    """Sorted rows: the kept set lies in a few tiles, and groups of neighbours are not alike."""
    for V in (5000, 100001, 300001):
        logits, u = rows(2, V, 20, seed=V)
        for desc in (False, True):
            ordered = torch.sort(logits, dim=1, descending=desc).values
            for setting in (dict(k=100), dict(k=1500, p=0.9), dict(p=0.9), dict(k=2500)):
                check(ordered, u, **setting)
                check(ordered.bfloat16(), u, **setting)


def test_many_rows_and_draws():
    logits, u = rows(600, 333, 3, seed=4)
    check(logits[:40], u[:40], k=30, p=0.9)
    ids, _ = ops.sample_logits(logits, u, top_k=30, top_p=0.9)
    assert torch.equal(ids[:40], ops.sample_logits(logits[:40], u[:40], top_k=30, top_p=0.9)[0])
    logits, u = rows(1, 70000, 5000, seed=6)
    check(logits, u, p=0.97)
    check(logits, u, k=100)


def test_refusals():
    logits, u = rows(4, 50, 2)
    calls = [lambda: ops.sample_logits(logits.half(), u), lambda: ops.sample_logits(logits.cpu(), u),
             lambda: ops.sample_logits(logits, u.cpu()), lambda: ops.sample_logits(logits, u[:3]),
             lambda: ops.sample_logits(logits, u.half()), lambda: ops.sample_logits(logits, u.view(4, 2, 1)),
             lambda: ops.sample_logits(logits[:, :0], u), lambda: ops.sample_logits(logits, u, temperature=-1.0),
             lambda: ops.sample_logits(logits, u, temperature=float("inf")), lambda: ops.sample_logits(logits, u, temperature=float("nan")),
             lambda: ops.sample_logits(logits, u, top_k=-1), lambda: ops.sample_logits(logits, u, top_p=1.5),
             lambda: ops.sample_logits(logits, u, min_p=-0.1), lambda: ops.sample_logits(logits, u, top_p=float("nan")),
             lambda: ops.sample_logits(logits, u, top_k=torch.ones(4, device=DEV)),
             lambda: ops.sample_logits(logits, u, top_p=torch.ones(3, device=DEV)),
             lambda: ops.sample_logits(logits, u, temperature=torch.ones(4))]
    for call in calls:
        with pytest.raises(hmx.HmxError):
            call()


def test_streams_and_graphs():
    logits, u = rows(5, 40001, 4, seed=31)
    big, ub = rows(2, 1_000_001, 4, torch.bfloat16, seed=32)
    settings = dict(temperature=0.9, top_k=0, top_p=0.9, min_p=0.0)
    graphs = []
    for _ in range(2):                                   # two graphs replayed in turn: neither meets the other's workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.sample_logits(logits, u, **settings) + ops.sample_logits(big, ub, **settings)
        graphs.append((graph, out))
    for k in range(4):
        logits.mul_(0.9)
        big.mul_(0.9)
        graph, out = graphs[k % 2]
        graph.replay()
        torch.cuda.synchronize()
        want = ops.sample_logits(logits, u, **settings) + ops.sample_logits(big, ub, **settings)
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = ops.sample_logits(big, ub, **settings)
    b = ops.sample_logits(big, ub, **settings)            # two calls at once
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
