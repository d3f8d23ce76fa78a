"""GPU tests of sampling against the definition in 64 bits: tokens are whole numbers and have to be equal.  (A draw or a border
nearer to u or top_p of the sum than the weights' precision, 2^-44 of the largest each, could fall either way; the reference's own
sums in 64 bits are no finer.  No row here comes that near.)"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(row, u, T, k, p, m):
    row = np.where(np.isnan(row), -np.inf, row)
    if row.max() == -np.inf:
        return -1
    if not T > 0:
        return int(np.argmax(row))
    by = np.lexsort((np.arange(row.size), -row))
    with np.errstate(invalid="ignore"):
        w = np.where(row[by] == row.max(), 1.0, np.exp((row[by] - row.max()) / T))
    n = max(1, int(np.sum(w >= m))) if m > 0 else row.size
    n = n if k <= 0 else min(n, k)
    before = np.concatenate([[0.0], np.cumsum(w[:n])])
    if not p >= 1:
        n = max(1, int(np.searchsorted(before[:n], p * before[n], side="left")))
    kept = np.sort(by[:n])
    weight = np.zeros(row.size)
    weight[by] = w
    cum = np.cumsum(weight[kept])
    return int(kept[min(np.searchsorted(cum, u * cum[-1], side="right"), len(kept) - 1)])


def both(kernels, logits, u, T=1.0, k=0, p=1.0, m=0.0):
    got = kernels.sample(logits, u, temperature=T, top_k=k, top_p=p, min_p=m)
    pick = lambda t, b: float(t[b]) if isinstance(t, torch.Tensor) else float(np.float32(t))
    x, un = logits.double().cpu().numpy(), u.double().cpu().numpy()
    want = [reference(x[b], un[b], pick(T, b), int(pick(k, b)), pick(p, b), pick(m, b)) for b in range(len(x))]
    assert got.tolist() == want
    return got


def rows(B, V, dtype, seed=0, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (spread * torch.randn(B, V, device="cuda", generator=g)).to(dtype), torch.rand(B, device="cuda", generator=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (2, 7), (5, 33), (9, 1000), (40, 4097), (1, 152064), (2, 151937), (70, 32000),
                                 (3, 262144)])
def test_filters(kernels, dtype, B, V):
    logits, u = rows(B, V, dtype, seed=V)
    for k, p, m, T in ((0, 1.0, 0.0, 1.0), (50, 0.9, 0.0, 0.8), (0, 0.95, 0.0, 1.3), (1, 1.0, 0.0, 1.0), (0, 1.0, 0.05, 0.7),
                       (300, 0.5, 0.01, 2.0), (0, 0.0, 0.0, 1.0), (0, 0.999, 0.0, 5.0), (7, 1.0, 1.0, 1.0), (0, 1.0, 0.0, 0.0),
                       (V - 1, 1.0, 0.0, 1.0), (V, 0.7, 0.0, 1.0)):
        both(kernels, logits, u, T, k, p, m)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_settings_of_each_row(kernels, dtype):
    B, V = 64, 20011
    logits, u = rows(B, V, dtype, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    pick = lambda *c: torch.tensor(c, device="cuda")[torch.randint(len(c), (B,), device="cuda", generator=g)]
    both(kernels, logits, u, pick(0.0, 0.3, 1.0, 2.0), pick(0, -1, 1, 5, 1000, 30000).to(torch.int32), pick(1.0, 0.9, 0.1, 0.0),
         pick(0.0, 0.1, 0.5, 1.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_equal_logits_keep_the_lowest_indices(kernels, dtype):
    """All logits equal, or few values: borders inside runs of equal logits, in every slice of the row."""
    V, B = 50000, 16
    u = torch.arange(B, device="cuda").float() / B + 0.03
    for logits in (torch.zeros(B, V, device="cuda"),
                   torch.randint(0, 4, (B, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).float() - 1,
                   torch.where(torch.arange(V, device="cuda") % 2 == 0, 0.0, -0.0).expand(B, V)):
        for k, p in ((10, 1.0), (20001, 1.0), (0, 0.5), (30000, 0.77), (0, 0.999)):
            both(kernels, logits.to(dtype).contiguous(), u, 1.0, k, p)


def test_not_numbers_and_infinities(kernels):
    inf, nan = float("inf"), float("nan")
    V = 3000
    logits, u = rows(8, V, torch.float32, seed=5)
    logits[0] = nan
    logits[1] = -inf
    logits[2, ::2] = -inf
    logits[3, 1::2] = nan
    logits[4, 7] = inf
    logits[5, [9, 77, 2999]] = inf
    logits[6] = torch.finfo(torch.float32).min
    logits[7] = -inf
    logits[7, 2500] = -5.0
    for dtype in (torch.float32, torch.bfloat16):
        x = logits.to(dtype)
        for k, p, T in ((0, 1.0, 1.0), (2500, 1.0, 1.0), (2, 0.5, 1.0), (0, 0.9, 0.5), (0, 1.0, 0.0)):
            both(kernels, x, u, T, k, p)
    # numbers outside [0, 1): the first, the last
    both(kernels, logits[2:], torch.tensor([0.0] * 6, device="cuda"))
    got = kernels.sample(logits[2:4], torch.tensor([1.0, 5.0], device="cuda"))
    assert got.tolist() == [2999, 2998]
    assert kernels.sample(logits[2:4], torch.tensor([nan, -1.0], device="cuda")).tolist() == [1, 0]


def test_far_apart_logits_and_small_temperature(kernels):
    logits, u = rows(20, 9000, torch.float32, seed=6, spread=40.0)
    for T in (0.01, 0.5, 1.0, 100.0):
        both(kernels, logits, u, T, 0, 0.95)


def test_strided_rows_and_out(kernels):
    logits, u = rows(6, 5000, torch.bfloat16, seed=7)
    wide = torch.full((6, 5003), 50.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:5001] = logits
    out = torch.empty(6, dtype=torch.int64, device="cuda")
    got = kernels.sample(wide[:, 1:5001], u, top_k=40, out=out)
    assert got is out and torch.equal(got, kernels.sample(logits, u, top_k=40))


def test_draws_follow_the_distribution(kernels):
    """100 000 equally spaced numbers hit every kept token in its share, to one draw."""
    n, V = 100000, 64
    logits, _ = rows(1, V, torch.float32, seed=8, spread=1.0)
    u = (torch.arange(n, device="cuda").float() + 0.5) / n
    got = torch.bincount(kernels.sample(logits.expand(n, V), u, top_k=20), minlength=V)
    kept = torch.zeros(V, dtype=torch.bool, device="cuda")
    kept[logits[0].topk(20).indices] = True
    share = torch.softmax(torch.where(kept, logits[0].double(), -torch.inf), -1) * n
    assert (got[~kept] == 0).all() and ((got - share).abs() <= 2).all()


def test_captured(kernels):
    logits, u = rows(4, 152064, torch.bfloat16, seed=9)
    kernels.sample(logits, u)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        got = kernels.sample(logits, u, top_k=50, top_p=0.9)
    for seed in (10, 11):
        x, v = rows(4, 152064, torch.bfloat16, seed=seed)
        logits.copy_(x)
        u.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        assert got.tolist() == both(kernels, x, v, 1.0, 50, 0.9).tolist()


def test_streams_and_settings_that_are_no_numbers(kernels):
    """Calls that overlap on two streams draw what single calls draw; settings that are not numbers, or infinite, are answered:
    a temperature that is no positive number takes the largest logit, an infinite one draws evenly, other nans filter as 0."""
    x = [rows(9, 50000, torch.bfloat16, seed=60 + i) for i in range(2)]
    draw = lambda i, **kw: kernels.sample(*x[i], **kw)
    ways = [dict(temperature=0.8), dict(top_k=50, top_p=0.9), dict(top_p=0.9, temperature=3.0)]
    want = [[draw(i, **kw) for i in range(2)] for kw in ways]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for w, kw in enumerate(ways):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got.append((w, i, draw(i, **kw)))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[w][i]) for w, i, t in got)
    inf, nan = float("inf"), float("nan")
    greedy = draw(0, temperature=0.0)
    for kw in (dict(temperature=nan), dict(temperature=-1.0), dict(temperature=-inf), dict(top_p=nan), dict(top_p=-1.0)):
        assert torch.equal(draw(0, **kw), greedy), kw
    assert torch.equal(draw(0, min_p=nan), draw(0))
    logits, u = rows(4, 1000, torch.float32, seed=70)
    assert torch.equal(kernels.sample(logits, u, temperature=1e-45), logits.argmax(-1))  # (no two are equal)
    logits[:, ::2] = -inf
    assert torch.equal(kernels.sample(logits, u, temperature=inf), 2 * (u.double() * 500).long() + 1)
