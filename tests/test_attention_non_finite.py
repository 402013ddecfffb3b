"""Attention over the paged cache where something it reads is NaN or infinite: the same elements as
in the 64-bit formula, whatever borders of the work the keys fall on."""
import math

import pytest
import torch

from test_paged_attention import BF, HF, call, case, drawn, exact

gpu = pytest.mark.gpu


def same(out, lse, want):
    """NaN and infinities where the formula has them, the rest within the bound."""
    o, ob, l, lb = want
    for got, right, bound in ((out.cpu().double().view(o.shape), o, ob), (lse.cpu().double(), l, lb)):
        assert torch.equal(torch.isnan(got), torch.isnan(right))
        inf, fin = torch.isinf(right), torch.isfinite(right)
        assert torch.equal(got[inf], right[inf])
        assert ((got - right).abs()[fin] <= bound[fin]).all()


# one request, cut by every border; many key heads, cut by none; requests of one tile and of none
BATCHES = [[4097], [33, 0, 700, 16, 1, 300], [90] * 40]
GEOMETRY = [(8, 2, 128, BF), (5, 1, 64, HF), (32, 8, 128, BF), (16, 1, 64, BF), (20, 1, 128, HF), (6, 2, 96, BF)]


@gpu
@pytest.mark.parametrize("prefix", [None, [200]])
@pytest.mark.parametrize("HQ,H,D,dtype", GEOMETRY)
@pytest.mark.parametrize("lengths", BATCHES)
def test_nan_queries_of_single_tokens(lengths, HQ, H, D, dtype, prefix):
    c = case(lengths, HQ=HQ, H=H, D=D, dtype=dtype, prefix=prefix)
    for b in range(0, len(lengths), 2):
        c["q"][b, (3 * b + 1) % HQ, 5] = math.nan
    same(*call(c, return_lse=True), exact(c))


@gpu
@pytest.mark.parametrize("new", [None, 1])
@pytest.mark.parametrize("HQ,H,D,dtype", GEOMETRY)
@pytest.mark.parametrize("lengths", BATCHES)
def test_nan_keys(lengths, HQ, H, D, dtype, new):
    """A page of them in one key head, in the middle of the longest request; the others stay clean."""
    c = case(lengths, [min(n, 9) for n in lengths] if new else None, HQ=HQ, H=H, D=D, dtype=dtype)
    at = lengths.index(max(lengths))
    pages = c["own"][1][c["own"][0][at]:c["own"][0][at + 1]]
    c["cache"][pages[len(pages) // 2].item(), 0, :, H - 1] = math.nan
    same(*call(c, return_lse=True), exact(c))


def bounded(c, clean, **kw):
    """The formula on `c`, with the bounds of the same call without what is infinite or NaN in V."""
    o, _, l, _ = exact(c, **kw)
    _, ob, _, lb = exact(clean, **kw)
    return o, ob, l, lb


def with_values(c, at, what):
    """(a copy of `c` with these values at (request, key, key head, element) of V, `c`)."""
    bs = c["cache"].shape[2]
    dirty = dict(c, cache=c["cache"].clone())
    for (b, key, h, e), x in zip(at, what):
        page = c["own"][1][c["own"][0][b] + key // bs].item()
        dirty["cache"][page, 1, key % bs, h, e] = x
    return dirty, c


PROMPTS = [([300], [300]), ([700, 40, 129], [500, 40, 1]), ([600, 2], [257, 2]), ([50, 260], [90, 300])]


@gpu
@pytest.mark.parametrize("prefix", [None, [150]])
@pytest.mark.parametrize("BS", [16, 12, 128])
@pytest.mark.parametrize("HQ,H,D,dtype", [(8, 2, 128, BF), (3, 3, 64, HF), (14, 2, 128, HF), (20, 1, 64, BF)])
@pytest.mark.parametrize("lengths,new", PROMPTS)
def test_infinite_values_of_prompts(lengths, new, HQ, H, D, dtype, BS, prefix):
    """Seen by some rows and hidden from others: among the first keys, in the middle, and the last."""
    n = lengths[0]
    at = [(0, 0, 0, 3), (0, n // 2, 0, 4), (0, n - 20, 0, 5), (0, n - 1, 0, 3), (0, n - 1, H - 1, D - 1), (0, n // 2, H - 1, 7), (0, n - 9, H - 1, 7)]
    what = [math.inf, -math.inf, math.nan, -math.inf, math.inf, math.inf, math.inf]
    dirty, clean = with_values(case(lengths, new, HQ=HQ, H=H, D=D, dtype=dtype, BS=BS, prefix=prefix, spread=0.5), at, what)
    same(*call(dirty, return_lse=True), bounded(dirty, clean))


@gpu
@pytest.mark.parametrize("what", ["query", "first value", "last value"])
def test_what_is_not_finite_costs_no_walk_over_the_keys(what):
    c = case([2048], [2048], HQ=8, H=2)
    if what == "query":
        dirty = dict(c, q=c["q"].clone())
        dirty["q"][:, :, 0] = math.nan
    else:
        key = 0 if what == "first value" else 2047
        dirty, _ = with_values(c, [(0, key, 0, 0), (0, key, 1, 0)], [math.inf, math.inf])
    from lmserve_b200.ops import paged_attention

    def time(c):
        args = [t.to("cuda:0") for t in (c["q"], c["cache"], *c["own"])]
        qo, best = c["qo"].to("cuda:0"), math.inf
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            paged_attention(*args, qo_indptr=qo)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert time(dirty) < 8 * time(c)


@gpu
def test_infinite_values_of_the_newest_tokens_of_a_long_request():
    n = 50_000
    c = case([9, n, 300], [9, 40, 1], HQ=2, H=1, D=64, spread=0.5)
    at = [(1, n - 1, 0, 1), (1, n - 30, 0, 2), (1, n - 41, 0, 3), (1, 3, 0, 4)]
    dirty, clean = with_values(c, at, [math.inf, -math.inf, math.inf, math.inf])
    same(*call(dirty, return_lse=True), bounded(dirty, clean))


@gpu
@pytest.mark.parametrize("prefix", [None, [150]])
@pytest.mark.parametrize("BS", [16, 12, 8])
@pytest.mark.parametrize("HQ,H,D,dtype", GEOMETRY)
@pytest.mark.parametrize("lengths", BATCHES)
def test_infinite_values_of_single_tokens(lengths, HQ, H, D, dtype, BS, prefix):
    c = case(lengths, HQ=HQ, H=H, D=D, dtype=dtype, BS=BS, prefix=prefix, spread=0.5)
    n = lengths[0]
    at = [(0, 0, 0, 3), (0, n // 2, 0, 4), (0, n // 3, 0, 5), (0, n - 1, H - 1, D - 1), (0, n - 2, 0, 6), (0, 1, 0, 6)]
    dirty, clean = with_values(c, at, [math.inf, -math.inf, math.nan, math.inf, math.inf, -math.inf])
    same(*call(dirty, return_lse=True), bounded(dirty, clean))


@gpu
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF)])
def test_an_infinite_value_of_a_key_that_carries_all(D, dtype):
    """Weights that the element type holds exactly leave no rest: 0 * infinity must not come of it."""
    for n in (1, 5, 2000):
        c = case([n, 3], HQ=4, H=2, D=D, dtype=dtype, spread=0.0)  # equal scores: every stored weight is the same power of two
        dirty, clean = with_values(c, [(0, n - 1, 0, 1), (1, 1, 1, 2)], [math.inf, -math.inf])
        same(*call(dirty, return_lse=True), bounded(dirty, clean))


@gpu
@pytest.mark.parametrize("seed", range(24))
def test_random_calls_with_something_not_finite(seed):
    """A random call with NaN and infinities in queries, keys and values: read, masked, behind the last
    keys of requests and in pages that no request has."""
    c, kw = drawn(500 + seed)
    g = torch.Generator().manual_seed(seed)
    pick = lambda n: int(torch.randint(n, (1,), generator=g))
    c["q"] = (0.5 * torch.randn(c["q"].shape, generator=g)).to(c["q"].dtype)  # no weight underflows
    clean = dict(c)
    T, HQ, D = c["q"].shape
    NB, _, BS, H, _ = c["cache"].shape
    c["q"], c["cache"] = c["q"].clone(), c["cache"].clone()
    for _ in range(1 + T // 40):
        c["q"][pick(T), pick(HQ), pick(D)] = math.nan
    for _ in range(1 + NB * BS // 600):
        c["cache"][pick(NB), 0, pick(BS), pick(H), pick(D)] = math.nan
    for _ in range(3 + NB * BS // 100):
        c["cache"][pick(NB), 1, pick(BS), pick(H), pick(D)] = [math.inf, -math.inf, math.nan][pick(3)]
    same(*call(c, return_lse=True, **kw), bounded(c, clean, **kw))
