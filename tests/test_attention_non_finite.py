"""Attention over the paged cache where something it reads is NaN or infinite: the same elements as
in the 64-bit formula, whatever borders of the work the keys fall on."""
import math

import pytest
import torch

from test_paged_attention import BF, HF, call, case, exact

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
