"""How exactly the attention kernels hold the weights of the keys: a largest one beside very many
small ones, and sums that cancel, against bounds without slack for a coarser weight."""
import math

import pytest
import torch

from oracle.attention_oracle import paged_attention as formula, weight_rounding
from test_paged_attention import BF, HF, call

gpu = pytest.mark.gpu


def sink(requests, n, score, new=None, HQ=16, H=8, D=64, dtype=HF, prefix=False):
    """Requests of one key of score 0 with V = 0 and n keys of this score with V = 1 and -1/2, on two
    pages; or their last page behind a prefix of all the others."""
    i32 = lambda a: torch.tensor(a, dtype=torch.int32)
    cache = torch.zeros(2, 2, 16, H, D)
    cache[:, 0, :, :, 0] = score
    cache[:, 1] = 1.0
    cache[:, 1, :, :, ::3] = -0.5
    cache[0, :, 0] = 0.0
    m = (n + 1) // 16
    whole = [0] + [1] * (m - 1)
    c = dict(prefix=None, groups=None, qo=None, cache=cache.to(dtype))
    c["own"] = (i32([m * i for i in range(requests + 1)]), i32(whole * requests), i32([16] * requests))
    if prefix:
        c["prefix"] = (i32([0, m - 1]), i32(whole[:-1]), i32([16]))
        c["own"] = (i32(range(requests + 1)), i32([1] * requests), i32([16] * requests))
    if new:
        c["qo"] = i32([new * i for i in range(requests + 1)])
    c["q"] = torch.zeros(requests * (new or 1), HQ, D, dtype=dtype)
    c["q"][..., 0] = 1.0
    return c


def first(c, rows):
    """The formula for the first request: all have the same."""
    own = (c["own"][0][:2], c["own"][1][:c["own"][0][1]], c["own"][2][:1])
    return dict(query=c["q"][:rows], k_cache=c["cache"][:, 0], v_cache=c["cache"][:, 1], own=own,
                qo_indptr=c["qo"][:2] if c["qo"] is not None else None, prefix=c["prefix"])


@gpu
@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("n,score", [(32767, -25.1), (32767, -17.0), (131071, -24.4), (131071, -30.0)])
@pytest.mark.parametrize("kind,requests,new,prefix", [("single", 300, None, False), ("single", 5, None, False), ("tiles", 40, 3, False), ("tiles", 128, None, True)])
def test_many_small_weights_beside_a_large_one(kind, requests, new, prefix, n, score, dtype):
    c = sink(requests, n, score * math.log(2.0), new, dtype=dtype, prefix=prefix)
    rows = new or 1
    out, lse = call(c, return_lse=True, scale=1.0)
    o, ob, l, lb = formula(**first(c, rows), scale=1.0, weights=weight_rounding(kind, dtype))
    out, lse = out.cpu().double().view(requests, *o.shape), lse.cpu().double().view(requests, *l.shape)
    assert ((out - o).abs() <= ob).all(), ((out - o).abs() / ob).max().item()
    assert ((lse - l).abs() <= lb).all()


SHARES = (3, 5, 7, 11, 13)


def cancelling(D, dtype):
    """Request i: a key of score 0 with V = -1, and SHARES[i] keys of about -log SHARES[i] with V = 1, in
    one tile, so that what is left of their sum shows how the weights were held."""
    i32 = lambda a: torch.tensor(a, dtype=torch.int32)
    B = len(SHARES)
    cache = torch.zeros(B, 2, 16, 1, D)
    cache[:, 1] = 1.0
    for b, n in enumerate(SHARES):
        cache[b, 0, 1:, 0, 0] = -math.log(n)
        cache[b, 1, 0] = -1.0
    q = torch.zeros(B, 4, D)
    q[:, :, 0] = 1.0
    return dict(q=q.to(dtype), cache=cache.to(dtype), own=(i32(range(B + 1)), i32(range(B)), i32([n + 1 for n in SHARES])),
                prefix=None, groups=None, qo=None)


def wanted(c, kind, dtype):
    return formula(c["q"], c["cache"][:, 0], c["cache"][:, 1], c["own"], scale=1.0, weights=weight_rounding(kind, dtype))


@gpu
@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("kind,D", [("single", 64), ("single", 128), ("rows", 96), ("rows", 8)])
def test_weights_of_sums_that_cancel(kind, D, dtype):
    c = cancelling(D, dtype)
    out, lse = call(c, return_lse=True, scale=1.0)
    o, ob, l, lb = wanted(c, kind, dtype)
    assert ((out.cpu().double() - o).abs() <= ob).all(), ((out.cpu().double() - o).abs() / ob).max().item()
    assert ((lse.cpu().double() - l).abs() <= lb).all()


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("kind", ["single", "rows"])
def test_weights_rounded_once_would_not_pass(kind, dtype):
    """The same sums with each weight rounded once to the element type, as for tiles of rows."""
    c = cancelling(64, dtype)
    o, ob, _, _ = wanted(c, kind, dtype)
    caught = 0
    for b, n in enumerate(SHARES):
        w = torch.exp(c["cache"][b, 0, :n + 1, 0, 0].double())
        once = (w.to(dtype).double() * c["cache"][b, 1, :n + 1, 0, 0].double()).sum() / w.sum()
        caught += int((once - o[b, 0, 0]).abs() > 2 * ob[b, 0, 0])
    assert caught >= 3  # a weight may lie near a value of the type by chance


@pytest.mark.parametrize("n,score", [(32767, -25.1), (131071, -24.4)])
def test_small_weights_held_against_one_would_not_pass(n, score):
    """fp16 weights of at most one: 2^-25.1 is stored as 0, 2^-24.4 as 2^-24."""
    c = sink(1, n, score * math.log(2.0), dtype=HF, HQ=1, H=1)
    o, ob, _, _ = formula(**first(c, 1), scale=1.0, weights=weight_rounding("single", HF))
    w = torch.exp(c["cache"][1, 0, 0, 0, 0].double())
    part = w.half().double()
    part = part + (w - part).half().double()
    assert (n * part / (1 + n * w) - o[0, 0, 1]).abs() > 2 * ob[0, 0, 1]


def test_the_bound_without_a_rounding_given_is_that_of_one():
    c = cancelling(64, BF)
    u = 2.0 ** -8
    a = formula(c["q"], c["cache"][:, 0], c["cache"][:, 1], c["own"], scale=1.0)
    b = formula(c["q"], c["cache"][:, 0], c["cache"][:, 1], c["own"], scale=1.0, weights=(u, 2.0 ** -126 * u))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
