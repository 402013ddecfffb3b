"""CPU oracle (torch, 64 bits) of the head norm + rotary embedding and of attention over the paged
cache, with the error bounds the tests hold the kernels to.

Each function returns the exact values next to ``bound``: how far a result may be from them that
holds scores, statistics and accumulators in fp32, rounds the weights ``exp(s - m)`` to the element
type for the second product and rounds the output once.
"""
from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def weight_rounding(kind, dtype):
    """(relative to the weight, relative to the largest one): how far the weights that a kernel
    takes into the second product may be from ``exp(s - m)``.  ``kind``: "tiles" (several tokens a
    request, shared prefixes) rounds them once; "single" (one token a request) feeds a part, rounded
    towards zero from 2^-12 less than the weight, and the rest, at most a step and 2^-12 of the weight,
    rounded; "rows" (head dims without matrix products) keeps them in fp32.  fp16 holds them 2^9 times
    as large, so that the half step 2^-25 of its smallest numbers is 2^-34 of the largest weight."""
    u = half_step(dtype)
    if kind == "rows":
        return 0.0, 2.0 ** -126
    return (u if kind == "tiles" else u * (2 * u + 2.0 ** -12)), 2.0 ** (-34 if dtype == torch.float16 else -126)


def qk_norm_rotary(x, weight, positions, cos_sin, head_dim, eps):
    """(exact, bound) of ``x`` [T, heads * head_dim] normalised by head and rotated."""
    D, E = head_dim, head_dim // 2
    T = x.shape[0]
    n = x.double().reshape(T, -1, D)
    n = n / torch.sqrt((n * n).mean(-1, keepdim=True) + eps) * weight.double()
    row = cos_sin.double()[positions.long()][:, None]
    a, b = n[..., :E], n[..., E:]
    c0, c1, s0, s1 = (row[..., i * E:(i + 1) * E] for i in range(4))
    exact = torch.cat((a * c0 - b * s0, b * c1 + a * s1), -1)
    size = torch.cat(((a * c0).abs() + (b * s0).abs(), (b * c1).abs() + (a * s1).abs()), -1)
    # the sum of D squares, its inverse root (two steps) and five products and sums in fp32
    fp32 = (D / 2 + 16) * F32
    u = half_step(x.dtype)
    tiny = torch.finfo(x.dtype).smallest_normal * u
    bound = (exact.abs() + fp32 * size) * u + fp32 * size + tiny
    return exact.reshape(T, -1), bound.reshape(T, -1)


def _listed(indptr, indices, last, i, block_size):
    a, z = int(indptr[i]), int(indptr[i + 1])
    return [int(x) for x in indices[a:z]], max(0, (z - a - 1) * block_size + int(last[i])) if z > a else 0


def paged_attention(query, k_cache, v_cache, own, qo_indptr=None, prefix=None, group_indptr=None,
                    scale=None, causal=True, weights=None):
    """(out, out bound, lse, lse bound) in float64; rows outside qo_indptr are NaN.

    ``query`` [T, HQ, D]; the caches [NB, BS, H, D]; ``own`` and ``prefix`` are
    ``(indptr, indices, last_page_len)``; ``weights`` what :func:`weight_rounding` gives (default: one
    rounding to the element type, with its smallest numbers)."""
    T, HQ, D = query.shape
    BS, H = k_cache.shape[1:3]
    group = HQ // H
    scale = D ** -0.5 if scale is None else scale
    B = len(own[2])
    first = list(range(B + 1)) if qo_indptr is None else [int(x) for x in qo_indptr]
    u = half_step(query.dtype)
    own_step, floor = weights or (u, torch.finfo(query.dtype).smallest_normal * u)
    out = torch.full((T, HQ, D), math.nan, dtype=torch.float64)
    bound, lse, lse_bound = torch.zeros_like(out), torch.full((T, HQ), math.nan, dtype=torch.float64), torch.zeros(T, HQ, dtype=torch.float64)

    def taken(pages, n):
        at = torch.tensor(pages, dtype=torch.long)
        return k_cache[at].double().reshape(-1, H, D)[:n], v_cache[at].double().reshape(-1, H, D)[:n]

    for b in range(B):
        keys, values = taken(*_listed(*own, b, BS))
        n_own, ahead = keys.shape[0], 0
        if prefix is not None:
            g = 0 if group_indptr is None else next(
                (i for i in range(len(group_indptr) - 1) if group_indptr[i] <= b < group_indptr[i + 1]), None)
            if g is not None:
                pk, pv = taken(*_listed(*prefix, g, BS))
                keys, values, ahead = torch.cat((pk, keys)), torch.cat((pv, values)), pk.shape[0]
        n_new = first[b + 1] - first[b]
        for i in range(n_new):
            t = first[b] + i
            seen = ahead + (max(0, min(n_own, n_own - n_new + i + 1)) if causal else n_own)
            if seen == 0:
                out[t], lse[t] = 0.0, -math.inf
                continue
            k = keys[:seen].repeat_interleave(group, 1)
            v = values[:seen].repeat_interleave(group, 1)
            q = query[t].double()
            s = scale * torch.einsum("hd,lhd->hl", q, k)
            # worst error of a score: D products and sums of this size in fp32
            s_err = ((D + 8) * F32 * abs(scale) * torch.einsum("hd,lhd->hl", q.abs(), k.abs())).amax(-1)
            s_err = s_err + 8 * F32 * s.abs().amax(-1)
            w = torch.softmax(s, -1)
            out[t] = torch.einsum("hl,lhd->hd", w, v)
            size = torch.einsum("hl,lhd->hd", w, v.abs())
            lse[t] = torch.logsumexp(s, -1)
            # the exponential (its argument rounded once more), the sums over the keys, a few joins
            sums = (seen + 64) * F32
            fp32 = 2 * s_err + 2.0 ** -20 + sums
            # weights below the normal range lose bits against the largest one
            tiny = seen * floor * v.abs().amax()
            bound[t] = u * out[t].abs() + (own_step + fp32[:, None]) * (1 + u) * size + tiny
            lse_bound[t] = s_err + 2.0 ** -20 + sums + 4 * F32 * lse[t].abs()
    return out, bound, lse, lse_bound
