"""Attention over the paged cache, with and without shared prefixes: the kernels against the formula
in 64 bits (GPU), the refusals (CPU and GPU)."""
import ctypes
import math

import pytest
import torch

from lmserve_b200 import _lib
from oracle import attention_oracle

DEV = "cuda:0"
gpu = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def table(lengths, pages, BS):
    """(indptr, indices, last) of lists of these lengths, on pages taken from the iterator."""
    indptr, indices, last = [0], [], []
    for n in lengths:
        m = -(-n // BS)
        indices += [next(pages) for _ in range(m)]
        indptr.append(len(indices))
        last.append(n - (m - 1) * BS if m else 0)
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (indptr, indices, last))


def case(lengths, new=None, HQ=8, H=2, D=128, BS=16, dtype=BF, prefix=None, groups=None, seed=1, spread=2.0):
    """Requests of these own lengths and new tokens (None: one each), behind these prefixes."""
    g = torch.Generator().manual_seed(seed)
    need = sum(-(-n // BS) for n in list(lengths) + list(prefix or []))
    NB = need + 3
    pages = iter(torch.randperm(NB, generator=g).tolist())
    c = dict(own=table(lengths, pages, BS), prefix=table(prefix, pages, BS) if prefix is not None else None,
             groups=torch.tensor(groups, dtype=torch.int32) if groups is not None else None, qo=None)
    T = len(lengths)
    if new is not None:
        T = sum(new)
        c["qo"] = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    c["cache"] = torch.randn(NB, 2, BS, H, D, generator=g).to(dtype)
    c["q"] = (spread * torch.randn(T, HQ, D, generator=g)).to(dtype)
    return c


def call(c, dev=DEV, **kw):
    from lmserve_b200.ops import paged_attention, shared_prefix_attention
    d = lambda t: t.to(dev) if t is not None else None
    cache = tuple(d(t) for t in c["cache"]) if isinstance(c["cache"], tuple) else d(c["cache"])
    q = d(kw.pop("query", c["q"]))
    own = [d(t) for t in c["own"]]
    if c["prefix"] is None:
        return paged_attention(q, cache, *own, qo_indptr=d(c["qo"]), **kw)
    return shared_prefix_attention(q, cache, *(d(t) for t in c["prefix"]), *own, group_indptr=d(c["groups"]),
                                   qo_indptr=d(c["qo"]), **kw)


def exact(c, **kw):
    k, v = c["cache"] if isinstance(c["cache"], tuple) else (c["cache"][:, 0], c["cache"][:, 1])
    return attention_oracle.paged_attention(c["q"], k, v, c["own"], c["qo"], c["prefix"],
                                            c["groups"].tolist() if c["groups"] is not None else None, **kw)


def compare(out, lse, want):
    o, ob, l, lb = want
    rows = ~torch.isnan(l[:, 0])
    out, lse = out.cpu().double().view(o.shape)[rows], lse.cpu().double()[rows]
    o, ob, l, lb = o[rows], ob[rows], l[rows], lb[rows]
    assert torch.isfinite(out).all()
    worst = ((out - o).abs() / ob.clamp(min=1e-30))[ob > 0].max().item() if (ob > 0).any() else 0.0
    assert ((out - o).abs() <= ob).all(), f"out off by {worst:.3f} of the bound"
    empty = torch.isinf(l)
    assert torch.equal(lse == -math.inf, empty)
    assert ((lse - l).abs()[~empty] <= lb[~empty]).all(), \
        f"lse off by {((lse - l).abs()[~empty] / lb[~empty]).max().item():.3f} of the bound"


def check(c, **kw):
    out, lse = call(c, return_lse=True, **kw)
    compare(out, lse, exact(c, **kw))
    return out


HEADS = [(1, 1), (8, 2), (7, 1), (32, 8), (6, 6), (24, 3), (16, 1), (20, 1)]


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("HQ,H", HEADS)
def test_decode(HQ, H, D, dtype):
    check(case([1, 0, 15, 16, 17, 130, 33, 500], HQ=HQ, H=H, D=D, dtype=dtype))


@gpu
@pytest.mark.parametrize("BS", [1, 3, 7, 8, 12, 16, 24, 32, 64, 128, 256])
@pytest.mark.parametrize("new", [None, [1, 5, 70, 2, 0]])
def test_page_sizes(BS, new):
    check(case([1, 300, 257, 64, 129], new, BS=BS))


@gpu
@pytest.mark.parametrize("n", [1, 2, 15, 16, 31, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 4099])
def test_decode_lengths(n):
    check(case([n], HQ=32, H=8))
    check(case([n, 0, 3 * n + 1], HQ=28, H=4, D=64, dtype=HF))


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,D", [(HF, 64), (BF, 128)])
@pytest.mark.parametrize("HQ,H", [(8, 2), (7, 1), (3, 3), (32, 1)])
def test_new_tokens(HQ, H, dtype, D, causal):
    # single tokens, a request without tokens, whole prompts, chunks behind a past
    check(case([9, 40, 300, 129, 128, 1], [1, 0, 300, 60, 128, 1], HQ=HQ, H=H, D=D, dtype=dtype), causal=causal)


@gpu
@pytest.mark.parametrize("n,past", [(1, 0), (1, 128), (2, 127), (63, 1), (64, 0), (65, 64), (127, 129), (129, 0), (257, 300)])
def test_prompt_lengths(n, past):
    check(case([n + past, 5], [n, 5], HQ=4, H=2))


@gpu
def test_more_new_tokens_than_keys_leave_rows_empty():
    c = case([10, 0, 200], [30, 4, 300], HQ=4, H=2)
    out = check(c)
    assert not out[:20].any() and not out[30:34].any() and not out[34:134].any()


@gpu
@pytest.mark.parametrize("dtype,D", [(HF, 64), (BF, 128)])
@pytest.mark.parametrize("HQ,H", [(8, 2), (7, 1), (4, 4), (16, 1), (20, 1)])
@pytest.mark.parametrize("length", [0, 1, 100, 128, 515])
def test_shared_prefix_decode(length, HQ, H, dtype, D):
    check(case([1, 17, 0, 200, 33], HQ=HQ, H=H, D=D, dtype=dtype, prefix=[length]))


@gpu
@pytest.mark.parametrize("new", [None, [1, 5, 70, 2, 0, 3, 9]])
@pytest.mark.parametrize("BS", [16, 12, 64])
def test_shared_prefix_groups(new, BS):
    # an empty prefix, an empty group, a request in front of and one behind all groups
    check(case([40, 30, 120, 7, 64, 3, 90], new, BS=BS, prefix=[70, 0, 300, 33], groups=[1, 3, 4, 4, 6]))


@gpu
def test_many_rows_behind_one_prefix():
    check(case([i % 40 for i in range(150)], HQ=32, H=8, prefix=[700]))
    check(case([3 + i for i in range(12)], [1 + i % 5 for i in range(12)], HQ=28, H=4, D=64, dtype=HF, prefix=[1500]))


@gpu
def test_prefix_in_front_is_the_same_as_one_table():
    c = case([50, 9, 130], prefix=[64])
    own, shared = c["own"], c["prefix"]
    lists = [shared[1].tolist() + own[1][own[0][i]:own[0][i + 1]].tolist() for i in range(3)]
    whole = dict(c, prefix=None, own=(torch.tensor([0, *torch.tensor([len(x) for x in lists]).cumsum(0)], dtype=torch.int32),
                                      torch.tensor(sum(lists, []), dtype=torch.int32), own[2]))
    compare(*call(c, return_lse=True), exact(whole))
    compare(*call(whole, return_lse=True), exact(c))


@gpu
def test_requests_that_name_the_same_pages():
    c = case([100, 100, 100])
    c["own"][1][7:] = c["own"][1][:7].repeat(2)
    check(c)


@gpu
@pytest.mark.parametrize("spread", [0.0, 40.0])
def test_flat_and_peaked_scores(spread):
    check(case([700, 90], HQ=8, H=2, spread=spread))
    check(case([700, 90], [150, 90], HQ=8, H=2, spread=spread))


@gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-4])
@pytest.mark.parametrize("new", [None, [3, 60, 1]])
def test_scales_of_any_sign(scale, new):
    check(case([100, 60, 3], new, prefix=[50]), scale=scale)


@gpu
def test_rising_scores_move_the_running_maximum():
    # every key scores higher than the ones before it, across all tile borders
    c = case([600, 400], [70, 1], HQ=2, H=1, D=64, dtype=HF)
    c["q"][:] = 0.5
    for b in range(2):
        pages = c["own"][1][c["own"][0][b]:c["own"][0][b + 1]].long()
        ramp = torch.linspace(-4, 4, len(pages) * 16).view(-1, 16, 1, 1).to(HF)
        c["cache"][pages, 0] = ramp.expand(-1, -1, 1, 64)
    check(c, scale=1.0)


@gpu
def test_values_beyond_the_last_key_do_not_leak():
    # the rest of the last page and every page outside the tables hold NaN and infinities
    c = case([37, 5, 129], [37, 1, 3], BS=16)
    clean = c["cache"].clone()
    dirty = torch.full_like(clean, math.nan)
    dirty[:, :, ::2] = math.inf
    for b, n in enumerate([37, 5, 129]):
        pages = c["own"][1][c["own"][0][b]:c["own"][0][b + 1]].tolist()
        for j in range(n):
            dirty[pages[j // 16], :, j % 16] = clean[pages[j // 16], :, j % 16]
    c["cache"] = dirty
    out, lse = call(c, return_lse=True)
    one = dict(c, qo=None, q=c["q"][[36, 37, 40]])
    out1, lse1 = call(one, return_lse=True)
    c["cache"] = clean
    one["cache"] = clean
    compare(out, lse, exact(c))
    compare(out1, lse1, exact(one))


@gpu
@pytest.mark.parametrize("new", [None, [40, 1, 9]])
def test_infinite_keys_of_later_tokens_stay_masked(new):
    c = case([40, 1, 300], new)
    c["cache"][c["own"][1][2].item(), 1, 7] = math.inf  # V of the last key of request 0: seen by its last token
    out = call(c)
    rows = [0] if new is None else list(range(40))
    last = rows[-1]
    assert not torch.isfinite(out[last]).any()
    others = [r for r in range(out.shape[0]) if r != last]
    assert torch.isfinite(out[others]).all()


@gpu
def test_strided_query_flat_shape_scale_and_out():
    c = case([100, 3, 64], HQ=8, H=2)
    packed = torch.randn(3, 12 * 128).to(BF)
    packed[:, 128:9 * 128] = c["q"].view(3, -1)
    flat = packed.to(DEV)[:, 128:9 * 128]
    want = exact(c, scale=0.3)
    compare(*call(c, query=flat, return_lse=True, scale=0.3), want)
    out = torch.full((5, 3, 8 * 128), 7.0, dtype=BF, device=DEV)[::2][:, :, :].select(0, 1)
    got = call(c, query=flat, scale=0.3, out=out)
    assert got is out
    o, ob, _, _ = want
    assert ((out.cpu().double().view(o.shape) - o).abs() <= ob).all()


@gpu
def test_separate_key_and_value_caches():
    c = case([100, 3, 64], [4, 1, 64])
    want = exact(c)
    k, v = c["cache"][:, 0].contiguous(), c["cache"][:, 1].contiguous()
    compare(*call(dict(c, cache=(k, v)), return_lse=True), want)


@gpu
def test_pages_of_a_layered_cache_are_strided():
    c = case([100, 3, 64], [4, 1, 64])
    want = exact(c)
    big = torch.zeros(c["cache"].shape[0], 3, *c["cache"].shape[1:], dtype=BF, device=DEV)
    big[:, 1] = c["cache"].to(DEV)
    compare(*call(dict(c, cache=big[:, 1]), return_lse=True), want)


@gpu
@pytest.mark.parametrize("prefix", [None, [100]])
def test_rows_behind_the_last_request_are_left_alone(prefix):
    c = case([50, 60], [20, 30], prefix=prefix)
    c["q"] = torch.cat((c["q"], c["q"][:9]))
    out = torch.full(c["q"].shape, 3.0, dtype=BF, device=DEV)
    got, lse = call(c, out=out, return_lse=True)
    assert (got[50:] == 3.0).all()
    compare(got, lse, exact(c))


@gpu
@pytest.mark.parametrize("new", [None, [2, 9, 1]])
def test_pages_outside_the_cache_read_as_zeros_and_are_reported(new):
    c = case([40, 35, 20], new, prefix=[30])
    NB = c["cache"].shape[0]
    zeros = torch.zeros(1, *c["cache"].shape[1:], dtype=BF)
    for which, bad in ((0, NB), (1, -1), (1, 2 ** 31 - 1)):
        d = dict(c, own=tuple(t.clone() for t in c["own"]), prefix=tuple(t.clone() for t in c["prefix"]))
        at = 4
        target = d["own"] if which else d["prefix"]
        at = 4 if which else 1
        target[1][at] = bad
        L = _lib.lib()
        L.lms_set_debug_checks(1)
        idx, val = ctypes.c_int64(), ctypes.c_int64()
        try:
            out, lse = call(d, return_lse=True)
            assert L.lms_check_device_errors(None, ctypes.byref(idx), ctypes.byref(val)) == _lib.LMS_ERR_INDEX
            assert (idx.value, val.value) == (at, bad)
        finally:
            L.lms_set_debug_checks(0)
        target[1][at] = NB
        compare(out, lse, exact(dict(d, cache=torch.cat((c["cache"], zeros)))))


@gpu
def test_table_entries_past_the_end_read_as_zeros():
    c = case([40, 35], [3, 2])
    short = tuple(t.clone() for t in c["own"])
    zeros = torch.zeros(1, *c["cache"].shape[1:], dtype=BF)
    cut = (short[0], short[1][:-1].clone(), short[2])
    out, lse = call(dict(c, own=cut), return_lse=True)
    whole = (short[0], torch.cat((cut[1], torch.tensor([c["cache"].shape[0]], dtype=torch.int32))), short[2])
    compare(out, lse, exact(dict(c, own=whole, cache=torch.cat((c["cache"], zeros)))))


@gpu
@pytest.mark.parametrize("kind", ["decode", "varlen", "prefix"])
def test_captured_calls_follow_the_arrays(kind):
    """One graph, replayed for steps of other lengths and a smaller total; two graphs in turn."""
    from lmserve_b200.ops import paged_attention, shared_prefix_attention
    first, second = [130, 400, 17, 90], [1, 0, 333, 50]
    new = ([5, 100, 1, 20], [1, 0, 77, 3]) if kind == "varlen" else (None, None)
    pre = ([200], [37]) if kind == "prefix" else (None, None)
    a = case(first, new[0], prefix=pre[0], seed=1)
    b = case(second, new[1], prefix=pre[1], seed=2)
    NB = max(a["cache"].shape[0], b["cache"].shape[0])
    T = a["q"].shape[0]

    def padded(t, n):
        return torch.cat((t, t.new_zeros(n - t.shape[0], *t.shape[1:])))

    def load(bufs, c):
        bufs["cache"].copy_(padded(c["cache"], NB))
        bufs["q"].copy_(padded(c["q"], T))
        for i in range(3):
            bufs["own"][i].copy_(padded(c["own"][i], bufs["own"][i].shape[0]))
            if c["prefix"] is not None:
                bufs["prefix"][i].copy_(padded(c["prefix"][i], bufs["prefix"][i].shape[0]))
        if c["qo"] is not None:
            bufs["qo"].copy_(c["qo"])

    def buffers():
        return dict(cache=torch.zeros(NB, *a["cache"].shape[1:], dtype=BF, device=DEV),
                    q=torch.zeros(a["q"].shape, dtype=BF, device=DEV),
                    own=[torch.zeros(60 if i == 1 else t.shape[0], dtype=torch.int32, device=DEV) for i, t in enumerate(a["own"])],
                    prefix=[torch.zeros(20 if i == 1 else t.shape[0], dtype=torch.int32, device=DEV) for i, t in enumerate(a["prefix"] or [])],
                    qo=torch.zeros(5, dtype=torch.int32, device=DEV) if new[0] else None)

    def run(w):
        if kind == "prefix":
            return shared_prefix_attention(w["q"], w["cache"], *w["prefix"], *w["own"], return_lse=True)
        return paged_attention(w["q"], w["cache"], *w["own"], qo_indptr=w["qo"], return_lse=True)

    sets, graphs, outs = [buffers(), buffers()], [], []
    for w in sets:
        load(w, a)
        run(w)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(w))
    for steps in ((a, b), (b, a)):
        for w, c in zip(sets, steps):
            load(w, c)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (out, lse), c in zip(outs, steps):
            n = c["q"].shape[0]
            compare(out[:n], lse[:n], exact(c))


@gpu
def test_two_streams_at_once():
    cs = [case([900, 20, 333], seed=i, prefix=[400] if i % 2 else None) for i in range(4)]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = []
    for c, s in zip(cs, streams):
        with torch.cuda.stream(s):
            got.append(call(c, return_lse=True))
    torch.cuda.synchronize()
    for c, g in zip(cs, got):
        compare(*g, exact(c))


@gpu
@pytest.mark.parametrize("new", [None, [3, 64, 200]])
def test_the_same_call_gives_the_same_bits(new):
    c = case([2000, 64, 777], new, HQ=32, H=8, prefix=[900])
    a = call(c)
    for _ in range(3):
        assert torch.equal(a.view(torch.int16), call(c).view(torch.int16))


@gpu
def test_offsets_past_32_bits():
    # the last pages of an 8.6 GB layer lie past 2^32 bytes and past 2^31 elements
    BS, H, D = 16, 8, 128
    NB = 2 ** 33 // (2 * BS * H * D * 2) + 64
    c = case([100, 33, 64], [1, 33, 2], HQ=32, H=H)
    big = torch.empty(NB, 2, BS, H, D, dtype=BF, device=DEV)
    n = c["cache"].shape[0]
    big[NB - n:] = c["cache"].to(DEV)
    far = dict(c, own=(c["own"][0], c["own"][1] + (NB - n), c["own"][2]), cache=big)
    compare(*call(far, return_lse=True), exact(c))
    one = dict(far, qo=None, q=c["q"][:3])
    compare(*call(one, return_lse=True), exact(dict(c, qo=None, q=c["q"][:3])))
    del big, far, one
    torch.cuda.empty_cache()


@gpu
def test_nothing_to_do():
    c = case([5, 6])
    d = lambda t: t.to(DEV)
    from lmserve_b200.ops import paged_attention
    none = (torch.zeros(1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.zeros(0, dtype=torch.int32))
    out, lse = paged_attention(d(c["q"])[:0], d(c["cache"]), *(d(t) for t in none), return_lse=True)
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)
    # requests, but not one key in the batch
    check(case([0, 0, 0]))
    check(case([0, 0], [2, 3], prefix=[0]))


@gpu
def test_refusals_gpu():
    from lmserve_b200.ops import paged_attention, shared_prefix_attention
    c = case([5, 6, 20])
    q, cache = c["q"].to(DEV), c["cache"].to(DEV)
    own = [t.to(DEV) for t in c["own"]]
    f = lambda q=q, cache=cache, own=own, **kw: paged_attention(q, cache, *own, **kw)
    with pytest.raises(RuntimeError, match="no CPU path"):
        f(q=c["q"])
    with pytest.raises(ValueError, match="cache's device"):
        f(own=list(c["own"]))
    with pytest.raises(TypeError, match="torch.Tensor"):
        f(own=[own[0], None, own[2]])
    with pytest.raises(TypeError, match="torch.Tensor"):
        f(q=None)
    with pytest.raises(TypeError, match="int32"):
        f(own=[own[0].long(), *own[1:]])
    with pytest.raises(TypeError, match="one dtype"):
        f(q=q.half())
    with pytest.raises(TypeError, match="fp16 and bf16"):
        f(q=q.float(), cache=cache.float())
    with pytest.raises(ValueError, match="cannot share"):
        f(q=q[:, :7])
    with pytest.raises(ValueError, match="one row a request"):
        f(q=q[:2])
    with pytest.raises(ValueError, match="dense heads"):
        f(q=q.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="one entry more"):
        f(qo_indptr=own[0][:3])
    with pytest.raises(ValueError, match="contiguous"):
        f(cache=cache.transpose(3, 4).contiguous().transpose(3, 4))
    with pytest.raises(ValueError, match="out must"):
        f(out=torch.empty_like(q, dtype=HF))
    two = [torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), own[1], torch.tensor([3, 4], dtype=torch.int32, device=DEV)]
    with pytest.raises(ValueError, match="group_indptr"):
        shared_prefix_attention(q, cache, *two, *own)
    x = torch.zeros(3, 2, 12, dtype=BF, device=DEV)
    with pytest.raises(_lib.LmsError) as e:
        f(q=x, cache=torch.zeros(4, 2, 16, 2, 12, dtype=BF, device=DEV))
    assert e.value.status == _lib.LMS_ERR_UNSUPPORTED


A = 0x10000  # aligned, never dereferenced


def c_args(**kw):
    d = dict(q=A, out=A, lse=0, kc=A, vc=A, qt=2048, ot=2048, bst=16384, sst=512, kp=A, ki=A, ke=A, nk=9, qo=0,
             pp=0, pi=0, pe=0, np=0, gp=0, T=4, B=4, G=0, NB=20, HQ=8, H=2, D=128, BS=16, dt=1, causal=1)
    d.update({k: v for k, v in kw.items() if k in d})
    words = (ctypes.c_int64 * (len(d) + 3))(*[v or 0 for v in d.values()], 0, 0, 0)
    ctypes.cast(ctypes.byref(words, 8 * len(d)), ctypes.POINTER(ctypes.c_double))[0] = kw.get("scale", 0.1)
    return words


def test_argument_errors_of_the_c_entry():
    L = _lib.lib()
    f = lambda **kw: L.lms_paged_attention(c_args(**kw), None)
    assert L.lms_paged_attention(None, None) == _lib.LMS_ERR_NULL
    assert f(T=0, B=0) == _lib.LMS_OK and L.lms_attention_workspace_bytes(c_args(T=0, B=0)) == 0
    for kw in (dict(T=-1), dict(T=3), dict(HQ=7), dict(H=0), dict(BS=0), dict(dt=2), dict(NB=-1), dict(nk=-1),
               dict(scale=math.inf), dict(scale=math.nan), dict(G=-1), dict(nk=2 ** 27), dict(G=1, np=2 ** 27),
               dict(T=2 ** 30, B=2 ** 30)):
        assert f(**kw) == _lib.LMS_ERR_RANGE, kw
        assert L.lms_attention_workspace_bytes(c_args(**kw)) == _lib.LMS_ERR_RANGE, kw
    for kw in (dict(D=100), dict(D=264)):
        assert f(**kw) == _lib.LMS_ERR_UNSUPPORTED, kw
    for kw in (dict(q=0), dict(out=0), dict(kc=0), dict(kp=0), dict(ke=0), dict(ki=0), dict(G=1), dict(G=2, pp=A, pe=A)):
        assert f(**kw) == _lib.LMS_ERR_NULL, kw
    for kw in (dict(q=A + 8), dict(vc=A + 4), dict(qt=2050), dict(sst=520), dict(kp=A + 2), dict(qo=A + 1)):
        assert f(**kw) == _lib.LMS_ERR_ALIGN, kw


def test_cpu_tensors_are_refused():
    for c in (case([5, 6]), case([5, 6], prefix=[3])):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call(c, dev="cpu")


def test_the_oracle_on_a_case_done_by_hand():
    """Two keys, head dim 8: weights 1/4 and 3/4."""
    q = torch.zeros(1, 1, 8)
    q[0, 0, 0] = 1
    cache = torch.zeros(1, 2, 2, 1, 8)
    cache[0, 0, 1, 0, 0] = math.log(3.0)
    cache[0, 1, 0], cache[0, 1, 1] = 4.0, 8.0
    own = (torch.tensor([0, 1]), torch.tensor([0]), torch.tensor([2]))
    out, _, lse, _ = attention_oracle.paged_attention(q, cache[:, 0], cache[:, 1], own, scale=1.0)
    assert torch.allclose(out, torch.full_like(out, 7.0)) and abs(lse.item() - math.log(4.0)) < 1e-6


def drawn(seed):
    """A random call: geometry, lengths (zeros and single keys often), groups, stray requests."""
    import random
    r = random.Random(seed)
    D = r.choice([64, 64, 128, 128, 128, 8, 40, 96, 256])
    H = r.choice([1, 1, 2, 3, 4, 5, 8, 9])
    G = r.choice([1, 2, 3, 4, 7, 8, 9, 16, 17, 33])
    B = r.choice([1, 2, 3, 9, 33, 70])
    most = r.choice([1, 20, 140, 600]) if B < 40 else r.choice([1, 20, 60])
    length = lambda: r.choice([0, 1, r.randint(0, most), r.randint(0, most), r.randint(0, most)])
    lengths = [length() for _ in range(B)]
    new = None
    if r.random() < 0.6:
        new = [r.choice([0, 1, r.randint(0, 6), r.randint(0, max(1, min(most, 2 * n)))]) for n in lengths]
        if sum(new) > 700:
            new = [min(n, 3) for n in new]
        if sum(new) == 0:
            new[0] = 1
    prefix = groups = None
    if r.random() < 0.5:
        n = r.choice([1, 1, 2, 4])
        prefix = [length() for _ in range(n)]
        if n > 1 or r.random() < 0.5:
            groups = sorted(r.randint(0, B) for _ in range(n + 1))
    c = case(lengths, new, HQ=H * G, H=H, D=D, BS=r.choice([1, 5, 8, 12, 16, 16, 16, 24, 32, 64, 128, 256]),
             dtype=r.choice([HF, BF]), prefix=prefix, groups=groups, seed=seed, spread=r.choice([0.5, 2.0, 6.0]))
    return c, dict(causal=r.random() < 0.8)


@gpu
@pytest.mark.parametrize("seed", range(40))
def test_random_calls(seed):
    c, kw = drawn(seed)
    check(c, **kw)


@gpu
def test_thousands_of_requests():
    """More requests than a warp's, a block's or an SM count's worth, single tokens and a few each."""
    lengths = [i % 7 for i in range(5000)]
    c = case(lengths, HQ=4, H=2, D=64, dtype=HF)
    out, lse = call(c, return_lse=True)
    some = torch.arange(0, 5000, 41)
    picked = dict(c, q=c["q"][some], own=(c["own"][0], c["own"][1], c["own"][2]))
    lists = [c["own"][1][c["own"][0][b]:c["own"][0][b + 1]].tolist() for b in some]
    picked["own"] = (torch.tensor([0, *torch.tensor([len(x) for x in lists]).cumsum(0)], dtype=torch.int32),
                     torch.tensor(sum(lists, []), dtype=torch.int32), c["own"][2][some])
    compare(out[some.to(DEV)], lse[some.to(DEV)], exact(picked))
    new = [1 + i % 3 for i in range(3000)]
    c = case([n + i % 5 for i, n in enumerate(new)], new, HQ=4, H=2, D=64, dtype=HF)
    out, lse = call(c, return_lse=True)
    first = c["qo"].tolist()
    some = list(range(0, 3000, 61))
    rows = [t for b in some for t in range(first[b], first[b + 1])]
    lists = [c["own"][1][c["own"][0][b]:c["own"][0][b + 1]].tolist() for b in some]
    picked = dict(c, q=c["q"][rows], qo=torch.tensor([0, *torch.tensor([new[b] for b in some]).cumsum(0)], dtype=torch.int32),
                  own=(torch.tensor([0, *torch.tensor([len(x) for x in lists]).cumsum(0)], dtype=torch.int32),
                       torch.tensor(sum(lists, []), dtype=torch.int32), c["own"][2][some]))
    compare(out[rows], lse[rows], exact(picked))


@gpu
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF)])
@pytest.mark.parametrize("prefix", [None, [1000]])
def test_many_bytes_of_keys(prefix, D, dtype):
    """Above the size where the decode kernel fetches rows in place of boxes: 0.6 GB of table, on few pages."""
    once, times = [4000, 17, 0, 4099, 1, 900], 30 * 256 // D
    c = case(once, HQ=16, H=8, D=D, dtype=dtype, prefix=prefix)
    indptr, indices, last = c["own"]
    ends = torch.cat([indptr[1:] + i * int(indptr[-1]) for i in range(times)])
    c["own"] = (torch.cat([indptr[:1], ends]).int(), indices.repeat(times), last.repeat(times))
    assert len(c["own"][1]) * 16 * 8 * D * 4 > 2**29
    g = torch.Generator().manual_seed(2)
    c["q"] = (2 * torch.randn(len(once) * times, 16, D, generator=g)).to(dtype)
    out, lse = call(c, return_lse=True)
    some = list(range(len(once) * 7, len(once) * 9)) + list(range(len(once) * (times - 1), len(once) * times))
    start = c["own"][0].tolist()
    lists = [c["own"][1][start[b]:start[b + 1]].tolist() for b in some]
    picked = dict(c, q=c["q"][some], own=(torch.tensor([0, *torch.tensor([len(x) for x in lists]).cumsum(0)], dtype=torch.int32),
                                          torch.tensor(sum(lists, []), dtype=torch.int32), c["own"][2][some]))
    compare(out[some], lse[some], exact(picked))


@gpu
def test_the_first_call_may_be_captured():
    """In a fresh process: per-device set-up, then a capture with no call before it."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch, sys
sys.path.insert(0, 'tests')
from lmserve_b200 import _lib
from lmserve_b200.ops import paged_attention
from test_paged_attention import case, exact, compare
torch.cuda.init(); torch.zeros(1, device='cuda')
_lib.check(_lib.lib().lms_init_device())
for new in (None, [30, 1, 200]):
    c = case([100, 7, 300], new)
    d = [t.cuda() for t in (c['q'], c['cache'], *c['own'])]
    qo = c['qo'].cuda() if new else None
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = paged_attention(*d, qo_indptr=qo, return_lse=True)
    g.replay(); torch.cuda.synchronize()
    compare(*got, exact(c))
print('captured')
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr
