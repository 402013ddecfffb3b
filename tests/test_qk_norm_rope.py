"""Head norm + rotary embedding + cache write: the kernel against the formula in 64 bits (GPU), its
refusals (CPU and GPU)."""
import ctypes

import pytest
import torch

from lmserve_b200 import _lib
from oracle import attention_oracle, rope_oracle

DEV = "cuda:0"
gpu = pytest.mark.gpu


def case(dtype=torch.bfloat16, T=37, NH=8, NKV=2, D=128, BS=16, max_pos=300, seed=3, pos_dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(T, (NH + 2 * NKV) * D, generator=g) * 1.5).to(dtype)
    q, k, v = qkv[:, :NH * D], qkv[:, NH * D:(NH + NKV) * D], qkv[:, (NH + NKV) * D:]
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype) for _ in range(2))
    pos = torch.randint(0, max_pos, (T,), generator=g).to(pos_dtype)
    pos[-1] = max_pos - 1
    cs = rope_oracle.build_cos_sin_cache(max_pos, D, dtype)
    NB = -(-T // BS) + 2
    cache = torch.randn(NB, 2, BS, NKV, D, generator=g).to(dtype)
    slots = torch.randperm(NB * BS, generator=g)[:T]
    return dict(q=q, k=k, v=v, qw=qw, kw=kw, pos=pos, cs=cs, D=D, cache=cache, slots=slots)


def on_gpu(c):
    # the three projections stay strided views of one tensor
    qkv = torch.cat((c["q"], c["k"], c["v"]), 1).to(DEV)
    a, b = c["q"].shape[1], c["q"].shape[1] + c["k"].shape[1]
    d = {n: (t.to(DEV) if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    return dict(d, q=qkv[:, :a], k=qkv[:, a:b], v=qkv[:, b:])


def call(d, eps=1e-6, return_key=True):
    from lmserve_b200.ops import qk_norm_rotary_pos_emb_and_cache
    return qk_norm_rotary_pos_emb_and_cache(d["q"], d["k"], d["v"], d["qw"], d["kw"], d["pos"], d["cs"], d["D"],
                                            d["cache"], d["slots"], eps=eps, return_key=return_key)


def close(got, exact, bound):
    off = (got.cpu().double() - exact).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), f"off by {(off / bound).max().item():.3f} of the bound"


def check(c, eps=1e-6):
    want = {n: attention_oracle.qk_norm_rotary(c[n], c[n + "w"], c["pos"], c["cs"], c["D"], eps) for n in "qk"}
    d = on_gpu(c)
    before = d["cache"].clone()
    q, k = call(d, eps)
    close(q, *want["q"])
    close(k, *want["k"])
    # the cache: rotated K bit for bit as returned, V as given, every other row as it was
    T, D = c["q"].shape[0], c["D"]
    BS = c["cache"].shape[2]
    keep = d["slots"] >= 0
    at = d["slots"][keep].long()
    before[at // BS, 0, at % BS] = k.view(T, -1, D)[keep]
    before[at // BS, 1, at % BS] = d["v"].reshape(T, -1, D)[keep]
    assert torch.equal(d["cache"].view(torch.int16), before.view(torch.int16))
    return q, k


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [16, 48, 64, 80, 128, 256, 512])
@pytest.mark.parametrize("T,NH,NKV", [(1, 4, 4), (37, 8, 2), (130, 7, 1)])
def test_against_the_formula(dtype, D, T, NH, NKV):
    check(case(dtype, T, NH, NKV, D))


@gpu
@pytest.mark.parametrize("T,NH,NKV,D,BS", [(1, 32, 8, 128, 16), (256, 28, 4, 128, 16), (2049, 32, 8, 128, 16),
                                           (1023, 16, 4, 64, 12), (5, 1, 1, 128, 7), (700, 40, 40, 96, 1)])
def test_sizes_on_both_sides_of_the_launch_rule(T, NH, NKV, D, BS):
    check(case(torch.bfloat16, T, NH, NKV, D, BS, seed=T))


@gpu
def test_padding_int64_positions_and_eps():
    c = case(torch.float16, T=50, pos_dtype=torch.int64)
    c["slots"][[0, 7, 49]] = -1
    check(c, eps=0.25)


@gpu
def test_heads_of_zeros_and_of_large_values():
    c = case(torch.bfloat16, T=9, seed=5)
    q = c["q"].clone()
    q[0], q[1] = 0.0, q[1] * 1e15  # squares up to 1e31 stay inside fp32
    q[2] = q[2] * 1e-12            # eps decides
    c["q"] = q
    q, _ = check(c)
    assert not q[0].any()


@gpu
def test_without_a_cache_and_without_the_key():
    from lmserve_b200.ops import qk_norm_rotary_pos_emb
    c = case(torch.bfloat16, T=21)
    d = on_gpu(c)
    q, k = call(d)
    q2, k2 = qk_norm_rotary_pos_emb(d["q"], d["k"], d["qw"], d["kw"], d["pos"], d["cs"], d["D"])
    d["cache"].zero_()
    q3 = call(d, return_key=False)
    assert isinstance(q3, torch.Tensor)
    for a, b in ((q2, q), (k2, k), (q3, q)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@gpu
def test_no_token_at_all():
    d = on_gpu(case(T=4))
    for n in ("q", "k", "v", "pos", "slots"):
        d[n] = d[n][:0]
    before = d["cache"].clone()
    q, k = call(d)
    assert q.shape == (0, 8 * 128) and k.shape == (0, 2 * 128)
    assert torch.equal(before.view(torch.int16), d["cache"].view(torch.int16))


@gpu
def test_on_another_stream_and_captured():
    c = case(torch.bfloat16, T=64)
    d = on_gpu(c)
    want_q, want_k = call(d)
    want = d["cache"].clone()
    d["cache"].zero_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q, k = call(d)
    s.synchronize()
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, k = call(d)
    d["cache"].copy_(c["cache"])
    d["pos"].copy_(c["pos"].flip(0))
    graph.replay()
    torch.cuda.synchronize()
    bound = attention_oracle.qk_norm_rotary(c["q"], c["qw"], c["pos"].flip(0), c["cs"], c["D"], 1e-6)
    close(q, *bound)
    assert torch.equal(want[:, 1].view(torch.int16), d["cache"][:, 1].view(torch.int16))


@gpu
def test_positions_and_slots_outside_are_left_out_and_reported():
    c = case(torch.bfloat16, T=8)
    L = _lib.lib()
    idx, val = ctypes.c_int64(), ctypes.c_int64()
    for name, value in (("pos", c["cs"].shape[0]), ("pos", -1), ("slots", c["cache"].shape[0] * 16)):
        d = on_gpu(c)
        before = d["cache"].clone()
        d[name] = d[name].clone()
        d[name][5] = value
        L.lms_set_debug_checks(1)
        try:
            call(d)
            assert L.lms_check_device_errors(None, ctypes.byref(idx), ctypes.byref(val)) == _lib.LMS_ERR_INDEX
            assert (idx.value, val.value) == (5, value)
        finally:
            L.lms_set_debug_checks(0)
        slot = int(c["slots"][5])
        row = d["cache"][slot // 16, 0, slot % 16]
        assert torch.equal(row, before[slot // 16, 0, slot % 16])  # K of that token was not written


@gpu
def test_refusals_gpu():
    from lmserve_b200.ops import qk_norm_rotary_pos_emb
    d = on_gpu(case(torch.bfloat16, T=4))
    f = lambda **kw: qk_norm_rotary_pos_emb(*({**d, **kw}[n] for n in ("q", "k", "qw", "kw", "pos", "cs", "D")))
    with pytest.raises(ValueError, match="query_weight"):
        f(qw=d["qw"][:64])
    with pytest.raises(ValueError, match="key_weight"):
        f(kw=d["kw"].float())
    with pytest.raises(RuntimeError, match="no CPU path"):
        f(qw=d["qw"].cpu())
    with pytest.raises(TypeError):
        f(pos=d["pos"][:3])
    with pytest.raises(_lib.LmsError) as e:  # 8 is not a multiple of 16
        x = torch.zeros(2, 16, dtype=torch.bfloat16, device=DEV)
        qk_norm_rotary_pos_emb(x, x, x[0, :8].contiguous(), x[0, :8].contiguous(), d["pos"][:2],
                               torch.zeros(4, 16, dtype=torch.bfloat16, device=DEV), 8)
    assert e.value.status == _lib.LMS_ERR_UNSUPPORTED


A = 0x10000  # aligned, never dereferenced


def test_argument_errors_of_the_c_entry():
    entry = _lib.lib().lms_qk_norm_rope_and_cache
    assert entry(None, None) == _lib.LMS_ERR_NULL

    def f(**kw):
        d = dict(q=A, k=A, v=A, qt=2048, kt=512, vt=512, qw=A, kw=A, eps=1e-6, pos=A, p64=0, cs=A, row=512, qo=A,
                 qot=2048, ko=0, kot=0, kc=A, vc=A, bst=8192, sst=512, slots=A, T=4, nh=8, nkv=2, hd=128, dt=1,
                 bs=16, ns=64, mp=32)
        d.update(kw)
        words = (ctypes.c_int64 * len(d))(*[int(v or 0) if n != "eps" else 0 for n, v in d.items()])
        ctypes.cast(ctypes.byref(words, 64), ctypes.POINTER(ctypes.c_double))[0] = d["eps"]
        return entry(words, None)

    assert f(T=0) == _lib.LMS_OK
    for kw in (dict(T=-1), dict(nh=0), dict(dt=2), dict(eps=-1.0), dict(eps=float("nan")), dict(bs=0), dict(mp=-1)):
        assert f(**kw) == _lib.LMS_ERR_RANGE, kw
    for kw in (dict(hd=24), dict(hd=528)):
        assert f(**kw) == _lib.LMS_ERR_UNSUPPORTED, kw
    for kw in (dict(q=None), dict(qw=None), dict(cs=None), dict(vc=None), dict(slots=None), dict(v=None)):
        assert f(**kw) == _lib.LMS_ERR_NULL, kw
    for kw in (dict(q=A + 8), dict(kw=A + 2), dict(qt=2050), dict(pos=A + 2), dict(slots=A + 4)):
        assert f(**kw) == _lib.LMS_ERR_ALIGN, kw


def test_cpu_tensors_are_refused():
    c = case(torch.bfloat16, T=4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        call(c)


@gpu
@pytest.mark.parametrize("pos_dtype,slot_dtype", [(torch.int32, torch.int64), (torch.int64, torch.int32)])
def test_positions_and_slots_of_any_shape(pos_dtype, slot_dtype):
    """One entry a token, as the other rotary calls take them: [batch, tokens], columns of a table."""
    from lmserve_b200.ops import rotary_pos_emb_and_cache
    d = on_gpu(case(T=24, pos_dtype=pos_dtype))
    want = call(d)
    cache = d["cache"].clone()
    table = torch.stack((d["slots"], d["slots"]), 1).to(slot_dtype)
    for pos, slots in ((d["pos"].view(4, 6), d["slots"].view(24, 1)), (d["pos"].view(24, 1).expand(24, 2)[:, 1], table[:, 1])):
        d["cache"].zero_()
        rotary_pos_emb_and_cache(d["q"], d["k"], d["v"], pos, d["cs"], d["D"], d["cache"], slots)
        got = call(dict(d, pos=pos, slots=slots))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        written = d["slots"]
        for plane in (0, 1):
            assert torch.equal(d["cache"][written // 16, plane, written % 16], cache[written // 16, plane, written % 16])
    with pytest.raises(TypeError, match="one entry per token"):
        call(dict(d, pos=d["pos"].view(4, 6)[:3]))
    with pytest.raises(ValueError, match="one entry per token"):
        call(dict(d, slots=d["slots"].view(4, 6)[:3]))
