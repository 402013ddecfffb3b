"""Attention of a batch over its pages of one layer's cache.

``paged_attention`` is the call LMServe's attention layer makes after the cache write
(``models/layers/attention.py:87-106``, flashinfer's paged prefill and decode wrappers), on the
index arrays that :class:`lmserve_b200.step_inputs.StepInputBuilder` leaves on the device:
``params.prefill`` and ``params.decode`` hold its arguments.  There is nothing to plan: the
kernels read the lengths from those arrays, so a call captured into a CUDA graph follows their
contents from replay to replay.  ``shared_prefix_attention`` is the same attention for requests
that share long prefixes, which it reads once a group instead of once a request.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from .. import _lib
from .cache_ops import _current_device, _packer, _raw_stream_of
from .rotary_embedding_ops import _DTYPE_CODE


Cache = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]

_entries: Optional[Tuple[int, int]] = None
_I32 = torch.int32


def _entry_points() -> Tuple[int, int]:
    """Addresses of ``lms_attention_workspace_bytes`` and ``lms_paged_attention`` (looked up once)."""
    global _entries
    if _entries is None:
        L = _lib.lib()
        _entries = tuple(ctypes.cast(f, ctypes.c_void_p).value
                         for f in (L.lms_attention_workspace_bytes, L.lms_paged_attention))
    return _entries


def _refuse(query, paged_kv_cache, lists, qo_indptr, group_indptr, out):
    """Names what is wrong with the arguments of an attention call."""
    if type(paged_kv_cache) is torch.Tensor:
        k_cache = v_cache = paged_kv_cache
        if k_cache.dim() != 5 or k_cache.shape[1] != 2:
            raise ValueError("paged_kv_cache must be [num_pages, 2, page_size, H, D]")
    else:
        k_cache, v_cache = paged_kv_cache
        if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
            raise ValueError("k_cache and v_cache must both be [num_pages, page_size, H, D]")
    BS, H, D = k_cache.shape[-3:]
    if not (query.is_cuda and k_cache.is_cuda and v_cache.is_cuda):
        raise RuntimeError("query and the cache must live on a CUDA device; the attention ops have no CPU path")
    dev, dtype = k_cache.device, k_cache.dtype
    if dtype not in _DTYPE_CODE:
        raise TypeError(f"attention supports fp16 and bf16, got {dtype}")
    if query.dtype != dtype or v_cache.dtype != dtype:
        raise TypeError("query and the cache must share one dtype")
    if query.device != dev or v_cache.device != dev:
        raise ValueError(f"query and both caches must be on one device ({dev}), got {query.device} and {v_cache.device}")
    if k_cache.stride()[-3:] != (H * D, D, 1):
        raise ValueError("the entries [page_size, H, D] of a page must be contiguous")
    T, HQ = query.shape[0] if query.dim() else 0, 0
    if query.dim() == 3 and query.shape[2] == D and (T == 0 or query.stride()[1:] == (D, 1) or query.shape[1] == 1 and query.stride(2) == 1):
        HQ = query.shape[1]
    elif query.dim() == 2 and D and query.shape[1] % D == 0 and (T == 0 or query.stride(1) == 1):
        HQ = query.shape[1] // D
    else:
        raise ValueError("query must be [T, num_heads, head_dim] or [T, num_heads * head_dim] with dense heads")
    if H == 0 or HQ == 0 or HQ % H:
        raise ValueError(f"{HQ} query heads cannot share {H} key heads")
    counts = []
    for what, who, (indptr, indices, last) in lists:
        for name, t in ((what + "indptr", indptr), (what + "indices", indices), (what + "last_page_len", last)):
            _check_index(name, t, dev)
        if indptr.shape[0] < 1 or last.shape[0] != indptr.shape[0] - 1:
            raise ValueError(f"{what}indptr must have one entry more than {what}last_page_len, one a {who}")
        counts.append(indptr.shape[0] - 1)
    if qo_indptr is not None:
        _check_index("qo_indptr", qo_indptr, dev)
        if qo_indptr.shape[0] != counts[0] + 1:
            raise ValueError("qo_indptr must have one entry more than there are requests")
    elif T != counts[0]:
        raise ValueError("without qo_indptr every request has one token: query needs one row a request")
    if len(counts) == 2:
        if group_indptr is not None:
            _check_index("group_indptr", group_indptr, dev)
            if group_indptr.shape[0] != counts[1] + 1:
                raise ValueError("group_indptr must have one entry more than there are prefixes")
        elif counts[1] != 1:
            raise ValueError("group_indptr says which requests share which of several prefixes")
    if out is not None:
        raise ValueError("out must match query in shape, dtype and device, with dense heads")
    raise ValueError("unsupported arguments of an attention call")


def _check_index(name: str, t: torch.Tensor, dev: torch.device) -> None:
    if t.dtype != _I32:
        raise TypeError(f"{name} must be int32 (got {t.dtype})")
    if t.device != dev or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector on the cache's device")


def _attention(query, paged_kv_cache: Cache, lists, group_indptr, qo_indptr, scale, causal, return_lse, out):
    # A layer of a decode step makes this call once, and the host's part of it is most of what a
    # small one costs: every attribute is read once, all checks are one expression, and only a call
    # that fails it is looked at again, to say what is wrong.
    _, _, (kv_indptr, kv_indices, kv_last) = lists[0]
    if type(paged_kv_cache) is torch.Tensor:
        k_cache = v_cache = paged_kv_cache
        cshape, cstride = k_cache.shape, k_cache.stride()
        ok = len(cshape) == 5 and cshape[1] == 2
    else:
        k_cache, v_cache = paged_kv_cache
        cshape, cstride = k_cache.shape, k_cache.stride()
        ok = (len(cshape) == 4 and cshape == v_cache.shape and cstride == v_cache.stride()
              and v_cache.dtype is k_cache.dtype and v_cache.get_device() == k_cache.get_device())
    dtype, idx = k_cache.dtype, k_cache.get_device()
    qshape, qstride = query.shape, query.stride()
    code = _DTYPE_CODE.get(dtype)
    if ok and idx >= 0 and code is not None and query.dtype is dtype and query.get_device() == idx:
        H, D = cshape[-2], cshape[-1]
        HD = H * D
        nk = kv_indices.shape[0] if kv_indices.dim() == 1 else -1
        B = kv_indptr.shape[0] - 1 if kv_indptr.dim() == 1 else -1
        T = qshape[0] if qshape else 0
        if len(qshape) == 3:
            HQ = qshape[1]
            ok = qshape[2] == D and (T == 0 or (qstride[2] == 1 and (HQ == 1 or qstride[1] == D)))
        elif len(qshape) == 2 and D:
            HQ = qshape[1] // D
            ok = HQ * D == qshape[1] and (T == 0 or qstride[1] == 1)
        else:
            HQ, ok = 0, False
        ok = (ok and HQ > 0 and H > 0 and HQ % H == 0 and cstride[-3:] == (HD, D, 1) and B >= 0 and nk >= 0
              and kv_indptr.dtype is _I32 and kv_indices.dtype is _I32 and kv_last.dtype is _I32
              and kv_indptr.get_device() == idx and kv_indices.get_device() == idx and kv_last.get_device() == idx
              and kv_indptr.is_contiguous() and kv_indices.is_contiguous() and kv_last.is_contiguous()
              and kv_last.shape == (B,))
    else:
        ok = False
    qo = pp = pi = pe = gp = None
    n_prefix = G = 0
    if ok:
        if qo_indptr is None:
            ok = T == B
        else:
            ok = (qo_indptr.shape == (B + 1,) and qo_indptr.dtype is _I32 and qo_indptr.get_device() == idx
                  and qo_indptr.is_contiguous())
            qo = qo_indptr.data_ptr()
    if ok and len(lists) == 2:
        _, _, (indptr, indices, last) = lists[1]
        n_prefix = indices.shape[0] if indices.dim() == 1 else -1
        G = indptr.shape[0] - 1 if indptr.dim() == 1 else -1
        ok = (G >= 0 and n_prefix >= 0 and last.shape == (G,)
              and indptr.dtype is _I32 and indices.dtype is _I32 and last.dtype is _I32
              and indptr.get_device() == idx and indices.get_device() == idx and last.get_device() == idx
              and indptr.is_contiguous() and indices.is_contiguous() and last.is_contiguous())
        pp, pi, pe = indptr.data_ptr(), indices.data_ptr(), last.data_ptr()
        if group_indptr is None:
            ok = ok and G == 1
        else:
            ok = (ok and group_indptr.shape == (G + 1,) and group_indptr.dtype is _I32
                  and group_indptr.get_device() == idx and group_indptr.is_contiguous())
            gp = group_indptr.data_ptr()
    if not ok:
        _refuse(query, paged_kv_cache, lists, qo_indptr, group_indptr, None)
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
        o_tok = HQ * D
    else:
        ostride = out.stride()
        if (out.shape != qshape or out.dtype is not dtype or out.get_device() != idx
                or T and (ostride[-1] != 1 or (len(qshape) == 3 and HQ > 1 and ostride[1] != D))):
            _refuse(query, paged_kv_cache, lists, qo_indptr, group_indptr, out)
        o_tok = ostride[0]
    lse = torch.empty((T, HQ), dtype=torch.float32, device=query.device) if return_lse else None
    if T and B:
        kptr = k_cache.data_ptr()
        words = [query.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None, kptr,
                 kptr + cstride[1] * 2 if v_cache is k_cache else v_cache.data_ptr(),
                 qstride[0] * 2 if T > 1 else 0, o_tok * 2 if T > 1 else 0, cstride[0] * 2, HD * 2,
                 kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_last.data_ptr(), nk, qo, pp, pi, pe, n_prefix, gp,
                 T, B, G, cshape[0], HQ, H, D, cshape[-3], code, 1 if causal else 0,
                 D ** -0.5 if scale is None else float(scale), None, 0]
        size_of, run = _entries or _entry_points()
        if idx != _current_device():
            with torch.cuda.device(idx):
                _enqueue(size_of, run, words, kv_indptr, idx)
        else:
            _enqueue(size_of, run, words, kv_indptr, idx)
    return (out, lse) if return_lse else out


def _enqueue(size_of, run, words, like, idx):
    need = _packer.call_words(size_of, None, words)
    if need > 0:
        # taken per call from the caching allocator: ordered by the stream it is used on, and a
        # captured call keeps its own
        workspace = like.new_empty(need >> 2)  # int32; `need` is a multiple of 256
        words[-2] = workspace.data_ptr()
        words[-1] = need
    elif need:
        _lib.check(need)
    rc = _packer.call_words(run, _raw_stream_of(idx), words)
    if rc:
        _lib.check(rc)


def paged_attention(query: torch.Tensor, paged_kv_cache: Cache, kv_indptr: torch.Tensor,
                    kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor,
                    qo_indptr: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    causal: bool = True, return_lse: bool = False,
                    out: Optional[torch.Tensor] = None):
    """Attention of every request's new tokens over its keys in the cache, those of the new
    tokens included (they were written before, by any of the cache-write operators).

    ``query``: ``[T, num_heads, head_dim]`` or ``[T, num_heads * head_dim]``, fp16 or bf16, the
    token stride is free; ``paged_kv_cache``: one layer's ``[num_pages, 2, page_size, H, D]``, or a
    ``(k_cache, v_cache)`` pair of ``[num_pages, page_size, H, D]``; ``num_heads`` is a multiple of
    ``H`` and head ``h`` reads key head ``h // (num_heads // H)``.  ``kv_indptr`` / ``kv_indices`` /
    ``kv_last_page_len`` (int32): the page table in CSR form.  ``qo_indptr`` (int32): the tokens
    of request ``b`` are rows ``qo_indptr[b]:qo_indptr[b + 1]``; without it every request has one.

    The ``n`` new tokens of a request are its last ``n`` keys: with ``causal`` token ``i`` of them
    reads the keys ``j <= len - n + i``, otherwise all ``len``.  ``scale`` multiplies ``q . k``
    (default ``head_dim ** -0.5``).  Returns the output in the shape of ``query``, and with
    ``return_lse`` also the natural logarithm of every row's sum of ``exp(scale q . k)``, fp32
    ``[T, num_heads]``.  A row that reads no key is 0, its logarithm ``-inf``.  Rows outside
    ``qo_indptr[0]:qo_indptr[-1]`` (a padded batch) are not written: pass ``out`` (same shape and
    dtype, sharing no memory with the inputs) to say what they hold.

    Head dims up to 256 that are multiples of 8.
    """
    return _attention(query, paged_kv_cache, (("kv_", "request", (kv_indptr, kv_indices, kv_last_page_len)),),
                      None, qo_indptr, scale, causal, return_lse, out)


def shared_prefix_attention(query: torch.Tensor, paged_kv_cache: Cache,
                            prefix_indptr: torch.Tensor, prefix_indices: torch.Tensor,
                            prefix_last_page_len: torch.Tensor, kv_indptr: torch.Tensor,
                            kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor,
                            group_indptr: Optional[torch.Tensor] = None,
                            qo_indptr: Optional[torch.Tensor] = None,
                            scale: Optional[float] = None, causal: bool = True,
                            return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """:func:`paged_attention` for requests that share prefixes, read once for all of them.

    The requests ``group_indptr[g]:group_indptr[g + 1]`` (int32; without it there is one group of
    all requests) read every key of the pages ``prefix_indices[prefix_indptr[g]:prefix_indptr[g +
    1]]`` - ``prefix_last_page_len[g]`` of the last one - and then their own, which
    ``kv_indptr`` / ``kv_indices`` / ``kv_last_page_len`` list *without* the prefix.  The result is
    that of :func:`paged_attention` with the prefix in front of every request's own keys; causality
    concerns the own keys only.  A prefix may be empty, a group too, and a request outside every
    group has no prefix.  The other arguments are those of :func:`paged_attention`.
    """
    return _attention(query, paged_kv_cache,
                      (("kv_", "request", (kv_indptr, kv_indices, kv_last_page_len)),
                       ("prefix_", "group", (prefix_indptr, prefix_indices, prefix_last_page_len))),
                      group_indptr, qo_indptr, scale, causal, return_lse, out)
