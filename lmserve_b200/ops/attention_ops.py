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
from .cache_ops import _OnDevice, _packer, _stream_ptr
from .rotary_embedding_ops import _DTYPE_CODE

Cache = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]

_entries: Optional[Tuple[int, int]] = None


def _entry_points() -> Tuple[int, int]:
    """Addresses of ``lms_attention_workspace_bytes`` and ``lms_paged_attention`` (looked up once)."""
    global _entries
    if _entries is None:
        L = _lib.lib()
        _entries = tuple(ctypes.cast(f, ctypes.c_void_p).value
                         for f in (L.lms_attention_workspace_bytes, L.lms_paged_attention))
    return _entries


def _index(name: str, t: torch.Tensor, dev: torch.device) -> int:
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32 (got {t.dtype})")
    if t.device != dev or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector on the cache's device")
    return t.data_ptr()


def _pages(what: str, n_name: str, indptr, indices, last, dev) -> Tuple[int, int, int, int, int]:
    """(indptr, indices, last pointers, entries of `indices`, number of lists)."""
    p = _index(f"{what}indptr", indptr, dev)
    i = _index(f"{what}indices", indices, dev)
    e = _index(f"{what}last_page_len", last, dev)
    n = indptr.shape[0] - 1
    if n < 0 or last.shape[0] != n:
        raise ValueError(f"{what}indptr must have one entry more than {what}last_page_len has {n_name}")
    return p, i, e, indices.shape[0], n


def _attention(query, paged_kv_cache: Cache, own, prefix, group_indptr, qo_indptr, scale, causal,
               return_lse, out):
    if type(paged_kv_cache) is torch.Tensor:
        k_cache = v_cache = paged_kv_cache
        if k_cache.dim() != 5 or k_cache.shape[1] != 2:
            raise ValueError("paged_kv_cache must be [num_pages, 2, page_size, H, D]")
        NB, _, BS, H, D = k_cache.shape
        page, plane, *inner = k_cache.stride()
    else:
        k_cache, v_cache = paged_kv_cache
        if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
            raise ValueError("k_cache and v_cache must both be [num_pages, page_size, H, D]")
        NB, BS, H, D = k_cache.shape
        page, *inner = k_cache.stride()
        plane = 0
    if not (query.is_cuda and k_cache.is_cuda and v_cache.is_cuda):
        raise RuntimeError("query and the cache must live on a CUDA device; the attention ops have no CPU path")
    dev, dtype = k_cache.device, k_cache.dtype
    if dtype not in _DTYPE_CODE:
        raise TypeError(f"attention supports fp16 and bf16, got {dtype}")
    if query.dtype is not dtype or v_cache.dtype is not dtype:
        raise TypeError("query and the cache must share one dtype")
    if query.device != dev or v_cache.device != dev:
        raise RuntimeError("query must be on the cache's device; the attention ops have no CPU path")
    if inner != [H * D, D, 1]:
        raise ValueError("the entries [page_size, H, D] of a page must be contiguous")
    shape = query.shape
    if query.dim() == 3:
        T, HQ, dq = shape
        dense = dq == D and (T == 0 or (query.stride(2) == 1 and (HQ == 1 or query.stride(1) == D)))
    elif query.dim() == 2 and D:
        T, HQ = shape[0], shape[1] // D
        dense = HQ * D == shape[1] and (T == 0 or query.stride(1) == 1)
    else:
        dense = False
    if not dense:
        raise ValueError("query must be [T, num_heads, head_dim] or [T, num_heads * head_dim] with dense heads")
    if H == 0 or HQ == 0 or HQ % H:
        raise ValueError(f"{HQ} query heads cannot share {H} key heads")
    kp, ki, ke, nk, B = _pages("kv_", "requests", *own, dev)
    if qo_indptr is not None:
        qo = _index("qo_indptr", qo_indptr, dev)
        if qo_indptr.shape[0] != B + 1:
            raise ValueError("qo_indptr must have one entry more than there are requests")
    else:
        qo = None
        if T != B:
            raise ValueError("without qo_indptr every request has one token: query needs one row a request")
    pp = pi = pe = gp = None
    np_ = G = 0
    if prefix is not None:
        pp, pi, pe, np_, G = _pages("prefix_", "groups", *prefix, dev)
        if group_indptr is not None:
            gp = _index("group_indptr", group_indptr, dev)
            if group_indptr.shape[0] != G + 1:
                raise ValueError("group_indptr must have one entry more than there are prefixes")
        elif G != 1:
            raise ValueError("group_indptr says which requests share which of several prefixes")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=dev)
    elif out.shape != shape or out.dtype is not dtype or out.device != dev:
        raise ValueError("out must match query in shape, dtype and device")
    elif T and (out.stride(-1) != 1 or (out.dim() == 3 and HQ > 1 and out.stride(1) != D)):
        raise ValueError("out must have dense heads")
    lse = torch.empty(T, HQ, dtype=torch.float32, device=dev) if return_lse else None
    if T and B:
        es = 2
        kptr = k_cache.data_ptr()
        words = [query.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None,
                 kptr, kptr + plane * es if v_cache is k_cache else v_cache.data_ptr(),
                 query.stride(0) * es, out.stride(0) * es, page * es, H * D * es,
                 kp, ki, ke, nk, qo, pp, pi, pe, np_, gp, T, B, G, NB, HQ, H, D, BS,
                 _DTYPE_CODE[dtype], 1 if causal else 0,
                 float(D ** -0.5 if scale is None else scale), None, 0]
        size_of, run = _entry_points()
        with _OnDevice(dev):
            need = _packer.call_words(size_of, None, words)
            if need < 0:
                _lib.check(need)
            if need:
                workspace = torch.empty(need, dtype=torch.uint8, device=dev)
                words[-2:] = workspace.data_ptr(), need
            rc = _packer.call_words(run, _stream_ptr(dev), words)
            if rc:
                _lib.check(rc)
    return (out, lse) if return_lse else out


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
    return _attention(query, paged_kv_cache, (kv_indptr, kv_indices, kv_last_page_len), None, None,
                      qo_indptr, scale, causal, return_lse, out)


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
    return _attention(query, paged_kv_cache, (kv_indptr, kv_indices, kv_last_page_len),
                      (prefix_indptr, prefix_indices, prefix_last_page_len), group_indptr,
                      qo_indptr, scale, causal, return_lse, out)
