"""Attention of a batch over its pages of one layer's cache.

``paged_attention`` is the step behind the cache write in LMServe's attention layer
(``models/layers/attention.py:87-106``), on the index arrays that :class:`lmserve_b200.step_inputs.StepInputBuilder` leaves on the device:
``params.prefill`` and ``params.decode`` hold its arguments.  There is nothing to plan: the
kernels read the lengths from those arrays, so a call captured into a CUDA graph follows their
contents from replay to replay.  ``shared_prefix_attention`` is the same attention for requests
that share long prefixes, which it reads once a group instead of once a request (heads of 64 and 128).
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
    if isinstance(paged_kv_cache, torch.Tensor):
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
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype != _I32:
        raise TypeError(f"{name} must be int32 (got {t.dtype})")
    if t.device != dev or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector on the cache's device")


def _attention(query, paged_kv_cache: Cache, own, prefix, group_indptr, qo_indptr, scale, causal, return_lse, out):
    if not isinstance(query, torch.Tensor):
        raise TypeError(f"query must be a torch.Tensor, got {type(query).__name__}")
    idx = query.get_device()
    if idx >= 0 and idx != _current_device():
        with torch.cuda.device(idx):
            return _attention(query, paged_kv_cache, own, prefix, group_indptr, qo_indptr, scale, causal, return_lse, out)
    if isinstance(paged_kv_cache, torch.Tensor):
        k_cache, v_cache = paged_kv_cache, None
    else:
        k_cache, v_cache = paged_kv_cache
    result = torch.empty_like(query, memory_format=torch.contiguous_format) if out is None else out
    lse = None
    if return_lse:
        shape = query.shape
        heads = shape[1] if len(shape) == 3 else shape[1] // max(1, k_cache.shape[-1]) if len(shape) == 2 else 0
        lse = torch.empty((shape[0] if shape else 0, heads), dtype=torch.float32, device=query.device)
    size_of, run = _entries or _entry_points()
    # all checks of the tensors are made there (csrc/packer.c)
    rc = _packer.attention(size_of, run, _raw_stream_of(idx) if idx >= 0 else 0, idx, query, k_cache, v_cache, *own,
                           qo_indptr, *prefix, group_indptr, scale, causal, result, lse)
    if rc:
        _lib.check(rc)
    elif rc is None:
        lists = [("kv_", "request", own)]
        if prefix[0] is not None:
            lists.append(("prefix_", "group", prefix))
        _refuse(query, paged_kv_cache, lists, qo_indptr, group_indptr, out)
    return (result, lse) if return_lse else result


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
    ``[T, num_heads]``.  A row that reads no key is 0, its logarithm ``-inf``.  NaN and infinities in
    keys and values reach the rows that read them, as in the formula (an infinity whose weight is
    below 2^-126 of the row's largest, in fp16 2^-22, may give NaN or be lost), and no other row.  Rows outside ``qo_indptr[0]:qo_indptr[-1]`` (a padded
    batch) are not written, their logarithms neither: pass ``out`` (same shape and dtype, sharing no
    memory with the inputs) to say what they hold.

    Head dims up to 256 that are multiples of 8; 64 and 128 run on the tensor cores, the others on the
    CUDA cores, which is slow for prompts.  Forward only: nothing is recorded for a gradient.
    """
    return _attention(query, paged_kv_cache, (kv_indptr, kv_indices, kv_last_page_len), (None, None, None), None,
                      qo_indptr, scale, causal, return_lse, out)


def shared_prefix_attention(query: torch.Tensor, paged_kv_cache: Cache,
                            prefix_indptr: torch.Tensor, prefix_indices: torch.Tensor,
                            prefix_last_page_len: torch.Tensor, kv_indptr: torch.Tensor,
                            kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor,
                            group_indptr: Optional[torch.Tensor] = None,
                            qo_indptr: Optional[torch.Tensor] = None,
                            scale: Optional[float] = None, causal: bool = True,
                            return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """:func:`paged_attention` for requests that share prefixes, read once for all of them where the
    head dim is 64 or 128 (once a row otherwise: right, but nothing is saved).

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
