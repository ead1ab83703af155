"""Attention over the tokens a selection names: the step behind the selector (no counterpart in the reference, which ends with
the indices). It reads the rows it is told of where they lie, in 16 bits or as the e4m3 codes of ``kv_cache``, and takes the
indices as ``fast_topk_v3`` and ``FusedIndexerTopk`` (with `offsets`: a sequence's first slot), ``fast_topk_transform_fused`` or
``fast_topk_transform_ragged_fused`` (slots already) hand them out. A tree of drafted tokens is a list of indices per token too:
the context's picks and the slots of the token's ancestors."""
from __future__ import annotations

import struct
from typing import Optional

import torch

from . import _native
from .norm_rope import _DENSE, FP8, _check_cache, _check_vector, _no_grad
from .topk_indexer import _launch

_TYPES = {torch.float16: 0, torch.bfloat16: 1}
#: fftopk_attend (include/fftopk.h)
_ARGS = struct.Struct("@PqqPqqPqqPqqPqqPqPPqqPqqiiiiif")


def sparse_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    indices: torch.Tensor,
    *,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    offsets: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
):
    """
    Args:
        q: [T, Hq, D], float16 or bfloat16, CUDA, D 64 or 128, unit inner stride, rows on 16 bytes.
        k_cache, v_cache: [slots, Hk, D], Hq a multiple of Hk (query head h uses head h // (Hq / Hk)); of q's type, or
            float8_e4m3fn with k_scale and v_scale, float32 [slots, Hk]. Any strides whose rows start on 16 bytes.
        indices: int32 [T, K], unit inner stride: the cache rows token t attends to, in any order, negative entries left out
            wherever they stand; shared by the heads. An index named twice counts twice; one beyond the cache is left out and
            shows up in kernel_status().
        offsets: int32 [T], added to the non-negative entries of a row.
        softmax_scale: default D ** -0.5.
        out: [T, Hq, D] of q's type for the result.
    Returns:
        out, or (out, lse) with lse float32 [T, Hq], the log of the sum of exponentials. A token without entries: 0 and -inf.
    """
    idx, shape, qs, dtype = q.get_device(), q.shape, q.stride(), q.dtype
    if idx < 0 or len(shape) != 3:
        raise RuntimeError("q must be a CUDA tensor [tokens, heads, D]")
    T, Hq, D = shape
    if dtype not in _TYPES:
        raise RuntimeError("q must be float16 or bfloat16")
    if D not in (64, 128):
        raise RuntimeError("D must be 64 or 128")
    if qs[2] != 1:
        raise RuntimeError("q must have unit inner stride")
    shape = k_cache.shape
    if len(shape) != 3 or v_cache.shape != shape or shape[2] != D:
        raise RuntimeError("k_cache and v_cache must be [slots, heads, D] with q's D")
    slots, Hk, _ = shape
    if Hk == 0 or Hq % Hk:
        raise RuntimeError("q's heads must be a multiple of the cache's")
    ka = va = 0
    if k_cache.dtype is FP8:
        _, ks, kss = _check_cache(k_cache, k_scale, "k", idx, Hk, D)
        _, vs, vss = _check_cache(v_cache, v_scale, "v", idx, Hk, D)
        ka, va = k_scale.data_ptr(), v_scale.data_ptr()
    else:
        if k_scale is not None or v_scale is not None:
            raise RuntimeError("k_scale and v_scale go with float8_e4m3fn caches")
        if k_cache.dtype is not dtype or v_cache.dtype is not dtype:
            raise RuntimeError("the caches must both be of q's type, or both float8_e4m3fn")
        if k_cache.get_device() != idx or v_cache.get_device() != idx:
            raise RuntimeError("the caches must be on q's device")
        ks, vs, kss, vss = k_cache.stride(), v_cache.stride(), (0, 0), (0, 0)
        if ks[2] != 1 or vs[2] != 1:
            raise RuntimeError("the caches must have unit inner stride")
    picks, step = indices.shape, indices.stride()
    if indices.dtype is not torch.int32 or len(picks) != 2 or picks[0] != T or indices.get_device() != idx \
            or (picks[1] > 1 and step[1] != 1) or picks[1] > 0x7fffffff:
        raise RuntimeError("indices must be an int32 tensor [tokens, K < 2^31] with unit inner stride on q's device")
    off = _check_vector(offsets, "offsets", idx, T)
    _no_grad(q, k_cache, v_cache, k_scale, v_scale, out)
    if out is None:
        out = torch.empty_like(q, memory_format=_DENSE)
        os = (Hq * D, D)
    else:
        os = out.stride()
        if out.dtype is not dtype or out.shape != q.shape or out.get_device() != idx or os[2] != 1:
            raise RuntimeError("out must have q's shape and type, unit inner stride, on q's device")
    lse = q.new_empty((T, Hq), dtype=torch.float32) if return_lse else None
    if T and Hq:
        args = _ARGS.pack(
            q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), ks[0], ks[1], v_cache.data_ptr(), vs[0], vs[1], ka, kss[0], kss[1], va, vss[0],
            vss[1], indices.data_ptr(), step[0], off, out.data_ptr(), os[0], os[1], lse.data_ptr() if return_lse else 0, T, slots, Hq, Hk, D,
            picks[1], _TYPES[dtype], D ** -0.5 if softmax_scale is None else softmax_scale)
        _launch(_native.lib().fftopk_sparse_attention, "fftopk_sparse_attention", idx, args)
    return (out, lse) if return_lse else out
