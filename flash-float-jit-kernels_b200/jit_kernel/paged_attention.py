"""Attention of every sequence's newest token over its whole context: the step of layers that select nothing, beside
``sparse_attention`` (no counterpart in the reference). The context lies in pages of a cache in 16 bits or as the e4m3 codes of
``kv_cache``. What every cached row has been given so far - what ``kv_cache.cache_evict`` goes by - is brought up to date on the way."""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional

import torch

from . import _native
from .kv_cache import _check_table, _check_weight
from .norm_rope import _DENSE, FP8, _check_cache, _check_vector, _no_grad
from .sparse_attention import _TYPES
from .topk_indexer import _launch

#: fftopk_paged (include/fftopk.h)
_ARGS = struct.Struct("@PqqPqqPqqPqqPqqPqPPqqPPqqPqqqqqiiiiiifi")


def paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    page_size: int,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    weight: Optional[torch.Tensor] = None,
    weight_out: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
):
    """
    Args:
        q: [B, Hq, D], float16 or bfloat16, CUDA, D 64 or 128, unit inner stride, rows on 16 bytes: one token of each sequence.
        k_cache, v_cache: [slots, Hk, D], Hq a multiple of Hk (query head h uses head h // (Hq / Hk)); of q's type, or
            float8_e4m3fn with k_scale and v_scale, float32 [slots, Hk]. Any strides whose rows start on 16 bytes.
        page_table: int32 [B, pages], unit inner stride. Position j of sequence b is row page_table[b, j // page_size] * page_size
            + j % page_size of the caches. Entries behind a sequence's length are not read; a negative page is left out with its
            positions; a row beyond the cache, and positions beyond the table, are left out and show up in kernel_status().
        lengths: int32 [B], the sequences' lengths, the newest token's own row among them; 0 for a row of a padded batch.
        page_size: rows of a page, any number from 1.
        softmax_scale: default D ** -0.5.
        weight, weight_out: float32 [B, Hk, N], unit inner stride, N at least the longest length: the attention weights each cached
            row has had. weight_out = weight + this call's, added up over the query heads of a key head. weight alone: updated in
            place; weight_out alone: this call's. Behind a sequence's length weight_out stays as it was. The call then takes
            4 bytes of workspace per query head (rounded up to eights of a key head's) and position the table has room for: hand in a
            page_table as wide as the longest sequence.
        out: [B, Hq, D] of q's type for the result, apart from q (and weight_out, where it is not weight, from weight): rows in one buffer
            are fine, on one another they are refused. (Neither is a broadcast view.)
    Returns:
        out, or (out, lse) with lse float32 [B, Hq], the log of the sum of exponentials. A sequence without rows: 0 and -inf.
    """
    idx, shape, qs, dtype = q.get_device(), q.shape, q.stride(), q.dtype
    if idx < 0 or len(shape) != 3:
        raise RuntimeError("q must be a CUDA tensor [sequences, heads, D]")
    B, Hq, D = shape
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
    if not 1 <= page_size <= 0x7fffffff:
        raise RuntimeError("page_size must be at least 1")
    table, row, pages = _check_table(page_table, "page_table", idx, B)
    if pages * page_size > 0x7ffffff0:
        raise RuntimeError("page_table names more than 2^31 - 16 positions of a sequence")
    at = _check_vector(lengths, "lengths", idx, B)
    if lengths is None:
        raise RuntimeError("lengths are missing")
    w = wo = 0
    ws = wos = (0, 0, 0)
    cols = 0
    if weight is not None:
        ws, cols = _check_weight(weight, "weight", idx, B, Hk)
        if weight_out is None:
            weight_out = weight
        w = weight.data_ptr()
    if weight_out is not None:
        wos, cols = _check_weight(weight_out, "weight_out", idx, B, Hk, cols if weight is not None else -1)
        wo = weight_out.data_ptr()
    _no_grad(q, k_cache, v_cache, k_scale, v_scale, weight, weight_out, out)
    if out is None:
        out = torch.empty_like(q, memory_format=_DENSE)
        os = (Hq * D, D)
    else:
        os = out.stride()
        if out.dtype is not dtype or out.shape != q.shape or out.get_device() != idx or os[2] != 1:
            raise RuntimeError("out must have q's shape and type, unit inner stride, on q's device")
    lse = torch.empty((B, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    if B and Hq:
        args = _ARGS.pack(
            q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), ks[0], ks[1], v_cache.data_ptr(), vs[0], vs[1], ka, kss[0], kss[1], va, vss[0],
            vss[1], table, row, at, out.data_ptr(), os[0], os[1], lse.data_ptr() if return_lse else 0, w, ws[0], ws[1], wo, wos[0], wos[1],
            cols, B, slots, Hq, Hk, D, pages, page_size, _TYPES[dtype], D ** -0.5 if softmax_scale is None else softmax_scale, 0)
        n = _workspace_bytes(idx, B, Hq, Hk, D, pages, page_size, ka != 0, wo != 0)
        space = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        _launch(_native.lib().fftopk_paged_attention, "fftopk_paged_attention", idx, args, space.data_ptr() if n else 0, n)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=256)
def _workspace_bytes(idx: int, B: int, Hq: int, Hk: int, D: int, pages: int, page_size: int, fp8: bool, weigh: bool) -> int:
    """What the library asks for a call of these sizes on device idx: no address of it counts, 256 stands for all that are there."""
    there = 256
    args = _ARGS.pack(there, 0, 0, there, 0, 0, there, 0, 0, there * fp8, 0, 0, there * fp8, 0, 0, there, 0, there, there, 0, 0, 0, 0, 0, 0,
                      there * weigh, 0, 0, 0, B, 1, Hq, Hk, D, pages, page_size, 0, 0.0, 0)
    n = ctypes.c_size_t()
    with torch.cuda.device(idx):
        rc = _native.lib().fftopk_paged_workspace_bytes(args, ctypes.byref(n))
    if rc:
        _native.check(rc, "fftopk_paged_attention")
    return n.value
