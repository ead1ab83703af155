"""A cache of keys or values in fp8: e4m3 codes [slots, heads, D] with a float32 scale per slot and head, quantised as it is
written and widened as it is read (no counterpart in the reference). A slot is a token's row; which one a token has is the
caller's affair (a page table's entry, a sequence's base plus the position). ``sparse_attention`` reads such caches as they are."""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from .norm_rope import _DTYPES, _check_cache, _check_first, _check_rows, _check_vector, _no_grad, _quantised, _rows
from .topk_indexer import _launch


def cache_write(
    k: torch.Tensor,
    slots: torch.Tensor,
    k_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v: Optional[torch.Tensor] = None,
    v_cache: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> None:
    """
    Quantise k - and v, in the same launch - into rows `slots` of their caches.
    Args:
        k, v: [T, H, D] of one type (float16, bfloat16, float32), CUDA, unit inner stride; D a multiple of 8 up to 256.
        slots: int32 [T]. A negative slot is padding: that token is not written. A slot beyond the cache is not written either
            and shows up in kernel_status(). The slots of one call differ from one another.
        k_cache, v_cache: float8_e4m3fn [slots, H, D], unit inner stride; k_scale, v_scale: float32 [slots, H].
    A row's largest finite magnitude becomes 448 (scale = amax / 448, codes to nearest even); infinities become the largest code,
    NaN stays NaN. Rows that no slot names keep what they hold.
    """
    idx, T, D, dtype = _check_first(k, "k")
    H, xs = _check_rows(k, "k", idx, dtype, T, D)
    at = _check_vector(slots, "slots", idx, T)
    n, cs, ss = _check_cache(k_cache, k_scale, "k", idx, H, D)
    _no_grad(k, k_cache, k_scale, v, v_cache, v_scale)
    parts = _quantised(k, xs, H, k_cache, cs, k_scale, ss, at, n)
    if v is not None:
        if v_cache is None:
            raise RuntimeError("v, v_cache and v_scale go together")
        H, xs = _check_rows(v, "v", idx, dtype, T, D)
        n, cs, ss = _check_cache(v_cache, v_scale, "v", idx, H, D)
        parts += _quantised(v, xs, H, v_cache, cs, v_scale, ss, at, n)
    elif v_cache is not None or v_scale is not None:
        raise RuntimeError("v, v_cache and v_scale go together")
    if T:
        _rows(idx, parts, T, D, dtype)


def cache_read(
    cache: torch.Tensor,
    scale: torch.Tensor,
    slots: torch.Tensor,
    *,
    offsets: Optional[torch.Tensor] = None,
    dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """
    Rows of a quantised cache, gathered and widened.
    Args:
        cache, scale: float8_e4m3fn [slots, H, D] and float32 [slots, H], as cache_write fills them.
        slots: int32 [B, K] or [K], contiguous: the rows to read, -1 for none (zeros) - what the selector hands out, for instance.
        offsets: int32 [B] (with slots [B, K]): added to the non-negative entries of row b.
        dtype: float16, bfloat16 or float32.
    Returns:
        slots.shape + [H, D], contiguous. A row beyond the cache gives zeros and shows up in kernel_status().
    """
    idx = cache.get_device()
    if idx < 0 or cache.dim() != 3:
        raise RuntimeError("cache must be a CUDA tensor [slots, heads, D]")
    _, H, D = cache.shape
    n, cs, ss = _check_cache(cache, scale, "the", idx, H, D)
    if D % 8 or not 8 <= D <= 256:
        raise RuntimeError("D must be a multiple of 8 up to 256")
    if dtype not in _DTYPES:
        raise RuntimeError("dtype must be float16, bfloat16 or float32")
    shape = slots.shape
    if slots.dtype is not torch.int32 or len(shape) not in (1, 2) or not slots.is_contiguous() or slots.get_device() != idx:
        raise RuntimeError("slots must be a contiguous int32 tensor [B, K] or [K] on the cache's device")
    rows, per_row = shape if len(shape) == 2 else (1, shape[0])
    if offsets is not None and len(shape) != 2:
        raise RuntimeError("offsets go with slots [B, K]")
    off = _check_vector(offsets, "offsets", idx, rows)
    _no_grad(cache, scale)
    out = scale.new_empty((*shape, H, D), dtype=dtype)
    if rows and per_row and H:
        _launch(_native.lib().fftopk_cache_read, "fftopk_cache_read", idx, cache.data_ptr(), cs[0], cs[1], n, H, D, scale.data_ptr(), ss[0],
                ss[1], slots.data_ptr(), rows, per_row, off, out.data_ptr(), _DTYPES[dtype])
    return out
