"""A cache of keys or values in fp8: e4m3 codes [slots, heads, D] with a float32 scale per slot and head, quantised as it is
written and widened as it is read (no counterpart in the reference). A slot is a token's row; which one a token has is the
caller's affair (a page table's entry, a sequence's base plus the position). ``sparse_attention`` and ``paged_attention`` read such
caches as they are; ``cache_evict`` thins them, or 16-bit ones, by the weights ``paged_attention`` adds up."""
from __future__ import annotations

import struct
from typing import Optional

import torch

from . import _native
from .norm_rope import _DENSE, _DTYPES, FP8, _check_cache, _check_first, _check_rows, _check_vector, _no_grad, _quantised, _rows
from .topk_indexer import _launch

#: fftopk_evict (include/fftopk.h)
_EVICT = struct.Struct("@PqqPqqPqqPqqPqqPqqPqPqPPPqqqiiiiiiiiii")


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


def _check_table(t: torch.Tensor, what: str, idx: int, seqs: int):
    """(address, row stride, columns) of a page table"""
    shape, step = t.shape, t.stride()
    if t.dtype is not torch.int32 or len(shape) != 2 or shape[0] != seqs or t.get_device() != idx or (shape[1] > 1 and step[1] != 1):
        raise RuntimeError(f"{what} must be an int32 tensor [sequences, pages] with unit inner stride on the cache's device")
    return t.data_ptr(), step[0], shape[1]


def _check_weight(t: torch.Tensor, what: str, idx: int, seqs: int, heads: int, cols: int = -1):
    """(strides, columns) of weights [sequences, key heads, positions]"""
    shape, step = t.shape, t.stride()
    if t.dtype is not torch.float32 or len(shape) != 3 or shape[0] != seqs or shape[1] != heads or t.get_device() != idx \
            or (cols >= 0 and shape[2] != cols) or (shape[2] > 1 and step[2] != 1):
        raise RuntimeError(f"{what} must be float32 [sequences, key heads, positions] with unit inner stride on the cache's device")
    return step, shape[2]


def cache_evict(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    weight: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    to_table: torch.Tensor,
    *,
    page_size: int,
    budget: int,
    recent: int = 0,
    sinks: int = 0,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    weight_out: Optional[torch.Tensor] = None,
):
    """
    Thin out sequences of a paged cache: of every sequence and key head the `budget` rows that have had the most attention move to other
    pages, in order. The old pages are the caller's to free (or stay with the sequences that share them).
    Args:
        k_cache, v_cache: [slots, Hk, D], float16, bfloat16, or float8_e4m3fn with k_scale and v_scale, float32 [slots, Hk]; unit inner
            stride, D a multiple of 8 up to 256. Written at the rows that to_table names.
        weight: float32 [B, Hk, N], unit inner stride, N at least the longest length: what paged_attention has added up.
        page_table: int32 [B, pages]; lengths: int32 [B]: as for paged_attention.
        to_table: int32 [B, pages for `budget` rows at least]: where the rows go; none of the pages that page_table names for any
            sequence of the call.
        budget: rows that a key head keeps; a sequence of up to that many keeps (and moves) all of them.
        recent, sinks: of those, the last and the first rows of the sequence, whatever their weight. Between them the largest weights
            stay, of equal ones the lower positions (NaN counts as the largest).
        weight_out: float32 [B, Hk, N] for the weights of what stays, zeros behind (default: a new tensor; apart from weight,
            no broadcast view).
    Returns:
        (kept, lengths, weight_out): int32 [B, Hk, budget], the positions that stayed in ascending order, -1 behind them; int32 [B],
        the new lengths; the weights. Rows on negative pages or beyond the cache are not copied and show up in kernel_status(), as do
        lengths beyond the table or the weights.
    """
    idx, shape, dtype = k_cache.get_device(), k_cache.shape, k_cache.dtype
    if idx < 0 or len(shape) != 3 or v_cache.shape != shape:
        raise RuntimeError("k_cache and v_cache must be CUDA tensors [slots, heads, D] of one shape")
    slots, H, D = shape
    if D % 8 or not 8 <= D <= 256:
        raise RuntimeError("D must be a multiple of 8 up to 256")
    ka = va = 0
    if dtype is FP8:
        _, ks, kss = _check_cache(k_cache, k_scale, "k", idx, H, D)
        _, vs, vss = _check_cache(v_cache, v_scale, "v", idx, H, D)
        ka, va = k_scale.data_ptr(), v_scale.data_ptr()
    else:
        if k_scale is not None or v_scale is not None:
            raise RuntimeError("k_scale and v_scale go with float8_e4m3fn caches")
        if dtype not in (torch.float16, torch.bfloat16) or v_cache.dtype is not dtype or v_cache.get_device() != idx:
            raise RuntimeError("the caches must be of one type, float16, bfloat16 or float8_e4m3fn, on one device")
        ks, vs, kss, vss = k_cache.stride(), v_cache.stride(), (0, 0), (0, 0)
        if ks[2] != 1 or vs[2] != 1:
            raise RuntimeError("the caches must have unit inner stride")
    if weight.dim() != 3:
        raise RuntimeError("weight must be float32 [sequences, key heads, positions]")
    B = weight.shape[0]
    ws, cols = _check_weight(weight, "weight", idx, B, H)
    if not 1 <= page_size <= 0x7fffffff:
        raise RuntimeError("page_size must be at least 1")
    table, row, pages = _check_table(page_table, "page_table", idx, B)
    to, to_row, to_pages = _check_table(to_table, "to_table", idx, B)
    if lengths is None:
        raise RuntimeError("lengths are missing")
    at = _check_vector(lengths, "lengths", idx, B)
    if budget < 0 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise RuntimeError("recent and sinks are parts of the budget")
    if budget > to_pages * page_size:
        raise RuntimeError("to_table has no room for the budget")
    _no_grad(k_cache, v_cache, k_scale, v_scale, weight, weight_out)
    if weight_out is None:
        weight_out = torch.empty_like(weight, memory_format=_DENSE)
        wos = (H * cols, cols)
    else:
        wos, _ = _check_weight(weight_out, "weight_out", idx, B, H, cols)
        if weight_out.data_ptr() == weight.data_ptr() and weight.numel():
            raise RuntimeError("weight_out must not be weight itself")
    kept = torch.empty((B, H, budget), dtype=torch.int32, device=lengths.device)
    left = torch.empty_like(lengths)
    if B and H:
        args = _EVICT.pack(
            k_cache.data_ptr(), ks[0], ks[1], v_cache.data_ptr(), vs[0], vs[1], ka, kss[0], kss[1], va, vss[0], vss[1], weight.data_ptr(),
            ws[0], ws[1], weight_out.data_ptr(), wos[0], wos[1], table, row, to, to_row, at, left.data_ptr(), kept.data_ptr(), cols, B, slots,
            H, D, 1 if dtype is FP8 else 2, pages, to_pages, page_size, budget, recent, sinks, 0)
        _launch(_native.lib().fftopk_cache_evict, "fftopk_cache_evict", idx, args)
    else:
        left.zero_()
    return kept, left, weight_out
