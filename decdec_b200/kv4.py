"""The 4-bit key/value cache of a decoder layer and what stands around it: positions into queries and keys, pages and slots of a
step, new rows into the cache, attention over it.  No counterpart in the reference binding, whose models keep a dense 16-bit cache
(end-to-end/model.py).

A step of a layer, for a batch of requests whose tokens lie one request after another:

    p = kv4.plan(lengths, new_lengths, block_table, free_pages, free_count, page_size, tokens)        # once for all layers
    q, k = kv4.rotary(q, k, p.positions, frequencies, factor=factor)
    kv4.append(cache, k, v, p.slots, group_size)
    y = kv4.attention(q, cache, block_table, p.lengths, p.query_starts, group_size, max_queries=n)

A batch of one with a contiguous cache is a block table that counts up.  Nothing synchronises and every call can be captured in a
CUDA graph once a call has run eagerly on the device; lengths, tables and slots are read on the device.  Elements are held as
offset + step * code with 16 codes and one (step, offset) for `group_size` elements of a head; `include/decdec_b200.h` gives the
format.  Tensors: fp16 or bf16, [tokens, heads, head_dim], any strides with neighbouring elements in a head.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional

import torch

from . import capi
from .ops import _DT, _call, _check, _stream

_INTS = (torch.int32, torch.int64)


class Plan(NamedTuple):
    positions: torch.Tensor       # int64 [tokens], 0 behind the last new token
    slots: torch.Tensor           # int64 [tokens], -1 behind it
    query_starts: torch.Tensor    # int32 [requests + 1]
    lengths: torch.Tensor         # int32 [requests], the new tokens included
    free_count: torch.Tensor      # int32 [1]
    status: torch.Tensor          # int32 [1]: 0, or why nothing was given (1 pages, 2 table, 4 tokens, 8 a negative count)


def cell_bytes(head_dim: int, group_size: int) -> int:
    """Bytes of 16 tokens of one head."""
    _check(head_dim in (64, 128, 256), f"head_dim must be 64, 128 or 256, got {head_dim}.")
    _check(group_size in (32, 64, 128) and group_size <= head_dim, f"group_size must be 32, 64 or 128 and not above head_dim, got {group_size}.")
    return 16 * (head_dim + 8 * head_dim // group_size)


def empty_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, group_size: int, device="cuda") -> torch.Tensor:
    """A cache of `pages` pages of `page_size` tokens (a multiple of 16): uint8 [pages, kv_heads, bytes of a page], zeros."""
    _check(page_size > 0 and page_size % 16 == 0, f"page_size must be a multiple of 16, got {page_size}.")
    return torch.zeros((pages, kv_heads, page_size // 16 * cell_bytes(head_dim, group_size)), dtype=torch.uint8, device=device)


def _cache(cache: torch.Tensor, head_dim: int, group_size: int):
    """pages, page_size, kv_heads of a cache."""
    _check(cache.dtype == torch.uint8 and cache.dim() == 3 and cache.is_contiguous(), "cache must be a contiguous uint8 tensor [pages, kv_heads, bytes].")
    pages, kv_heads, size = cache.shape
    cell = cell_bytes(head_dim, group_size)
    _check(size > 0 and size % cell == 0, f"a page of {size} bytes is no whole number of cells of {cell} bytes (head_dim {head_dim}, group_size {group_size}).")
    return pages, size // cell * 16, kv_heads


def _rows(t: torch.Tensor, name: str) -> tuple:
    _check(t.dim() == 3, f"{name} must be of shape (tokens, heads, head_dim).")
    _check(t.stride(2) == 1 or t.size(2) <= 1, f"elements of a head of {name} must be neighbours.")
    return t.data_ptr(), t.stride(0), t.stride(1)


def _same_device(first: torch.Tensor, *others) -> None:
    _check(first.is_cuda, "tensors must be on GPU.")
    for t in others:
        _check(t is None or t.device == first.device, "all tensors must be on the same GPU.")


def _index(t: torch.Tensor, n: int, name: str) -> tuple:
    _check(t.dtype in _INTS and t.dim() == 1 and t.is_contiguous() and t.numel() == n, f"{name} must be a contiguous int32 or int64 tensor of {n} entries.")
    return t.data_ptr(), int(t.dtype == torch.int64)


def _int32(t: torch.Tensor, n: Optional[int], name: str) -> int:
    _check(t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous() and (n is None or t.numel() == n),
           f"{name} must be a contiguous int32 tensor" + ("." if n is None else f" of {n} entries."))
    return t.data_ptr()


def _table(t: torch.Tensor, requests: int) -> tuple:
    _check(t.dtype == torch.int32 and t.dim() == 2 and t.size(0) == requests and (t.size(1) <= 1 or t.stride(1) == 1),
           "block_table must be an int32 tensor of shape (requests, pages) with neighbouring entries.")
    return t.data_ptr(), t.stride(0), t.size(1)


# ---- rotary positions ---------------------------------------------------------------------------------------

def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None, device="cuda") -> tuple:
    """Rotation per position of each pair, float64 [rotary_dim / 2], and the factor of the rotated values.

    `scaling` for contexts beyond the trained ones, by its "type":
      "linear"  {"factor"}: all pairs turn `factor` times slower
      "llama3"  {"factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"}: pairs with fewer than low_freq_factor
                turns over the trained length turn slower, those with more than high_freq_factor do not, between them a blend
      "yarn"    {"factor", "original_max_position_embeddings", "beta_fast" (32), "beta_slow" (1), "attention_factor" (0.1 ln factor + 1)}: the
                same with a ramp over the pair's index, and a factor on the rotated values
    """
    _check(rotary_dim > 0 and rotary_dim % 2 == 0, f"rotary_dim must be even and above 0, got {rotary_dim}.")
    f = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    factor = 1.0
    if scaling is not None:
        kind, by = scaling.get("type"), float(scaling.get("factor", 1.0))
        _check(by >= 1.0, f"the factor of a scaling must be at least 1, got {by}.")
        if kind == "linear":
            f = f / by
        elif kind == "llama3":
            lo, hi = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
            _check(hi > lo, "high_freq_factor must be above low_freq_factor.")
            keep = ((scaling["original_max_position_embeddings"] * f / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1)
            f = f * (keep + (1 - keep) / by)
        elif kind == "yarn":
            far = scaling["original_max_position_embeddings"]

            def pair(turns):
                return rotary_dim * math.log(far / (turns * 2 * math.pi)) / (2 * math.log(base))

            lo = max(math.floor(pair(scaling.get("beta_fast", 32.0))), 0)
            hi = min(math.ceil(pair(scaling.get("beta_slow", 1.0))), rotary_dim // 2 - 1)
            slow = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
            f = f * (1 - slow + slow / by)
            factor = float(scaling.get("attention_factor", 0.1 * math.log(by) + 1.0))
        else:
            _check(False, f"unknown scaling type {kind!r}: linear, llama3 or yarn.")
    return f.to(device), factor


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, interleaved: bool = False,
           factor: float = 1.0, out: Optional[tuple] = None) -> tuple:
    """Positions into queries and keys (k may be None): the first 2 * len(frequencies) elements of each head are turned, the rest copied.
    Pairs are neighbours if `interleaved`, else half of the turned elements apart.  Angles are taken in 64 bits.  fp16, bf16, fp32.
    out=(q', k'): where to, which may be q and k themselves.  Returns (q', k')."""
    _check(q.dtype in _DT, "Unsupported data type.")
    tokens, heads, d = q.shape if q.dim() == 3 else (0, 0, 0)
    args = [*_rows(q, "q"), heads]
    _same_device(q, k, positions, frequencies)
    if k is not None:
        args += [*_rows(k, "k"), k.size(1)]
        _check(k.dtype == q.dtype and k.size(0) == tokens and k.size(2) == d, "q and k must share data type, tokens and head_dim.")
    else:
        args += [None, 0, 0, 0]
    _check(frequencies.dtype == torch.float64 and frequencies.dim() == 1 and frequencies.is_contiguous(), "frequencies must be a contiguous float64 vector.")
    _check(0 < 2 * frequencies.numel() <= d, "there are more frequencies than pairs in a head, or none.")
    at, wide = _index(positions, tokens, "positions")
    if out is None:
        q_out = torch.empty((tokens, heads, d), dtype=q.dtype, device=q.device)
        k_out = None if k is None else torch.empty((tokens, k.size(1), d), dtype=q.dtype, device=q.device)
    else:
        q_out, k_out = out
        _check(q_out.shape == q.shape and q_out.dtype == q.dtype and (k is None) == (k_out is None), "out must have the shapes and types of q and k.")
        _check(k is None or (k_out.shape == k.shape and k_out.dtype == k.dtype), "out must have the shapes and types of q and k.")
        _same_device(q, q_out, k_out)
    args += _rows(q_out, "out")
    args += [None, 0, 0] if k is None else _rows(k_out, "out")
    with torch.cuda.device(q.device):
        _call("decdec_rotary", *args, at, wide, frequencies.data_ptr(), tokens, d, 2 * frequencies.numel(), int(interleaved), float(factor),
              _DT[q.dtype], _stream())
    return q_out, k_out


# ---- pages and slots of a step ---------------------------------------------------------------------------------

def plan(lengths: torch.Tensor, new_lengths: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
         page_size: int, tokens: int) -> Plan:
    """Pages, slots and positions of the next step from lengths[b] tokens held and new_lengths[b] to come (int32), on the device.

    A request that outgrows its pages takes the last of free_pages[:free_count]; they are entered in `block_table`, which is
    written in place.  `tokens`: entries of positions and slots, at least the sum of new_lengths.  All or nothing: if status is not 0
    no page is given, slots are -1, query_starts 0, lengths and free_count as they were."""
    requests = lengths.numel()
    _same_device(lengths, new_lengths, block_table, free_pages, free_count)
    device = lengths.device
    args = [_int32(lengths, None, "lengths"), _int32(new_lengths, requests, "new_lengths"), requests, *_table(block_table, requests),
            _int32(free_pages, None, "free_pages"), free_pages.numel(), _int32(free_count, 1, "free_count"), int(page_size), int(tokens)]
    _check(tokens >= 0, "tokens must not be negative.")
    wide = torch.empty((2, tokens), dtype=torch.int64, device=device)
    narrow = torch.empty(2 * requests + 3, dtype=torch.int32, device=device)
    starts, after, left, status = narrow.split([requests + 1, requests, 1, 1])
    with torch.cuda.device(device):
        _call("decdec_kv4_plan", *args, wide[0].data_ptr(), wide[1].data_ptr(), starts.data_ptr(), after.data_ptr(), left.data_ptr(), status.data_ptr(),
              _stream())
    return Plan(wide[0], wide[1], starts, after, left, status)


# ---- rows into the cache and out of it ---------------------------------------------------------------------------

def append(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, group_size: int) -> None:
    """Writes rows of keys and values [tokens, kv_heads, head_dim] to their slots (page * page_size + place; negative: skipped).
    Slots must differ: of two rows with the same slot any mixture may stay."""
    _check(k.dtype in (torch.float16, torch.bfloat16) and v.dtype == k.dtype, "k and v must both be half or both bfloat16.")
    args = [*_rows(k, "k"), *_rows(v, "v")]
    _check(k.shape == v.shape, "k and v must have the same shape.")
    _same_device(k, v, slots, cache)
    pages, page_size, kv_heads = _cache(cache, k.size(2), group_size)
    _check(k.size(1) == kv_heads, f"the cache has {kv_heads} heads, k and v have {k.size(1)}.")
    at, wide = _index(slots, k.size(0), "slots")
    with torch.cuda.device(k.device):
        _call("decdec_kv4_append", *args, at, wide, k.size(0), cache.data_ptr(), pages, page_size, kv_heads, k.size(2), group_size, _DT[k.dtype], _stream())


def gather(cache: torch.Tensor, slots: torch.Tensor, head_dim: int, group_size: int, dtype: torch.dtype) -> tuple:
    """Dense keys and values [len(slots), kv_heads, head_dim] of slots, in any order; zeros for negative ones."""
    _check(dtype in (torch.float16, torch.bfloat16), "dtype must be half or bfloat16.")
    _same_device(cache, slots)
    pages, page_size, kv_heads = _cache(cache, head_dim, group_size)
    n = slots.numel()
    at, wide = _index(slots, n, "slots")
    out = torch.empty((2, n, kv_heads, head_dim), dtype=dtype, device=cache.device)
    k, v = out[0], out[1]
    with torch.cuda.device(cache.device):
        _call("decdec_kv4_gather", cache.data_ptr(), pages, page_size, kv_heads, head_dim, group_size, at, wide, n, k.data_ptr(), v.data_ptr(), _DT[dtype],
              _stream())
    return k, v


# ---- attention ---------------------------------------------------------------------------------------------------

def attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, query_starts: torch.Tensor, group_size: int,
              max_queries: Optional[int] = None, scale: Optional[float] = None, window: int = 0, out: Optional[torch.Tensor] = None,
              return_lse: bool = False):
    """softmax(scale q k^T) v over the cache, causal: request b has the rows query_starts[b]..query_starts[b+1]-1 of q [tokens, heads,
    head_dim], which are its last tokens, and lengths[b] tokens in the cache with them.  Query head h reads key head h * kv_heads // heads.

    window > 0: each row sees the last `window` tokens up to its own.  A row that sees no token gives zeros.  max_queries: the most rows of a
    request (default: all rows), which chooses the kernel.  scale: default head_dim ** -0.5.  Rows behind the last request are left as
    they are in `out`, zeros where `out` is not given.  return_lse: also the fp32 logarithms [tokens, heads] of the sums of exp(scale q k^T)."""
    _check(q.dtype in (torch.float16, torch.bfloat16), "q must be half or bfloat16.")
    at = _rows(q, "q")
    tokens, heads, d = q.shape
    _same_device(q, cache, block_table, lengths, query_starts, out)
    pages, page_size, kv_heads = _cache(cache, d, group_size)
    _check(kv_heads > 0 and heads > 0 and heads % kv_heads == 0, f"heads of q must be a multiple of the cache's {kv_heads}, got {heads}.")
    requests = lengths.numel()
    table = _table(block_table, requests)
    lens, starts = _int32(lengths, None, "lengths"), _int32(query_starts, requests + 1, "query_starts")
    _check(window >= 0, "window must not be negative.")
    _check(max_queries is None or max_queries >= 1, "max_queries must be at least 1.")
    max_queries = max(1, tokens if max_queries is None else min(int(max_queries), tokens))
    scale = d ** -0.5 if scale is None else float(scale)
    given = out is not None
    if given:
        _check(out.shape == q.shape and out.dtype == q.dtype, "out must have the shape and type of q.")
    else:
        out = torch.empty((tokens, heads, d), dtype=q.dtype, device=q.device)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float32, device=q.device) if return_lse else None
    dt = _DT[q.dtype]
    with torch.cuda.device(q.device):
        size = C.c_size_t(0)
        _call("decdec_kv4_attention_workspace", requests, tokens, heads, kv_heads, d, group_size, max_queries, dt, C.byref(size))
        workspace = torch.empty(size.value, dtype=torch.uint8, device=q.device)
        _call("decdec_kv4_attention", *at, *_rows(out, "out"), lse.data_ptr() if return_lse else None, cache.data_ptr(), pages, page_size, *table, lens, starts,
              requests, tokens, heads, kv_heads, d, group_size, max_queries, scale, min(int(window), 0x7fffffff), int(not given), workspace.data_ptr(),
              workspace.numel(), dt, _stream())
    return (out, lse) if return_lse else out
