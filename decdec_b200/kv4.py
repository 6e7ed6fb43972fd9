"""The 4-bit key/value cache of a decoder layer and what stands around it: positions into queries and keys, pages and slots of a
step, new rows into the cache, attention over it.  No counterpart in the reference binding, whose models keep a dense 16-bit cache
(end-to-end/model.py).

A step of a layer, for a batch of requests whose tokens lie one request after another:

    p = kv4.plan(lengths, new_lengths, block_table, free_pages, free_count, page_size, tokens)        # once for all layers
    q, k = kv4.rotary(q, k, p.positions, frequencies, factor=factor)
    kv4.append(cache, k, v, p.slots, group_size)
    y = kv4.attention(q, cache, block_table, p.lengths, p.query_starts, group_size, max_queries=n)

A batch of one with a contiguous cache is a block table that counts up.  Nothing synchronises but the first append, gather or attention on
a stream, which allocates its error word; every call can be captured in a CUDA graph once a call has run eagerly on the device; lengths, tables and
slots are read on the device.  Elements are held as
offset + step * code with 16 codes and one (step, offset) for `group_size` elements of a head; `include/decdec_b200.h` gives the
format.  Tensors: fp16 or bf16, [tokens, heads, head_dim], any strides with neighbouring elements in a head.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _kv4
from .ops import _check


class Plan(NamedTuple):
    positions: torch.Tensor       # int64 [tokens], 0 behind the last new token
    slots: torch.Tensor           # int64 [tokens], -1 behind it
    query_starts: torch.Tensor    # int32 [requests + 1]
    lengths: torch.Tensor         # int32 [requests], the new tokens included
    free_count: torch.Tensor      # int32 [1]
    status: torch.Tensor          # int32 [1]: 0, or why nothing was given (1 pages, 2 table, 4 tokens, 8 a negative count)


def cell_bytes(head_dim: int, group_size: int) -> int:
    """Bytes of 16 tokens of one head."""
    return _kv4.cell_bytes(head_dim, group_size)


def empty_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, group_size: int, device="cuda") -> torch.Tensor:
    """A cache of `pages` pages of `page_size` tokens (a multiple of 16): uint8 [pages, kv_heads, bytes of a page], zeros."""
    _check(page_size > 0 and page_size % 16 == 0, f"page_size must be a multiple of 16, got {page_size}.")
    return torch.zeros((pages, kv_heads, page_size // 16 * cell_bytes(head_dim, group_size)), dtype=torch.uint8, device=device)


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
            hi = min(math.ceil(pair(scaling.get("beta_slow", 1.0))), rotary_dim - 1)
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
    return _kv4.rotary(q, k, positions, frequencies, interleaved, factor, *((None, None) if out is None else out))


# ---- pages and slots of a step ---------------------------------------------------------------------------------

def plan(lengths: torch.Tensor, new_lengths: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
         page_size: int, tokens: int) -> Plan:
    """Pages, slots and positions of the next step from lengths[b] tokens held and new_lengths[b] to come (int32), on the device.

    A request that outgrows its pages takes the last of free_pages[:free_count]; they are entered in `block_table`, which is
    written in place.  `tokens`: entries of positions and slots, at least the sum of new_lengths.  All or nothing: if status is not 0
    no page is given, slots are -1, query_starts 0, lengths and free_count as they were."""
    return Plan(*_kv4.plan(lengths, new_lengths, block_table, free_pages, free_count, page_size, tokens))


# ---- rows into the cache and out of it ---------------------------------------------------------------------------

def append(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, group_size: int) -> None:
    """Writes rows of keys and values [tokens, kv_heads, head_dim] to their slots (page * page_size + place; negative: skipped).
    Slots must differ: of two rows with the same slot any mixture may stay."""
    _kv4.append(cache, k, v, slots, group_size)


def gather(cache: torch.Tensor, slots: torch.Tensor, head_dim: int, group_size: int, dtype: torch.dtype) -> tuple:
    """Dense keys and values [len(slots), kv_heads, head_dim] of slots, in any order; zeros for negative ones."""
    return _kv4.gather(cache, slots, head_dim, group_size, dtype)


# ---- attention ---------------------------------------------------------------------------------------------------

def attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, query_starts: torch.Tensor, group_size: int,
              max_queries: Optional[int] = None, scale: Optional[float] = None, window: int = 0, out: Optional[torch.Tensor] = None,
              return_lse: bool = False):
    """softmax(scale q k^T) v over the cache, causal: request b has the rows query_starts[b]..query_starts[b+1]-1 of q [tokens, heads,
    head_dim], which are its last tokens, and lengths[b] tokens in the cache with them.  Query head h reads key head h * kv_heads // heads.

    window > 0: each row sees the last `window` tokens up to its own.  A row that sees no token gives zeros.  max_queries: the most rows of a
    request, which chooses the kernel; the default, all rows, is meant for one request: a decoding batch without it may run on the kernel for
    prompts, several times slower.  scale: default head_dim ** -0.5.  Rows of no request, before the first or
    behind the last, are left as they are in `out`, zeros where `out` is not given.  return_lse: also the fp32 logarithms [tokens, heads] of the sums of exp(scale q k^T)."""
    out, lse = _kv4.attention(q, cache, block_table, lengths, query_starts, group_size, max_queries, scale, window, out, return_lse)
    return (out, lse) if return_lse else out
