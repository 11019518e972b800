"""A decoder layer around its products, on the B200: rotary positions, norms and residual, and a paged cache in 8 bits.

  rotary_frequencies, rotary   rotary positions, with the norm of queries and keys before them
  add_norm                     the norms around a block, its gate and its residual in one pass
  paged_cache, cache_append    a cache of keys and values in pages and 8 bits, and what puts new tokens into it
  paged_attention              attention of the newest tokens over such a cache

The reference keeps no cache and leaves these to the compiled graph. Calls, errors and autograd are as in generate.py;
the same calls are the ops torch.ops.xdna.* of these names (without rotary_frequencies and paged_cache).
"""

import math
from typing import NamedTuple

import torch

from . import generate, kernels
from .generate import ERR_INVALID, _account, _ready

SCALINGS = (None, "linear", "ntk", "yarn", "llama3")


def rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, original=None, low=1.0, high=None, device="cuda"):
    """(inv_freq f32 [dim / 2], attention factor) of rotary positions over dim entries of a head.

    The frequencies are base ** (-2 i / dim). For contexts `factor` times as long as the model's: "linear" divides all
    of them by factor; "ntk" raises the base to base * factor ** (dim / (dim - 2)); "yarn" divides those that turn less
    than `low` times in the `original` context, leaves those that turn more than `high` (32) times, and goes evenly from
    one to the other over the entries between, with the attention factor 1 + 0.1 ln(factor); "llama3" does the same with
    `high` 4, evenly in the number of turns, and the attention factor 1. Both results go to rotary and cache_append."""
    if scaling not in SCALINGS:
        raise kernels.XdnaError("rotary_frequencies", ERR_INVALID, f"scaling {scaling!r} (one of {SCALINGS})")
    if dim < 2 or dim % 2 or not base > 1 or not factor >= 1 or not math.isfinite(base * factor) or (scaling == "ntk" and dim < 4):
        raise kernels.XdnaError("rotary_frequencies", ERR_INVALID, f"dim {dim}, base {base}, factor {factor}")
    high = high if high is not None else 32.0 if scaling == "yarn" else 4.0
    if scaling in ("yarn", "llama3") and (original is None or not original > 0 or not 0 < low < high):
        raise kernels.XdnaError("rotary_frequencies", ERR_INVALID, f"original {original}, low {low}, high {high}")
    if scaling == "ntk":
        base = base * factor ** (dim / (dim - 2))
    freq = [base ** (-2 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "yarn":
        def entry(turns):  # where a frequency turns so often in the original context
            return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        first, last = max(math.floor(entry(high)), 0), min(math.ceil(entry(low)), dim - 1)
        way = [min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0) for i in range(dim // 2)]
        freq = [f * (1 - w) + f / factor * w for f, w in zip(freq, way)]
    elif scaling == "llama3":
        turns = [original * f / (2 * math.pi) for f in freq]
        way = [min(max((t - low) / (high - low), 0.0), 1.0) for t in turns]
        freq = [f * w + f / factor * (1 - w) for f, w in zip(freq, way)]
    return (torch.tensor(freq, dtype=torch.float64).float().to(device),
            1 + 0.1 * math.log(factor) if scaling == "yarn" else 1.0)


def rotary(x, positions, inv_freq, factor=1.0, interleaved=False, norm=None, eps=1e-6):
    """x [T, H, D] (f32, bf16 or f16; D a multiple of 8 up to 256; any strides) with each head turned to its token's place.

    positions [T] int32 or int64, inv_freq f32 [R / 2] (rotary_frequencies): of each head's first R entries the pairs
    (p, p + R / 2), or (2 p, 2 p + 1) with interleaved, turn by the angle positions * inv_freq[p], taken in 64 bits, and
    are multiplied with factor; the entries from R on stay. norm: weights [D], or [H, D] where heads differ (queries and
    keys of one projection in one call), of an RMS norm of each head before that. Returns a new [T, H, D], rounded once."""
    t0 = _ready(x)
    out = generate._native.rotary(x, positions, inv_freq, factor, interleaved, norm, eps)
    if out is None:  # autograd records this call
        return torch.ops.xdna.rotary(x, positions, inv_freq, factor, interleaved, norm, eps)
    _account(t0)
    return out


def add_norm(x, y, weight, post=None, gate=None, scale=1.0, eps=1e-6):
    """(x', h): a block's result y added to the residual stream x, and the next block's input. All in f32, per row:

      z = y / sqrt(mean y^2 + eps) * post, or y without post;  x' = x + scale * gate * z;
      h = x' / sqrt(mean x'^2 + eps) * weight

    x, y [..., D] of one shape, each f32, bf16 or f16 (any strides), D up to 16384; weight, post [D]; gate [D] or x's
    shape. x' has x's type, h y's; h is of x' before it is rounded."""
    t0 = _ready(x)
    out = generate._native.add_norm(x, y, weight, post, gate, scale, eps)
    if out is None:  # autograd records this call
        return torch.ops.xdna.add_norm(x, y, weight, post, gate, scale, eps)
    _account(t0)
    return out


class PagedCache(NamedTuple):
    """Codes [pages, Hkv, page, D] (int8 or float8_e4m3fn) and scales f32 [pages, Hkv] of one layer's keys and values:
    key = code * scale. A scale is of one head's part of a page, zero or more; those of cache_append are powers of two."""

    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor


def paged_cache(pages, heads, dim, page=64, dtype=torch.int8, device="cuda"):
    """An empty PagedCache. page: 16, 32, 64 or 128 tokens; dim: 64 or 128; dtype: int8 or float8_e4m3fn."""
    if pages < 0 or heads < 1 or dim not in (64, 128) or page not in (16, 32, 64, 128):
        raise kernels.XdnaError("paged_cache", ERR_INVALID, f"{pages} pages of {page} tokens, {heads} heads of {dim}")
    if dtype not in (torch.int8, torch.float8_e4m3fn):
        raise kernels.XdnaError("paged_cache", ERR_INVALID, f"codes in {dtype} (int8 or float8_e4m3fn)")
    codes = torch.zeros(2, pages, heads, page, dim, dtype=torch.int8, device=device).view(dtype)
    scales = torch.zeros(2, pages, heads, device=device)
    return PagedCache(codes[0], codes[1], scales[0], scales[1])


def cache_append(k, v, k_cache, v_cache, k_scales, v_scales, table, starts, cu_seqlens=None, inv_freq=None, factor=1.0,
                 interleaved=False, k_norm=None, q=None, q_norm=None, eps=1e-6):
    """Puts new keys and values k, v [T, Hkv, D] (bf16 or f16; any strides) into a paged cache (PagedCache's four, in
    place), the keys normed (k_norm) and turned to their places (inv_freq, factor, interleaved: as rotary; none without
    inv_freq) on the way.

    Without cu_seqlens token i is the next one of sequence i (a decode step), with it [N + 1] (int32) tokens
    cu_seqlens[i] .. cu_seqlens[i + 1] - 1 are sequence i's next ones. starts [N] int32: how many tokens of a sequence
    the cache has before the call; below zero, nothing of it is stored. table [N, M] int32: page table[i, j] holds
    sequence i's tokens j * page on; tokens whose entry is no page, and those past M pages, are not stored. No two
    sequences may append to one page. All lengths stay on the GPU.

    A block's (one head's part of a page) scale is the least power of two that holds its largest value in 127 (int8) or
    448 (e4m3) of it. Where it grows with a later token, the older codes are rounded to it; a page whose first slot is
    written starts anew; one that is given an infinity or a NaN reads as NaN until then. Other slots are left alone.

    q [T, Hq, D], any heads in k's type that turn with their tokens (q_norm: their norm): returned as a new tensor, zeros
    where starts is below zero and for tokens of no sequence. Without q the call returns None."""
    t0 = _ready(k)
    args = (k, v, k_cache, v_cache, k_scales, v_scales, table, starts, cu_seqlens, inv_freq, factor, interleaved, k_norm,
            q, q_norm, eps)
    out = generate._native.cache_append(*args)
    if out is None:  # autograd records this call
        return torch.ops.xdna.cache_append(*args)
    _account(t0)
    return None if out is False else out


def paged_attention(q, k_cache, v_cache, k_scales, v_scales, table, lens, scale=None):
    """Attention over a paged cache: softmax(scale q k^T) v of the newest tokens of B sequences.

    q [B, Hq, D], one token each, or [B, T, Hq, D], the last T of each (bf16 or f16, D 64 or 128, Hq a multiple of the
    cache's Hkv; any strides); lens [B] int32: the sequence's tokens in the cache, q's own among them (clamped to what
    table [B, M] int32 can hold). Token t attends to the first lens - T + t + 1; tokens whose table entry is no page do
    not count; a row that sees nothing is zero. scale: 1 / sqrt(D) unless given. T is meant to be small (one, or a few
    proposed tokens). Returns q's shape. The lengths stay on the GPU and the work is shared out by them there."""
    t0 = _ready(q)
    out = generate._native.paged_attention(q, k_cache, v_cache, k_scales, v_scales, table, lens, scale)
    if out is None:  # autograd records this call
        return torch.ops.xdna.paged_attention(q, k_cache, v_cache, k_scales, v_scales, table, lens, scale)
    _account(t0)
    return out
