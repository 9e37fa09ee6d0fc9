"""Layout of a key / value cache held in 4 bits, and its plain form (the CPU path, the kernels' oracle).

One uint8 tensor each for keys and values, [pages, kv heads, page_size / 16, 9 * D]: a page of a head is blocks of 16 tokens, a
block 16 rows of D / 2 bytes and behind them 16 x D / 64 pairs (scale, low) of bf16, one pair for each 64 dims of a token's head.
A block is one contiguous copy, codes and pairs together, whatever the page size.

Each 64 dims y of a token's head are coded by themselves: low = min y, scale = bf16((max y - low) / 15) (below 2^-126: 0), code =
min(15, round((y - low) / scale)), ties to even; 0 where the scale is 0. A code c stands for c * scale + low. Four bits and, for the
pair, half a bit a value. Keys are coded as rotated and rounded to bf16, so that low is exact. A group that holds a NaN or an
infinity (or spans more than fp32 holds) reads back as NaN.

What attention makes of held values on the GPU: decoding sequences take codes, scales and low ends as they are; a query's dims are exact down to
2^-28 of its head's largest, sums are fp32, and a probability times a value's scale is rounded to fp16: 2^-11, or 2^-31 of the largest scale among
the head's values (2^-60 at least) where that is more. Prompt portions see held values rounded to bf16 (2^-8, as `kv_cache_rows` gives
them) and round probabilities to bf16, as over a bf16 cache. The plain form keeps fp32.

A row's 32-bit unit u holds eight dims, the first in the lowest four bits: those from 64 (u % (D / 64)) + 8 (u // (D / 64)) on. So
16 bytes hold as many dims of each group, which is what a lane of the attention kernel takes (csrc/attn/kv4_attention.cu).
"""
from __future__ import annotations

import functools

import torch

BLOCK = 16
MOST_PAGE = 512          # tokens; the attention kernel divides by it with one multiplication
HEAD_DIMS = (64, 128)


def cache_shape(num_pages: int, num_kv_heads: int, head_dim: int, page_size: int):
    if head_dim not in HEAD_DIMS or not BLOCK <= page_size <= MOST_PAGE or page_size % BLOCK:
        raise ValueError(f"a 4-bit cache holds heads of 64 or 128 in pages of a multiple of {BLOCK} tokens up to {MOST_PAGE}: got heads "
                         f"of {head_dim}, pages of {page_size}")
    return (num_pages, num_kv_heads, page_size // BLOCK, 9 * head_dim)


@functools.lru_cache(maxsize=256)
def sizes(shape):
    """(pages, kv heads, page_size, head_dim) of a shape, or None if it is no 4-bit cache's."""
    if len(shape) != 4 or shape[3] % 9 or shape[3] // 9 not in HEAD_DIMS or not 1 <= shape[2] <= MOST_PAGE // BLOCK:
        return None
    return shape[0], shape[1], shape[2] * BLOCK, shape[3] // 9


def geometry(cache: torch.Tensor):
    """(pages, kv heads, page_size, head_dim) of a 4-bit cache."""
    geo = sizes(cache.shape)
    if geo is None or cache.dtype != torch.uint8 or not cache.is_contiguous():
        raise ValueError(f"not a 4-bit cache: {cache.dtype} {tuple(cache.shape)}")
    return geo


def held(cache) -> bool:
    """Whether this is a 4-bit cache."""
    return cache is not None and cache.dtype == torch.uint8


@functools.lru_cache(maxsize=None)
def _order(dim: int):
    """Dim of each code of a row, in storage order, and where each dim's code is."""
    g = dim // 64
    dims = torch.tensor([64 * (u % g) + 8 * (u // g) + e for u in range(dim // 8) for e in range(8)])
    return dims, torch.argsort(dims)


def encode(x: torch.Tensor):
    """Rows [..., D] (rounded to bf16 first) -> (codes [..., D / 2], pairs [..., D / 16]), bytes."""
    d = x.shape[-1]
    y = x.to(torch.bfloat16).float().unflatten(-1, (d // 64, 64))
    low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    scale = ((high - low) / 15).to(torch.bfloat16).float()
    scale = torch.where(scale < 2.0 ** -126, 0.0, torch.where(torch.isfinite(scale), scale, torch.nan))
    codes = torch.where(scale > 0, torch.round((y - low) / scale), 0.0).clamp(0, 15).to(torch.uint8).flatten(-2)
    codes = codes[..., _order(d)[0].to(x.device)].unflatten(-1, (d // 2, 2))
    pairs = torch.cat((scale, low), -1).to(torch.bfloat16).view(torch.uint8).flatten(-2)
    return codes[..., 0] | (codes[..., 1] << 4), pairs


def decode(codes: torch.Tensor, pairs: torch.Tensor):
    """The inverse: fp32 values."""
    d = 2 * codes.shape[-1]
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., _order(d)[1].to(codes.device)]
    scale, low = pairs.contiguous().view(torch.bfloat16).float().unflatten(-1, (d // 64, 2)).unbind(-1)
    return (c.float().unflatten(-1, (d // 64, 64)) * scale.unsqueeze(-1) + low.unsqueeze(-1)).flatten(-2)


def _views(cache: torch.Tensor):
    """Codes [pages, heads, blocks, 16, D / 2] and pairs [pages, heads, blocks, 16, D / 16] of a cache, as views."""
    d = geometry(cache)[3]
    return cache[..., : 8 * d].unflatten(-1, (BLOCK, d // 2)), cache[..., 8 * d:].unflatten(-1, (BLOCK, d // 16))


def _places(cache, slots):
    _, _, page, _ = geometry(cache)
    slots = slots.long()
    at = slots % page
    return torch.div(slots, page, rounding_mode="floor"), torch.div(at, BLOCK, rounding_mode="floor"), at % BLOCK


def write_rows(cache: torch.Tensor, slots: torch.Tensor, x: torch.Tensor):
    """x [T, heads, D] into `slots` (negative ones, and ones behind the last page: left out)."""
    pages, _, page, _ = geometry(cache)
    keep = (slots >= 0) & (slots < pages * page)
    for view, rows in zip(_views(cache), encode(x[keep])):
        p, b, r = _places(cache, slots[keep])
        view[p, :, b, r] = rows


def read_rows(cache: torch.Tensor, slots: torch.Tensor):
    """What the cache holds at `slots`, [T, heads, D] fp32 (zeros for slots that write_rows leaves out)."""
    pages, heads, page, d = geometry(cache)
    out = torch.zeros(slots.shape[0], heads, d, dtype=torch.float32, device=cache.device)
    keep = (slots >= 0) & (slots < pages * page)
    p, b, r = _places(cache, slots[keep])
    codes, pairs = _views(cache)
    out[keep] = decode(codes[p, :, b, r], pairs[p, :, b, r])
    return out
