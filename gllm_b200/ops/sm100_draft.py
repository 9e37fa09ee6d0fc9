"""Python front-ends of the kernels for drafted tokens (csrc/draft): plan, attention, verification, rows that move. Definitions and checks:
`ops.draft`. Each function validates, allocates its output and its scratch and launches on the current stream; no fallback.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from gllm_b200.ops import draft, lib as _lib
from gllm_b200.ops.lib import check, on_this_device, stream_ptr
from gllm_b200.ops.sm100 import NUM_SMS, _BF16, _count

_MOST_CACHES = 256       # of one launch (csrc/draft/tree_ops.cu)


def plan(parents: torch.Tensor, inp, page_size: int):
    """(seen int64 [T], positions int32 [T], slots int32 [T]) of the nodes; 0, 0 and -1 in rows behind the last sequence."""
    b = draft.check_plan(parents, inp, page_size)
    t = parents.shape[0]
    seen = parents.new_empty(t, dtype=torch.int64)
    positions, slots = parents.new_empty(t), parents.new_empty(t)
    if t == 0:
        return seen, positions, slots
    table = inp.block_table
    on_this_device(parents, inp.query_start_loc, inp.seq_lens, table)
    check(_lib.load().gllm_draft_plan(parents.data_ptr(), inp.query_start_loc.data_ptr(), inp.seq_lens.data_ptr(), table.data_ptr(),
                                      table.stride(0), table.shape[1], b, t, page_size, seen.data_ptr(), positions.data_ptr(),
                                      slots.data_ptr(), stream_ptr()), "draft_plan")
    _count()
    return seen, positions, slots


@functools.lru_cache(maxsize=None)
def _attention_scratch(head_dim: int) -> int:
    return _lib.load().gllm_draft_attention_scratch(head_dim, NUM_SMS)


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, inp, seen: torch.Tensor, scale: float, num_q_heads: int,
              head_dim: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [T, Hq * D] bf16 (any row stride) -> [T, Hq * D]; rows behind the last sequence are left as they are."""
    b = draft.check_attention(q, k_cache, v_cache, inp, seen, scale, num_q_heads, head_dim, out)
    pages, hkv, _, page_size, w = k_cache.shape
    t = q.shape[0]
    if q.dtype != _BF16 or w != 64 or head_dim not in draft.HEAD_DIMS or page_size not in draft.PAGE_SIZES:
        raise ValueError(f"drafted tokens are attended in bf16, heads of 64 or 128, pages of 8 to 128 tokens (a power of two): got {q.dtype}, "
                         f"heads of {head_dim}, pages of {page_size}")
    q_ts = q.stride(0) if t > 1 else num_q_heads * head_dim      # the stride of a dimension of one may be anything
    if t and (q.data_ptr() | 2 * q_ts | k_cache.data_ptr() | v_cache.data_ptr()) % 16:
        raise ValueError("queries and caches of drafted tokens must lie on 16-byte boundaries")
    if out is None:
        out = q.new_empty((t, num_q_heads * head_dim))
    if t == 0 or b == 0:
        return out
    table = inp.block_table
    on_this_device(q, k_cache, v_cache, table, inp.seq_lens, inp.query_start_loc, seen, out)
    size = _attention_scratch(head_dim)
    scratch = k_cache.new_empty(size, dtype=torch.uint8)       # of this call: captured graphs and streams share none
    check(_lib.load().gllm_draft_attention(q.data_ptr(), q_ts, out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), pages,
                                           table.data_ptr(), table.stride(0), table.shape[1], inp.seq_lens.data_ptr(),
                                           inp.query_start_loc.data_ptr(), seen.data_ptr(), b, t, inp.max_q_len, num_q_heads, hkv,
                                           head_dim, page_size, scale, NUM_SMS, scratch.data_ptr(), size, stream_ptr()), "draft_attention")
    _count(2)
    return out


def _verify_parts(b: int) -> int:
    return 1


def verify(tokens: torch.Tensor, parents: torch.Tensor, inp, target: torch.Tensor, draft_probs: Optional[torch.Tensor] = None,
           uniform: Optional[torch.Tensor] = None):
    """(tokens int32 [T], path int32 [T], count int32 [sequences]); -1 behind a sequence's last and in rows behind the last sequence."""
    b = draft.check_verify(tokens, parents, inp, target, draft_probs, uniform)
    t = tokens.shape[0]
    said, path, count = tokens.new_empty(t), tokens.new_empty(t), tokens.new_empty(b)
    if b == 0 and t == 0:
        return said, path, count
    on_this_device(tokens, parents, inp.query_start_loc, target, draft_probs, uniform)
    by_token = not target.is_floating_point()
    check(_lib.load().gllm_draft_verify(
        tokens.data_ptr(), parents.data_ptr(), inp.query_start_loc.data_ptr(), target.data_ptr() if by_token else None,
        None if by_token else target.data_ptr(), 0 if by_token else target.stride(0), None if draft_probs is None else draft_probs.data_ptr(),
        0 if draft_probs is None else draft_probs.stride(0), None if uniform is None else uniform.data_ptr(),
        0 if by_token else target.shape[1], b, t, said.data_ptr(), path.data_ptr(), count.data_ptr(),
        1 if by_token else _verify_parts(b), stream_ptr()), "draft_verify")
    _count()
    return said, path, count


def keep(k_caches, v_caches, inp, path: torch.Tensor, count: torch.Tensor) -> None:
    """Rows of the nodes in `path` move up behind their contexts, in every cache; a launch for each shape of cache."""
    b = draft.check_keep(inp, path, count)
    caches = draft.cache_list(k_caches, v_caches)
    t = path.shape[0]
    if t == 0 or b == 0:
        return
    table = inp.block_table
    on_this_device(path, count, table, inp.seq_lens, inp.query_start_loc, *caches)
    shapes = {}
    for c in caches:
        shapes.setdefault((c.shape, c.element_size()), []).append(c.data_ptr())
    for (shape, size), at in shapes.items():
        pages, heads, slabs, page_size, w = shape
        for i in range(0, len(at), _MOST_CACHES):
            some = at[i:i + _MOST_CACHES]
            check(_lib.load().gllm_draft_keep((ctypes.c_void_p * len(some))(*some), len(some), pages, heads * slabs, page_size,
                                              w * size // 16, path.data_ptr(), count.data_ptr(), inp.query_start_loc.data_ptr(),
                                              inp.seq_lens.data_ptr(), table.data_ptr(), table.stride(0), table.shape[1], b, t,
                                              stream_ptr()), "draft_keep")
            _count()
