"""Python front-ends of the kernels for drafted tokens (csrc/draft): plan, attention, verification, rows that move. Definitions and checks:
`ops.draft`. Each function validates, allocates its output and its scratch and launches on the current stream; no fallback.
"""
from __future__ import annotations

import array
import functools
from typing import Optional

import torch

from gllm_b200.ops import draft, lib as _lib
from gllm_b200.ops.lib import check, on_this_device, stream_ptr
from gllm_b200.ops.sm100 import NUM_SMS, _BF16, _count

_MOST_CACHES = 256       # of one launch (csrc/draft/tree_ops.cu)


def plan(parents: torch.Tensor, inp, page_size: int):
    """(seen int64 [T], positions int32 [T], slots int32 [T]) of the nodes; 0, 0 and -1 in rows behind the last sequence."""
    b, start, lens, table = draft.check_plan(parents, inp, page_size)
    t = parents.shape[0]
    seen = parents.new_empty(t, dtype=torch.int64)
    positions, slots = torch.empty_like(parents), torch.empty_like(parents)
    if t == 0:
        return seen, positions, slots
    on_this_device(parents, start, lens, table)
    check(_lib.load().gllm_draft_plan(parents.data_ptr(), start.data_ptr(), lens.data_ptr(), table.data_ptr(), table.stride(0),
                                      table.shape[1], b, t, page_size, seen.data_ptr(), positions.data_ptr(), slots.data_ptr(),
                                      stream_ptr()), "draft_plan")
    _count()
    return seen, positions, slots


@functools.lru_cache(maxsize=None)
def _attention_scratch(head_dim: int, max_rows: int) -> int:
    return _lib.load().gllm_draft_attention_scratch(head_dim, max_rows, NUM_SMS)


def _whole_units(seqs: int, kv_heads: int, group: int, nodes: int, max_len: int) -> bool:
    """Whether no unit of the attention kernel (a sequence's kv head and block of rows) is cut: nothing is joined then, in a second launch of some
    5 us, but the SM with the most has up to a unit more than its share. Cut and whole, us: 8 units of 1, 4, 12 and 47
    tiles (32 / 8 heads of 128, 8 nodes) 11.5 / 10.3, 14.1 / 12.4, 15.7 / 16.5, 19.0 / 39.4; 128 of 4 and 47 17.3 / 14.4, 57.4 / 66.3; 1024 of
    4 and 12 53.4 / 47.5, 111 / 108. The longest length is all that is known of them, and the others may be short, so longer units are cut
    however many there are: 18 sequences, all of 16 tiles 39.0 / 32.9, one of 16 beside 17 of one 18.3 / 22.6; all of 32 60.6 / 54.4, one 22.1 /
    34.9; 37 sequences, all of 32 101.6 / 100.4, one of 32 24.7 / 35.9, one of 470 116 / 394. Results are right either way, whatever the lengths are
    when a captured call is replayed."""
    tiles = (max_len + 127) // 128
    if tiles <= 8 or tiles > 16:
        return tiles <= 8
    rows = nodes * group
    block = (32 if rows <= 32 else 64 if rows <= 64 else 128 if rows <= 128 else 256) // group
    units = seqs * kv_heads * -(-nodes // max(block, 1))
    return (-(-units // NUM_SMS) - units / NUM_SMS) * tiles <= 2.5


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, inp, seen: torch.Tensor, scale: float, num_q_heads: int,
              head_dim: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [T, Hq * D] bf16 (any row stride) -> [T, Hq * D]; rows behind the last sequence are not written: in a result that is made here they hold
    whatever the memory held."""
    b, start, lens, table = draft.check_attention(q, k_cache, v_cache, inp, seen, scale, num_q_heads, head_dim, out)
    pages, hkv, _, page_size, w = k_cache.shape
    t, q_ts = q.shape[0], q.stride(0)
    if q.dtype is not _BF16 or w != 64 or head_dim not in draft.HEAD_DIMS or page_size not in draft.PAGE_SIZES or \
            num_q_heads // hkv > draft.MOST_GROUP:
        raise ValueError(f"drafted tokens are attended in bf16, heads of 64 or 128, at most {draft.MOST_GROUP} query heads a kv head, pages of 8 "
                         f"to 128 tokens (a power of two): got {q.dtype}, {num_q_heads} / {hkv} heads of {head_dim}, pages of {page_size}")
    if t <= 1:
        q_ts = num_q_heads * head_dim                          # the stride of a dimension of one may be anything
    q_at, k_at, v_at = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    if out is None:
        out = q.new_empty((t, num_q_heads * head_dim))
    out_at = out.data_ptr()
    if t and (q_at | 2 * q_ts | k_at | v_at | out_at) % 16:
        raise ValueError("queries, caches and results of drafted tokens must lie on 16-byte boundaries")
    if t == 0 or b == 0:
        return out
    on_this_device(q, k_cache, v_cache, table, lens, start, seen, out)
    most = inp.max_q_len
    whole = _whole_units(b, hkv, num_q_heads // hkv, most, inp.max_seq_len)
    scratch_at, size = None, 0
    if not whole:
        size = _attention_scratch(head_dim, min(most, draft.MOST_NODES) * (num_q_heads // hkv))
        scratch = k_cache.new_empty(size, dtype=torch.uint8)   # of this call: captured graphs and streams share none
        scratch_at = scratch.data_ptr()
    check(_lib.load().gllm_draft_attention(q_at, q_ts, out_at, k_at, v_at, pages, table.data_ptr(), table.stride(0), table.shape[1],
                                           lens.data_ptr(), start.data_ptr(), seen.data_ptr(), b, t, most, whole, num_q_heads, hkv,
                                           head_dim, page_size, scale, NUM_SMS, scratch_at, size, stream_ptr()), "draft_attention")
    _count(1 if whole else 2)
    return out


def _verify_parts(b: int, vocab: int) -> int:
    """CTAs of a cluster that share a sequence: as many as leave all clusters resident, two CTAs an SM. One sequence, 151,936 tokens, 1 to 16
    CTAs: 24, 16.5, 12.3, 10.0, 9.2 us; 64 of 128,257: 36, 20.5, 18.0, 24, 40; 256 of 151,936: 60, 67, 78, 104. Sixteen are for few sequences and
    long rows (8 and 16 CTAs: 4 chains of 32,000 8.0 / 8.5, of 100,352 9.8 / 9.0, of 151,936 10.8 / 9.5; 8 chains 11.0 / 11.0, 8 trees of 32
    nodes 19.7 / 15.8; 8 chains of 100,352 10.0 / 10.3; 12 of 151,936 11.5 / 11.6)."""
    if vocab > 1 << 16 and b <= (8 if vocab > 1 << 17 else 4):
        return 16
    return 8 if b <= 37 else 4 if b <= 74 else 2 if b <= 148 else 1


def verify(tokens: torch.Tensor, parents: torch.Tensor, inp, target: torch.Tensor, draft_probs: Optional[torch.Tensor] = None,
           uniform: Optional[torch.Tensor] = None):
    """(tokens int32 [T], path int32 [T], count int32 [sequences]); -1 behind a sequence's last and in rows behind the last sequence."""
    b, start, by_token = draft.check_verify(tokens, parents, inp, target, draft_probs, uniform)
    t = tokens.shape[0]
    said, path, count = tokens.new_empty(t), tokens.new_empty(t), tokens.new_empty(b)
    if b == 0 and t == 0:
        return said, path, count
    on_this_device(tokens, parents, start, target, draft_probs, uniform)
    chosen_at = target_at = draft_at = uniform_at = None
    ld_target = ld_draft = vocab = 0
    if by_token:
        chosen_at = target.data_ptr()
    else:
        target_at, ld_target, vocab, uniform_at = target.data_ptr(), target.stride(0), target.shape[1], uniform.data_ptr()
        if draft_probs is not None:
            draft_at, ld_draft = draft_probs.data_ptr(), draft_probs.stride(0)
    check(_lib.load().gllm_draft_verify(tokens.data_ptr(), parents.data_ptr(), start.data_ptr(), chosen_at, target_at, ld_target, draft_at,
                                        ld_draft, uniform_at, vocab, b, t, said.data_ptr(), path.data_ptr(), count.data_ptr(),
                                        1 if by_token else _verify_parts(b, vocab), stream_ptr()), "draft_verify")
    _count()
    return said, path, count


def keep(k_caches, v_caches, inp, path: torch.Tensor, count: torch.Tensor) -> None:
    """Rows of the nodes in `path` move up behind their contexts, in every cache; a launch for each shape of cache."""
    b, start, lens, table = draft.check_keep(inp, path, count)
    groups = draft.cache_groups(k_caches, v_caches)
    t = path.shape[0]
    if t == 0 or b == 0:
        return
    on_this_device(path, count, table, lens, start)
    here = path.get_device()
    for (pages, heads, slabs, page_size, w), size, at, caches in groups:
        if list(map(torch.Tensor.get_device, caches)).count(here) != len(caches):
            on_this_device(*caches)
        for i in range(0, len(at), _MOST_CACHES):
            some = at[i:i + _MOST_CACHES]
            ptrs = array.array("Q", some)
            check(_lib.load().gllm_draft_keep(ptrs.buffer_info()[0], len(some), pages, heads * slabs, page_size, w * size // 16,
                                              path.data_ptr(), count.data_ptr(), start.data_ptr(), lens.data_ptr(), table.data_ptr(),
                                              table.stride(0), table.shape[1], b, t, stream_ptr()), "draft_keep")
            _count()
