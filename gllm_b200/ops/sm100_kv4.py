"""Python front-ends of the 4-bit cache kernels (csrc/elemwise/rope_kv4.cu, csrc/attn/kv4_attention.cu): rotary write, attention, rows
read back. Layout: `ops.kv4`. Each function validates, allocates its output and its scratch and launches on the current stream; no fallback.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from gllm_b200.ops import kv4, lib as _lib
from gllm_b200.ops.lib import check, on_this_device, stream_ptr
from gllm_b200.ops.sm100 import NUM_SMS, _BF16, _count

_DECODE_CTAS = NUM_SMS               # one an SM
EXPAND_BYTES = 1 << 30               # bf16 keys and values that prompts have at a time (one sequence at least)


def _pair(k_cache, v_cache):
    """(pages, kv heads, page_size, head_dim) of a layer's caches."""
    shape = k_cache.shape
    geo = kv4.sizes(shape)
    if geo is not None and k_cache.dtype is v_cache.dtype is torch.uint8 and v_cache.shape == shape and k_cache.is_contiguous() and \
            v_cache.is_contiguous():
        return geo
    geo = kv4.geometry(k_cache)                               # raises for what is no cache
    if kv4.geometry(v_cache) != geo:
        raise ValueError(f"4-bit caches of unequal shape: {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    return geo


def _index(t: torch.Tensor, what: str, dims: int = 1):
    assert t.dtype == torch.int32 and t.dim() == dims and (t.stride(-1) == 1 or t.shape[-1] < 2), f"{what}: int32, contiguous rows"


def _refuse_write(q, k, v, positions, cos_sin, rot, neox, q_norm_w, k_norm_w, heads, dim, slots, mrope):
    """Raises for arguments that `rope_kv_write` does not take (the common ones do not come here)."""
    t, hq, d = q.shape
    assert q.dtype == k.dtype == v.dtype == _BF16 and q.stride(2) == k.stride(2) == v.stride(2) == 1
    assert d == dim and k.shape == v.shape == (t, heads, d), (q.shape, k.shape, v.shape, heads, dim)
    _index(slots, "slots")
    assert slots.shape[0] >= t
    if rot < 0 or rot > d or rot % (16 if neox else 8):
        raise ValueError(f"a 4-bit cache takes rotations of a multiple of 16 dims (of 8 in neighbouring pairs): got {rot} of {d}")
    if rot:
        assert cos_sin.dtype == torch.float32 and cos_sin.is_contiguous() and cos_sin.shape[1] == rot, (cos_sin.shape, rot)
    for w in (q_norm_w, k_norm_w):
        assert w is None or (w.dtype == _BF16 and w.shape == (d,) and w.is_contiguous())
    _index(positions, "positions", 2 if mrope else 1)
    assert positions.shape[-1] >= t and (not mrope or positions.shape[0] >= 3), positions.shape
    rows = [x for x in (q, k, v) if x.numel()]
    if any(x.data_ptr() % 16 or any(n > 1 and s % 8 for n, s in zip(x.shape[:2], x.stride())) for x in rows) or \
            any(w is not None and w.data_ptr() % 16 for w in (q_norm_w, k_norm_w)):
        raise ValueError("rows and norm weights written to a 4-bit cache must lie on 16-byte boundaries")


def rope_kv_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, cos_sin: Optional[torch.Tensor],
                  rot_dim: int, neox: bool, q_norm_w: Optional[torch.Tensor], k_norm_w: Optional[torch.Tensor], eps: float,
                  k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, mrope_section=None):
    """`sm100.rope_kv_write` on 4-bit caches: q [T, Hq, D] is normed and rotated in place; k and v [T, Hkv, D] are read only. Rows (all three
    may be strided views) lie on 16-byte boundaries; rot_dim is a multiple of 16, of 8 for neighbouring pairs."""
    pages, heads, page_size, dim = _pair(k_cache, v_cache)
    if v is None or slots is None:
        raise ValueError("a 4-bit cache is written with keys, values and their slots")
    t, hq, d = q.shape
    rot = rot_dim if cos_sin is not None else 0
    mrope = False
    if positions.dim() == 2:
        mrope = mrope_section is not None
        if not mrope:
            positions = positions[0]
    (qt, qh, qd), (kt, kh, kd), (vt, vh, vd) = q.stride(), k.stride(), v.stride()
    if t == 1:                                                # the stride of a dimension of one may be anything
        qt = kt = vt = d
    if hq == 1:
        qh = d
    if heads == 1:
        kh = vh = d
    q_at, k_at, v_at = q.data_ptr(), k.data_ptr(), v.data_ptr()
    ends = q_at | k_at | v_at | 2 * (qt | qh | kt | kh | vt | vh)
    qw_at = kw_at = None
    common = not mrope and d == dim and qd == kd == vd == 1 and rot % 16 == 0 and 0 <= rot <= d
    if q_norm_w is not None:
        qw_at = q_norm_w.data_ptr()
        ends |= qw_at
        common = common and q_norm_w.dtype is _BF16 and q_norm_w.numel() == d and q_norm_w.is_contiguous()
    if k_norm_w is not None:
        kw_at = k_norm_w.data_ptr()
        ends |= kw_at
        common = common and k_norm_w.dtype is _BF16 and k_norm_w.numel() == d and k_norm_w.is_contiguous()
    if not (common and ends % 16 == 0 and q.dtype is k.dtype is v.dtype is _BF16 and k.shape == v.shape == (t, heads, d) and
            slots.dtype is positions.dtype is torch.int32 and slots.dim() == positions.dim() == 1 and slots.numel() >= t and
            positions.numel() >= t and slots.is_contiguous() and positions.is_contiguous() and
            (rot == 0 or (cos_sin.dtype is torch.float32 and cos_sin.shape[1] == rot and cos_sin.is_contiguous()))):
        _refuse_write(q, k, v, positions, cos_sin, rot, neox, q_norm_w, k_norm_w, heads, dim, slots, mrope)
    if t == 0:
        return
    on_this_device(q, k, v, positions, slots, k_cache, v_cache, cos_sin, q_norm_w, k_norm_w)
    sec0 = sec1 = pos_stride = 0
    if mrope:
        if len(mrope_section) > 3 and mrope_section[3]:       # interleaved; otherwise chunks (see sm100.rope_kv_write)
            sec0, sec1 = -int(mrope_section[1]), int(mrope_section[2])
        else:
            sec0, sec1 = int(mrope_section[0]), int(mrope_section[1])
        pos_stride = positions.stride(0)
    check(_lib.load().gllm_rope_kv4_write(
        q_at, qt, qh, hq, k_at, kt, kh, heads, v_at, vt, vh, qw_at, kw_at, cos_sin.data_ptr() if rot else None, d, rot,
        neox, t, positions.data_ptr(), slots.data_ptr(), eps, k_cache.data_ptr(), v_cache.data_ptr(), pages, sec0, sec1, page_size,
        pos_stride, stream_ptr()), "rope_kv4_write")
    _count()


def kv_cache_rows(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor):
    """(keys, values) [T, Hkv, D] bf16 that 4-bit caches hold at `slots`; zeros for slots outside of the cache."""
    pages, heads, page_size, d = _pair(k_cache, v_cache)
    _index(slots, "slots")
    on_this_device(k_cache, v_cache, slots)
    t = slots.shape[0]
    k = k_cache.new_empty((t, heads, d), dtype=_BF16)
    v = torch.empty_like(k)
    if t:
        check(_lib.load().gllm_kv4_rows(k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), t, heads,
                                        d, page_size, pages, stream_ptr()), "kv4_rows")
        _count()
    return k, v


@functools.lru_cache(maxsize=None)
def _decode_scratch(d: int) -> int:
    return _lib.load().gllm_kv4_decode_scratch(d, _DECODE_CTAS)


def scratch_bytes(kv_heads: int, d: int, max_len: int, max_seqs: int = 256) -> int:
    """The most that one step's `paged_attention` allocates beside its result: expanded tiles of prompts and their table, parts of decoding
    sequences."""
    table = 4 * max_seqs * ((max_len + 63) // 64)
    return max(EXPAND_BYTES, 4 * kv_heads * d * (max_len + 63)) + table + _DECODE_CTAS * (2 * 16 * (d + 2) * 4 + 16) + (1 << 20)


def expand_rounds(lens, token_bytes: int, limit: int):
    """(first, end, tiles of 64 tokens) of consecutive sequences whose expanded keys and values stay below `limit` bytes together, one
    sequence at least. lens: their lengths, on the host."""
    rounds, first, tiles = [], 0, 0
    for s, n in enumerate(lens):
        more = (n + 63) // 64
        if s > first and (tiles + more) * 64 * token_bytes > limit:
            rounds.append((first, s, tiles))
            first, tiles = s, 0
        tiles += more
    if len(lens) > first:
        rounds.append((first, len(lens), tiles))
    return rounds


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    query_start_loc: torch.Tensor, scale: float, num_q_heads: int, head_dim: int, num_decode_seqs: int,
                    num_seqs: int, max_q_len: int, max_seq_len: int, out: Optional[torch.Tensor] = None, host_lens=None):
    """`sm100.paged_attention` on 4-bit caches. Decoding sequences read the codes (csrc/attn/kv4_attention.cu). Prompt portions have their
    sequences' keys and values expanded to bf16 first, EXPAND_BYTES of them at a time, and take the tcgen05 prefill kernel.
    host_lens: the lengths [num_seqs] on the host, no shorter than those on the device; without them every prompt is given room for
    max_seq_len, and while a graph is captured for all that its row of the table holds."""
    pages, hkv, page_size, d = _pair(k_cache, v_cache)
    (t, width), (q_ts, one), hq = q.shape, q.stride(), num_q_heads
    assert q.dtype is _BF16 and width >= hq * d and one == 1 and d == head_dim and hq % hkv == 0
    _index(block_table, "block_table", 2)
    _index(seq_lens, "seq_lens")
    assert block_table.shape[0] >= num_seqs and seq_lens.shape[0] >= num_seqs and t >= num_decode_seqs and 0 <= num_decode_seqs <= num_seqs
    prompts = num_seqs - num_decode_seqs if max_q_len > 0 else 0
    if prompts:
        _index(query_start_loc, "query_start_loc")
        assert query_start_loc.shape[0] > num_seqs and (host_lens is None or len(host_lens) >= num_seqs), (query_start_loc.shape, num_seqs)
    q_at = q.data_ptr()
    if t == 1:                                                # the stride of a dimension of one may be anything
        q_ts = hq * d
    if (q_at | 2 * q_ts) % 16 and t:
        raise ValueError("queries over a 4-bit cache must lie on 16-byte boundaries")
    if out is None:
        out = q.new_empty((t, hq * d))
    else:
        assert out.dtype == _BF16 and out.shape == (t, hq * d) and out.is_contiguous()
    on_this_device(q, out, k_cache, v_cache, block_table, seq_lens, query_start_loc if prompts else None)
    L, st = _lib.load(), stream_ptr()
    pitch, width = block_table.stride(0), block_table.shape[1]
    k_at, v_at, out_at, table_at, lens_at = k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr()
    if num_decode_seqs > 0:
        size = _decode_scratch(d)
        scratch = k_cache.new_empty(size)                     # of this call: captured graphs and streams share none
        check(L.gllm_kv4_decode(q_at, q_ts, out_at, k_at, v_at, pages, table_at, pitch, width, lens_at, num_decode_seqs, hq, hkv, d, page_size,
                                scale, _DECODE_CTAS, scratch.data_ptr(), size, st), "kv4_decode")
        _count(2)
    if prompts:
        if torch.cuda.is_current_stream_capturing():          # replayed at other lengths
            lens = [width * page_size] * prompts
        else:
            lens = [max_seq_len] * prompts if host_lens is None else host_lens[num_decode_seqs:num_seqs]
            lens = lens.tolist() if hasattr(lens, "tolist") else list(lens)
        start_at = query_start_loc.data_ptr()
        # (first sequence, sequences, the longest's tokens, tiles), a round each
        rounds = [(a, b - a, max(lens[a:b]), tiles) for a, b, tiles in expand_rounds(lens, 4 * hkv * d, EXPAND_BYTES) if tiles]
        # the tiles' table, keys, values, in one buffer for all rounds, which follow one another. The table comes first: a sequence that is
        # longer than its room (not what the caller said) has entries read behind it, which lie in the keys, and tiles that do not exist,
        # which are read as zeros
        tile = hkv * d * 128
        heads = [(4 * n * ((longest + 63) // 64) + 255) // 256 * 256 for _, n, longest, _ in rounds]
        room = k_cache.new_empty(max((head + 2 * r[3] * tile for head, r in zip(heads, rounds)), default=0))
        t_at = room.data_ptr()
        for head, (first, n, longest, tiles) in zip(heads, rounds):
            a, max_tiles = num_decode_seqs + first, (longest + 63) // 64
            kt_at = t_at + head
            vt_at = kt_at + tiles * tile
            check(L.gllm_kv4_expand(k_at, v_at, table_at + 4 * a * pitch, pitch, width, lens_at + 4 * a, n, hkv, d, page_size, pages, tiles,
                                    kt_at, vt_at, t_at, max_tiles, longest, st), "kv4_expand")
            check(L.gllm_attn_prefill_tc_tiles(q_at, q_ts, out_at, kt_at, vt_at, tiles, t_at, max_tiles,
                                               lens_at + 4 * a, start_at + 4 * a, t, n, max_q_len, hq, hkv, d, scale, st),
                  "attn_prefill_tc_tiles")
            _count(2)
    return out
