"""Decoding with drafted tokens: what its operators are, their checks, and their plain form (the CPU path, the kernels' oracle).

A step drafts a tree of tokens for every sequence and lets the model look at all of them at once. A sequence's nodes are its rows
[query_start_loc[s], query_start_loc[s + 1]) of the batch, at most 64. Node 0 is the token that stands already, as in a step without
drafts; a parent is a node's index within its sequence and comes before it, anything else counts as none (such a node sees the context and
itself, and is never taken). `seq_lens` counts the nodes: ctx = seq_len - nodes tokens are in the cache, node i lies at cache position
ctx + i while the step runs; what would lie behind the last entry of `block_table` has no place (slot -1) and is seen by nobody. A
sequence without rows takes no part; rows behind the last sequence belong to none.

  plan     who sees whom, one 64-bit word a node (bit j: node j), the nodes' rotary positions (ctx + depth) and cache slots
  attend   softmax over the context and over the nodes whose bits are set; a row that sees nothing is zero
  verify   which nodes the target model takes, one path from node 0 on, and the token behind the last of them
  keep     keys and values of the nodes that were taken move up behind the context; the others' rows are free

A step: draft_plan, then in each layer rope_kv_write at the plan's positions and slots and draft_attention, then draft_verify on the nodes'
logits or probabilities, then draft_keep over all layers; the sequences are count tokens longer than their contexts then, and the last of
`tokens` is the next step's node 0.

Verification by tokens: the target's token at every node is known (argmax, or drawn by the sampler with all of its filters); a child that
is that token is taken. By probabilities: node 0's children are tried in order, then those of the one that is taken. With target row p and draft
row q of the node, M_0 = 1, S_0 = 0, child k, token x, is taken where

  u M_k q(x) < max(p(x) - S_k q(x), 0)         otherwise S_k+1 = S_k + M_k,  M_k+1 = sum_y max(p(y) - S_k+1 q(y), 0)

which is the rule for drafts that were drawn independently from q: behind a token that is not taken p becomes what of it is over q. The next
token is the first whose running sum of r = max(p - S q, 0) is over u_0 sum r. Drafts without a distribution (looked up, or the likeliest)
have q(x) = 1 at their token: M falls by p(x) (0 at least), r is p without the tokens that were not taken. Where r has no mass it is p; where p has
none the token is 0. Probabilities are fp32, what is computed from them fp64: a token changes only where u lies within some 2^-50 of a border. Values
that are not over 0 (NaN among them) have no mass, and a token outside of the vocabulary none either.

On the GPU attention takes bf16 queries and caches, heads of 64 or 128, at most 128 query heads a kv head, pages of 8 to 128 tokens; its
probabilities are rounded to bf16 (half a step, at most 2^-8 of the value) before their product with V, sums are fp32. `keep` moves rows of any type.
"""
from __future__ import annotations

import functools
import operator

import torch

from gllm_b200.ops import kv4

MOST_NODES = 64
PAGE_SIZES = (8, 16, 32, 64, 128)
HEAD_DIMS = (64, 128)
MOST_GROUP = 128          # query heads a kv head


# -- checks, the same on either device. What a common call passes comes first: a step makes one call a layer ---------------------
_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32


def num_seqs(inp) -> int:
    return getattr(inp, "padded_tokens", 0) or inp.num_seqs


def _index(t, what: str, n: int, dims: int = 1):
    if isinstance(t, torch.Tensor) and t.dtype is _I32 and t.dim() == dims and t.shape[0] >= n and (t.is_contiguous() or t.stride(-1) == 1):
        return t
    if not isinstance(t, torch.Tensor) or t.dtype != _I32 or t.dim() != dims or (t.stride(-1) != 1 and t.shape[-1] > 1):
        raise ValueError(f"{what}: int32 with contiguous rows, {dims}-dimensional")
    if t.shape[0] < n:
        raise ValueError(f"{what}: {t.shape[0]} entries for {n}")
    return t


def _starts(inp):
    b = num_seqs(inp)
    if inp.max_q_len > MOST_NODES:
        raise ValueError(f"a sequence has at most {MOST_NODES} drafted nodes: got {inp.max_q_len}")
    return b, _index(inp.query_start_loc, "query_start_loc", b + 1)


def check_batch(inp):
    """(sequences, query_start_loc, seq_lens, block_table): each looked up once, since an engine's batch makes a view of it."""
    b, start = _starts(inp)
    return b, start, _index(inp.seq_lens, "seq_lens", b), _index(inp.block_table, "block_table", b, 2)


def check_plan(parents, inp, page_size):
    _index(parents, "parents", 0)
    if page_size < 1:
        raise ValueError(f"pages of {page_size} tokens")
    return check_batch(inp)


def check_attention(q, k_cache, v_cache, inp, seen, scale, num_q_heads, head_dim, out):
    batch = check_batch(inp)
    if kv4.held(k_cache) or kv4.held(v_cache):
        raise ValueError("drafted tokens are attended over bf16 caches, not over one held in 4 bits")
    shape = k_cache.shape
    if len(shape) != 5 or v_cache.shape != shape or not k_cache.dtype is v_cache.dtype is q.dtype:
        raise ValueError(f"caches [pages, heads, slabs, page, slab] of the queries' type: got {tuple(shape)}, {tuple(v_cache.shape)}, "
                         f"{k_cache.dtype}, {v_cache.dtype}, {q.dtype}")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()) or shape[0] < 1 or batch[3].shape[1] < 1:
        raise ValueError("caches are contiguous and have pages, block_table has columns")
    _, hkv, slabs, _, w = shape
    rows, width = q.shape if q.dim() == 2 else (0, -1)
    if slabs * w != head_dim or num_q_heads % hkv or width < num_q_heads * head_dim or q.stride(1) != 1:
        raise ValueError(f"queries {tuple(q.shape)} of {num_q_heads} heads of {head_dim} over {hkv} heads of {slabs * w}")
    if seen.dtype is not _I64 or seen.dim() != 1 or seen.shape[0] < rows or not seen.is_contiguous():
        raise ValueError("seen: int64, contiguous, a word for each row of q")
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"a scale over 0: got {scale}")
    if out is not None and (out.dtype != q.dtype or out.shape != (rows, num_q_heads * head_dim) or not out.is_contiguous()):
        raise ValueError("out: contiguous, [rows of q, heads * dim], of its type")
    return batch


def check_verify(tokens, parents, inp, target, draft, uniform):
    """(sequences, query_start_loc, whether the target's tokens are given)"""
    b, start = _starts(inp)
    t = _index(tokens, "tokens", 0).shape[0]
    _index(parents, "parents", t)
    if target.dtype is not _F32 and not target.is_floating_point():
        _index(target, "target tokens", t)
        if draft is not None or uniform is not None:
            raise ValueError("target tokens are compared: no draft probabilities and no random numbers go with them")
        return b, start, True
    for x, what in ((target, "target"), (draft, "draft")):
        if x is not None and (x.dtype is not _F32 or x.dim() != 2 or x.shape[0] < t or (x.stride(1) != 1 and x.shape[1] > 1)):
            raise ValueError(f"{what}: fp32 probabilities [rows, vocabulary], rows contiguous")
    if target.shape[1] < 1 or (draft is not None and draft.shape[1] != target.shape[1]):
        raise ValueError("target and draft are over one vocabulary")
    if uniform is None or uniform.dtype is not _F32 or uniform.dim() != 1 or uniform.shape[0] < t or not uniform.is_contiguous():
        raise ValueError("uniform: fp32 in [0, 1), one for each row")
    return b, start, False


_shape_of, _dtype_of = operator.attrgetter("shape"), operator.attrgetter("dtype")


def cache_groups(k_caches, v_caches):
    """[(shape, bytes of an element, addresses, tensors)]: the tensors of all layers by shape, each once (layers may share one; None: a
    layer without)."""
    caches = [c for c in (*k_caches, *(v_caches or ())) if c is not None]
    if not caches:
        return []
    shape, dtype, n = caches[0].shape, caches[0].dtype, len(caches)
    at = list(map(torch.Tensor.data_ptr, caches))
    size = caches[0].element_size()
    if len(shape) == 5 and dtype is not torch.uint8 and shape[4] * size % 16 == 0 and all(map(torch.Tensor.is_contiguous, caches)) and \
            list(map(_shape_of, caches)).count(shape) == n and list(map(_dtype_of, caches)).count(dtype) == n and len(set(at)) == n and \
            functools.reduce(operator.or_, at) % 16 == 0:
        return [(shape, size, at, caches)]
    groups, seen = {}, set()
    for c, a in zip(caches, at):
        if kv4.held(c):
            raise ValueError("rows of a cache held in 4 bits are not moved")
        if c.dim() != 5 or not c.is_contiguous() or c.shape[4] * c.element_size() % 16 or a % 16:
            raise ValueError(f"caches [pages, heads, slabs, page, slab], contiguous, slabs of whole 16-byte words: got {tuple(c.shape)} {c.dtype}")
        if a not in seen and c.numel():
            seen.add(a)
            _, _, some, tensors = groups.setdefault((c.shape, c.element_size()), (c.shape, c.element_size(), [], []))
            some.append(a)
            tensors.append(c)
    return list(groups.values())


def check_keep(inp, path, count):
    batch = check_batch(inp)
    _index(path, "path", 0)
    _index(count, "count", batch[0])
    return batch


# -- plain form ------------------------------------------------------------------------------------------------------------
def _sequences(inp, rows: int):
    """(sequence, first row, nodes) of those that have any."""
    b = num_seqs(inp)
    start = inp.query_start_loc[: b + 1].tolist()
    return [(s, start[s], min(start[s + 1], rows) - start[s]) for s in range(b) if min(start[s + 1], rows) > start[s]]


def plan(parents, inp, page_size: int):
    check_plan(parents, inp, page_size)
    t = parents.shape[0]
    seen = torch.zeros(t, dtype=torch.int64)
    positions = torch.zeros(t, dtype=torch.int32)
    slots = torch.full((t,), -1, dtype=torch.int32)
    table, lens, up = inp.block_table, inp.seq_lens.tolist(), parents.tolist()
    for s, a, n in _sequences(inp, t):
        ctx = max(lens[s] - n, 0)
        masks = []
        for i in range(min(n, MOST_NODES)):
            p = up[a + i]
            masks.append((masks[p] if 0 <= p < i else 0) | 1 << i)
            positions[a + i] = ctx + bin(masks[i]).count("1") - 1
            page = (ctx + i) // page_size
            if page < table.shape[1]:
                slots[a + i] = int(table[s, page]) * page_size + (ctx + i) % page_size
            seen[a + i] = masks[i] - (1 << 64 if masks[i] >> 63 else 0)
    return seen, positions, slots


def attention(q, k_cache, v_cache, inp, seen, scale, num_q_heads, head_dim, out=None):
    from gllm_b200.ops.ref import gather_kv
    check_attention(q, k_cache, v_cache, inp, seen, scale, num_q_heads, head_dim, out)
    if out is None:
        out = torch.zeros(q.shape[0], num_q_heads * head_dim, dtype=q.dtype)
    g, lens = num_q_heads // k_cache.shape[1], inp.seq_lens.tolist()
    for s, a, n in _sequences(inp, q.shape[0]):
        ctx = max(lens[s] - n, 0)
        length = min(ctx + n, inp.block_table.shape[1] * k_cache.shape[3])
        k, v = (gather_kv(c, inp.block_table[s], length).float().repeat_interleave(g, 1) for c in (k_cache, v_cache))
        qq = q[a:a + n, : num_q_heads * head_dim].reshape(n, num_q_heads, head_dim).float()
        z = torch.einsum("qhd,khd->hqk", qq, k) * scale
        sees = torch.ones(n, ctx + n, dtype=torch.bool)
        sees[:, ctx:] = (seen[a:a + n, None] >> torch.arange(n)) & 1 > 0
        sees = sees[:, :length]
        z = z.masked_fill(~sees, float("-inf"))
        p = torch.where(sees.any(-1)[:, None], z.softmax(-1), 0.0)
        hidden = torch.where(sees[None, :, :, None], p[..., None] * v.permute(1, 0, 2)[:, None], 0.0)    # 0 times what is no number: 0
        out[a:a + n] = hidden.sum(2).permute(1, 0, 2).reshape(n, -1).to(q.dtype)
    return out


def _mass(x):
    return torch.where(x > 0, x, 0.0)


def verify(tokens, parents, inp, target, draft=None, uniform=None):
    check_verify(tokens, parents, inp, target, draft, uniform)
    t, b = tokens.shape[0], num_seqs(inp)
    said, path = (torch.full((t,), -1, dtype=torch.int32) for _ in range(2))
    count = torch.zeros(b, dtype=torch.int32)
    word, up = tokens.tolist(), parents.tolist()
    vocab = target.shape[1] if target.dim() == 2 else 0
    for s, a, n in _sequences(inp, t):
        n, node, taken = min(n, MOST_NODES), 0, [0]
        while True:
            children = [i for i in range(node + 1, n) if up[a + i] == node]
            step = None
            if not vocab:
                after = int(target[a + node])
                step = next((i for i in children if word[a + i] == after), None)
            else:
                p = target[a + node].double()
                rest, mass, past = _mass(p), 1.0, 0.0
                for i in children:
                    x, u = word[a + i], float(uniform[a + i])
                    inside = 0 <= x < vocab
                    have = float(rest[x]) if inside else 0.0
                    if u * mass * (float(draft[a + node, x]) if draft is not None and inside else 1.0) < have:
                        step = i
                        break
                    if draft is None:
                        mass = max(mass - have, 0.0)
                        if inside:
                            rest[x] = 0.0
                    else:
                        past += mass
                        rest = _mass(p - past * draft[a + node].double())
                        mass = float(rest.sum())
                if step is None:
                    after = _draw(rest if float(rest.sum()) > 0 else _mass(p), float(uniform[a]))
            if step is None:
                break
            taken.append(step)
            node = step
        k = len(taken)
        count[s] = k
        path[a:a + k] = torch.tensor(taken, dtype=torch.int32)
        said[a:a + k] = torch.tensor([word[a + i] for i in taken[1:]] + [after], dtype=torch.int32)
    return said, path, count


def _draw(rest, u: float) -> int:
    total = rest.cumsum(0)
    if not float(total[-1]) > 0:
        return 0
    return min(int((total <= u * total[-1]).sum()), int(rest.nonzero().max()))


def keep(k_caches, v_caches, inp, path, count):
    check_keep(inp, path, count)
    table, lens, way, taken = inp.block_table, inp.seq_lens.tolist(), path.tolist(), count.tolist()
    moves = []
    for s, a, n in _sequences(inp, path.shape[0]):
        ctx = max(lens[s] - n, 0)
        moves += [(s, ctx + way[a + j], ctx + j) for j in range(1, min(taken[s], n, MOST_NODES)) if j < way[a + j] < min(n, MOST_NODES)]
    for c in (c for group in cache_groups(k_caches, v_caches) for c in group[3]):
        pages, page = c.shape[0], c.shape[3]
        places = []
        for s, old, new in moves:
            if max(old, new) // page < table.shape[1]:
                places.append((int(table[s, old // page]), old % page, int(table[s, new // page]), new % page))
        places = torch.tensor([x for x in places if 0 <= x[0] < pages and 0 <= x[2] < pages], dtype=torch.long).reshape(-1, 4)
        c[places[:, 2], :, :, places[:, 3]] = c[places[:, 0], :, :, places[:, 1]]
