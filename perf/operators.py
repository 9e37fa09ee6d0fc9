"""Operators of quantised serving: products in 8-bit integers and a key / value cache held in 4 bits.

Four entry points of `gllm_b200.layers.functional`, each in a plain form (elementary torch operations) and as the
framework's kernels:

  append   rope_kv_write on a 4-bit cache: per-head norm, rotation, keys and values quantised into their pages, the rows
           read back with kv_cache_rows
  attend   paged_attention over a 4-bit cache: decoding sequences, prompt portions, or both in one batch
  linear   linear with an 8-bit weight: rows quantised with a scale per token, products summed in integers, scales per
           token and output channel (and a bias)
  gated    linear_silu_mul with an 8-bit weight: the same with silu(gate) * up behind it

The 4-bit cache, one uint8 tensor each for keys and values, is [pages, kv heads, page_size / 16, 9 * D]: blocks of 16 tokens, a
block 16 rows of D / 2 bytes and then 16 x D / 64 pairs (scale, low) of bf16, one pair for each 64 dims of a token's head. A
row's 32-bit unit u holds eight dims, the first in the lowest four bits: those from 64 (u % (D / 64)) + 8 (u // (D / 64)) on. A
code c stands for c * scale + low.

`listed()`, `draw(rng)`, `prepare(case, seed)`, `run(state)`, `work(case)`, `exact(case, seed)`.
"""
import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
PAGE = 16
EPS = 1e-6


def listed():
    return [
        # a lone chat: the token of one sequence, normed heads
        {"name": "append_decode_1", "kind": "append", "tokens": 1, "hq": 32, "hkv": 8, "dim": 128, "norm": True, "rot": 128,
         "neox": True},
        # a large decode batch: one token each, no norms
        {"name": "append_decode_256", "kind": "append", "tokens": 256, "hq": 64, "hkv": 8, "dim": 128, "norm": False, "rot": 128,
         "neox": True},
        # a chunk of prompts where half of each head is rotated in neighbouring pairs and few heads hold keys; an odd length
        {"name": "append_prompt_2047", "kind": "append", "tokens": 2047, "hq": 32, "hkv": 2, "dim": 128, "norm": False, "rot": 64,
         "neox": False},
        # a full prefill chunk of the throughput workload
        {"name": "append_prompt_4096", "kind": "append", "tokens": 4096, "hq": 32, "hkv": 8, "dim": 128, "norm": True, "rot": 128,
         "neox": True},
        # a lone chat over a short history: latency
        {"name": "attend_decode_1", "kind": "attend", "hq": 32, "hkv": 8, "dim": 128, "decodes": 1, "prompts": 0, "tokens": 0,
         "ctx": 700, "mix": 1},
        # a decode batch over ragged histories
        {"name": "attend_decode_64", "kind": "attend", "hq": 32, "hkv": 8, "dim": 128, "decodes": 64, "prompts": 0, "tokens": 0,
         "ctx": 2500, "mix": 2},
        # few sequences with long histories: what a 4-bit cache is taken for
        {"name": "attend_long_4", "kind": "attend", "hq": 64, "hkv": 8, "dim": 128, "decodes": 4, "prompts": 0, "tokens": 0,
         "ctx": 60000, "mix": 3},
        # a chunked-prefill step: ragged prompts, some with cached prefixes, beside decoding sequences; heads of 64
        {"name": "attend_step_3000", "kind": "attend", "hq": 32, "hkv": 8, "dim": 64, "decodes": 8, "prompts": 3, "tokens": 3000,
         "ctx": 1200, "mix": 4},
        # decoding: the fused projection of queries, keys and values for one token
        {"name": "linear_1", "kind": "linear", "rows": 1, "n": 6144, "k": 4096, "bias": False},
        # a prompt of odd length through a wide projection with a bias
        {"name": "linear_777", "kind": "linear", "rows": 777, "n": 10240, "k": 8192, "bias": True},
        # the gated projection of a decode batch: weights are the traffic
        {"name": "gated_64", "kind": "gated", "rows": 64, "n": 24576, "k": 4096, "bias": False},
        # the gated projection of a full prefill chunk
        {"name": "gated_4096", "kind": "gated", "rows": 4096, "n": 24576, "k": 4096, "bias": False},
    ]


def draw(rng):
    most = max(_plain_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _plain_cost(case) <= most:
            return case


def _draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("append", "attend", "linear", "gated"))
    if kind == "append":
        hkv, g, dim = rng.choice((1, 2, 4, 8, 32)), rng.choice((1, 2, 4, 5, 7, 8)), rng.choice((64, 128))
        return {"kind": kind, "tokens": log(1, 4096), "hq": hkv * g, "hkv": hkv, "dim": dim, "norm": rng.random() < 0.5,
                "rot": rng.choice((dim, dim, dim // 2)), "neox": rng.random() < 0.7}
    if kind == "attend":
        hkv, g, dim = rng.choice((1, 2, 4, 8, 32)), rng.choice((1, 2, 4, 5, 7, 8)), rng.choice((64, 128))
        case = {"kind": kind, "hq": hkv * g, "hkv": hkv, "dim": dim, "decodes": 0, "prompts": 0, "tokens": 0,
                "ctx": log(20, 60000), "mix": rng.randrange(1 << 20)}
        what = rng.random()
        if what < 0.8:
            case["decodes"] = log(1, 128)
        if what > 0.6:
            case["prompts"] = rng.randint(1, 4)
            case["tokens"] = log(8, 2048)
            case["ctx"] = min(case["ctx"], 3000)
            case["decodes"] = min(case["decodes"], 8)
        return case
    k = 16 * log(4, 768)
    if kind == "linear":
        return {"kind": kind, "rows": log(1, 4096), "n": 8 * log(16, 2048), "k": k, "bias": rng.random() < 0.5}
    return {"kind": kind, "rows": log(1, 4096), "n": 16 * log(16, 1536), "k": k, "bias": False}


# ------------------------------------------------------------------------------------------------------------------------
# what a case does
# ------------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """(tokens in the cache, new tokens) of each sequence, decoding ones first."""
    rng = np.random.RandomState(case["mix"])
    ctx = case["ctx"]
    lens = [int(x) for x in rng.randint(max(1, ctx // 2), ctx + 1, case["decodes"])]
    new = [1] * case["decodes"]
    if case["prompts"]:
        n = case["prompts"]
        share = rng.dirichlet([4.0] * n) * max(0, case["tokens"] - n)
        for i in range(n):
            q = 1 + int(share[i])
            prior = int(rng.randint(0, ctx + 1)) if rng.rand() < 0.5 else 0
            lens.append(q + prior)
            new.append(q)
    return lens, new


def work(case):
    if case["kind"] == "append":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
        row = 9 * d / 16
        # q in and out, k and v in, codes out; read back: codes in, rows out; angles, positions and slots
        return {"bytes": t * (4 * hq * d + 2 * 2 * hkv * d + 2 * 2 * hkv * row + 2 * 2 * hkv * d + 4 * case["rot"] + 8),
                "flops": t * (hq + 2 * hkv) * d * 4}
    if case["kind"] == "attend":
        lens, new = _lengths(case)
        hq, hkv, d = case["hq"], case["hkv"], case["dim"]
        pairs = sum(q * (n - q) + q * (q + 1) / 2 for n, q in zip(lens, new))
        return {"bytes": sum(lens) * 2 * hkv * 9 * d / 16 + 2 * sum(new) * hq * d * 2, "flops": 4 * pairs * hq * d}
    m, n, k = case["rows"], case["n"], case["k"]
    return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * (n if case["kind"] == "linear" else n // 2), "flops": 2 * m * n * k}


def _plain_cost(case):
    """Seconds that the plain form takes, roughly: a drawn case costs no more than the largest listed one."""
    if case["kind"] == "attend":
        lens, new = _lengths(case)
        pad = len(lens) * max(lens)
        return (pad * case["hkv"] * case["dim"] * 60 + pad * max(new) * case["hq"] * 40) / 3e12
    w = work(case)
    return w["bytes"] * 8 / 3e12 if case["kind"] == "append" else w["flops"] / 5e13 + w["bytes"] / 1e12


# ------------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------------
def _units(dim):
    """Dim of each nibble of a cached row, in storage order."""
    g = dim // 64
    u = torch.arange(dim // 8, device=DEV).unsqueeze(1)
    return (64 * (u % g) + 8 * torch.div(u, g, rounding_mode="floor") + torch.arange(8, device=DEV)).reshape(-1)


def _coded(x):
    """Rows [..., D] as they lie in a cache: codes [..., D / 2] and pairs [..., D / 16], bytes."""
    dim = x.shape[-1]
    grouped = x.float().unflatten(-1, (dim // 64, 64))
    low, high = grouped.amin(-1, keepdim=True), grouped.amax(-1, keepdim=True)
    scale = ((high - low) / 15).to(BF16).float()
    codes = torch.where(scale > 0, torch.round((grouped - low) / scale), 0.0).clamp(0, 15).to(torch.uint8).flatten(-2)
    codes = codes[..., _units(dim)].unflatten(-1, (dim // 2, 2))
    return codes[..., 0] | (codes[..., 1] << 4), torch.cat((scale, low), -1).to(BF16).view(torch.uint8).flatten(-2)


def _pack(x):
    """[..., 16, D] -> blocks [..., 9 D] of a 4-bit cache."""
    return torch.cat([y.flatten(-2) for y in _coded(x)], -1)


def _keys_values(gen, n, heads, dim):
    """Rows as a trained model has them: dims with offsets and widths of their own."""
    offset = torch.randn(1, heads, dim, generator=gen, device=DEV) * 0.7
    width = 0.5 + torch.rand(1, heads, dim, generator=gen, device=DEV)
    return (torch.randn(n, heads, dim, generator=gen, device=DEV) * width + offset).to(BF16)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "append":
        return _prepare_append(case, gen)
    if case["kind"] == "attend":
        return _prepare_attend(case, gen)
    m, n, k = case["rows"], case["n"], case["k"]
    x = torch.randn(m, k, generator=gen, device=DEV)
    x = (x * (0.2 + 2 * torch.rand(m, 1, generator=gen, device=DEV))).to(BF16)
    w = torch.clamp(torch.round(torch.randn(n, k, generator=gen, device=DEV) * 32), -127, 127).to(torch.int8)
    scale = (0.5 + torch.rand(n, generator=gen, device=DEV)) * (0.03 / 32)
    bias = torch.randn(n, generator=gen, device=DEV).to(BF16) if case["bias"] else None
    return SimpleNamespace(case=case, x=x, w=w, scale=scale, bias=bias)


def _prepare_append(case, gen):
    t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
    # the fused projection's output: q, k and v are views of its rows
    qkv = torch.empty(t, (hq + 2 * hkv) * d, dtype=BF16, device=DEV)
    q, k, v = (x.view(t, -1, d) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
    q.copy_(torch.randn(t, hq, d, generator=gen, device=DEV))
    k.copy_(_keys_values(gen, t, hkv, d))
    v.copy_(_keys_values(gen, t, hkv, d))
    half = case["rot"] // 2
    most = 8192
    angles = torch.arange(most, device=DEV, dtype=F64).unsqueeze(1) * 1e6 ** (-torch.arange(half, device=DEV, dtype=F64) / half)
    cos_sin = torch.cat((angles.cos(), angles.sin()), 1).float()
    positions = torch.randint(0, most, (t,), generator=gen, device=DEV, dtype=torch.int32)
    pages = -(-t // PAGE) + 3
    caches = [torch.zeros(pages, hkv, PAGE // 16, 9 * d, dtype=torch.uint8, device=DEV) for _ in range(2)]
    slots = torch.randperm(pages * PAGE, generator=gen, device=DEV)[:t].to(torch.int32)
    norms = [(1 + 0.1 * torch.randn(d, generator=gen, device=DEV)).to(BF16) if case["norm"] else None for _ in range(2)]
    return SimpleNamespace(case=case, q=q, k=k, v=v, cos_sin=cos_sin, positions=positions, caches=caches, slots=slots, norms=norms)


def _prepare_attend(case, gen):
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    lens, new = _lengths(case)
    blocks = [-(-n // PAGE) for n in lens]
    pages = sum(blocks) + 1
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros(len(lens), max(blocks), dtype=torch.int32, device=DEV)
    at = 0
    for s, b in enumerate(blocks):
        table[s, :b] = order[at:at + b]
        at += b
    caches = []
    for _ in range(2):
        cache = torch.empty(pages, hkv, PAGE // 16, 9 * d, dtype=torch.uint8, device=DEV)
        for p0 in range(0, pages, 4096):
            p1 = min(p0 + 4096, pages)
            rows = _keys_values(gen, (p1 - p0) * PAGE, hkv, d).view(p1 - p0, PAGE // 16, 16, hkv, d)
            cache[p0:p1] = _pack(rows.permute(0, 3, 1, 2, 4))
        caches.append(cache)
    q = torch.randn(sum(new), hq * d, generator=gen, device=DEV).to(BF16)
    start = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    inp = SimpleNamespace(block_table=table, seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV), query_start_loc=start.to(DEV),
                          num_decode_seqs=case["decodes"], num_seqs=len(lens), num_tokens=sum(new), padded_tokens=0,
                          max_q_len=max(new), max_seq_len=max(lens), decode_splits=None,
                          batch=SimpleNamespace(seq_lens=np.array(lens, np.int32), query_start_loc=start.numpy()))
    return SimpleNamespace(case=case, q=q, caches=caches, inp=inp)


# ------------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------------
def run(state):
    c = state.case
    if own:
        from gllm_b200.layers import functional as Fn
        if c["kind"] == "append":
            Fn.rope_kv_write(state.q, state.k, state.v, state.positions, state.cos_sin, c["rot"], c["neox"], state.norms[0],
                             state.norms[1], EPS, state.caches[0], state.caches[1], state.slots)
            return (state.q, *Fn.kv_cache_rows(state.caches[0], state.caches[1], state.slots))
        if c["kind"] == "attend":
            return Fn.paged_attention(state.q, state.caches[0], state.caches[1], state.inp, c["dim"] ** -0.5, c["hq"], c["dim"])
        if c["kind"] == "linear":
            return Fn.linear(state.x, (state.w, state.scale), state.bias)
        return Fn.linear_silu_mul(state.x, (state.w, state.scale))
    return {"append": _append, "attend": _attend, "linear": _linear, "gated": _gated}[c["kind"]](state)


def _turned(x, weight, state):
    """Norm and rotation of [T, heads, D] in 32 bits, rounded behind each."""
    c = state.case
    x = x.float()
    if weight is not None:
        x = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()).to(BF16).float()
    half = c["rot"] // 2
    rows = state.cos_sin[state.positions.long()].unsqueeze(1)
    cos, sin = rows[..., :half], rows[..., half:]
    if c["neox"]:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, x[..., 2 * half:]), -1).to(BF16)


def _decoded(rows, pairs, dim):
    """[..., D / 2] codes and [..., D / 16] pairs, bytes -> [..., D] in 32 bits."""
    codes = torch.stack((rows & 15, rows >> 4), -1).flatten(-2)
    back = torch.empty(dim, dtype=torch.long, device=rows.device)
    back[_units(dim)] = torch.arange(dim, device=rows.device)
    scale, low = pairs.contiguous().view(BF16).float().unflatten(-1, (dim // 64, 2)).unbind(-1)
    return (codes[..., back].float().unflatten(-1, (dim // 64, 64)) * scale.unsqueeze(-1) + low.unsqueeze(-1)).flatten(-2)


def _append(state):
    c = state.case
    state.q.copy_(_turned(state.q, state.norms[0], state))
    page, row = torch.div(state.slots, PAGE, rounding_mode="floor").long(), (state.slots % PAGE).long()
    out = [state.q]
    for x, cache in zip((_turned(state.k, state.norms[1], state), state.v), state.caches):
        d = c["dim"]
        codes = cache[:, :, 0, : 8 * d].unflatten(-1, (16, d // 2))
        pairs = cache[:, :, 0, 8 * d:].unflatten(-1, (16, d // 16))
        codes[page, :, row], pairs[page, :, row] = _coded(x)
        out.append(_decoded(codes[page, :, row], pairs[page, :, row], d).to(BF16))
    return tuple(out)


def _attend(state):
    c, inp = state.case, state.inp
    d, hkv, g = c["dim"], c["hkv"], c["hq"] // c["hkv"]
    n_seq, longest, most = inp.num_seqs, inp.max_seq_len, inp.max_q_len
    held = []
    for cache in state.caches:
        blocks = cache[inp.block_table.long()][:, :, :, 0]                          # [B, blocks, Hkv, 9 D]
        x = _decoded(blocks[..., : 8 * d].unflatten(-1, (16, d // 2)), blocks[..., 8 * d:].unflatten(-1, (16, d // 16)), d)
        held.append(x.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :longest])         # [B, Hkv, keys, D]
    start, lens = inp.query_start_loc.long(), inp.seq_lens.long()
    new = start[1:] - start[:-1]
    step = torch.arange(most, device=DEV)
    rows = (start[:-1, None] + torch.minimum(step, new[:, None] - 1))               # [B, queries]; the last one again behind the end
    q = state.q.float()[rows].view(n_seq, most, hkv, g, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = (q @ held[0].transpose(-1, -2) * d ** -0.5).view(n_seq, hkv, g, most, -1)
    last = (lens - new)[:, None] + step
    hidden = torch.arange(scores.shape[-1], device=DEV) > last[..., None]           # [B, queries, keys]
    scores = scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.flatten(2, 3) @ held[1]).view(n_seq, hkv, g, most, d) / total
    out = out.permute(0, 3, 1, 2, 4).flatten(2)                                     # [B, queries, Hq D]
    return out[step < new[:, None]].to(BF16)


def _sums(state):
    x = state.x.float()
    most = x.abs().amax(1, keepdim=True)
    codes = torch.where(most > 0, torch.round(x * 127 / most), 0.0)
    return (codes @ state.w.float().t()) * (most / 127) * state.scale


def _linear(state):
    y = _sums(state)
    return (y if state.bias is None else y + state.bias.float()).to(BF16)


def _gated(state):
    gate, up = _sums(state).chunk(2, 1)
    return (gate / (1 + (-gate).exp()) * up).to(BF16)


# ------------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "attend":
        return _exact_attend(s)
    x = s.x.double()
    unit = x.abs().max(dim=1).values / 127
    whole = (x / unit[:, None]).round()
    near = (x * 254 / x.abs().max(dim=1).values[:, None]).abs()                     # halves are ties: to the even number
    tie = (near == near.round()) & (near % 2 == 1)
    even = 2 * (x.abs() * 127 / x.abs().max(dim=1).values[:, None] / 2).round() * x.sign()
    whole = torch.where(tie, even, whole)
    y = torch.einsum("mk,nk->mn", whole * unit[:, None], s.w.double() * s.scale.double()[:, None])
    if case["kind"] == "gated":
        n = case["n"] // 2
        return torch.sigmoid(y[:, :n]) * y[:, :n] * y[:, n:]
    return y if s.bias is None else y + s.bias.double()


def _exact_append(s):
    c = s.case
    d, half = c["dim"], c["rot"] // 2
    first = torch.arange(half, device=DEV) * (1 if c["neox"] else 2)
    second = first + (half if c["neox"] else 1)
    cs = s.cos_sin.double()[s.positions.long()][:, None]

    def turned(x, w):
        x = x.double()
        if w is not None:                                                           # the norm rounds to bf16, as the rotation does
            x = (x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w.double()).to(BF16).double()
        y = x.clone()
        y[..., first] = x[..., first] * cs[..., :half] - x[..., second] * cs[..., half:]
        y[..., second] = x[..., second] * cs[..., :half] + x[..., first] * cs[..., half:]
        return y

    def held(x):
        parts = []
        for g0 in range(0, d, 64):
            y = x.to(BF16).double()[..., g0:g0 + 64]
            low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
            step = ((high - low) / 15).to(BF16).double()
            code = ((y - low) / torch.where(step == 0, 1.0, step)).round().clamp(max=15)
            parts.append(low + code * step)
        return torch.cat(parts, -1)

    return turned(s.q, s.norms[0]), held(turned(s.k, s.norms[1])), held(s.v)


def _exact_attend(s):
    c, inp = s.case, s.inp
    d, hkv = c["dim"], c["hkv"]
    g, groups = c["hq"] // hkv, d // 64
    lens, start = inp.batch.seq_lens.tolist(), inp.batch.query_start_loc.tolist()
    if sum(n * (b - a) for n, a, b in zip(lens, start, start[1:])) * c["hq"] * d > 3e13:
        return None
    out = torch.empty(s.q.shape[0], c["hq"], d, dtype=F64, device=DEV)
    for i, n in enumerate(lens):
        pages = inp.block_table[i, : -(-n // PAGE)].long()
        ql = start[i + 1] - start[i]
        for h in range(hkv):
            kv = []
            for cache in s.caches:
                block = cache[pages, h, 0]
                byte = block[:, : 8 * d].reshape(-1, d // 8, 4).long()                # tokens x units x bytes
                word = byte[..., 0] + (byte[..., 1] << 8) + (byte[..., 2] << 16) + (byte[..., 3] << 24)
                eight = torch.stack([(word >> (4 * e)) % 16 for e in range(8)], -1)   # tokens x units x dims
                x = eight.view(-1, d // 8 // groups, groups, 8).transpose(1, 2).reshape(-1, groups, 64).double()
                pair = block[:, 8 * d:].reshape(-1, 4 * groups).contiguous().view(BF16).double().view(-1, groups, 2)
                kv.append((x * pair[..., :1] + pair[..., 1:]).reshape(-1, d)[:n])
            q = s.q[start[i]:start[i + 1]].view(ql, hkv, g, d)[:, h].double()
            z = torch.einsum("qgd,kd->gqk", q, kv[0]) / math.sqrt(d)
            z = z + torch.full((ql, n), -math.inf, dtype=F64, device=DEV).triu(n - ql + 1)
            out[start[i]:start[i + 1], h * g:(h + 1) * g] = torch.einsum("gqk,kd->qgd", z.softmax(-1), kv[1])
    return out.flatten(1)
