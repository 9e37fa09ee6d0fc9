"""Operators of decoding with drafted tokens: a tree of drafts is laid out behind a paged cache, attended, verified and kept.

Four entry points of `gllm_b200.layers.functional`, each in a plain form (elementary torch operations) and as the framework's
kernels:

  plan     draft_plan: the parents of every sequence's nodes -> who sees whom, positions, cache slots
  attend   draft_attention: the nodes' queries over the paged cache; a node sees the context, itself and its ancestors
  verify   draft_verify: which of the drafted tokens the target model takes, and the token behind them: drafts drawn from
           distributions ("draws"), drafts without one ("given"), or tokens already drawn from the target at every node ("match")
  keep     draft_keep: keys and values of the nodes that were taken move up behind the context, in all layers

A sequence's nodes are its rows [query_start_loc[s], query_start_loc[s + 1]), at most 64. Node 0 is the last token that stands, a
parent comes before its node, -1 is none. `seq_lens` counts the nodes: node i lies at cache position seq_len - nodes + i.

Verification. At a node with target distribution p and draft distribution q its children are tried in order. With M_0 = 1 and S_0 = 0
child k, token x, is taken where u M_k q(x) < max(p(x) - S_k q(x), 0); otherwise S_k+1 = S_k + M_k and M_k+1 = sum_y max(p(y) -
S_k+1 q(y), 0). Behind the last node taken the next token is the first whose running sum of max(p - S q, 0) is over u times the
whole. A draft without a distribution has q(x) = 1: M falls by p(x), the token leaves p.

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
TAKEN = 0.4                     # share of nodes that the keep cases move


def listed():
    return [
        # one chat: a small tree behind a few hundred tokens
        {"name": "plan_1", "kind": "plan", "seqs": 1, "nodes": 8, "reach": 3, "ctx": 700, "mix": 11},
        # a large batch of full trees
        {"name": "plan_256", "kind": "plan", "seqs": 256, "nodes": 64, "reach": 9, "ctx": 2500, "mix": 12},
        # one chat: latency
        {"name": "attend_1", "kind": "attend", "hq": 32, "hkv": 8, "dim": 128, "seqs": 1, "nodes": 8, "reach": 3, "ctx": 700, "mix": 1},
        # a batch of small trees over ragged histories, heads of 64, seven query heads a kv head
        {"name": "attend_batch_48", "kind": "attend", "hq": 14, "hkv": 2, "dim": 64, "seqs": 48, "nodes": 13, "reach": 4, "ctx": 1500,
         "mix": 2},
        # two long documents
        {"name": "attend_long_2", "kind": "attend", "hq": 64, "hkv": 8, "dim": 128, "seqs": 2, "nodes": 16, "reach": 6, "ctx": 60000,
         "mix": 3},
        # full trees: the keys are read for 256 rows a head
        {"name": "attend_wide_16", "kind": "attend", "hq": 32, "hkv": 8, "dim": 128, "seqs": 16, "nodes": 64, "reach": 12, "ctx": 4000,
         "mix": 4},
        # greedy decoding of a batch: the target's own tokens are known
        {"name": "verify_match_64", "kind": "verify", "form": "match", "seqs": 64, "nodes": 12, "reach": 4, "vocab": 151936, "mix": 5},
        # one chat: a chain of four drafts from a small model
        {"name": "verify_chain_1", "kind": "verify", "form": "draws", "seqs": 1, "nodes": 5, "reach": 1, "vocab": 151936, "mix": 6},
        # a batch of chains; an odd vocabulary
        {"name": "verify_chain_64", "kind": "verify", "form": "draws", "seqs": 64, "nodes": 6, "reach": 1, "vocab": 128257, "mix": 7},
        # trees of looked-up continuations, which have no distribution
        {"name": "verify_tree_16", "kind": "verify", "form": "given", "seqs": 16, "nodes": 32, "reach": 6, "vocab": 151936, "mix": 8},
        # one chat: some rows of every layer
        {"name": "keep_1", "kind": "keep", "layers": 36, "heads": 8, "dim": 128, "seqs": 1, "nodes": 8, "ctx": 100, "mix": 9},
        # a batch of trees
        {"name": "keep_64", "kind": "keep", "layers": 36, "heads": 8, "dim": 128, "seqs": 64, "nodes": 24, "ctx": 100, "mix": 10},
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

    kind = rng.choice(("plan", "attend", "attend", "verify", "verify", "keep"))
    case = {"kind": kind, "nodes": log(1, 64), "mix": rng.randrange(1 << 20)}
    if kind == "keep":
        return {**case, "layers": log(1, 64), "heads": rng.choice((1, 2, 4, 8, 32)), "dim": rng.choice((64, 128)), "seqs": log(1, 128),
                "ctx": log(1, 300)}
    case["reach"] = rng.randint(1, 12)
    if kind == "plan":
        return {**case, "seqs": log(1, 256), "ctx": log(1, 10000)}
    if kind == "attend":
        hkv, g = rng.choice((1, 2, 4, 8, 32)), rng.choice((1, 2, 4, 5, 7, 8))
        return {**case, "hq": hkv * g, "hkv": hkv, "dim": rng.choice((64, 128)), "seqs": log(1, 128), "ctx": log(4, 60000)}
    return {**case, "form": rng.choice(("match", "draws", "draws", "given")), "seqs": log(1, 64), "vocab": log(1000, 152000)}


# ------------------------------------------------------------------------------------------------------------------------
# what a case does
# ------------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """(context, nodes) of each sequence."""
    rng = np.random.RandomState(case["mix"])
    n, ctx = case["nodes"], case.get("ctx", 0)
    nodes = [n] + [int(x) for x in rng.randint((n + 1) // 2, n + 1, case["seqs"] - 1)]
    return [int(x) for x in rng.randint(ctx // 2, ctx + 1, case["seqs"])], nodes


def work(case):
    ctx, nodes = _lengths(case)
    rows = sum(nodes)
    if case["kind"] == "plan":      # parents in; masks, positions and slots out; pages of the nodes
        return {"bytes": rows * (4 + 8 + 4 + 4) + 4 * sum(n // PAGE + 1 for n in nodes), "flops": rows * math.log2(case["nodes"] + 1)}
    if case["kind"] == "attend":    # every key and value once; a node sees the context and itself at least
        hq, hkv, d = case["hq"], case["hkv"], case["dim"]
        return {"bytes": (sum(ctx) + rows) * 2 * hkv * d * 2 + rows * (2 * hq * d * 2 + 8),
                "flops": 4 * sum(n * (c + 1) for c, n in zip(ctx, nodes)) * hq * d}
    if case["kind"] == "verify":    # the row behind the last node taken, and the drafts' where it has one; single values of the others
        each = {"match": 0, "given": 1, "draws": 2}[case["form"]] * case["vocab"]
        return {"bytes": 4 * case["seqs"] * each + rows * (4 + 4 + 4 + 4 * 3), "flops": 3 * case["seqs"] * each + rows}
    # rows that move, in and out
    moved = sum(TAKEN * (n - 1) - sum(TAKEN ** j for j in range(1, n)) for n in nodes)
    return {"bytes": moved * 2 * 2 * case["layers"] * case["heads"] * case["dim"] * 2 + 8 * rows, "flops": rows}


def _plain_cost(case):
    """Seconds that the plain form takes, roughly: a drawn case costs no more than the largest listed one."""
    ctx, nodes = _lengths(case)
    seqs, most = case["seqs"], case["nodes"]
    if case["kind"] == "attend":
        pad = seqs * (max(ctx) + most)
        return (pad * case["hkv"] * case["dim"] * 20 + pad * most * case["hq"] * 40) / 3e12
    if case["kind"] == "verify":
        return seqs * case["vocab"] * {"match": 0, "given": 60, "draws": 30 * most}[case["form"]] / 3e12
    if case["kind"] == "keep":
        return (sum(ctx) + sum(nodes)) * 4 * case["layers"] * case["heads"] * case["dim"] / 3e12
    return seqs * most * most * 100 / 3e12


# ------------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------------
def _batch(case, gen):
    """What a step knows of its sequences, and the parents of their nodes: one of the `reach` nodes before each."""
    ctx, nodes = _lengths(case)
    blocks = [-(-(c + n) // PAGE) for c, n in zip(ctx, nodes)]
    pages = sum(blocks) + 1
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros(len(nodes), max(blocks), dtype=torch.int32, device=DEV)
    held = torch.arange(max(blocks), device=DEV) < torch.tensor(blocks, device=DEV).unsqueeze(1)
    table[held] = order[: sum(blocks)]
    start = torch.tensor([0] + nodes).cumsum(0).to(torch.int32)
    inp = SimpleNamespace(block_table=table, seq_lens=torch.tensor([c + n for c, n in zip(ctx, nodes)], dtype=torch.int32, device=DEV),
                          query_start_loc=start.to(DEV), num_seqs=len(nodes), num_tokens=sum(nodes), max_q_len=max(nodes),
                          max_seq_len=max(c + n for c, n in zip(ctx, nodes)))
    node = torch.cat([torch.arange(n) for n in nodes]).to(DEV)
    back = 1 + (torch.rand(sum(nodes), generator=gen, device=DEV) * node.clamp(max=case.get("reach", 1))).floor().long()
    parents = torch.where(node > 0, (node - back).clamp(min=0), -1).to(torch.int32)
    return inp, parents, pages


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    inp, parents, pages = _batch(case, gen)
    s = SimpleNamespace(case=case, inp=inp, parents=parents)
    if case["kind"] == "attend":
        hq, hkv, d = case["hq"], case["hkv"], case["dim"]
        s.q = torch.randn(inp.num_tokens, hq * d, generator=gen, device=DEV).to(BF16)
        s.caches = [torch.empty(pages, hkv, d // 64, PAGE, 64, dtype=BF16, device=DEV).normal_(generator=gen) for _ in range(2)]
        s.seen = _plan(s)[0]        # of the whole step: its layers share it
    elif case["kind"] == "verify":
        _prepare_verify(s, gen)
    elif case["kind"] == "keep":
        # one buffer, of which every layer's keys and values are views
        s.held = torch.empty(2, case["layers"], pages, case["heads"], case["dim"] // 64, PAGE, 64, dtype=BF16, device=DEV).normal_(generator=gen)
        s.caches = [list(x.unbind()) for x in s.held]
        taken = torch.rand(inp.num_tokens, generator=gen, device=DEV) < TAKEN
        first, at = inp.query_start_loc[:-1].long(), torch.arange(inp.num_tokens, device=DEV)
        taken[first] = True
        seq = torch.bucketize(at, inp.query_start_loc[1:].long(), right=True)
        before = taken.cumsum(0) - 1
        place = first[seq] + before - before[first][seq]
        s.path = torch.full((inp.num_tokens,), -1, dtype=torch.int32, device=DEV)
        s.path[place[taken]] = (at - first[seq])[taken].to(torch.int32)
        s.count = torch.zeros(inp.num_seqs, dtype=torch.int32, device=DEV).index_add_(0, seq, taken.to(torch.int32))
    return s


def _prepare_verify(s, gen):
    """Targets as trained models have them (a few likely tokens), drafts from a model that is near; two of three are taken."""
    case, t, v = s.case, s.inp.num_tokens, s.case["vocab"]
    s.draft = s.uniform = None
    first = s.inp.query_start_loc[:-1].long()
    seq = torch.bucketize(torch.arange(t, device=DEV), s.inp.query_start_loc[1:].long(), right=True)
    above = first[seq] + s.parents.long().clamp(min=0)
    if case["form"] == "match":
        s.target = torch.randint(0, v, (t,), generator=gen, device=DEV, dtype=torch.int32)
        other = torch.randint(0, v, (t,), generator=gen, device=DEV, dtype=torch.int32)
        s.tokens = torch.where(torch.rand(t, generator=gen, device=DEV) < 0.6, s.target[above], other)
        return
    z = torch.randn(t, v, generator=gen, device=DEV) * 3
    s.target = z.softmax(-1)
    if case["form"] == "draws":
        s.draft = z.add_(torch.randn(t, v, generator=gen, device=DEV) * 0.8).softmax(-1)
    del z
    s.tokens = torch.multinomial((s.target if s.draft is None else s.draft)[above], 1, generator=gen)[:, 0].to(torch.int32)
    s.uniform = torch.rand(t, generator=gen, device=DEV)


# ------------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------------
def run(state):
    c = state.case
    if own:
        from gllm_b200.layers import functional as Fn
        if c["kind"] == "plan":
            return Fn.draft_plan(state.parents, state.inp, PAGE)
        if c["kind"] == "attend":
            return Fn.draft_attention(state.q, state.caches[0], state.caches[1], state.inp, state.seen, c["dim"] ** -0.5, c["hq"], c["dim"])
        if c["kind"] == "verify":
            return Fn.draft_verify(state.tokens, state.parents, state.inp, state.target, state.draft, state.uniform)
        Fn.draft_keep(state.caches[0], state.caches[1], state.inp, state.path, state.count)
        return state.held
    return {"plan": _plan, "attend": _attend, "verify": _verify, "keep": _keep}[c["kind"]](state)


def _nodes(inp):
    """Rows of the nodes [B, most] (the sequence's last one again behind its end) and which there are."""
    start = inp.query_start_loc.long()
    n = start[1:] - start[:-1]
    step = torch.arange(inp.max_q_len, device=DEV)
    return start[:-1, None] + torch.minimum(step, n[:, None] - 1), step < n[:, None]


def _lines(parents):
    """[B, n, n]: whether j is i or an ancestor of i."""
    n = parents.shape[1]
    at = torch.arange(n, device=DEV)
    up = (parents.unsqueeze(2) == at).float() + torch.eye(n, device=DEV)
    return torch.linalg.matrix_power(up, 64) > 0


def _plan(state):
    inp = state.inp
    rows, there = _nodes(inp)
    at = torch.arange(inp.max_q_len, device=DEV)
    lines = _lines(state.parents.long()[rows])
    seen = (lines.long() << at).sum(-1)
    ctx = (inp.seq_lens - inp.query_start_loc[1:] + inp.query_start_loc[:-1]).long()
    positions = ctx[:, None] + lines.sum(-1) - 1
    place = ctx[:, None] + at
    blocks = torch.div(place, PAGE, rounding_mode="floor").clamp(max=inp.block_table.shape[1] - 1)
    slots = inp.block_table.gather(1, blocks).long() * PAGE + place % PAGE
    return seen[there], positions[there].to(torch.int32), slots[there].to(torch.int32)


def _attend(state):
    c, inp = state.case, state.inp
    d, hkv, g = c["dim"], c["hkv"], c["hq"] // c["hkv"]
    longest, most = inp.max_seq_len, inp.max_q_len
    held = [x[inp.block_table.long()].permute(0, 2, 1, 4, 3, 5).flatten(4).flatten(2, 3)[:, :, :longest].float() for x in state.caches]
    rows, there = _nodes(inp)
    q = state.q[rows].float().view(inp.num_seqs, most, hkv, g, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = (q @ held[0].transpose(-1, -2) * d ** -0.5).view(inp.num_seqs, hkv, g, most, longest)
    place = torch.arange(longest, device=DEV)
    node = place - (inp.seq_lens - there.sum(1))[:, None]                            # [B, keys]: which node a key is
    bit = (state.seen[rows].unsqueeze(2) >> node.clamp(0, 63).unsqueeze(1)) & 1      # [B, nodes, keys]
    hidden = (node.unsqueeze(1) >= 0) & ((bit == 0) | (place >= inp.seq_lens[:, None]).unsqueeze(1))
    scores = scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.flatten(2, 3) @ held[1]).view(inp.num_seqs, hkv, g, most, d) / total
    return out.permute(0, 3, 1, 2, 4).flatten(2)[there].to(BF16)


def _verify(state):
    inp, form = state.inp, state.case["form"]
    n = inp.max_q_len
    rows, there = _nodes(inp)
    tokens, parents = state.tokens.long()[rows], torch.where(there, state.parents.long()[rows], -2)
    above = inp.query_start_loc[:-1, None].long() + parents.clamp(min=0)
    at = torch.arange(n, device=DEV)
    elder = (parents.unsqueeze(2) == parents.unsqueeze(1)) & (at < at[:, None]) & (parents >= 0).unsqueeze(2)
    children = ((parents.unsqueeze(2) == at) & there.unsqueeze(2)).sum(1)            # of each node
    if form == "match":
        taken = state.target.long()[above] == tokens
    else:
        u, p = state.uniform.double()[rows], state.target[above, tokens].double()
        if form == "given":
            again = (elder & (tokens.unsqueeze(2) == tokens.unsqueeze(1))).any(-1)
            p = torch.where(again, 0.0, p)
            left = (1 - (elder * p.unsqueeze(1)).sum(-1)).clamp(min=0)
            taken = u * left < p
        else:
            mass, past = [torch.ones(state.target.shape[0], dtype=F64, device=DEV)], [torch.zeros(state.target.shape[0], dtype=F64, device=DEV)]
            for _ in range(int(children.max())):                                     # a child that is not taken each
                past.append(past[-1] + mass[-1])
                mass.append(_rest(state, slice(None), past[-1]).sum(-1))
            mass, past, rank = torch.stack(mass, 1), torch.stack(past, 1), elder.sum(-1)
            q = state.draft[above, tokens].double()
            taken = u * mass[above, rank] * q < (p - past[above, rank] * q).clamp(min=0)
    good = (taken & (parents >= 0) & ~(elder & taken.unsqueeze(1)).any(-1)) | (at == 0)
    stands = there & ~(_lines(parents) & ~good.unsqueeze(1)).any(-1)
    count = stands.sum(1)
    last = (stands * at).amax(1)
    row = rows.gather(1, last[:, None])[:, 0]
    if form == "match":
        after = state.target.long()[row]
    else:
        if form == "given":
            mine = (parents == last[:, None]) & there
            rest = torch.cat((state.target[row].double(), torch.zeros_like(u[:, :1])), 1)
            rest = rest.scatter_(1, torch.where(mine, tokens, rest.shape[1] - 1), 0.0)[:, :-1]
        else:
            rest = _rest(state, row, past[row, children.gather(1, last[:, None])[:, 0]])
        rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, state.target[row].double())
        run_sum = rest.cumsum(-1)
        after = (run_sum <= u[:, :1] * run_sum[:, -1:]).sum(-1)
        final = rest.shape[1] - 1 - (rest.flip(1) > 0).to(torch.uint8).argmax(1)
        after = torch.minimum(after, final)
    place = torch.where(stands, stands.cumsum(1) - 1, n)
    path = torch.full((inp.num_seqs, n + 1), -1, dtype=torch.long, device=DEV).scatter_(1, place, at.expand_as(place))[:, :n]
    out = torch.where(path >= 0, tokens.gather(1, path.clamp(min=0)), -1).roll(-1, 1)
    out = torch.where(at < count[:, None] - 1, out, torch.where(at == count[:, None] - 1, after[:, None], -1))
    return out[there].to(torch.int32), path[there].to(torch.int32), count.to(torch.int32)


def _rest(state, rows, past):
    """max(p - past q, 0) of these rows, in 64 bits."""
    return (state.target[rows].double() - past[:, None] * state.draft[rows].double()).clamp_(min=0)


def _keep(state):
    inp = state.inp
    rows, there = _nodes(inp)
    step = torch.arange(inp.max_q_len, device=DEV)
    ctx = (inp.seq_lens - there.sum(1)).long()[:, None]
    move = there & (step < state.count[:, None])
    seq = torch.arange(inp.num_seqs, device=DEV)[:, None].expand_as(rows)[move]
    old, new = (ctx + state.path.long()[rows])[move], (ctx + step)[move]
    (old_page, old_row), (new_page, new_row) = ((inp.block_table[seq, torch.div(x, PAGE, rounding_mode="floor")].long(), x % PAGE)
                                                for x in (old, new))
    for cache in (*state.caches[0], *state.caches[1]):
        cache[new_page, :, :, new_row] = cache[old_page, :, :, old_row]
    return state.held


# ------------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "plan":
        return None
    s = prepare(case, seed)
    start = s.inp.query_start_loc.tolist()
    if case["kind"] == "attend":
        return _exact_attend(s, start)
    if case["kind"] == "keep":      # bits that move: bf16 values are the same in 64
        if s.held.numel() > 1e9:
            return None
        moves = []
        path, count, table, lens = s.path.tolist(), s.count.tolist(), s.inp.block_table.tolist(), s.inp.seq_lens.tolist()
        for i, (a, b) in enumerate(zip(start, start[1:])):
            ctx = lens[i] - (b - a)
            for j in range(count[i]):
                moves.append([(table[i][k // PAGE], k % PAGE) for k in (ctx + path[a + j], ctx + j)])
        at = torch.tensor(moves, device=DEV)
        out = s.held.double()
        out[:, :, at[:, 1, 0], :, :, at[:, 1, 1]] = s.held[:, :, at[:, 0, 0], :, :, at[:, 0, 1]].double()
        return out
    return _exact_verify(s, start)


def _exact_attend(s, start):
    c, inp = s.case, s.inp
    d, hkv, g = c["dim"], c["hkv"], c["hq"] // c["hkv"]
    lens, parents = inp.seq_lens.tolist(), s.parents.tolist()
    if sum(n * (b - a) for n, a, b in zip(lens, start, start[1:])) * c["hq"] * d > 3e13:
        return None
    out = torch.empty(s.q.shape[0], c["hq"], d, dtype=F64, device=DEV)
    for i, (a, b) in enumerate(zip(start, start[1:])):
        n, ctx = lens[i], lens[i] - (b - a)
        hide = torch.full((b - a, n), -math.inf, dtype=F64)
        hide[:, :ctx] = 0
        for k in range(b - a):
            j = k
            while j >= 0:
                hide[k, ctx + j] = 0
                j = parents[a + j]
        hide = hide.to(DEV)
        pages = inp.block_table[i, : -(-n // PAGE)].long()
        for h in range(hkv):
            k, v = (x[pages, h].transpose(1, 2).reshape(-1, d)[:n].double() for x in s.caches)
            q = s.q[a:b].view(b - a, hkv, g, d)[:, h].double()
            z = torch.einsum("qgd,kd->gqk", q, k) / math.sqrt(d) + hide
            out[a:b, h * g:(h + 1) * g] = torch.einsum("gqk,kd->qgd", z.softmax(-1), v)
    return out.flatten(1)


def _exact_verify(s, start):
    tokens, parents = s.tokens.tolist(), s.parents.tolist()
    words, paths, counts = [], [], []
    for a, b in zip(start, start[1:]):
        node, path, said = 0, [0], []
        while True:
            children = [i for i in range(1, b - a) if parents[a + i] == node]
            if s.case["form"] == "match":
                after = int(s.target[a + node])
                step = next((i for i in children if tokens[a + i] == after), None)
            else:
                p = s.target[a + node].double()
                rest, mass, step = p.clone(), 1.0, None
                for i in children:
                    x = tokens[a + i]
                    q = torch.zeros_like(p).index_fill_(0, torch.tensor([x], device=DEV), 1.0) if s.draft is None else s.draft[a + node].double()
                    if float(s.uniform[a + i]) * mass * float(q[x]) < float(rest[x]):
                        step = i
                        break
                    if s.draft is None:
                        mass, rest = max(mass - float(rest[x]), 0.0), rest * (1 - q)
                    else:
                        rest = (rest - mass * q).clamp(min=0)
                        mass = float(rest.sum())
                if step is None:
                    rest = rest if float(rest.sum()) > 0 else p
                    after = int(torch.searchsorted(rest.cumsum(0), float(s.uniform[a]) * rest.sum(), right=True))
                    after = min(after, int(rest.nonzero().max()))
            if step is None:
                break
            path.append(step)
            said.append(tokens[a + step])
            node = step
        counts.append(len(path))
        free = [-1] * (b - a - len(path))
        words += said + [after] + free
        paths += path + free
    return tuple(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (words, paths, counts))
