"""64-bit definitions of the operators for drafted tokens, and batches for their tests."""
import math
import types

import torch

BF16, F64 = torch.bfloat16, torch.float64


def batch(ctx, nodes, page, device, seed=0, spare=2, pad_seqs=0):
    """A step's description: contexts and nodes of each sequence, pages in random order; the table's entries behind a sequence's are no pages."""
    gen = torch.Generator().manual_seed(seed)
    blocks = [-(-(c + n) // page) for c, n in zip(ctx, nodes)]
    pages = sum(blocks) + spare
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(ctx), max([*blocks, 1]) + 1), -7, dtype=torch.int32)
    at = 0
    for s, b in enumerate(blocks):
        table[s, :b] = order[at:at + b]
        at += b
    start = torch.tensor([0, *nodes]).cumsum(0).to(torch.int32)
    return types.SimpleNamespace(block_table=table.to(device), seq_lens=torch.tensor([c + n for c, n in zip(ctx, nodes)], dtype=torch.int32, device=device),
                                 query_start_loc=start.to(device), num_seqs=len(ctx), num_tokens=sum(nodes), max_q_len=max([*nodes, 0]),
                                 max_seq_len=max(c + n for c, n in zip(ctx, nodes)), padded_tokens=0, num_decode_seqs=0, pages=pages,
                                 ctx=list(ctx), nodes=list(nodes), page=page)


def trees(nodes, reach, seed=0):
    """Parents [T] (list): one of the `reach` nodes before each."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for n in nodes:
        out += [-1 if i == 0 else i - 1 - int(torch.randint(0, min(i, reach), (1,), generator=gen)) for i in range(n)]
    return out


def line(parents, first, i):
    """Node i and its ancestors."""
    out = []
    while i >= 0:
        out.append(i)
        p = parents[first + i]
        i = p if 0 <= p < i else -1
    return out


def plan(parents, b, rows):
    seen, pos, slots = [0] * rows, [0] * rows, [-1] * rows
    table, at = b.block_table.tolist(), 0
    for s, (c, n) in enumerate(zip(b.ctx, b.nodes)):
        for i in range(n):
            up = line(parents, at, i)
            word = sum(1 << j for j in up)
            seen[at + i] = word - (1 << 64) if word >> 63 else word
            pos[at + i] = c + len(up) - 1
            slots[at + i] = table[s][(c + i) // b.page] * b.page + (c + i) % b.page
        at += n
    return torch.tensor(seen), torch.tensor(pos, dtype=torch.int32), torch.tensor(slots, dtype=torch.int32)


def sees(seen, b):
    """[nodes, keys] for each sequence, from the words."""
    out, at = [], 0
    for c, n in zip(b.ctx, b.nodes):
        m = torch.zeros(n, c + n, dtype=torch.bool)
        m[:, :c] = True
        for i in range(n):
            w = int(seen[at + i])
            for j in range(n):
                m[i, c + j] = bool((w >> j) & 1)
        out.append(m)
        at += n
    return out


def rows_of(cache, b, s):
    """[keys, heads, D] of sequence s, fp64."""
    n = b.ctx[s] + b.nodes[s]
    blk = cache[b.block_table[s, : -(-n // b.page)].long()].permute(0, 3, 1, 2, 4)
    return blk.reshape(-1, cache.shape[1], cache.shape[2] * cache.shape[4])[:n].to(F64)


def attention(q, k_cache, v_cache, b, masks, scale, hq):
    """(result, tolerance) [T, Hq, D], fp64.

    Roundings of the kernels: the result once to bf16 (2^-8 of it), probabilities once to bf16 (2^-8 of sum p |v|). Scores are fp32 sums of
    products that fp32 holds exactly: at most 2 D roundings of 2^-24 of the largest partial sum, which is below sum |q k|: with D = 128 2^-16 of
    scale sum |q k| in the exponent at the very worst; the sums of probabilities and results are fp32 too (2^-24 a step, 2^-16 for 256 steps
    of the longest chains of additions here), and the exponential is good to 2^-22."""
    out, tol, at = [], [], 0
    d = k_cache.shape[2] * k_cache.shape[4]
    g = hq // k_cache.shape[1]
    for s, (c, n) in enumerate(zip(b.ctx, b.nodes)):
        qq = q[at:at + n, : hq * d].reshape(n, hq, d).to(F64)
        at += n
        k, v = (rows_of(x, b, s).repeat_interleave(g, 1) for x in (k_cache, v_cache))
        m = masks[s].to(q.device)
        if not n:
            continue
        z = torch.einsum("qhd,khd->hqk", qq, k) * scale
        z = torch.where(m, z, -math.inf)
        p = torch.where(m.any(-1)[:, None], z.softmax(-1), 0.0)
        size = torch.einsum("qhd,khd->hqk", qq.abs(), k.abs()).nan_to_num(0.0, 0.0, 0.0) * scale
        err = 2.0 ** -8 + 2.0 ** -15 + 2.0 ** -15 * torch.where(m, size, 0.0).amax(-1)
        # what a row does not see is not in it, whatever it is
        term = torch.where(m[None, :, :, None], p[..., None] * v.permute(1, 0, 2)[:, None], 0.0)
        o = term.sum(2).permute(1, 0, 2)
        out.append(o)
        tol.append((err[..., None] * term.abs().sum(2)).permute(1, 0, 2) + 2.0 ** -8 * o.abs() + 1e-30)
    return torch.cat(out), torch.cat(tol)


def verify(tokens, parents, b, target, draft=None, uniform=None):
    said, ways, counts, first = [], [], [], 0
    tok = tokens.tolist()
    up = parents.tolist()
    u = None if uniform is None else [float(x) for x in uniform]
    for n in b.nodes:
        if n == 0:
            counts.append(0)
            continue
        way = [0]
        while True:
            c = way[-1]
            kids = [i for i in range(c + 1, n) if up[first + i] == c]
            nxt = None
            if u is None:
                last = int(target[first + c])
                for i in kids:
                    if tok[first + i] == last:
                        nxt = i
                        break
            else:
                p = target[first + c].to(F64)
                v = p.shape[0]
                q = None if draft is None else draft[first + c].to(F64)
                r, mass, off = torch.where(p > 0, p, 0.0), 1.0, 0.0
                for i in kids:
                    x = tok[first + i]
                    ok = 0 <= x < v
                    have = float(r[x]) if ok else 0.0
                    if u[first + i] * mass * (1.0 if q is None or not ok else float(q[x])) < have:
                        nxt = i
                        break
                    if q is None:
                        mass = max(mass - have, 0.0)
                        if ok:
                            r = r.clone()
                            r[x] = 0.0
                    else:
                        off = off + mass
                        r = p - off * q
                        r = torch.where(r > 0, r, 0.0)
                        mass = float(r.sum())
                if nxt is None:
                    if not float(r.sum()) > 0:
                        r = torch.where(p > 0, p, 0.0)
                    run = r.cumsum(0)
                    if not float(run[-1]) > 0:
                        last = 0
                    else:
                        hit = (run > u[first] * run[-1]).nonzero()
                        last = int(hit[0]) if len(hit) else int(r.nonzero()[-1])
            if nxt is None:
                break
            way.append(nxt)
        said += [tok[first + i] for i in way[1:]] + [last] + [-1] * (n - len(way))
        ways += way + [-1] * (n - len(way))
        counts.append(len(way))
        first += n
    return [torch.tensor(x, dtype=torch.int32, device=tokens.device) for x in (said, ways, counts)]


def drafts(nodes, parents, vocab, form, device, seed=0, sharp=2.0):
    """Tokens of the nodes, target, draft probabilities and random numbers of a form of verification."""
    gen = torch.Generator(device=device).manual_seed(seed)
    t = sum(nodes)
    first = [sum(nodes[:s]) for s, n in enumerate(nodes) for _ in range(n)]
    above = torch.tensor([f + max(p, 0) for f, p in zip(first, parents)], device=device, dtype=torch.long)
    i32 = dict(dtype=torch.int32, device=device)
    if form == "match":
        target = torch.randint(0, vocab, (t,), generator=gen, **i32)
        tokens = torch.where(torch.rand(t, generator=gen, device=device) < 0.6, target[above], torch.randint(0, vocab, (t,), generator=gen, **i32))
        return tokens, target, None, None
    z = torch.randn(t, vocab, generator=gen, device=device) * sharp
    target = z.softmax(-1)
    draft = (z + torch.randn(t, vocab, generator=gen, device=device)).softmax(-1) if form == "draws" else None
    tokens = torch.multinomial((target if draft is None else draft)[above], 1, generator=gen)[:, 0].to(torch.int32)
    return tokens, target, draft, torch.rand(t, generator=gen, device=device)


def kept(caches, b, path, count):
    """The caches after the moves, new tensors."""
    way, taken, table = path.tolist(), count.tolist(), b.block_table.tolist()
    out = [c.clone() for c in caches]
    at = 0
    for s, (c, n) in enumerate(zip(b.ctx, b.nodes)):
        for j in range(taken[s]):
            a, z = c + way[at + j], c + j
            for x, y in zip(caches, out):
                y[table[s][z // b.page], :, :, z % b.page] = x[table[s][a // b.page], :, :, a % b.page]
        at += n
    return out


def paths(nodes, share, device, seed=0):
    """Ascending paths from node 0 on: (path [T], count [sequences])."""
    gen = torch.Generator().manual_seed(seed)
    path, count = [], []
    for n in nodes:
        way = [i for i in range(n) if i == 0 or float(torch.rand((), generator=gen)) < share]
        path += way + [-1] * (n - len(way))
        count.append(len(way))
    i32 = dict(dtype=torch.int32, device=device)
    return torch.tensor(path, **i32), torch.tensor(count, **i32)
