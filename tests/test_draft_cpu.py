"""Operators for drafted tokens on the CPU: the plain forms against the definitions in 64 bits, and what is refused."""
import types

import pytest
import torch

from gllm_b200.layers import functional as Fn
from gllm_b200.ops import draft as D, kv4
from gllm_b200.ops.ref import kv_cache_shape
from tests import draft_util as U

BF16 = torch.bfloat16
I32 = torch.int32


def _i32(x):
    return torch.tensor(x, dtype=I32)


@pytest.mark.parametrize("ctx,nodes,page,reach", [([0], [1], 16, 1), ([5, 0, 31], [8, 0, 3], 16, 3), ([100, 7], [64, 33], 8, 9), ([63], [64], 32, 1)])
def test_plan(ctx, nodes, page, reach):
    b = U.batch(ctx, nodes, page, "cpu")
    up = U.trees(nodes, reach)
    got = Fn.draft_plan(_i32(up + [3, 4]), b, page)            # two rows behind the last sequence
    for x, y in zip(got, U.plan(up, b, len(up) + 2)):
        assert x.dtype == y.dtype and torch.equal(x, y)


def test_plan_of_parents_that_are_none():
    b = U.batch([4], [5], 16, "cpu")
    up = [-1, 3, 1, -9, 4]                                      # behind the node, itself, no node
    seen, pos, _ = Fn.draft_plan(_i32(up), b, 16)
    assert seen.tolist() == [1, 2, 6, 8, 16] and pos.tolist() == [4, 4, 5, 4, 4]


@pytest.mark.parametrize("dim,hq,hkv,dtype", [(64, 4, 2, BF16), (128, 3, 3, torch.float32), (32, 8, 1, BF16)])
def test_attention(dim, hq, hkv, dtype):
    torch.manual_seed(0)
    b = U.batch([21, 0, 3], [6, 0, 9], 8, "cpu")
    up = U.trees(b.nodes, 3)
    seen = Fn.draft_plan(_i32(up), b, 8)[0]
    seen[7] = 0                                                 # sees the context alone
    k, v = (torch.randn(kv_cache_shape(b.pages, hkv, dim, 8)).to(dtype) for _ in range(2))
    q = torch.randn(len(up) + 2, hq * dim + 8).to(dtype)
    out = torch.full((len(up) + 2, hq * dim), 7.0, dtype=dtype)
    got = Fn.draft_attention(q, k, v, b, torch.cat((seen, seen[:2])), dim ** -0.5, hq, dim, out=out)
    want, tol = U.attention(q[: len(up)], k, v, b, U.sees(seen, b), dim ** -0.5, hq)
    assert got is out and ((got[: len(up)].double().view(-1, hq, dim) - want).abs() <= tol).all() and (got[len(up):] == 7).all()


def test_attention_of_rows_that_see_nothing_or_no_numbers():
    torch.manual_seed(1)
    b = U.batch([0], [4], 16, "cpu")
    k, v = (torch.randn(kv_cache_shape(b.pages, 2, 64, 16)).to(BF16) for _ in range(2))
    v[b.block_table[0, 0], 0, 0, 2, 5], k[b.block_table[0, 0], 1, 0, 2] = float("inf"), float("nan")
    q = torch.randn(4, 128).to(BF16)
    out = Fn.draft_attention(q, k, v, b, torch.tensor([1, 3, 7, 0]), 0.125, 2, 64).view(4, 2, 64)
    assert torch.isfinite(out[:2]).all() and (out[3] == 0).all()
    assert out[2, 0, 5] == float("inf") and torch.isnan(out[2, 1]).all()


@pytest.mark.parametrize("form", ["match", "given", "draws"])
@pytest.mark.parametrize("nodes,reach,vocab", [([1], 1, 5), ([5, 0, 9], 1, 11), ([16, 30], 6, 40), ([64], 12, 3), ([4, 2], 3, 1)])
def test_verify(form, nodes, reach, vocab):
    for seed in range(4):
        b = U.batch([3] * len(nodes), nodes, 16, "cpu")
        up = U.trees(nodes, reach, seed)
        tok, target, draft, u = U.drafts(nodes, up, vocab, form, "cpu", seed)
        pad = torch.tensor([1, 1], dtype=I32)
        want = U.verify(tok, _i32(up), b, target, draft, u)
        got = Fn.draft_verify(tok, _i32(up), b, target, draft, u)
        for x, y in zip(got, want):
            assert x.dtype == I32 and torch.equal(x, y)
        # rows behind the last sequence
        more = [None if x is None else torch.cat((x, x[:1].expand(2, *x.shape[1:]))) for x in (target, draft, u)]
        got = Fn.draft_verify(torch.cat((tok, pad)), torch.cat((_i32(up), pad)), b, *more)
        assert torch.equal(got[0][:-2], want[0]) and got[0][-2:].tolist() == got[1][-2:].tolist() == [-1, -1]


@pytest.mark.parametrize("form,ups", [("draws", [-1, 0, 0, 0]), ("draws", [-1, 0, 1]), ("given", [-1, 0, 0]), ("draws", [-1, 0, 1, 0, 3])])
def test_verify_keeps_the_targets_distribution(form, ups):
    """What a sequence says first is distributed as the target's row: 6000 draws, five standard deviations of a share at most."""
    gen = torch.Generator().manual_seed(5)
    n, draws = len(ups), 6000
    p, q = (torch.rand(n, 4, generator=gen).add_(0.05) for _ in range(2))
    p, q = p / p.sum(1, keepdim=True), q / q.sum(1, keepdim=True)
    b = U.batch([3] * draws, [n] * draws, 16, "cpu")
    above = torch.tensor([max(x, 0) for x in ups])
    tok = torch.multinomial(q[above], draws, replacement=True, generator=gen).t().reshape(-1).to(I32)
    if form == "given":                                         # the same two guesses each time
        tok = torch.tensor([0, 2, 1]).repeat(draws).to(I32)
    u = torch.rand(n * draws, generator=gen)
    said = Fn.draft_verify(tok, _i32(ups * draws), b, p.repeat(draws, 1), q.repeat(draws, 1) if form == "draws" else None, u)[0]
    share = torch.bincount(said.view(draws, n)[:, 0].long(), minlength=4) / draws
    assert ((share - p[0]).abs() <= 5 * (p[0] * (1 - p[0]) / draws).sqrt()).all()


def test_verify_without_mass():
    b = U.batch([0], [2], 16, "cpu")
    z, u = torch.zeros(2, 4), torch.tensor([0.5, 0.0])
    for target in (z, torch.full((2, 4), float("nan")), torch.full((2, 4), -1.0)):
        assert Fn.draft_verify(_i32([1, 2]), _i32([-1, 0]), b, target, None, u)[0].tolist() == [0, -1]
    same = torch.tensor([[0.25, 0.5, 0.25, 0.0]] * 2)           # token 3 has no mass; nothing of p is over q: p itself
    assert Fn.draft_verify(_i32([1, 3]), _i32([-1, 0]), b, same, same, u)[0].tolist() == [1, -1]
    assert Fn.draft_verify(_i32([1, -5]), _i32([-1, 0]), b, same, None, u)[0].tolist() == [1, -1]


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (torch.float32, 128), (BF16, 32)])
def test_keep(dtype, dim):
    torch.manual_seed(2)
    b = U.batch([21, 0, 3, 40], [6, 0, 9, 1], 8, "cpu")
    path, count = U.paths(b.nodes, 0.5, "cpu")
    ks = [torch.randn(kv_cache_shape(b.pages, 2, dim, 8)).to(dtype) for _ in range(3)]
    vs = [torch.randn(kv_cache_shape(b.pages, 3, 64, 8)).to(dtype) for _ in range(2)]
    want = U.kept(ks + vs, b, path, count)
    Fn.draft_keep([ks[0], None, ks[1], ks[0], ks[2]], vs, b, path, count)      # a layer without, one that shares
    for x, y in zip(ks + vs, want):
        assert torch.equal(x, y)
    Fn.draft_keep(ks, [], b, path, count)                       # latent caches have no values


def _args(b, **over):
    torch.manual_seed(0)
    t = b.num_tokens
    a = dict(q=torch.randn(t, 256).to(BF16), k_cache=torch.randn(kv_cache_shape(b.pages, 2, 64, 16)).to(BF16), inp=b,
             v_cache=torch.randn(kv_cache_shape(b.pages, 2, 64, 16)).to(BF16), seen=torch.ones(t, dtype=torch.int64), scale=0.1,
             num_q_heads=4, head_dim=64)
    a.update(over)
    return a


def test_attention_refuses():
    b = U.batch([20], [3], 16, "cpu")
    ok = _args(b)
    Fn.draft_attention(**ok)
    four = torch.zeros(kv4.cache_shape(4, 2, 64, 16), dtype=torch.uint8)
    bad = [dict(k_cache=four, v_cache=four), dict(k_cache=ok["k_cache"].float()), dict(q=ok["q"].float()), dict(v_cache=ok["v_cache"][:1]),
           dict(k_cache=ok["k_cache"][..., ::2]), dict(k_cache=ok["k_cache"][:0], v_cache=ok["v_cache"][:0]), dict(num_q_heads=3), dict(head_dim=128), dict(q=ok["q"][:, :128]), dict(seen=ok["seen"].to(I32)),
           dict(seen=ok["seen"][:2]), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
           dict(out=torch.zeros(3, 256)), dict(out=torch.zeros(2, 256, dtype=BF16)), dict(out=torch.zeros(3, 512, dtype=BF16)[:, ::2])]
    for over in bad:
        with pytest.raises(ValueError):
            Fn.draft_attention(**{**ok, **over})


@pytest.mark.parametrize("name,value", [("max_q_len", 65), ("query_start_loc", torch.zeros(2, dtype=torch.int64)), ("query_start_loc", _i32([0])),
                                        ("seq_lens", torch.zeros(0, dtype=I32)), ("block_table", _i32([1, 2])), ("block_table", torch.zeros(1, 4)),
                                        ("seq_lens", None), ("block_table", torch.zeros(1, 8, dtype=I32)[:, ::2])])
def test_batches_are_refused(name, value):
    b = U.batch([20], [3], 16, "cpu")
    setattr(b, name, value)
    path, count = _i32([0, 1, 2]), _i32([3])
    with pytest.raises(ValueError):
        Fn.draft_plan(_i32([-1, 0, 1]), b, 16)
    with pytest.raises(ValueError):
        Fn.draft_attention(**_args(types.SimpleNamespace(**{**vars(U.batch([20], [3], 16, "cpu")), name: value})))
    with pytest.raises(ValueError):
        Fn.draft_keep([], [], b, path, count)
    if name in ("max_q_len", "query_start_loc"):
        with pytest.raises(ValueError):
            Fn.draft_verify(_i32([0, 1, 2]), _i32([-1, 0, 1]), b, _i32([0, 1, 2]))


def test_verify_and_keep_refuse():
    b = U.batch([20], [3], 16, "cpu")
    tok, up, p, u = _i32([0, 1, 2]), _i32([-1, 0, 1]), torch.rand(3, 8), torch.rand(3)
    Fn.draft_verify(tok, up, b, p, p, u)
    for args in [(tok.long(), up, b, p, p, u), (tok, up[:2], b, p, p, u), (tok, up, b, p.double(), None, u), (tok, up, b, p, p.half(), u),
                 (tok, up, b, p[:2], None, u), (tok, up, b, p, p[:, :7], u), (tok, up, b, p, p, None), (tok, up, b, p, p, u.double()),
                 (tok, up, b, p, p, u[:2]), (tok, up, b, p[:, ::2], None, u), (tok, up, b, p[:, :0], None, u), (tok, up, b, tok, p, u),
                 (tok, up, b, tok, None, u), (tok, up, b, tok.long()), (tok, up, b, p[0], None, u)]:
        with pytest.raises(ValueError):
            Fn.draft_verify(*args)
    c = torch.zeros(kv_cache_shape(4, 2, 64, 16), dtype=BF16)
    path, count = _i32([0, 1, 2]), _i32([3])
    four = torch.zeros(kv4.cache_shape(4, 2, 64, 16), dtype=torch.uint8)
    for args in [([four], [four], b, path, count), ([c.transpose(1, 3)], [], b, path, count), ([c[0]], [], b, path, count),
                 ([torch.zeros(kv_cache_shape(4, 2, 4, 16), dtype=BF16)], [], b, path, count), ([c], [c], b, path.long(), count),
                 ([c], [c], b, path, count[:0])]:
        with pytest.raises(ValueError):
            Fn.draft_keep(*args)


def test_plan_refuses():
    b = U.batch([20], [3], 16, "cpu")
    for up, page in [(torch.tensor([-1, 0, 1]), 16), (_i32([[-1, 0, 1]]), 16), (_i32([-1, 0, 0, 0, 1])[::2], 16), (_i32([-1, 0, 1]), 0)]:
        with pytest.raises(ValueError):
            Fn.draft_plan(up, b, page)


def test_64_nodes_at_most_and_names_of_limits():
    assert D.MOST_NODES == 64
    b = U.batch([20], [64], 16, "cpu")
    seen = Fn.draft_plan(_i32(list(range(-1, 63))), b, 16)[0]
    assert seen[-1] == -1 and seen[0] == 1                       # the last of a chain sees every node: all 64 bits


@pytest.mark.parametrize("seqs", [1, 18, 37, 74, 111, 148, 300])
@pytest.mark.parametrize("nodes,group", [(1, 1), (8, 4), (24, 4), (64, 8)])
def test_long_units_of_attention_are_cut_however_many_there_are(seqs, nodes, group):
    """One long context beside short ones: what counts is how long it may be, not whether the units go evenly into the SMs."""
    from gllm_b200.ops import sm100_draft
    for length in (32 * 128, 60000, 1 << 20):
        assert not sm100_draft._whole_units(seqs, 8, group, nodes, length)
    assert sm100_draft._whole_units(seqs, 8, group, nodes, 600)


def test_attention_of_tables_that_end():
    torch.manual_seed(4)
    b = U.batch([14, 0, 24, 5], [8, 20, 3, 7], 16, "cpu")
    b.block_table = b.block_table[:, :1]
    seen = Fn.draft_plan(_i32(U.trees(b.nodes, 3)), b, 16)[0]
    k, v = (torch.randn(kv_cache_shape(b.pages, 2, 64, 16)).to(BF16) for _ in range(2))
    q = torch.randn(38, 256).to(BF16)
    got = Fn.draft_attention(q, k, v, b, seen, 0.125, 4, 64).double().view(38, 4, 64)
    want, tol = U.attention(q, k, v, b, [m[:, :16] for m in U.sees(seen.tolist(), b)], 0.125, 4)
    assert ((got - want).abs() <= tol).all()
