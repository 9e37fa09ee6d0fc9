"""Kernels for drafted tokens against the definitions in 64 bits (GPU)."""
import time
import types

import pytest
import torch

from gllm_b200.layers import functional as Fn
from gllm_b200.ops import lib, ref, sm100, sm100_draft
from gllm_b200.ops.ref import kv_cache_shape
from tests import draft_util as U

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


# -- plan -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("ctx,nodes,page,reach", [
    ([0], [1], 16, 1), ([700], [8], 16, 3), ([5, 0, 31, 2], [8, 0, 3, 1], 16, 3), ([100, 7, 0], [64, 33, 64], 8, 9), ([63, 1], [64, 64], 128, 1),
    ([3 * i for i in range(300)], [i % 7 for i in range(300)], 16, 2)])
def test_plan(ctx, nodes, page, reach):
    b = U.batch(ctx, nodes, page, DEV)
    up = U.trees(nodes, reach)
    got = Fn.draft_plan(_i32(up + [3] * 70), b, page)
    for x, y in zip(got, U.plan(up, b, len(up) + 70)):
        assert x.dtype == y.dtype and torch.equal(x.cpu(), y)


def test_plan_of_parents_that_are_none_and_tables_that_end():
    b = U.batch([4, 30], [5, 3], 16, DEV)
    b.block_table = b.block_table[:, :2]
    seen, pos, slots = Fn.draft_plan(_i32([-1, 3, 1, -9, 4, -1, 0, 7]), b, 16)
    assert seen.tolist() == [1, 2, 6, 8, 16, 1, 3, 4] and pos.tolist() == [4, 4, 5, 4, 4, 30, 31, 30]
    last = int(b.block_table[1, 1]) * 16
    assert slots.tolist()[5:] == [last + 14, last + 15, -1]
    assert Fn.draft_plan(_i32([]), U.batch([3], [0], 16, DEV), 16)[0].shape == (0,)


# -- attention ------------------------------------------------------------------------------------------------------------
def _attention_case(ctx, nodes, hq, hkv, d, page, reach=4, extra=0, seed=0, size=1.0):
    """Caches whose rows outside of the sequences are no numbers."""
    torch.manual_seed(seed + sum(ctx) + d)
    b = U.batch(ctx, nodes, page, DEV, seed)
    shape = kv_cache_shape(b.pages, hkv, d, page)
    caches = [torch.full(shape, float("nan"), dtype=BF16, device=DEV) for _ in range(2)]
    for s, (c, n) in enumerate(zip(ctx, nodes)):
        at = torch.arange(c + n, device=DEV)
        for x in caches:
            x[b.block_table[s][at // page].long(), :, :, at % page] = torch.randn(c + n, hkv, d // 64, 64, device=DEV).mul_(size).to(BF16)
    q = (torch.randn(sum(nodes) + 3, hq * d + extra, device=DEV) * size).to(BF16)[:, extra:]
    up = U.trees(nodes, reach, seed)
    seen = Fn.draft_plan(_i32(up + [-1] * 3), b, page)[0]
    return types.SimpleNamespace(b=b, k=caches[0], v=caches[1], q=q, up=up, seen=seen, hq=hq, d=d)


def _check_attention(x, scale=None, masks=None):
    t = x.b.num_tokens
    scale = scale or x.d ** -0.5
    out = torch.full((t + 3, x.hq * x.d), 5.0, dtype=BF16, device=DEV)
    got = Fn.draft_attention(x.q, x.k, x.v, x.b, x.seen, scale, x.hq, x.d, out=out)
    assert got is out and (out[t:] == 5).all()
    if t == 0:
        return out
    want, tol = U.attention(x.q[:t], x.k, x.v, x.b, masks or U.sees(x.seen.tolist(), x.b), scale, x.hq)
    off = (out[:t].double().view(-1, x.hq, x.d) - want).abs()
    assert (off <= tol).all(), (off - tol).max()
    return out


@pytest.mark.parametrize("ctx,nodes,hq,hkv,d,page,extra", [
    ([0], [1], 1, 1, 64, 16, 0), ([0], [64], 4, 2, 128, 16, 8), ([127], [1], 4, 1, 128, 16, 0), ([128], [1], 32, 8, 128, 16, 0),
    ([100], [64], 8, 1, 64, 8, 0), ([120, 64, 0], [16, 64, 5], 7, 1, 128, 16, 8), ([700], [8], 32, 8, 128, 16, 0),
    ([5, 0, 31, 2, 300], [8, 0, 3, 1, 64], 6, 2, 64, 32, 0), ([1000, 3, 517], [13, 64, 2], 14, 2, 64, 64, 0), ([255, 256, 257], [7, 7, 7], 5, 5, 128, 128, 0),
    ([2000], [64], 64, 8, 128, 16, 0), ([1500] * 3, [40, 17, 64], 16, 1, 128, 16, 0), ([33] * 70, [3] * 70, 8, 2, 128, 16, 0),
    ([5000, 1], [26, 26], 32, 4, 128, 16, 0), ([300, 90], [5, 2], 128, 1, 64, 16, 0), ([200, 700], [3, 64], 71, 1, 64, 16, 8), ([260], [40], 100, 2, 128, 32, 0),
    ([500, 2, 1300], [43, 44, 9], 9, 3, 128, 16, 0), ([1000, 200], [22, 64], 12, 2, 128, 16, 8), ([130] * 30, [11] * 30, 6, 1, 64, 16, 0), ([9000], [5], 8, 8, 64, 16, 0), ([4000], [1], 4, 1, 128, 16, 0),
    ([17 * i % 900 for i in range(40)], [1 + i % 20 for i in range(40)], 10, 2, 64, 16, 0)])
def test_attention(ctx, nodes, hq, hkv, d, page, extra):
    _check_attention(_attention_case(ctx, nodes, hq, hkv, d, page, extra=extra))


@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_a_long_context(d):
    _check_attention(_attention_case([40000, 100], [9, 64], 8, 2, d, 16))


@pytest.mark.parametrize("size,scale", [(1.0, 3.0), (1.0, 1e-3), (8.0, None), (0.01, None)])
def test_attention_of_sharp_and_flat_scores(size, scale):
    _check_attention(_attention_case([300, 1200], [20, 9], 8, 2, 128, 16, size=size), scale)


@pytest.mark.parametrize("d,ctx", [(64, 0), (128, 0), (128, 37), (64, 100)])
def test_attention_with_any_words(d, ctx):
    """Words that are no tree: any bits, none, bits behind the last node."""
    x = _attention_case([ctx, 5], [64, 21], 8, 2, d, 16)
    gen = torch.Generator(device=DEV).manual_seed(3)
    x.seen = torch.randint(-2 ** 62, 2 ** 62, x.seen.shape, generator=gen, device=DEV) * 3
    x.seen[3], x.seen[70] = 0, -1
    out = _check_attention(x)
    if ctx == 0:
        assert (out[3] == 0).all()


def test_attention_whatever_lies_in_nodes_that_are_not_seen():
    """Keys and values of one branch are no numbers: the other branch does not notice, those that see them do."""
    for d, ctx in ((128, 0), (128, 120), (64, 300)):
        x = _attention_case([ctx], [40], 8, 2, d, 16, reach=6)
        place = [(int(x.b.block_table[0, (ctx + i) // 16]), (ctx + i) % 16) for i in range(40)]
        seen = x.seen.tolist()
        bad = {7: float("nan"), 11: float("inf"), 18: float("-inf"), 30: float("nan")}
        for i, (what, (page, row)) in enumerate((w, place[n]) for n, w in bad.items()):
            x.v[page, :, :, row, i::5] = what
        x.k[place[30][0], :, :, place[30][1]] = float("nan")
        out = Fn.draft_attention(x.q, x.k, x.v, x.b, x.seen, d ** -0.5, 8, d).view(-1, 8, d // 64, 64)[:40]
        clean = x.v.clone()
        k = x.k.clone()
        for n in bad:
            clean[place[n][0], :, :, place[n][1]] = 0
        k[place[30][0], :, :, place[30][1]] = 0
        want, tol = U.attention(x.q[:40], k, clean, x.b, U.sees(seen, x.b), d ** -0.5, 8)
        want, tol = want.view(out.shape), tol.view(out.shape)
        for i in range(40):
            hit = [n for n in bad if seen[i] >> n & 1]
            if not hit:
                assert ((out[i].double() - want[i]).abs() <= tol[i]).all(), i
            elif 30 in hit:
                assert torch.isnan(out[i]).all()
            else:
                cols = torch.zeros(64, dtype=torch.bool, device=DEV)
                for j, n in enumerate(bad):
                    if n in hit:
                        cols[j::5] = True
                assert torch.isfinite(out[i][..., ~cols]).all() and not torch.isfinite(out[i][..., cols]).any(), i


def test_attention_of_pages_that_do_not_exist():
    """Table entries inside a sequence that are no pages: nothing outside of the cache is read, other sequences are what they were."""
    x = _attention_case([300, 200], [9, 9], 8, 2, 128, 16)
    x.b.block_table[0, 3], x.b.block_table[0, 7] = 10 ** 6, -5
    out = Fn.draft_attention(x.q, x.k, x.v, x.b, x.seen, 0.1, 8, 128)
    want, tol = U.attention(x.q[:18], x.k, x.v, types.SimpleNamespace(**{**vars(x.b), "block_table": x.b.block_table.clamp(0, x.b.pages - 1)}),
                            U.sees(x.seen.tolist(), x.b), 0.1, 8)
    assert ((out[9:18].double().view(-1, 8, 128) - want[9:]).abs() <= tol[9:]).all()
    torch.cuda.synchronize()


def test_attention_is_the_same_twice_and_on_another_stream():
    x = _attention_case([700, 2300, 90], [9, 17, 64], 32, 8, 128, 16)
    a = _check_attention(x)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        b = Fn.draft_attention(x.q, x.k, x.v, x.b, x.seen, 128 ** -0.5, 32, 128)
    other = _attention_case([50] * 20, [30] * 20, 32, 8, 128, 16, seed=4)
    _check_attention(other)                                     # at the same time
    st.synchronize()
    t = x.b.num_tokens
    assert torch.equal(a[:t], b[:t])


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("ctx,nodes,hq,hkv,d", [
    ([9000], [5], 8, 8, 64), ([9000], [5], 8, 8, 128), ([30000], [4], 2, 1, 128), ([3000] * 9, [8] * 9, 32, 8, 128), ([2500, 9000, 40], [12, 3, 7], 8, 2, 64),
    ([9000], [40], 8, 8, 128), ([5000, 700], [50, 64], 2, 2, 64), ([3000] * 9, [15] * 9, 32, 8, 128), ([9000], [32], 16, 4, 128), ([4000] * 5, [24] * 5, 10, 2, 64),
    ([4000] * 5, [18] * 5, 49, 7, 128), ([6000, 300], [64, 40], 16, 4, 128), ([2000] * 8, [33] * 8, 16, 2, 64), ([7000] * 2, [20, 64], 24, 3, 128)])
def test_attention_with_units_cut_and_whole(ctx, nodes, hq, hkv, d, whole, monkeypatch):
    """Shares of several tiles and several units, for every number of lanes a row and for blocks of two halves."""
    from gllm_b200.ops import sm100_draft
    monkeypatch.setattr(sm100_draft, "_whole_units", lambda *a: whole)
    for seed in range(2):
        _check_attention(_attention_case(ctx, nodes, hq, hkv, d, 16, seed=seed))


def test_attention_refuses_on_the_gpu():
    x = _attention_case([50], [3], 4, 2, 64, 16)
    args = dict(q=x.q, k_cache=x.k, v_cache=x.v, inp=x.b, seen=x.seen, scale=0.1, num_q_heads=4, head_dim=64)
    wide = torch.zeros(kv_cache_shape(4, 1, 256, 16), dtype=BF16, device=DEV)
    odd = torch.zeros(kv_cache_shape(4, 2, 64, 24), dtype=BF16, device=DEV)
    many = torch.zeros(6, 129 * 64, dtype=BF16, device=DEV)
    for over in [dict(q=many, k_cache=x.k[:, :1].contiguous(), v_cache=x.v[:, :1].contiguous(), num_q_heads=129), dict(q=torch.zeros(6, 264, dtype=BF16, device=DEV)[:, 1:257]), dict(q=torch.zeros(6, 257, dtype=BF16, device=DEV)[:, :256]),
                 dict(k_cache=odd, v_cache=odd), dict(k_cache=wide, v_cache=wide, num_q_heads=1, head_dim=256), dict(seen=x.seen.cpu()),
                 dict(k_cache=x.k.float(), v_cache=x.v.float(), q=x.q.float())]:
        with pytest.raises(ValueError):
            Fn.draft_attention(**{**args, **over})


# -- verification ---------------------------------------------------------------------------------------------------------
def _same(got, want):
    for x, y in zip(got, want):
        assert x.dtype == I32 and torch.equal(x, y), (x, y)


@pytest.mark.parametrize("form", ["match", "given", "draws"])
@pytest.mark.parametrize("nodes,reach,vocab", [
    ([1], 1, 1), ([5], 1, 2), ([5, 0, 9], 1, 5), ([16, 30, 1], 6, 127), ([64], 12, 1000), ([64, 64], 64, 4099), ([4, 2, 64], 3, 32000),
    ([6] * 40, 1, 8191), ([3, 5], 2, 151936), ([1, 8], 4, 128257)])
def test_verify(form, nodes, reach, vocab):
    for seed in range(3):
        b = U.batch([3] * len(nodes), nodes, 16, DEV)
        up = U.trees(nodes, reach, seed)
        args = U.drafts(nodes, up, vocab, form, DEV, seed, 1 + seed)
        up = _i32(up)
        _same(Fn.draft_verify(args[0], up, b, *args[1:]), U.verify(args[0], up, b, *args[1:]))


@pytest.mark.parametrize("form", ["given", "draws"])
@pytest.mark.parametrize("seqs", [1, 2, 5, 17, 100])
def test_verify_of_more_and_fewer_sequences(form, seqs):
    nodes = [3 + s % 4 for s in range(seqs)]
    b, up = U.batch([3] * seqs, nodes, 16, DEV), U.trees(nodes, 2)
    args = U.drafts(nodes, up, 20011, form, DEV)
    up = _i32(up)
    _same(Fn.draft_verify(args[0], up, b, *args[1:]), U.verify(args[0], up, b, *args[1:]))


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("most", [8, 16, 30, 64])
def test_attention_of_nodes_that_are_no_numbers_in_every_form(most, d, whole, monkeypatch):
    """Rows of four heads: four, two and one lane a row, blocks of 256. Two calls at once give the same bits."""
    monkeypatch.setattr(sm100_draft, "_whole_units", lambda *a: whole)
    ctx, nodes = [0, 120, 127, 900, 250, 3], [most, 1, most, most // 2 + 1, 0, most]
    x = _attention_case(ctx, nodes, 8, 2, d, 16)
    seen, bad, first = x.seen.tolist(), {}, [sum(nodes[:s]) for s in range(len(nodes))]
    gen = torch.Generator().manual_seed(most)
    for s, n in enumerate(nodes):
        for i in (torch.rand(n, generator=gen) < 0.2).nonzero()[:, 0].tolist():
            what = (float("nan"), float("inf"), float("-inf"))[i % 3]
            x.v[int(x.b.block_table[s, (ctx[s] + i) // 16]), :, :, (ctx[s] + i) % 16, i % 7::7] = what
            bad[s, i] = torch.arange(d, device=DEV) % 64 % 7 == i % 7
    got = []
    torch.cuda.synchronize()
    for stream in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            got.append(Fn.draft_attention(x.q, x.k, x.v, x.b, x.seen, d ** -0.5, 8, d)[:x.b.num_tokens])
    torch.cuda.synchronize()
    assert torch.equal(got[0].view(torch.int16), got[1].view(torch.int16))
    want, tol = U.attention(x.q[:x.b.num_tokens], x.k, torch.where(x.v.isfinite(), x.v, 0), x.b, U.sees(seen, x.b), d ** -0.5, 8)
    out = got[0].double().view(-1, 8, d)
    fits = (out - want).abs() <= tol
    for (s, i), cols in bad.items():
        for row in range(first[s], first[s] + nodes[s]):
            if seen[row] >> i & 1:
                fits[row][:, cols] = ~out[row][:, cols].isfinite()
    assert bad and fits.all()


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("most", [8, 16, 30, 64])
def test_attention_whose_waits_run_out(most, d, whole, monkeypatch):
    """Limits of nothing, 1 ns and 2 us: the roles give up at different places, nothing is waited for that was never issued (two seconds), the
    host learns of it, and the next call is right again."""
    monkeypatch.setattr(sm100_draft, "_whole_units", lambda *a: whole)
    x = _attention_case([700, 90, 5, 3000], [most, 3, most, most], 8, 2, d, 16)
    want = _check_attention(x)
    assert sm100.waits_given_up() == 0
    try:
        for limit in (0, 1, 2000):
            lib.watch_waits(limit_ns=limit)
            for _ in range(3):
                t0 = time.monotonic()
                Fn.draft_attention(x.q, x.k, x.v, x.b, x.seen, d ** -0.5, 8, d)
                torch.cuda.synchronize()
                assert time.monotonic() - t0 < 0.5, limit
            assert lib.waits_gave_up(clear=True) or limit > 0
    finally:
        lib.watch_waits()
        lib.waits_gave_up(clear=True)
    assert torch.equal(_check_attention(x), want) and sm100.waits_given_up() == 0


@pytest.mark.parametrize("form", ["given", "draws"])
@pytest.mark.parametrize("seqs,vocab", [(1, 65537), (4, 65536), (4, 99991), (5, 99991), (8, 131073), (9, 131073)])
def test_verify_of_long_rows(form, seqs, vocab):
    """Few sequences have larger clusters; the rows' starts lie off the 16-byte boundaries."""
    nodes = [1 + (3 + s) % 5 for s in range(seqs)]
    b, up = U.batch([3] * seqs, nodes, 16, DEV), U.trees(nodes, 2)
    for seed in range(2):
        args = U.drafts(nodes, up, vocab, form, DEV, seed)
        _same(Fn.draft_verify(args[0], _i32(up), b, *args[1:]), U.verify(args[0], _i32(up), b, *args[1:]))


@pytest.mark.parametrize("shift_p,shift_q", [(0, 0), (1, 1), (1, 3), (2, 0), (3, 2)])
@pytest.mark.parametrize("vocab", [3, 1001])
def test_verify_of_views(vocab, shift_p, shift_q):
    nodes = [7, 3, 12]
    b, up = U.batch([3] * 3, nodes, 16, DEV), U.trees(nodes, 3)
    tok, p, q, u = U.drafts(nodes, up, vocab, "draws", DEV)
    wide_p, wide_q = torch.full((22, vocab + 5), 9.0, device=DEV), torch.full((22, vocab + 7), 9.0, device=DEV)
    wide_p[:, shift_p:shift_p + vocab], wide_q[:, shift_q:shift_q + vocab] = p, q
    got = Fn.draft_verify(tok, _i32(up), b, wide_p[:, shift_p:shift_p + vocab], wide_q[:, shift_q:shift_q + vocab], u)
    _same(got, U.verify(tok, _i32(up), b, p, q, u))


@pytest.mark.parametrize("form", ["given", "draws"])
def test_verify_of_many_siblings_and_the_same_token_twice(form):
    """A star whose children are tried one after the other, most of them not taken."""
    for seed in range(6):
        nodes = [64, 40]
        b = U.batch([3, 9], nodes, 16, DEV)
        up = [-1] + [0] * 63 + [-1] + [0] * 39
        tok, p, q, u = U.drafts(nodes, up, 5000, form, DEV, seed, 0.3)
        tok[1::3] = tok[1]
        tok[5], tok[9] = -1, 5000                               # outside of the vocabulary
        u[1:60] = 0.9999
        _same(Fn.draft_verify(tok, _i32(up), b, p, q, u), U.verify(tok, _i32(up), b, p, q, u))


def test_verify_at_the_ends_of_the_random_numbers_and_without_mass():
    nodes = [3] * 8
    b, up = U.batch([3] * 8, nodes, 16, DEV), U.trees(nodes, 1)
    tok, p, q, u = U.drafts(nodes, up, 3000, "draws", DEV)
    p[:, :100], p[:, -50:] = 0, 0                               # borders at both ends
    u[0::3], u[1::3] = 0.0, 1.0
    u[12:] = 1.0 - 2.0 ** -24
    p[3:6], p[6], q[9:12] = 0, float("nan"), p[9:12]            # nothing; no numbers; nothing of p over q
    p[15:18, 7] = float("inf")
    p[18:21] = -1.0
    _same(Fn.draft_verify(tok, _i32(up), b, p, q, u), U.verify(tok, _i32(up), b, p, q, u))
    _same(Fn.draft_verify(tok, _i32(up), b, p, None, u), U.verify(tok, _i32(up), b, p, None, u))


def test_verify_of_one_hot_and_even_rows():
    """Sums that fp64 holds exactly, random numbers on the borders."""
    nodes = [2] * 16
    b, up = U.batch([3] * 16, nodes, 16, DEV), U.trees(nodes, 1)
    p = torch.full((32, 4096), 2.0 ** -12, device=DEV)
    p[0:2] = 0
    p[0:2, 4000] = 1
    u = (torch.arange(32, device=DEV) * 128).remainder(4096) / 4096
    tok = (torch.arange(32, device=DEV) * 37).to(I32)
    for q in (None, p.roll(1, 1), p.clone()):
        _same(Fn.draft_verify(tok, _i32(up), b, p, q, u), U.verify(tok, _i32(up), b, p, q, u))


def test_verify_leaves_rows_behind_the_last_sequence():
    nodes = [5, 2]
    b, up = U.batch([3, 3], nodes, 16, DEV), U.trees(nodes, 1)
    tok, p, q, u = U.drafts(nodes, up, 50, "draws", DEV)
    more = [torch.cat((x, x[:1].expand(80, *x.shape[1:]))) for x in (tok, _i32(up), p, q, u)]
    got = Fn.draft_verify(more[0], more[1], b, *more[2:])
    _same([got[0][:7], got[1][:7], got[2]], U.verify(tok, _i32(up), b, p, q, u))
    assert (got[0][7:] == -1).all() and (got[1][7:] == -1).all()


def test_verify_refuses_on_the_gpu():
    b = U.batch([3], [2], 16, DEV)
    p, u = torch.rand(2, 9, device=DEV), torch.rand(2, device=DEV)
    for args in [(_i32([1, 2]), _i32([-1, 0]), b, p.cpu(), None, u), (_i32([1, 2]), _i32([-1, 0]), b, p, p.cpu(), u),
                 (_i32([1, 2]), _i32([-1, 0]).cpu(), b, p, p, u)]:
        with pytest.raises(ValueError):
            Fn.draft_verify(*args)


# -- rows that move -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("ctx,nodes,heads,d,page,layers,dtype", [
    ([0], [1], 1, 64, 16, 1, BF16), ([700], [8], 8, 128, 16, 36, BF16), ([5, 0, 31, 2], [8, 0, 3, 1], 2, 64, 8, 3, BF16),
    ([100, 7, 0], [64, 33, 64], 3, 128, 128, 2, torch.float32), ([63, 9], [64, 64], 4, 192, 16, 2, torch.float16), ([20] * 40, [9] * 40, 2, 32, 16, 300, BF16)])
@pytest.mark.parametrize("share", [0.3, 0.9])
def test_keep(ctx, nodes, heads, d, page, layers, dtype, share):
    torch.manual_seed(3)
    b = U.batch(ctx, nodes, page, DEV)
    path, count = U.paths(nodes, share, DEV)
    caches = [torch.randn(kv_cache_shape(b.pages, heads, d, page), device=DEV).to(dtype) for _ in range(layers + 1)]
    want = U.kept(caches, b, path, count)
    Fn.draft_keep(caches[:layers], [None, *caches[layers:], caches[0]], b, path, count)
    for x, y in zip(caches, want):
        assert torch.equal(x, y)


def test_keep_of_paths_that_are_none():
    """Nothing outside of the sequence's nodes is moved, pages that are none are left out."""
    b = U.batch([20, 20], [6, 6], 16, DEV)
    cache = torch.randn(kv_cache_shape(b.pages, 2, 64, 16), device=DEV).to(BF16)
    before = cache.clone()
    Fn.draft_keep([cache], [], b, _i32([0, 9, 60, -1, 2, 3, 0, 1, 2, 3, 4, 5]), _i32([6, 99]))
    assert torch.equal(cache, before)
    b.block_table[0, 1], b.block_table[1, 1] = -3, 10 ** 6
    Fn.draft_keep([cache], [], b, _i32([0, 2, 4, 5, -1, -1] * 2), _i32([4, 4]))
    assert torch.equal(cache, before)


# -- together -------------------------------------------------------------------------------------------------------------
class Model:
    """Two attention layers of random weights: what a step calls, for drafted trees and for one token."""

    def __init__(self, b, hq=8, hkv=2, d=64, vocab=512, layers=2):
        gen = torch.Generator(device=DEV).manual_seed(9)

        def w(*shape):
            return (torch.randn(*shape, generator=gen, device=DEV) * shape[-1] ** -0.5).to(BF16)
        self.hq, self.hkv, self.d, self.wide = hq, hkv, d, hq * d
        self.table, self.head = w(vocab, self.wide) * 16, w(vocab, self.wide)
        self.layers = [(w((hq + 2 * hkv) * d, self.wide), w(self.wide, self.wide)) for _ in range(layers)]
        self.k, self.v = ([torch.zeros(kv_cache_shape(b.pages, hkv, d, 16), dtype=BF16, device=DEV) for _ in range(layers)] for _ in range(2))
        self.angles = ref.build_cos_sin_cache(d, 4096, 1e4).to(DEV)

    def __call__(self, tokens, positions, slots, attend):
        x = Fn.embedding(tokens, self.table)
        for (qkv_w, o_w), k, v in zip(self.layers, self.k, self.v):
            q, kk, vv = Fn.linear(x, qkv_w).split([self.hq * self.d, self.hkv * self.d, self.hkv * self.d], 1)
            Fn.rope_kv_write(q.unflatten(1, (-1, self.d)), kk.unflatten(1, (-1, self.d)), vv.unflatten(1, (-1, self.d)), positions, self.angles,
                             self.d, True, None, None, 1e-6, k, v, slots)
            x = x + Fn.linear(attend(q, k, v), o_w)
        return Fn.linear(x, self.head)


def _step(model, b, tokens, up):
    seen, positions, slots = Fn.draft_plan(up, b, 16)
    return model(tokens, positions, slots, lambda q, k, v: Fn.draft_attention(q, k, v, b, seen, 0.125, model.hq, model.d))


def test_a_run_with_drafts_is_the_run_without():
    """Trees of guesses, right ones among them, verified by the target's own tokens: what a sequence says, and its cache, is what single
    tokens give (paged_attention); logits agree to the roundings of two layers in bf16 (some 2^-8 of a row's largest each)."""
    lens = [37, 5, 90]
    b = U.batch(lens, [64] * 3, 16, DEV)                        # room for what is to come
    table = b.block_table
    gen = torch.Generator(device=DEV).manual_seed(4)
    prompts = [torch.randint(0, 500, (n,), generator=gen, device=DEV, dtype=I32) for n in lens]

    def batch(ctx, nodes):
        x = U.batch(ctx, nodes, 16, DEV)
        x.block_table = table
        return x

    def prefill(model):                                         # chains behind nothing, 64 tokens at a time
        for at in range(0, 90, 64):
            part = [p[at:at + 64] for p in prompts]
            x = batch([min(at, n) for n in lens], [len(p) for p in part])
            up = [i - 1 for p in part for i in range(len(p))]
            _step(model, x, torch.cat(part), _i32(up))

    one = Model(b)
    prefill(one)
    said, logits = [[11, 22, 33]], []
    for step in range(12):                                      # single tokens
        x = batch([n + step for n in lens], [1] * 3)
        seen, pos, slots = Fn.draft_plan(_i32([-1] * 3), x, 16)
        dec = types.SimpleNamespace(**{**vars(x), "num_decode_seqs": 3, "decode_splits": None, "batch": None})
        z = one(_i32(said[-1]), pos, slots, lambda q, k, v: Fn.paged_attention(q, k, v, dec, 0.125, one.hq, one.d))
        logits.append(z)
        said.append(Fn.sample(z, types.SimpleNamespace(batch=types.SimpleNamespace(all_greedy=True, need_penalty=False))).tolist())

    two = Model(b)
    prefill(two)
    for x, y in zip(one.k + one.v, two.k + two.v):
        pages = table[0, :2].long()
        assert torch.equal(x[pages], y[pages])
    done, now, sure = [0, 0, 0], [11, 22, 33], 0
    while min(done) < 8:
        tokens, up, nodes = [], [], []
        for s in range(3):                                      # node 0, two wrong guesses, then right ones below them with wrong beside
            right = [said[min(done[s] + 1 + j, 12)][s] for j in range(3)]
            tokens += [now[s], 7, 9, right[0], 3, right[1], right[2]]
            up += [-1, 0, 0, 0, 3, 3, 5]
            nodes.append(7)
        x = batch([n + d for n, d in zip(lens, done)], nodes)
        z = _step(two, x, _i32(tokens), _i32(up))
        for s in range(3):
            want = logits[done[s]][s].float()
            assert (z[7 * s].float() - want).abs().max() <= 8 * 2 ** -8 * want.abs().max()
        chosen = Fn.sample(z, types.SimpleNamespace(batch=types.SimpleNamespace(all_greedy=True, need_penalty=False)))
        out, path, count = Fn.draft_verify(_i32(tokens), _i32(up), x, chosen)
        Fn.draft_keep(two.k, two.v, x, path, count)
        for s in range(3):
            n = int(count[s])
            for j, t in enumerate(out[7 * s:7 * s + n].tolist()):
                if done[s] + 1 + j <= 12:
                    assert t == said[done[s] + 1 + j][s], (s, done, j)
            sure = max(sure, n)
            done[s] += n
            now[s] = int(out[7 * s + n - 1])
    assert sure == 4                                            # all of a tree's right guesses are taken
    for s in range(3):                                          # the caches of what was said
        keep = lens[s] + min(done[s], 12)
        at = torch.arange(keep, device=DEV)
        for x, y in zip(one.k + one.v, two.k + two.v):
            a, c = (z[table[s][at // 16].long(), :, :, at % 16].float() for z in (x, y))
            assert (a - c).abs().max() <= 8 * 2 ** -8 * a.abs().max()


@pytest.mark.parametrize("form", ["given", "draws", "match"])
def test_a_captured_step(form):
    """One graph of plan, attention, verification and moves, replayed on other lengths, trees, tokens and pages; two graphs in turn."""
    seqs, most, hq, hkv, d, vocab = 3, 9, 8, 2, 128, 3001
    t = seqs * most
    made = []
    for g in range(2):
        torch.manual_seed(g)
        pages = 120
        s = types.SimpleNamespace(
            inp=types.SimpleNamespace(block_table=torch.zeros(seqs, 40, dtype=I32, device=DEV), seq_lens=_i32([1] * seqs),
                                      query_start_loc=_i32([0, 1, 2, 3]), num_seqs=seqs, num_tokens=t, max_q_len=most, max_seq_len=640, padded_tokens=0),
            up=_i32([-1] * t), tok=_i32([0] * t), q=torch.randn(t, hq * d, device=DEV).to(BF16),
            caches=[torch.randn(kv_cache_shape(pages, hkv, d, 16), device=DEV).to(BF16) for _ in range(2)],
            target=torch.zeros(t, dtype=I32, device=DEV) if form == "match" else torch.rand(t, vocab, device=DEV),
            draft=torch.rand(t, vocab, device=DEV) if form == "draws" else None, u=None if form == "match" else torch.rand(t, device=DEV))

        def step(s=s):
            s.plan = Fn.draft_plan(s.up, s.inp, 16)
            s.out = Fn.draft_attention(s.q, *s.caches, s.inp, s.plan[0], d ** -0.5, hq, d)
            s.said = Fn.draft_verify(s.tok, s.up, s.inp, s.target, s.draft, s.u)
            Fn.draft_keep([s.caches[0]], [s.caches[1]], s.inp, s.said[1], s.said[2])
        step()
        torch.cuda.synchronize()
        s.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s.graph):
            step()
        made.append(s)
    for ctx, nodes in [([0, 0, 0], [1, 1, 1]), ([600, 3, 250], [9, 0, 5]), ([127, 128, 500], [9, 9, 9]), ([10, 20, 30], [0, 0, 4])]:
        for g, s in enumerate(made):
            b = U.batch(ctx, nodes, 16, DEV, seed=g)
            up = U.trees(nodes, 3, g)
            n = len(up)
            tok, target, draft, u = U.drafts(nodes, up, vocab, form, DEV, g)
            s.inp.block_table.fill_(-7)
            s.inp.block_table[:, : b.block_table.shape[1]] = b.block_table
            s.inp.seq_lens.copy_(b.seq_lens)
            s.inp.query_start_loc.copy_(b.query_start_loc)
            for x, y in ((s.up, _i32(up)), (s.tok, tok), (s.target, target), (s.draft, draft), (s.u, u)):
                if x is not None:
                    x[:n] = y
            s.before = [c.clone() for c in s.caches]
            s.b, s.n = b, n
            s.graph.replay()
        torch.cuda.synchronize()
        for s in made:
            up, n = s.up[:n], s.n
            want, tol = U.attention(s.q[:n], *s.before, s.b, U.sees(s.plan[0].tolist(), s.b), d ** -0.5, hq)
            assert ((s.out[:n].double().view(-1, hq, d) - want).abs() <= tol).all()
            said = U.verify(s.tok[:n], up, s.b, s.target, s.draft, s.u)
            assert torch.equal(s.said[0][:n], said[0]) and torch.equal(s.said[1][:n], said[1]) and torch.equal(s.said[2], said[2])
            assert (s.said[0][n:] == -1).all() and (s.plan[0][n:] == 0).all()
            for x, y in zip(s.caches, U.kept(s.before, s.b, said[1], said[2])):
                assert torch.equal(x, y)


@pytest.mark.parametrize("parts", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("vocab", [5, 3001, 70001])
def test_verify_whatever_draft_rows_hold_that_no_child_was_drawn_from(parts, vocab, monkeypatch):
    """The draft's row of a node without children, or whose child is taken, is not part of the answer; nor is one that leaves nothing of p."""
    monkeypatch.setattr(sm100_draft, "_verify_parts", lambda *a: parts)
    nodes = [1, 4, 3, 2, 1, 5, 2]
    b, up = U.batch([3] * len(nodes), nodes, 16, DEV), U.trees(nodes, 1)
    for seed in range(3):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        tok, p, _, u = U.drafts(nodes, up, vocab, "given", DEV, seed)
        q = 1.5 * p                                             # nothing of p is over it: a refused child's rest is p itself
        tok[:] = torch.arange(len(up), device=DEV) % 2          # tokens 0 and 1 keep their numbers
        first, what = 0, (float("nan"), float("inf"), float("-inf"))
        for s, n in enumerate(nodes):
            u[first + 1:first + n] = 0.0                        # taken
            q[first + n - 1] = what[(s + seed) % 3]             # without children
            if s % 2 == 0 and n > 1:                            # the last child is refused
                u[first + n - 1] = 1 - 2.0 ** -24
                hit = torch.rand(vocab - 2, generator=gen, device=DEV) < 0.5
                q[first + n - 2, 2:] = torch.where(hit, torch.where(hit.roll(1), float("nan"), float("inf")), q[first + n - 2, 2:])
            first += n
        want = U.verify(tok, _i32(up), b, p, q, u)
        assert want[2].tolist() == [n - (s % 2 == 0 and n > 1) for s, n in enumerate(nodes)]
        _same(Fn.draft_verify(tok, _i32(up), b, p, q, u), want)


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_many_items_with_and_without_a_second_half(d, whole, monkeypatch):
    """Some seven items an SM in blocks of 256 rows, few of them with more than 128; values of nodes that are no numbers in one sequence of two."""
    monkeypatch.setattr(sm100_draft, "_whole_units", lambda *a: whole)
    nodes = [(64, 2, 5, 1, 40, 3, 33, 7, 1, 2)[s % 10] for s in range(500)]
    ctx = [(7 * s) % 140 for s in range(500)]
    x = _attention_case(ctx, nodes, 8, 2, d, 16)
    t, seen = x.b.num_tokens, x.seen.tolist()
    hit = torch.zeros(t, d, dtype=torch.bool, device=DEV)         # columns of a row with a value that is no number
    first = 0
    for s, n in enumerate(nodes):
        if s % 2 == 0:
            i = s // 2 % n
            x.v[int(x.b.block_table[s, (ctx[s] + i) // 16]), :, :, (ctx[s] + i) % 16, s % 7::7] = (float("nan"), float("inf"), float("-inf"))[s % 3]
            rows = [r for r in range(first, first + n) if seen[r] >> i & 1]
            hit[rows] = torch.arange(d, device=DEV) % 64 % 7 == s % 7
        first += n
    out = Fn.draft_attention(x.q, x.k, x.v, x.b, x.seen, d ** -0.5, 8, d)[:t].double().view(-1, 8, d)
    want, tol = U.attention(x.q[:t], x.k, torch.where(x.v.isfinite(), x.v, 0), x.b, U.sees(seen, x.b), d ** -0.5, 8)
    assert hit.any() and torch.where(hit[:, None], ~out.isfinite(), (out - want).abs() <= tol).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("most", [8, 16, 30, 64])
@pytest.mark.parametrize("pages", [1, 2, 9])
def test_attention_of_tables_that_end(pages, most, d):
    """Tokens behind a table's last page have no place: nobody sees them, context or nodes."""
    x = _attention_case([16 * pages - 2, 0, 16 * pages + 8, 5, 16 * pages], [most, most, 3, 7, 2], 8, 2, d, 16)
    x.b.block_table = x.b.block_table[:, :pages]
    masks = [m[:, :16 * pages] for m in U.sees(x.seen.tolist(), x.b)]
    _check_attention(x, masks=masks)


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("most", [8, 16, 30, 64])
def test_captured_attention_with_units_cut_and_whole(most, d, whole, monkeypatch):
    """Two graphs in turn, replayed with lengths that change which shares begin, end and join units: many parts, then none, then others."""
    monkeypatch.setattr(sm100_draft, "_whole_units", lambda *a: whole)
    seqs, made = 4, []
    for g in range(2):
        torch.manual_seed(g)
        inp = types.SimpleNamespace(block_table=torch.zeros(seqs, 640, dtype=I32, device=DEV), seq_lens=_i32([1] * seqs), query_start_loc=_i32(range(seqs + 1)),
                                    num_seqs=seqs, num_tokens=seqs * most, max_q_len=most, max_seq_len=10000, padded_tokens=0)
        s = types.SimpleNamespace(inp=inp, q=torch.randn(seqs * most, 8 * d, device=DEV).to(BF16), seen=torch.ones(seqs * most, dtype=torch.int64, device=DEV),
                                  caches=[torch.randn(kv_cache_shape(1800, 2, d, 16), device=DEV).to(BF16) for _ in range(2)],
                                  out=torch.zeros(seqs * most, 8 * d, dtype=BF16, device=DEV))

        def step(s=s):
            Fn.draft_attention(s.q, *s.caches, s.inp, s.seen, d ** -0.5, 8, d, out=s.out)
        step()
        torch.cuda.synchronize()
        s.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s.graph):
            step()
        made.append(s)
    for ctx, nodes in [([9000, 40, 9000, 8000], [most] * 4), ([0, 0, 0, 0], [1, 0, 0, 0]), ([9900, 0, 0, 0], [most, 0, 1, 0]), ([60, 700, 5, 9000], [1, most, most, 3]),
                       ([0] * 4, [0] * 4), ([2000] * 4, [most] * 4), ([127, 9000, 128, 1], [most, 1, most, 2])]:
        for g, s in enumerate(made):
            b, n = U.batch(ctx, nodes, 16, DEV, seed=g), sum(nodes)
            s.inp.block_table.fill_(-7)
            s.inp.block_table[:, : b.block_table.shape[1]] = b.block_table
            s.inp.seq_lens.copy_(b.seq_lens)
            s.inp.query_start_loc.copy_(b.query_start_loc)
            s.seen[:n] = Fn.draft_plan(_i32(U.trees(nodes, 3, g)), b, 16)[0]
            s.out.fill_(5)
            s.b, s.n = b, n
            s.graph.replay()
        torch.cuda.synchronize()
        for s in made:
            assert (s.out[s.n:] == 5).all()
            if s.n:
                want, tol = U.attention(s.q[:s.n], *s.caches, s.b, U.sees(s.seen.tolist(), s.b), d ** -0.5, 8)
                assert ((s.out[:s.n].double().view(-1, 8, d) - want).abs() <= tol).all(), ctx
