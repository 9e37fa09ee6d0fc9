"""Kernels of the cache held in 4 bits against the definitions in 64 bits (GPU)."""
import types

import numpy as np
import pytest
import torch

from gllm_b200.ops import kv4, ref
from tests import kv4_util as U

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# -- writing ------------------------------------------------------------------------------------------------------------
def _write_inputs(t, hq, hkv, d, rot, page, norms, extra=0):
    torch.manual_seed(t + hq + d + rot)
    pages = -(-t // page) + 2
    buf = torch.randn(t, (hq + 2 * hkv) * d + extra, device=DEV).to(BF16)
    q, k, v = buf[:, extra:].split([hq * d, hkv * d, hkv * d], 1)
    q, k, v = q.unflatten(1, (hq, d)), k.unflatten(1, (hkv, d)), v.unflatten(1, (hkv, d))
    k += torch.randn(hkv, d, device=DEV).to(BF16)
    pos = torch.randint(0, 4000, (t,), device=DEV, dtype=torch.int32)
    cs = ref.build_cos_sin_cache(rot, 4096, 1e4).to(DEV) if rot else None
    slots = torch.randperm(pages * page, device=DEV)[:t].to(torch.int32)
    w = [(1 + 0.1 * torch.randn(d, device=DEV)).to(BF16) if n in norms else None for n in "qk"]
    caches = [torch.randint(0, 256, kv4.cache_shape(pages, hkv, d, page), dtype=torch.uint8, device=DEV) for _ in range(2)]
    return types.SimpleNamespace(buf=buf, q=q, k=k, v=v, pos=pos, cs=cs, slots=slots, w=w, caches=caches, pages=pages)


@pytest.mark.parametrize("t,hq,hkv,d,rot,neox,page,extra", [
    (1, 1, 1, 64, 64, True, 16, 0), (1, 32, 8, 128, 128, True, 16, 0), (83, 7, 1, 64, 32, True, 16, 8), (83, 5, 3, 128, 64, False, 48, 8),
    (200, 14, 2, 64, 64, False, 32, 0), (33, 8, 8, 128, 96, True, 16, 8), (33, 4, 4, 128, 0, True, 16, 0), (700, 32, 8, 128, 128, True, 64, 0),
    (900, 16, 4, 64, 64, True, 16, 0), (5, 3, 1, 128, 8, False, 16, 0)])
def test_write_gives_the_plain_forms_bits(t, hq, hkv, d, rot, neox, page, extra):
    """Without norms every step is one rounded operation: queries and caches agree bit for bit, slots that are left out and rows of
    other tokens included."""
    from gllm_b200.ops import sm100_kv4
    x = _write_inputs(t, hq, hkv, d, rot, page, "", extra)
    if t > 2:
        x.slots[t // 2], x.slots[0] = -1, x.pages * page + 5
    want, q0, k0 = [c.clone() for c in x.caches], x.q.clone(), x.k.clone()
    sm100_kv4.rope_kv_write(x.q, x.k, x.v, x.pos, x.cs, rot, neox, None, None, 1e-6, *x.caches, x.slots)
    assert torch.equal(x.k, k0)
    ref.rope_kv_write(q0, x.k, x.v, x.pos, x.cs, rot, neox, None, None, 1e-6, *want, x.slots)
    assert torch.equal(x.q, q0)
    for a, b in zip(x.caches, want):
        assert torch.equal(a, b)
    rows = sm100_kv4.kv_cache_rows(*x.caches, x.slots)
    for a, c in zip(rows, want):
        assert torch.equal(a, kv4.read_rows(c, x.slots).to(BF16))


@pytest.mark.parametrize("norms", ["q", "k", "qk"])
@pytest.mark.parametrize("t,hq,hkv,d,rot,neox", [(1, 4, 2, 64, 64, True), (65, 32, 8, 128, 128, True), (300, 6, 2, 128, 64, False)])
def test_write_with_norms(t, hq, hkv, d, rot, neox, norms):
    """Against 64 bits: a query is rounded behind the norm and behind the rotation (a value that lies next to a border may go to
    either side: two steps of 2^-8 of the largest it is turned from); a held key is within half a code's step of it, the step itself good to
    2^-8 and, through the ends of its group, to those roundings."""
    from gllm_b200.ops import sm100_kv4
    x = _write_inputs(t, hq, hkv, d, rot, 16, norms)
    half = rot // 2
    rows = x.cs[x.pos.long()]
    want_q, want_k = (U.turned(y, w, rows[:, :half], rows[:, half:], rot, neox, 1e-6) for y, w in zip((x.q, x.k), x.w))
    sm100_kv4.rope_kv_write(x.q, x.k, x.v, x.pos, x.cs, rot, neox, *x.w, 1e-6, *x.caches, x.slots)
    most = want_q.abs().amax(-1, keepdim=True)
    assert ((x.q.double() - want_q).abs() <= 2 ** -7 * 2 ** 0.5 * most).all()
    keys, vals = sm100_kv4.kv_cache_rows(*x.caches, x.slots)
    y = want_k.unflatten(-1, (-1, 64))
    most = y.abs().amax(-1, keepdim=True).amax(-2, keepdim=True)
    turn = 2 ** -7 * 2 ** 0.5 * most
    step = (y.amax(-1, keepdim=True) - y.amin(-1, keepdim=True) + 2 * turn) / 15
    assert ((keys.double().unflatten(-1, (-1, 64)) - y).abs() <= step * (0.5 + 16 * 2 ** -8) + turn + 2 ** -8 * most).all()
    assert torch.equal(vals, U.values(x.v).float().to(BF16))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", [3, 900])
def test_write_in_both_forms_gives_the_same_bits(t, d):
    """Three equal rows of positions take the form with a lane per eight dims, one row the one with both halves of a pair in a lane."""
    from gllm_b200.ops import sm100_kv4
    x = _write_inputs(t, 16, 8, d, d, 16, "qk")
    other, q0 = [c.clone() for c in x.caches], x.q.clone()
    sm100_kv4.rope_kv_write(x.q, x.k, x.v, x.pos, x.cs, d, True, *x.w, 1e-6, *x.caches, x.slots)
    sm100_kv4.rope_kv_write(q0, x.k, x.v, x.pos.expand(3, -1).contiguous(), x.cs, d, True, *x.w, 1e-6, *other, x.slots, [d // 4, d // 8, d // 8])
    assert torch.equal(x.q, q0) and all(torch.equal(a, b) for a, b in zip(x.caches, other))


@pytest.mark.parametrize("section", [[8, 12, 12], [16, 8, 8], [12, 10, 10, True]])
def test_write_with_three_position_rows(section):
    from gllm_b200.ops import sm100_kv4
    x = _write_inputs(50, 4, 2, 64, 64, 16, "")
    pos = torch.randint(0, 4000, (3, 64), device=DEV, dtype=torch.int32)[:, :50]
    want, q0 = [c.clone() for c in x.caches], x.q.clone()
    sm100_kv4.rope_kv_write(x.q, x.k, x.v, pos, x.cs, 64, True, None, None, 1e-6, *x.caches, x.slots, section)
    ref.rope_kv_write(q0, x.k, x.v, pos, x.cs, 64, True, None, None, 1e-6, *want, x.slots, section)
    assert torch.equal(x.q, q0) and all(torch.equal(a, b) for a, b in zip(x.caches, want))


def test_write_of_values_that_are_no_numbers_and_of_flat_groups():
    from gllm_b200.ops import sm100_kv4
    x = _write_inputs(6, 2, 2, 128, 0, 16, "")
    x.v[0, 0, 3], x.v[1, 1, 70], x.v[2, 0] = float("nan"), float("inf"), 2.5
    x.v[3, 1, :64], x.k[4] = 0.0, 1e30
    sm100_kv4.rope_kv_write(x.q, x.k, x.v, x.pos, None, 0, True, None, None, 1e-6, *x.caches, x.slots)
    keys, vals = sm100_kv4.kv_cache_rows(*x.caches, x.slots)
    assert torch.isnan(vals[0, 0, :64]).all() and torch.isnan(vals[1, 1, 64:]).all()
    bad = torch.isnan(vals)
    assert bad.sum() == 128 and torch.equal(vals[~bad], U.values(x.v).float().to(BF16)[~bad])
    assert (vals[2, 0] == 2.5).all() and (vals[3, 1, :64] == 0).all() and torch.equal(keys[4], x.k[4])


def test_write_of_no_tokens():
    from gllm_b200.ops import sm100_kv4
    x = _write_inputs(4, 2, 2, 64, 64, 16, "")
    before = [c.clone() for c in x.caches]
    sm100_kv4.rope_kv_write(x.q[:0], x.k[:0], x.v[:0], x.pos[:0], x.cs, 64, True, None, None, 1e-6, *x.caches, x.slots[:0])
    assert all(torch.equal(a, b) for a, b in zip(x.caches, before))
    assert sm100_kv4.kv_cache_rows(*x.caches, x.slots[:0])[0].shape == (0, 2, 64)


# -- attention ----------------------------------------------------------------------------------------------------------
def _filled(lens, hkv, d, page, seed=0):
    """Caches whose free rows hold bytes that stand for NaN, the sequences' rows and their table (entries behind them are no pages)."""
    torch.manual_seed(seed + sum(lens) + d)
    blocks = [-(-n // page) for n in lens]
    pages = sum(blocks) + 3
    order = torch.randperm(pages)
    table = torch.full((len(lens), max(max(blocks), 1) + 1), -7, dtype=torch.int32)
    caches = [torch.full(kv4.cache_shape(pages, hkv, d, page), 255, dtype=torch.uint8, device=DEV) for _ in range(2)]
    rows, at = [], 0
    for s, (n, b) in enumerate(zip(lens, blocks)):
        table[s, :b] = order[at:at + b]
        at += b
        i = torch.arange(n)
        slots = (table[s].long()[i // page] * page + i % page).to(torch.int32).to(DEV)
        kv = [(torch.randn(n, hkv, d, device=DEV) * (0.5 + torch.rand(hkv, d, device=DEV)) + torch.randn(hkv, d, device=DEV)).to(BF16)
              for _ in range(2)]
        for c, x in zip(caches, kv):
            kv4.write_rows(c, slots, x)
        rows.append(kv)
    return caches, rows, table.to(DEV)


def _attend(q, caches, table, lens, news, decodes, hq, hkv, d, **kw):
    from gllm_b200.ops import sm100_kv4
    start = _i32([0] + np.cumsum(news).tolist())
    return sm100_kv4.paged_attention(q, *caches, table, _i32(lens), start, kw.pop("scale", d ** -0.5), hq, d, decodes, len(lens),
                                     max(news), max(lens), host_lens=lens, **kw)


@pytest.mark.parametrize("lens", [[1], [16], [17], [31, 32, 33], [0, 5, 0], [700], [64] * 3 + [1, 2000, 3]])
@pytest.mark.parametrize("hq,hkv,d,page", [(4, 1, 128, 16), (7, 1, 64, 16), (8, 8, 64, 48), (16, 2, 128, 32), (24, 2, 128, 16), (32, 1, 64, 16),
                                           (20, 2, 64, 16)])
def test_decode(lens, hq, hkv, d, page):
    caches, rows, table = _filled(lens, hkv, d, page)
    buf = torch.randn(len(lens), hq * d + 64, device=DEV).to(BF16)          # rows of a wider projection
    q = buf[:, 64:]
    got = _attend(q, caches, table, lens, [1] * len(lens), len(lens), hq, hkv, d)
    want, tol = U.attention(q.unflatten(1, (hq, d)), rows, lens, [1] * len(lens), d ** -0.5, hkv, False)
    assert ((got.view_as(want).double() - want).abs() <= tol).all()


@pytest.mark.parametrize("b,longest,hq,hkv,d", [(300, 90, 4, 2, 64), (700, 40, 8, 1, 128), (256, 100, 32, 8, 128), (1100, 150, 4, 2, 64), (3, 30000, 8, 2, 128), (1, 50000, 16, 1, 64), (64, 1500, 8, 8, 128)])
def test_decode_of_many_and_of_long_sequences(b, longest, hq, hkv, d):
    rng = np.random.RandomState(b)
    lens = rng.randint(1, longest + 1, b).tolist()
    caches, rows, table = _filled(lens, hkv, d, 16)
    q = torch.randn(b, hq * d, device=DEV).to(BF16) * 2
    got = _attend(q, caches, table, lens, [1] * b, b, hq, hkv, d)
    want, tol = U.attention(q.view(b, hq, d), rows, lens, [1] * b, d ** -0.5, hkv, False)
    assert ((got.view_as(want).double() - want).abs() <= tol).all()
    again = _attend(q, caches, table, lens, [1] * b, b, hq, hkv, d)
    assert torch.equal(got, again)                         # sums in a fixed order


@pytest.mark.parametrize("size", [0.0, 1e-30, 1e-4, 300.0])
def test_decode_over_the_range_of_queries(size):
    """Scores up to thousands (one key takes all), queries of zeros and far below what fp16 holds."""
    lens, hq, hkv, d = [150, 37], 8, 2, 128
    caches, rows, table = _filled(lens, hkv, d, 16)
    q = (torch.randn(2, hq * d, device=DEV) * size).to(BF16)
    got = _attend(q, caches, table, lens, [1, 1], 2, hq, hkv, d)
    want, tol = U.attention(q.view(2, hq, d), rows, lens, [1, 1], d ** -0.5, hkv, False)
    if size == 300.0:                                      # scores of some 3000: fp32 holds them to 2^-12, products likewise
        tol = tol + 2 ** -9 * 8
    assert ((got.view_as(want).double() - want).abs() <= tol).all()


@pytest.mark.parametrize("loud", [1.0, 2.0 ** 12, 2.0 ** -12])
def test_decode_of_values_of_very_different_sizes(loud):
    """One token's values are `loud` times the others', and it is not what the queries look for, or all that they look for."""
    lens, hq, hkv, d = [333, 64], 8, 2, 128
    torch.manual_seed(5)
    caches, rows, table = _filled(lens, hkv, d, 16)
    for i, at in ((0, 300), (1, 5)):
        rows[i][1][at] = (rows[i][1][at].float() * loud).to(BF16)
        kv4.write_rows(caches[1], (table[i, at // 16] * 16 + at % 16).view(1), rows[i][1][at:at + 1])
    q = torch.randn(2, hq * d, device=DEV).to(BF16)
    q[1] = (rows[1][0][5].float() * (2.0 if loud < 1 else -0.2)).to(BF16).repeat_interleave(hq // hkv, 0).flatten()
    got = _attend(q, caches, table, lens, [1, 1], 2, hq, hkv, d)
    want, tol = U.attention(q.view(2, hq, d), rows, lens, [1, 1], d ** -0.5, hkv, False)
    assert ((got.view_as(want).double() - want).abs() <= tol).all()


def test_decode_of_a_key_that_is_no_number():
    lens, hq, hkv, d = [90, 40], 4, 2, 128
    caches, rows, table = _filled(lens, hkv, d, 16)
    bad = rows[0][0][70:71].clone()
    bad[0, 1, 5] = float("nan")
    slot = table[0, 70 // 16] * 16 + 70 % 16
    kv4.write_rows(caches[0], slot.view(1), bad)
    q = torch.randn(2, hq * d, device=DEV).to(BF16)
    got = _attend(q, caches, table, lens, [1, 1], 2, hq, hkv, d).view(2, hq, d)
    assert torch.isnan(got[0, 2:]).all() and torch.isfinite(got[0, :2].float()).all() and torch.isfinite(got[1].float()).all()


@pytest.mark.parametrize("lens,news,decodes", [
    ([1], [1], 0), ([5, 64, 200], [5, 64, 200], 0), ([300, 129], [17, 128], 0), ([33, 900, 90, 65], [1, 1, 90, 3], 2),
    ([40, 7, 500, 130], [1, 7, 260, 1], 1)])
@pytest.mark.parametrize("hq,hkv,d,page", [(4, 1, 128, 16), (14, 2, 64, 16), (8, 8, 64, 48), (32, 4, 128, 64)])
def test_prompts_beside_decodes(lens, news, decodes, hq, hkv, d, page, monkeypatch):
    from gllm_b200.ops import sm100_kv4
    monkeypatch.setattr(sm100_kv4, "EXPAND_BYTES", 256 * 4 * hkv * d)       # several rounds
    caches, rows, table = _filled(lens, hkv, d, page)
    q = torch.randn(sum(news), hq * d, device=DEV).to(BF16)
    got = _attend(q, caches, table, lens, news, decodes, hq, hkv, d)
    want, tol = U.attention(q.view(-1, hq, d), rows, lens, news, d ** -0.5, hkv, True)
    assert ((got.view_as(want).double() - want).abs() <= tol).all()


def test_prompts_without_lengths_on_the_host():
    from gllm_b200.ops import sm100_kv4
    lens, news, hq, hkv, d = [20, 190, 64], [20, 100, 1], 4, 2, 64
    caches, rows, table = _filled(lens, hkv, d, 16)
    q = torch.randn(sum(news), hq * d, device=DEV).to(BF16)
    args = (q, *caches, table, _i32(lens), _i32([0, 20, 120, 121]), 0.1, hq, d, 0, 3, 100, 190)
    assert torch.equal(sm100_kv4.paged_attention(*args), sm100_kv4.paged_attention(*args, host_lens=lens))


def test_decode_of_more_sequences_than_a_block_keeps_lengths_of():
    """A sequence of one tile is never cut, so it has the same bits in any batch."""
    b, d = 90000, 64
    caches, rows, table = _filled([16], 1, d, 16)
    lens = np.random.RandomState(0).randint(0, 17, b).tolist()
    q = torch.randn(b, d, device=DEV).to(BF16)
    got = _attend(q, caches, table.expand(b, -1), lens, [1] * b, b, 1, 1, d)
    for at in (0, 44000, b - 300):
        part = _attend(q[at:at + 300], caches, table.expand(300, -1), lens[at:at + 300], [1] * 300, 300, 1, 1, d)
        assert torch.equal(got[at:at + 300], part)
    want, tol = U.attention(q[:40].view(40, 1, d), rows * 40, lens[:40], [1] * 40, d ** -0.5, 1, False)
    assert ((got[:40].view_as(want).double() - want).abs() <= tol).all()


def test_rows_behind_the_last_sequence_stay():
    lens, hq, hkv, d = [30, 50], 4, 2, 64
    caches, rows, table = _filled(lens, hkv, d, 16)
    q = torch.randn(5, hq * d, device=DEV).to(BF16)
    out = torch.full((5, hq * d), 7.0, dtype=BF16, device=DEV)
    _attend(q, caches, table, lens, [1, 1], 2, hq, hkv, d, out=out)
    assert (out[2:] == 7).all() and (out[:2] != 7).any()


def test_decode_captured_and_replayed_with_other_lengths_beside_another_graph():
    """Two graphs on two streams at once, each with scratch of its own; lengths and table are read at replay."""
    from gllm_b200.ops import sm100_kv4
    hq, hkv, d, b = 8, 2, 128, 5
    lens = [[3, 800, 40, 1, 77], [2000, 16, 17, 300, 5]]
    made = [_filled([2048] * b, hkv, d, 16, seed=i) for i in range(2)]
    runs = []
    for caches, rows, table in made:
        q = torch.randn(b, hq * d, device=DEV).to(BF16)
        n = _i32([1] * b)
        out = torch.empty(b, hq * d, dtype=BF16, device=DEV)

        def call():
            sm100_kv4.paged_attention(q, *caches, table, n, None, d ** -0.5, hq, d, b, b, 1, 2048, out=out)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        runs.append((graph, q, n, out, torch.cuda.Stream()))
    for turn in range(4):
        for i, (graph, q, n, out, stream) in enumerate(runs):
            n.copy_(_i32(lens[(i + turn) % 2]))
        torch.cuda.synchronize()
        for graph, q, n, out, stream in runs:
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for i, ((graph, q, n, out, stream), (caches, rows, table)) in enumerate(zip(runs, made)):
            want, tol = U.attention(q.view(b, hq, d), rows, lens[(i + turn) % 2], [1] * b, d ** -0.5, hkv, False)
            assert ((out.view_as(want).double() - want).abs() <= tol).all()


def test_prompts_captured_and_replayed_with_other_lengths():
    """A graph has room for what its block table holds, whatever the lengths were when it was captured."""
    from gllm_b200.ops import sm100_kv4
    hq, hkv, d, news = 4, 2, 64, [1, 30, 70]
    caches, rows, table = _filled([512] * 3, hkv, d, 16)
    q = torch.randn(sum(news), hq * d, device=DEV).to(BF16)
    n, starts = _i32([5, 40, 70]), _i32([0, 1, 31, 101])
    out = torch.empty(sum(news), hq * d, dtype=BF16, device=DEV)

    def call():
        sm100_kv4.paged_attention(q, *caches, table, n, starts, d ** -0.5, hq, d, 1, 3, 70, 70, out=out, host_lens=[5, 40, 70])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([5, 40, 70], [400, 512, 333], [1, 30, 512]):
        n.copy_(_i32(lens))
        graph.replay()
        torch.cuda.synchronize()
        for a, b, at, rounded in ((0, 1, 0, False), (1, 3, 1, True)):
            want, tol = U.attention(q[at:sum(news[:b])].view(-1, hq, d), rows[a:b], lens[a:b], news[a:b], d ** -0.5, hkv, rounded)
            assert ((out[at:sum(news[:b])].view_as(want).double() - want).abs() <= tol).all(), (lens, a)


@pytest.mark.parametrize("news", [[1, 1, 1], [1, 40, 3]])
def test_tables_that_are_views(news):
    """Rows of a wider table, and one row for all sequences."""
    hq, hkv, d, lens, tokens, first = 4, 2, 64, [40, 100, 77], sum(news), news[0]
    caches, rows, table = _filled([112] * 3, hkv, d, 16)
    q = torch.randn(tokens, hq * d, device=DEV).to(BF16)
    decodes = 3 if max(news) == 1 else 1
    wide = torch.full((3, 21), 0x7fffffff, dtype=torch.int32, device=DEV)
    wide[:, 13:] = table
    for t, r in ((wide[:, 13:], rows), (table[1:2].expand(3, -1), [rows[1]] * 3)):
        got = _attend(q, caches, t, lens, news, decodes, hq, hkv, d).view(-1, hq, d).double()
        for a, b, rounded in ((0, decodes, False), (decodes, 3, True)):
            at = slice(sum(news[:a]), sum(news[:b]))
            if a < b:
                want, tol = U.attention(q[at].view(-1, hq, d), r[a:b], lens[a:b], news[a:b], d ** -0.5, hkv, rounded)
                assert ((got[at] - want).abs() <= tol).all()


def test_one_row_of_a_buffer_of_any_width():
    """The stride of a dimension of one does not matter."""
    from gllm_b200.ops import sm100_kv4
    hq, hkv, d = 4, 1, 64
    x = _write_inputs(1, hq, hkv, d, d, 16, "qk")
    odd = [torch.zeros(1, y.shape[1] * d + 5, dtype=BF16, device=DEV)[:, :y.shape[1] * d] for y in (x.q, x.k, x.v)]
    for a, b in zip(odd, (x.q, x.k, x.v)):
        a.copy_(b.flatten(1))
    got = [c.clone() for c in x.caches]
    views = [y.as_strided((1, y.shape[1] // d, d), (y.stride(0), d, 1)) for y in odd]
    assert all(y.stride(0) % 8 for y in odd + views)
    sm100_kv4.rope_kv_write(*views, x.pos, x.cs, d, True, *x.w, 1e-6, *got, x.slots)
    sm100_kv4.rope_kv_write(x.q, x.k, x.v, x.pos, x.cs, d, True, *x.w, 1e-6, *x.caches, x.slots)
    assert torch.equal(views[0], x.q) and all(torch.equal(a, b) for a, b in zip(got, x.caches))
    caches, rows, table = _filled([50], hkv, d, 16)
    for decodes in (1, 0):
        a, b = (_attend(q, caches, table, [50], [1], decodes, hq, hkv, d) for q in (odd[0], x.q.flatten(1).clone()))
        assert torch.equal(a, b)


def test_attention_refuses():
    from gllm_b200.ops import sm100_kv4
    caches, rows, table = _filled([20], 2, 64, 16)
    q = torch.randn(1, 4 * 64 + 4, device=DEV).to(BF16)
    with pytest.raises(ValueError):
        _attend(q[:, 4:], caches, table, [20], [1], 1, 4, 2, 64)             # rows off 16-byte boundaries
    with pytest.raises(AssertionError):
        _attend(q[:, :256].contiguous(), caches, table, [20], [1], 1, 2, 2, 128)
    with pytest.raises(RuntimeError):
        _attend(q[:, :256].contiguous(), caches, table[:, :0], [20], [1], 1, 4, 2, 64)                   # a table without columns
    with pytest.raises(ValueError):
        sm100_kv4.paged_attention(q[:, :256].contiguous(), caches[0], caches[1][:1], table, _i32([20]), None, 1.0, 4, 64, 1, 1, 1, 20)


def test_tensors_elsewhere_are_refused():
    from gllm_b200.ops import sm100, sm100_kv4
    caches, rows, table = _filled([20], 2, 64, 16)
    q = torch.randn(1, 4 * 64, device=DEV).to(BF16)
    with pytest.raises(ValueError):
        sm100_kv4.paged_attention(q, *caches, table.cpu(), _i32([20]), None, 1.0, 4, 64, 1, 1, 1, 20)
    with pytest.raises(ValueError):
        sm100_kv4.kv_cache_rows(*caches, torch.zeros(3, dtype=torch.int32))
    x = _write_inputs(4, 2, 2, 64, 64, 16, "")
    with pytest.raises(ValueError):
        sm100_kv4.rope_kv_write(x.q, x.k, x.v, x.pos.cpu(), x.cs, 64, True, None, None, 1e-6, *x.caches, x.slots)
    with pytest.raises(ValueError):
        sm100.linear_int8(q, torch.zeros(16, 256, dtype=torch.int8), torch.ones(16, device=DEV))


def test_waits_that_run_out_are_reported():
    from gllm_b200.ops import lib as _lib, sm100
    lens, hq, hkv, d = [4000, 300], 8, 2, 128
    caches, rows, table = _filled(lens, hkv, d, 16)
    q = torch.randn(2, hq * d, device=DEV).to(BF16)
    assert sm100.waits_given_up() == 0
    try:
        _lib.watch_waits(0)
        _attend(q, caches, table, lens, [1, 1], 2, hq, hkv, d)
        torch.cuda.synchronize()
        assert _lib.waits_gave_up(clear=True)
    finally:
        _lib.watch_waits()
    got = _attend(q, caches, table, lens, [1, 1], 2, hq, hkv, d)
    want, tol = U.attention(q.view(2, hq, d), rows, lens, [1, 1], d ** -0.5, hkv, False)
    assert ((got.view_as(want).double() - want).abs() <= tol).all() and not _lib.waits_gave_up()
