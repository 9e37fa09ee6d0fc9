"""Cache held in 4 bits: layout and plain form against the definition in 64 bits, refusals, the engine on it (CPU)."""
import types

import numpy as np
import pytest
import torch

from gllm_b200.layers import functional as Fn
from gllm_b200.ops import kv4, ref, sm100_kv4
from tests import kv4_util as U

BF16 = torch.bfloat16


@pytest.mark.parametrize("d", [64, 128])
def test_rows_read_back_as_the_definition_says(d):
    torch.manual_seed(d)
    x = (torch.randn(9, 3, d) * torch.rand(9, 3, 1) * 20 + torch.randn(9, 3, d)).to(BF16)
    x[0, 0] = 0.0                                          # a group without a span
    x[1, 1, :64] = 1.5
    x[2, 2, 5] = 300.0                                     # one dim far out
    x[3, 0, 7], x[3, 1, d - 1] = float("nan"), float("-inf")
    codes, pairs = kv4.encode(x)
    assert codes.shape == (9, 3, d // 2) and pairs.shape == (9, 3, d // 16)
    got, want = kv4.decode(codes, pairs), U.values(x)
    bad = ~torch.isfinite(x.float()).unflatten(-1, (-1, 64)).all(-1, keepdim=True).expand(-1, -1, -1, 64).flatten(-2)
    assert torch.isnan(got[bad]).all()                     # a group with a value that is no number reads back as NaN
    torch.testing.assert_close(got[~bad].double(), want[~bad], rtol=2 ** -23, atol=0)
    span = x.float().unflatten(-1, (-1, 64)).amax(-1) - x.float().unflatten(-1, (-1, 64)).amin(-1)
    off = (got - x.float()).abs().unflatten(-1, (-1, 64)).amax(-1)
    ok = torch.isfinite(span)
    # half a step; the scale's own rounding (2^-8) can leave the upper end 15 2^-8 of a step behind
    assert (off[ok] <= span[ok] / 15 * (0.5 + 16 * 2 ** -8)).all()


@pytest.mark.parametrize("page", [16, 48])
@pytest.mark.parametrize("d", [64, 128])
def test_write_then_read(d, page):
    torch.manual_seed(1)
    pages, heads, t = 5, 3, 29
    cache = torch.randint(0, 256, kv4.cache_shape(pages, heads, d, page), dtype=torch.uint8)
    before = cache.clone()
    slots = torch.randperm(pages * page)[:t].to(torch.int32)
    slots[4], slots[7] = -1, pages * page                  # left out
    x = torch.randn(t, heads, d).to(BF16)
    kv4.write_rows(cache, slots, x)
    got = kv4.read_rows(cache, slots)
    keep = torch.ones(t, dtype=torch.bool)
    keep[[4, 7]] = False
    torch.testing.assert_close(got[keep].double(), U.values(x[keep]), rtol=2 ** -23, atol=0)
    assert (got[~keep] == 0).all()
    other = torch.ones(pages * page, dtype=torch.bool)
    other[slots[keep].long()] = False
    rest = torch.nonzero(other)[:, 0].to(torch.int32)
    a, b = kv4.read_rows(cache, rest), kv4.read_rows(before, rest)
    assert torch.equal(a.view(torch.int32), b.view(torch.int32))           # nothing else moved


def test_layout_of_a_row():
    """Code of dim 64 g + 8 chunk + e: nibble e of unit chunk * groups + g."""
    x = torch.zeros(128)
    x[64 + 8 * 3 + 5] = 15.0
    codes, pairs = kv4.encode(x.to(BF16))
    word = codes.view(torch.int32)
    assert torch.nonzero(word)[:, 0].tolist() == [3 * 2 + 1] and int(word[7]) == 15 << 20
    assert pairs.view(BF16).tolist() == [0.0, 0.0, 1.0, 0.0]


def test_ref_write_rotates_queries_and_leaves_keys():
    torch.manual_seed(2)
    t, hq, hkv, d = 6, 4, 2, 64
    q, k, v = (torch.randn(t, h, d).to(BF16) for h in (hq, hkv, hkv))
    cs = ref.build_cos_sin_cache(d, 64, 1e4)
    pos = torch.arange(t, dtype=torch.int32)
    slots = torch.arange(t, dtype=torch.int32) + 3
    caches = [torch.zeros(kv4.cache_shape(1, hkv, d, 16), dtype=torch.uint8) for _ in range(2)]
    q0, k0 = q.clone(), k.clone()
    Fn.rope_kv_write(q, k, v, pos, cs, d, True, None, None, 1e-6, *caches, slots)
    half = d // 2
    want = U.turned(q0, None, cs[:t, :half], cs[:t, half:], d, True, 1e-6)
    assert torch.equal(k, k0) and (q.double() - want).abs().max() <= 2 ** -8 * want.abs().max()
    keys, vals = Fn.kv_cache_rows(*caches, slots)
    assert keys.dtype == BF16 and keys.shape == (t, hkv, d)
    turned = U.turned(k0, None, cs[:t, :half], cs[:t, half:], d, True, 1e-6).float().to(BF16)
    assert torch.equal(keys, U.values(turned).float().to(BF16)) and torch.equal(vals, U.values(v).float().to(BF16))


def test_ref_attention():
    torch.manual_seed(3)
    hq, hkv, d, page = 4, 2, 64, 16
    lens, news = [21, 7, 40], [1, 7, 9]
    table = torch.randperm(9)[: 3 * 3].view(3, 3).to(torch.int32)
    caches = [torch.zeros(kv4.cache_shape(9, hkv, d, page), dtype=torch.uint8) for _ in range(2)]
    rows = []
    for s, n in enumerate(lens):
        at = torch.arange(n)
        slots = (table[s].long()[at // page] * page + at % page).to(torch.int32)
        rows.append([torch.randn(n, hkv, d).to(BF16) for _ in range(2)])
        for c, x in zip(caches, rows[-1]):
            kv4.write_rows(c, slots, x)
    q = torch.randn(sum(news), hq * d).to(BF16)
    inp = types.SimpleNamespace(block_table=table, seq_lens=torch.tensor(lens, dtype=torch.int32),
                                query_start_loc=torch.tensor([0, 1, 8, 17], dtype=torch.int32))
    got = Fn.paged_attention(q, *caches, inp, d ** -0.5, hq, d)
    want, tol = U.attention(q.view(-1, hq, d), rows, lens, news, d ** -0.5, hkv, False)
    assert ((got.view_as(want).double() - want).abs() <= tol + 1e-6).all()


def test_rounds_of_expansion():
    assert sm100_kv4.expand_rounds([64, 65, 1], 10, limit=64 * 10 * 3) == [(0, 2, 3), (2, 3, 1)]
    assert sm100_kv4.expand_rounds([1000, 10], 1, limit=1) == [(0, 1, 16), (1, 2, 1)]       # one at least
    assert sm100_kv4.expand_rounds([], 1, 1) == [] and sm100_kv4.expand_rounds([0, 0], 1, 1) == [(0, 2, 0)]


@pytest.mark.parametrize("d,page", [(32, 16), (96, 16), (256, 16), (64, 8), (128, 24), (128, 0), (64, 528)])
def test_shapes_that_a_cache_does_not_take(d, page):
    with pytest.raises(ValueError):
        kv4.cache_shape(4, 2, d, page)


def _call(**over):
    t, hq, hkv, d = 4, 4, 2, 128
    a = dict(q=torch.zeros(t, hq, d, dtype=BF16), k=torch.zeros(t, hkv, d, dtype=BF16), v=torch.zeros(t, hkv, d, dtype=BF16),
             positions=torch.zeros(t, dtype=torch.int32), cos_sin=torch.zeros(8, d), rot_dim=d, neox=True, q_norm_w=None, k_norm_w=None,
             eps=1e-6, k_cache=torch.zeros(kv4.cache_shape(2, hkv, d, 16), dtype=torch.uint8),
             v_cache=torch.zeros(kv4.cache_shape(2, hkv, d, 16), dtype=torch.uint8), slots=torch.zeros(t, dtype=torch.int32))
    a.update(over)
    return sm100_kv4.rope_kv_write(**a)


@pytest.mark.parametrize("over", [
    dict(v_cache=torch.zeros(kv4.cache_shape(3, 2, 128, 16), dtype=torch.uint8)),
    dict(k_cache=torch.zeros(2, 2, 1, 9 * 96, dtype=torch.uint8)),
    dict(k_cache=torch.zeros(2, 4, 1, 9 * 128, dtype=torch.uint8)[:, ::2]),
    dict(v=None), dict(slots=None), dict(rot_dim=24, cos_sin=torch.zeros(8, 24)), dict(rot_dim=4, neox=False, cos_sin=torch.zeros(8, 4)),
    dict(rot_dim=192, cos_sin=torch.zeros(8, 192)), dict(q=torch.zeros(4, 4 * 128 + 4, dtype=BF16)[:, 4:].view(4, 4, 128)),
])
def test_write_refuses(over):
    with pytest.raises(ValueError):
        _call(**over)


@pytest.mark.parametrize("over", [
    dict(q=torch.zeros(4, 4, 128)), dict(k=torch.zeros(4, 1, 128, dtype=BF16)), dict(q=torch.zeros(4, 4, 64, dtype=BF16)),
    dict(slots=torch.zeros(4, dtype=torch.int64)), dict(slots=torch.zeros(3, dtype=torch.int32)), dict(cos_sin=torch.zeros(8, 64)),
    dict(positions=torch.zeros(4, dtype=torch.int64)), dict(q_norm_w=torch.ones(64, dtype=BF16)),
])
def test_write_checks_its_arguments(over):
    with pytest.raises(AssertionError):
        _call(**over)


@pytest.mark.parametrize("power", [-110, -122, -126, -130, -133])
def test_groups_of_tiny_values(power):
    """A scale below 2^-126 counts as 0: its group reads back as its lowest value, within 15 2^-126 of what was written."""
    torch.manual_seed(0)
    x = (torch.randn(40, 1, 64).double() * 2.0 ** power).to(BF16)
    low, scale, _ = U.coded(x)
    got, want = kv4.decode(*kv4.encode(x)), U.values(x)
    flat = (scale < 2.0 ** -126)[..., 0].expand(-1, -1, 64)
    assert flat.all() == flat.any() == (power <= -126)     # spans of 64 normal numbers: some 4.7, 0.3 of a scale at 2^-126, 5 at 2^-122
    assert torch.equal(got[flat].double(), low[..., 0].expand_as(x)[flat]) and float((got.double() - x.double()).abs().max()) <= max(
        15 * 2.0 ** -126, float((want - x.double()).abs().max()))
    torch.testing.assert_close(got[~flat].double(), want[~flat], rtol=2 ** -23, atol=2 ** -149)


def _attend(**over):
    d = 64
    a = dict(q=torch.zeros(5, 4 * d, dtype=BF16), k_cache=torch.zeros(kv4.cache_shape(4, 2, d, 16), dtype=torch.uint8),
             v_cache=torch.zeros(kv4.cache_shape(4, 2, d, 16), dtype=torch.uint8), block_table=torch.zeros(3, 2, dtype=torch.int32),
             seq_lens=torch.ones(3, dtype=torch.int32), query_start_loc=torch.zeros(4, dtype=torch.int32), scale=1.0, num_q_heads=4, head_dim=d,
             num_decode_seqs=1, num_seqs=3, max_q_len=2, max_seq_len=20)
    a.update(over)
    return sm100_kv4.paged_attention(**a)


@pytest.mark.parametrize("over", [
    dict(query_start_loc=torch.zeros(3, dtype=torch.int32)), dict(query_start_loc=torch.zeros(4, dtype=torch.int64)),
    dict(host_lens=[5, 6]), dict(num_decode_seqs=4), dict(num_decode_seqs=-1), dict(block_table=torch.zeros(2, 2, dtype=torch.int32)),
    dict(seq_lens=torch.ones(2, dtype=torch.int32)), dict(q=torch.zeros(0, 256, dtype=BF16)), dict(num_q_heads=3),
])
def test_attention_checks_its_arguments_before_it_launches(over):
    """Indexes that end before the last sequence would be read past their end on the device."""
    with pytest.raises(AssertionError):
        _attend(**over)


def test_write_takes_three_rows_of_positions():
    positions = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(AssertionError):
        _call(positions=positions, mrope_section=[16, 24, 24])
