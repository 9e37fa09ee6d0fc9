"""Decode attention over a 4-bit cache within the roundings that it makes, and what a step allocates (GPU)."""
import pytest
import torch

from tests import kv4_util as U
from tests.test_kv4_gpu import BF16, DEV, _attend, _filled

pytestmark = pytest.mark.gpu
F64 = torch.float64


def _bound(q, rows, lens, scale, hkv):
    """q [B, Hq, D] of one new token a sequence -> (result, tolerance without its last rounding), fp64.

    Codes and factors of queries enter the products of a score as they are (factors 2^-28 of a head's largest and more; below, they are good to
    2^-36 of it). D / 16 instructions add 16 products each to what is there, with at most 2^-22 of the sum of the magnitudes, and as much again
    goes to scales, low ends, the exponent and the subtraction of the maximum, eight operations: (D / 16 + 8) 2^-22 of sum |q| (s c + |low|). A
    probability times a value's scale is rounded to fp16 (2^-11), sums over n keys take n / 16 steps of 2^-23 and 32 to be joined, products
    below fp16's normal numbers are good to 2^-31 of the largest that can stand beside them, and the result is rounded once: 2^-8, over all
    values 2^-8 / sqrt 3 of their norm (uniform within half a step)."""
    out, tol = [], []
    for s, ((k, v), n) in enumerate(zip(rows, lens)):
        hq, d = q.shape[1:]
        qq = q[s].to(F64).unflatten(0, (hkv, hq // hkv))
        kk, vv = U.values(k[:n]), U.values(v[:n])
        klow, ks, kc = U.coded(k[:n])
        vlow, vs, vc = U.coded(v[:n])
        p = (torch.einsum("hgd,khd->hgk", qq, kk) * scale).softmax(-1)
        o = torch.einsum("hgk,khd->hgd", p, vv)
        steps = torch.einsum("hgk,khd->hgd", p, (vs * vc).flatten(-2))
        size = steps + torch.einsum("hgk,khd->hgd", p, vlow.expand_as(vc).flatten(-2).abs())
        dz = (d / 16 + 8) * 2.0 ** -22 * (torch.einsum("hgd,khd->hgk", qq.abs(), (ks * kc + klow.abs()).flatten(-2)) * scale).amax(-1, keepdim=True)
        least = 2.0 ** -31 * 15 * n * vs.amax((0, 2, 3))[:, None, None] * p.amax(-1, keepdim=True)
        slack = 2.0 ** -11 * steps + least + (2 * dz + (n / 16 + 32) * 2.0 ** -23) * size
        out.append(o.flatten(0, 1))
        tol.append(slack.flatten(0, 1))
    return torch.stack(out), torch.stack(tol)


@pytest.mark.parametrize("parity", [0, 1])
@pytest.mark.parametrize("loud", [1.0, 16.0, 32.0])
@pytest.mark.parametrize("lens,hq,hkv,d", [([700], 8, 2, 128), ([40, 1500, 333], 7, 1, 64), ([900, 64], 32, 2, 128)])
def test_queries_with_a_few_large_dims(lens, hq, hkv, d, loud, parity):
    """A sixteenth of a head's dims are `loud` times the rest, all of them even or all odd: trained models have such dims."""
    caches, rows, table = _filled(lens, hkv, d, 16)
    q = torch.randn(len(lens), hq, d, device=DEV)
    q[..., parity::16] *= loud
    q = q.to(BF16)
    got = _attend(q.flatten(1), caches, table, lens, [1] * len(lens), len(lens), hq, hkv, d)
    want, slack = _bound(q, rows, lens, d ** -0.5, hkv)
    off = (got.view_as(want).to(F64) - want).abs()
    assert float((off / (slack + 2.0 ** -8 * (want.abs() + slack))).max()) <= 1
    assert off.norm() <= 1.1 * 2.0 ** -8 / 3 ** 0.5 * want.norm() + slack.norm(), (off.norm() / want.norm(), slack.norm() / want.norm())


def test_rounds_of_prompts_allocate_what_is_counted(monkeypatch):
    """Several rounds of expanded prompts, of unequal sizes: no more is live at a time than `scratch_bytes`, by which the engine sizes its pages."""
    from gllm_b200.ops import sm100_kv4
    hq, hkv, d = 8, 8, 128
    monkeypatch.setattr(sm100_kv4, "EXPAND_BYTES", 4 * hkv * d * 4096)
    lens, news = [2000, 2096, 4000, 3000, 1000, 4096], [3, 40, 1, 7, 200, 9]
    caches, rows, table = _filled(lens, hkv, d, 16)
    q = torch.randn(sum(news), hq * d, device=DEV).to(BF16)
    want = _attend(q, caches, table, lens, news, 0, hq, hkv, d)
    del want
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = _attend(q, caches, table, lens, news, 0, hq, hkv, d)
    most = torch.cuda.max_memory_allocated() - before - got.numel() * 2
    counted = sm100_kv4.scratch_bytes(hkv, d, max(lens))
    assert most <= counted, (most, counted)
