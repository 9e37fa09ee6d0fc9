"""8-bit products: plain form and refusals (CPU)."""
import pytest
import torch

from gllm_b200.layers import functional as Fn
from gllm_b200.ops import ref, sm100

BF16 = torch.bfloat16


def test_plain_form():
    torch.manual_seed(0)
    x = torch.randn(5, 48).to(BF16)
    x[2] = 0.0
    x[0, 0], x[0, 1] = 254.0, 1.0                          # 127 / 254: a tie, to the even 0
    q, s = ref.int8_quant_rows(x)
    assert int(q[0, 0]) == 127 and int(q[0, 1]) == 0 and (q[2] == 0).all() and float(s[0]) == 2.0
    w8 = torch.randint(-128, 128, (32, 48), dtype=torch.int8)
    ws = torch.rand(32) * 0.01
    b = torch.randn(32).to(BF16)
    want = (q.double() * s.double()[:, None]) @ (w8.double() * ws.double()[:, None]).t()
    y = Fn.linear(x, (w8, ws), b)
    assert ((y.double() - want - b.double()).abs() <= 2 ** -8 * (want + b.double()).abs() + 1e-5).all()
    g, u = want.chunk(2, 1)
    y = Fn.linear_silu_mul(x, (w8, ws))
    assert ((y.double() - g * torch.sigmoid(g) * u).abs() <= 2 ** -8 * (g * u).abs() + 1e-5).all()
    out = torch.zeros(5, 32).to(BF16)
    assert Fn.linear(x, (w8, ws), out=out) is out and out.any()


def _call(**over):
    a = dict(x=torch.zeros(4, 64, dtype=BF16), w8=torch.zeros(32, 64, dtype=torch.int8), w_scale=torch.ones(32))
    a.update(over)
    return sm100.linear_int8(**a)


@pytest.mark.parametrize("over", [
    dict(x=torch.zeros(4, 40, dtype=BF16), w8=torch.zeros(32, 40, dtype=torch.int8)),
    dict(x=torch.zeros(1, sm100.INT8_MOST_K + 16, dtype=BF16), w8=torch.zeros(8, sm100.INT8_MOST_K + 16, dtype=torch.int8)),
    dict(x=torch.zeros(4, 68, dtype=BF16)[:, 4:]), dict(w8=torch.zeros(12, 64, dtype=torch.int8), w_scale=torch.ones(12)),
    dict(w8=torch.zeros(24, 64, dtype=torch.int8), w_scale=torch.ones(24), silu=True), dict(bias=torch.zeros(32, dtype=BF16), silu=True),
    dict(out=torch.zeros(4, 36, dtype=BF16)[:, 4:]), dict(w_scale=torch.ones(33)[1:]),
])
def test_refuses(over):
    with pytest.raises(ValueError):
        _call(**over)


@pytest.mark.parametrize("over", [
    dict(x=torch.zeros(4, 64)), dict(w8=torch.zeros(32, 64, dtype=torch.uint8)), dict(w8=torch.zeros(32, 48, dtype=torch.int8)),
    dict(w_scale=torch.ones(31)), dict(w_scale=torch.ones(32, dtype=BF16)), dict(bias=torch.zeros(32)), dict(bias=torch.zeros(16, dtype=BF16)),
    dict(out=torch.zeros(4, 16, dtype=BF16)), dict(out=torch.zeros(4, 32)), dict(w8=torch.zeros(64, 64, dtype=torch.int8)[::2]),
])
def test_checks_its_arguments(over):
    with pytest.raises(AssertionError):
        _call(**over)


@pytest.mark.parametrize("rows,form", [(9, 0), (5, 3), (1, 4), (1, 2)])
def test_the_entry_refuses_before_it_launches(rows, form):
    """No room for the quantised rows; more rows than the form for few takes; no such form; a cluster without rows."""
    from gllm_b200.ops import lib
    at = 1 << 20
    assert lib.load().gllm_linear_int8(at, 64, None, None, at, at, at, 16, rows, 16, 64, None, False, form, 0, 0, 0, None) == 1


def _definition(x):
    """(whole numbers, scales), fp64: the step is the largest magnitude, 2^-100 at least, / 127."""
    a = x.double().abs().amax(1, keepdim=True).clamp_min(2.0 ** -100)
    return torch.round(127 * x.double() / a), a / 127


def test_small_rows_have_the_least_step():
    """Rows whose largest magnitude lies on either side of 2^-100, zeros and rows that are not finite."""
    torch.manual_seed(1)
    x = torch.randn(12, 64).clamp(-1, 1)
    x[:, 0] = 1.0
    x = (x.double() * 2.0 ** -torch.arange(98, 110).double()[:, None]).to(BF16)
    x = torch.cat([x, torch.zeros(1, 64, dtype=BF16)])
    q, s = ref.int8_quant_rows(x)
    want, scale = _definition(x)
    assert torch.equal(q.double(), want) and (q[3] != 0).any() and (q[:, 0] <= 127).all()
    torch.testing.assert_close(s.double(), scale[:, 0], rtol=2 ** -24, atol=0)
    bad = torch.randn(2, 64).to(BF16)
    bad[0, 3], bad[1, 4] = float("nan"), float("-inf")
    q, s = ref.int8_quant_rows(bad)
    assert (q == 0).all() and not torch.isfinite(s).any()
