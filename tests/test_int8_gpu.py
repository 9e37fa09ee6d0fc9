"""8-bit products with scales per token and output channel against their definition in 64 bits (GPU)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F64 = torch.bfloat16, torch.float64
DEV = "cuda"


def quantised(x):
    """(whole numbers, unit) per row in 64 bits: x 127 / max to the nearest, ties to even."""
    x = x.to(F64)
    a = x.abs().amax(1, keepdim=True)
    a = torch.where(a == 0, 1.0, a)
    near = 127 * x.abs() / a                               # 15 by 8 bits: fp64 has every tie exactly
    return torch.round(near) * x.sign(), a / 127


def product(x, w8, ws, bias=None, silu=False):
    """-> (y, tolerance), fp64. Integer sums are exact; a sum to fp32, the scale of the row, that of the row and column and their
    product with it are one rounding of 2^-24 each; the bias another. With the gate: those of its two factors (its own slope is at most 1.1,
    the exponential and the division good to 2^-21), then the result's 2^-8."""
    q, unit = quantised(x)
    y = (q @ w8.to(F64).t()) * unit * ws.to(F64)
    if silu:
        g, u = y.chunk(2, 1)
        y = g * torch.sigmoid(g) * u
        slack = 2 ** -22 * 1.1 * g.abs() * u.abs() + 2 ** -22 * y.abs() + 2 ** -20 * y.abs()
    else:
        slack = 2 ** -22 * y.abs()
        if bias is not None:
            slack = slack + 2 ** -23 * bias.to(F64).abs()
            y = y + bias.to(F64)
    return y, 2 ** -8 * (y.abs() + slack) + slack + 1e-30


def _inputs(m, n, k, seed=0):
    torch.manual_seed(seed + m + n + k)
    x = (torch.randn(m, k, device=DEV) * (0.05 + 5 * torch.rand(m, 1, device=DEV))).to(BF16)
    w8 = torch.randint(-128, 128, (n, k), device=DEV, dtype=torch.int8)
    ws = (0.5 + torch.rand(n, device=DEV)) * 0.01
    return x, w8, ws


@pytest.mark.parametrize("m,k", [(1, 16), (3, 512), (9, 528), (5, 1024), (70, 2048), (2, 4096), (33, 5008), (4, 12288), (3, 28672), (2, 131072)])
def test_rows_are_quantised_to_the_nearest(m, k):
    from gllm_b200.ops import sm100
    torch.manual_seed(k)
    x = (torch.randn(m, k + 8, device=DEV) * 3).to(BF16)[:, 8:]             # rows of a wider tensor
    x[0, 0] = 254 * 2.0 ** -4                                               # 127 / 2^k: many quotients are ties
    x[0, 1:] = torch.randint(-254, 255, (k - 1,), device=DEV).to(BF16) * 2.0 ** -4
    q, s = sm100.int8_quant_rows(x)
    want, unit = quantised(x)
    assert torch.equal(q.to(F64), want)
    torch.testing.assert_close(s.to(F64), unit[:, 0], rtol=2 ** -24, atol=0)


@pytest.mark.parametrize("power", [-90, 0, 117])
def test_every_quotient_of_two_bf16(power):
    """Each largest magnitude beside each other value that does not vanish, ties among them: a bf16 has eight bits."""
    from gllm_b200.ops import sm100
    bits = torch.arange(128, 256, device=DEV, dtype=F64)
    below = torch.cat([bits * 2.0 ** -e for e in range(1, 10)])
    x = torch.cat([bits[:, None], torch.minimum(bits[None], bits[:, None]), -below.expand(128, -1), torch.zeros(128, 15, device=DEV)], 1)
    x = (x * 2.0 ** power).to(BF16)
    q, s = sm100.int8_quant_rows(x)
    assert torch.equal(q.to(F64), torch.round(x.to(F64) * 127 / x[:, :1].to(F64))) and (q == 127).any(1).all()


def test_rows_of_zeros_tiny_rows_and_rows_that_are_no_numbers():
    from gllm_b200.ops import sm100
    x = torch.randn(6, 64, device=DEV).to(BF16)
    x[0], x[1] = 0.0, x[1] * 2.0 ** -110
    x[2, 5], x[3, 9] = float("nan"), float("inf")
    x[4] *= 2.0 ** 120
    q, s = sm100.int8_quant_rows(x)
    assert (q[:2] == 0).all() and torch.isfinite(s[:2]).all() and not torch.isfinite(s[2:4]).any()
    want, unit = quantised(x[4:])
    assert torch.equal(q[4:].to(F64), want)
    w8, ws = torch.ones(16, 64, device=DEV, dtype=torch.int8), torch.ones(16, device=DEV)
    y = sm100.linear_int8(x, w8, ws)
    assert (y[:2] == 0).all() and not torch.isfinite(y[2:4]).any() and torch.isfinite(y[4:]).all()


SHAPES = [(1, 8, 16), (1, 6144, 4096), (2, 136, 80), (17, 264, 1040), (48, 1024, 4096), (64, 4096, 512), (130, 392, 272), (255, 2048, 1024),
          (257, 640, 400), (300, 1000, 2064), (777, 1280, 1024), (1030, 520, 144)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("with_bias", [False, True])
def test_product(m, n, k, with_bias):
    from gllm_b200.layers import functional as Fn
    x, w8, ws = _inputs(m, n, k)
    bias = torch.randn(n, device=DEV).to(BF16) if with_bias else None
    y = Fn.linear(x, (w8, ws), bias)
    want, tol = product(x, w8, ws, bias)
    assert y.dtype == BF16 and ((y.to(F64) - want).abs() <= tol).all()


@pytest.mark.parametrize("m,n,k", [(m, 2 * n, k) for m, n, k in SHAPES])
def test_gated_product(m, n, k):
    from gllm_b200.layers import functional as Fn
    x, w8, ws = _inputs(m, n, k)
    ws = ws / k ** 0.5 * 0.3
    y = Fn.linear_silu_mul(x, (w8, ws))
    want, tol = product(x, w8, ws, silu=True)
    assert y.shape == (m, n // 2) and ((y.to(F64) - want).abs() <= tol).all()


@pytest.mark.parametrize("m", [1, 2, 3, 4])
@pytest.mark.parametrize("n,k", [(16, 16), (48, 528), (2384, 80), (4768, 2064), (272, 4096), (1040, 4112), (64, 12288), (48, 40960)])
@pytest.mark.parametrize("silu", [False, True])
def test_few_rows_give_the_bits_of_the_other_forms(m, n, k, silu):
    """Sums are exact and the same operations follow. More units than warps, fewer than SMs, K that ends inside a warp's loads."""
    from gllm_b200.ops import sm100
    x, w8, ws = _inputs(m, n, k)
    wide = torch.zeros(m, k + 8, dtype=BF16, device=DEV)
    wide[:, 8:] = x
    ws = ws / k ** 0.5 * 0.3 if silu else ws
    bias = None if silu else torch.randn(n, device=DEV).to(BF16)
    y = sm100.linear_int8(wide[:, 8:], w8, ws, bias, silu=silu, plan=(3, 0, 0, 0))
    want, tol = product(x, w8, ws, bias, silu=silu)
    assert ((y.to(F64) - want).abs() <= tol).all()
    assert torch.equal(y, sm100.linear_int8(x, w8, ws, bias, silu=silu, plan=(1, 0, 0, 0)))
    assert torch.equal(y, sm100.linear_int8(x, w8, ws, bias, silu=silu))


def test_one_row_of_a_buffer_of_any_width():
    """The stride of a dimension of one does not matter."""
    from gllm_b200.ops import sm100
    x, w8, ws = _inputs(1, 16, 64)
    odd, out = torch.zeros(1, 67, dtype=BF16, device=DEV)[:, :64], torch.zeros(1, 19, dtype=BF16, device=DEV)[:, :16]
    odd.copy_(x)
    for plan in (None, (1, 0, 0, 0), (2, 16, 1, 108 * 1024)):
        assert torch.equal(sm100.linear_int8(odd, w8, ws, out=out, plan=plan), sm100.linear_int8(x, w8, ws))
    assert torch.equal(sm100.int8_quant_rows(odd)[0], sm100.int8_quant_rows(x)[0])


def test_few_rows_that_are_no_numbers():
    from gllm_b200.ops import sm100
    x, w8, ws = _inputs(4, 16, 64)
    x[0], x[1, 5], x[2, 9] = 0.0, float("nan"), float("inf")
    y = sm100.linear_int8(x, w8, ws, plan=(3, 0, 0, 0))
    want, tol = product(x[3:], w8, ws)
    assert (y[0] == 0).all() and torch.isnan(y[1:3]).all() and ((y[3:].to(F64) - want).abs() <= tol).all()


@pytest.mark.parametrize("plan", [(1, 0, 0, 0), (2, 16, 1, 108 * 1024), (2, 64, 3, 108 * 1024), (2, 32, 8, 220 * 1024), (2, 256, 2, 220 * 1024),
                                  (2, 112, 5, 108 * 1024)])
@pytest.mark.parametrize("silu", [False, True])
def test_forms_by_name(plan, silu):
    """Every form at a size that the choice by size would give to another: the same bits, since the sums are integers."""
    from gllm_b200.ops import sm100
    x, w8, ws = _inputs(139, 1104, 1168)
    ws = ws * 0.01
    y = sm100.linear_int8(x, w8, ws, silu=silu, plan=plan)
    want, tol = product(x, w8, ws, silu=silu)
    assert ((y.to(F64) - want).abs() <= tol).all()
    assert torch.equal(y, sm100.linear_int8(x, w8, ws, silu=silu))


@pytest.mark.parametrize("m", [3, 300])
def test_largest_sums_are_exact(m):
    """127 x -128 over the longest rows: 2.13e9, next to the end of int32."""
    from gllm_b200.ops import sm100
    k = sm100.INT8_MOST_K
    x = torch.full((m, k), 3.0, device=DEV).to(BF16)
    w8 = torch.full((16, k), -128, device=DEV, dtype=torch.int8)
    w8[3] = 127
    ws = torch.full((16,), 2.0 ** -20, device=DEV)
    y = sm100.linear_int8(x, w8, ws)
    want, tol = product(x, w8, ws)
    assert ((y.to(F64) - want).abs() <= tol).all()


@pytest.mark.parametrize("m", [5, 400])
def test_strided_rows_results_in_place_and_rows_behind(m):
    from gllm_b200.ops import sm100
    x, w8, ws = _inputs(m, 264, 256)
    wide = torch.randn(m, 512, device=DEV).to(BF16)
    wide[:, 128:384] = x
    out = torch.full((m + 3, 512), 7.0, dtype=BF16, device=DEV)
    y = sm100.linear_int8(wide[:, 128:384], w8, ws, out=out[:m, 64:328])
    want, tol = product(x, w8, ws)
    assert y.data_ptr() == out[:m, 64:328].data_ptr() and ((y.to(F64) - want).abs() <= tol).all()
    assert (out[m:] == 7).all() and (out[:, :64] == 7).all() and (out[:, 328:] == 7).all()


def test_no_rows():
    from gllm_b200.ops import sm100
    _, w8, ws = _inputs(1, 64, 64)
    assert sm100.linear_int8(torch.empty(0, 64, dtype=BF16, device=DEV), w8, ws).shape == (0, 64)
    assert sm100.int8_quant_rows(torch.empty(0, 64, dtype=BF16, device=DEV))[0].shape == (0, 64)


def test_captured_products_on_two_streams():
    """Two graphs replayed at once: each has its quantised rows in memory of its own."""
    from gllm_b200.ops import sm100
    runs = []
    for m in (7, 600):
        x, w8, ws = _inputs(m, 1024, 2048, seed=m)
        out = torch.empty(m, 1024, dtype=BF16, device=DEV)
        sm100.linear_int8(x, w8, ws, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            sm100.linear_int8(x, w8, ws, out=out)
        runs.append((graph, x, w8, ws, out, torch.cuda.Stream()))
    for turn in range(3):
        for graph, x, w8, ws, out, stream in runs:
            x.copy_(torch.randn_like(x.float()).to(BF16))
            out.zero_()
        torch.cuda.synchronize()
        for graph, x, w8, ws, out, stream in runs:
            with torch.cuda.stream(stream):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for graph, x, w8, ws, out, stream in runs:
            want, tol = product(x, w8, ws)
            assert ((out.to(F64) - want).abs() <= tol).all()


@pytest.mark.parametrize("plan", [(1, 0, 0, 0), (2, 64, 2, 108 * 1024)])
def test_waits_that_run_out_are_reported(plan):
    from gllm_b200.ops import lib as _lib, sm100
    x, w8, ws = _inputs(300, 1024, 4096)
    assert sm100.waits_given_up() == 0
    try:
        _lib.watch_waits(0)
        sm100.linear_int8(x, w8, ws, plan=plan)
        torch.cuda.synchronize()
        assert _lib.waits_gave_up(clear=True)
    finally:
        _lib.watch_waits()
    want, tol = product(x, w8, ws)
    assert ((sm100.linear_int8(x, w8, ws, plan=plan).to(F64) - want).abs() <= tol).all() and not _lib.waits_gave_up()


@pytest.mark.parametrize("m", [1, 4, 7, 200, 1200])
@pytest.mark.parametrize("n,k", [(64, 256), (2048, 4096), (9728, 1024)])
def test_weights_quantised_just_before_their_product(m, n, k):
    """The quantiser's pair is a weight: both calls behind one another in one graph, where no gap of the host lies between them, with other
    weights at every replay. The same bits as with all the time in the world between them."""
    from gllm_b200.layers import functional as Fn
    from gllm_b200.ops import sm100
    torch.manual_seed(m + n)
    x, w = torch.randn(m, k, device=DEV).to(BF16), torch.empty(n, k, dtype=BF16, device=DEV)
    weights = [(torch.randn(n, k, device=DEV) * 0.1).to(BF16) for _ in range(3)]
    w.copy_(weights[0])
    Fn.linear(x, sm100.int8_quant_rows(w))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s = sm100.int8_quant_rows(w)
        y = Fn.linear(x, (q, s))
    for turn in range(6):
        w.copy_(weights[turn % 3])
        q.zero_()                                          # what a product that came too early would find
        graph.replay()
        got = y.clone()
        torch.cuda.synchronize()
        q1, s1 = sm100.int8_quant_rows(weights[turn % 3])
        torch.cuda.synchronize()
        assert torch.equal(q, q1) and torch.equal(s, s1)
        assert torch.equal(got, Fn.linear(x, (q1, s1)))


@pytest.mark.parametrize("m,k", [(24, 64), (24, 2048), (3, 32768)])
def test_small_rows_are_quantised_as_the_plain_form_does(m, k):
    """Largest magnitudes on either side of 2^-100, the least step: codes and scales of the plain form, in the product of few rows too."""
    from gllm_b200.ops import ref, sm100
    torch.manual_seed(k)
    x = torch.randn(m, k, device=DEV, dtype=F64).clamp(-1, 1)
    x[:, 0] = 1.0
    x = (x * 2.0 ** -(96 + torch.arange(m, device=DEV) % 12).double()[:, None]).to(BF16)
    q, s = sm100.int8_quant_rows(x)
    want_q, want_s = ref.int8_quant_rows(x.cpu())
    assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s) and (want_q[5:] != 0).any() == (m > 5)
    w8 = torch.randint(-128, 128, (32, k), device=DEV, dtype=torch.int8)
    ws = torch.full((32,), 2.0 ** 60, device=DEV)
    for rows in (x[:1], x[m // 4:m // 4 + 2], x):
        y = sm100.linear_int8(rows, w8, ws)
        want = (ref.int8_quant_rows(rows.cpu())[0].double() @ w8.cpu().double().t()) * ref.int8_quant_rows(rows.cpu())[1].double()[:, None] * 2.0 ** 60
        # the definition's value through one rounding to bf16 (2^-8) behind three of fp32
        assert ((y.cpu().double() - want).abs() <= (2 ** -8 + 2 ** -22) * want.abs()).all()
