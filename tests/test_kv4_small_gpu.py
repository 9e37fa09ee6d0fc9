"""Rotary write to a 4-bit cache at the lower end of bf16 (GPU)."""
import pytest
import torch

from gllm_b200.ops import kv4
from tests.test_kv4_gpu import BF16, DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rot", [0, 1])
@pytest.mark.parametrize("power", [-100, -118, -122, -123, -124, -126, -130, -133])
def test_write_of_tiny_values_gives_the_plain_forms_bits(power, rot, d):
    """Scales on either side of 2^-126, below which they count as 0; many spans are 15 times a number halfway between two scales."""
    from gllm_b200.ops import sm100_kv4
    t, h = 96, 2
    torch.manual_seed(power + d)
    v = (torch.randn(t, h, d, device=DEV).double() * 2.0 ** power).to(BF16)
    ties = (torch.randint(128, 256, (t // 2, h), device=DEV) * 2 + 1).double() * 15 * 2.0 ** (power - 12)          # nine bits of quotient
    v[: t // 2, :, 1:64] = 0
    v[: t // 2, :, 0] = (ties / 16).to(BF16)
    v[: t // 2, :, 1] = (v[: t // 2, :, 0].double() - ties).to(BF16)
    k, q = v.flip(0).contiguous(), torch.zeros(t, 2, d, dtype=BF16, device=DEV)
    pos, slots = torch.zeros(t, dtype=torch.int32, device=DEV), torch.arange(t, dtype=torch.int32, device=DEV) + 5
    turn = torch.cat((torch.ones(2, d // 2), torch.zeros(2, d // 2)), 1).to(DEV) if rot else None                     # by nothing
    got = [torch.zeros(kv4.cache_shape(8, h, d, 16), dtype=torch.uint8, device=DEV) for _ in range(2)]
    want = [c.clone() for c in got]
    sm100_kv4.rope_kv_write(q, k, v, pos, turn, rot * d, True, None, None, 1e-6, *got, slots)
    for c, x in zip(want, (k, v)):
        kv4.write_rows(c, slots, x)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for rows, c in zip(sm100_kv4.kv_cache_rows(*got, slots), want):
        assert torch.equal(rows, kv4.read_rows(c, slots).to(BF16))
