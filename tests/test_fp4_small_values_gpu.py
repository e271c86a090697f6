"""4-bit products of activations whose groups are tiny, and 4-bit weights with the smallest exponents, against 64 bits.

Tolerances are those of ``test_fp4_products_gpu``.  The two e4m3 terms of a group share an exponent that is never below 4, 2^-123, and
the lo term's smallest step is 2^-9 / 16 of it: below that exponent a value is off by up to 2^-14 2^-123 more."""
import pytest
import torch

from gcore_b200.ops import quant
from test_fp4_products_gpu import bound, rand

pytestmark = pytest.mark.gpu


def large_weight(N, K, exponent):
    """Random codes, all groups with one exponent."""
    g = torch.Generator(device="cuda").manual_seed(N + K)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    return quant.Fp4Weight(codes, torch.full((N, K // 32), exponent, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("T", [1, 5, 40, 200])
@pytest.mark.parametrize("exponent", [1, 4, 10, 11, 12, 13, 14])
def test_groups_of_tiny_values(T, exponent):
    """The largest of each group has this biased exponent and a mantissa on either side of e4m3's largest, 1.75."""
    N, K = 130, 256
    W = large_weight(N, K, 220)
    w = W.values(torch.float32).double()
    x = rand(T, K, seed=exponent).bfloat16() * 2.0 ** (exponent - 128)
    mantissas = torch.tensor([0x5f, 0x60, 0x61, 0x62, 0x70, 0x7e, 0x7f, 0x00], device="cuda")
    tops = (exponent * 128 + mantissas).to(torch.int16).view(torch.bfloat16)
    x = torch.minimum(x.abs(), tops[None].repeat_interleave(32, 1)) * torch.sign(x)
    x[:, ::32] = tops * torch.where(torch.arange(T, device="cuda")[:, None] % 2 == 0, 1.0, -1.0).bfloat16()
    y = x.double() @ w.t()
    b = bound(x.double(), w, y, torch.bfloat16) + 2.0 ** -137 * w.abs().sum(1)
    assert ((quant.linear_fp4(x, W).double() - y).abs() <= b).all()
