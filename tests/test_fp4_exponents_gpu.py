"""4-bit weights with the smallest exponents: the values, the product and its gradient belong to one weight."""
import pytest
import torch

from gcore_b200.ops import quant
from test_fp4_products_gpu import bound, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exponent", [0, 1, 2, 3])
@pytest.mark.parametrize("T", [3, 40, 300])
def test_smallest_exponents(exponent, T):
    N, K = 200, 256
    g = torch.Generator(device="cuda").manual_seed(exponent)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    e = torch.full((N, K // 32), exponent, dtype=torch.uint8, device="cuda")
    e[::7, 3] = 40
    W = quant.Fp4Weight(codes, e)
    on_cpu = quant.Fp4Weight(codes.cpu(), e.cpu()).values(torch.float32)
    assert torch.equal(W.values().view(torch.int16).cpu(), on_cpu.bfloat16().view(torch.int16))
    w = on_cpu.double().cuda()
    x = (rand(T, K, seed=1) * 2.0 ** 110).bfloat16().requires_grad_()
    y = quant.linear_fp4(x, W)
    want = x.detach().double() @ w.t()
    assert ((y.detach().double() - want).abs() <= bound(x.detach().double(), w, want, torch.bfloat16)).all()
    dy = (rand(T, N, seed=2) * 2.0 ** 110).bfloat16()
    dx = torch.autograd.grad(y, x, dy)[0]
    want = dy.double() @ w
    tol = (N / 16 + 16) * 2.0 ** -23 * (dy.double().abs() @ w.abs()) + 1e-30
    assert ((dx.double() - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol)).all()
