"""Derivatives of the low-precision serving operators: what carries one, what refuses one."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from gcore_b200.ops import fused, quant


def rows(T, W, seed):
    return torch.randn(T, W, generator=torch.Generator().manual_seed(seed))


def test_operators_without_derivatives_refuse_tangents():
    x, gain = rows(3, 256, 1), torch.ones(256)
    W = quant.Fp4Weight.of(rows(40, 256, 2))
    q, s = quant.quant_act_1x32(x)
    with fw.dual_level():
        d = fw.make_dual(x, x)
        for call in (lambda: fused.rmsnorm_fp8(d, gain), lambda: fused.rmsnorm_fp8(x, gain, residual=d),
                     lambda: fused.rmsnorm_fp8(x, fw.make_dual(gain, gain)), lambda: fused.swiglu_fp8(d),
                     lambda: quant.gemm_fp4(q, s, W, fw.make_dual(x[0, :40], x[0, :40]))):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
        fused.rmsnorm_fp8(x, gain)   # others of the same level are none of its concern


def test_product_carries_tangents_and_refuses_a_second_derivative(monkeypatch):
    W = quant.Fp4Weight.of(rows(40, 256, 2))
    w = W.values(torch.float32)
    x, t, b = rows(3, 256, 1), rows(3, 256, 3), rows(1, 40, 4)[0]
    with fw.dual_level():
        y = fw.unpack_dual(quant.linear_fp4(fw.make_dual(x, t), W))
        assert torch.allclose(y.tangent, t @ w.t(), rtol=1e-5, atol=1e-5)
    # the function that a GPU's products go through, with their definitions in place of the kernels
    monkeypatch.setattr(quant, "_fp4_product", lambda x2, xs, weight, bias, dtype:
                        torch.nn.functional.linear(x2, w, bias).to(dtype))
    monkeypatch.setattr(quant, "_fp4_dgrad", lambda dy, weight: dy.detach().float() @ w)
    with fw.dual_level():
        y = fw.unpack_dual(quant._LinearFp4Tangent.apply(fw.make_dual(x, t), W, fw.make_dual(b, 2 * b)))
        assert torch.allclose(y.tangent, t @ w.t() + 2 * b, rtol=1e-5, atol=1e-5)
        y = fw.unpack_dual(quant._LinearFp4Tangent.apply(x, W, fw.make_dual(b, 2 * b)))
        assert y.tangent.shape == (3, 40) and torch.allclose(y.tangent.float(), (2 * b).expand(3, 40), rtol=2 ** -8)
    x.requires_grad_()
    g, = torch.autograd.grad(quant._LinearFp4.apply(x, W, None).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):   # not x's gradient alone, without the product's part
        (g.sum() + x.sum()).backward()


def test_quantiser_refuses_a_gradient_and_a_tangent():
    x = rows(3, 64, 1)
    want = quant.quant_act_1x32(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        quant.quant_act_1x32(x.clone().requires_grad_())
    with fw.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
        quant.quant_act_1x32(fw.make_dual(x, x))
    with torch.no_grad():
        q, s = quant.quant_act_1x32(x.clone().requires_grad_())
    assert not q.requires_grad and torch.equal(q.float(), want[0].float()) and torch.equal(s.float(), want[1].float())
