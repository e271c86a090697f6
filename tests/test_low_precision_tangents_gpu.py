"""Forward-mode derivatives of the low-precision serving operators on the GPU: carried or refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from gcore_b200.ops import fused, quant
from test_fp4_products_gpu import bound, rand, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [2, 40, 200])
def test_product_carries_tangents(T):
    W = weight(300, 256, seed=1)
    w = W.values(torch.float32).double()
    x, t = rand(T, 256, seed=2).bfloat16(), rand(T, 256, seed=3).bfloat16()
    b, bt = rand(300, seed=4).bfloat16(), rand(300, seed=5).bfloat16()
    want = t.double() @ w.t()
    with fw.dual_level():
        y = fw.unpack_dual(quant.linear_fp4(fw.make_dual(x, t), W))
        z = fw.unpack_dual(quant.linear_fp4(x, W, fw.make_dual(b, bt)))
        both = fw.unpack_dual(quant.linear_fp4(fw.make_dual(x, t), W, fw.make_dual(b, bt)))
    assert torch.equal(y.primal, quant.linear_fp4(x, W)) and torch.equal(z.tangent, bt.expand(T, 300))
    assert ((y.tangent.double() - want).abs() <= bound(t.double(), w, want, torch.bfloat16)).all()
    want = want + bt.double()
    assert ((both.tangent.double() - want).abs() <= bound(t.double(), w, want, torch.bfloat16)).all()


def test_operators_without_derivatives_refuse_tangents():
    x = rand(3, 256, seed=1).bfloat16()
    gain = torch.ones(256, device="cuda").bfloat16()
    W = weight(40, 256, seed=2)
    q, s = quant.quant_act_1x32(x)
    with fw.dual_level():
        d = fw.make_dual(x, x)
        for call in (lambda: fused.rmsnorm_fp8(d, gain), lambda: fused.rmsnorm_fp8(x, gain, residual=d),
                     lambda: fused.rmsnorm_fp8(x, fw.make_dual(gain, gain)), lambda: fused.swiglu_fp8(d),
                     lambda: quant.quant_act_1x32(d), lambda: quant.gemm_fp4(q, s, W, fw.make_dual(x[0, :40], x[0, :40]))):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
