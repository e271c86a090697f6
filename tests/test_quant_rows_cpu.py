"""Norm and activation with e4m3 outputs, 4-bit weights and their products: the PyTorch definitions and every refusal."""
import pytest
import torch

from gcore_b200.ops import fused, quant


def rows(T, W, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, W, generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rounded_norm_is_the_norm_followed_by_the_quantiser(dtype):
    x, r, w = rows(5, 256, 0).to(dtype), rows(5, 256, 1).to(dtype), (1 + 0.1 * rows(1, 256, 2)[0]).to(dtype)
    q, s, out = fused.rmsnorm_fp8(x, w, 1e-5, r, as_rounded=True)
    y, res = fused.rmsnorm(x, w, 1e-5, r)
    q0, s0 = quant.act_quant_1x128_ref(y)
    assert torch.equal(q.float(), q0.float()) and torch.equal(s, s0) and torch.equal(out, res)
    q, s, out = fused.rmsnorm_fp8(x, w, 1e-5)
    assert out is x and q.dtype == torch.float8_e4m3fn and s.shape == (5, 2)


def test_rounded_activation_is_the_activation_followed_by_the_quantiser():
    x = rows(3, 512, 3).to(torch.bfloat16).view(3, 1, 512)
    q, s = fused.swiglu_fp8(x, as_rounded=True)
    q0, s0 = quant.act_quant_1x128_ref(fused.swiglu(x).view(3, 256))
    assert q.shape == (3, 1, 256) and torch.equal(q.float().view(3, 256), q0.float()) and torch.equal(s.view(3, 2), s0)


def test_power_of_two_scales_are_the_smallest_that_fit():
    x = torch.zeros(1, 32 * 8)
    tops = [448.0, 448.0 * (1 + 2 ** -23), 1.0, 2.0 ** -40, 0.0, 3e38, float("inf"), float("nan")]
    for i, t in enumerate(tops):
        x[0, 32 * i + 5] = -t
    q, s = quant.quant_act_1x32(x)
    assert s.dtype == torch.float8_e8m0fnu
    e = s.view(torch.uint8)[0].tolist()
    # 2^-8 * 1.75 * 2^8 = 1.75 >= 1; the floor of 1e-10 has the exponent -42; 3e38 = 1.76 * 2^127
    assert e == [127, 128, 119, 85, 85, 247, 255, 255]
    dq = quant.dequant_1x128(torch.zeros(1, 128), torch.zeros(1, 1))  # the block-fp8 form is untouched
    assert dq.abs().sum() == 0
    back = q.float().view(8, 32) * s.float()[0][:, None]
    assert back[0, 5] == -448 and back[2, 5] == -1 and back[4].abs().sum() == 0 and back[6:].isnan().all()
    assert abs(back[1, 5] + 448) <= 448 / 16


def test_weight_keeps_codes_exponents_and_values():
    for N, K in ((1, 32), (40, 96), (130, 256), (257, 160)):
        w = rows(N, K, N + K)
        W = quant.Fp4Weight.of(w)
        codes, s, dq = quant.fp4_quant_1x32_ref(w)
        assert W.shape == (N, K) and W.padded % 128 == 0 and W.codes.data_ptr() % 32 == 0
        assert torch.equal(W.values(torch.float32), dq) and torch.equal(W.values(), dq.bfloat16())
        e = W.exponents
        assert torch.equal(torch.exp2(e.float() - 127), s.view(N, K // 32))
        # row r of a tile at (r % 32) * 16 + (r / 32) * 4
        r, c = N - 1, K // 32 - 1
        flat = W.tiles.reshape(-1)
        at = (((r >> 7) * (W.padded // 128) + (c >> 2)) * 512) + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (c & 3)
        assert flat[at] == e[r, c]
        again = quant.Fp4Weight(W.codes[:, :K // 2], e.contiguous().view(torch.float8_e8m0fnu))
        assert torch.equal(again.values(torch.float32), dq)


def test_product_and_its_gradient():
    W = quant.Fp4Weight.of(rows(37, 96, 1))
    dq = W.values(torch.float32)
    x = rows(6, 96, 2).view(2, 3, 96).requires_grad_()
    b = rows(1, 37, 3)[0].requires_grad_()
    y = quant.linear_fp4(x, W, b)
    assert y.shape == (2, 3, 37) and torch.allclose(y, x @ dq.t() + b, rtol=1e-6, atol=1e-6)
    gx, gb = torch.autograd.grad(y, (x, b), torch.ones_like(y))
    assert torch.allclose(gx, dq.sum(0).expand(2, 3, 96), rtol=1e-5, atol=1e-5) and torch.equal(gb, torch.full((37,), 6.0))
    q, s = quant.quant_act_1x32(x.detach())
    xq = (q.float().unflatten(-1, (-1, 32)) * s.float()[..., None]).flatten(-2)
    assert torch.allclose(quant.gemm_fp4(q, s, W, out_dtype=torch.float32), xq @ dq.t(), rtol=1e-6, atol=1e-6)
    assert quant.linear_fp4(x[:, :0], W).shape == (2, 0, 37)


def test_refusals():
    x, w = rows(2, 256, 0), torch.ones(256)
    with pytest.raises(ValueError, match="scales"):
        fused.rmsnorm_fp8(x, w, scales="fp16")
    with pytest.raises(ValueError, match="multiple of 128"):
        fused.rmsnorm_fp8(x[:, :192], w[:192])
    with pytest.raises(ValueError, match="multiple of 32"):
        fused.rmsnorm_fp8(x[:, :40], w[:40], scales="e8m0")
    with pytest.raises(ValueError, match="gain"):
        fused.rmsnorm_fp8(x, w[:128])
    with pytest.raises(ValueError, match="residual"):
        fused.rmsnorm_fp8(x, w, residual=x[:1])
    with pytest.raises(RuntimeError, match="no gradient"):
        fused.rmsnorm_fp8(x.clone().requires_grad_(), w)
    with torch.no_grad():
        fused.rmsnorm_fp8(x.clone().requires_grad_(), w)
    with pytest.raises(ValueError, match="gate"):
        fused.swiglu_fp8(x[:, :255])
    with pytest.raises(ValueError, match="multiple of 128"):
        fused.swiglu_fp8(x[:, :128])
    with pytest.raises(RuntimeError, match="no gradient"):
        fused.swiglu_fp8(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="multiple of 32"):
        quant.quant_act_1x32(x[:, :33])
    W = quant.Fp4Weight.of(rows(8, 64, 1))
    codes, e = W.codes[:, :32].contiguous(), W.exponents.contiguous()
    for bad in ((codes.float(), e), (codes[0], e), (codes[:, :20], e), (codes, e[:, :1]), (codes, e.int()), (codes[:0], e[:0])):
        with pytest.raises(ValueError, match="Fp4Weight"):
            quant.Fp4Weight(*bad)
    with pytest.raises(ValueError, match="groups of 32"):
        quant.Fp4Weight.of(rows(4, 40, 0))
    with pytest.raises(TypeError, match="Fp4Weight"):
        quant.linear_fp4(rows(2, 64, 0), torch.ones(8, 64))
    with pytest.raises(ValueError, match="against"):
        quant.linear_fp4(rows(2, 32, 0), W)
    with pytest.raises(ValueError, match="bias"):
        quant.linear_fp4(rows(2, 64, 0), W, torch.ones(7))
    q, s = quant.quant_act_1x32(rows(2, 64, 0))
    with pytest.raises(ValueError, match="float8"):
        quant.gemm_fp4(q.float(), s, W)
    with pytest.raises(ValueError, match="float8"):
        quant.gemm_fp4(q, s.float(), W)
    with pytest.raises(ValueError, match="scales"):
        quant.gemm_fp4(q, s[:1], W)
    with pytest.raises(ValueError, match="results"):
        quant.gemm_fp4(q, s, W, out_dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no gradient"):
        quant.gemm_fp4(q, s, W, torch.ones(8, requires_grad=True))


def test_single_rows_without_a_batch():
    x, w = rows(1, 256, 0)[0], torch.ones(256)
    q, s, out = fused.rmsnorm_fp8(x, w, residual=x)
    assert q.shape == (256,) and s.shape == (2,) and out.shape == (256,)
    q, s = fused.swiglu_fp8(x, scales="e8m0")
    assert q.shape == (128,) and s.shape == (4,)
    W = quant.Fp4Weight.of(rows(8, 256, 1))
    q, s = quant.quant_act_1x32(x)
    assert quant.linear_fp4(x, W).shape == (8,) and quant.gemm_fp4(q, s, W).shape == (8,)


def test_gemm_fp4_refuses_activations_and_scales_that_want_a_gradient():
    q, s = quant.quant_act_1x32(rows(3, 64, 5))
    W = quant.Fp4Weight.of(rows(8, 64, 6))
    with pytest.raises(RuntimeError, match="no gradient"):
        quant.gemm_fp4(q.clone().requires_grad_(), s, W)
    with pytest.raises(RuntimeError, match="no gradient"):
        quant.gemm_fp4(q, s.clone().requires_grad_(), W)
    with torch.no_grad():
        assert torch.equal(quant.gemm_fp4(q.clone().requires_grad_(), s, W), quant.gemm_fp4(q, s, W))
