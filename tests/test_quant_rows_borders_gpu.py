"""Norms and activations that end in e4m3 where a rounding or a range decides: ties between two codes, gates far below zero."""
import pytest
import torch

from gcore_b200.ops import fused, quant
from test_quant_rows_gpu import check, rand

pytestmark = pytest.mark.gpu


def e4m3_of(v):
    """The nearest e4m3 value, halves to even, of 64-bit values within 448."""
    step = torch.exp2(torch.frexp(v)[1].clamp_min(-5).double() - 4)
    return torch.round(v / step) * step


@pytest.mark.parametrize("T,H,residual", [(1, 3584, True), (64, 128, False), (301, 1536, False), (33, 7168, True), (4, 16384, False)])
def test_codes_of_a_norm_are_those_of_the_definition(T, H, residual):
    """A value over its group's largest does not depend on the norm, and numerator and denominator are products of two bf16 values:
    the quotient is known exactly in 64 bits, ties among it."""
    g = torch.Generator(device="cuda").manual_seed(H)
    x = torch.randint(-40, 41, (T, H), generator=g, device="cuda").bfloat16()
    x[:, ::3] = rand(T, H, seed=T)[:, ::3]
    r = torch.randint(-40, 41, (T, H), generator=g, device="cuda").bfloat16() if residual else None
    w = (torch.randint(16, 33, (H,), generator=g, device="cuda") / 32).bfloat16()
    q, s, out = fused.rmsnorm_fp8(x, w, 1e-6, r)
    p = (out.double() * w.double()).unflatten(-1, (-1, 128))
    top = p.abs().amax(-1, keepdim=True).clamp_min(1e-300)
    want = e4m3_of(448 * p / top).flatten(-2)
    half = 448 * p / top / torch.exp2(torch.frexp(448 * p / top)[1].clamp_min(-5).double() - 4) % 1 == 0.5
    assert half.sum() > 0 and torch.equal(q.double(), want)
    y = out.double() / torch.sqrt(out.double().pow(2).mean(-1, keepdim=True) + 1e-6) * w.double()
    check(q, s, y, "fp32", 2 ** -18)


@pytest.mark.parametrize("scales", ["fp32", "e8m0"])
def test_rows_below_the_floor_of_a_scale(scales):
    """Groups that are all below 1e-10 keep the floor's scale; codes are values over it."""
    x, w = rand(5, 512, seed=1), torch.ones(512, device="cuda").bfloat16()
    w[:128] = 1e-12
    w[128:256] = 3e-11
    w[256:384] = 1e-30
    q, s, _ = fused.rmsnorm_fp8(x, w, 1e-6, scales=scales)
    xd = x.double()
    check(q, s, xd / torch.sqrt(xd.pow(2).mean(-1, keepdim=True) + 1e-6) * w.double(), scales, 2 ** -18)
    x = rand(3, 256, seed=2) * 1e-30          # eps carries the norm: 1000 x
    q, s, _ = fused.rmsnorm_fp8(x, w[384:].repeat(2), 1e-6, scales=scales)
    assert (q.float() == 0).all() and (s.float() < 1e-12).all()


@pytest.mark.parametrize("scales", ["fp32", "e8m0"])
def test_activation_with_gates_far_below_zero(scales):
    """silu(gate) leaves the normal 32-bit range below a gate of -87, but a large partner brings the product back."""
    T, F = 6, 512
    gate = -(86 + 4 * torch.rand(T, F, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"))
    gate[1] = gate[1] * 0.9
    gate[2] = -gate[2]
    gate[3, ::2] = 0.3
    up = rand(T, F, seed=3)
    up[0] *= 1e30
    up[3] *= 1e37
    up[4] *= 1e37
    up[5, :128] *= 1e36
    x = torch.cat([gate.bfloat16(), up], -1)
    q, s = fused.swiglu_fp8(x, scales=scales)
    g, u = x.double().chunk(2, -1)
    # the exponential of a gate of 90 is off by 90 2^-24 and the rest by 2^-18
    check(q, s, g * torch.sigmoid(g) * u, scales, 2 ** -16)


@pytest.mark.parametrize("scales", ["fp32", "e8m0"])
def test_a_few_far_gates_in_a_large_batch(scales):
    """Several units a thread: a row of far gates changes itself only."""
    T, F = 1203, 4096
    x = rand(T, 2 * F, seed=5, scale=2)
    base = fused.swiglu_fp8(x, scales=scales)
    rows = [0, 1, 600, 1201, 1202]
    x[rows, :F] = -(80 + 10 * torch.rand(5, F, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")).bfloat16()
    x[rows, F:] *= 1e30
    q, s = fused.swiglu_fp8(x, scales=scales)
    g, u = x.double().chunk(2, -1)
    check(q, s, g * torch.sigmoid(g) * u, scales, 2 ** -16)
    keep = [i for i in range(T) if i not in rows]
    # units whose warp has none of the rows' gates are the same bits; the others may be off by a rounding of 32 bits
    same = (q.view(torch.uint8)[keep] == base[0].view(torch.uint8)[keep]).float().mean()
    assert same > 0.999


def test_far_gates_late_in_a_share():
    """More than 32 iterations a thread: those beyond share a bit of what is to be done over."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    F = 16384
    T = 36 * sms * 32 * 512 // (F // 8)
    x = torch.randn(2, 2 * F, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").bfloat16().repeat(T // 2, 1)
    T = x.shape[0]
    rows = [0, 3, T // 36 * 30, T // 36 * 34 + 1, T - 1]
    x[rows, :F] = (-84 - 6 * torch.rand(5, F, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")).bfloat16()
    x[rows, F:] *= 1e30
    q, s = fused.swiglu_fp8(x, scales="e8m0")
    some = rows + [1, 2, T // 2, T - 2]
    g, u = x[some].double().chunk(2, -1)
    check(q[some], s[some], g * torch.sigmoid(g) * u, "e8m0", 2 ** -16)
    plain = [i for i in range(100, T - 100, 2) if i not in rows]   # copies of row 0 as it was
    assert (q.view(torch.uint8)[plain] == q.view(torch.uint8)[plain[0]]).all()


@pytest.mark.parametrize("T,H", [(1, 3584), (37, 4096), (200, 96), (3, 8192)])
def test_rounded_forms_with_powers_of_two_are_the_chains_bit_for_bit(T, H):
    x, r, w = rand(T, H, seed=1), rand(T, H, seed=2, scale=3), 1 + rand(H, seed=3, scale=0.2)
    y, res = fused.rmsnorm(x, w, 1e-6, r)
    q0, s0 = quant.quant_act_1x32(y)
    q, s, out = fused.rmsnorm_fp8(x, w, 1e-6, r, scales="e8m0", as_rounded=True)
    assert torch.equal(out, res)
    assert torch.equal(s.view(torch.uint8), s0.view(torch.uint8)) and torch.equal(q.view(torch.uint8), q0.view(torch.uint8))
    q0, s0 = quant.quant_act_1x32(fused.swiglu(torch.cat([x, r], -1)))
    q, s = fused.swiglu_fp8(torch.cat([x, r], -1), scales="e8m0", as_rounded=True)
    assert torch.equal(s.view(torch.uint8), s0.view(torch.uint8)) and torch.equal(q.view(torch.uint8), q0.view(torch.uint8))
