"""Norm and activation with e4m3 outputs on the GPU, against 64 bits and against the chains they replace.

Tolerances.  A code is off by half a step: |y| / 16 relative, or 2^-10 of the scale below e4m3's smallest normal value.  The
32-bit value in front of it: a thread adds at most 64 squares one after the other and the rest in a tree of 8 + 5 steps, half of
which relative error the root keeps, and a handful of roundings and approximate functions (2 units each) follow: below 2^-18.
The approximate exponential of the activation is off by 2^-21 of its argument's size (|gate| < 16 here) beside 2 units: 2^-17."""
import pytest
import torch

from gcore_b200.ops import fused, quant

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g, device="cuda")).bfloat16()


def check(q, s, y, scales, slack):
    """Codes and scales against the exact values ``y`` (64 bits)."""
    n = 128 if scales == "fp32" else 32
    g = y.unflatten(-1, (-1, n))
    top = g.abs().amax(-1).clamp_min(1e-10)
    sd = s.double()
    if scales == "fp32":
        assert ((sd - top / 448).abs() <= slack * top / 448).all()
    else:
        e = torch.log2(top / 448)
        lo, hi = torch.ceil(e - 2 * slack), torch.ceil(e + 2 * slack)   # they differ only beside a border
        got = torch.frexp(sd)[1] - 1                                    # the logarithm of a power of two, exactly
        assert ((got >= lo) & (got <= hi)).all()
    back = q.double().unflatten(-1, (-1, n)) * sd[..., None]
    bound = g.abs() * (2 ** -4 + 2 * slack) + sd[..., None] * 2 ** -10 * (1 + 2 * slack)
    assert ((back - g).abs() <= bound).all()


@pytest.mark.parametrize("scales", ["fp32", "e8m0"])
@pytest.mark.parametrize("T,H,residual", [(1, 128, True), (7, 256, False), (3, 1536, True), (1, 3584, True), (65, 7168, False),
                                          (5, 8192, True), (2, 8320, True), (3, 16384, False), (1500, 384, True)])
def test_norm(T, H, residual, scales):
    x, r, w = rand(T, H, seed=T), rand(T, H, seed=T + 1, scale=3) if residual else None, 1 + rand(H, seed=2, scale=0.2)
    q, s, out = fused.rmsnorm_fp8(x, w, 1e-6, r, scales=scales)
    xs = x if r is None else (x.float() + r.float()).bfloat16()
    assert torch.equal(out, xs)
    xd = xs.double()
    check(q, s, xd / torch.sqrt(xd.pow(2).mean(-1, keepdim=True) + 1e-6) * w.double(), scales, 2 ** -18)


@pytest.mark.parametrize("H", [32, 96, 160, 4128])
def test_norm_of_widths_that_are_whole_groups_of_32(H):
    x, r, w = rand(9, H, seed=H), rand(9, H, seed=H + 1), 1 + rand(H, seed=2, scale=0.2)
    q, s, out = fused.rmsnorm_fp8(x, w, 1e-5, r, scales="e8m0")
    xd = out.double()
    check(q, s, xd / torch.sqrt(xd.pow(2).mean(-1, keepdim=True) + 1e-5) * w.double(), "e8m0", 2 ** -18)


@pytest.mark.parametrize("scales", ["fp32", "e8m0"])
@pytest.mark.parametrize("T,F", [(1, 128), (3, 384), (64, 18944), (777, 8960), (1, 14336)])
def test_activation(T, F, scales):
    x = rand(T, 2 * F, seed=F, scale=2)
    q, s = fused.swiglu_fp8(x, scales=scales)
    g, u = x.double().chunk(2, -1)
    check(q, s, g * torch.sigmoid(g) * u, scales, 2 ** -17)


@pytest.mark.parametrize("T,F", [(5, 32), (11, 96), (2, 4128)])
def test_rows_and_activation_of_whole_groups_of_32(T, F):
    x = rand(T, 2 * F, seed=F)
    q, s = fused.swiglu_fp8(x, scales="e8m0")
    g, u = x.double().chunk(2, -1)
    check(q, s, g * torch.sigmoid(g) * u, "e8m0", 2 ** -17)
    q, s = quant.quant_act_1x32(x)
    q0, s0 = quant.quant_rows_ref(x, "e8m0")
    assert torch.equal(q.view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s.view(torch.uint8), s0.view(torch.uint8))


@pytest.mark.parametrize("T,H", [(1, 3584), (37, 4096), (200, 1024), (3, 8192)])
def test_rounded_forms_are_the_chains_bit_for_bit(T, H):
    x, r, w = rand(T, H, seed=1), rand(T, H, seed=2, scale=3), 1 + rand(H, seed=3, scale=0.2)
    y, res = fused.rmsnorm(x, w, 1e-6, r)
    q0, s0 = quant.quant_act_1x128(y)
    q, s, out = fused.rmsnorm_fp8(x, w, 1e-6, r, as_rounded=True)
    assert torch.equal(out, res) and torch.equal(s, s0) and torch.equal(q.view(torch.uint8), q0.view(torch.uint8))
    q, s, out = fused.rmsnorm_fp8(x, w, 1e-6, as_rounded=True)
    q0, s0 = quant.quant_act_1x128(fused.rmsnorm(x, w, 1e-6)[0])
    assert out is x and torch.equal(s, s0) and torch.equal(q.view(torch.uint8), q0.view(torch.uint8))
    q0, s0 = quant.quant_act_1x128(fused.swiglu(x.view(T, H)))
    q, s = fused.swiglu_fp8(x, as_rounded=True)
    assert torch.equal(s, s0) and torch.equal(q.view(torch.uint8), q0.view(torch.uint8))


def test_zeros_non_finite_rows_strides_and_empty_batches():
    x, w = rand(6, 256, seed=5), torch.ones(256, dtype=torch.bfloat16, device="cuda")
    x[1] = 0
    x[2, 7] = float("nan")
    x[4, 9] = float("inf")
    for scales in ("fp32", "e8m0"):
        q, s, _ = fused.rmsnorm_fp8(x, w, 1e-6, scales=scales)
        assert q[1].float().abs().sum() == 0 and s[1].float().isfinite().all()
        n = 256 // s.shape[1]
        back = q.float().unflatten(-1, (-1, n)) * s.float()[..., None]
        assert back[2].isnan().any() and back[4].isnan().any() and back[[0, 1, 3, 5]].isfinite().all()
        wide = torch.randn(6, 512, device="cuda").bfloat16()
        a, b, _ = fused.rmsnorm_fp8(wide[:, 3:259], w, 1e-6, wide[:, 130:386], scales=scales)   # neither packed nor aligned
        c, d, _ = fused.rmsnorm_fp8(wide[:, 3:259].clone(), w, 1e-6, wide[:, 130:386].clone(), scales=scales)
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8)) and torch.equal(b.view(torch.uint8), d.view(torch.uint8))
        q, s, out = fused.rmsnorm_fp8(x[:0], w, 1e-6, x[:0], scales=scales)
        assert q.shape == (0, 256) and s.shape[0] == 0 and out.shape == (0, 256)
        assert fused.swiglu_fp8(x[:0], scales=scales)[0].shape == (0, 128)
    # an infinite gate with a finite product partner: the group is NaN, its neighbours are not
    z = rand(1, 512, seed=6)
    z[0, 3] = float("inf")
    q, s = fused.swiglu_fp8(z, scales="e8m0")
    back = q.float().view(8, 32) * s.float()[0][:, None]
    assert back[0].isnan().all() and back[1:].isfinite().all()


def test_norm_in_a_graph_on_another_stream():
    x, r, w = rand(12, 512, seed=1), rand(12, 512, seed=2), torch.ones(512, dtype=torch.bfloat16, device="cuda")
    want = fused.rmsnorm_fp8(x, w, 1e-6, r, scales="e8m0")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fused.rmsnorm_fp8(x, w, 1e-6, r, scales="e8m0")
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s, out = fused.rmsnorm_fp8(x, w, 1e-6, r, scales="e8m0")
    x.mul_(2)
    r.mul_(2)
    graph.replay()
    x0, r0 = x / 2, r / 2
    # twice the stream: the norm is the same up to eps, the residual stream doubles
    assert torch.equal(out, 2 * want[2]) and torch.equal(x0 + r0, want[2])
    again = fused.rmsnorm_fp8(x, w, 1e-6, r, scales="e8m0")
    assert torch.equal(q.view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(s.view(torch.uint8), again[1].view(torch.uint8))
