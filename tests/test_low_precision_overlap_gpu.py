"""The low-precision serving kernels overlapped as the rollout engine launches them, against launches one after another: overlap off,
and the stream waited for behind every operator."""
import pytest
import torch

from gcore_b200.ops import _lib, fused, quant
from test_fp4_products_gpu import rand, weight

pytestmark = pytest.mark.gpu


def layer(x, res, gain, up, down, eight, then):
    if eight:
        q, s, res = then(fused.rmsnorm_fp8(x, gain, 1e-6, res, scales="e8m0"))
        q, s = then(fused.swiglu_fp8(then(quant.gemm_fp4(q, s, up)), scales="e8m0"))
        return then(quant.gemm_fp4(q, s, down)), res
    h, res = then(fused.rmsnorm(x, gain, 1e-6, res))
    return then(quant.linear_fp4(then(fused.swiglu(then(quant.linear_fp4(h, up)))), down)), res


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("T", [1, 6, 24, 160, 600])
def test_a_chain_of_layers(T, eight):
    up, down = weight(2048, 512, seed=1), weight(512, 1024, seed=2)
    gain = torch.ones(512, device="cuda").bfloat16()
    x0 = rand(T, 512, seed=3, scale=0.1).bfloat16()

    def run(then):
        x, res, seen = x0, torch.zeros_like(x0), []
        for i in range(12):
            x, res = layer(x, res, gain, up, down, eight, then)
            x = (x / 16).clamp(-8, 8) if i % 3 == 2 else x    # the weights' groups are large: values stay finite
            seen += [x, res]
        return seen

    def alone(out):
        torch.cuda.synchronize()
        return out

    lib = _lib.kernels()
    with torch.no_grad():
        was = lib.gk_set_overlap(0)
        try:
            want = run(alone)
        finally:
            lib.gk_set_overlap(was)
        torch.cuda.synchronize()
        outside = run(lambda out: out)
        lib.gk_set_pdl(1)
        try:
            inside = run(lambda out: out)
        finally:
            lib.gk_set_pdl(0)
    assert all(a.isfinite().all() for a in want)
    for got in (outside, inside):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
