"""Products with 4-bit weights on the GPU against 64 bits.

Tolerances.  Codes times powers of two are exact in the operands, so what is left is the sum and the result's rounding.  The tensor
core adds 16 or 32 products at a time to a 32-bit sum, each addition off by at most 2^-23 of what has been added: (K / 16 + 16)
2^-23 of sum |x w|.  Where 16-bit activations are two e4m3 terms a term's rest below 2^-22 of the largest of its group of 32 is
lost: 2^-21 of sum (group's largest |x|) |w|.  A bf16 result adds half a step, 2^-8 relative to it (2^-9 for an exact one)."""
import pytest
import torch

from gcore_b200.ops import quant

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return scale * torch.randn(*shape, generator=g, device="cuda")


def weight(N, K, seed=0):
    # groups of very different size, some of them zero
    w = rand(N, K // 32, 32, seed=seed) * torch.exp2(torch.randint(-12, 3, (N, K // 32, 1), device="cuda").float())
    w[:: 5, 0] = 0
    return quant.Fp4Weight.of(w.view(N, K).bfloat16())


def bound(x, w, y, dtype):
    K = x.shape[1]
    top = x.abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, 32).flatten(-2)
    b = (K / 16 + 16) * 2.0 ** -23 * (x.abs() @ w.abs().t()) + 2.0 ** -21 * (top @ w.abs().t())
    return b + (2.0 ** -8 * (y.abs() + b) if dtype == torch.bfloat16 else 0) + 1e-30


SIZES = [(1, 128, 32), (1, 300, 3584), (3, 1, 64), (8, 129, 256), (13, 4608, 3584), (16, 513, 1184), (33, 3584, 4128), (64, 896, 18944),
         (100, 1027, 512), (128, 256, 1536), (129, 640, 1024), (257, 2293, 1056), (1000, 384, 2048),
         # few tiles: chunks of the tokens, with and without a divided sum; many tiles of the widths that are not whole units
         (150, 130, 4608), (300, 70, 2080), (129, 129, 128), (641, 513, 672), (1300, 6401, 256), (700, 12802, 160), (520, 9999, 384)]


@pytest.mark.parametrize("T,N,K", SIZES)
def test_products(T, N, K):
    W = weight(N, K, seed=N + K)
    w = W.values(torch.float32).double()
    x = (rand(T, K, seed=T) * torch.exp(rand(K, seed=1))).bfloat16()
    bias = rand(N, seed=3).bfloat16()
    for b in (None, bias, bias.float()):
        y = x.double() @ w.t() + (b.double() if b is not None else 0)
        got = quant.linear_fp4(x, W, b)
        assert got.shape == (T, N) and got.dtype == torch.bfloat16
        assert ((got.double() - y).abs() <= bound(x.double(), w, y, torch.bfloat16)).all()
    q, s = quant.quant_act_1x32(x)
    xq = (q.double().unflatten(-1, (-1, 32)) * s.double()[..., None]).flatten(-2)
    y = xq @ w.t()
    for dtype in (torch.bfloat16, torch.float32):
        got = quant.gemm_fp4(q, s, W, out_dtype=dtype)
        assert got.dtype == dtype and ((got.double() - y).abs() <= bound(xq, w, y, dtype)).all()
    got = quant.gemm_fp4(q, s, W, bias)
    assert ((got.double() - y - bias.double()).abs() <= bound(xq, w, y + bias.double(), torch.bfloat16)).all()


def test_every_code_and_column_is_read_once_and_in_order():
    """One token with a single 1: the product is one column of the weight, exactly."""
    N, K = 130, 256
    W = weight(N, K, seed=9)
    w = W.values(torch.bfloat16)
    eye = torch.eye(K, device="cuda").bfloat16()
    assert torch.equal(quant.linear_fp4(eye, W), w.t())
    for k in (0, 1, 31, 32, 63, 127, 128, 200, 255):
        assert torch.equal(quant.linear_fp4(eye[k:k + 1], W)[0], w[:, k])
        q, s = quant.quant_act_1x32(eye[k:k + 1])
        assert torch.equal(quant.gemm_fp4(q, s, W)[0], w[:, k])


@pytest.mark.parametrize("T", [1, 5, 40, 200])
def test_activations_of_any_size(T):
    """Outliers, tiny values, zeros and whole rows of nothing; rows do not touch one another."""
    N, K = 384, 640
    W = weight(N, K, seed=4)
    w = W.values(torch.float32).double()
    x = rand(T, K, seed=6)
    x[:, 5] *= 3000
    x[:, 70] = 1e-6
    x[:, 96:128] = 0
    x[:, 200:210] *= 1e-20
    if T > 2:
        x[1] = 0
        x[2] *= 1e30
    x = x.bfloat16()
    y = x.double() @ w.t()
    got = quant.linear_fp4(x, W)
    assert ((got.double() - y).abs() <= bound(x.double(), w, y, torch.bfloat16)).all()
    if T > 2:
        assert (got[1] == 0).all()
        x[2, 3] = float("nan")
        bad = quant.linear_fp4(x, W)
        keep = [i for i in range(T) if i != 2]
        assert bad[2].isnan().all() and torch.equal(bad[keep], got[keep])


def test_row_strides_batches_and_empty():
    W = weight(256, 512, seed=2)
    x = rand(6, 1024, seed=1).bfloat16()
    want = quant.linear_fp4(x[:, 3:515].clone(), W)
    assert torch.equal(quant.linear_fp4(x[:, 3:515], W), want)
    assert torch.equal(quant.linear_fp4(x[:, 3:515].unflatten(0, (2, 3)), W), want.view(2, 3, 256))
    assert quant.linear_fp4(x[:0, :512], W).shape == (0, 256)
    q, s = quant.quant_act_1x32(x[:0, :512])
    assert quant.gemm_fp4(q, s, W).shape == (0, 256)
    # rows of three exponents that start on any byte, scales and codes of wider buffers
    V = weight(40, 96, seed=3)
    q, s = quant.quant_act_1x32(x[:, :96])
    want = quant.gemm_fp4(q, s, V)
    for i in range(1, 5):
        assert torch.equal(quant.gemm_fp4(q[i:], s[i:], V), want[i:])
    wide_q, wide_s = torch.zeros(6, 200, device="cuda").to(torch.float8_e4m3fn), torch.empty(6, 7, dtype=torch.uint8, device="cuda")
    wide_q[:, 5:101], wide_s[:, 2:5] = q, s.view(torch.uint8)
    assert torch.equal(quant.gemm_fp4(wide_q[:, 5:101], wide_s.view(torch.float8_e8m0fnu)[:, 2:5], V), want)
    # a weight cut out of a larger one
    big = quant.Fp4Weight.of(rand(80, 512, seed=9).bfloat16())
    part = quant.Fp4Weight(big.codes[3:44, 16:64], big.exponents[3:44, 1:4])
    assert torch.equal(part.values(), big.values()[3:44, 32:128])
    y = x[:, :96].double() @ part.values().double().t()
    assert ((quant.linear_fp4(x[:, :96], part).double() - y).abs() <= bound(x[:, :96].double(), part.values().double(), y,
                                                                            torch.bfloat16)).all()


@pytest.mark.parametrize("T,N,K", [(1, 64, 96), (40, 257, 320), (300, 1024, 512), (513, 130, 1152), (257, 1, 64), (131, 903, 256)])
def test_gradient(T, N, K):
    W = weight(N, K, seed=N)
    w = W.values(torch.float32).double()
    x = rand(T, K, seed=1).bfloat16().requires_grad_()
    b = rand(N, seed=2).bfloat16().requires_grad_()
    dy = rand(T, N, seed=3).bfloat16()
    gx, gb = torch.autograd.grad(quant.linear_fp4(x, W, b), (x, b), dy)
    want = dy.double() @ w
    tol = (N / 16 + 16) * 2.0 ** -23 * (dy.double().abs() @ w.abs()) + 1e-30
    assert ((gx.double() - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol)).all()
    s = dy.double().sum(0)
    assert ((gb.double() - s).abs() <= 2.0 ** -8 * s.abs() + T * 2.0 ** -23 * dy.double().abs().sum(0)).all()
    # along a direction: the product is linear, so the difference quotient is the gradient's product with it
    d = rand(T, K, seed=8).bfloat16()
    with torch.no_grad():
        two = (quant.linear_fp4(x + d, W).double() - quant.linear_fp4(x - d, W).double()) / 2
    lhs, rhs = (two * dy.double()).sum(), (gx.double() * d.double()).sum()
    x2 = x.detach().double().abs() + d.double().abs()
    slack = 2.0 ** -7 * ((x2 @ w.abs().t()) * dy.double().abs()).sum() + 2.0 ** -8 * (gx.double().abs() * d.double().abs()).sum()
    assert (lhs - rhs).abs() <= slack


@pytest.mark.parametrize("tokens", [(1, 16, 40), (300, 5, 2100), (128, 2500, 64)])
def test_graphs_and_streams_side_by_side(tokens):
    """Two captured graphs and eager calls of the same weight at once: no shared scratch."""
    W = weight(1536, 2048, seed=3)
    xs = [rand(t, 2048, seed=t).bfloat16() for t in tokens]
    want = [quant.linear_fp4(x, W) for x in xs]
    graphs = []
    for x in xs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = quant.linear_fp4(x, W)
        graphs.append((g, y))
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            graphs[0][0].replay()
        with torch.cuda.stream(streams[1]):
            graphs[1][0].replay()
        with torch.cuda.stream(streams[2]):
            y = quant.linear_fp4(xs[2], W)
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want[0]) and torch.equal(graphs[1][1], want[1]) and torch.equal(y, want[2])


@pytest.mark.parametrize("T", [2, 20, 150])
def test_tokens_that_are_not_numbers_stay_by_themselves(T):
    """e4m3 rows with the scale of NaN, bf16 rows with an infinity: their tokens come out as NaN, the others as they were."""
    W = weight(200, 384, seed=1)
    x = rand(T, 384, seed=2).bfloat16()
    want = quant.linear_fp4(x, W)
    q, s = quant.quant_act_1x32(x)
    want8 = quant.gemm_fp4(q, s, W)
    x[1, 100] = float("-inf")
    got = quant.linear_fp4(x, W)
    s.view(torch.uint8)[1, 3] = 255
    got8 = quant.gemm_fp4(q, s, W)
    keep = [i for i in range(T) if i != 1]
    assert got[1].isnan().all() and got8[1].isnan().all()
    assert torch.equal(got[keep], want[keep]) and torch.equal(got8[keep], want8[keep])


def test_single_rows_and_rows_in_a_batch_agree():
    W = weight(640, 512, seed=5)
    x = rand(12, 512, seed=3).bfloat16()
    assert torch.equal(quant.linear_fp4(x[3], W), quant.linear_fp4(x[3:4], W)[0])
    q, s = quant.quant_act_1x32(x[3])
    assert torch.equal(quant.gemm_fp4(q, s, W), quant.gemm_fp4(*quant.quant_act_1x32(x[3:4]), W)[0])


def test_a_layer_as_it_is_served_with_overlapped_launches():
    """Norm, product, activation, product of a decode batch, launched as the rollout engine does (each kernel set up while the one
    in front drains), thirty times over: the bits of launches one after another."""
    from gcore_b200.ops import _lib, fused
    up, down = weight(2048, 512, seed=1), weight(512, 1024, seed=2)
    gain = torch.ones(512, device="cuda").bfloat16()
    x0 = rand(24, 512, seed=3, scale=0.1).bfloat16()

    def layer(x, res, eight):
        if eight:
            q, s, res = fused.rmsnorm_fp8(x, gain, 1e-6, res, scales="e8m0")
            return quant.gemm_fp4(*fused.swiglu_fp8(quant.gemm_fp4(q, s, up), scales="e8m0"), down), res
        h, res = fused.rmsnorm(x, gain, 1e-6, res)
        return quant.linear_fp4(fused.swiglu(quant.linear_fp4(h, up)), down), res

    def run(eight, T):
        x, res, seen = x0[:T], torch.zeros_like(x0[:T]), []
        for _ in range(30):
            x, res = layer(x, res, eight)
            seen += [x, res]
        return seen

    lib = _lib.kernels()
    for T in (1, 6, 24):
        for eight in (False, True):
            with torch.no_grad():
                want = run(eight, T)
                torch.cuda.synchronize()
                lib.gk_set_pdl(1)
                try:
                    got = run(eight, T)
                finally:
                    lib.gk_set_pdl(0)
            assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(got, want))
