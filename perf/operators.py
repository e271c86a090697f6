"""Operators of low-precision serving, as a list of measurable cases.

A rollout engine that serves quantised projections runs, per layer, a norm, a projection, an activation and a projection.
Three of the four operators below are what stands between and in them:

* ``norm``    residual addition and RMSNorm, the result in e4m3 with scales (``fused.rmsnorm_fp8``);
* ``swiglu``  the gated activation, the result in e4m3 with scales (``fused.swiglu_fp8``);
* ``linear``  bf16 activations times a 4-bit weight with one power of two per 32 codes (``quant.linear_fp4``), with
  ``grad`` its gradient in the activations too;
* ``gemm``    e4m3 activations with a power of two per 32 values times such a weight (``quant.gemm_fp4``).

``scales`` of ``norm`` and ``swiglu``: ``fp32`` is one 32-bit scale per 128 values, what the block-fp8 product reads;
``e8m0`` one power of two per 32 values, what the 4-bit product reads.

Where ``own`` is false every operator is written with elementary torch operations in 32 bits.
"""
import math

import torch

own = False

EPS = 1e-6
E4M3_MAX, E2M1_MAX = 448.0, 6.0
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------------------------------------------------- cases
def _norm(name, tokens, width, scales, residual=True):
    return dict(name=name, op="norm", tokens=tokens, width=width, scales=scales, residual=residual)


def _swiglu(name, tokens, width, scales):
    return dict(name=name, op="swiglu", tokens=tokens, width=width, scales=scales)


def _product(name, op, tokens, inner, outer, bias=False, grad=False):
    return dict(name=name, op=op, tokens=tokens, inner=inner, outer=outer, bias=bias, grad=grad)


def listed():
    return [
        # one request decodes on the dense 7B recipe: nothing but latency
        _norm("norm_one_token", 1, 3584, "fp32"),
        # a decode batch of the widest preset, in front of a 4-bit projection
        _norm("norm_decode_batch", 96, 7168, "e8m0"),
        # packed prompts of one prefill pass (16384 tokens is the engine's limit), the long-context recipe's width
        _norm("norm_prompts", 16384, 4096, "e8m0"),
        # the first norm of a pass has no residual yet; a ragged number of prompt tokens
        _norm("norm_first_layer", 3001, 1536, "fp32", residual=False),
        # activation of a decode batch of the 7B recipe, in front of its block-fp8 down projection
        _swiglu("swiglu_decode_batch", 64, 18944, "fp32"),
        # activation of packed prompts of the long-context recipe
        _swiglu("swiglu_prompts", 8191, 14336, "e8m0"),
        # one request decodes: gate and up projection of the 7B recipe, 68 MB of codes for one row
        _product("linear_one_token", "linear", 1, 3584, 37888),
        # a small decode batch through the query, key and value projection with its bias
        _product("linear_bias", "linear", 13, 3584, 4608, bias=True),
        # a rollout's decode batch through the down projection: a long sum, few output rows
        _product("linear_decode_batch", "linear", 64, 18944, 3584),
        # a packed micro-batch through a frozen 4-bit projection under trained adapters: forward and the gradient
        _product("linear_train", "linear", 3391, 4096, 6144, grad=True),
        # a decode batch with 8-bit activations through gate and up projection of the long-context recipe
        _product("gemm_decode_batch", "gemm", 96, 4096, 28672),
        # packed prompts with 8-bit activations through the same projection
        _product("gemm_prompts", "gemm", 8192, 4096, 28672),
    ]


MOST_NORM = 16384 * 4096          # values of the largest listed norm
MOST_SWIGLU = 8191 * 14336
MOST_LINEAR = 3391 * 4096 * 6144  # multiplications; forward and gradient are twice that
MOST_GEMM = 8192 * 4096 * 28672


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "swiglu", "linear", "linear", "gemm"))
    if op in ("norm", "swiglu"):
        scales = rng.choice(("fp32", "e8m0"))
        unit = 128 if scales == "fp32" else 32
        widest, most = (8192, MOST_NORM) if op == "norm" else (18944, MOST_SWIGLU)
        width = unit * _log_uniform(rng, 256 // unit, widest // unit)
        tokens = _log_uniform(rng, 1, min(16384, most // width))
        if op == "norm":
            return dict(op=op, tokens=tokens, width=width, scales=scales, residual=rng.random() < 0.8)
        return dict(op=op, tokens=tokens, width=width, scales=scales)
    inner = 32 * _log_uniform(rng, 512 // 32, 18944 // 32)
    outer = _log_uniform(rng, 100, 37888)
    if op == "gemm":
        tokens = _log_uniform(rng, 1, max(1, min(8192, MOST_GEMM // (inner * outer))))
        return dict(op=op, tokens=tokens, inner=inner, outer=outer, bias=rng.random() < 0.3, grad=False)
    tokens = _log_uniform(rng, 1, max(1, min(4096, MOST_LINEAR // (inner * outer))))
    return dict(op=op, tokens=tokens, inner=inner, outer=outer, bias=rng.random() < 0.3,
                grad=tokens >= 256 and rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------------------ inputs
def _activations(gen, tokens, width):
    """Normal values whose columns differ in size, as hidden states do, with some columns far larger than the rest."""
    size = torch.exp(0.4 * torch.randn(width, generator=gen, device="cuda"))
    size = torch.where(torch.rand(width, generator=gen, device="cuda") < 0.004, size * 30, size)
    return torch.randn(tokens, width, generator=gen, device="cuda").mul_(size).to(torch.bfloat16)


def _weight_codes(gen, rows, width):
    """A normal weight in 4 bits: codes [rows, width / 2], two a byte, the even column in the low half; exponents
    [rows, width / 32] as biased bytes.  Each group's power of two is the smallest that keeps its values within 6."""
    w = torch.randn(rows, width // 32, 32, generator=gen, device="cuda").mul_(0.02)
    m, e = torch.frexp(w.abs().amax(-1))
    e = e - 3 + (m > 0.75)
    w = torch.ldexp(w, -e[..., None])
    bounds = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    code = torch.bucketize(w.abs(), bounds).to(torch.uint8) | ((w < 0).to(torch.uint8) << 3)
    code = code.view(rows, width)
    return code[:, 0::2] | (code[:, 1::2] << 4), (e + 127).to(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, T = case["op"], case["tokens"]
    st = dict(case=dict(case))
    if op == "norm":
        st["x"] = _activations(gen, T, case["width"])
        st["gain"] = (1 + 0.2 * torch.randn(case["width"], generator=gen, device="cuda")).to(torch.bfloat16)
        st["residual"] = _activations(gen, T, case["width"]) if case["residual"] else None
    elif op == "swiglu":
        st["x"] = torch.randn(T, 2 * case["width"], generator=gen, device="cuda").to(torch.bfloat16)
    else:
        K, N = case["inner"], case["outer"]
        st["codes"], st["exponents"] = _weight_codes(gen, N, K)
        st["bias"] = (0.1 * torch.randn(N, generator=gen, device="cuda")).to(torch.bfloat16) if case["bias"] else None
        x = _activations(gen, T, K)
        if op == "linear":
            st["x"] = x
            st["dy"] = torch.randn(T, N, generator=gen, device="cuda").to(torch.bfloat16) if case["grad"] else None
        else:
            st["q"], st["s"] = _to_e4m3(x.float(), "e8m0")
        if own:  # the handle that a server makes of a weight when it is loaded
            from gcore_b200.ops import quant
            st["weight"] = quant.Fp4Weight(st["codes"], st["exponents"])
    return st


# -------------------------------------------------------------------------------------------------------- plain form
def _to_e4m3(y, scales):
    T, W = y.shape
    if scales == "fp32":
        y = y.view(T, W // 128, 128)
        s = y.abs().amax(-1).clamp_min(1e-10) / E4M3_MAX
        q = (y / s[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
        return q.view(T, W).to(torch.float8_e4m3fn), s
    y = y.view(T, W // 32, 32)
    m, e = torch.frexp(y.abs().amax(-1).clamp_min(1e-10))
    e = e - 9 + (m > 0.875)   # smallest power of two that keeps the group within 448 = 0.875 * 2^9
    q = torch.ldexp(y, -e[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
    return q.view(T, W).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _weight_values(codes, exponents):
    N, half = codes.shape
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], dim=-1).view(N, 2 * half)
    w = table[both.int()].view(N, half // 16, 32)
    return torch.ldexp(w, exponents.int()[..., None] - 127).view(N, 2 * half)


def _plain(st):
    c = st["case"]
    if c["op"] == "norm":
        x = st["x"]
        if st["residual"] is not None:
            x = (x.float() + st["residual"].float()).to(x.dtype)
        f = x.float()
        y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * st["gain"].float()
        return (*_to_e4m3(y, c["scales"]), x)
    if c["op"] == "swiglu":
        g, u = st["x"].float().chunk(2, dim=-1)
        return _to_e4m3(g / (1 + torch.exp(-g)) * u, c["scales"])
    w = _weight_values(st["codes"], st["exponents"])
    if c["op"] == "linear":
        x = st["x"].float()
    else:
        x = st["q"].float().view(c["tokens"], -1, 32) * st["s"].float()[..., None]
    y = x.view(c["tokens"], -1) @ w.t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    y = y.to(torch.bfloat16)
    return (y, (st["dy"].float() @ w).to(torch.bfloat16)) if c["grad"] else y


def _kernels(st):
    from gcore_b200.ops import fused, quant
    c = st["case"]
    if c["op"] == "norm":
        return fused.rmsnorm_fp8(st["x"], st["gain"], EPS, st["residual"], scales=c["scales"])
    if c["op"] == "swiglu":
        return fused.swiglu_fp8(st["x"], scales=c["scales"])
    if c["op"] == "gemm":
        return quant.gemm_fp4(st["q"], st["s"], st["weight"], st["bias"])
    if not c["grad"]:
        return quant.linear_fp4(st["x"], st["weight"], st["bias"])
    x = st["x"].detach().requires_grad_()
    y = quant.linear_fp4(x, st["weight"], st["bias"])
    return y.detach(), torch.autograd.grad(y, x, st["dy"])[0]


def run(state):
    return _kernels(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------- in 64 bits
def _e4m3_of(v):
    """The nearest e4m3 value, halves to even: steps of an eighth of the power of two below, of 2^-9 under 2^-6."""
    v = v.clamp(-E4M3_MAX, E4M3_MAX)
    step = torch.exp2(torch.frexp(v)[1].clamp_min(-5).double() - 4)
    return torch.round(v / step) * step


def _groups(y, scales):
    n = 128 if scales == "fp32" else 32
    g = y.unflatten(-1, (-1, n))
    top = g.abs().amax(-1, keepdim=True).clamp_min(1e-10) / E4M3_MAX
    if scales == "e8m0":
        top = torch.exp2(torch.ceil(torch.log2(top)))
    return _e4m3_of(g / top).flatten(-2), top.squeeze(-1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        x = st["x"].double()
        if case["residual"]:
            x = (x + st["residual"].double()).to(torch.bfloat16).double()   # the stream is kept in 16 bits
        y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["width"] + EPS) * st["gain"].double()
        return (*_groups(y, case["scales"]), x)
    if case["op"] == "swiglu":
        W = case["width"]
        x = st["x"].double()
        return _groups(x[:, :W] * torch.sigmoid(x[:, :W]) * x[:, W:], case["scales"])
    N, K = case["outer"], case["inner"]
    w = torch.empty(N, K, dtype=torch.float64, device="cuda")
    for half, at in ((st["codes"] & 15, 0), (st["codes"] >> 4, 1)):
        e, m = ((half >> 1) & 3).double(), (half & 1).double()
        size = torch.where(e == 0, m / 2, torch.exp2(e - 1) * (1 + m / 2))
        w[:, at::2] = torch.where(half >= 8, -size, size)
    w *= torch.exp2(st["exponents"].double() - 127).repeat_interleave(32, dim=1)
    x = st["x"].double() if case["op"] == "linear" else st["q"].double() * st["s"].double().repeat_interleave(32, dim=1)
    y = torch.matmul(x, w.T)
    if case["bias"]:
        y += st["bias"].double()
    return (y, torch.matmul(st["dy"].double(), w)) if case["grad"] else y


# ---------------------------------------------------------------------------------------------------------- its work
def work(case):
    """Inputs read once, outputs written once; two operations a multiplication of the products, as many as there are roundings,
    additions and multiplications for the rest."""
    T = case["tokens"]
    if case["op"] in ("norm", "swiglu"):
        W = case["width"]
        scale_bytes = T * W / 32   # four bytes per 128 values, or one per 32
        if case["op"] == "norm":
            return dict(bytes=T * W * (2 + 1 + (4 if case["residual"] else 0)) + 2 * W + scale_bytes, flops=8 * T * W)
        return dict(bytes=T * W * (4 + 1) + scale_bytes, flops=8 * T * W)
    K, N = case["inner"], case["outer"]
    weight = N * K / 2 + N * K / 32
    x = T * K * 2 if case["op"] == "linear" else T * K * (1 + 1 / 32)
    total = weight + x + 2 * T * N + (2 * N if case["bias"] else 0)
    if case["grad"]:
        total += 2 * T * N + 2 * T * K
    return dict(bytes=total, flops=(4 if case["grad"] else 2) * T * N * K)
