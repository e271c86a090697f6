"""Block-scaled fp8 / fp4 quantisation and the block-scaled fp8 GEMM (``csrc/quant.cu``, ``csrc/gemm_fp8.cu``).

Eager definitions (``*_ref``) are the oracle and the CPU path; they follow the reference's eager quantisers
(gpatch_v4/kernel/quantize/eager_quant_kernels.py:63-233): e4m3 with 1x128 (activations) or 128x128 (weights) blocks,
fp32 or power-of-two scales, e2m1 1x32 with e8m0 scales, and quantise->dequantise round trips for QAT.
"""
from __future__ import annotations


import torch

from . import _lib

E4M3_MAX = 448.0
E2M1_MAX = 6.0
E2M1_VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
LAUNCHES = {"quant": 0}


def _pow2_ceil(s: torch.Tensor) -> torch.Tensor:
    return torch.exp2(torch.ceil(torch.log2(s)))


def act_quant_1x128_ref(x: torch.Tensor, pow2: bool = False):
    M, K = x.shape
    xb = x.float().view(M, K // 128, 128)
    s = xb.abs().amax(-1).clamp_min(1e-10) / E4M3_MAX
    if pow2:
        s = _pow2_ceil(s)
    q = (xb / s[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(M, K), s


def weight_quant_128x128_ref(w: torch.Tensor, pow2: bool = False):
    N, K = w.shape
    nb, kb = (N + 127) // 128, (K + 127) // 128
    wp = torch.zeros(nb * 128, kb * 128, dtype=torch.float32, device=w.device)
    wp[:N, :K] = w.float()
    blk = wp.view(nb, 128, kb, 128)
    s = blk.abs().amax(dim=(1, 3)).clamp_min(1e-10) / E4M3_MAX
    if pow2:
        s = _pow2_ceil(s)
    q = (blk / s[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(nb * 128, kb * 128)[:N, :K].contiguous(), s


def dequant_1x128(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    M, K = q.shape
    return (q.float().view(M, K // 128, 128) * s[..., None]).view(M, K)


def dequant_128x128(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    N, K = q.shape
    return q.float() * s.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]


def dequant_128x128_as(q: torch.Tensor, s: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """``dequant_128x128(q, s).to(dtype)``, in one pass for bf16 on a GPU."""
    N, K = q.shape
    if (dtype == torch.bfloat16 and _lib.use_native(q) and K % 128 == 0 and q.dtype == torch.float8_e4m3fn and q.is_contiguous()
            and s.dtype == torch.float32 and s.is_contiguous() and tuple(s.shape) == ((N + 127) // 128, K // 128)
            and q.data_ptr() % 16 == 0 and N > 0):
        out = torch.empty(N, K, dtype=dtype, device=q.device)
        LAUNCHES["quant"] += 1
        _lib.check(_lib.kernels().gk_dequant_128x128(_lib.ptr(q), _lib.ptr(s), _lib.ptr(out), N, K, _lib.stream_ptr()),
                   "dequant_128x128")
        return out
    return dequant_128x128(q, s).to(dtype)


def fp4_quant_1x32_ref(x: torch.Tensor):
    """Returns (codes uint8 [numel] with sign in bit 3, scale fp32 [numel/32], dequantised fp32)."""
    xf = x.float().reshape(-1, 32)
    s = _pow2_ceil(xf.abs().amax(-1).clamp_min(1e-10) / E2M1_MAX)
    y = (xf / s[:, None]).clamp(-E2M1_MAX, E2M1_MAX)
    vals = E2M1_VALUES.to(x.device)
    a = y.abs()
    # nearest representable, ties to the even code (bounds 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5)
    bounds = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    closed_right = torch.tensor([True, False, True, False, True, False, True], device=x.device)
    code = torch.zeros_like(a, dtype=torch.int64)
    for b, cr in zip(bounds.tolist(), closed_right.tolist()):
        code += (a > b).long() if cr else (a >= b).long()
    dq = vals[code] * torch.sign(y) * s[:, None]
    codes = (code | ((y < 0).long() << 3)).to(torch.uint8)
    return codes.reshape(-1), s, dq.reshape(x.shape)


# ------------------------------------------------------------------------------------------------ native wrappers
def quant_act_1x128(x: torch.Tensor, pow2: bool = False):
    """x bf16 [M, K] (K % 128 == 0) -> (q float8_e4m3fn [M, K], scales fp32 [M, K/128])."""
    if not (_lib.use_native(x) and x.dtype == torch.bfloat16 and x.is_contiguous()):
        return act_quant_1x128_ref(x, pow2)
    M, K = x.shape
    q = torch.empty(M, K, dtype=torch.uint8, device=x.device)
    s = torch.empty(M, K // 128, dtype=torch.float32, device=x.device)
    LAUNCHES["quant"] += 1
    _lib.check(_lib.kernels().gk_act_quant_1x128(_lib.ptr(x), _lib.ptr(q), _lib.ptr(s), None, M, K, int(pow2),
                                                 _lib.stream_ptr()), "act_quant")
    return q.view(torch.float8_e4m3fn), s


def quant_weight_128x128(w: torch.Tensor, pow2: bool = False):
    if not (_lib.use_native(w) and w.dtype == torch.bfloat16 and w.is_contiguous()):
        return weight_quant_128x128_ref(w, pow2)
    N, K = w.shape
    q = torch.empty(N, K, dtype=torch.uint8, device=w.device)
    s = torch.empty((N + 127) // 128, (K + 127) // 128, dtype=torch.float32, device=w.device)
    LAUNCHES["quant"] += 1
    _lib.check(_lib.kernels().gk_weight_quant_128x128(_lib.ptr(w), _lib.ptr(q), _lib.ptr(s), None, N, K, int(pow2),
                                                      _lib.stream_ptr()), "weight_quant")
    return q.view(torch.float8_e4m3fn), s


def qat_fp8_(x: torch.Tensor, block: str = "1x128", pow2: bool = True) -> torch.Tensor:
    """In-place quantise -> dequantise round trip (fake quant for QAT) on a bf16 tensor."""
    if _lib.use_native(x) and x.dtype == torch.bfloat16 and x.is_contiguous():
        lib = _lib.kernels()
        LAUNCHES["quant"] += 1
        if block == "1x128":
            x2 = x.view(-1, x.shape[-1])
            _lib.check(lib.gk_act_quant_1x128(_lib.ptr(x2), None, None, _lib.ptr(x2), x2.shape[0], x2.shape[1], int(pow2),
                                              _lib.stream_ptr()), "qat_1x128")
        else:
            _lib.check(lib.gk_weight_quant_128x128(_lib.ptr(x), None, None, _lib.ptr(x), x.shape[0], x.shape[1],
                                                   int(pow2), _lib.stream_ptr()), "qat_128x128")
        return x
    if block == "1x128":
        q, s = act_quant_1x128_ref(x.view(-1, x.shape[-1]), pow2)
        x.copy_(dequant_1x128(q, s).view(x.shape).to(x.dtype))
    else:
        q, s = weight_quant_128x128_ref(x, pow2)
        x.copy_(dequant_128x128(q, s).to(x.dtype))
    return x


def quant_fp4_1x32(x: torch.Tensor):
    """bf16 -> (packed uint8 [numel/2] two e2m1 codes per byte, scale_e8m0 uint8 [numel/32], scale fp32)."""
    n = x.numel()
    if not (_lib.use_native(x) and x.dtype == torch.bfloat16 and x.is_contiguous()):
        codes, s, _ = fp4_quant_1x32_ref(x)
        packed = (codes[0::2] | (codes[1::2] << 4)).to(torch.uint8)
        e8 = (torch.log2(s).round().long() + 127).clamp(0, 254).to(torch.uint8)
        return packed, e8, s
    packed = torch.empty(n // 2, dtype=torch.uint8, device=x.device)
    e8 = torch.empty(n // 32, dtype=torch.uint8, device=x.device)
    s = torch.empty(n // 32, dtype=torch.float32, device=x.device)
    LAUNCHES["quant"] += 1
    _lib.check(_lib.kernels().gk_fp4_quant_1x32(_lib.ptr(x), _lib.ptr(packed), _lib.ptr(e8), _lib.ptr(s), None, n,
                                                _lib.stream_ptr()), "fp4_quant")
    return packed, e8, s


def fp4_to_fp8_rebase(packed: torch.Tensor, scale_f32: torch.Tensor, shape):
    """Lossless re-base of fp4 (e2m1 x power-of-two scale) into e4m3 codes with one fp32 scale per 1x128 block
    (deployment format of the reference's ``fp4_qat_then_to_fp8``): every e2m1 value times a power of two is exactly
    representable in e4m3 as long as the four 1x32 scales inside a 128 block differ by at most 2^6."""
    codes = torch.stack([packed & 0xF, packed >> 4], dim=-1).reshape(-1).long()
    vals = E2M1_VALUES.to(packed.device)[codes & 7] * torch.where((codes & 8) > 0, -1.0, 1.0)
    x = (vals.view(-1, 32) * scale_f32[:, None]).view(shape)
    M, K = x.shape
    blk = x.view(M, K // 128, 128)
    s128 = scale_f32.view(M, K // 128, 4).amax(-1)  # power of two
    q = (blk / s128[..., None]).to(torch.float8_e4m3fn)
    return q.view(M, K), s128


def gemm_fp8_blockscaled(a_q, a_s, b_q, b_s, out_dtype=torch.bfloat16):
    """``C = dequant(a_q, a_s) @ dequant(b_q, b_s)^T`` with a_q [M,K] (1x128 scales [M,K/128]) and b_q [N,K]
    (128x128 scales)."""
    M, K = a_q.shape
    N = b_q.shape[0]
    if not _lib.use_native(a_q):
        return (dequant_1x128(a_q, a_s) @ dequant_128x128(b_q, b_s).t()).to(out_dtype)
    out = torch.empty(M, N, dtype=out_dtype, device=a_q.device)
    LAUNCHES["quant"] += 1
    a_s, b_s = a_s.contiguous(), b_s.contiguous()   # named: a temporary must outlive the asynchronous launch
    rc = _lib.kernels().gk_gemm_fp8_blockscaled(_lib.ptr(a_q), a_q.stride(0), _lib.ptr(b_q), b_q.stride(0),
                                                _lib.ptr(a_s), _lib.ptr(b_s), _lib.ptr(out),
                                                out.stride(0), int(out_dtype == torch.float32), M, N, K,
                                                _lib.ptr(_lib.err_flag(a_q.device)), _lib.stream_ptr())
    _lib.check(rc, "gemm_fp8_blockscaled")
    return out


def transpose_weight_128x128(q: torch.Tensor, s: torch.Tensor, groups: int = 1):
    """Transposed copy of a 128x128-block-scaled e4m3 weight (``[G * N, K]`` -> ``[G * K, N]``, scales alike): a
    square scale block is its own transpose, so the codes move and no value is re-quantised.  This is the B operand
    of the fp8 data-gradient GEMM ``dX = dY W``."""
    GN, K = q.shape
    N = GN // groups
    assert N % 128 == 0 and K % 128 == 0, (N, K)
    qt = q.view(torch.uint8).view(groups, N, K).transpose(1, 2).contiguous().view(groups * K, N).view(q.dtype)
    st = s.view(groups, N // 128, K // 128).transpose(1, 2).contiguous().view(groups * (K // 128), N // 128)
    return qt, st


def fp8_dgrad(dy: torch.Tensor, cache: dict, out_dtype, offsets=None, groups: int = 1):
    """``dX = dY W`` on the block-fp8 GEMM: dY quantised 1x128 along the output features (the contraction), W taken
    from the forward's e4m3 cache in transposed form (built once per weight version).  With ``offsets`` the grouped
    (per-expert) form."""
    if cache.get("t_ver") != cache["ver"]:
        qt, st = transpose_weight_128x128(cache["q"], cache["s"], groups)
        cache.update(t_ver=cache["ver"], qt=qt, st=st)
    gq, gs = quant_act_1x128(dy.to(torch.bfloat16).contiguous())
    od = out_dtype if out_dtype in (torch.bfloat16, torch.float32) else torch.bfloat16
    if offsets is None:
        return gemm_fp8_blockscaled(gq, gs, cache["qt"], cache["st"], out_dtype=od)
    return gemm_fp8_grouped(gq, gs, cache["qt"], cache["st"], offsets, groups, out_dtype=od)


def fp8_wgrad(dy: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """``dW = dY^T X`` (fp32 [N, K]) on the block-fp8 GEMM: the contraction runs over tokens, so dY^T is quantised
    1x128 along tokens and X^T in 128x128 blocks; token counts are padded to a multiple of 128 with zero rows."""
    M = dy.shape[0]
    pad = (-M) % 128
    dyt = torch.nn.functional.pad(dy.to(torch.bfloat16), (0, 0, 0, pad)).t().contiguous()   # [N, M']
    xt = torch.nn.functional.pad(x.to(torch.bfloat16), (0, 0, 0, pad)).t().contiguous()     # [K, M']
    aq, as_ = quant_act_1x128(dyt)
    bq, bs = quant_weight_128x128(xt)
    return gemm_fp8_blockscaled(aq, as_, bq, bs, out_dtype=torch.float32)


def gemm_fp8_grouped(a_q, a_s, b_q, b_s, offsets, num_groups: int, out_dtype=torch.bfloat16):
    """Ragged-M grouped block-fp8 GEMM (experts): rows ``offsets[g]:offsets[g+1]`` of ``a_q`` [R, K] (multiples of
    128; scales ``a_s`` [R, K/128]) multiply group g's weight ``b_q[g * N:(g + 1) * N]`` ([G * N, K] e4m3, 128x128
    scales ``b_s`` [G * N / 128, K / 128]; N a multiple of 128 so that no scale block spans two experts).  Rows of the
    output beyond ``offsets[G]`` are zero."""
    R, K = a_q.shape
    N = b_q.shape[0] // num_groups
    assert N % 128 == 0 and R % 128 == 0, (N, R)
    if not _lib.use_native(a_q) or not hasattr(_lib.kernels(), "gk_gemm_fp8_grouped"):
        a = dequant_1x128(a_q, a_s)
        b = dequant_128x128(b_q, b_s)[:num_groups * N, :K].view(num_groups, N, K)
        out = torch.zeros(R, N, dtype=torch.float32, device=a_q.device)
        off = offsets.tolist()
        for g in range(num_groups):
            if off[g + 1] > off[g]:
                out[off[g]:off[g + 1]] = a[off[g]:off[g + 1]].float() @ b[g].float().t()
        return out.to(out_dtype)
    out = torch.zeros(R, N, dtype=out_dtype, device=a_q.device)
    LAUNCHES["quant"] += 1
    a_s, b_s, offs = a_s.contiguous(), b_s.contiguous(), offsets.int().contiguous()   # named: they must outlive the launch
    rc = _lib.kernels().gk_gemm_fp8_grouped(_lib.ptr(a_q), a_q.stride(0), _lib.ptr(b_q), b_q.stride(0),
                                            _lib.ptr(a_s), _lib.ptr(b_s), _lib.ptr(out),
                                            out.stride(0), int(out_dtype == torch.float32), R, N, K,
                                            _lib.ptr(offs), num_groups,
                                            _lib.ptr(_lib.err_flag(a_q.device)), _lib.stream_ptr())
    _lib.check(rc, "gemm_fp8_grouped")
    return out


class Fp8Linear(torch.nn.Module):
    """Frozen block-fp8 base weight (e4m3 + 128x128 fp32 scales); activations are quantised 1x128 on the fly.  Used
    for the fp8 rollout path and as the frozen base under LoRA."""

    def __init__(self, weight_bf16: torch.Tensor):
        super().__init__()
        q, s = quant_weight_128x128(weight_bf16.contiguous())
        self.register_buffer("weight_q", q)
        self.register_buffer("weight_scale", s)

    def forward(self, x):
        shp = x.shape
        x2 = x.reshape(-1, shp[-1]).contiguous()
        pad = (-x2.shape[1]) % 128
        assert pad == 0, "fp8 linear needs K % 128 == 0"
        aq, as_ = quant_act_1x128(x2)
        y = gemm_fp8_blockscaled(aq, as_, self.weight_q, self.weight_scale, out_dtype=x.dtype
                                 if x.dtype in (torch.bfloat16, torch.float32) else torch.bfloat16)
        return y.reshape(*shp[:-1], self.weight_q.shape[0])


# ------------------------------------------------------------------------------------------------ 4-bit weights
def quant_rows_ref(y: torch.Tensor, scales: str):
    """``(q, s)`` of the rows of ``y``: e4m3 codes with one fp32 scale per 128 values (``fp32``) or the smallest power of two per
    32 values that keeps them within 448 (``e8m0``); a group that holds a NaN or an infinity has the exponent of NaN."""
    if scales == "fp32":
        q, s = act_quant_1x128_ref(y.reshape(-1, y.shape[-1]))
        return q.view(y.shape), s.view(*y.shape[:-1], -1)
    g = y.float().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1).clamp_min(1e-10)
    m, e = torch.frexp(torch.where(torch.isfinite(top), top, torch.ones_like(top)))
    e = e - 9 + (m > 0.875)                     # 448 = 0.875 * 2^9
    q = torch.ldexp(g, -e[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    code = torch.where(torch.isfinite(top), e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return q.view(y.shape), code.view(torch.float8_e8m0fnu)


def quant_act_1x32(x: torch.Tensor):
    """``x`` [..., K] (K a multiple of 32) -> ``(q float8_e4m3fn [..., K], s float8_e8m0fnu [..., K / 32])``, the activations of
    ``gemm_fp4``.  Inference only."""
    K = x.shape[-1]
    if K == 0 or K % 32:
        raise ValueError(f"quant_act_1x32: a width of {K} is not a multiple of 32")
    if _lib.differentiated(x):
        raise RuntimeError("quant_act_1x32 has no gradient: call it under torch.no_grad()")
    if not (_lib.use_native(x) and x.dtype == torch.bfloat16):
        return quant_rows_ref(x, "e8m0")
    if not _lib.is_current(x):
        with torch.cuda.device(x.device):
            return quant_act_1x32(x)
    x2 = _lib.packed16(x)
    q = torch.empty_like(x2, dtype=torch.float8_e4m3fn)
    s = torch.empty((*x.shape[:-1], K // 32), dtype=torch.float8_e8m0fnu, device=x.device)
    LAUNCHES["quant"] += 1
    _lib.check(_lib.kernels().gk_rows_quant(x2.data_ptr(), q.data_ptr(), s.data_ptr(), x2.numel() // K, K, 0, 1, 0,
                                            _lib.stream_ptr()), "rows_quant")
    return q, s


class Fp4Weight:
    """A frozen projection weight ``[N, K]`` in 4 bits, laid out once for the kernels that read it: e2m1 codes, two a byte with
    the even column in the low half, and one power of two per 32 columns.  ``codes`` uint8 [N, K / 2] and ``exponents`` (biased
    by 127; uint8 or float8_e8m0fnu, [N, K / 32]) are what ``quant_fp4_1x32`` makes and what published 4-bit checkpoints hold;
    ``Fp4Weight.of(w)`` quantises.  K is a multiple of 32.  Codes that are laid out as the kernels read them (whole tiles of 128
    columns, packed) are kept as they are, not copied."""

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor):
        if codes.dtype != torch.uint8 or codes.dim() != 2:
            raise ValueError(f"Fp4Weight: codes are uint8 [N, K / 2], got {codes.dtype} {tuple(codes.shape)}")
        N, K = codes.shape[0], 2 * codes.shape[1]
        if N == 0 or K == 0 or K % 32:
            raise ValueError(f"Fp4Weight: [{N}, {K}] (rows, and columns in whole groups of 32, are needed)")
        if exponents.dtype not in (torch.uint8, torch.float8_e8m0fnu) or tuple(exponents.shape) != (N, K // 32):
            raise ValueError(f"Fp4Weight: exponents are uint8 or float8_e8m0fnu [{N}, {K // 32}], got {exponents.dtype} "
                             f"{tuple(exponents.shape)}")
        if exponents.device != codes.device:
            raise ValueError(f"Fp4Weight: codes on {codes.device}, exponents on {exponents.device}")
        self.shape, self.device = (N, K), codes.device
        # columns in whole tiles of 128 (codes behind the last one are zero), rows on 32-byte boundaries
        self.padded = (K + 127) // 128 * 128
        if self.padded != K:
            codes = torch.nn.functional.pad(codes, (0, (self.padded - K) // 2))
        self.codes = codes if codes.is_contiguous() and codes.data_ptr() % 32 == 0 else codes.clone(
            memory_format=torch.contiguous_format)
        # exponents in tiles of 128 rows x 128 columns, 512 bytes: row r at (r % 32) * 16 + (r / 32) * 4
        nt, kt = (N + 127) // 128, self.padded // 128
        e = torch.nn.functional.pad(exponents.view(torch.uint8), (0, 4 * kt - K // 32, 0, 128 * nt - N), value=127)
        self.tiles = _lib.packed16(e.view(nt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4))

    @classmethod
    def of(cls, w: torch.Tensor) -> "Fp4Weight":
        """``w`` [N, K] in 4 bits, each group of 32 columns with the power of two of ``quant_fp4_1x32``."""
        N, K = w.shape
        if K % 32:
            raise ValueError(f"Fp4Weight: {K} columns are not whole groups of 32")
        if _lib.use_native(w) and not _lib.is_current(w):
            with torch.cuda.device(w.device):
                return cls.of(w)
        packed, e8, _ = quant_fp4_1x32(w.detach().contiguous())
        return cls(packed.view(N, K // 2), e8.view(N, K // 32))

    @property
    def exponents(self) -> torch.Tensor:
        """Biased exponents uint8 [N, K / 32]."""
        nt, kt = self.tiles.shape[:2]
        return self.tiles.permute(0, 3, 2, 1, 4).reshape(nt * 128, kt * 4)[:self.shape[0], :self.shape[1] // 32]

    def _bf16(self, rows: int) -> torch.Tensor:
        """On a GPU: values [rows, padded columns] in bf16, zero from the last row of the weight on (rows of the same tile)."""
        out = torch.empty(rows, self.padded, dtype=torch.bfloat16, device=self.device)
        LAUNCHES["quant"] += 1
        _lib.check(_lib.kernels().gk_fp4_dequant(self.codes.data_ptr(), self.tiles.data_ptr(), out.data_ptr(), self.shape[0], rows,
                                                 self.padded, _lib.stream_ptr()), "fp4_dequant")
        return out

    def values(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The weight [N, K] in ``dtype`` (bf16 holds every value below 2^128; the result may be a view of wider rows)."""
        N, K = self.shape
        if dtype == torch.bfloat16 and _lib.use_native(self.codes):
            if not _lib.is_current(self.codes):
                with torch.cuda.device(self.device):
                    return self.values(dtype)
            return self._bf16(N)[:, :K]
        c = torch.stack([self.codes & 15, self.codes >> 4], dim=-1).view(N, self.padded)[:, :K].int()
        v = E2M1_VALUES.to(self.device)[c & 7] * torch.where(c >= 8, -1.0, 1.0)
        e = self.exponents.int()
        scale = torch.where(e == 255, torch.full_like(e, 0, dtype=torch.float32) + float("nan"),
                            torch.ldexp(torch.ones_like(e, dtype=torch.float32), e - 127))
        return (v.view(N, K // 32, 32) * scale[..., None]).view(N, K).to(dtype)


def _check_fp4(what, x, weight, bias):
    if not isinstance(weight, Fp4Weight):
        raise TypeError(f"{what}: weight is an Fp4Weight, got {type(weight).__name__}")
    N, K = weight.shape
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"{what}: x {tuple(x.shape)} against a weight {weight.shape}")
    if x.device != weight.device or (bias is not None and bias.device != x.device):
        raise ValueError(f"{what}: tensors on {x.device}, {weight.device}" + (f", {bias.device}" if bias is not None else ""))
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"{what}: bias {tuple(bias.shape)} for {N} outputs")


def _fp4_product(x2, xs, weight: Fp4Weight, bias, out_dtype):
    """``x2`` [T, K] bf16, or e4m3 with exponents ``xs`` [T, K / 32] (packed, on a GPU), times the weight."""
    (T, K), N = x2.shape, weight.shape[0]
    terms = 2 if xs is None else 1
    lib, dev = _lib.kernels(), x2.device
    y = torch.empty_strided((T, N), (N, 1), dtype=out_dtype, device=dev)
    if T == 0:
        return y
    need = lib.gk_fp4_product_scratch(T, terms, N, weight.padded)
    scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    if bias is not None:
        bias = (bias if bias.dtype in (torch.bfloat16, torch.float32) else bias.float()).contiguous()
    LAUNCHES["quant"] += 2 if need else 1
    _lib.check(lib.gk_fp4_product(
        weight.codes.data_ptr(), weight.tiles.data_ptr(), x2.data_ptr(), xs.data_ptr() if xs is not None else None,
        scratch.data_ptr() if need else None, y.data_ptr(), N, out_dtype == torch.float32,
        bias.data_ptr() if bias is not None else None, bias is not None and bias.dtype == torch.float32, T, terms, N, K,
        weight.padded, _lib.err_flag(dev).data_ptr(), _lib.stream_ptr()), "fp4_product")
    return y


def _fp4_dgrad(dy, weight: Fp4Weight):
    """``dy`` [T, N] times the weight [N, K]: its bf16 values, exact below 2^128, on the framework's GEMM.  The product reads rows
    of ``dy`` in 16-byte units: other widths get columns of zero, and the weight as many rows of zero."""
    from .gemm import linear_dgrad
    (N, K), T = weight.shape, dy.shape[0]
    wide = (N + 7) // 8 * 8
    dy = _lib.packed16(dy)
    if wide != N:
        packed, dy = dy, torch.empty(T, wide, dtype=dy.dtype, device=dy.device)
        LAUNCHES["quant"] += 1
        _lib.check(_lib.kernels().gk_pad_rows16(packed.data_ptr(), dy.data_ptr(), T, N, wide, _lib.stream_ptr()), "pad_rows16")
    return linear_dgrad(dy, weight._bf16(wide)[:, :K])


class _LinearFp4(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, weight, bias):
        ctx.weight, ctx.bias_dtype = weight, bias.dtype if bias is not None else None
        ctx.rows = x2.shape[0]
        return _fp4_product(x2, None, weight, bias, x2.dtype)

    @staticmethod
    def backward(ctx, dy):
        # a graph of the gradient is asked for: it ends here with an error (the decorator's 3 us are not paid otherwise)
        return (_linear_fp4_once if torch.is_grad_enabled() else _linear_fp4_gradients)(ctx, dy)


def _linear_fp4_gradients(ctx, dy):
    dx = db = None
    if ctx.needs_input_grad[0]:
        N, K = ctx.weight.shape
        if dy.shape[0] == 0:
            dx = dy.new_empty(0, K)
        else:
            dx = _fp4_dgrad(dy.to(torch.bfloat16), ctx.weight)
    if ctx.needs_input_grad[2]:
        db = dy.float().sum(0).to(ctx.bias_dtype)
    return dx, None, db


_linear_fp4_once = torch.autograd.function.once_differentiable(_linear_fp4_gradients)


class _LinearFp4Tangent(_LinearFp4):
    """With the forward-mode rule, which alone makes every call of a function 5 us longer."""

    @staticmethod
    def jvp(ctx, x_t, _, bias_t):
        if x_t is None:
            return bias_t.to(torch.bfloat16).expand(ctx.rows, -1).clone()
        return _fp4_product(_lib.packed16(x_t), None, ctx.weight, bias_t, x_t.dtype)


def linear_fp4(x: torch.Tensor, weight: Fp4Weight, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``y = x W^T (+ bias)`` for a frozen 4-bit weight and 16-bit activations, ``x`` [..., K] -> [..., N] in ``x``'s type: the
    product that a model trained with ``fp4_qat`` computes.  Differentiable once in ``x`` and ``bias``, in reverse and forward mode.
    On a GPU bf16 activations run on the kernels; others are multiplied in 32 bits by PyTorch with the weight's values, made anew."""
    _check_fp4("linear_fp4", x, weight, bias)
    N, K = weight.shape
    if not (_lib.use_native(x) and x.dtype == torch.bfloat16):
        y = torch.nn.functional.linear(x.float(), weight.values(torch.float32), bias.float() if bias is not None else None)
        return y.to(x.dtype)
    if not _lib.is_current(x):
        with torch.cuda.device(x.device):
            return linear_fp4(x, weight, bias)
    x2 = _lib.packed16(x if x.dim() == 2 else x.reshape(-1, K))
    if _lib.differentiated(x, bias):
        y = (_LinearFp4Tangent if _lib.has_tangent(x, bias) else _LinearFp4).apply(x2, weight, bias)
    else:
        y = _fp4_product(x2, None, weight, bias, x.dtype)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


def gemm_fp4(a_q: torch.Tensor, a_s: torch.Tensor, weight: Fp4Weight, bias: torch.Tensor | None = None,
             out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``y = dequant(a_q, a_s) W^T (+ bias)``: e4m3 activations ``a_q`` [..., K] with one power of two per 32 values ``a_s``
    (float8_e8m0fnu [..., K / 32]; ``rmsnorm_fp8``, ``swiglu_fp8`` and ``quant_act_1x32`` make them) times a 4-bit weight, in
    ``out_dtype`` (bf16 or fp32).  No gradient."""
    if a_q.dtype != torch.float8_e4m3fn or a_s.dtype != torch.float8_e8m0fnu:
        raise ValueError(f"gemm_fp4: activations are float8_e4m3fn with float8_e8m0fnu scales, got {a_q.dtype}, {a_s.dtype}")
    _check_fp4("gemm_fp4", a_q, weight, bias)
    N, K = weight.shape
    if tuple(a_s.shape) != (*a_q.shape[:-1], K // 32) or a_s.device != a_q.device:
        raise ValueError(f"gemm_fp4: scales {tuple(a_s.shape)} on {a_s.device} for activations {tuple(a_q.shape)} on {a_q.device}")
    if _lib.differentiated(a_q, a_s, bias):
        raise RuntimeError("gemm_fp4 has no gradient: call it under torch.no_grad()")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"gemm_fp4: results are bfloat16 or float32, not {out_dtype}")
    if not _lib.use_native(a_q):
        x = (a_q.float().unflatten(-1, (-1, 32)) * a_s.float()[..., None]).flatten(-2)
        y = torch.nn.functional.linear(x, weight.values(torch.float32), bias.float() if bias is not None else None)
        return y.to(out_dtype)
    if not _lib.is_current(a_q):
        with torch.cuda.device(a_q.device):
            return gemm_fp4(a_q, a_s, weight, bias, out_dtype)
    flat = a_q.dim() == 2
    q2, s2 = _lib.packed16(a_q if flat else a_q.reshape(-1, K)), _lib.packed16(a_s if flat else a_s.reshape(-1, K // 32))
    y = _fp4_product(q2, s2, weight, bias, out_dtype)
    return y if flat else y.view(*a_q.shape[:-1], N)
