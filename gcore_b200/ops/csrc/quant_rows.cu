// Rows that end in e4m3: residual addition + RMSNorm, SwiGLU and plain rows, each quantised in the pass that computes it.
//
//   SC32 = false  one fp32 scale per 128 values, amax / 448 (what gemm_fp8.cu reads)
//   SC32 = true   one power of two per 32 values as its biased exponent (e8m0, what gemm_fp4.cu reads): the smallest that keeps
//                 the group within 448.  A NaN or an infinity in the group makes the exponent 255, which is NaN.
//
// Values stay in 32 bits from the input to the one rounding at the end.  AS16 rounds them to bf16 first, so that the codes and
// scales are those of the unfused kernels (norm or activation to bf16, then the quantiser) bit for bit: the order of every sum
// is rmsnorm_fwd_kernel's (elementwise.cu).
//
// Bound by memory: a norm reads 4 and writes 3 bytes a value with its residual, the activation reads 4 and writes 1; the chains
// they replace write and read the bf16 value in between (4 bytes more) and launch twice.
#include "host_utils.h"
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <type_traits>

namespace gqr {
using namespace gk;

struct alignas(16) Row8 { __nv_bfloat162 v[4]; };

__device__ __forceinline__ void unpack(const Row8& a, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(a.v[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ Row8 pack(const float (&f)[8]) {
  Row8 a;
#pragma unroll
  for (int i = 0; i < 4; ++i) a.v[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  return a;
}

__device__ __forceinline__ uint2 codes8(const float (&f)[8], float inv) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i] * inv, f[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// The largest of the three sizes; NaN if one of them is.
__device__ __forceinline__ float largest(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The upper 22 of 24 bits, to nearest (Veltkamp's splitting).
__device__ __forceinline__ float upper22(float t) {
  const float c = __fmul_rn(t, 5.f);
  return __fadd_rn(c, __fsub_rn(t, c));
}

// Eight values of a thread, f * unit, to codes; the 16 (SC32: 4) neighbouring lanes of its group hold the group's other values.
// All lanes of the warp call this; `at` counts units of eight values over the whole matrix and picks the group's scale.
//
// fp32 scales of a norm that is not rounded in between (TIES): the code is that of f times 448 / amax, one division a group that
// rounds to nearest.  f = x * gain * 2^n is the exact product of two bf16 values, and `unit`, what is left of the norm's factor, is
// not in f / amax.  448 f / amax is then a ratio of 19 bits to 16, so either a tie between two codes (one value in 2 10^4 of bf16
// rows) or more than 2^-21 away from one, 4.1 units in the last place; the product is off by 1.5 of them at most, and rounded to a
// multiple of four it is a tie where the ratio is one, which goes to the even code.  3001 x 1536 values: 289 codes wrong where the
// norm in 32 bits is multiplied by 1 / s, 269 where it is divided by s, none here; us, multiplied / here / a division for each
// value: 3001 x 1536 6.9 / 7.9 / 14.0, 16384 x 4096 with residual 81.3 / 84.4 / 110.
template <bool SC32, bool AS16, bool TIES>
__device__ __forceinline__ void quantise(float (&f)[8], float unit, bool live, long long at, uint2* q, void* scales) {
  if (AS16) unpack(pack(f), f);
  if (SC32) {
    float amax = 1e-10f;
#pragma unroll
    for (int j = 0; j < 8; j += 2) amax = largest(amax, f[j], f[j + 1]);
    amax = largest(amax, __shfl_xor_sync(0xffffffffu, amax, 1), 0.f);
    amax = largest(amax, __shfl_xor_sync(0xffffffffu, amax, 2), 0.f);
    const uint32_t top = __float_as_uint(amax);
    // 448 = 1.75 * 2^8: the exponent is amax's less 8, and one more where the mantissa is above 1.75
    const uint32_t e = top >= 0x7f800000u ? 255u : (top >> 23) - 8u + ((top & 0x7fffffu) > 0x600000u ? 1u : 0u);
    const float inv = __uint_as_float((254u - min(e, 253u)) << 23);
    if (live) {
      q[at] = codes8(f, inv);
      if ((threadIdx.x & 3) == 0) static_cast<uint8_t*>(scales)[at >> 2] = static_cast<uint8_t>(e);
    }
  } else {
    float amax = fabsf(f[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) amax = fmaxf(amax, fabsf(f[j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    float s, inv = 1.f;
    if (AS16 || !TIES) {   // as the chain's quantiser computes them: 2^-22, less than an activation is off
      s = fmaxf(amax, 1e-10f) / 448.f;
      inv = 1.f / s;
    } else {
      // one division for both: the scale in the lane that stores it, 448 / amax in the others
      const bool lead = (threadIdx.x & 15) == 0;
      const float top = amax * unit, under = top > 1e-10f ? amax : 1e-10f / unit;
      s = __fdiv_rn(lead ? fmaxf(top, 1e-10f) : 448.f, lead ? 448.f : under);
      inv = __shfl_sync(0xffffffffu, s, (threadIdx.x & 16) | 1);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = upper22(__fmul_rn(f[j], inv));
      inv = 1.f;
    }
    if (live) {
      q[at] = codes8(f, inv);
      if ((threadIdx.x & 15) == 0) static_cast<float*>(scales)[at >> 4] = s;
    }
  }
}

__device__ __forceinline__ float block_sum(float v, float* red) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) red[w] = v;
  __syncthreads();
  const int nw = (blockDim.x + 31) >> 5;
  float t = lane < nw ? red[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

// A CTA per row, SLOTS units of eight values per thread, kept in registers between the sum and the scaling.
template <int SLOTS, bool SC32, bool AS16>
__global__ void __launch_bounds__(256) norm_quant_kernel(const Row8* __restrict__ x, const Row8* __restrict__ res,
                                                         const Row8* __restrict__ w, uint2* __restrict__ q,
                                                         void* __restrict__ scales, Row8* __restrict__ res_out, int T, int H,
                                                         float eps, float inv_h, int early) {
  __shared__ float red[32];
  pdl_launch_dependents();
  if (!early) pdl_wait();   // the gains may be read before the kernel in front has ended in a decode chain only
  const int nv = H >> 3;
  constexpr bool WIDE = SLOTS <= 2;   // the gains stay in 32 bits where there are registers for it
  Row8 gain[SLOTS];
  float gain32[WIDE ? SLOTS : 1][8];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int i = threadIdx.x + s * 256;
    if (i < nv) {
      gain[s] = w[i];
      if (WIDE) unpack(gain[s], gain32[WIDE ? s : 0]);
    }
  }
  pdl_wait();
  Row8 v[SLOTS], r[SLOTS], vn[SLOTS], rn[SLOTS];
  auto load = [&](int row) {   // the next row's, under way while this one's squares are added up
    if (row >= T) return;
    const long long at = static_cast<long long>(row) * nv;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int i = threadIdx.x + s * 256;
      if (i < nv) {
        vn[s] = x[at + i];
        if (res) rn[s] = res[at + i];
      }
    }
  };
  load(blockIdx.x);
  for (int row = blockIdx.x; row < T; row += gridDim.x) {
    const long long at = static_cast<long long>(row) * nv;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) { v[s] = vn[s]; r[s] = rn[s]; }
    load(row + gridDim.x);
    float ss = 0.f;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int i = threadIdx.x + s * 256;
      if (i < nv) {
        float f[8];
        unpack(v[s], f);
        if (res) {
          float g[8];
          unpack(r[s], g);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] += g[j];
          v[s] = pack(f);
          res_out[at + i] = v[s];
          unpack(v[s], f);  // the norm is that of the 16-bit stream
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
      }
    }
    ss = block_sum(ss, red);
    float factor = rsqrtf((AS16 ? ss / H : ss * inv_h) + eps), unit = 1.f;
    if (!SC32 && !AS16) {   // the power of two and, in `unit`, the rest; zero, infinity and NaN as they are
      const uint32_t bits = __float_as_uint(factor);
      unit = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
      if (bits < 0x7f800000u) factor = __uint_as_float(bits & 0x7f800000u);
    }
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int i = threadIdx.x + s * 256;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (i < nv) {
        float g[8];
        unpack(v[s], f);
        if (!WIDE) unpack(gain[s], g);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = f[j] * factor * (WIDE ? gain32[WIDE ? s : 0][j] : g[j]);
      }
      quantise<SC32, AS16, true>(f, unit, i < nv, at + i, q, scales);
    }
  }
}

// A unit of the activation whose gates may be far below zero: e^-gate or its reciprocal leaves the 32-bit range there, and a large
// partner brings the product back.  With h = e^(-|gate| / 2): gate / (1 + h^2), times h^2 where the gate is negative, half of it in
// front of the partner and half behind.  (For all units it takes 99.7 us instead of 90.2, 8191 x 14336: a second pass of
// rows_quant_kernel does it where it is needed.)
template <bool SC32>
__device__ __noinline__ void far_gates(const Row8* __restrict__ in, long long u, bool live, int nv, uint2* __restrict__ q,
                                       void* __restrict__ scales) {
  float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, p[8];
  if (live) {
    const long long t = u / nv;
    const Row8* gate = in + t * (2 * nv) + (u - t * nv);
    unpack(gate[0], f);
    unpack(gate[nv], p);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float h = __expf(-0.5f * fabsf(f[j])), n = f[j] < 0.f ? h : 1.f;
      f[j] = __fdividef(f[j] * n, fmaf(h, h, 1.f)) * p[j] * n;
    }
  }
  quantise<SC32, false, false>(f, 1.f, live, u, q, scales);
}

// ACT: in = [gate | up] of 2 F values a row, silu(gate) * up; otherwise the row itself.  One unit of eight values per thread.
// Index: int where the units fit (a 64-bit division costs more than the activation).
template <bool ACT, bool SC32, bool AS16, int U, typename Index>
__global__ void __launch_bounds__(256) rows_quant_kernel(const Row8* __restrict__ in, uint2* __restrict__ q,
                                                         void* __restrict__ scales, Index units, int nv) {
  pdl_launch_dependents();
  pdl_wait();
  const long long step = static_cast<long long>(gridDim.x) * (256 * U);
  uint32_t redo = 0, turn = 1;   // iterations with gates far below zero; the last bit stands for all from the 32nd on
  for (long long u0 = blockIdx.x * (256ll * U); u0 < units; u0 += step) {
    uint32_t far = 0;   // the largest bit patterns of gates: those furthest below zero
    Row8 a[U], b[U];
    // one division for all units of an iteration where they span two rows at most
    const bool few = ACT && nv >= 256 * U;
    const Index t0 = few ? static_cast<Index>(u0) / nv : 0, first = few ? static_cast<Index>(u0) - t0 * nv : 0;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const Index u = static_cast<Index>(u0) + k * 256 + static_cast<Index>(threadIdx.x);
      if (u < units) {
        if (ACT) {
          Index t = t0, i = first + k * 256 + static_cast<Index>(threadIdx.x);
          if (!few) {
            t = u / nv;
            i = u - t * nv;
          } else if (i >= nv) {
            ++t;
            i -= nv;
          }
          const Row8* gate = in + static_cast<long long>(t) * (2 * nv) + i;
          a[k] = gate[0];
          b[k] = gate[nv];
        } else {
          a[k] = in[u];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const Index u = static_cast<Index>(u0) + k * 256 + static_cast<Index>(threadIdx.x);
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (u < units) {
        unpack(a[k], f);
        if (ACT) {
          if (!AS16) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(a[k].v);
            far = __vimax3_u16x2(__vimax3_u16x2(far, w[0], w[1]), w[2], w[3]);
          }
          float p[8];
          unpack(b[k], p);
          // Off by 2^-20 + |gate| 2^-23: the exponential by two units and by its argument's rounding, the quotient by two.
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = __fdividef(f[j], 1.f + __expf(-f[j])) * p[j];
        }
      }
      quantise<SC32, AS16, false>(f, 1.f, u < units, u, q, scales);
    }
    if (ACT && !AS16) {
      if (max(far >> 16, far & 0xffffu) > 0xc2a0u) redo |= turn;
      if (turn < 0x80000000u) turn <<= 1;
    }
  }
  // Below a gate of -87 that is zero, as in swiglu.  Where nothing is rounded in between, a warp does the units of the iterations over
  // in which it has a gate below -80 (0xc2a0).  us, 8191 x 14336, without such gates / with a channel of them / with a token in 100 /
  // nothing else: this 91.0 / 99 / 93 / 208, the whole share of a warp over 90.5 / 133 / 102 / 202, no second pass 90.1.
  if (ACT && !AS16) {
    redo = __reduce_or_sync(0xffffffffu, redo);
    turn = 1;
    for (long long u0 = blockIdx.x * (256ll * U); redo && u0 < units; u0 += step) {
      if (redo & turn) {
#pragma unroll 1
        for (int k = 0; k < U; ++k) {
          const long long u = u0 + k * 256 + static_cast<int>(threadIdx.x);
          far_gates<SC32>(in, u, u < units, nv, q, scales);
        }
      }
      if (turn < 0x80000000u) turn <<= 1;
    }
  }
}

inline bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; }

}  // namespace gqr

using namespace gqr;

// x, res (optional, with res_out) [T, H] bf16, w [H] bf16, all 16-byte aligned; q [T, H] e4m3, scales [T, H / 128] fp32 or, with
// sc32, [T, H / 32] e8m0.  H a multiple of 128 (sc32: 32), at most 16384.
GK_EXPORT int gk_norm_quant(const void* x, const void* res, const void* w, void* q, void* scales, void* res_out, int T, int H,
                            float eps, int sc32, int as16, void* stream) {
  if (T < 0 || H <= 0 || H % (sc32 ? 32 : 128) || H > 16384) return -1;
  if (!aligned16(x) || !aligned16(res) || !aligned16(w) || !aligned16(q) || !aligned16(res_out)) return -2;
  if (T == 0) return 0;
  const int sms = gk::sm_count(), grid = T < sms * 8 ? T : sms * 8, nv = H / 8;
  auto go = [&](auto kernel) {
    return gk::launch_waiting(kernel, grid, 256, static_cast<cudaStream_t>(stream), static_cast<const Row8*>(x),
                              static_cast<const Row8*>(res), static_cast<const Row8*>(w), static_cast<uint2*>(q), scales,
                              static_cast<Row8*>(res_out), T, H, eps, 1.f / static_cast<float>(H), gk::pdl_flag());
  };
  auto slots = [&](auto sc, auto as) {
    constexpr bool S = decltype(sc)::value, A = decltype(as)::value;
    if (nv <= 256) return go(norm_quant_kernel<1, S, A>);
    if (nv <= 512) return go(norm_quant_kernel<2, S, A>);
    if (nv <= 1024) return go(norm_quant_kernel<4, S, A>);
    return go(norm_quant_kernel<8, S, A>);
  };
  using Y = std::true_type;
  using N = std::false_type;
  if (sc32) return as16 ? slots(Y{}, Y{}) : slots(Y{}, N{});
  return as16 ? slots(N{}, Y{}) : slots(N{}, N{});
}

// act: in [T, 2 F] bf16 = [gate | up]; otherwise in [T, F], with sc32 and without as16 only.  q [T, F], scales as above; 16-byte aligned.
GK_EXPORT int gk_rows_quant(const void* in, void* q, void* scales, long long T, int F, int act, int sc32, int as16,
                            void* stream) {
  if (T < 0 || F <= 0 || F % (sc32 ? 32 : 128) || (!act && (!sc32 || as16))) return -1;
  if (!aligned16(in) || !aligned16(q)) return -2;
  if (T == 0) return 0;
  const int nv = F / 8;
  // two units under way per thread once every thread of the GPU has one (us, one / two, before the units' rows shared a division:
  // 8191 x 14336 101.7 / 99.5, 64 x 18944 3.6 / 3.9; as it stands 91 and 3.0 in a graph)
  const long long units = T * nv, most = gk::sm_count() * 32ll;
  const bool two = units > gk::sm_count() * 2048ll;
  const long long blocks = two ? (units + 511) / 512 : (units + 255) / 256;
  auto go = [&](auto kernel, auto n) {
    return gk::launch_waiting(kernel, static_cast<unsigned>(blocks < most ? blocks : most), 256, static_cast<cudaStream_t>(stream),
                              static_cast<const Row8*>(in), static_cast<uint2*>(q), scales, n, nv);
  };
  auto pick = [&](auto width, auto n) {
    using I = decltype(n);
    constexpr int U = decltype(width)::value;
    if (!act) return go(rows_quant_kernel<false, true, false, U, I>, n);
    if (sc32) return as16 ? go(rows_quant_kernel<true, true, true, U, I>, n) : go(rows_quant_kernel<true, true, false, U, I>, n);
    return as16 ? go(rows_quant_kernel<true, false, true, U, I>, n) : go(rows_quant_kernel<true, false, false, U, I>, n);
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  if (!two) return pick(One{}, static_cast<int>(units));
  return units < (1ll << 30) ? pick(Two{}, static_cast<int>(units)) : pick(Two{}, units);
}
