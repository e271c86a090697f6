// 4-bit weights: e2m1 codes [N, K / 2] (two a byte, the even column in the low half) with one power of two per 32 columns.
//
// The exponents (e8m0) are kept in tiles of 128 rows x 128 columns, 512 bytes each, row tile by row tile: row r of a tile has the
// four exponents of its columns at byte (r % 32) * 16 + (r / 32) * 4.  K is a multiple of 128 here (padded with zero codes).
#include "host_utils.h"
#include <cuda_bf16.h>
#include <cuda_fp8.h>

namespace gq4 {

// 2^(e - 127); 255 is NaN.  2^-127 and values below 2^-126 become zero (subnormals are flushed).
__device__ __forceinline__ float pow2_of(uint32_t e) {
  return e == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(e << 23);
}
__device__ __forceinline__ float e2m1_value(uint32_t c) {
  const uint32_t m = c & 7u;  // 0, 0.5, then (1 + m0 / 2) * 2^(e - 1)
  const float a = m < 2u ? 0.5f * m : __uint_as_float((126u + (m >> 1)) << 23 | (m & 1u) << 22);
  return c & 8u ? -a : a;
}
__device__ __forceinline__ uint32_t two_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// bf16 values (exact: two significant bits) of the weight, eight per thread.
__global__ void __launch_bounds__(256) fp4_dequant_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ tiles,
                                                          uint4* __restrict__ out, long long units, int per_row) {
  for (long long u = blockIdx.x * 256ll + threadIdx.x; u < units; u += gridDim.x * 256ll) {
    const long long row = u / per_row;
    const int col = static_cast<int>(u - row * per_row) * 8;
    const long long tile = (row >> 7) * (per_row >> 4) + (col >> 7);
    const int r = static_cast<int>(row & 127);
    const float s = pow2_of(tiles[tile * 512 + (r & 31) * 16 + (r >> 5) * 4 + ((col >> 5) & 3)]);
    const uint32_t c = __ldcs(codes + u);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = two_bf16(e2m1_value(c >> (8 * i) & 15u) * s, e2m1_value(c >> (8 * i + 4) & 15u) * s);
    out[u] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// bf16 values (exact: four significant bits) of e4m3 codes with one exponent per 32, eight per thread.
__global__ void __launch_bounds__(256) mxfp8_dequant_kernel(const uint2* __restrict__ q, const uint8_t* __restrict__ e,
                                                            uint4* __restrict__ out, long long units) {
  for (long long u = blockIdx.x * 256ll + threadIdx.x; u < units; u += gridDim.x * 256ll) {
    const float s = pow2_of(e[u >> 2]);
    const uint2 c = q[u];
    const uint32_t w[2] = {c.x, c.y};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3));
      o[i] = two_bf16(__low2float(h) * s, __high2float(h) * s);
    }
    out[u] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

inline unsigned grid_for(long long units) {
  const long long want = (units + 255) / 256, most = gk::sm_count() * 32ll;
  return static_cast<unsigned>(want < most ? want : most);
}

}  // namespace gq4

// codes [N, K / 2], tiles [ceil(N / 128), K / 128, 512], out [N, K] bf16; K a multiple of 128, 16-byte aligned.
GK_EXPORT int gk_fp4_dequant(const void* codes, const void* tiles, void* out, long long N, int K, void* stream) {
  if (N < 0 || K <= 0 || K % 128 || ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(out)) & 15)) return -1;
  const long long units = N * (K / 8);
  if (units == 0) return 0;
  gq4::fp4_dequant_kernel<<<gq4::grid_for(units), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint32_t*>(codes), static_cast<const uint8_t*>(tiles), static_cast<uint4*>(out), units, K / 8);
  return gk::launch_status();
}

// q [T, K] e4m3, e [T, K / 32] e8m0, out [T, K] bf16; K a multiple of 32, 16-byte aligned.
GK_EXPORT int gk_mxfp8_dequant(const void* q, const void* e, void* out, long long T, int K, void* stream) {
  if (T < 0 || K <= 0 || K % 32 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)) return -1;
  const long long units = T * (K / 8);
  if (units == 0) return 0;
  gq4::mxfp8_dequant_kernel<<<gq4::grid_for(units), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint2*>(q), static_cast<const uint8_t*>(e), static_cast<uint4*>(out), units);
  return gk::launch_status();
}
