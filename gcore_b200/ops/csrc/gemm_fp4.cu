// 4-bit weights: e2m1 codes [N, K / 2] (two a byte, the even column in the low half) with one power of two per 32 columns.
//
// The exponents (e8m0) are kept in tiles of 128 rows x 128 columns, 512 bytes each, row tile by row tile: row r of a tile has the
// four exponents of its columns at byte (r % 32) * 16 + (r / 32) * 4.  K is a multiple of 128 here (padded with zero codes).
#include "ptx.cuh"
#include "host_utils.h"
#include <cuda_bf16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

namespace gq4 {
using namespace gk;

inline unsigned grid_for(long long units) {
  const long long want = (units + 255) / 256, most = gk::sm_count() * 32ll;
  return static_cast<unsigned>(want < most ? want : most);
}

// A product whose operands and result may be below 2^-126 (the file is compiled with such values flushed to zero).
__device__ __forceinline__ float times(float a, float b) {
  float c;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
// 2^(e - 127); 255 is NaN.
__device__ __forceinline__ float pow2_of(uint32_t e) {
  return __uint_as_float(e == 255u ? 0x7fffffffu : e == 0u ? 0x400000u : e << 23);
}
__device__ __forceinline__ uint32_t two_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// bf16 values of the weight (exact: two significant bits; infinity from 2^128 on).  A CTA per tile of 128 x 128: sixteen threads a row, eight values each,
// eight rows a thread, so that a warp writes whole lines and eight loads are under way.  Two and a half bytes a value: 6144 x
// 4096 12.3 us (floor 9.9; one row a thread and a division each 22.7).
__global__ void __launch_bounds__(256) fp4_dequant_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ tiles,
                                                          uint4* __restrict__ out, long long N, long long rows, int kb) {
  const int k = blockIdx.x % kb;
  const long long row0 = static_cast<long long>(blockIdx.x / kb) * 128;
  const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const uint8_t* sf = tiles + static_cast<long long>(blockIdx.x) * 512 + (c >> 2);
  const long long at = (row0 + r0) * kb * 16 + k * 16 + c, step = 16ll * kb * 16;   // units of eight values
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = row0 + r0 + 16 * i < N ? __ldcs(codes + at + i * step) : 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i;
    if (row0 + r >= rows) break;
    const float s = pow2_of(sf[(r & 31) * 16 + (r >> 5) * 4]);
    uint32_t o[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const __half2 h = __half2(__nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(w[i] >> (8 * b)), __NV_E2M1));
      o[b] = two_bf16(times(__low2float(h), s), times(__high2float(h), s));
    }
    out[at + i * step] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// Rows of N 16-bit values to rows of 16-byte units, zero behind the last value: what a tensor-core operand's rows start on.  A
// thread makes a unit out of the five words that its values lie in, whatever boundary they start on.
__global__ void __launch_bounds__(256) pad_rows16_kernel(const uint32_t* __restrict__ src, uint4* __restrict__ dst, long long units,
                                                         int N, int per, long long values) {
  for (long long u = blockIdx.x * 256ll + threadIdx.x; u < units; u += gridDim.x * 256ll) {
    const long long row = u / per;
    const int c = static_cast<int>(u - row * per) * 8, left = N - c;   // values of the row from here on
    const long long at = row * N + c, word = at >> 1;
    uint32_t w[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      const long long k = 2 * (word + j);
      w[j] = 0;
      if (k + 1 < values) w[j] = src[word + j];
      else if (k < values) w[j] = reinterpret_cast<const uint16_t*>(src)[k];   // the last of an odd number
    }
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[j] = at & 1 ? __funnelshift_r(w[j], w[j + 1], 16) : w[j];
      if (2 * j + 1 >= left) o[j] = 2 * j < left ? o[j] & 0xffffu : 0u;
    }
    dst[u] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ---------------------------------------------------------------------------------------------- few tokens
// y[T, N] = x[T, K] W[N, K]^T (+ bias) on the block-scaled tensor core (kind::mxf8f6f4), which takes e2m1 and e4m3 operands with
// one e8m0 exponent per 32 values of K: the codes of the weight go from memory to the product as they are.
//
//   * The 128-row tile runs over output features, the tokens are the product's N (swap-AB).  A product instruction takes the same 70
//     cycles for 16 columns as for 128, and its operands' and descriptors' way to the tensor core is what the issuing warp spends
//     its time on: with one lane in a branch of its own 64 tokens of 3584 x 18944 took 79 us in one piece, now 46.
//   * 16-bit activations enter as two e4m3 terms, x = 2^e (hi + lo / 16) with one e per 32 values: hi keeps four significant bits, lo
//     the four behind them down to a step of 2^-9, 2^-13 of hi's unit.  With the group's largest between 224 and 448 of it a
//     bf16 value at most 2^13 below that largest is exact, and a smaller one is off by less than 2^-21 of it (half a step, 2^-14,
//     of 224).  The terms are separate columns of one product; the epilogue adds them.
//   * K is divided over a cluster of `ks` CTAs where there are few tiles: CTA r finishes tokens r, r + ks, ..., whose partial sums
//     the others send it through distributed shared memory in one copy each (stores of 128 bytes a warp took 20 us for 64
//     tokens); it adds them in the order of the CTAs.
//
// The weight's bytes bound it with a token or two (half a byte a value and a 32nd for the exponents), the tokens' operand on its way
// out of L2, 16 KB a K block of 64 tokens for 8.7 KB of weight, from a few dozen on.
constexpr int BM = 128, BK = 128, UK = 32;
constexpr int THREADS = 320;          // one warp loads, one issues, eight read the result (the first four also prepare tokens)
constexpr int MAX_STAGES = 8;
constexpr int A_BYTES = BM * BK;      // a row of 128 codes takes 128 bytes in shared memory: 16 codes and 8 bytes of gap a unit
constexpr int SF_BYTES = 512;         // exponents of 128 rows x 128 columns

// Where the product's token operand comes from.
enum Tokens : int {
  SPLIT = 0,   // the two terms of bf16 rows and their exponents, made by fp4_split_kernel
  ROWS16 = 1,  // bf16 rows, split into each stage of the ring by four of the epilogue's warps (up to 8 tokens)
  ROWS8 = 2,   // e4m3 rows; the same warps bring the exponents into place
};

struct Fp4Params {
  int total, Tc, Tp, terms, N, kb, ks, stages, cols;   // tokens in all and per CTA; cols: columns of the product (Tp * terms)
  int K;                                       // columns that the tokens really have
  int ring;                                    // bytes of the operands' ring, or of the partial sums that use it later
  const uint8_t* tiles;                        // weight exponents
  const void* x;                               // ROWS16: rows
  const uint8_t* sf;                           // SPLIT: exponents [chunk, kb, ceil(cols / 128), 512]; ROWS8: [total, K / 32]
  void* Y;
  long long ldy;
  int out_fp32;
  const void* bias;
  int bias_fp32;
  int early;                                   // the weight may be read before the kernel in front has ended
  int* err;
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// The tensor core's instructions of the decode kernel: the whole warp runs up to them and one lane (`go`) issues, so that
// addresses and descriptors stay in uniform registers.  512 bytes of exponents (32 rows of 16) to four columns of tensor memory,
// the same for each quarter of the lanes:
__device__ __forceinline__ void sf_to_tmem(uint32_t go, uint32_t taddr, uint32_t smem_addr) {
  const uint64_t desc = static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) |
                        (static_cast<uint64_t>(1) << 46);
  asm volatile(
      "{\n"
      ".reg .pred q;\n"
      "setp.ne.b32 q, %2, 0;\n"
      "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n"
      "}\n" ::"r"(taddr),
      "l"(desc), "r"(go)
      : "memory");
}
__device__ __forceinline__ void umma_mx(uint32_t go, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "setp.ne.b32 q, %7, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(go)
      : "memory");
}
__device__ __forceinline__ void umma_commit_if(uint32_t go, uint64_t* bar) {
  asm volatile(
      "{\n"
      ".reg .pred q;\n"
      "setp.ne.b32 q, %1, 0;\n"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
      "}\n" ::"r"(smem_u32(bar)),
      "r"(go)
      : "memory");
}
// fmt: 0 = e4m3, 5 = e2m1; exponents are e8m0.  Bits 4 and 29 and the ones above each count the byte of the four exponents that a
// lane holds per column (B's and A's).
__device__ __forceinline__ uint32_t mx_idesc(int m, int n, int a_fmt, int b_fmt) {
  return (static_cast<uint32_t>(a_fmt) << 7) | (static_cast<uint32_t>(b_fmt) << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (1u << 23) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t in_cta(uint32_t local, uint32_t cta) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(cta));
  return at;
}
// Own shared memory to another CTA's of the cluster; `bar` is that CTA's.
__device__ __forceinline__ void bulk_send(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "r"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}

// Eight bf16 values of a group of 32 (four neighbouring lanes; the whole warp calls this) as two e4m3 terms and the exponents of
// both; 255 where the group holds a NaN or an infinity.
struct Terms {
  uint2 hi, lo;
  uint32_t e_hi, e_lo;
};
__device__ __forceinline__ Terms split8(const uint4& raw) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  // bf16 pattern of the largest: eight bits of exponent, seven of mantissa; 448 = 1.75 * 2^8 as in quant_rows.cu.  The lo term's
  // exponent is four less, so the hi term's is at least 4: a group whose largest is below 2^-115 keeps steps of 2^-136.
  const uint32_t e = static_cast<uint32_t>(max(static_cast<int>(top >> 7) - 8 + ((top & 0x7fu) > 0x60u ? 1 : 0), 4));
  const bool bad = top >= 0x7f80u;
  const float inv = __uint_as_float((254u - (bad ? 127u : e)) << 23);
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = times(__uint_as_float(w[i] << 16), inv), b = times(__uint_as_float(w[i] & 0xffff0000u), inv);
    hi[i] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(hi[i]), __NV_E4M3));
    lo[i] = __nv_cvt_float2_to_fp8x2(make_float2((a - __low2float(h)) * 16.f, (b - __high2float(h)) * 16.f), __NV_SATFINITE,
                                     __NV_E4M3);
  }
  Terms t;
  t.hi = make_uint2(hi[0] | (hi[1] << 16), hi[2] | (hi[3] << 16));
  t.lo = make_uint2(lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16));
  t.e_hi = bad ? 255u : e;
  t.e_lo = bad ? 255u : e - 4u;
  return t;
}
// Byte of exponent k4 of row r in tiles of 128 rows x 128 columns.
__device__ __forceinline__ int sf_at(int r, int k4) { return (r >> 7) * SF_BYTES + (r & 31) * 16 + ((r >> 5) & 3) * 4 + k4; }

// SRC: Tokens.  UNITS (ROWS16): units of eight values per lane of a preparing warp and K block, two tokens each.
template <int SRC, int UNITS>
__global__ void __launch_bounds__(THREADS)
fp4_decode_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, Fp4Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int nsf = (p.cols + 127) / 128, ks_log = 31 - __clz(p.ks);    // ks is 1, 2, 4 or 8
  const int b_bytes = p.cols * BK;                                    // a multiple of 2048
  const int stage_bytes = A_BYTES + b_bytes;
  const int sf_stage = SF_BYTES * (1 + nsf);
  const int chunk = blockIdx.y, tok0 = chunk * p.Tc, T = min(p.Tc, p.total - tok0);   // this CTA's tokens
  const int cs = (p.Tc + p.ks - 1) / p.ks;                            // token columns that a CTA of the cluster finishes
  float* part = reinterpret_cast<float*>(smem);                       // own partial sums [ks][cs][128], over the finished ring
  uint8_t* sf_smem = smem + p.ring;                                   // per stage: the weight's exponents, the tokens'
  float* red = reinterpret_cast<float*>(sf_smem + p.stages * sf_stage);   // the other CTAs' [ks][cs][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(red + (p.ks > 1 ? p.ks * cs * BM : 0));
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* tfull = empty + MAX_STAGES;
  uint64_t* rfull = tfull + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(rfull + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x % p.ks;   // in the cluster
  const int tile = blockIdx.x / p.ks;
  const int n0 = tile * BM;
  // K blocks in shares that differ by one at most
  const int kb0 = static_cast<int>(static_cast<long long>(p.kb) * rank / p.ks);
  const int kblocks = static_cast<int>(static_cast<long long>(p.kb) * (rank + 1) / p.ks) - kb0;
  const int acc_cols = (p.cols + 31) & ~31, sf_cols = 4 * (1 + nsf);
  uint32_t tmem_cols = 32;
  while (tmem_cols < static_cast<uint32_t>(acc_cols + p.stages * sf_cols)) tmem_cols <<= 1;
  // the gaps between the codes do not count
  const uint32_t stage_tx = A_BYTES / 2 + SF_BYTES + (SRC == ROWS16 ? 0 : b_bytes) + (SRC == SPLIT ? nsf * SF_BYTES : 0);

  const uint8_t* tile_sf = p.tiles + (static_cast<long long>(tile) * p.kb + kb0) * SF_BYTES;
  const uint8_t* token_sf = p.sf + (SRC == SPLIT ? (static_cast<long long>(chunk) * p.kb + kb0) * nsf * SF_BYTES : 0);
  const int token_row = SRC == SPLIT ? chunk * p.cols : tok0;
  auto load_weight = [&](int s, int kb) {
    mbar_expect_tx(&full[s], stage_tx);
    tma_load_2d(smem + s * stage_bytes, &tmW, &full[s], (kb0 + kb) * BK, n0);
    bulk_load(sf_smem + s * sf_stage, tile_sf + kb * SF_BYTES, SF_BYTES, &full[s]);
  };
  auto load_tokens = [&](int s, int kb) {
    if (SRC != ROWS16) tma_load_2d(smem + s * stage_bytes + A_BYTES, &tmX, &full[s], (kb0 + kb) * BK, token_row);
    if (SRC == SPLIT)
      bulk_load(sf_smem + s * sf_stage + SF_BYTES, token_sf + static_cast<long long>(kb) * nsf * SF_BYTES, SF_BYTES * nsf, &full[s]);
  };

  int pre = 0, loaded = 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(&full[s], SRC == SPLIT ? 1 : 2); mbar_init(&empty[s], 1); }
    mbar_init(tfull, 1);
    mbar_init(rfull, 1);
    fence_barrier_init();
    if (p.ks > 1) mbar_expect_tx(rfull, (p.ks - 1) * cs * BM * 4);
    pre = kblocks < p.stages ? kblocks : p.stages;
    if (!p.early) pdl_wait();
    for (int kb = 0; kb < pre; ++kb) load_weight(kb, kb);
    pdl_wait();
    for (int kb = 0; kb < pre; ++kb) load_tokens(kb, kb);
  }
  // Tensor memory is taken behind the wait, and the kernel behind this one is let go when it has been: a CTA that held some while
  // it waited for a kernel whose CTA still wanted some could stop both.
  pdl_wait();
  if (warp == 2) { tmem_alloc(tmem_holder, tmem_cols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_holder);
  pdl_launch_dependents();
  if (p.ks > 1) cluster_arrive();   // "this CTA runs"; the wait is in front of what it is sent

  bool ok = true;
  if (warp == 0) {
    pre = __shfl_sync(0xffffffffu, pre, 0);
    loaded = pre;
    int s = pre == p.stages ? 0 : pre;
    uint32_t ph = pre == p.stages ? 1 : 0;
    for (int kb = pre; kb < kblocks; ++kb) {
      ok = mbar_wait_warp(&empty[s], ph ^ 1, p.err, ERR_WAIT_EMPTY);
      if (!ok) break;
      if (lane == 0) { load_weight(s, kb); load_tokens(s, kb); }
      __syncwarp();
      ++loaded;
      if (++s == p.stages) { s = 0; ph ^= 1; }
    }
    if (p.ks > 1) cluster_wait();
  } else if (warp == 1) {
    const uint32_t go = elect_one() ? 1 : 0, idesc = mx_idesc(BM, p.cols, 5, 0);
    int s = 0;
    uint32_t ph = 0;
    for (int kb = 0; kb < kblocks; ++kb) {
      ok = mbar_wait_warp(&full[s], ph, p.err, ERR_WAIT_FULL);
      if (!ok) break;
      tc_fence_after();
      const uint32_t a = smem_u32(smem + s * stage_bytes), b = a + A_BYTES, f = smem_u32(sf_smem + s * sf_stage);
      const uint32_t sfa = tmem_base + acc_cols + s * sf_cols, sfb = sfa + 4;
      for (int j = 0; j < 1 + nsf; ++j) sf_to_tmem(go, sfa + 4 * j, f + SF_BYTES * j);
#pragma unroll
      for (int k4 = 0; k4 < BK / UK; ++k4)
        umma_mx(go, tmem_base, make_smem_desc_sw128(a + k4 * UK, 16, 1024), make_smem_desc_sw128(b + k4 * UK, 16, 1024),
                idesc + k4 * ((1u << 4) + (1u << 29)), sfa, sfb, (kb > 0 || k4 > 0) ? 1u : 0u);
      umma_commit_if(go, &empty[s]);
      if (kb == kblocks - 1) umma_commit_if(go, tfull);
      if (++s == p.stages) { s = 0; ph ^= 1; }
    }
    if (!ok) {   // products under way end before the CTA gives its memory back
      umma_commit_if(go, tfull);
      mbar_land(tfull, 0);
    }
    if (p.ks > 1) cluster_wait();
  } else {
    // A K block's tokens are one warp's: its chain of load, split, store and fence takes 0.4 us, so four blocks are under way at a
    // time, and each warp has its next block's loads in flight.  Never more warps than stages: a warp's last block is then at most
    // a round of the ring behind, and the parity of a stage's barrier tells it whether the stage is free.
    const int workers = p.stages < 4 ? p.stages : 4;
    if (SRC == ROWS16 && warp - 2 < workers) {
      constexpr int U = UNITS > 0 ? UNITS : 1;
      const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x);
      const int c = lane & 15, t0 = lane >> 4;   // unit j: token 2 j + t0, eight values from column 8 c
      uint4 raw[U];
      auto fetch = [&](int kb) {
        const int col = (kb0 + kb) * BK + c * 8;
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int t = 2 * j + t0;
          raw[j] = kb < kblocks && t < T && col < p.K ? *reinterpret_cast<const uint4*>(x + static_cast<long long>(t) * p.K + col)
                                                        : make_uint4(0, 0, 0, 0);
        }
      };
      fetch(warp - 2);
      int s = warp - 2;
      uint32_t ph = 0;
      for (int kb = warp - 2; kb < kblocks; kb += workers, s += workers) {
        while (s >= p.stages) { s -= p.stages; ph ^= 1; }
        Terms v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) v[j] = split8(raw[j]);
        fetch(kb + workers);
        ok = mbar_wait_warp(&empty[s], ph ^ 1, p.err, ERR_WAIT_EMPTY);
        if (!ok) break;
        uint8_t* b = smem + s * stage_bytes + A_BYTES;
        uint8_t* f = sf_smem + s * sf_stage + SF_BYTES;
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int t = 2 * j + t0, l = p.Tp + t;
          if (t >= T) continue;
          // 16-byte piece c / 2 of the row, in the order of the 128-byte swizzle
          *reinterpret_cast<uint2*>(b + t * BK + (((c >> 1) ^ (t & 7)) << 4) + (c & 1) * 8) = v[j].hi;
          *reinterpret_cast<uint2*>(b + l * BK + (((c >> 1) ^ (l & 7)) << 4) + (c & 1) * 8) = v[j].lo;
          if ((c & 3) == 0) {
            f[sf_at(t, c >> 2)] = static_cast<uint8_t>(v[j].e_hi);
            f[sf_at(l, c >> 2)] = static_cast<uint8_t>(v[j].e_lo);
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[s]);
      }
    } else if (SRC == ROWS8 && warp - 2 < workers) {
      const int per = p.K / 32;
      uint32_t w[4], next[4];
      auto fetch = [&](uint32_t (&to)[4], int kb) {   // exponents of a K block for tokens lane, lane + 32, ...; 1 behind the last column
        const int at = (kb0 + kb) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = lane + 32 * j;
          to[j] = 0;
          if (t >= T || kb >= kblocks) continue;
          const uint8_t* mine = p.sf + static_cast<long long>(tok0 + t) * per + at;
          if ((per & 3) == 0) {
            to[j] = *reinterpret_cast<const uint32_t*>(mine);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) to[j] |= (at + i < per ? mine[i] : 127u) << (8 * i);
          }
        }
      };
      fetch(w, warp - 2);
      fetch(next, warp - 2 + workers);
      int s = warp - 2;
      uint32_t ph = 0;
      for (int kb = warp - 2; kb < kblocks; kb += workers, s += workers) {
        while (s >= p.stages) { s -= p.stages; ph ^= 1; }
        ok = mbar_wait_warp(&empty[s], ph ^ 1, p.err, ERR_WAIT_EMPTY);
        if (!ok) break;
        uint8_t* f = sf_smem + s * sf_stage + SF_BYTES;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (lane + 32 * j < T) *reinterpret_cast<uint32_t*>(f + sf_at(lane + 32 * j, 0)) = w[j];
          w[j] = next[j];
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[s]);
        fetch(next, kb + 2 * workers);
      }
    }
    // Epilogue: a lane per output feature; the warps of the two halves take eight tokens in turn.
    const int quad = warp & 3, half = (warp - 2) >> 2, row = quad * 32 + lane, feat = n0 + row;
    ok = ok && mbar_wait_warp(tfull, 0, p.err, ERR_WAIT_TMEM_FULL) && *reinterpret_cast<volatile int*>(p.err) == 0;
    ok = __all_sync(0xffffffffu, ok) != 0;
    tc_fence_after();
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    float bias = 0.f;
    if (p.bias && feat < p.N)
      bias = p.bias_fp32 ? static_cast<const float*>(p.bias)[feat] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[feat]);
    const long long y0 = tok0 * p.ldy + feat;
    auto store = [&](int tok, float v) {
      if (p.out_fp32) static_cast<float*>(p.Y)[y0 + tok * p.ldy] = v;
      else static_cast<__nv_bfloat16*>(p.Y)[y0 + tok * p.ldy] = __float2bfloat16(v);
    };
    if (ok) {
      for (int c = half * 16; c < T; c += 32) {
        uint32_t r[2][8], l[2][8];   // sixteen tokens a wait
        tmem_ld8(taddr + c, r[0]);
        if (c + 8 < T) tmem_ld8(taddr + c + 8, r[1]);
        if (p.terms == 2) {
          tmem_ld8(taddr + p.Tp + c, l[0]);
          if (c + 8 < T) tmem_ld8(taddr + p.Tp + c + 8, l[1]);
        }
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int tok = c + j;
          if (tok >= T) break;
          float v = __uint_as_float(r[j >> 3][j & 7]);
          if (p.terms == 2) v += __uint_as_float(l[j >> 3][j & 7]);
          if (p.ks > 1) part[((tok & (p.ks - 1)) * cs + (tok >> ks_log)) * BM + row] = v;
          else if (feat < p.N) store(tok, v + bias);
        }
      }
    }
    if (p.ks > 1) {
      fence_proxy_async();
      cluster_wait();   // every CTA of the cluster runs: it may be sent something
      asm volatile("bar.sync 1, 256;" ::: "memory");
      // sent whether or not this CTA is well: the others wait for it
      if (threadIdx.x == 64) {
        for (int o = 1; o < p.ks; ++o) {
          const uint32_t to = (rank + o) % p.ks;
          bulk_send(in_cta(smem_u32(red + static_cast<int>(rank) * cs * BM), to), smem_u32(part + static_cast<int>(to) * cs * BM),
                    cs * BM * 4, in_cta(smem_u32(rfull), to));
        }
      }
      __syncwarp();
      const bool got = mbar_wait_warp(rfull, 0, p.err, ERR_WAIT_MISC);
      if (!got) mbar_land(rfull, 0);
      ok = __all_sync(0xffffffffu, ok && got && *reinterpret_cast<volatile int*>(p.err) == 0) != 0;
      if (ok && feat < p.N) {
        for (int j = half; j * p.ks + static_cast<int>(rank) < T; j += 2) {
          float v = 0.f;
          for (int r = 0; r < p.ks; ++r) v += (r == static_cast<int>(rank) ? part : red)[(r * cs + j) * BM + row];
          store(j * p.ks + rank, v + bias);
        }
      }
    }
    tc_fence_before();
  }
  if (p.ks > 1) {   // what this CTA sent has been read: its owners have seen it arrive
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_before();
  const bool failed = __syncthreads_or(!ok);
  if (failed && warp == 0) {   // copies that nobody waits for any more land before the CTA gives its memory back
    for (int kb = loaded > p.stages ? loaded - p.stages : 0; kb < loaded; ++kb)
      mbar_land(&full[kb % p.stages], static_cast<uint32_t>(kb / p.stages) & 1);
  }
  if (warp == 2) { tc_fence_after(); tmem_dealloc(tmem_base, tmem_cols); }
}

// bf16 rows to their terms, eight values a thread, chunk by chunk of `Tc` tokens: codes [2 Tp, Kp] of a chunk, hi rows first, and
// exponents in tiles of 128 code rows x 128 columns, `per_chunk`, `per_kb` and `per_tile` tiles from one chunk, K block and 128
// rows to the next.  Columns from K to Kp become zero.
struct SplitLayout {
  int T, Tc, Tp, K, Kp, per_chunk, per_kb, per_tile;
};
__global__ void __launch_bounds__(256) fp4_split_kernel(const uint4* __restrict__ x, uint2* __restrict__ codes,
                                                        uint8_t* __restrict__ sf, SplitLayout p) {
  pdl_wait();
  pdl_launch_dependents();
  const int per = p.Kp / 8, live = p.K / 8;
  const long long units = static_cast<long long>(p.T) * per;   // a multiple of 16
  for (long long u0 = blockIdx.x * 256ll; u0 < units; u0 += gridDim.x * 256ll) {
    const long long u = u0 + threadIdx.x;
    const int tok = static_cast<int>(u / per), c = static_cast<int>(u - static_cast<long long>(tok) * per);
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (u < units && c < live) raw = x[static_cast<long long>(tok) * live + c];
    const Terms v = split8(raw);
    if (u < units) {
      const int chunk = tok / p.Tc, t = tok - chunk * p.Tc, l = p.Tp + t;
      const long long row = static_cast<long long>(chunk) * (2 * p.Tp) + t;
      codes[row * per + c] = v.hi;
      codes[(row + p.Tp) * per + c] = v.lo;
      if ((c & 3) == 0) {
        const int k4 = (c >> 2) & 3;
        const long long at = static_cast<long long>(chunk) * p.per_chunk + static_cast<long long>(c >> 4) * p.per_kb;
        sf[(at + static_cast<long long>(t >> 7) * p.per_tile) * SF_BYTES + sf_at(t & 127, k4)] = static_cast<uint8_t>(v.e_hi);
        sf[(at + static_cast<long long>(l >> 7) * p.per_tile) * SF_BYTES + sf_at(l & 127, k4)] = static_cast<uint8_t>(v.e_lo);
      }
    }
  }
}

// Exponents [T, K / 32] to tiles of 128 rows x 128 columns, row tile by row tile; 1 behind the last column.
__global__ void __launch_bounds__(256) fp4_tiles_kernel(const uint8_t* __restrict__ s, uint8_t* __restrict__ sf, int T, int per,
                                                        int kb) {
  pdl_wait();
  pdl_launch_dependents();
  const long long n = static_cast<long long>(T) * kb;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int t = static_cast<int>(i / kb), k = static_cast<int>(i - static_cast<long long>(t) * kb);
    const uint8_t* from = s + static_cast<long long>(t) * per + k * 4;
    uint32_t w = 0;
    if ((per & 3) == 0) {
      w = *reinterpret_cast<const uint32_t*>(from);
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b) w |= (k * 4 + b < per ? from[b] : 127u) << (8 * b);
    }
    *reinterpret_cast<uint32_t*>(sf + (static_cast<long long>(t >> 7) * kb + k) * SF_BYTES + sf_at(t & 127, 0)) = w;
  }
}

// ---------------------------------------------------------------------------------------------- many tokens
// The same product with the tokens as its rows: tiles of 128 tokens x 256 output features, one after another on each SM.  The
// 256 columns of the sum and the exponents' columns leave no room for a second sum, so the eight epilogue warps take it to
// registers (128 a thread) before they round and store it, and the next tile's products begin meanwhile.  TERMS = 2: both
// terms of a bf16 row meet the weight tile in one K block, so a weight byte serves twice the operations.
// The tensor core takes 512 cycles for a term's K block; what it needs from L2 meanwhile, 33.5 KB (TERMS = 2: 50 KB in 1024
// cycles), is about what an SM gets.
constexpr int PM = 128, PN = 256;
constexpr int P_THREADS = 320;
template <int TERMS>
struct PromptCfg {
  static constexpr int A_TILE = PM * BK, B_TILE = PN * BK, OPERANDS = TERMS * A_TILE + B_TILE;
  static constexpr int SF = SF_BYTES * (TERMS + 2);
  static constexpr int STAGES = TERMS == 1 ? 4 : 3;
  static constexpr int PATCH = 32 * 80;       // a warp's 32 tokens x 64 bytes on their way to memory, rows 80 bytes apart
  static constexpr int SMEM = STAGES * (OPERANDS + SF) + 8 * PATCH + 1024 + 256;
  static constexpr uint32_t TX = TERMS * A_TILE + B_TILE / 2 + SF;
};

struct PromptParams {
  int T, N, kb, mt, nt, lo_rows, band;   // mt, nt: tiles; lo_rows: code rows from a hi term to its lo term
  const uint8_t* tiles;                  // weight exponents
  const uint8_t* sf;                     // token exponents [code rows / 128, kb, 512]
  void* Y;
  long long ldy;
  int out_fp32;
  const void* bias;
  int bias_fp32;
  int* err;
};

template <int TERMS>
__global__ void __launch_bounds__(P_THREADS, 1)
fp4_prompt_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, PromptParams p) {
  using C = PromptCfg<TERMS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sf_smem = smem + C::STAGES * C::OPERANDS;
  uint8_t* patches = sf_smem + C::STAGES * C::SF;
  uint64_t* full = reinterpret_cast<uint64_t*>(sf_smem + C::STAGES * C::SF + 8 * C::PATCH);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tempty + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ntiles = p.mt * p.nt;
  const int last_w = (p.N + BM - 1) / BM - 1;
  constexpr int SF_COLS = 4 * (TERMS + 2);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(tfull, 1);
    mbar_init(tempty, 8);
    fence_barrier_init();
  }
  pdl_wait();                // tensor memory is taken behind it, as in the kernel above
  if (warp == 2) { tmem_alloc(tmem_holder, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_holder);
  pdl_launch_dependents();

  bool ok = true;
  int loaded = 0;
  if (warp == 0) {
    int s = 0;
    uint32_t ph = 0;
    for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x) {
      int mi, ni;
      raster_tile(t, p.mt, p.nt, p.band, mi, ni);
      for (int kb = 0; kb < p.kb; ++kb) {
        ok = mbar_wait_warp(&empty[s], ph ^ 1, p.err, ERR_WAIT_EMPTY);
        if (!ok) break;
        if (lane == 0) {
          uint8_t* a = smem + s * C::OPERANDS;
          uint8_t* f = sf_smem + s * C::SF;
          mbar_expect_tx(&full[s], C::TX);
#pragma unroll
          for (int i = 0; i < TERMS; ++i) {
            tma_load_2d(a + i * C::A_TILE, &tmX, &full[s], kb * BK, mi * PM + i * p.lo_rows);
            bulk_load(f + i * SF_BYTES, p.sf + (static_cast<long long>(mi + i * (p.lo_rows / PM)) * p.kb + kb) * SF_BYTES, SF_BYTES,
                      &full[s]);
          }
          tma_load_2d(a + TERMS * C::A_TILE, &tmW, &full[s], kb * BK, ni * PN);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int w = 2 * ni + i < last_w ? 2 * ni + i : last_w;   // exponents behind the last tile meet zero codes
            bulk_load(f + (TERMS + i) * SF_BYTES, p.tiles + (static_cast<long long>(w) * p.kb + kb) * SF_BYTES, SF_BYTES, &full[s]);
          }
        }
        __syncwarp();
        ++loaded;
        if (++s == C::STAGES) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    const uint32_t go = elect_one() ? 1 : 0, idesc = mx_idesc(PM, PN, 0, 5);
    int s = 0, n = 0;
    uint32_t ph = 0;
    for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x, ++n) {
      ok = mbar_wait_warp(tempty, (n & 1) ^ 1, p.err, ERR_WAIT_TMEM_EMPTY);
      if (!ok) break;
      tc_fence_after();
      for (int kb = 0; kb < p.kb; ++kb) {
        ok = mbar_wait_warp(&full[s], ph, p.err, ERR_WAIT_FULL);
        if (!ok) break;
        tc_fence_after();
        const uint32_t a = smem_u32(smem + s * C::OPERANDS), b = a + TERMS * C::A_TILE, f = smem_u32(sf_smem + s * C::SF);
        const uint32_t sfa = tmem_base + PN + s * SF_COLS, sfb = sfa + 4 * TERMS;
#pragma unroll
        for (int i = 0; i < TERMS + 2; ++i) sf_to_tmem(go, sfa + 4 * i, f + SF_BYTES * i);
#pragma unroll
        for (int i = 0; i < TERMS; ++i)
#pragma unroll
          for (int k4 = 0; k4 < BK / UK; ++k4)
            umma_mx(go, tmem_base, make_smem_desc_sw128(a + i * C::A_TILE + k4 * UK, 16, 1024),
                    make_smem_desc_sw128(b + k4 * UK, 16, 1024), idesc + k4 * ((1u << 4) + (1u << 29)), sfa + 4 * i, sfb,
                    (kb > 0 || i > 0 || k4 > 0) ? 1u : 0u);
        umma_commit_if(go, &empty[s]);
        if (kb == p.kb - 1) umma_commit_if(go, tfull);
        if (++s == C::STAGES) { s = 0; ph ^= 1; }
      }
    }
    if (!ok) {   // products under way end before the CTA gives its memory back
      umma_commit_if(go, tfull);
      const long long t0 = clock64();
      while (clock64() - t0 < LAND_BUDGET_CYCLES / 10) {}
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + half * 128;
    int n = 0;
    for (int t = blockIdx.x; t < ntiles; t += gridDim.x, ++n) {
      ok = mbar_wait_warp(tfull, n & 1, p.err, ERR_WAIT_TMEM_FULL) && *reinterpret_cast<volatile int*>(p.err) == 0;
      ok = __all_sync(0xffffffffu, ok) != 0;
      if (!ok) break;
      tc_fence_after();
      uint32_t r[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(taddr + 32 * c, r[c]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty);
      int mi, ni;
      raster_tile(t, p.mt, p.nt, p.band, mi, ni);
      const int tok0 = mi * PM + quad * 32, col0 = ni * PN + half * 128;
      if (p.bias) {   // one branch for all values: asked for each, it took longer than the stores
#pragma unroll
        for (int c = 0; c < 128; ++c) {
          const int col = col0 + c < p.N ? col0 + c : p.N - 1;
          const float b = p.bias_fp32 ? static_cast<const float*>(p.bias)[col]
                                      : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[col]);
          r[c >> 5][c & 31] = __float_as_uint(__uint_as_float(r[c >> 5][c & 31]) + b);
        }
      }
      // A lane has a token's 128 features; through shared memory four lanes write 64 bytes of a token together, eight tokens an
      // instruction (16 bytes of 32 tokens each: half-filled sectors, 3 % longer for 8192 x 28672 x 4096).
      uint8_t* patch = patches + (warp - 2) * C::PATCH;
      if ((p.ldy & 7) == 0 && col0 + 128 <= p.N) {
        const int width = p.out_fp32 ? 16 : 32;   // features of a patch
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (!p.out_fp32 && (c & 1)) continue;
          uint4* mine = reinterpret_cast<uint4*>(patch + lane * 80);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (p.out_fp32) {
              float v[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(r[c >> 1][(c & 1) * 16 + g * 4 + j]);
              mine[g] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            } else {
              float v[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[c >> 1][g * 8 + j]);
              mine[g] = make_uint4(two_bf16(v[0], v[1]), two_bf16(v[2], v[3]), two_bf16(v[4], v[5]), two_bf16(v[6], v[7]));
            }
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int t = k * 8 + (lane >> 2);
            const uint4 v = *reinterpret_cast<const uint4*>(patch + t * 80 + (lane & 3) * 16);
            if (tok0 + t < p.T) {
              const long long at = static_cast<long long>(tok0 + t) * p.ldy + col0 + c * 16 + (lane & 3) * (width / 4);
              if (p.out_fp32) *reinterpret_cast<uint4*>(static_cast<float*>(p.Y) + at) = v;
              else *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.Y) + at) = v;
            }
          }
          __syncwarp();
        }
      } else if (p.out_fp32) {   // rows on any boundary, the last columns: sixteen features of two tokens per store
        float* rows = reinterpret_cast<float*>(patch);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (col0 + c * 16 >= p.N) break;
#pragma unroll
          for (int j = 0; j < 16; ++j) rows[lane * 17 + j] = __uint_as_float(r[c >> 1][(c & 1) * 16 + j]);
          __syncwarp();
          const int col = col0 + c * 16 + (lane & 15);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int t = 2 * k + (lane >> 4);
            if (tok0 + t < p.T && col < p.N)
              static_cast<float*>(p.Y)[static_cast<long long>(tok0 + t) * p.ldy + col] = rows[t * 17 + (lane & 15)];
          }
          __syncwarp();
        }
      } else {   // in bf16 a token's 128 features at a time: 128 bytes an instruction, from the row's first or second feature as it
                 // starts on an even or odd one (1485 x 34790 x 768: 103 us, 34816 features 70; two bytes a lane 118)
        const int lim = p.N - col0 < 128 ? p.N - col0 : 128;
        for (int step = 0; step < 4 && lim > 0; ++step) {
          if (lane >> 3 == step) {
            uint4* mine = reinterpret_cast<uint4*>(patch + (lane & 7) * 272);
#pragma unroll
            for (int g = 0; g < 16; ++g) {
              float v[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[g >> 2][(g & 3) * 8 + j]);
              mine[g] = make_uint4(two_bf16(v[0], v[1]), two_bf16(v[2], v[3]), two_bf16(v[4], v[5]), two_bf16(v[6], v[7]));
            }
          }
          __syncwarp();
          const int rows = p.T - tok0 - step * 8 < 8 ? p.T - tok0 - step * 8 : 8;
#pragma unroll 2
          for (int k = 0; k < rows; ++k) {
            const long long at = static_cast<long long>(tok0 + step * 8 + k) * p.ldy + col0;
            const int odd = static_cast<int>(at & 1);
            uint16_t* to = static_cast<uint16_t*>(p.Y) + at;
            const uint32_t* row = reinterpret_cast<const uint32_t*>(patch + k * 272);
            if (odd && lane == 0) to[0] = static_cast<uint16_t>(row[0]);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int word = q * 32 + lane, e = 2 * word + odd;
              const uint32_t v = odd ? __funnelshift_r(row[word], row[word + 1], 16) : row[word];
              if (e + 1 < lim) *reinterpret_cast<uint32_t*>(to + e) = v;
              else if (e < lim) to[e] = static_cast<uint16_t>(v);
            }
          }
          __syncwarp();
        }
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  const bool failed = __syncthreads_or(!ok);
  if (failed && warp == 0) {
    for (int kb = loaded > C::STAGES ? loaded - C::STAGES : 0; kb < loaded; ++kb)
      mbar_land(&full[kb % C::STAGES], static_cast<uint32_t>(kb / C::STAGES) & 1);
  }
  if (warp == 2) { tc_fence_after(); tmem_dealloc(tmem_base, 512); }
}


}  // namespace gq4

// codes [N, K / 2], tiles [ceil(N / 128), K / 128, 512], out [rows, K] bf16, zero from row N on; N <= rows, both in the same last
// tile; K a multiple of 128, 16-byte aligned.
GK_EXPORT int gk_fp4_dequant(const void* codes, const void* tiles, void* out, long long N, long long rows, int K, void* stream) {
  if (N < 0 || rows < N || (rows + 127) / 128 != (N + 127) / 128 || K <= 0 || K % 128) return -1;
  if (((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(out)) & 15)) return -1;
  const long long ctas = (N + 127) / 128 * (K / 128);
  if (ctas == 0) return 0;
  if (ctas > 0x7fffffffll) return -3;
  gq4::fp4_dequant_kernel<<<static_cast<unsigned>(ctas), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint32_t*>(codes), static_cast<const uint8_t*>(tiles), static_cast<uint4*>(out), N, rows, K / 128);
  return gk::launch_status();
}

// src [T, N] to dst [T, Np], zero from column N on; 16-bit values; src 4-byte and dst 16-byte aligned, Np a multiple of 8.
GK_EXPORT int gk_pad_rows16(const void* src, void* dst, long long T, int N, int Np, void* stream) {
  if (T < 0 || N < 1 || Np < N || Np % 8 || (reinterpret_cast<uintptr_t>(src) & 3) || (reinterpret_cast<uintptr_t>(dst) & 15)) return -1;
  const long long units = T * (Np / 8);
  if (units == 0) return 0;
  gq4::pad_rows16_kernel<<<gq4::grid_for(units), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint32_t*>(src), static_cast<uint4*>(dst), units, N, Np / 8, T * N);
  return gk::launch_status();
}

namespace gq4 {

// Codes [rows, K] (K a multiple of 128) as tiles of box_rows x 128 whose rows are spread to 128 bytes.
inline int make_tmap_fp4(CUtensorMap* out, const void* base, uint64_t rows, uint64_t K, uint32_t box_rows) {
  gk::EncodeTiledFn fn = gk::get_encode_fn();
  if (!fn) return -1;
  cuuint64_t dims[2] = {K, rows}, strides[1] = {K / 2};
  cuuint32_t box[2] = {128, box_rows}, estr[2] = {1, 1};
  CUresult r = CUDA_SUCCESS;
  for (int attempt = 0; attempt < 2; ++attempt) {
    r = fn(out, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 2, const_cast<void*>(base), dims, strides, box, estr,
           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_ERROR_INVALID_CONTEXT) break;
    gk::bind_primary_context();
  }
  return r == CUDA_SUCCESS ? 0 : -2;
}

typedef void (*DecodeKernel)(CUtensorMap, CUtensorMap, Fp4Params);

inline DecodeKernel decode_kernel(int src, int T) {
  if (src == SPLIT) return fp4_decode_kernel<SPLIT, 0>;
  if (src == ROWS8) return fp4_decode_kernel<ROWS8, 0>;
  return T <= 2 ? fp4_decode_kernel<ROWS16, 1> : fp4_decode_kernel<ROWS16, 4>;
}

// Allows `kernel` all of an SM's shared memory, once per device; `done` has a bit for each.
template <typename Kernel>
inline int allow_shared(Kernel kernel, unsigned long long& done) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return -13;
  const unsigned long long bit = 1ull << (device & 63);
  if (done & bit) return 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return -13;
  done |= bit;
  return 0;
}

struct Fp4Plan {
  int T, Tc, chunks, Tp, cols, nsf, src, ks, stages, ring, smem;
  float cost;
};

// The decode kernel's plan: tokens per CTA (`Tc`, in whole columns of the product), how many CTAs share a tile's K, how deep the
// ring is.  The cheapest by a model of what was measured (B200, us).  A K block of a lone CTA takes 0.26 (the issuing warp's
// chain) or 0.0085 a KB of operands (60 bytes a cycle, what an SM gets out of L2); two CTAs on an SM share its 0.2 of the memory's
// rate; all together get 9.5 KB a ns out of L2.  A round of CTAs costs 2 and Tc / 50 for each CTA of an SM, a launch 2, the
// exchange in a cluster 2 + Tc / 33 and 1 more for eight CTAs, of which fewer fit into a GPC.  Chosen against the others that were
// run, ks = 1 / 2 / 4 / 8: 1 x 4608 x 3584 12.0 / 9.5 / [9.0] / 9.8, 64 x 4608 x 3584 [14.1] / 14.6 / 21.0 / 26.1, 64 x 3584 x 18944
// 45.7 / 31.8 / [20.6] / 27.6, 16 x 3584 x 18944 - / 25.4 / [16.7] / 15.2 (a second round
// of few CTAs counts as a whole one: 26 by the model), 96 x 28672 x 4096 (e4m3) [23.1] / 67 / 89 / 154; one or two
// CTAs an SM: 1 x 37888 x 3584 22.6 / [16.0], 64 x 4608 x 3584 [14.1] / 16.3.
inline Fp4Plan decode_plan(int T, int Tc, int terms, int N, int kb) {
  Fp4Plan p = {}, best = {};
  p.T = T;
  p.Tc = Tc;
  p.chunks = (T + Tc - 1) / Tc;
  p.Tp = terms == 2 ? (Tc + 7) / 8 * 8 : (Tc + 15) / 16 * 16;
  p.cols = p.Tp * terms;
  p.nsf = (p.cols + 127) / 128;
  p.src = terms == 1 ? ROWS8 : T <= 8 ? ROWS16 : SPLIT;
  const int sms = gk::sm_count();
  const long long tiles = (N + BM - 1ll) / BM * p.chunks;
  if (tiles * 8 > 0x3fffffff || p.chunks > 65535) return best;
  const int tile_bytes = A_BYTES + p.cols * BK, sf = SF_BYTES * (1 + p.nsf), stage = tile_bytes + sf;
  const float kbytes = 8.7f + 0.128f * p.cols;
  for (p.ks = 1; p.ks <= 8 && p.ks <= kb; p.ks *= 2) {
    const int share = (kb + p.ks - 1) / p.ks, red = p.ks > 1 ? p.ks * ((Tc + p.ks - 1) / p.ks) * BM * 4 : 0;
    const int fixed = 1024 + red + (2 * MAX_STAGES + 3) * 8;
    for (int resident = 1; resident <= 2; ++resident) {
      p.stages = (228 * 1024 / resident - 1024 - fixed) / stage;
      if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
      if (p.stages > share) p.stages = share;
      if (p.stages < 1 || (p.stages < 3 && p.stages < share)) continue;
      int tmem = 32;
      while (tmem < (p.cols + 31) / 32 * 32 + p.stages * 4 * (1 + p.nsf)) tmem *= 2;
      p.ring = p.stages * tile_bytes > red ? p.stages * tile_bytes : (red + 1023) / 1024 * 1024;
      p.smem = p.ring + p.stages * sf + fixed;
      // As much of an SM's shared memory as of its tensor memory (512 columns): CTAs that fit side by side, of one launch or of
      // several streams', all get their columns.  One that waited for columns while its cluster waited for it could stop both.
      if (p.smem < tmem * 456 - 1024) p.smem = tmem * 456 - 1024;
      if (p.smem > 228 * 1024 / resident - 1024) continue;
      const int n = static_cast<int>(tiles) * p.ks, slots = sms * resident * (p.ks == 8 ? 7 : p.ks == 4 ? 9 : 10) / 10;
      const int rounds = (n + slots - 1) / slots, each = n > slots ? resident : (n + sms - 1) / sms;
      float one = (0.0085f * kbytes > 0.2f ? 0.0085f * kbytes : 0.2f) * each;
      if (one < 0.26f) one = 0.26f;
      float loop = rounds * (2.f + 0.02f * Tc * each + share * one);
      const float l2 = static_cast<float>(tiles) * kb * kbytes / 9500.f;
      if (loop < l2) loop = l2;
      p.cost = loop + 2.f + (p.ks > 1 ? 2.f + 0.03f * Tc + (p.ks == 8 ? 1.f : 0.f) : 0.f);
      if (best.ks == 0 || p.cost < best.cost) best = p;
    }
  }
  return best;
}

// Which kernel, and its plan: ks = 0 for the prompt kernel.  Its tiles of 128 x 256 leave SMs without work where there are few of
// them, and nothing divides a long K: there the decode kernel runs on chunks of the tokens.  A K block of a prompt tile takes
// 0.45 us (0.72 of two terms), a tile 1.5 more, a launch 4.  us, prompt kernel / chunks of 128 / 64 / 32: 150 x 410 x 18912 of e4m3
// 66 / 19.4 / [14.5] / 14.0, 936 x 417 x 1664 21.5 / 14.1 / 11.8 / [10.9], 512 x 4608 x 3584 of e4m3 17.8 / [16.6] / 17.6 / 27.4, 2048 x 1536 x
// 1536 of e4m3 [11.7] / 13.8 / 18.4 / 25.0, 1024 x 3584 x 3584 [31.4] / 37.0 / 36.1 / 50.9.
inline Fp4Plan plan_for(int T, int terms, int N, int kb) {
  Fp4Plan best = {};
  float cost = 0.f;
  if (T > 128) {
    const long long tiles = (T + 127ll) / 128 * ((N + 255ll) / 256), sms = gk::sm_count();
    cost = 4.f + (tiles + sms - 1) / sms * (1.5f + kb * (terms == 1 ? 0.45f : 0.72f));
    best.cost = cost;
  }
  for (int Tc = T < 128 ? T : 128; Tc >= 32 || Tc == T; Tc = Tc > 64 ? 64 : Tc > 32 ? 32 : 0) {
    const Fp4Plan p = decode_plan(T, Tc, terms, N, kb);
    if (p.ks > 0 && (cost == 0.f || p.cost < cost)) {
      best = p;
      cost = p.cost;
    }
  }
  return best;
}

inline int decode_launch(const void* codes, const void* xq, long long xq_rows, int xq_cols, const Fp4Plan& pl, Fp4Params& p,
                         cudaStream_t st) {
  CUtensorMap tmW, tmX;
  if (make_tmap_fp4(&tmW, codes, p.N, static_cast<uint64_t>(p.kb) * BK, BM)) return -11;
  if (pl.src == ROWS16) tmX = tmW;   // not used
  else if (gk::make_tmap_2d(&tmX, xq, 1, xq_rows, xq_cols, xq_cols, pl.cols, BK, true)) return -12;
  p.total = pl.T; p.Tc = pl.Tc; p.Tp = pl.Tp; p.ks = pl.ks; p.stages = pl.stages; p.cols = pl.cols; p.ring = pl.ring;
  cudaLaunchConfig_t cfg = {};
  const DecodeKernel kernel = decode_kernel(pl.src, pl.T);
  static unsigned long long done[3][2];
  if (int rc = allow_shared(kernel, done[pl.src][pl.T <= 2])) return rc;
  cfg.gridDim = dim3((p.N + BM - 1) / BM * pl.ks, pl.chunks, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = pl.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = pl.ks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  // Set up while the kernel in front drains.  What that kernel may have written is read behind the wait; the weight only where it
  // cannot have: behind the split of the same call, in a decode chain.
  attr[1].val.programmaticStreamSerializationAllowed = gk::overlap_flag();
  p.early = pl.src == SPLIT || gk::pdl_flag();
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return gk::launch_ex(cfg, kernel, tmW, tmX, p);
}

}  // namespace gq4

namespace gq4 {
template <int TERMS>
inline int prompt_launch(const void* codes, const void* xq, long long xq_rows, int xq_cols, const PromptParams& p, int Kp,
                         cudaStream_t st) {
  using C = PromptCfg<TERMS>;
  CUtensorMap tmW, tmX;
  if (make_tmap_fp4(&tmW, codes, p.N, Kp, PN)) return -11;
  if (gk::make_tmap_2d(&tmX, xq, 1, xq_rows, xq_cols, xq_cols, PM, BK, true)) return -12;
  static unsigned long long done = 0;
  if (int rc = allow_shared(fp4_prompt_kernel<TERMS>, done)) return rc;
  const long long tiles = static_cast<long long>(p.mt) * p.nt;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles < gk::sm_count() ? tiles : gk::sm_count()), 1, 1);
  cfg.blockDim = dim3(P_THREADS, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = gk::overlap_flag();   // behind the kernel of the same call that prepares the tokens
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return gk::launch_ex(cfg, fp4_prompt_kernel<TERMS>, tmW, tmX, p);
}
}  // namespace gq4

// Bytes of scratch (16-byte aligned) that gk_fp4_product wants; 0: none.
GK_EXPORT long long gk_fp4_product_scratch(int T, int terms, int N, int Kp) {
  const gq4::Fp4Plan pl = gq4::plan_for(T, terms, N, Kp / 128);
  const long long kb = Kp / 128;
  if (pl.ks > 0) return pl.src == gq4::SPLIT ? pl.chunks * (static_cast<long long>(pl.cols) * Kp + kb * pl.nsf * 512) : 0;
  const long long rows = (T + 127) / 128 * 128ll * terms;
  return (terms == 2 ? rows * Kp : 0) + rows / 128 * kb * 512;
}

// y [T, N] (bf16 or fp32, row stride ldy) of activations and a weight: codes [N, Kp / 2] on a 32-byte boundary, tiles of its
// exponents.  x: bf16 [T, K] (terms 2) or e4m3 [T, K] with exponents xs [T, K / 32] (terms 1), rows packed, 16-byte aligned as
// is Y (xs 4-byte); K a multiple of 32, Kp of 128 and less than 128 above it.
GK_EXPORT int gk_fp4_product(const void* codes, const void* tiles, const void* x, const void* xs, void* scratch, void* Y,
                             long long ldy, int out_fp32, const void* bias, int bias_fp32, int T, int terms, int N, int K, int Kp,
                             int* err, void* stream) {
  using namespace gq4;
  if ((terms != 1 && terms != 2) || T < 1 || N < 1 || K < 32 || K % 32 || Kp % 128 || Kp < K || Kp - K >= 128) return -1;
  if ((reinterpret_cast<uintptr_t>(codes) & 31) || (reinterpret_cast<uintptr_t>(xs) & 3) ||
      ((reinterpret_cast<uintptr_t>(tiles) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(scratch) |
        reinterpret_cast<uintptr_t>(Y)) & 15))
    return -2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int kb = Kp / 128;
  const Fp4Plan pl = plan_for(T, terms, N, kb);
  uint8_t* ws = static_cast<uint8_t*>(scratch);
  const unsigned split_grid = grid_for(static_cast<long long>(T) * (Kp / 8));
  if (pl.ks > 0) {
    Fp4Params p = {};
    p.terms = terms; p.N = N; p.kb = kb; p.K = K;
    p.tiles = static_cast<const uint8_t*>(tiles);
    p.Y = Y; p.ldy = ldy; p.out_fp32 = out_fp32; p.bias = bias; p.bias_fp32 = bias_fp32; p.err = err;
    if (pl.src == ROWS8) {
      p.sf = static_cast<const uint8_t*>(xs);
      return decode_launch(codes, x, T, K, pl, p, st);
    }
    if (pl.src == ROWS16) {
      p.x = x;
      return decode_launch(codes, nullptr, 0, 0, pl, p, st);
    }
    if (!ws) return -2;
    const long long rows = static_cast<long long>(pl.chunks) * pl.cols;
    uint8_t* sf = ws + rows * Kp;
    p.sf = sf;
    const SplitLayout lay = {T, pl.Tc, pl.Tp, K, Kp, kb * pl.nsf, pl.nsf, 1};
    if (int rc = gk::launch_waiting(fp4_split_kernel, split_grid, 256, st, static_cast<const uint4*>(x),
                                    reinterpret_cast<uint2*>(ws), sf, lay))
      return rc;
    return decode_launch(codes, ws, rows, Kp, pl, p, st);
  }
  if (!ws) return -2;
  const int mt = (T + PM - 1) / PM, nt = (N + PN - 1) / PN;
  if (static_cast<long long>(mt) * nt > 0x7fffffffll) return -3;
  PromptParams p = {};
  p.T = T; p.N = N; p.kb = kb; p.mt = mt; p.nt = nt; p.band = gk::raster_group_m();
  p.tiles = static_cast<const uint8_t*>(tiles);
  p.Y = Y; p.ldy = ldy; p.out_fp32 = out_fp32; p.bias = bias; p.bias_fp32 = bias_fp32; p.err = err;
  if (terms == 1) {
    p.sf = ws;
    if (int rc = gk::launch_waiting(fp4_tiles_kernel, grid_for(static_cast<long long>(T) * kb), 256, st,
                                    static_cast<const uint8_t*>(xs), ws, T, K / 32, kb))
      return rc;
    return prompt_launch<1>(codes, x, T, K, p, Kp, st);
  }
  const int rows = mt * PM;
  uint8_t* sf = ws + 2ll * rows * Kp;
  p.sf = sf;
  p.lo_rows = rows;
  const SplitLayout lay = {T, rows, rows, K, Kp, 0, 1, kb};
  if (int rc = gk::launch_waiting(fp4_split_kernel, split_grid, 256, st, static_cast<const uint4*>(x), reinterpret_cast<uint2*>(ws),
                                  sf, lay))
    return rc;
  return prompt_launch<2>(codes, ws, 2ll * rows, Kp, p, Kp, st);
}
