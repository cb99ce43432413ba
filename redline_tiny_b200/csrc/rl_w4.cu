// Products of a few rows with 4-bit weights: C[m][n] = sum_k x[m][k] (u[n][k] - 8) s[n][k / G] (+ bias), m <= 64.
//
// Bound by the weight bytes (K N / 2) on paper at one row; the kernels stay above that floor with no unit saturated (ALU pipe
// 44 %, issue 50 %): streams are short, and every CTA pays a start and a join for 16 columns. One row, weights from HBM / left
// in the L2 by the call before: 50 MB of codes (4096 x 24576) 14.5 / 13.5 - 14.3 us = 3.7 TB/s, 12.6 MB (4096 x 6144)
// 5.3 / 4.7 - 5.0 us, of which a launch and one load are 4. The weights are the A operand of
// mma.m16n8k16 (16 columns of B on the M side, up to 8 rows of x per n-tile), turned from 4 bits to bf16 in registers,
// exactly (nibbles_lo). A group's products are summed by the tensor core in fp32 and scaled once as they are added to the
// fp32 result, so the only rounding is the output's (and fp32's). Rejected for one row: two column tiles a warp (17.4 us),
// 2 - 4 warps a CTA (16.8 - 18.4), CTAs that go on to further columns (15.2), deeper rings (no change).
//
// Native layout, 0.5 byte a weight: tiles of 16 columns x 128 k, 1 KB, K running fastest. Lane 4g + c owns 16 bytes for
// column g (first 512 bytes) and 16 for column g + 8; word q of them holds k = 32q + 8c .. + 7, nibble i the k 2i and
// nibble i + 4 the k 2i + 1. A 32-deep group is then one word per lane, and a word's x values are 16 contiguous bytes.
// Scales: [tile][group][8] pairs (s_g, s_{g + 8}) in bf16. For an up matrix (swiglu) the first 8 columns of a tile are
// gate units and the last 8 the same units' projections, so one lane holds both.
#include "rl_common.cuh"
#include "rl_host.h"

namespace rl {
namespace w4 {

constexpr int TN = 16;          // columns per tile
constexpr int TK = 128;         // k per tile
constexpr int TILE = TN * TK / 2;
constexpr int kMaxRows = 64;

__host__ __device__ inline int64_t tiles_n(int64_t N) { return (N + TN - 1) / TN; }
__host__ __device__ inline int64_t tiles_k(int64_t K) { return (K + TK - 1) / TK; }

// The column of B that row `r` of native tile `t` holds (N or more: padding).
__host__ __device__ inline int64_t column_of(int64_t t, int r, int swiglu) {
  if (!swiglu) return t * TN + r;
  const int64_t unit = t * 8 + (r & 7);
  return unit / 64 * 128 + unit % 64 + (r >= 8 ? 64 : 0);
}

// One thread per 32-bit word of the native codes; padding holds u = 8 (a zero weight).
__global__ void __launch_bounds__(256) pack_kernel(const uint8_t* codes, int64_t K, int64_t N, int swiglu, uint32_t* out,
                                                   int64_t words) {
  const int64_t kt = tiles_k(K);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < words;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t tile = i / (TILE / 4);
    const int at = static_cast<int>(i % (TILE / 4));
    const int q = at & 3, lane = at >> 2 & 31, half = at >> 7;
    const int64_t col = column_of(tile / kt, (lane >> 2) + 8 * half, swiglu);
    const int64_t k0 = tile % kt * TK + 32 * q + 8 * (lane & 3);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t u = col < N && k0 + j < K ? codes[(k0 + j) * N + col] & 15u : 8u;
      w |= u << (4 * (j >> 1) + 16 * (j & 1));
    }
    out[i] = w;
  }
}

__global__ void __launch_bounds__(256) pack_scales_kernel(const uint16_t* scales, int64_t groups, int64_t pad_groups,
                                                          int64_t N, int swiglu, uint32_t* out, int64_t count) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < count;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int g = static_cast<int>(i & 7);
    const int64_t gr = i / 8 % pad_groups, t = i / 8 / pad_groups;
    const int64_t c0 = column_of(t, g, swiglu), c1 = column_of(t, g + 8, swiglu);
    const uint32_t lo = gr < groups && c0 < N ? scales[gr * N + c0] : 0u;
    const uint32_t hi = gr < groups && c1 < N ? scales[gr * N + c1] : 0u;
    out[i] = lo | (hi << 16);
  }
}

// Round a float B (K, N) to 4 bits: per group and column s = bf16(e / -8), e the value of largest magnitude (the
// first, among equals), u = clip(rint(w / s) + 8, 0, 15). A signed s lets the extreme use the code -8, so the step is
// 1/8 of the extreme and not 1/7. A group with a NaN or an infinity takes a NaN scale; an all-zero group takes zero.
template <typename X>
__global__ void __launch_bounds__(256) quantize_kernel(const X* B, int64_t K, int64_t N, int G, uint8_t* codes,
                                                       uint16_t* scales) {
  const int64_t n = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (n >= N) return;
  for (int64_t gr = blockIdx.y; gr < K / G; gr += gridDim.y) {
    float ext = 0.0f;
    bool bad = false;
    for (int j = 0; j < G; ++j) {
      const X raw = B[(gr * G + j) * N + n];
      const float w = sizeof(X) == 2 ? bf16_bits_to_float(static_cast<uint32_t>(raw)) : static_cast<float>(raw);
      bad |= !(fabsf(w) <= 3.4028235e38f);
      if (fabsf(w) > fabsf(ext)) ext = w;
    }
    const __nv_bfloat16 sb = __float2bfloat16_rn(bad ? __uint_as_float(0x7FC00000u) : ext * -0.125f);
    const float s = __bfloat162float(sb);
    scales[gr * N + n] = __bfloat16_as_ushort(sb);
    for (int j = 0; j < G; ++j) {
      const X raw = B[(gr * G + j) * N + n];
      const float w = sizeof(X) == 2 ? bf16_bits_to_float(static_cast<uint32_t>(raw)) : static_cast<float>(raw);
      const float m = s == 0.0f || bad ? 0.0f : fminf(fmaxf(rintf(__fdiv_rn(w, s)), -8.0f), 7.0f);
      codes[(gr * G + j) * N + n] = static_cast<uint8_t>(static_cast<int>(m) + 8);
    }
  }
}

struct Args {
  const uint16_t* x;
  const uint4* w;
  const uint32_t* s;
  const uint16_t* bias;
  void* out;
  int64_t K, N;
  int M, out_f32;
};

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// Nibbles 0 and 4 (lo) or 1 and 5 (hi) of a word as bf16 values (u - 8) / 64. Taken as bf16 bits, a field in the low 8
// bits is that integer times 2^-133 (subnormal, or the first binade, whose spacing is the same), so one FMA scales it and
// takes the offset off, exactly. Three ALU instructions less per word than shifting every nibble to the same place and
// setting an exponent beside it (the ALU pipe runs at half rate and was the busiest: 16.3 -> 13.3 us for 50 MB of codes).
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t nibbles_lo(uint32_t w) { return fma_bf16x2(w & 0x000F000Fu, 0x7F007F00u, 0xBE00BE00u); }
__device__ __forceinline__ uint32_t nibbles_hi(uint32_t w) { return fma_bf16x2(w & 0x00F000F0u, 0x7D007D00u, 0xBE00BE00u); }
constexpr float kUnit = 64.0f;   // what the sums are short of

// A k tile's operands on their way: the lane's codes of columns g and g + 8 and the groups' scales.
template <int G>
struct Tile {
  uint4 w0, w1;
  uint32_t s[TK / G];
};
template <int G>
__device__ __forceinline__ void load_tile(Tile<G>& t, const uint4* w, const uint32_t* sc) {
  t.w0 = __ldcs(w), t.w1 = __ldcs(w + 32);
#pragma unroll
  for (int j = 0; j < TK / G; ++j) t.s[j] = __ldcs(sc + j * 8);
}

// acc += the products of CT tiles with the same x fragments: x(q, nt) gives the 16 bytes of word q for row nt * 8 + g.
template <int CT, int NT, int G, typename X>
__device__ __forceinline__ void tile_product(const Tile<G> (&t)[CT], X x, float (&acc)[CT][NT][4]) {
  float part[CT][NT][4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 xv[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) xv[nt] = x(q, nt);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const uint32_t v0 = q == 0 ? t[ct].w0.x : q == 1 ? t[ct].w0.y : q == 2 ? t[ct].w0.z : t[ct].w0.w;
      const uint32_t v1 = q == 0 ? t[ct].w1.x : q == 1 ? t[ct].w1.y : q == 2 ? t[ct].w1.z : t[ct].w1.w;
      const uint32_t h0 = v0 >> 8, h1 = v1 >> 8;
      const uint32_t A[8] = {nibbles_lo(v0), nibbles_lo(v1), nibbles_hi(v0), nibbles_hi(v1),
                             nibbles_lo(h0), nibbles_lo(h1), nibbles_hi(h0), nibbles_hi(h1)};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (q % (G / 32) == 0) mma_zero(part[ct][nt], A[0], A[1], A[2], A[3], xv[nt].x, xv[nt].y);
        else mma(part[ct][nt], A[0], A[1], A[2], A[3], xv[nt].x, xv[nt].y);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma(part[ct][nt], A[4], A[5], A[6], A[7], xv[nt].z, xv[nt].w);
      if (q % (G / 32) == G / 32 - 1) {
        const uint32_t s = t[ct].s[q / (G / 32)];
        const float s0 = __uint_as_float(s << 16), s1 = __uint_as_float(s & 0xFFFF0000u);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          acc[ct][nt][0] = fmaf(s0, part[ct][nt][0], acc[ct][nt][0]);
          acc[ct][nt][1] = fmaf(s0, part[ct][nt][1], acc[ct][nt][1]);
          acc[ct][nt][2] = fmaf(s1, part[ct][nt][2], acc[ct][nt][2]);
          acc[ct][nt][3] = fmaf(s1, part[ct][nt][3], acc[ct][nt][3]);
        }
      }
    }
  }
}

// Bias, activation and store of one output: v (and for SwiGLU the unit's projection) of row m, tile row r of tile t.
template <bool kSwiglu>
__device__ __forceinline__ void finish(const Args& a, int m, int64_t t, int r, float v, float up) {
  const int64_t col = column_of(t, r, kSwiglu);
  if (col >= a.N) return;
  int64_t at = m * a.N + col;
  if (a.bias) v += bf16_bits_to_float(a.bias[col]);
  if (kSwiglu) {
    if (a.bias) up += bf16_bits_to_float(a.bias[col + 64]);
    v = v / (1.0f + __expf(-v)) * up;
    at = m * (a.N / 2) + t * 8 + r;
  }
  if (a.out_f32) static_cast<float*>(a.out)[at] = v;
  else static_cast<uint16_t*>(a.out)[at] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// Up to 8 rows: one CTA per 16 columns; its warps take the k tiles in turn, each with kDepth tiles on their way, and
// are joined in shared memory in warp order. x comes straight from L1 and L2: it is small next to the weights. Lanes of
// rows beyond M read the last row: a column of the B operand reaches its own column of the result only.
constexpr int kFew = 8, kDepth = 2;
template <int G, bool kSwiglu>
__global__ void __launch_bounds__(32 * kFew, 4) few_kernel(const Args a) {
  __shared__ float red[kFew][8][TN + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int K = static_cast<int>(a.K), kt = static_cast<int>(tiles_k(a.K));
  constexpr int kSc = TK / G * 8;                                 // scale words of a tile
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kt + warp;
  const uint4* w = a.w + at * (TILE / 16) + lane;
  const uint32_t* sc = a.s + at * kSc + g;
  const uint16_t* x = a.x + static_cast<int64_t>(min(g, a.M - 1)) * K + warp * TK + 8 * c;
  const int n = kt > warp ? (kt - warp + kFew - 1) / kFew : 0;    // this warp's tiles
  const int tail = K % TK != 0 && (kt - 1) % kFew == warp ? n - 1 : n;   // the one whose k ends inside it
  float acc[1][1][4] = {{{0.0f, 0.0f, 0.0f, 0.0f}}};
  Tile<G> ring[kDepth][1];
#pragma unroll
  for (int j = 0; j < kDepth; ++j)
    if (j < n) load_tile<G>(ring[j][0], w + j * kFew * (TILE / 16), sc + j * kFew * kSc);
  for (int t0 = 0; t0 < n; t0 += kDepth) {
#pragma unroll
    for (int j = 0; j < kDepth; ++j) {
      if (t0 + j < n) {
        uint4 xv[4];
        if (t0 + j != tail) {
#pragma unroll
          for (int q = 0; q < 4; ++q) xv[q] = __ldg(reinterpret_cast<const uint4*>(x + j * kFew * TK + 32 * q));
        } else {
          const int left = K % TK - 8 * c;                        // k left of this lane's first
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            xv[q] = make_uint4(0, 0, 0, 0);
            if (32 * q < left) xv[q] = __ldg(reinterpret_cast<const uint4*>(x + j * kFew * TK + 32 * q));
          }
        }
        tile_product<1, 1, G>(ring[j], [&](int q, int) { return xv[q]; }, acc);
        if (t0 + j + kDepth < n)
          load_tile<G>(ring[j][0], w + (j + kDepth) * kFew * (TILE / 16), sc + (j + kDepth) * kFew * kSc);
      }
    }
    x += kDepth * kFew * TK, w += kDepth * kFew * (TILE / 16), sc += kDepth * kFew * kSc;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[warp][2 * c + (i & 1)][g + 8 * (i >> 1)] = acc[0][0][i] * kUnit;
  __syncthreads();
  constexpr int kOut = kSwiglu ? 8 : TN;
  for (int i = threadIdx.x; i < a.M * kOut; i += 32 * kFew) {
    const int m = i / kOut, r = i % kOut;
    float v = 0.0f, up = 0.0f;
#pragma unroll
    for (int k = 0; k < kFew; ++k) {
      v += red[k][m][r];
      if (kSwiglu) up += red[k][m][r + 8];
    }
    finish<kSwiglu>(a, m, blockIdx.x, r, v, up);
  }
}

// 9 to 64 rows: one CTA per 128 columns and share of K, a warp per CT x 16 columns; the x of a share is brought into
// shared memory once (with one warp per 16 columns reading x itself, x is M / 8 times the weights' bytes of L2 traffic)
// and each fragment serves CT tiles of codes. The CTAs of a cluster hold the shares of K of the same columns and are
// joined through distributed shared memory in rank order. 23 rows, 12288 x 4096: 14.3 - 14.8 us, weights cold or not.
// mma.sync issues one m16n8k16 in two cycles an SM (1024 products a cycle): 24 of them a tile and 192 tiles on the fullest SMs
// are 5 us, start, joins and clusters that leave SMs empty the rest. 16 / 32 / 48 / 64 rows (groups of 64, weights cold):
// 4096 x 24576 20.7 / 35.7 / 53.1 / 66.8 us, 12288 x 4096 13.4 / 16.5 / 23.9 / 28.8, 4096 x 6144 8.8 / 13.9 / 17.8 / 22.3. The
// packed bfp16 GEMM takes 65, 28 and 22 us there at any of these row counts: at 64 rows the two meet. Rejected: K split over
// warps as well (17 - 19 us).
template <int NT>
struct Many {
  static constexpr int CT = NT <= 3 ? 2 : 1;
  static constexpr int kCols = 128, kWarps = kCols / (CT * TN), kThreads = 32 * kWarps;
  static constexpr int kRows = 8 * NT;
  static constexpr int kX = kRows * TK * 2;                       // bytes of x per k tile
  static constexpr int kCtas = NT <= 3 ? 3 : NT <= 4 ? 2 : 1;  // resident per SM
  static constexpr int kDepth = 2;                                // k tiles of codes on their way
  static constexpr int kPanel = 221184 / kCtas / kX / kDepth * kDepth;   // k tiles of x in shared memory at a time
  static constexpr int kOut = kRows * (kCols + 4) * 4;            // this CTA's sums [row][column], padded
  static constexpr int kSmem = kPanel * kX > kOut ? kPanel * kX : kOut;
};

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

template <int NT, int G, bool kSwiglu>
__global__ void __launch_bounds__(Many<NT>::kThreads, Many<NT>::kCtas) many_kernel(const Args a, int shares, int log_shares) {
  using C = Many<NT>;
  constexpr int D = C::kDepth, CT = C::CT;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int K = static_cast<int>(a.K), kt = static_cast<int>(tiles_k(a.K));
  const int rank = blockIdx.x & (shares - 1);
  const int64_t tile0 = static_cast<int64_t>(blockIdx.x >> log_shares) * (C::kCols / TN), tiles = tiles_n(a.N);
  const int t_begin = (kt * rank) >> log_shares, t_end = (kt * (rank + 1)) >> log_shares;
  constexpr int kSc = TK / G * 8;                                 // scale words of a tile
  const uint4* w[CT];
  const uint32_t* sc[CT];
  Tile<G> ring[D][CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {                               // (a tile beyond the last is the last again, unused)
    const int64_t at = min(tile0 + warp * CT + ct, tiles - 1) * kt + t_begin;
    w[ct] = a.w + at * (TILE / 16) + lane;
    sc[ct] = a.s + at * kSc + g;
#pragma unroll
    for (int j = 0; j < D; ++j)
      if (t_begin + j < t_end) load_tile<G>(ring[j][ct], w[ct] + j * (TILE / 16), sc[ct] + j * kSc);
  }
  // Row m of a k tile keeps its 16-byte chunk j at chunk j ^ 4 (m & 1): the eight lanes of a phase (two rows, four
  // chunks) then read eight different bank groups. A thread copies chunk tid % 16 of rows tid / 16, + kStep, ..; rows
  // beyond M repeat the last (their results are not stored), k beyond K are zeros.
  constexpr int kStep = C::kThreads / 16, kCopies = (C::kRows + kStep - 1) / kStep;
  static_assert(kStep % 2 == 0, "rows of x per pass");
  const int xm = threadIdx.x >> 4, xj = threadIdx.x & 15;
  const uint32_t xdst = smem_u32(smem) + xm * (TK * 2) + ((xj ^ ((xm & 1) * 4)) << 4);
  const uint16_t* xsrc[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i)
    xsrc[i] = a.x + static_cast<int64_t>(min(xm + kStep * i, a.M - 1)) * K + t_begin * TK + 8 * xj;
  float acc[CT][NT][4];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[ct][nt][0] = acc[ct][nt][1] = acc[ct][nt][2] = acc[ct][nt][3] = 0.0f;
  const uint8_t* xa = smem + g * (TK * 2);
  const uint32_t xc = (c ^ ((g & 1) * 4)) << 4;
  // (few k tiles a share are one panel; 64 rows of 4096 x 24576 take three)
  for (int p0 = t_begin; p0 < t_end; p0 += C::kPanel) {
    const int p1 = min(p0 + C::kPanel, t_end);
    if (p0 > t_begin) __syncthreads();                            // every warp is done with the panel before
    for (int t = p0; t < p1; ++t) {
      const bool in = t * TK + 8 * xj < K;
      const uint32_t dst = xdst + (t - p0) * C::kX;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        if (xm + kStep * i >= C::kRows) break;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i * kStep * (TK * 2)),
                     "l"(in ? xsrc[i] : a.x), "r"(in ? 16 : 0)
                     : "memory");
        xsrc[i] += TK;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    for (int t0 = p0; t0 < p1; t0 += D) {
#pragma unroll
      for (int j = 0; j < D; ++j) {
        const int t = t0 + j;
        if (t < p1) {
          const uint8_t* at = xa + (t - p0) * C::kX;
          tile_product<CT, NT, G>(ring[j], [&](int q, int nt) {
            return *reinterpret_cast<const uint4*>(at + nt * 8 * (TK * 2) + (xc ^ (q << 6)));
          }, acc);
          if (t + D < t_end) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
              load_tile<G>(ring[j][ct], w[ct] + (j + D) * (TILE / 16), sc[ct] + (j + D) * kSc);
          }
        }
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) w[ct] += D * (TILE / 16), sc[ct] += D * kSc;
    }
  }
  __syncthreads();                                                // the panel becomes the sums
  float* sums = reinterpret_cast<float*>(smem);
  constexpr int kLd = C::kCols + 4;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sums[(nt * 8 + 2 * c + (i & 1)) * kLd + (warp * CT + ct) * TN + g + 8 * (i >> 1)] = acc[ct][nt][i] * kUnit;
  if (shares > 1) cluster_sync(); else __syncthreads();
  // this CTA finishes every shares-th (row, column) of the cluster's 128 columns
  constexpr int kOut = kSwiglu ? C::kCols / 2 : C::kCols;
  for (int i = threadIdx.x + rank * C::kThreads; i < a.M * kOut; i += C::kThreads << log_shares) {
    const int m = i / kOut, n = i % kOut;
    const int t = kSwiglu ? n >> 3 : n >> 4, r = kSwiglu ? n & 7 : n & 15;
    const float* at = sums + m * kLd + t * TN + r;
    float v = 0.0f, up = 0.0f;
#pragma unroll 8
    for (int k = 0; k < shares; ++k) {
      const uint32_t remote = mapa_shared(smem_u32(at), k);
      v += ld_cluster(remote);
      if (kSwiglu) up += ld_cluster(remote + 32);
    }
    if (tile0 + t < tiles) finish<kSwiglu>(a, m, tile0 + t, r, v, up);
  }
  if (shares > 1) cluster_sync();                                 // no CTA leaves while its sums are read
}

template <int NT, int G, bool kSwiglu>
inline int launch_many(const Args& a, cudaStream_t s) {
  auto kern = many_kernel<NT, G, kSwiglu>;
  static PerDevice ready;
  RL_TRY_CUDA(ready.once([=] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Many<NT>::kSmem); }));
  // shares of K: as many as keep the grid within the GPU's resident CTAs and leave each at least two k tiles
  const int64_t groups = (a.N + Many<NT>::kCols - 1) / Many<NT>::kCols, kt = tiles_k(a.K);
  const int64_t slots = static_cast<int64_t>(sm_count()) * Many<NT>::kCtas;
  int log_shares = 0;
  while (log_shares < 3 && (groups << (log_shares + 1)) <= slots && kt >= (4 << log_shares)) ++log_shares;
  const int shares = 1 << log_shares;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(groups * shares));
  cfg.blockDim = dim3(Many<NT>::kThreads);
  cfg.dynamicSmemBytes = Many<NT>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = shares;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  RL_TRY_CUDA(cudaLaunchKernelEx(&cfg, kern, a, shares, log_shares));
  return RL_OK;
}

template <int G, bool kSwiglu>
inline int launch(const Args& a, cudaStream_t s) {
  if (a.M <= 8) {
    few_kernel<G, kSwiglu><<<static_cast<unsigned>(tiles_n(a.N)), 32 * kFew, 0, s>>>(a);
    RL_TRY_CUDA(cudaGetLastError());
    return RL_OK;
  }
  switch ((a.M + 7) / 8) {
    case 2: return launch_many<2, G, kSwiglu>(a, s);
    case 3: return launch_many<3, G, kSwiglu>(a, s);
    case 4: return launch_many<4, G, kSwiglu>(a, s);
    case 5:
    case 6: return launch_many<6, G, kSwiglu>(a, s);
    default: return launch_many<8, G, kSwiglu>(a, s);
  }
}

inline int check_shape(const char* fn, int64_t K, int64_t N, int group, int swiglu) {
  RL_REQUIRE(group == 32 || group == 64 || group == 128, RL_ERR_ARGUMENT, "%s: groups of %d (32, 64 or 128)", fn, group);
  RL_REQUIRE(K > 0 && K % group == 0 && K <= (1 << 24), RL_ERR_ARGUMENT, "%s: K = %lld must be a multiple of the group",
             fn, (long long)K);
  RL_REQUIRE(N > 0 && N <= (1 << 24) && (!swiglu || N % 128 == 0), RL_ERR_ARGUMENT,
             "%s: N = %lld (an up matrix needs N %% 128 == 0)", fn, (long long)N);
  return RL_OK;
}

}  // namespace w4
}  // namespace rl

extern "C" {

int rl_w4_bytes(int64_t K, int64_t N, int group, int swiglu, size_t* code_bytes, size_t* scale_bytes) {
  using namespace rl;
  int st;
  if ((st = w4::check_shape("rl_w4_bytes", K, N, group, swiglu)) != RL_OK) return st;
  RL_REQUIRE(code_bytes && scale_bytes, RL_ERR_ARGUMENT, "rl_w4_bytes: NULL pointer");
  const size_t tiles = static_cast<size_t>(w4::tiles_n(N)) * w4::tiles_k(K);
  *code_bytes = tiles * w4::TILE;
  *scale_bytes = tiles * (w4::TK / group) * w4::TN * 2;
  return RL_OK;
}

int rl_w4_quantize(const void* B, int dtype, int64_t K, int64_t N, int group, uint8_t* codes, uint16_t* scales,
                   rl_stream_t stream) {
  using namespace rl;
  int st;
  if ((st = w4::check_shape("rl_w4_quantize", K, N, group, 0)) != RL_OK) return st;
  RL_REQUIRE(B && codes && scales, RL_ERR_ARGUMENT, "rl_w4_quantize: NULL pointer");
  RL_REQUIRE(dtype == RL_F32 || dtype == RL_BF16, RL_ERR_ARGUMENT, "rl_w4_quantize: unknown dtype %d", dtype);
  RL_REQUIRE(aligned(B, dtype == RL_F32 ? 4 : 2) && aligned(scales, 2), RL_ERR_ALIGNMENT,
             "rl_w4_quantize: operands must be aligned to their type");
  RL_REQUIRE(device_is_sm100(), RL_ERR_UNSUPPORTED, "rl_w4_quantize: needs an sm_100 device");
  const int64_t gr = K / group;
  const dim3 grid(static_cast<unsigned>((N + 255) / 256), static_cast<unsigned>(gr < 65535 ? gr : 65535));
  if (dtype == RL_F32)
    w4::quantize_kernel<float><<<grid, 256, 0, stream>>>(static_cast<const float*>(B), K, N, group, codes, scales);
  else
    w4::quantize_kernel<uint16_t><<<grid, 256, 0, stream>>>(static_cast<const uint16_t*>(B), K, N, group, codes, scales);
  RL_TRY_CUDA(cudaGetLastError());
  return RL_OK;
}

int rl_w4_pack(const uint8_t* codes, const uint16_t* scales, int64_t K, int64_t N, int group, int swiglu, uint8_t* w_out,
               uint8_t* s_out, rl_stream_t stream) {
  using namespace rl;
  size_t cb = 0, sb = 0;
  const int st = rl_w4_bytes(K, N, group, swiglu, &cb, &sb);
  if (st != RL_OK) return st;
  RL_REQUIRE(codes && scales && w_out && s_out, RL_ERR_ARGUMENT, "rl_w4_pack: NULL pointer");
  RL_REQUIRE(aligned(w_out, 16) && aligned(s_out, 16) && aligned(scales, 2), RL_ERR_ALIGNMENT,
             "rl_w4_pack: outputs must be 16-byte aligned");
  RL_REQUIRE(device_is_sm100(), RL_ERR_UNSUPPORTED, "rl_w4_pack: needs an sm_100 device");
  const int64_t words = static_cast<int64_t>(cb / 4), count = static_cast<int64_t>(sb / 4);
  const int64_t most = static_cast<int64_t>(sm_count()) * 16;
  auto ctas = [&](int64_t n) { return static_cast<unsigned>((n + 255) / 256 < most ? (n + 255) / 256 : most); };
  w4::pack_kernel<<<ctas(words), 256, 0, stream>>>(codes, K, N, swiglu, reinterpret_cast<uint32_t*>(w_out), words);
  RL_TRY_CUDA(cudaGetLastError());
  w4::pack_scales_kernel<<<ctas(count), 256, 0, stream>>>(scales, K / group, w4::tiles_k(K) * (w4::TK / group), N, swiglu,
                                                          reinterpret_cast<uint32_t*>(s_out), count);
  RL_TRY_CUDA(cudaGetLastError());
  return RL_OK;
}

int rl_linear_w4(const uint16_t* x, int64_t M, int64_t K, const uint8_t* w, const uint8_t* scales, int64_t N, int group,
                 const uint16_t* bias, int epilogue, void* out, int out_dtype, rl_stream_t stream) {
  using namespace rl;
  const int swiglu = epilogue == RL_EPI_SWIGLU;
  int st;
  if ((st = w4::check_shape("rl_linear_w4", K, N, group, swiglu)) != RL_OK) return st;
  RL_REQUIRE(M >= 0 && M <= w4::kMaxRows, RL_ERR_ARGUMENT,
             "rl_linear_w4: %lld rows (at most %d; rl_linear_bfp16 takes more)", (long long)M, w4::kMaxRows);
  RL_REQUIRE(epilogue == RL_EPI_NONE || epilogue == RL_EPI_BIAS || epilogue == RL_EPI_SWIGLU, RL_ERR_ARGUMENT,
             "rl_linear_w4: unknown epilogue %d", epilogue);
  RL_REQUIRE(epilogue != RL_EPI_BIAS || bias, RL_ERR_ARGUMENT, "rl_linear_w4: the bias epilogue needs a bias");
  RL_REQUIRE(out_dtype == RL_F32 || out_dtype == RL_BF16, RL_ERR_ARGUMENT, "rl_linear_w4: unknown dtype %d", out_dtype);
  if (M == 0) return RL_OK;
  RL_REQUIRE(x && w && scales && out, RL_ERR_ARGUMENT, "rl_linear_w4: NULL pointer");
  RL_REQUIRE(aligned(x, 16) && aligned(w, 16) && aligned(scales, 16) && aligned(bias, 2) &&
                 aligned(out, out_dtype == RL_F32 ? 4 : 2),
             RL_ERR_ALIGNMENT, "rl_linear_w4: x and the weights must be 16-byte aligned");
  RL_REQUIRE(device_is_sm100(), RL_ERR_UNSUPPORTED, "rl_linear_w4: needs an sm_100 device");
  const w4::Args a{x, reinterpret_cast<const uint4*>(w), reinterpret_cast<const uint32_t*>(scales),
                   epilogue == RL_EPI_NONE ? nullptr : bias, out, K, N, static_cast<int>(M), out_dtype == RL_F32};
  switch (group) {
    case 32: return swiglu ? w4::launch<32, true>(a, stream) : w4::launch<32, false>(a, stream);
    case 64: return swiglu ? w4::launch<64, true>(a, stream) : w4::launch<64, false>(a, stream);
    default: return swiglu ? w4::launch<128, true>(a, stream) : w4::launch<128, false>(a, stream);
  }
}

}  // extern "C"
