// Products of a few rows with 4-bit weights: C[m][n] = sum_k x[m][k] (u[n][k] - 8) s[n][k / G] (+ bias), m < 64.
//
// Bound by the weight bytes (K N / 2) up to about 16 rows. The weights are the A operand of mma.m16n8k16 (16 columns of
// B on the M side, up to 8 rows of x per n-tile), turned from 4 bits to bf16 in registers: the word's nibbles i and
// i + 4 become the halves of one register, (w >> 4i) & 0x000F000F | 0x43004300 = 128 + u, minus 136, exact. A group's
// products are summed by the tensor core in fp32 and scaled once as they are added to the fp32 result, so the only
// rounding is the output's (and fp32's).
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
constexpr int kWarps = 8;

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
// Nibbles i and i + 4 of a word as bf16 integers u - 8.
__device__ __forceinline__ uint32_t nibbles(uint32_t w, int i) {
  const uint32_t b = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(b), "r"(0x43084308u));
  return d;
}

// One CTA per 16 columns: its warps take the k tiles in turn and are joined in shared memory in warp order.
template <int NT, int G, bool kSwiglu>
__global__ void __launch_bounds__(32 * kWarps) linear_kernel(const Args a) {
  __shared__ float red[kWarps][8 * NT][TN + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int64_t kt = tiles_k(a.K);
  const uint4* w = a.w + static_cast<int64_t>(blockIdx.x) * kt * (TILE / 16) + lane;
  const uint32_t* sc = a.s + static_cast<int64_t>(blockIdx.x) * kt * (TK / G) * 8 + g;
  float acc[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.0f;
  for (int64_t t = warp; t < kt; t += kWarps) {
    const uint4 w0 = __ldcs(w + t * (TILE / 16)), w1 = __ldcs(w + t * (TILE / 16) + 32);
    const uint32_t v0[4] = {w0.x, w0.y, w0.z, w0.w}, v1[4] = {w1.x, w1.y, w1.z, w1.w};
    float part[NT][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q % (G / 32) == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) part[nt][0] = part[nt][1] = part[nt][2] = part[nt][3] = 0.0f;
      }
      uint32_t A[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) A[2 * i] = nibbles(v0[q], i), A[2 * i + 1] = nibbles(v1[q], i);
      const int64_t k = t * TK + 32 * q + 8 * c;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int m = nt * 8 + g;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (m < a.M && k < a.K) x = *reinterpret_cast<const uint4*>(a.x + m * a.K + k);
        mma(part[nt], A[0], A[1], A[2], A[3], x.x, x.y);
        mma(part[nt], A[4], A[5], A[6], A[7], x.z, x.w);
      }
      if (q % (G / 32) == G / 32 - 1) {
        const uint32_t s = __ldg(sc + (t * (TK / G) + q / (G / 32)) * 8);
        const float s0 = __uint_as_float(s << 16), s1 = __uint_as_float(s & 0xFFFF0000u);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          acc[nt][0] = fmaf(s0, part[nt][0], acc[nt][0]);
          acc[nt][1] = fmaf(s0, part[nt][1], acc[nt][1]);
          acc[nt][2] = fmaf(s1, part[nt][2], acc[nt][2]);
          acc[nt][3] = fmaf(s1, part[nt][3], acc[nt][3]);
        }
      }
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < 4; ++i) red[warp][nt * 8 + 2 * c + (i & 1)][g + 8 * (i >> 1)] = acc[nt][i];
  }
  __syncthreads();
  constexpr int kOut = kSwiglu ? 8 : TN;
  for (int i = threadIdx.x; i < a.M * kOut; i += 32 * kWarps) {
    const int m = i / kOut, r = i % kOut;
    float v = 0.0f, up = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      v += red[k][m][r];
      if (kSwiglu) up += red[k][m][r + 8];
    }
    const int64_t col = column_of(blockIdx.x, r, kSwiglu);
    if (col >= a.N) continue;
    int64_t at = m * a.N + col;
    if (a.bias) v += bf16_bits_to_float(a.bias[col]);
    if (kSwiglu) {
      if (a.bias) up += bf16_bits_to_float(a.bias[col + 64]);
      v = v / (1.0f + __expf(-v)) * up;
      at = m * (a.N / 2) + static_cast<int64_t>(blockIdx.x) * 8 + r;
    }
    if (a.out_f32) static_cast<float*>(a.out)[at] = v;
    else static_cast<uint16_t*>(a.out)[at] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
  }
}

template <int NT, int G>
inline void launch(const Args& a, bool swiglu, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(tiles_n(a.N));
  if (swiglu) linear_kernel<NT, G, true><<<grid, 32 * kWarps, 0, s>>>(a);
  else linear_kernel<NT, G, false><<<grid, 32 * kWarps, 0, s>>>(a);
}

template <int G>
inline void launch_rows(const Args& a, bool swiglu, cudaStream_t s) {
  if (a.M <= 8) launch<1, G>(a, swiglu, s);
  else if (a.M <= 16) launch<2, G>(a, swiglu, s);
  else if (a.M <= 32) launch<4, G>(a, swiglu, s);
  else launch<8, G>(a, swiglu, s);
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
    case 32: w4::launch_rows<32>(a, swiglu, stream); break;
    case 64: w4::launch_rows<64>(a, swiglu, stream); break;
    default: w4::launch_rows<128>(a, swiglu, stream); break;
  }
  RL_TRY_CUDA(cudaGetLastError());
  return RL_OK;
}

}  // extern "C"
