// Attention of many new tokens per sequence (prompts and their chunks) over the 8-bit paged cache, on tcgen05.
//
// One CTA per 256 rows (two 128-row tiles; rows = new tokens x query heads of one K/V head, token-major) of one
// sequence, over 128-key blocks, with the schedule of the dense two-tile attention kernel (rl_attn.cu): per block and
// tile S_t = Q_t K^T (M128 N128, bf16) into TMEM, softmax of one row per thread, P written back over S_t, and
// O_t += P_t V, the two tiles interleaved so that one's MMAs run under the other's softmax. What differs is the operands:
//
//  * three converter warps read the pages' codes and write the MMA operands into shared memory. K: bf16 (u - 128) / 64,
//    exact (a byte taken as bf16 bits is u 2^-133, so one FMA scales it and takes the offset off); the block's scale
//    2^(ek - 133) is applied to S, 16 columns at a time, where the softmax scales them anyway. V: fp16 (u - 128) 2^(5 + ev - e),
//    exact down to 2^-24, with e the largest V exponent that any row of the tile sees, found before the first block; O is
//    multiplied by 2^(e - 138) at the end. Blocks more than kReach = 29 below e become zeros (they hold less than 2^-29 of
//    the largest value that e admits). That is done only while every row sees a block of e or e - 1; elsewhere a tile with
//    blocks that far down goes by the split kernel's steps (far_tile), whose unit is each row's own, so that no hidden key
//    reaches a row. Both are written [key][64 dims] with the 128-byte swizzle: K-major for S, and for P V the
//    same layout read as MN-major B. The codes wait in the converters' registers for the time of a block (with one item in
//    flight their latency bound the kernel: 791 us for the case below, staged through shared memory 346).
//  * P is fp16 (11 significant bits), V too; the row sum adds P before its rounding. P is kept times 2^kUpP (at most
//    2^(kTau + kUpP) = 2^15), so a weight is off by half a step, 2^-11 of it, down to 2^-21 of the row's largest and by
//    2^-32 of the largest below that: without it weights below 2^-25 were lost whole, 0.4 % of the row in a tail of 131072.
//  * the tile's rows need not be consecutive in memory, so Q is copied by plain loads, all warps taking part.
//
// The chain of a tile bounds it, 4000 cycles per block of both tiles: softmax 2700 (it shares the issue slots and the shared
// memory with the converters), the rest of P V and the next S 1300, about twice their arithmetic, since their operands and
// the converters' stores share the shared memory too (the dense kernel takes 3300). A task adds 5.5 us until its first S and
// about 2 behind its last block.
// Three prompt chunks of 1021, 650 and 279 tokens over 8191, 5214 and 2245 (32 heads over 8): 235 us, 809 TFLOP/s; a fifth
// of it is the tail of 256 tasks of three lengths on 148 SMs. Steps: Q and the exponents by the converters alone, 272; by
// all warps, loads ahead of stores, 242; the wait for K taken off the chain, 233; values and weights right over their whole
// range, 235. A tile that goes by far_tile takes about 1.2 ms for 8191 keys. Rejected: reading S twice to free
// registers (361 - 424 against 267), scales read from shared memory where they are used (280), part of the exponentials by a
// polynomial (289 - 311 against 279), four converter warps (487), P handed over as 96 + 32 keys (248 against 233) or in
// quarters (236), one thread for the issuer's waits (240), the first codes loaded ahead of the start's barrier (266).
#include "rl_common.cuh"
#include "rl_host.h"

namespace rl {
namespace kvprompt {

using kv::BT;
using kv::HD;
using kvattn::Div;

constexpr int BQ = 128;
constexpr int ROWS = 2 * BQ;          // rows per CTA
constexpr int BKV = 128;              // keys per block
constexpr int kThreads = 384;
constexpr int KS = 3, VS = 2;         // operand stages
constexpr int RING = 8;               // blocks whose scales are kept
constexpr int SUB = 128 * 128;        // 128 rows of 64 16-bit values
constexpr int TILE = 2 * SUB;
constexpr int kQ = 0, kK = 2 * TILE, kV = kK + KS * TILE, kBar = kV + VS * TILE;
constexpr int kBytes = 1024 + kBar + 1024;
static_assert(kBytes <= 232448, "shared memory");
constexpr int kTmemCols = 512, kOCol = 256;
constexpr float kTau = 8.0f;
constexpr float kUpP = 7.0f;
constexpr int kUpV = 5;               // V is kept times 2^kUpV: 1152 2^kUpV, the offset, has to be an fp16 number
constexpr int kReach = 24 + kUpV;
constexpr int kConv = 3;              // converter warps: 0, 2 and 3 (1 issues the MMAs)

struct Barriers {
  uint64_t k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], s_full[2], p_full[2][2], o_full, drain;
  uint32_t tmem_base;
  int abort;
  int e_max, e_min;                   // largest and smallest V exponent of the tile's keys
  int e_all;                          // largest V exponent of the blocks that every row (with any key) sees
  int lim_min, lim_max;               // the smallest and largest limit of its rows (with any key)
  int task[6];                        // sequence (or -1), head, tile; the sequence's first row, rows and length
  int v_poison;                       // first position of the first V block with a NaN or an infinity
  alignas(8) uint8_t flag[RING][8];              // per block of 16 keys: 1 = K with a NaN or an infinity, 2 = absent
  alignas(16) float scale[RING][8];   // per block of 16 keys: what its raw scores are multiplied by
};
static_assert(sizeof(Barriers) <= 1024, "barrier block");

struct Args {
  const uint16_t* q;
  int64_t q_st, q_sh;
  kv::Pool pool;
  kv::Batch batch;
  const int32_t* row_limit;
  float scale_log2;
  uint16_t* o;
  int64_t ldo;
  Div group, hkv;
  int page_sh, vec;                   // vec: rows of o are 16-byte aligned
};

// B operand stored [k][64 n] with the 128-byte swizzle (MN-major): 64-column groups SUB bytes apart, 8-row groups 1024.
__device__ __forceinline__ uint64_t sdesc_mnmajor_sw128(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(SUB >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
// kind::f16 with fp16 A and B, B MN-major, fp32 D.
__host__ __device__ constexpr uint32_t idesc_f16_bmn(int M, int N) {
  return (1u << 4) | (1u << 16) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// 16 keys of a block in the lane's registers, with the block's exponent byte (0x100: absent or beyond the keys).
struct Unit {
  uint4 c[4];
  uint32_t e;
};

// Turn a unit into 16 rows of an operand tile (rows r0 ..): 32 bytes of 16-bit values per 16 codes, as two
// 16-byte chunks at swizzled positions. Step i of a lane is row l / 4 + 8 (i / 2), codes 16 (l % 4) + 64 (i % 2) ..: the
// eight lanes of a shared-memory phase then write an even and an odd row, whose chunks lie in eight different bank groups.
__device__ __forceinline__ int unit_row(int i, int lane) { return (lane >> 2) + 8 * (i >> 1); }
__device__ __forceinline__ int unit_code(int i, int lane) { return 16 * (lane & 3) + 64 * (i & 1); }
template <bool kIsV>
__device__ __forceinline__ void write_unit(uint8_t* tile, int r0, const Unit& u, uint32_t mul, uint32_t add, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w[4] = {u.c[i].x, u.c[i].y, u.c[i].z, u.c[i].w};
    uint32_t v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t lo = __byte_perm(w[k], kIsV ? 0x64646464u : 0u, 0x4140), hi = __byte_perm(w[k], kIsV ? 0x64646464u : 0u, 0x4342);
      v[2 * k] = kIsV ? fma_f16x2(lo, mul, add) : fma_bf16x2(lo, mul, add);
      v[2 * k + 1] = kIsV ? fma_f16x2(hi, mul, add) : fma_bf16x2(hi, mul, add);
    }
    uint8_t* at = tile + (i & 1) * SUB + (r0 + unit_row(i, lane)) * 128;
    const int c0 = 2 * (lane & 3), x = (lane >> 2) & 7;             // r0 and 8 (i / 2) are multiples of 8
    *reinterpret_cast<uint4*>(at + ((c0 ^ x) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<uint4*>(at + (((c0 + 1) ^ x) << 4)) = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// One 128-key block of the online softmax of the thread's row, as rl_attn.cu's softmax_block with a scale per 16 keys.
__device__ __forceinline__ void softmax_block(uint32_t ta, uint32_t to, int key0, int lim, const float* scale_at,
                                              uint2 flags, bool o_live, float& m_run, float& l_run, uint64_t* p_bar,
                                              int lane) {
  const float4 sa = *reinterpret_cast<const float4*>(scale_at), sb = *reinterpret_cast<const float4*>(scale_at + 4);
  const float scale[8] = {sa.x, sa.y, sa.z, sa.w, sb.x, sb.y, sb.z, sb.w};
  uint32_t s[BKV];
#pragma unroll
  for (int c = 0; c < BKV / 32; ++c) {
    uint32_t (&sc)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]);
    RL_TMEM_LD32(ta + 32 * c, sc);
  }
  tmem_ld_wait_regs(s);
  if (key0 + BKV - 1 > lim) {
#pragma unroll
    for (int c = 0; c < BKV; ++c)
      if (key0 + c > lim) s[c] = 0xFF800000u;  // -inf
  }
  if (flags.x | flags.y) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t f = (i < 4 ? flags.x : flags.y) >> (8 * (i & 3));
      if (f & 2) {
#pragma unroll
        for (int c = 16 * i; c < 16 * i + 16; ++c) s[c] = 0xFF800000u;
      }
      if ((f & 1) && key0 + 16 * i <= lim) l_run = __uint_as_float(0x7FC00000u);
    }
  }
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float a = -INFINITY, b = -INFINITY;
#pragma unroll
    for (int c = 16 * i; c < 16 * i + 16; c += 4) {
      a = attn::max3f(a, __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
      b = attn::max3f(b, __uint_as_float(s[c + 2]), __uint_as_float(s[c + 3]));
    }
    mx = fmaxf(mx, fmaxf(a, b) * scale[i]);
  }
  const bool raise = mx > m_run + kTau;
  float alpha = 1.0f;
  if (raise) {
    alpha = exp2f(m_run - mx);
    l_run *= alpha;
    m_run = mx;
  }
  const bool rescale = o_live && __any_sync(0xffffffffu, raise);
  const float mz = m_run == -INFINITY ? 0.0f : m_run - kUpP;      // a row that has seen no key: every score is -inf
  const float2 nm2 = make_float2(-mz, -mz);
  float2 acc[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t pk[32];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float f = scale[4 * h + g];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int i = 64 * h + 16 * g + 2 * c;
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), make_float2(f, f), nm2);
        const float2 e = make_float2(attn::ex2_approx(x.x), attn::ex2_approx(x.y));
        pk[8 * g + c] = kvattn::pack_h2(e.x, e.y);
        acc[c & 1] = __fadd2_rn(acc[c & 1], e);
      }
    }
    RL_TMEM_ST32(ta + 32 * h, pk);
    if (h == 0 && rescale) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t o[16];
        RL_TMEM_LD16(to + 16 * c, o);
        tmem_ld_wait_regs(o);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
        RL_TMEM_ST16(to + 16 * c, o);
        tmem_st_wait_regs(o);
      }
    }
    tmem_st_wait_regs(pk);
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&p_bar[h]);
  }
  const float2 a = __fadd2_rn(acc[0], acc[1]);
  l_run += a.x + a.y;
}

// The last key that new token j of a sequence sees (-1: none).
__device__ __forceinline__ int limit_of(const Args& a, const kv::Seq& s, uint32_t j) {
  if (!a.row_limit) return static_cast<int>(s.len - s.n + j);
  return max(-1, min(static_cast<int>(s.len) - 1, __ldg(a.row_limit + s.s0 + j)));
}

// A tile whose values lie too far apart for one fp16 unit (rare): eight rows a warp, over all their keys, block by block as
// the split kernel does. Right for every tile, at a small part of the rate.
__device__ __noinline__ void far_tile(const Args& a, const int (&task)[6]) {
  const int b = task[0], h = task[1];
  const kv::Seq s{task[3], task[4], task[5], true};
  const uint32_t row0 = static_cast<uint32_t>(task[2]) * ROWS, rows = static_cast<uint32_t>(s.n) * a.group.d;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int32_t* table = a.batch.table + b * a.batch.ld;
  const uint32_t end = min(rows, row0 + ROWS);
  for (uint32_t r0 = row0 + 8 * warp; r0 < end; r0 += 8 * (kThreads / 32)) {
    uint4 qw[4] = {};
    if (r0 + g < end) {
      const uint32_t j = (r0 + g) / a.group;
      const uint16_t* p = a.q + (s.s0 + j) * a.q_st + (h * a.group.d + r0 + g - j * a.group.d) * a.q_sh + 16 * c;
#pragma unroll
      for (int i = 0; i < 4; ++i) qw[i] = *reinterpret_cast<const uint4*>(p + 64 * (i >> 1) + 8 * (i & 1));
    }
    uint32_t qf[16];
    const uint32_t e = kvattn::q_fragments(qw, qf);
    float qs[1][2];
    int lim[1][2], lim_min = INT32_MAX, lim_max = -1;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t r = r0 + 2 * c + k;
      qs[0][k] = kvattn::q_scale(e, 2 * c + k, a.scale_log2);
      lim[0][k] = INT32_MAX;                                         // (rows behind the last are not stored)
      if (r < end) {
        lim[0][k] = limit_of(a, s, r / a.group);
        lim_min = min(lim_min, lim[0][k]), lim_max = max(lim_max, lim[0][k]);
      }
    }
#pragma unroll
    for (int d = 1; d <= 2; d <<= 1) {
      lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, d));
      lim_max = max(lim_max, __shfl_xor_sync(0xffffffffu, lim_max, d));
    }
    kvattn::Acc<1> acc = {};
    acc.m[0][0] = acc.m[0][1] = kvattn::kNone;
    for (int u = 0; u * BT <= lim_max; ++u) {
      const int pg = __ldg(table + (u >> (a.page_sh - 4)));
      if (static_cast<uint32_t>(pg) >= a.pool.pages) continue;       // (reported at the tile's start)
      const int64_t blk = (static_cast<int64_t>(pg * a.pool.hkv + h) << (a.page_sh - 4)) + (u & ((1 << (a.page_sh - 4)) - 1));
      const uint8_t* kp = a.pool.k + blk * (BT * HD) + g * HD + 16 * c;
      const uint8_t* vp = a.pool.v + blk * (BT * HD) + 2 * c * HD + 16 * g;
      uint4 kr[4], vr[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        kr[i] = *reinterpret_cast<const uint4*>(kp + (i >> 1) * 8 * HD + (i & 1) * 64);
        vr[i] = *reinterpret_cast<const uint4*>(vp + (i >> 1) * 8 * HD + (i & 1) * HD);
      }
      kvattn::block_step<1>(kr, vr, a.pool.ke[blk], a.pool.ve[blk], u * BT, qf, nullptr, qs, lim, lim_min, g, acc);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float l = acc.l[0][k];
#pragma unroll
      for (int d = 4; d <= 16; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
      const uint32_t r = r0 + 2 * c + k, j = r / a.group;
      if (r >= end) continue;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l, unit = bfp16_scale(static_cast<uint32_t>(acc.unit[0][k]));
      uint16_t* o = a.o + (s.s0 + j) * a.ldo + (h * a.group.d + r - j * a.group.d) * HD + 16 * g;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int y = 0; y < 2; ++y)
          o[2 * i + y] = __bfloat16_as_ushort(__float2bfloat16_rn(acc.o[0][i][k + 2 * y] * inv * unit));
    }
  }
}

__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const __grid_constant__ Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Barriers* bars = reinterpret_cast<Barriers*>(smem + kBar);
  volatile int* abort = &bars->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0) {
    // the task of this CTA: sequences in order, each with kv_heads x ceil(rows / 256) tiles, the last tile first
    int64_t before = 0;
    int found = -1, at = 0;
    for (int b0 = 0; b0 < a.batch.B && found < 0; b0 += 32) {
      const int b = b0 + lane;
      int64_t n = 0;
      if (b < a.batch.B) {
        const kv::Seq s = kv::load_seq(a.batch, b, a.pool.page);
        if (s.ok) n = (s.n * a.group.d + ROWS - 1) / ROWS * a.pool.hkv;
        else if (blockIdx.x == 0) report(kErrBadArgument);
      }
      int64_t end = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, end, d);
        if (lane >= d) end += v;
      }
      const bool mine = static_cast<int64_t>(blockIdx.x) - before < end;
      const uint32_t hit = __ballot_sync(0xffffffffu, mine);
      if (hit) {
        const int l = __ffs(hit) - 1;
        found = b0 + l;
        at = static_cast<int>(blockIdx.x - before - __shfl_sync(0xffffffffu, end - n, l));
      }
      before += __shfl_sync(0xffffffffu, end, 31);
    }
    if (lane == 0) {
      bars->task[0] = found;
      if (found >= 0) {
        const kv::Seq s = kv::load_seq(a.batch, found, a.pool.page);
        const int tiles = static_cast<int>((s.n * a.group.d + ROWS - 1) / ROWS);
        const uint32_t t = static_cast<uint32_t>(at) / a.hkv;
        bars->task[1] = at - static_cast<int>(t) * a.pool.hkv;
        bars->task[2] = tiles - 1 - static_cast<int>(t);
        bars->task[3] = static_cast<int>(s.s0), bars->task[4] = static_cast<int>(s.n), bars->task[5] = static_cast<int>(s.len);
      }
      for (int i = 0; i < KS; ++i) mbar_init(&bars->k_full[i], kConv), mbar_init(&bars->k_empty[i], 1);
      for (int i = 0; i < VS; ++i) mbar_init(&bars->v_full[i], kConv), mbar_init(&bars->v_empty[i], 1);
      for (int t = 0; t < 2; ++t) {
        mbar_init(&bars->s_full[t], 1);
        mbar_init(&bars->p_full[t][0], 4);
        mbar_init(&bars->p_full[t][1], 4);
      }
      mbar_init(&bars->o_full, 1);
      mbar_init(&bars->drain, 1);
      bars->abort = 0;
      bars->e_max = bars->e_all = 0;
      bars->e_min = 255;
      bars->lim_min = INT32_MAX, bars->lim_max = -1;
      bars->v_poison = INT32_MAX;
      fence_mbar_init();
    }
  }
  __syncthreads();
  const int b = bars->task[0];
  if (b < 0) return;   // (the grid is an upper bound)
  const int h = bars->task[1];
  const uint32_t row0 = static_cast<uint32_t>(bars->task[2]) * ROWS;
  const kv::Seq s{bars->task[3], bars->task[4], bars->task[5], true};
  const uint32_t rows = static_cast<uint32_t>(s.n) * a.group.d;
  const uint32_t last_row = min(row0 + ROWS, rows) - 1;
  if (a.row_limit && warp < ROWS / 32) {
    const uint32_t r = row0 + threadIdx.x;
    const int L = r <= last_row ? limit_of(a, s, r / a.group) : -1;
    const int lo = __reduce_min_sync(0xffffffffu, L < 0 ? INT32_MAX : L), hi = __reduce_max_sync(0xffffffffu, L);
    if (lane == 0) atomicMin(&bars->lim_min, lo), atomicMax(&bars->lim_max, hi);
  }
  if (warp == 0) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  // the keys that any row sees, and those that every row sees which sees any: limits grow along the rows, unless row_limit
  // gives them
  const int kmax = a.row_limit ? max(bars->lim_max, 0) + 1 : limit_of(a, s, last_row / a.group) + 1;
  const int lim_all = a.row_limit ? bars->lim_min : limit_of(a, s, row0 / a.group);
  const int nblk = (kmax + BKV - 1) / BKV;                        // >= 1

  // the page of the sequence's 16-key block u (-1 beyond the keys), and the block's pool index in it
  const int32_t* table = a.batch.table + b * a.batch.ld;
  const int units = (kmax + BT - 1) / BT;
  auto page_of = [&](int u) -> int { return u < units ? __ldg(table + (u >> (a.page_sh - 4))) : -1; };
  auto present = [&](int pg) -> bool { return static_cast<uint32_t>(pg) < a.pool.pages; };
  auto block_in = [&](int pg, int u) -> int {
    return ((pg * a.pool.hkv + h) << (a.page_sh - 4)) + (u & ((1 << (a.page_sh - 4)) - 1));
  };
  {
    // Q (256 rows x 16 chunks of 16 bytes) and the largest V exponent, by all warps and with the loads ahead of the stores:
    // this start is paid per task (the converters alone, a load at a time, took 15 us to the first product)
    constexpr int kQLoads = (ROWS * 16 + kThreads - 1) / kThreads;
    uint4 v[kQLoads];
#pragma unroll
    for (int i = 0; i < kQLoads; ++i) {
      const int x = threadIdx.x + i * kThreads;
      const uint32_t rr = row0 + (x >> 4);
      v[i] = make_uint4(0, 0, 0, 0);
      if (x < ROWS * 16 && rr < rows) {
        const uint32_t j = rr / a.group;
        v[i] = *reinterpret_cast<const uint4*>(a.q + (s.s0 + j) * a.q_st + (h * a.group.d + rr - j * a.group.d) * a.q_sh +
                                               8 * (x & 15));
      }
    }
    int e = 0, e_all = 0, e_min = 255;
#pragma unroll 2
    for (int u = threadIdx.x; u < units; u += kThreads) {
      const int pg = page_of(u);
      if (!present(pg)) {
        report(kErrBadArgument);
        continue;
      }
      const int ve = a.pool.ve[block_in(pg, u)];
      if (ve != 255) {
        e = max(e, ve), e_min = min(e_min, ve);
        if (u * BT <= lim_all) e_all = max(e_all, ve);
      } else {
        atomicMin(&bars->v_poison, u * BT);
      }
    }
    e = __reduce_max_sync(0xffffffffu, e);
    e_all = __reduce_max_sync(0xffffffffu, e_all);
    e_min = __reduce_min_sync(0xffffffffu, e_min);
    if (lane == 0) atomicMax(&bars->e_max, e), atomicMax(&bars->e_all, e_all), atomicMin(&bars->e_min, e_min);
#pragma unroll
    for (int i = 0; i < kQLoads; ++i) {
      const int x = threadIdx.x + i * kThreads, r = x >> 4, c = x & 15, y = r & 127;
      if (x < ROWS * 16)
        *reinterpret_cast<uint4*>(smem + kQ + (r >> 7) * TILE + (c >> 3) * SUB + y * 128 + (((c & 7) ^ (y & 7)) << 4)) = v[i];
    }
    fence_proxy_async_smem();
  }
  __syncthreads();

  if (bars->e_max - bars->e_min > kReach && bars->e_max - bars->e_all > 1) {
    far_tile(a, bars->task);
  } else if (warp < 4) {
    if (warp != 1) {
      // ---------------- converters ----------------
      const int cw = warp == 0 ? 0 : warp - 1;
      const int em = bars->e_max;

      // Warp cw converts units cw, cw + 3 and cw + 6 of each block's eight. The codes of block j + 1 are loaded into
      // registers as soon as block j's have been converted, so a load has the time of a whole block; page lookups run
      // one block further ahead.
      Unit ku[3], vu[3];
      int pg[3];                                                  // pages of the next block's units
      auto lookup = [&](int j) {
#pragma unroll
        for (int i = 0; i < 3; ++i) pg[i] = page_of(j < nblk ? j * 8 + cw + 3 * i : units);
      };
      auto load = [&](const uint8_t* codes, const uint8_t* exps, int j, Unit (&u)[3]) {
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          const int k = cw + 3 * i;
          const bool in = present(pg[i]);
          const int64_t blk = in ? block_in(pg[i], j * 8 + k) : 0;   // beyond the keys, or absent: any block, of weight zero
          u[i].e = in ? exps[blk] : 0x100u;
          const uint8_t* p = codes + blk * (BT * HD) + unit_row(0, lane) * HD + unit_code(0, lane);
#pragma unroll
          for (int y = 0; y < 4; ++y) u[i].c[y] = *reinterpret_cast<const uint4*>(p + 8 * (y >> 1) * HD + 64 * (y & 1));
        }
      };
      lookup(0);
      load(a.pool.k, a.pool.ke, 0, ku);
      load(a.pool.v, a.pool.ve, 0, vu);
      lookup(1);
      for (int j = 0; j < nblk; ++j) {
        const int ks = j % KS, vs = j % VS;
        if (!mbar_wait_warp(&bars->k_empty[ks], ((j / KS) & 1) ^ 1, abort)) break;
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (cw + 3 * i < 8) write_unit<false>(smem + kK + ks * TILE, 16 * (cw + 3 * i), ku[i], 0x7F007F00u, 0xC000C000u, lane);
        if (lane < 3 && cw + 3 * lane < 8) {                      // (the last use of this slot was eight blocks ago)
          const uint32_t e = lane == 0 ? ku[0].e : lane == 1 ? ku[1].e : ku[2].e;
          // (never zero: a masked score is -inf times this)
          bars->scale[j % RING][cw + 3 * lane] =
              e == 255u ? 1.0f : fmaxf(bfp16_scale(e & 255u) * 64.0f * a.scale_log2, 1.17549435e-38f);
          bars->flag[j % RING][cw + 3 * lane] = static_cast<uint8_t>((e == 255u ? 1 : 0) | (e & 0x100u ? 2 : 0));
        }
        load(a.pool.k, a.pool.ke, j + 1, ku);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->k_full[ks]);
        if (!mbar_wait_warp(&bars->v_empty[vs], ((j / VS) & 1) ^ 1, abort)) break;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          // 2^(kUpV - d) and -1152 times it in fp16. P = 0 for keys beyond the end or absent; a poisoned block's codes count as
          // they are (the rows that see it become NaN).
          const int d = vu[i].e == 255u ? 0 : em - static_cast<int>(vu[i].e & 255u);
          const float f = d > kReach ? 0.0f : __uint_as_float(static_cast<uint32_t>(127 + kUpV - d) << 23);
          if (cw + 3 * i < 8)
            write_unit<true>(smem + kV + vs * TILE, 16 * (cw + 3 * i), vu[i], kvattn::pack_h2(f, f),
                             kvattn::pack_h2(-1152.0f * f, -1152.0f * f), lane);
        }
        load(a.pool.v, a.pool.ve, j + 1, vu);
        lookup(j + 2);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->v_full[vs]);
      }
    } else {
      // ---------------- MMA issuer (warp-wide, elected lane issues) ----------------
      constexpr uint32_t idesc_s = idesc_bf16(BQ, BKV);
      constexpr uint32_t idesc_o = idesc_f16_bmn(BQ, HD);
      bool any = false;
      const uint32_t qa0 = smem_u32(smem + kQ);
      auto k_ready = [&](int j) -> bool { return mbar_wait_warp(&bars->k_full[j % KS], (j / KS) & 1, abort); };
      auto qk = [&](int t, int j) {
        const int st = j % KS;
        tc_fence_after();
        const uint32_t qa = qa0 + t * TILE, kb = smem_u32(smem + kK + st * TILE);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            const uint64_t adesc = sdesc_kmajor_sw128(qa + (k >> 2) * SUB) + 2 * (k & 3);
            const uint64_t bdesc = sdesc_kmajor_sw128(kb + (k >> 2) * SUB) + 2 * (k & 3);
            umma_ss(tmem + t * BKV, adesc, bdesc, idesc_s, k ? 1u : 0u);
          }
          umma_commit(&bars->s_full[t]);
          if (t == 1) umma_commit(&bars->k_empty[st]);
        }
        __syncwarp();
        any = true;
      };
      auto pv = [&](int t, int j) -> bool {
        const int st = j % VS;
        if (!mbar_wait_warp(&bars->v_full[st], (j / VS) & 1, abort)) return false;
        const uint32_t vb = smem_u32(smem + kV + st * TILE);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          // (K of the product behind this one is waited for here, where the wait is hidden)
          if (hh == 1 && j + 1 < nblk && !k_ready(j + 1)) return false;
          if (!mbar_wait_warp(&bars->p_full[t][hh], j & 1, abort)) return false;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 4 * hh; k < 4 * hh + 4; ++k)
              umma_ts(tmem + kOCol + t * HD, tmem + t * BKV + k * 8, sdesc_mnmajor_sw128(vb + k * 2048), idesc_o,
                      (j | k) ? 1u : 0u);
            if (hh == 1 && t == 1) umma_commit(&bars->v_empty[st]);
          }
          __syncwarp();
        }
        return true;
      };
      bool ok = k_ready(0);
      if (ok) qk(0, 0), qk(1, 0);
      for (int j = 0; ok && j < nblk; ++j)
        for (int t = 0; ok && t < 2; ++t) {
          ok = pv(t, j);
          if (ok && j + 1 < nblk) qk(t, j + 1);
        }
      if (elect_one()) {
        if (ok) umma_commit(&bars->o_full);
        if (!ok && any) {
          umma_commit(&bars->drain);
          mbar_drain(&bars->drain, 0);
        }
      }
      __syncwarp();
    }
  } else {
    // ---------------- softmax of tile t (thread = row = TMEM lane) ----------------
    const int t = (warp - 4) >> 2, q = warp & 3;
    const uint32_t row = row0 + t * BQ + 32 * q + lane;
    const uint32_t lane_off = (32u * q) << 16;
    const uint32_t ta = tmem + t * BKV + lane_off, to = tmem + kOCol + t * HD + lane_off;
    const uint32_t jr = row / a.group;
    // (rows behind the last, which are not stored, see what it sees: a mask in every block would cost their warp 1000 cycles)
    const uint32_t jl = min(jr, static_cast<uint32_t>(s.n) - 1);
    const int lim = limit_of(a, s, jl);
    float m_run = -INFINITY, l_run = 0.0f;
    bool ok = true;
    for (int j = 0; j < nblk; ++j) {
      if (!mbar_wait(&bars->s_full[t], j & 1, abort)) { ok = false; break; }
      tc_fence_after();
      softmax_block(ta, to, j * BKV, lim, bars->scale[j % RING], *reinterpret_cast<const uint2*>(bars->flag[j % RING]), j > 0,
                    m_run, l_run, bars->p_full[t], lane);
    }
    if (ok && mbar_wait(&bars->o_full, 0, abort)) {
      tc_fence_after();
      if (bars->v_poison <= lim) l_run = __uint_as_float(0x7FC00000u);
      // (two factors: their product may leave the range of a float)
      const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run, unit = bfp16_scale(static_cast<uint32_t>(bars->e_max)) * 0x1p-5f;
      static_assert(kUpV == 5, "unit of O");
      uint16_t* orow = a.o + (s.s0 + jr) * a.ldo + (h * a.group.d + row - jr * a.group.d) * HD;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        RL_TMEM_LD32(to + 32 * c, o);
        tmem_ld_wait_regs(o);
        if (row < rows) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            w[i] = attn::pack_bf16x2(__uint_as_float(o[2 * i]) * inv * unit, __uint_as_float(o[2 * i + 1]) * inv * unit);
          if (a.vec) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              reinterpret_cast<uint4*>(orow + 32 * c)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              orow[32 * c + 2 * i] = static_cast<uint16_t>(w[i]);
              orow[32 * c + 2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

inline int launch(int64_t tasks, const Args& a, cudaStream_t stream) {
  static PerDevice ready;
  RL_TRY_CUDA(ready.once([] { return cudaFuncSetAttribute(prompt_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes); }));
  prompt_kernel<<<static_cast<unsigned>(tasks), kThreads, kBytes, stream>>>(a);
  RL_TRY_CUDA(cudaGetLastError());
  return RL_OK;
}

}  // namespace kvprompt
}  // namespace rl
