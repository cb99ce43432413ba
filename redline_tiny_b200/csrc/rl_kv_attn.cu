// Attention of a few new tokens per sequence over the 8-bit paged cache (rl_kv.cu), head dim 128.
//
// o_r = sum_k p_rk v_k / sum_k p_rk, p_rk = 2^(s_rk - m_r), s_rk = scale_log2 * q_r . k_k over the keys k <= limit_r.
// With K = 2^(ek-133) mk per block of 16 tokens, s is an fp16 product q~ . mk (mk is an integer in [-128, 127], exact;
// q~ is q times a power of two per row that puts the row's largest value in [2^14, 2^15), exact for every value within
// 2^-28 of it) times one fp32 factor per block and row. P is rounded to fp16 (11 significant bits, half a step 2^-11
// of each weight; the row sum adds the rounded weights) and P . mv of a block, again with exact integers, is scaled by
// 2^(ev-133) as it is added to the fp32 accumulator. So the only roundings are P's and fp32's.
//
// The rows of one K/V head that share its keys (tokens of a sequence x query heads of the group) are the N side of
// mma.m16n8k16: S^T (16 tokens x 8 rows) = K q~^T and O^T (16 dims x 8 rows) += V^T P^T. The cache is then the A
// operand and is turned from bytes to fp16 in registers once for all rows: u -> 1024 + u by a byte permute, minus 1152
// in one packed subtraction. P^T goes from the accumulator layout to the B layout with movmatrix. The k index of both
// products may be permuted freely, so each lane's bytes are its own 16-byte loads: dims 16c.. and 64 + 16c.. of tokens
// g and g + 8 for K, dims 16g.. of tokens 2c, 2c + 1, 2c + 8, 2c + 9 for V (lane = 4g + c).
//
// Work is split evenly over the CTAs whatever the lengths are: a task is (sequence, K/V head, 8 NT rows), its units
// are 64 keys; CTA i takes units [i U / C, (i + 1) U / C) of the whole list. A task that a CTA does not finish leaves
// (O, m, l) in the workspace, and combine_kernel joins the pieces in CTA order, so results do not depend on timing.
#include "rl_common.cuh"
#include "rl_host.h"

namespace rl {
namespace kvattn {

using kv::BT;
using kv::HD;

constexpr int UNIT = 64;         // keys per unit of work
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kRaise = 8.0f;   // the running maximum rises only when a score exceeds it by more (log2): P <= 2^8

struct Args {
  const uint16_t* q;
  int64_t q_st, q_sh;
  kv::Pool pool;
  kv::Batch batch;
  const int32_t* row_limit;
  float scale_log2;
  uint16_t* o;
  int64_t ldo;
  int group;                     // query heads per K/V head
  float* part;                   // workspace: 2 slots per CTA of R x (128 + 2) floats
  int4* rec;                     // workspace: per CTA, the task it began and did not finish
};

// A piece record: rows [row0, row0 + R) of task (b, h) in `n` pieces, the first in slot `slot` of this CTA.
struct Piece {
  int b, h, tile, n;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2sub(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float2 unpack_h2(uint32_t h) {
  float2 f;
  asm("{.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;}" : "=f"(f.x), "=f"(f.y) : "r"(h));
  return f;
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Bytes (u0, u1) of a word pair, as fp16 integers u - 128.
template <int kSel>
__device__ __forceinline__ uint32_t codes_h2(uint32_t w) {
  return h2sub(__byte_perm(w, 0x64646464u, kSel), 0x64806480u);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}

// The list of units: sequence b has hkv * tiles(b) tasks of chunks(b) units each.
__device__ __forceinline__ int64_t tiles_of(const Args& a, const kv::Seq& s, int R) {
  return (s.n * a.group + R - 1) / R;
}
__device__ __forceinline__ int64_t chunks_of(const kv::Seq& s) { return s.len > 0 ? (s.len + UNIT - 1) / UNIT : 1; }

// Prefix sums of the sequences' units into `pre` (B + 1 values), by the whole CTA.
__device__ __forceinline__ void unit_prefix(const Args& a, int R, int64_t* pre, int64_t* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) pre[0] = 0;
  int64_t base = 0;
  for (int b0 = 0; b0 < a.batch.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int64_t u = 0;
    if (b < a.batch.B) {
      const kv::Seq s = kv::load_seq(a.batch, b, a.pool.page);
      if (s.ok) u = tiles_of(a, s, R) * chunks_of(s) * a.pool.hkv;
      else if (blockIdx.x == 0) report(kErrBadArgument);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, u, d);
      if (lane >= d) u += v;
    }
    if (lane == 31) warp_sum[warp] = u;
    __syncthreads();
    int64_t before = base;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    if (b < a.batch.B) pre[b + 1] = before + u;
    for (int w = 0; w < kWarps; ++w) base += warp_sum[w];
    __syncthreads();
  }
}

template <int NT>
struct Acc {
  float o[NT][8][4];     // O^T: dims 16g + 2i (+1 for [2], [3]), rows 2c, 2c + 1 of n-tile nt
  float m[NT][2], l[NT][2];
};

// One warp, one block of 16 keys starting at position pos0.
template <int NT>
__device__ __forceinline__ void block_step(const uint4 (&kr)[4], const uint4 (&vr)[4], uint32_t ke, uint32_t ve,
                                           int64_t pos0, const uint32_t (&qf)[16], uint32_t q_at, const float (&qs)[NT][2],
                                           const int (&lim)[NT][2], int lim_min, int g, Acc<NT>& acc) {
  float s[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
  const uint32_t* k0[2] = {&kr[0].x, &kr[1].x};   // token g: dims 16c.., 64 + 16c..
  const uint32_t* k1[2] = {&kr[2].x, &kr[3].x};   // token g + 8
#pragma unroll
  for (int jj = 0; jj < 4; ++jj) {
    uint32_t A[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = 2 * jj + i;
      const uint32_t w0 = k0[j >> 2][j & 3], w1 = k1[j >> 2][j & 3];
      A[i][0] = codes_h2<0x4140>(w0), A[i][2] = codes_h2<0x4342>(w0);
      A[i][1] = codes_h2<0x4140>(w1), A[i][3] = codes_h2<0x4342>(w1);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint4 q = make_uint4(qf[4 * jj], qf[4 * jj + 1], qf[4 * jj + 2], qf[4 * jj + 3]);
      if (NT > 1) q = lds128(q_at + (nt * 4 + jj) * 512);
      mma(s[nt], A[0][0], A[0][1], A[0][2], A[0][3], q.x, q.y);
      mma(s[nt], A[1][0], A[1][1], A[1][2], A[1][3], q.z, q.w);
    }
  }
  const float ks = ke == 255u ? __uint_as_float(0x7FC00000u) : bfp16_scale(ke);
  bool raise = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s[nt][i] = s[nt][i] * ks * qs[nt][i & 1];
    if (pos0 + BT - 1 > lim_min) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (pos0 + g + 8 * (i >> 1) > lim[nt][i & 1]) s[nt][i] = -INFINITY;
    }
    raise |= fmaxf(s[nt][0], s[nt][2]) > acc.m[nt][0] + kRaise || fmaxf(s[nt][1], s[nt][3]) > acc.m[nt][1] + kRaise;
  }
  if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float mx = fmaxf(s[nt][c], s[nt][c + 2]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float m = fmaxf(acc.m[nt][c], mx);
        const float alpha = m == acc.m[nt][c] ? 1.0f : exp2_approx(acc.m[nt][c] - m);
        acc.m[nt][c] = m;
        acc.l[nt][c] *= alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc.o[nt][i][c] *= alpha;
          acc.o[nt][i][c + 2] *= alpha;
        }
      }
  }
  uint32_t p[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float m0 = acc.m[nt][0] == -INFINITY ? 0.0f : acc.m[nt][0];
    const float m1 = acc.m[nt][1] == -INFINITY ? 0.0f : acc.m[nt][1];
    const uint32_t lo = pack_h2(exp2_approx(s[nt][0] - m0), exp2_approx(s[nt][1] - m1));
    const uint32_t hi = pack_h2(exp2_approx(s[nt][2] - m0), exp2_approx(s[nt][3] - m1));
    const float2 f = unpack_h2(lo), h = unpack_h2(hi);
    acc.l[nt][0] += f.x + h.x;
    acc.l[nt][1] += f.y + h.y;
    p[nt][0] = movmatrix(lo);
    p[nt][1] = movmatrix(hi);
  }
  if (ve == 255u) {   // a block with a NaN or an infinity: NaN for the rows that see it, nothing for the others
    const float nan = __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (pos0 <= lim[nt][c]) {
#pragma unroll
          for (int i = 0; i < 8; ++i) acc.o[nt][i][c] = acc.o[nt][i][c + 2] = nan;
        }
    return;
  }
  const float vs = bfp16_scale(ve);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t t0 = (&vr[0].x)[w], t1 = (&vr[1].x)[w], t2 = (&vr[2].x)[w], t3 = (&vr[3].x)[w];
#pragma unroll
    for (int hl = 0; hl < 2; ++hl) {
      const uint32_t x = __byte_perm(t0, t1, hl ? 0x7362 : 0x5140), y = __byte_perm(t2, t3, hl ? 0x7362 : 0x5140);
      const uint32_t a0 = codes_h2<0x4140>(x), a1 = codes_h2<0x4342>(x);
      const uint32_t a2 = codes_h2<0x4140>(y), a3 = codes_h2<0x4342>(y);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma(t, a0, a1, a2, a3, p[nt][0], p[nt][1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc.o[nt][2 * w + hl][i] = fmaf(vs, t[i], acc.o[nt][2 * w + hl][i]);
      }
    }
  }
}

// Shared memory of a CTA: the ring that brings blocks in (per warp kStages x [K 2 KB | V 2 KB]), reused at the end of a
// run for the warps' results (kWarps x R x 128 floats), then their maxima and sums, then the unit prefix.
template <int NT>
struct Cfg {
  static constexpr int R = 8 * NT;
  static constexpr int kStages = NT == 4 ? 4 : 3;
  static constexpr int kCtas = NT == 1 ? 4 : 2;                       // resident per SM
  static constexpr int kRing = kWarps * kStages * 2 * BT * HD;
  static constexpr int kOut = kWarps * R * HD * 4;
  static constexpr int kBody = kRing > kOut ? kRing : kOut;
  static constexpr int kQ = NT == 1 ? 0 : NT * 16 * 32 * 4;            // q fragments, where registers cannot hold them
  static size_t smem(int B) { return kBody + kQ + kWarps * R * 8 + (kWarps + B + 1) * sizeof(int64_t); }
};

template <int NT>
__global__ void __launch_bounds__(kThreads, Cfg<NT>::kCtas) attend_kernel(const Args a) {
  constexpr int R = 8 * NT;
  constexpr int S = Cfg<NT>::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  float* so = reinterpret_cast<float*>(smem);                        // [warp][row][128]
  uint8_t* sq = smem + Cfg<NT>::kBody;                               // [n-tile][4][lane] x 16 bytes
  float* sm = reinterpret_cast<float*>(sq + Cfg<NT>::kQ);            // [warp][row] maxima
  float* sl = sm + kWarps * R;                                       // [warp][row] sums
  int64_t* warp_sum = reinterpret_cast<int64_t*>(sl + kWarps * R);
  int64_t* pre = warp_sum + kWarps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  unit_prefix(a, R, pre, warp_sum);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t U = pre[a.batch.B];
  const int64_t C = min(static_cast<int64_t>(gridDim.x), U);        // every working CTA has at least one unit
  const bool idle = blockIdx.x >= C;
  const int64_t u_end = idle ? 0 : (blockIdx.x + 1) * U / C;
  int64_t u = idle ? 0 : blockIdx.x * U / C;
  bool first = true;
  Piece rec{0, 0, 0, 0};
  int b = 0;

  // ring addresses of this lane. Row r of a block keeps its 16-byte chunk j at chunk j ^ f(r), f = 4 (r & 1) for K and
  // 2 ((r >> 1) & 3) for V, so that the eight lanes of a shared-memory phase read eight different bank groups.
  const uint32_t ring = smem_u32(smem) + warp * (S * 2 * BT * HD);
  const int wr = lane >> 3, wc = lane & 7;                           // copies: rows wr, wr + 4, ..; chunk wc
  const uint32_t k_ld = g * HD + ((c ^ ((g & 1) * 4)) << 4);
  const uint32_t v_ld = BT * HD + 2 * c * HD + ((g ^ (2 * c)) << 4);

  while (u < u_end) {
    // the task of unit u
    int lo = b, hi = a.batch.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= u) lo = mid; else hi = mid;
    }
    b = lo;
    const kv::Seq s = kv::load_seq(a.batch, b, a.pool.page);
    const int64_t nch = chunks_of(s);
    const int64_t task = (u - pre[b]) / nch, ch0 = (u - pre[b]) - task * nch;
    const int64_t ch1 = min(nch, ch0 + (u_end - u));
    const int h = static_cast<int>(task % a.pool.hkv);
    const int64_t tile = task / a.pool.hkv;
    const int64_t rows = s.n * a.group;                              // rows of this K/V head

    uint32_t qf[16];
    float qs[NT][2];
    int lim[NT][2];
    int lim_min = INT32_MAX, lim_max = -1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int64_t rr = tile * R + nt * 8 + 2 * c + k;
        int64_t L = -1;
        if (rr < rows) {
          L = s.len - s.n + rr / a.group;
          if (a.row_limit) L = min(s.len - 1, static_cast<int64_t>(__ldg(a.row_limit + s.s0 + rr / a.group)));
        }
        lim[nt][k] = static_cast<int>(max(L, static_cast<int64_t>(-1)));
        lim_max = max(lim_max, lim[nt][k]);
        lim_min = min(lim_min, lim[nt][k]);
      }
    }
    lim_max = max(lim_max, __shfl_xor_sync(0xffffffffu, lim_max, 1));
    lim_max = max(lim_max, __shfl_xor_sync(0xffffffffu, lim_max, 2));
    lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 1));
    lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 2));

    // the warp's blocks: every fourth of the run. Lane j holds the pool index of block 32 t + j, one chunk ahead.
    const int64_t key_end = min(ch1 * UNIT, static_cast<int64_t>(lim_max) + 1);
    const int64_t pos0 = ch0 * UNIT + warp * BT;
    const int n = key_end > pos0 ? static_cast<int>((key_end - pos0 + UNIT - 1) / UNIT) : 0;
    auto block_of = [&](int k) -> int {
      if (k >= n) return -1;
      const int64_t blk = kv::block_index(a.pool, a.batch, b, pos0 + static_cast<int64_t>(k) * UNIT, h);
      if (blk < 0) report(kErrBadArgument);                          // a page outside the pool: its keys are absent
      return static_cast<int>(blk);
    };
    int idx = block_of(lane), idx_next = block_of(32 + lane);
    uint32_t ex[S];                                                  // ke | ve << 8 | present << 16 of the ring's blocks
    auto issue = [&](int k, uint32_t& e) {
      if (k < n) {
        if ((k & 31) == 0 && k > 0) {
          idx = idx_next;
          idx_next = block_of(k + 32 + lane);
        }
        const int64_t blk = __shfl_sync(0xffffffffu, idx, k & 31);
        e = 0;
        if (blk >= 0) {
          e = a.pool.ke[blk] | (a.pool.ve[blk] << 8) | 0x10000u;
          const uint8_t* kp = a.pool.k + blk * (BT * HD) + lane * 16;
          const uint8_t* vp = a.pool.v + blk * (BT * HD) + lane * 16;
          const uint32_t d = ring + (k % S) * (2 * BT * HD) + wr * HD;
#pragma unroll
          for (int j = 0; j < 4; ++j) cp_async16(d + j * 4 * HD + ((wc ^ ((wr & 1) * 4)) << 4), kp + j * 512);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            cp_async16(d + BT * HD + j * 4 * HD + ((wc ^ ((((wr + 4 * j) >> 1) & 3) * 2)) << 4), vp + j * 512);
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int k = 0; k < S - 1; ++k) issue(k, ex[k]);

    // q of the tile, while the first blocks are on their way
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int64_t r = tile * R + nt * 8 + g;                       // the row whose q this lane loads
      uint4 w[4] = {};
      if (r < rows) {
        const uint16_t* p = a.q + (s.s0 + r / a.group) * a.q_st + (h * a.group + r % a.group) * a.q_sh + 16 * c;
        w[0] = *reinterpret_cast<const uint4*>(p), w[1] = *reinterpret_cast<const uint4*>(p + 8);
        w[2] = *reinterpret_cast<const uint4*>(p + 64), w[3] = *reinterpret_cast<const uint4*>(p + 72);
      }
      const uint32_t x[16] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w,
                              w[2].x, w[2].y, w[2].z, w[2].w, w[3].x, w[3].y, w[3].z, w[3].w};
      uint32_t mx = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = max(mx, max(x[i] & 0x7FFFu, x[i] >> 16 & 0x7FFFu));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const uint32_t e = max(mx >> 7, 32u);                          // exponent field (values below 2^-95 keep less)
      const float up = __uint_as_float((268u - e) << 23);            // 2^(141 - e)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        qf[i] = pack_h2(__uint_as_float(x[i] << 16) * up, __uint_as_float(x[i] & 0xFFFF0000u) * up);
      if (NT > 1 && nt % kWarps == warp) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          reinterpret_cast<uint4*>(sq)[(nt * 4 + i) * 32 + lane] =
              make_uint4(qf[4 * i], qf[4 * i + 1], qf[4 * i + 2], qf[4 * i + 3]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int ec = __shfl_sync(0xffffffffu, static_cast<int>(e), (2 * c + k) * 4);
        qs[nt][k] = __uint_as_float(static_cast<uint32_t>(ec - 14) << 23) * a.scale_log2;   // 2^(e - 141)
      }
    }

    if (NT > 1) __syncthreads();
    const uint32_t q_at = smem_u32(sq) + lane * 16;

    Acc<NT> acc;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      acc.m[nt][0] = acc.m[nt][1] = -INFINITY;
      acc.l[nt][0] = acc.l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc.o[nt][i][0] = acc.o[nt][i][1] = acc.o[nt][i][2] = acc.o[nt][i][3] = 0.0f;
    }
    for (int i0 = 0; i0 < n; i0 += S) {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const int i = i0 + j;
        if (i < n) {
          cp_wait<S - 2>();
          __syncwarp();        // block i of every lane is in; every lane is done with block i - 1
          issue(i + S - 1, ex[(j + S - 1) % S]);
          if (ex[j] & 0x10000u) {
            const uint32_t at = ring + j * (2 * BT * HD);
            uint4 kr[4], vr[4];
            kr[0] = lds128(at + k_ld), kr[1] = lds128(at + (k_ld ^ 64));
            kr[2] = lds128(at + k_ld + 8 * HD), kr[3] = lds128(at + (k_ld ^ 64) + 8 * HD);
            vr[0] = lds128(at + v_ld), vr[1] = lds128(at + v_ld + HD);
            vr[2] = lds128(at + v_ld + 8 * HD), vr[3] = lds128(at + v_ld + 9 * HD);
            block_step<NT>(kr, vr, ex[j] & 255u, ex[j] >> 8 & 255u, pos0 + static_cast<int64_t>(i) * UNIT, qf, q_at, qs, lim,
                           lim_min, g, acc);
          }
        }
      }
    }
    cp_wait<0>();
    __syncthreads();           // every warp is done with the ring

    // join the warps: (O, m, l) of each through shared memory
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float l = acc.l[nt][k];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int row = nt * 8 + 2 * c + k;
        if (g == 0) sm[warp * R + row] = acc.m[nt][k], sl[warp * R + row] = l;
        float* d = so + (warp * R + row) * HD + 16 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          reinterpret_cast<float4*>(d)[i] = make_float4(acc.o[nt][2 * i][k], acc.o[nt][2 * i][k + 2],
                                                        acc.o[nt][2 * i + 1][k], acc.o[nt][2 * i + 1][k + 2]);
      }
    __syncthreads();
    const bool whole = ch0 == 0 && ch1 == nch;
    float* part = a.part + (static_cast<int64_t>(blockIdx.x) * 2 + (first ? 0 : 1)) * R * (HD + 2);
    const int d = threadIdx.x;
    for (int row = 0; row < R; ++row) {
      const int64_t r = tile * R + row;
      if (r >= rows) break;
      float m = sm[row];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) m = fmaxf(m, sm[w * R + row]);
      const float mz = m == -INFINITY ? 0.0f : m;
      float l = 0.0f, o = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2f(sm[w * R + row] - mz);
        l += f * sl[w * R + row];
        o += f * so[(w * R + row) * HD + d];
      }
      if (whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        a.o[(s.s0 + r / a.group) * a.ldo + (h * a.group + r % a.group) * HD + d] =
            __bfloat16_as_ushort(__float2bfloat16_rn(o * inv));
      } else {
        part[row * HD + d] = o;
        if (d == 0) part[R * HD + row] = m, part[R * HD + R + row] = l;
      }
    }
    if (!whole && ch0 == 0) {
      // the pieces end in the CTA that holds the task's last unit x: floor(j U / C) <= x < floor((j + 1) U / C)
      const int64_t x = u + nch - 1;
      rec = Piece{b, h, static_cast<int>(tile), static_cast<int>(((x + 1) * C - 1) / U - blockIdx.x) + 1};
      if (!first) rec.n = -rec.n;                                    // the first piece lies in the CTA's second slot
    }
    u += ch1 - ch0;
    first = false;
    __syncthreads();
  }
  if (threadIdx.x == 0) a.rec[blockIdx.x] = make_int4(rec.b, rec.h, rec.tile, rec.n);
}

// CTA i joins the pieces of the task that CTA i of attend_kernel began and did not finish: a warp per row, 4 dims a lane.
// Launched while attend_kernel still runs (its CTAs need no more than a slot), it waits for that grid's end.
constexpr int kJoin = 8;   // warps
template <int NT>
__global__ void __launch_bounds__(32 * kJoin) combine_kernel(const Args a) {
  constexpr int R = 8 * NT;
  constexpr int64_t kSlot = R * (HD + 2);
  const int lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 rec = a.rec[blockIdx.x];
  if (rec.w == 0) return;
  const int pieces = abs(rec.w);
  const kv::Seq s = kv::load_seq(a.batch, rec.x, a.pool.page);
  const int64_t rows = s.n * a.group;
  // piece 0 may lie in the CTA's second slot; the others in the first slots of the CTAs behind
  const float* base = a.part + static_cast<int64_t>(blockIdx.x) * 2 * kSlot;
  auto piece = [&](int j) { return base + (j == 0 ? (rec.w < 0 ? kSlot : 0) : j * 2 * kSlot); };
  for (int row = threadIdx.x >> 5; row < R; row += kJoin) {
    const int64_t r = static_cast<int64_t>(rec.z) * R + row;
    if (r >= rows) break;
    float m = -INFINITY;
    for (int j = lane; j < pieces; j += 32) m = fmaxf(m, piece(j)[R * HD + row]);
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float z = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int j = 0; j < pieces; ++j) {
      const float* p = piece(j);
      const float4 v = *reinterpret_cast<const float4*>(p + row * HD + 4 * lane);
      const float f = exp2f(p[R * HD + row] - z);
      l = fmaf(f, p[R * HD + R + row], l);
      o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* d = a.o + (s.s0 + r / a.group) * a.ldo + (rec.y * a.group + r % a.group) * HD + 4 * lane;
    const float v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = __bfloat16_as_ushort(__float2bfloat16_rn(v[i]));
  }
}

inline int tile_n(int64_t T, int B, int group) {
  // rows of a K/V head per sequence, on average: the smallest tile that holds them. A wider tile reads the cache fewer
  // times, a narrower one computes fewer empty rows; any choice is right for any batch.
  const int64_t rows = B > 0 ? (T * group + B - 1) / B : 0;
  return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}
inline int ctas_of(int nt) { return sm_count() * (nt == 1 ? Cfg<1>::kCtas : nt == 2 ? Cfg<2>::kCtas : Cfg<4>::kCtas); }
inline size_t part_bytes(int nt) { return static_cast<size_t>(ctas_of(nt)) * 2 * 8 * nt * (HD + 2) * 4; }

template <int NT>
inline int launch(const Args& a, cudaStream_t st) {
  const size_t smem = Cfg<NT>::smem(a.batch.B);
  const int ctas = ctas_of(NT);
  RL_TRY_CUDA(cudaFuncSetAttribute(attend_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   static_cast<int>(Cfg<NT>::smem(kv::kMaxBatch))));
  attend_kernel<NT><<<ctas, kThreads, smem, st>>>(a);
  RL_TRY_CUDA(cudaGetLastError());
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(32 * kJoin);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  RL_TRY_CUDA(cudaLaunchKernelEx(&cfg, combine_kernel<NT>, a));
  return RL_OK;
}

}  // namespace kvattn
}  // namespace rl

extern "C" {

size_t rl_kv_attention_workspace(int64_t T, int B, int heads, int kv_heads) {
  using namespace rl;
  if (T <= 0 || B <= 0 || kv_heads <= 0 || heads <= 0) return 0;
  const int nt = kvattn::tile_n(T, B, heads / kv_heads);
  return kvattn::part_bytes(nt) + static_cast<size_t>(kvattn::ctas_of(nt)) * sizeof(int4);
}

int rl_kv_attention(const uint16_t* q, int64_t q_st, int64_t q_sh, int64_t T, int heads, const uint8_t* pool_k,
                    const uint8_t* pool_v, const uint8_t* pool_ke, const uint8_t* pool_ve, int64_t pages, int kv_heads,
                    int page, const int32_t* table, int64_t table_ld, const int32_t* kv_len, const int32_t* q_start,
                    int B, const int32_t* row_limit, float scale_log2, uint16_t* o, int64_t ldo, void* workspace,
                    size_t workspace_bytes, rl_stream_t stream) {
  using namespace rl;
  kvattn::Args a;
  a.pool = kv::Pool{const_cast<uint8_t*>(pool_k), const_cast<uint8_t*>(pool_v), const_cast<uint8_t*>(pool_ke),
                    const_cast<uint8_t*>(pool_ve), pages, kv_heads, page};
  a.batch = kv::Batch{table, table_ld, kv_len, q_start, B, T};
  int st;
  if ((st = kv::check_pool("rl_kv_attention", a.pool)) != RL_OK ||
      (st = kv::check_batch("rl_kv_attention", a.batch)) != RL_OK)
    return st;
  RL_REQUIRE(heads > 0 && heads % kv_heads == 0, RL_ERR_ARGUMENT, "rl_kv_attention: %d query heads over %d K/V heads",
             heads, kv_heads);
  RL_REQUIRE(pages * kv_heads * (page / kv::BT) <= INT32_MAX, RL_ERR_ARGUMENT, "rl_kv_attention: %lld pages",
             (long long)pages);
  RL_REQUIRE(table_ld * page <= (1 << 30), RL_ERR_ARGUMENT, "rl_kv_attention: sequences of up to %lld tokens",
             (long long)(table_ld * page));
  if (T == 0 || B == 0) return RL_OK;
  RL_REQUIRE(q && q_start && o, RL_ERR_ARGUMENT, "rl_kv_attention: NULL pointer");
  RL_REQUIRE(aligned(q, 16) && q_st % 8 == 0 && q_sh % 8 == 0 && aligned(o, 2) && aligned(row_limit, 4), RL_ERR_ALIGNMENT,
             "rl_kv_attention: q must be 16-byte aligned, its strides multiples of 8");
  RL_REQUIRE(ldo >= static_cast<int64_t>(heads) * kv::HD, RL_ERR_ARGUMENT, "rl_kv_attention: ldo < heads * 128");
  const size_t need = rl_kv_attention_workspace(T, B, heads, kv_heads);
  RL_REQUIRE(workspace && workspace_bytes >= need, RL_ERR_ARGUMENT, "rl_kv_attention: workspace of %zu bytes, needs %zu",
             workspace_bytes, need);
  RL_REQUIRE(aligned(workspace, 16), RL_ERR_ALIGNMENT, "rl_kv_attention: the workspace must be 16-byte aligned");
  RL_REQUIRE(device_is_sm100(), RL_ERR_UNSUPPORTED, "rl_kv_attention: needs an sm_100 device");
  a.q = q, a.q_st = q_st, a.q_sh = q_sh;
  a.row_limit = row_limit, a.scale_log2 = scale_log2;
  a.o = o, a.ldo = ldo, a.group = heads / kv_heads;
  const int nt = kvattn::tile_n(T, B, a.group);
  a.part = static_cast<float*>(workspace);
  a.rec = reinterpret_cast<int4*>(static_cast<uint8_t*>(workspace) + kvattn::part_bytes(nt));
  switch (nt) {
    case 1: return kvattn::launch<1>(a, stream);
    case 2: return kvattn::launch<2>(a, stream);
    default: return kvattn::launch<4>(a, stream);
  }
}

}  // extern "C"
