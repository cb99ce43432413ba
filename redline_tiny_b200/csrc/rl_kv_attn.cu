// Attention of a few new tokens per sequence over the 8-bit paged cache (rl_kv.cu), head dim 128.
//
// o_r = sum_k p_rk v_k / sum_k p_rk, p_rk = 2^(s_rk - m_r), s_rk = scale_log2 * q_r . k_k over the keys k <= limit_r.
// With K = 2^(ek-133) mk per block of 16 tokens, s is an fp16 product q~ . mk (mk is an integer in [-128, 127], exact;
// q~ is q times a power of two per row that puts the row's largest value in [2^14, 2^15), exact for every value within
// 2^-28 of it) times one fp32 factor per block and row. P is rounded to fp16 (11 significant bits, half a step 2^-11
// of each weight; the row sum adds them unrounded). P . mv, again with exact integers, accumulates in fp32 in units of
// 2^(er-133), er the largest V exponent so far; a block's own scale 2^(ev-er) goes into its P. So the only roundings are
// P's and fp32's. A row keeps the er of the last block that it sees, so that no hidden key reaches it.
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
//
// Bound by the cache's bytes for one token a sequence: 269 MB (one sequence of 131071 tokens, 8 heads) in 54 us, of which
// the loop over the keys takes 35 - 46 us a CTA (7.6 - 5.8 TB/s), its start 4 and the joins 5; 564 MB (64 sequences of up
// to 8192) in 100 us = 5.7 TB/s. Steps, for the two: plain loads 114 / 166 us; copies through a per-warp ring 67 / 114; V
// scales in P and no 64-bit divisions 55 / 102. A step of 777 keys takes 5.6 us in one launch of clusters (7.0 in two
// launches): the launch, three dependent loads, a block or two a warp, the joins.
#include "rl_common.cuh"
#include "rl_host.h"

namespace rl {
namespace kvattn {

using kv::BT;
using kv::HD;

constexpr int UNIT = 64;         // keys per unit of work
constexpr float kRaise = 8.0f;   // the running maximum rises only when a score exceeds it by more (log2)
// P is kept times 2^kUp (<= 2^12). A V block whose scale is 2^-d of the unit of O lowers its P by 2^d, which costs a
// weight bits only below 2^(d - 18) of the largest; with d <= kWindow, below 2^-10, where they are off by 2^-21.
constexpr int kUp = 4;
constexpr uint32_t kWindow = 8;
constexpr float kNone = -1e30f;  // running maximum before any key (finite: no inf - inf)
// Pieces are joined in float, weights up to 2^12 and their sums included. A row whose unit is above 2^(kMostUnit - 133) is
// joined 2^x smaller, its sum too and its maximum x larger, which is the same piece: x = unit - kMostUnit.
constexpr int kMostUnit = 190;

// n / d for 0 <= n < 2^31 by a multiplication: mul = ceil(2^(31 + s) / d), s = ceil(log2 d); mul d exceeds
// 2^(31 + s) by e < d <= 2^s, so n e < 2^(31 + s) and the quotient is exact.
struct Div {
  uint32_t d, mul, sh;
  static Div of(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return Div{d, static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d), s};
  }
};
__device__ __forceinline__ uint32_t operator/(uint32_t n, const Div& v) {
  return static_cast<uint32_t>((static_cast<uint64_t>(n) * v.mul) >> 31) >> v.sh;
}

// What CTA i's task that it began and did not finish needs to be joined: its sequence's first row, the rows of a K/V
// head, the head, the tile, and the pieces (none: 0; negative: the first lies in the CTA's second slot).
struct Record {
  int s0, rows, h, tile, n, pad[3];
};

struct Args {
  const uint16_t* q;
  int64_t q_st, q_sh;
  kv::Pool pool;
  kv::Batch batch;
  const int32_t* row_limit;
  float scale_log2;
  uint16_t* o;
  int64_t ldo;
  Div group, hkv;                // query heads per K/V head, K/V heads
  int page_sh;                   // log2 of the page size
  int vec;                       // rows of o are 8-byte aligned
  float* part;                   // workspace: 2 slots per CTA of R x (128 + 2) floats
  Record* rec;                   // workspace: per CTA, the task it began and did not finish
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
__device__ __forceinline__ void mma_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
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
// (a plain load, which the compiler may place among the matrix instructions)
__device__ __forceinline__ uint4 lds128(const uint8_t* a) { return *reinterpret_cast<const uint4*>(a); }

// A row's q (the lane's dims 16c.. and 64 + 16c..) as fp16 times 2^(141 - e), which puts the row's largest value in
// [2^14, 2^15). Returns e, its exponent field.
__device__ __forceinline__ uint32_t q_fragments(const uint4 (&w)[4], uint32_t (&qf)[16]) {
  const uint32_t x[16] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w,
                          w[2].x, w[2].y, w[2].z, w[2].w, w[3].x, w[3].y, w[3].z, w[3].w};
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) mx = max(mx, max(x[i] & 0x7FFFu, x[i] >> 16 & 0x7FFFu));
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  const uint32_t e = max(mx >> 7, 32u);                              // (values below 2^-95 keep less)
  const float up = __uint_as_float((268u - e) << 23);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    qf[i] = pack_h2(__uint_as_float(x[i] << 16) * up, __uint_as_float(x[i] & 0xFFFF0000u) * up);
  return e;
}
// What the scores of row k (of the lanes that hold e) are multiplied by: 2^(e - 141) scale.
__device__ __forceinline__ float q_scale(uint32_t e, int row, float scale_log2) {
  const int er = __shfl_sync(0xffffffffu, static_cast<int>(e), row * 4);
  return __uint_as_float(static_cast<uint32_t>(er - 14) << 23) * scale_log2;
}

// The list of units: sequence b has hkv * tiles(b) tasks of chunks(b) units each.
__device__ __forceinline__ int64_t tiles_of(const Args& a, const kv::Seq& s, int R) {
  return (s.n * a.group.d + R - 1) / R;
}
__device__ __forceinline__ int64_t chunks_of(const kv::Seq& s) { return s.len > 0 ? (s.len + UNIT - 1) / UNIT : 1; }

// Prefix sums of the sequences' units (kTasks: of their tasks) into `pre` (B + 1 values), by the whole CTA.
template <int kWarps, bool kTasks>
__device__ __forceinline__ void unit_prefix(const Args& a, int R, int64_t* pre, int64_t* warp_sum, int4* seqs) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) pre[0] = 0;
  int64_t base = 0;
  for (int b0 = 0; b0 < a.batch.B; b0 += 32 * kWarps) {
    const int b = b0 + threadIdx.x;
    int64_t u = 0;
    if (b < a.batch.B) {
      const kv::Seq s = kv::load_seq(a.batch, b, a.pool.page);
      seqs[b] = make_int4(static_cast<int>(s.s0), static_cast<int>(s.n), static_cast<int>(s.len), 0);
      if (s.ok) u = tiles_of(a, s, R) * (kTasks ? 1 : chunks_of(s)) * a.hkv.d;
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

// floor(i U / C), in 32 bits where that holds the product.
__device__ __forceinline__ int64_t share(uint32_t i, int64_t U, int64_t C) {
  if (U < (1 << 20)) return i * static_cast<uint32_t>(U) / static_cast<uint32_t>(C);   // (a grid has fewer than 2^12 CTAs)
  return i * U / C;
}

template <int NT>
struct Acc {
  float o[NT][8][4];     // O^T: dims 16g + 2i (+1 for [2], [3]), rows 2c, 2c + 1 of n-tile nt
  float m[NT][2], l[NT][2];
  int er;                // the largest V exponent of the warp's blocks so far
  int unit[NT][2];       // O of a row is in units of 2^(unit - 133): er of the last block that the row sees
};

// P^T of a block times 2^shift, in the B layout; the row sums add the weights, before their rounding, times `unit`.
template <int NT>
__device__ __forceinline__ void weights(const float (&s)[NT][4], Acc<NT>& acc, float shift, float unit, uint32_t (&p)[NT][2]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float m0 = acc.m[nt][0] - shift, m1 = acc.m[nt][1] - shift;
    const float e0 = exp2_approx(s[nt][0] - m0), e1 = exp2_approx(s[nt][1] - m1);
    const float e2 = exp2_approx(s[nt][2] - m0), e3 = exp2_approx(s[nt][3] - m1);
    acc.l[nt][0] = fmaf(unit, e0 + e2, acc.l[nt][0]);
    acc.l[nt][1] = fmaf(unit, e1 + e3, acc.l[nt][1]);
    p[nt][0] = movmatrix(pack_h2(e0, e1));
    p[nt][1] = movmatrix(pack_h2(e2, e3));
  }
}

// The eight V^T fragments of a block (dims 16g + 2i, + 1), each handed to `f` for every n-tile.
template <int NT, typename F>
__device__ __forceinline__ void add_values(const uint4 (&vr)[4], F f) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t t0 = (&vr[0].x)[w], t1 = (&vr[1].x)[w], t2 = (&vr[2].x)[w], t3 = (&vr[3].x)[w];
#pragma unroll
    for (int hl = 0; hl < 2; ++hl) {
      const uint32_t x = __byte_perm(t0, t1, hl ? 0x7362 : 0x5140), y = __byte_perm(t2, t3, hl ? 0x7362 : 0x5140);
      const uint32_t a0 = codes_h2<0x4140>(x), a1 = codes_h2<0x4342>(x);
      const uint32_t a2 = codes_h2<0x4140>(y), a3 = codes_h2<0x4342>(y);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) f(2 * w + hl, a0, a1, a2, a3, nt);
    }
  }
}

// One warp, one block of 16 keys starting at position pos0.
template <int NT>
__device__ __forceinline__ void block_step(const uint4 (&kr)[4], const uint4 (&vr)[4], uint32_t ke, uint32_t ve,
                                           int pos0, const uint32_t (&qf)[16], const uint8_t* q_at, const float (&qs)[NT][2],
                                           const int (&lim)[NT][2], int lim_min, int g, Acc<NT>& acc) {
  float s[NT][4];
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
      if (jj == 0) mma_zero(s[nt], A[0][0], A[0][1], A[0][2], A[0][3], q.x, q.y);
      else mma(s[nt], A[0][0], A[0][1], A[0][2], A[0][3], q.x, q.y);
      mma(s[nt], A[1][0], A[1][1], A[1][2], A[1][3], q.z, q.w);
    }
  }
  const float ks = ke == 255u ? __uint_as_float(0x7FC00000u) : bfp16_scale(ke);
  // units of O: V blocks bring their scale in through P while it is within 2^kWindow of the unit
  const int ev = ve == 255u ? acc.er : static_cast<int>(ve);
  int d = acc.er - ev;
  uint32_t p[NT][2];
  bool change = static_cast<uint32_t>(d) > kWindow;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float f0 = ks * qs[nt][0], f1 = ks * qs[nt][1];
    s[nt][0] *= f0, s[nt][1] *= f1, s[nt][2] *= f0, s[nt][3] *= f1;
    if (pos0 + BT - 1 > lim_min) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (pos0 + g + 8 * (i >> 1) > lim[nt][i & 1]) s[nt][i] = -INFINITY;
    }
    change |= fmaxf(s[nt][0], s[nt][2]) > acc.m[nt][0] + kRaise || fmaxf(s[nt][1], s[nt][3]) > acc.m[nt][1] + kRaise;
  }
  if (__any_sync(0xffffffffu, change)) {
    // (a row that does not see this block, nor any behind it, keeps its unit: what is hidden may be 2^200 times its values)
    float to = 1.0f;
    if (ev > acc.er) {
      to = exp2f(static_cast<float>(acc.er - ev));
      acc.er = ev;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          acc.unit[nt][c] = pos0 <= lim[nt][c] ? ev : acc.unit[nt][c];
    }
    d = acc.er - ev;
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
        const float f = pos0 <= lim[nt][c] ? alpha * to : alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc.o[nt][i][c] *= f;
          acc.o[nt][i][c + 2] *= f;
        }
      }
    if (d > static_cast<int>(kWindow)) {
      // a block far below the unit (zeros, for one): its product is scaled as it is added, and the code below adds none
      const float vs = exp2f(static_cast<float>(-d));
      weights<NT>(s, acc, static_cast<float>(kUp), 1.0f, p);
      add_values<NT>(vr, [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, int nt) {
        float t[4];
        mma_zero(t, a0, a1, a2, a3, p[nt][0], p[nt][1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc.o[nt][i][j] = fmaf(vs, t[j], acc.o[nt][i][j]);
      });
      d = 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = -INFINITY;
    }
  }
  weights<NT>(s, acc, static_cast<float>(kUp - d), __uint_as_float(static_cast<uint32_t>(127 + d) << 23), p);
  add_values<NT>(vr, [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, int nt) {
    mma(acc.o[nt][i], a0, a1, a2, a3, p[nt][0], p[nt][1]);
  });
  if (ve == 255u) {   // a block with a NaN or an infinity: NaN for the rows that see it (the codes are small integers)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (pos0 <= lim[nt][c]) acc.l[nt][c] = __uint_as_float(0x7FC00000u);
  }
}

// O / l of one row as bf16, 4 dims a lane.
__device__ __forceinline__ void store_row(const Args& a, int64_t token, uint32_t head, int lane, const float4& o, float l) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* d = a.o + token * a.ldo + head * HD + 4 * lane;
  const float v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  if (a.vec) {
    uint2 w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w.x) : "f"(v[1]), "f"(v[0]));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w.y) : "f"(v[3]), "f"(v[2]));
    *reinterpret_cast<uint2*>(d) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = __bfloat16_as_ushort(__float2bfloat16_rn(v[i]));
  }
}

// Shared memory of a CTA: the ring that brings blocks in (per warp kStages x [K 2 KB | V 2 KB]), reused at the end of a
// run for the warps' results (kWarps x R x 128 floats), then their maxima and sums, then the unit prefix.
template <int NT>
struct Cfg {
  static constexpr int R = 8 * NT;
  // NT = 1: 4 CTAs of 4 warps hide each other's starts and ends of tasks. Medians on one box, 64 sequences of up to 8192
  // tokens (564 MB) / one of 131071 (269 MB): 4 x 4 warps 102 / 55 us, 2 x 8 116 / 51, 1 x 16 144 / 57; 2 stages instead
  // of 3 the same.
  static constexpr int kWarps = 4;
  static constexpr int kCtas = NT == 1 ? 4 : 2;                       // resident per SM
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kStages = NT == 1 ? 3 : 5;
  static constexpr int kRing = kWarps * kStages * 2 * BT * HD;
  static constexpr int kOut = kWarps * R * HD * 4;
  static constexpr int kJoined = R * (HD + 2) * 4;                    // the CTA's own piece, for its cluster
  static constexpr int kBody = kRing > kOut + kJoined ? kRing : kOut + kJoined;
  static constexpr int kQ = NT == 1 ? 0 : NT * 16 * 32 * 4;            // q fragments, where registers cannot hold them
  static size_t smem(int B) { return kBody + kQ + kWarps * R * 8 + B * 16 + (kWarps + B + 1) * 8; }
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float ld_cluster1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// kCluster: short contexts in one launch. A task is one cluster of eight CTAs, which share its keys evenly and join their
// pieces through distributed shared memory; otherwise units are spread over the grid and combine_kernel joins the pieces.
constexpr int kClusterCtas = 8;
template <int NT, bool kCluster>
__global__ void __launch_bounds__(Cfg<NT>::kThreads, Cfg<NT>::kCtas) attend_kernel(const Args a) {
  constexpr int R = 8 * NT, kWarps = Cfg<NT>::kWarps;
  constexpr int S = Cfg<NT>::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  float* so = reinterpret_cast<float*>(smem);                        // [warp][row][128]
  uint8_t* sq = smem + Cfg<NT>::kBody;                               // [n-tile][4][lane] x 16 bytes
  float* sm = reinterpret_cast<float*>(sq + Cfg<NT>::kQ);            // [warp][row] maxima
  float* sl = sm + kWarps * R;                                       // [warp][row] sums
  int4* seqs = reinterpret_cast<int4*>(sl + kWarps * R);              // first row, rows and length of each sequence
  int64_t* warp_sum = reinterpret_cast<int64_t*>(seqs + a.batch.B);
  int64_t* pre = warp_sum + kWarps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  unit_prefix<kWarps, kCluster>(a, R, pre, warp_sum, seqs);
  const int64_t U = pre[a.batch.B];
  int64_t C = 1, u, u_end;
  const int rank = blockIdx.x % kClusterCtas;
  if (kCluster) {
    u = blockIdx.x / kClusterCtas, u_end = u + 1;
    if (u >= U) return;                                              // (the whole cluster: the grid is an upper bound)
  } else {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    C = min(static_cast<int64_t>(gridDim.x), U);                    // every working CTA has at least one unit
    const bool idle = blockIdx.x >= C;
    u_end = idle ? 0 : share(blockIdx.x + 1, U, C);
    u = idle ? 0 : share(blockIdx.x, U, C);
  }
  bool first = true;
  Record rec = {};
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
    const int4 sq4 = seqs[b];
    const kv::Seq s{sq4.x, sq4.y, sq4.z, true};
    const int64_t nch = chunks_of(s), off = u - pre[b];
    uint32_t task;
    int64_t ch0, ch1;                                                // the run: chunks of 64 keys of the task
    if (kCluster) {
      task = static_cast<uint32_t>(off);
      ch0 = nch * rank / kClusterCtas, ch1 = nch * (rank + 1) / kClusterCtas;
    } else {
      task = static_cast<uint32_t>(off < (1ll << 31) ? static_cast<uint32_t>(off) / static_cast<uint32_t>(nch) : off / nch);
      ch0 = off - task * nch;
      ch1 = min(nch, ch0 + (u_end - u));
    }
    const uint32_t tile = task / a.hkv;
    const int h = static_cast<int>(task - tile * a.hkv.d);
    const uint32_t rows = static_cast<uint32_t>(s.n) * a.group.d;    // rows of this K/V head
    const uint32_t row0 = tile * R;

    uint32_t qf[16];
    float qs[NT][2];
    int lim[NT][2];
    int lim_min = INT32_MAX, lim_max = -1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t rr = row0 + nt * 8 + 2 * c + k;
        lim[nt][k] = INT32_MAX;                                      // rows behind the last: never stored, no reason to mask
        if (rr < rows) {
          const uint32_t j = rr / a.group;
          int64_t L = s.len - s.n + j;
          if (a.row_limit) L = min(s.len - 1, static_cast<int64_t>(__ldg(a.row_limit + s.s0 + j)));
          lim[nt][k] = static_cast<int>(max(L, static_cast<int64_t>(-1)));
          lim_max = max(lim_max, lim[nt][k]);
          lim_min = min(lim_min, lim[nt][k]);
        }
      }
    }
    lim_max = max(lim_max, __shfl_xor_sync(0xffffffffu, lim_max, 1));
    lim_max = max(lim_max, __shfl_xor_sync(0xffffffffu, lim_max, 2));
    lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 1));
    lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 2));

    // q of the rows this lane loads: asked for before the copies fill the memory system's queues
    uint4 qw[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t r = row0 + nt * 8 + g;
#pragma unroll
      for (int i = 0; i < 4; ++i) qw[nt][i] = make_uint4(0, 0, 0, 0);
      if (r < rows) {
        const uint32_t j = r / a.group;
        const uint16_t* p = a.q + (s.s0 + j) * a.q_st + (h * a.group.d + r - j * a.group.d) * a.q_sh + 16 * c;
#pragma unroll
        for (int i = 0; i < 4; ++i) qw[nt][i] = *reinterpret_cast<const uint4*>(p + 64 * (i >> 1) + 8 * (i & 1));
      }
    }

    // the warp's blocks: every kWarps-th of the run. Lane j holds the pool index of block 32 t + j, one chunk ahead.
    const int64_t key_end = min(ch1 * UNIT, static_cast<int64_t>(lim_max) + 1);
    const int64_t pos0 = ch0 * UNIT + warp * BT;
    const int n = key_end > pos0 ? static_cast<int>((key_end - pos0 + kWarps * BT - 1) / (kWarps * BT)) : 0;
    const int32_t* table = a.batch.table + b * a.batch.ld;
    auto page_of = [&](int k) -> int {                               // (a plain load: nothing waits for it here)
      return k < n ? __ldg(table + ((static_cast<uint32_t>(pos0) + k * (kWarps * BT)) >> a.page_sh)) : 0;
    };
    auto block_in = [&](int pg, int k) -> int {
      if (k >= n) return -1;
      if (static_cast<uint32_t>(pg) >= a.pool.pages) {               // a page outside the pool: its keys are absent
        report(kErrBadArgument);
        return -1;
      }
      const uint32_t pos = static_cast<uint32_t>(pos0) + k * (kWarps * BT);
      return ((pg * a.pool.hkv + h) << (a.page_sh - 4)) + ((pos & (a.pool.page - 1)) >> 4);
    };
    const int page0 = page_of(lane);
    int page_next = page_of(32 + lane), idx = block_in(page0, lane);
    uint32_t ke[S], ve[S];                                           // of the ring's blocks
    int at_pos[S];                                                   // first position, or beyond every limit
    auto issue = [&](int k, int j) {
      if (k < n) {
        if ((k & 31) == 0 && k > 0) {
          idx = block_in(page_next, k + lane);
          page_next = page_of(k + 32 + lane);
        }
        const int found = __shfl_sync(0xffffffffu, idx, k & 31);
        // an absent block reads as block 0, fully masked, with an exponent (255) that moves no unit
        const int64_t blk = max(found, 0);
        at_pos[j] = found < 0 ? 0x7FFFFF00 : static_cast<int>(pos0) + k * (kWarps * BT);
        ke[j] = a.pool.ke[blk], ve[j] = 255u;
        if (found >= 0) ve[j] = a.pool.ve[blk];
        const uint8_t* kp = a.pool.k + blk * (BT * HD) + lane * 16;
        const uint8_t* vp = a.pool.v + blk * (BT * HD) + lane * 16;
        const uint32_t d = ring + j * (2 * BT * HD) + wr * HD;
#pragma unroll
        for (int i = 0; i < 4; ++i) cp_async16(d + i * 4 * HD + ((wc ^ ((wr & 1) * 4)) << 4), kp + i * 512);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          cp_async16(d + BT * HD + i * 4 * HD + ((wc ^ ((((wr + 4 * i) >> 1) & 3) * 2)) << 4), vp + i * 512);
      }
      cp_commit();
    };
#pragma unroll
    for (int k = 0; k < S - 1; ++k) issue(k, k);

    // q of the tile, while the first blocks are on their way
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t e = q_fragments(qw[nt], qf);
      if (NT > 1 && nt % kWarps == warp) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          reinterpret_cast<uint4*>(sq)[(nt * 4 + i) * 32 + lane] =
              make_uint4(qf[4 * i], qf[4 * i + 1], qf[4 * i + 2], qf[4 * i + 3]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) qs[nt][k] = q_scale(e, 2 * c + k, a.scale_log2);
    }

    if (NT > 1) __syncthreads();
    const uint8_t* q_at = sq + lane * 16;

    Acc<NT> acc;
    acc.er = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc.unit[nt][0] = acc.unit[nt][1] = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      acc.m[nt][0] = acc.m[nt][1] = kNone;
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
          issue(i + S - 1, (j + S - 1) % S);
          const uint8_t* at = smem + warp * (S * 2 * BT * HD) + j * (2 * BT * HD);
          uint4 kr[4], vr[4];
          kr[0] = lds128(at + k_ld), kr[1] = lds128(at + (k_ld ^ 64));
          kr[2] = lds128(at + k_ld + 8 * HD), kr[3] = lds128(at + (k_ld ^ 64) + 8 * HD);
          vr[0] = lds128(at + v_ld), vr[1] = lds128(at + v_ld + HD);
          vr[2] = lds128(at + v_ld + 8 * HD), vr[3] = lds128(at + v_ld + 9 * HD);
          block_step<NT>(kr, vr, ke[j], ve[j], at_pos[j], qf, q_at, qs, lim, lim_min, g, acc);
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
        const int unit = acc.unit[nt][k], over = max(unit - kMostUnit, 0);
        const float ou = bfp16_scale(static_cast<uint32_t>(unit - over));
        float m = acc.m[nt][k];
        if (over) l *= __uint_as_float(static_cast<uint32_t>(127 - over) << 23), m += static_cast<float>(over);
        if (g == 0) sm[warp * R + row] = m, sl[warp * R + row] = l;
        float* d = so + (warp * R + row) * HD + 16 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          reinterpret_cast<float4*>(d)[i] = make_float4(acc.o[nt][2 * i][k] * ou, acc.o[nt][2 * i][k + 2] * ou,
                                                        acc.o[nt][2 * i + 1][k] * ou, acc.o[nt][2 * i + 1][k + 2] * ou);
      }
    __syncthreads();
    const bool whole = !kCluster && ch0 == 0 && ch1 == nch;
    float* part = kCluster ? reinterpret_cast<float*>(smem + Cfg<NT>::kOut)
                           : a.part + (static_cast<int64_t>(blockIdx.x) * 2 + (first ? 0 : 1)) * R * (HD + 2);
    // a warp per row, 4 dims a lane
#pragma unroll 2
    for (int row = warp; row < R; row += kWarps) {
      const uint32_t r = row0 + row, j = r / a.group;
      if (r >= rows) break;
      float mw[kWarps], m = kNone;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mw[w] = sm[w * R + row], m = fmaxf(m, mw[w]);
      float l = 0.0f;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2_approx(mw[w] - m);
        const float4 v = reinterpret_cast<const float4*>(so + (w * R + row) * HD)[lane];
        l = fmaf(f, sl[w * R + row], l);
        o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
      }
      if (whole) {
        store_row(a, s.s0 + j, h * a.group.d + r - j * a.group.d, lane, o, l);
      } else {
        reinterpret_cast<float4*>(part + row * HD)[lane] = o;
        if (lane == 0) part[R * HD + row] = m, part[R * HD + R + row] = l;
      }
    }
    if (kCluster) {
      cluster_sync();
      for (int i = warp; i < NT; i += kWarps) {                      // this CTA joins every eighth row
        const int row = rank + kClusterCtas * i;
        const uint32_t r = row0 + row, j = r / a.group;
        if (r >= rows) break;
        const uint32_t at = smem_u32(part);
        float mj[kClusterCtas], lj[kClusterCtas], m = kNone, l = 0.0f;
        float4 v[kClusterCtas], o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kClusterCtas; ++k) {
          const uint32_t remote = mapa_shared(at, k);
          v[k] = ld_cluster4(remote + (row * HD + 4 * lane) * 4);
          mj[k] = ld_cluster1(remote + (R * HD + row) * 4), lj[k] = ld_cluster1(remote + (R * HD + R + row) * 4);
        }
#pragma unroll
        for (int k = 0; k < kClusterCtas; ++k) m = fmaxf(m, mj[k]);
#pragma unroll
        for (int k = 0; k < kClusterCtas; ++k) {
          const float f = exp2_approx(mj[k] - m);
          l = fmaf(f, lj[k], l);
          o.x = fmaf(f, v[k].x, o.x), o.y = fmaf(f, v[k].y, o.y), o.z = fmaf(f, v[k].z, o.z), o.w = fmaf(f, v[k].w, o.w);
        }
        store_row(a, s.s0 + j, h * a.group.d + r - j * a.group.d, lane, o, l);
      }
      cluster_sync();                                                // no CTA leaves while its piece is read
      return;
    }
    if (!whole && ch0 == 0) {
      // the pieces end in the CTA that holds the task's last unit x: floor(j U / C) <= x < floor((j + 1) U / C)
      const int64_t x = u + nch - 1;
      const int pieces = static_cast<int>(((x + 1) * C - 1) / U - blockIdx.x) + 1;
      rec = Record{static_cast<int>(s.s0), static_cast<int>(rows), h, static_cast<int>(tile), first ? pieces : -pieces, {}};
    }
    u += ch1 - ch0;
    first = false;
    __syncthreads();
  }
  if (threadIdx.x == 0) a.rec[blockIdx.x] = rec;
}

// CTA i joins the pieces of the task that CTA i of attend_kernel began and did not finish: kJoin / 8 warps to a row, each
// a share of the pieces with a running maximum (all loads independent of it), then the shares in order. Launched while
// attend_kernel still runs, it waits for that grid's end.
constexpr int kJoin = 16;   // warps
template <int NT>
__global__ void __launch_bounds__(32 * kJoin) combine_kernel(const Args a) {
  constexpr int R = 8 * NT;
  constexpr int64_t kSlot = R * (HD + 2);
  constexpr int kShares = kJoin / 8;
  __shared__ float4 so[kShares][8][32];
  __shared__ float2 sml[kShares][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Record rec = a.rec[blockIdx.x];
  if (rec.n == 0) return;
  const int pieces = abs(rec.n);
  // piece 0 may lie in the CTA's second slot; the others in the first slots of the CTAs behind
  const float* base = a.part + static_cast<int64_t>(blockIdx.x) * 2 * kSlot;
  const int share = warp >> 3;
  for (int row0 = 0; row0 < R; row0 += 8) {
    const int row = row0 + (warp & 7);
    const uint32_t r = static_cast<uint32_t>(rec.tile) * R + row;
    float m = kNone, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < static_cast<uint32_t>(rec.rows)) {
      for (int j0 = share; j0 < pieces; j0 += 8 * kShares) {
        float4 v[8];
        float mj[8], lj[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {       // eight pieces on their way at once
          const int j = j0 + i * kShares;
          v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f), mj[i] = kNone, lj[i] = 0.0f;
          if (j < pieces) {
            const float* p = base + (j == 0 ? (rec.n < 0 ? kSlot : 0) : j * 2 * kSlot);
            v[i] = __ldcg(reinterpret_cast<const float4*>(p + row * HD) + lane);
            mj[i] = __ldcg(p + R * HD + row), lj[i] = __ldcg(p + R * HD + R + row);
          }
        }
        float mn = m;
#pragma unroll
        for (int i = 0; i < 8; ++i) mn = fmaxf(mn, mj[i]);
        const float fa = exp2_approx(m - mn);
        m = mn;
        l *= fa, o.x *= fa, o.y *= fa, o.z *= fa, o.w *= fa;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = exp2_approx(mj[i] - mn);
          l = fmaf(f, lj[i], l);
          o.x = fmaf(f, v[i].x, o.x), o.y = fmaf(f, v[i].y, o.y), o.z = fmaf(f, v[i].z, o.z), o.w = fmaf(f, v[i].w, o.w);
        }
      }
    }
    if (share > 0) {
      so[share][warp & 7][lane] = o;
      if (lane == 0) sml[share][warp & 7] = make_float2(m, l);
    }
    __syncthreads();
    if (share == 0 && r < static_cast<uint32_t>(rec.rows)) {
#pragma unroll
      for (int j = 1; j < kShares; ++j) {
        const float4 v = so[j][warp][lane];
        const float2 ml = sml[j][warp];
        const float mn = fmaxf(m, ml.x);
        const float fa = exp2_approx(m - mn), fb = exp2_approx(ml.x - mn);
        m = mn;
        l = fmaf(fb, ml.y, l * fa);
        o.x = fmaf(fb, v.x, o.x * fa), o.y = fmaf(fb, v.y, o.y * fa);
        o.z = fmaf(fb, v.z, o.z * fa), o.w = fmaf(fb, v.w, o.w * fa);
      }
      const uint32_t jr = r / a.group;
      store_row(a, rec.s0 + jr, rec.h * a.group.d + r - jr * a.group.d, lane, o, l);
    }
    __syncthreads();
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

// Clusters of the one-launch form: at most this many tasks, whatever the batch holds.
inline int64_t tasks_of(int nt, int64_t T, int B, int group, int hkv) { return (T * group / (8 * nt) + B) * hkv; }

template <int NT>
inline int launch_cluster(const Args& a, int64_t tasks, cudaStream_t st) {
  static PerDevice ready;
  RL_TRY_CUDA(ready.once([] {
    return cudaFuncSetAttribute(attend_kernel<NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(Cfg<NT>::smem(kv::kMaxBatch)));
  }));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tasks * kClusterCtas));
  cfg.blockDim = dim3(Cfg<NT>::kThreads);
  cfg.dynamicSmemBytes = Cfg<NT>::smem(a.batch.B);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = kClusterCtas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  RL_TRY_CUDA(cudaLaunchKernelEx(&cfg, attend_kernel<NT, true>, a));
  return RL_OK;
}

template <int NT>
inline int launch(const Args& a, cudaStream_t st) {
  const size_t smem = Cfg<NT>::smem(a.batch.B);
  const int ctas = ctas_of(NT);
  static PerDevice ready;
  RL_TRY_CUDA(ready.once([] {
    return cudaFuncSetAttribute(attend_kernel<NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(Cfg<NT>::smem(kv::kMaxBatch)));
  }));
  attend_kernel<NT, false><<<ctas, Cfg<NT>::kThreads, smem, st>>>(a);
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
