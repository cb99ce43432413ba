// The 8-bit paged cache of keys and values: writing new tokens, reading positions back, copying pages.
//
// A page holds `page` tokens (16, 32, 64, 128 or 256) of every K/V head of one layer: codes [Hkv][page][128] and one
// exponent byte per block of 16 tokens and head, [Hkv][page / 16]. A block is the bfp16 format with 16 x 128 values
// instead of 8: value = (u - 128) * 2^(E - 133), u = m + 128 in offset binary (as the native weight tiles), E the
// largest float32 exponent field in the block. The scale is a power of two because then every decoded value is exact
// in bf16 (8 significant bits), and a block whose later tokens need a larger E is rewritten by a shift. E = 255 marks
// a block that took in a NaN or an infinity; it reads as NaN.
//
// The kernels are bound by bytes where they are large: page copies 6.7 TB/s read and written (203 pages of 36 layers, 1.9 GB,
// 285 us); 8321 tokens of 8 heads written in 12.2 us (51 MB, 4.2 TB/s; a start of four dependent loads is 3 of them) and
// 3007 positions of four sequences read back in 13.8 us (49 MB written). K and V in another layout than rows of bf16 at 16-byte
// boundaries go by 2-byte loads, both of them: with V transposed, as the decoder layers hand it over, 49 us for the same tokens,
// 13.4 against 4.5 for 2048, 3.7 against 2.4 for one.
#include <cstdlib>

#include "rl_common.cuh"
#include "rl_host.h"

namespace rl {
namespace kv {

constexpr int HD = 128;     // head dim
constexpr int BT = 16;      // tokens per block (one exponent)
constexpr int kMaxBatch = 1024;

struct Pool {               // one layer
  uint8_t *k, *v, *ke, *ve;
  int64_t pages;
  int hkv, page;
};

struct Batch {
  const int32_t* table;     // (B, ld): page of each `page` tokens of each sequence
  int64_t ld;
  const int32_t* kv_len;    // (B): tokens in the cache, the new ones included
  const int32_t* q_start;   // (B + 1): rows of the new tokens
  int B;
  int64_t T;                // rows
};

// One sequence of a batch, checked against the sizes that the host knows. An impossible one is reported and dropped.
struct Seq {
  int64_t s0, n, len;
  bool ok;
};
__device__ __forceinline__ Seq load_seq(const Batch& bt, int b, int page) {
  Seq s;
  s.s0 = __ldg(bt.q_start + b);
  s.n = __ldg(bt.q_start + b + 1) - s.s0;
  s.len = __ldg(bt.kv_len + b);
  s.ok = s.s0 >= 0 && s.n >= 0 && s.s0 + s.n <= bt.T && s.len >= s.n && s.len <= bt.ld * page;
  return s;
}

// Index of the block (layer-wide) that holds token position `pos` of sequence b for head h, or -1 for a bad page.
__device__ __forceinline__ int64_t block_index(const Pool& p, const Batch& bt, int b, int64_t pos, int h) {
  const int sh = 31 - __clz(p.page);                                 // the page size is a power of two
  const int64_t pg = __ldg(bt.table + b * bt.ld + (pos >> sh));
  if (pg < 0 || pg >= p.pages) return -1;
  return ((pg * p.hkv + h) << (sh - 4)) + ((pos & (p.page - 1)) >> 4);
}

// m / 2^d for a code of an older token, rounded half to even (d >= 1), as an offset-binary byte.
__device__ __forceinline__ uint32_t shift_code(uint32_t u, int d) {
  const int m = static_cast<int>(u) - 128;
  if (d >= 9) return 128u;
  return static_cast<uint32_t>(((m + (1 << (d - 1)) - 1 + ((m >> d) & 1)) >> d) + 128);
}

// Codes of four new values (float32 bits) under exponent E: min(rint_half_even(x 2^(133 - E)), 127) + 128 as bytes. E is
// no smaller than the values' own exponent fields, so |x 2^(133 - E)| < 128 and only + 128 has to be clipped. The rounding is
// one FMA against 1.5 * 2^23, whose low byte is then the code but for its top bit; exponents near the ends of the range
// take the integer form.
__device__ __forceinline__ uint32_t codes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t E) {
  if (E >= 7u && E < 255u) {
    constexpr float kMagic = 12582912.0f;
    const float s = __uint_as_float((260u - E) << 23);
    auto q = [&](uint32_t x) { return __float_as_uint(fminf(fmaf(__uint_as_float(x), s, kMagic), kMagic + 127.0f)); };
    return __byte_perm(__byte_perm(q(a), q(b), 0x0040), __byte_perm(q(c), q(d), 0x0040), 0x5410) ^ 0x80808080u;
  }
  auto q = [&](uint32_t x) { return static_cast<uint32_t>(bfp16_quant_one(x, E) + 128); };
  return q(a) | q(b) << 8 | q(c) << 16 | q(d) << 24;
}

struct Source {             // rows of new keys or values: element (t, h, d) at t * st + h * sh + d * sd
  const void* x;
  int64_t st, sh, sd;
};

// The new values of a block in a warp's registers: up to 16 tokens x 128 dims.
//
// Any type and strides: lane l holds dims 4 l .. + 3 of every token, as float32 bits.
template <typename X>
struct AnyBlock {
  uint32_t x[BT][4];
  __device__ __forceinline__ void load(const Source& s, int64_t t0, int cnt, int h, int lane) {
    const bool vec = s.sd == 1 && ((reinterpret_cast<uintptr_t>(s.x) | (s.st * sizeof(X)) | (s.sh * sizeof(X))) &
                                   (4 * sizeof(X) - 1)) == 0;
    const X* p0 = static_cast<const X*>(s.x) + t0 * s.st + h * s.sh + 4 * lane * s.sd;
#pragma unroll
    for (int t = 0; t < BT; ++t) {
      x[t][0] = x[t][1] = x[t][2] = x[t][3] = 0u;
      if (t >= cnt) continue;
      const X* p = p0 + t * s.st;
      if (sizeof(X) == 2) {
        if (vec) {
          const uint2 w = *reinterpret_cast<const uint2*>(p);
          x[t][0] = w.x << 16, x[t][1] = w.x & 0xFFFF0000u, x[t][2] = w.y << 16, x[t][3] = w.y & 0xFFFF0000u;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[t][i] = static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + i * s.sd)) << 16;
        }
      } else {
        if (vec) {
          const uint4 w = *reinterpret_cast<const uint4*>(p);
          x[t][0] = w.x, x[t][1] = w.y, x[t][2] = w.z, x[t][3] = w.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[t][i] = *reinterpret_cast<const uint32_t*>(p + i * s.sd);
        }
      }
    }
  }
  __device__ __forceinline__ uint32_t exponent() const {
    uint32_t mx = 0;
#pragma unroll
    for (int t = 0; t < BT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = max(mx, x[t][i] & 0x7FFFFFFFu);
    return __reduce_max_sync(0xffffffffu, mx) >> 23;
  }
  __device__ __forceinline__ void store(uint8_t* row, int cnt, uint32_t E, int lane) const {
    uint32_t* p = reinterpret_cast<uint32_t*>(row) + lane;
#pragma unroll
    for (int t = 0; t < BT; ++t)
      if (t < cnt) p[t * (HD / 4)] = codes4(x[t][0], x[t][1], x[t][2], x[t][3], E);
  }
};

// bf16 rows at 16-byte boundaries: lanes 0 - 15 hold the even tokens and 16 - 31 the odd ones, 8 dims each. Half the
// registers of the form above and loads of 16 bytes: 26.4 -> 12.6 us for 8321 tokens of 8 heads.
struct WideBlock {
  uint4 x[BT / 2];
  __device__ __forceinline__ void load(const Source& s, int64_t t0, int cnt, int h, int lane) {
    const uint16_t* p = static_cast<const uint16_t*>(s.x) + (t0 + (lane >> 4)) * s.st + h * s.sh + 8 * (lane & 15);
#pragma unroll
    for (int t = 0; t < BT / 2; ++t) {
      x[t] = make_uint4(0, 0, 0, 0);
      if (2 * t + (lane >> 4) < cnt) x[t] = __ldcs(reinterpret_cast<const uint4*>(p + 2 * t * s.st));
    }
  }
  __device__ __forceinline__ uint32_t exponent() const {
    uint32_t m = 0;                                         // two 16-bit maxima
#pragma unroll
    for (int t = 0; t < BT / 2; ++t) {
      m = __vmaxu2(m, x[t].x & 0x7FFF7FFFu), m = __vmaxu2(m, x[t].y & 0x7FFF7FFFu);
      m = __vmaxu2(m, x[t].z & 0x7FFF7FFFu), m = __vmaxu2(m, x[t].w & 0x7FFF7FFFu);
    }
    return __reduce_max_sync(0xffffffffu, max(m & 0xFFFFu, m >> 16)) >> 7;
  }
  __device__ __forceinline__ void store(uint8_t* row, int cnt, uint32_t E, int lane) const {
    uint2* p = reinterpret_cast<uint2*>(row + (lane >> 4) * HD) + (lane & 15);
#pragma unroll
    for (int t = 0; t < BT / 2; ++t)
      if (2 * t + (lane >> 4) < cnt)
        p[t * (2 * HD / 8)] = make_uint2(codes4(x[t].x << 16, x[t].x & 0xFFFF0000u, x[t].y << 16, x[t].y & 0xFFFF0000u, E),
                                         codes4(x[t].z << 16, x[t].z & 0xFFFF0000u, x[t].w << 16, x[t].w & 0xFFFF0000u, E));
  }
};

// One warp per (group of `rows` rows, head, K or V). A row leads when it is the first of its block among the new
// tokens; the warp writes the blocks of its leading rows: the block's new values are read once into registers, their
// largest exponent field is joined with the exponent of the older tokens of the block, and the codes are stored. The last
// CTA reports impossible sequences, whichever rows they claim.
template <typename Block>
__global__ void __launch_bounds__(128) append_kernel(const Source sk, const Source sv, const Pool p, const Batch bt,
                                                     int rows, int64_t groups) {
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == gridDim.x - 1) {
    for (int b = threadIdx.x; b < bt.B; b += blockDim.x)
      if (!load_seq(bt, b, p.page).ok) report(kErrBadArgument);
    return;
  }
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (w >= groups * p.hkv * 2) return;
  const int is_v = static_cast<int>(w & 1);
  const int h = static_cast<int>((w >> 1) % p.hkv);
  const int64_t r0 = (w >> 1) / p.hkv * rows;
  const Source src = is_v ? sv : sk;
  uint8_t* codes = is_v ? p.v : p.k;
  uint8_t* exps = is_v ? p.ve : p.ke;
  // the sequence of row r0: the last b with q_start[b] <= r0
  int lo = 0, hi = bt.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(bt.q_start + mid) <= r0) lo = mid; else hi = mid;
  }
  int b = lo;
  Seq s = load_seq(bt, b, p.page);
  for (int64_t r = r0; r < min(r0 + rows, bt.T);) {
    while (b + 1 < bt.B && r >= s.s0 + s.n) s = load_seq(bt, ++b, p.page);
    if (r < s.s0 || r >= s.s0 + s.n) { ++r; continue; }   // a row of no sequence
    if (!s.ok) {
      r = s.s0 + s.n;
      continue;
    }
    const int64_t pos = s.len - s.n + (r - s.s0);
    const int a = static_cast<int>(pos % BT);             // place of row r in its block
    if (a != 0 && r != s.s0) {                            // led by an earlier row
      r = min(r + BT - a, s.s0 + s.n);
      continue;
    }
    const int cnt = static_cast<int>(min(static_cast<int64_t>(BT - a), s.s0 + s.n - r));
    Block x;
    x.load(src, r, cnt, h, lane);
    const int64_t blk = block_index(p, bt, b, pos, h);
    if (blk < 0) {
      if (lane == 0) report(kErrBadArgument);
      r += cnt;
      continue;
    }
    uint32_t E = x.exponent();
    uint8_t* row = codes + blk * (BT * HD);
    if (a > 0) {
      const uint32_t Eo = exps[blk];
      if (Eo >= E) {
        E = Eo;
      } else {
        const int d = static_cast<int>(E - Eo);
        uint32_t* old = reinterpret_cast<uint32_t*>(row) + lane;
        for (int t = 0; t < a; ++t) {
          const uint32_t u = old[t * (HD / 4)];
          old[t * (HD / 4)] = shift_code(u & 255u, d) | (shift_code(u >> 8 & 255u, d) << 8) |
                              (shift_code(u >> 16 & 255u, d) << 16) | (shift_code(u >> 24, d) << 24);
        }
      }
      __syncwarp();   // every lane has read the exponent before lane 0 replaces it
    }
    x.store(row + a * HD, cnt, E, lane);
    if (lane == 0) exps[blk] = static_cast<uint8_t>(E);
    r += cnt;
  }
}

// Two 16-byte stores of decoded values per 16 codes.
__device__ __forceinline__ void decode16(const uint4& u, uint32_t e, uint16_t* out) {
  uint32_t w[2][4];
  bfp16_decode_block_ob(e, u.x, u.y, w[0]);
  bfp16_decode_block_ob(e, u.z, u.w, w[1]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool nan = e == 255u;
    __stcs(reinterpret_cast<uint4*>(out) + i, nan ? make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u)
                                                  : make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]));
  }
}

// One thread per 16 values of the output (B, count, Hkv, 128), blockIdx.y = the sequence: token start[b] + i of sequence
// b, zero at and after its length (and on a bad page, which is reported).
__global__ void __launch_bounds__(256) read_kernel(const Pool p, const int32_t* table, int64_t ld, const int32_t* kv_len,
                                                   const int32_t* start, uint32_t count, uint16_t* ko, uint16_t* vo) {
  const int b = blockIdx.y;
  const uint32_t per = count * p.hkv * (HD / 16);
  const int64_t base = static_cast<int64_t>(b) * per;
  const int64_t first = __ldg(start + b), len = __ldg(kv_len + b);
  const Batch bt{table, ld, kv_len, nullptr, 0, 0};
  for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < per; i += gridDim.x * blockDim.x) {
    const uint32_t c = i % (HD / 16), th = i / (HD / 16), tok = th / p.hkv;
    const int h = static_cast<int>(th - tok * p.hkv);
    const int64_t pos = first + tok;
    uint16_t* k = ko + (base + i) * 16;
    uint16_t* v = vo + (base + i) * 16;
    const bool in = pos >= 0 && pos < len;
    const int64_t blk = in && pos < ld * p.page ? block_index(p, bt, b, pos, h) : -1;
    if (in && blk < 0) report(kErrBadArgument);
    if (blk < 0) {
      const uint4 z = make_uint4(0, 0, 0, 0);
      __stcs(reinterpret_cast<uint4*>(k), z), __stcs(reinterpret_cast<uint4*>(k) + 1, z);
      __stcs(reinterpret_cast<uint4*>(v), z), __stcs(reinterpret_cast<uint4*>(v) + 1, z);
    } else {
      const int64_t off = blk * (BT * HD) + (pos % BT) * HD + c * 16;
      const uint4 uk = *reinterpret_cast<const uint4*>(p.k + off), uv = *reinterpret_cast<const uint4*>(p.v + off);
      decode16(uk, p.ke[blk], k);
      decode16(uv, p.ve[blk], v);
    }
  }
}

// Page pairs travel as a kernel argument: no host-to-device copy, and nothing that the caller has to keep alive.
template <int N>
struct Pairs {
  int32_t src[N], dst[N];
};

constexpr int kPiece = 16384;   // bytes of a page that one CTA copies: 256 threads x 4 loads of 16 bytes in flight

template <int N>
__global__ void __launch_bounds__(256) copy_kernel(const Pool p, int64_t layer_codes, int64_t layer_exps,
                                                   const __grid_constant__ Pairs<N> pairs) {
  const int64_t bytes = static_cast<int64_t>(p.hkv) * p.page * HD;
  const int ne = p.hkv * p.page / BT;
  const int piece = blockIdx.x >> 1;
  const bool is_v = blockIdx.x & 1;
  const int64_t src = pairs.src[blockIdx.y], dst = pairs.dst[blockIdx.y];
  uint8_t* codes = (is_v ? p.v : p.k) + blockIdx.z * layer_codes;
  const uint4* s = reinterpret_cast<const uint4*>(codes + src * bytes);
  uint4* d = reinterpret_cast<uint4*>(codes + dst * bytes);
  const int64_t n16 = bytes / 16;
  uint4 r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t i = static_cast<int64_t>(piece) * (kPiece / 16) + j * 256 + threadIdx.x;
    if (i < n16) r[j] = __ldcs(s + i);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t i = static_cast<int64_t>(piece) * (kPiece / 16) + j * 256 + threadIdx.x;
    if (i < n16) __stcs(d + i, r[j]);
  }
  if (piece == 0) {
    uint8_t* e = (is_v ? p.ve : p.ke) + blockIdx.z * layer_exps;
    for (int i = threadIdx.x; i < ne; i += 256) e[dst * ne + i] = e[src * ne + i];
  }
}

// dst[at[i]] = value[i]: page tables and lengths follow the host's bookkeeping without a host-to-device copy, whose source
// the caller would have to keep unchanged until it ran.
template <int N>
__global__ void __launch_bounds__(N < 1024 ? N : 1024) set_kernel(int32_t* dst, int n, const __grid_constant__ Pairs<N> p) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) dst[p.src[i]] = p.dst[i];
}

inline int check_pool(const char* fn, const Pool& p) {
  RL_REQUIRE(p.k && p.v && p.ke && p.ve, RL_ERR_ARGUMENT, "%s: NULL pool pointer", fn);
  RL_REQUIRE(p.hkv > 0 && p.hkv <= 65535 && p.pages > 0 && p.pages <= INT32_MAX, RL_ERR_ARGUMENT,
             "%s: need kv_heads >= 1 and 1 <= pages < 2^31", fn);
  RL_REQUIRE(p.page == 16 || p.page == 32 || p.page == 64 || p.page == 128 || p.page == 256, RL_ERR_ARGUMENT,
             "%s: page size %d (16, 32, 64, 128 or 256 tokens)", fn, p.page);
  RL_REQUIRE(aligned(p.k, 16) && aligned(p.v, 16), RL_ERR_ALIGNMENT, "%s: the pool must be 16-byte aligned", fn);
  return RL_OK;
}

inline int check_batch(const char* fn, const Batch& bt) {
  RL_REQUIRE(bt.table && bt.kv_len, RL_ERR_ARGUMENT, "%s: NULL table or kv_len", fn);
  RL_REQUIRE(bt.B >= 0 && bt.B <= kMaxBatch, RL_ERR_ARGUMENT, "%s: %d sequences (at most %d)", fn, bt.B, kMaxBatch);
  RL_REQUIRE(bt.ld > 0 && bt.ld <= (1 << 24), RL_ERR_ARGUMENT, "%s: page table of %lld columns", fn, (long long)bt.ld);
  RL_REQUIRE(bt.T >= 0 && bt.T <= (1 << 24), RL_ERR_ARGUMENT, "%s: %lld rows", fn, (long long)bt.T);
  RL_REQUIRE(aligned(bt.table, 4) && aligned(bt.kv_len, 4) && aligned(bt.q_start, 4), RL_ERR_ALIGNMENT,
             "%s: int32 arrays must be 4-byte aligned", fn);
  return RL_OK;
}

template <int N>
inline int copy_launch(const Pool& p, int layers, int64_t lc, int64_t le, const int32_t* src, const int32_t* dst, int n,
                       cudaStream_t s) {
  Pairs<N> a;
  for (int i = 0; i < N; ++i) a.src[i] = i < n ? src[i] : 0, a.dst[i] = i < n ? dst[i] : 0;
  const int64_t bytes = static_cast<int64_t>(p.hkv) * p.page * HD;
  const dim3 grid(static_cast<unsigned>((bytes + kPiece - 1) / kPiece * 2), static_cast<unsigned>(n),
                  static_cast<unsigned>(layers));
  copy_kernel<N><<<grid, 256, 0, s>>>(p, lc, le, a);
  RL_TRY_CUDA(cudaGetLastError());
  return RL_OK;
}

}  // namespace kv
}  // namespace rl

extern "C" {

int rl_kv_append(const void* k, int64_t k_st, int64_t k_sh, int64_t k_sd, const void* v, int64_t v_st, int64_t v_sh,
                 int64_t v_sd, int dtype, int64_t T, uint8_t* pool_k, uint8_t* pool_v, uint8_t* pool_ke,
                 uint8_t* pool_ve, int64_t pages, int kv_heads, int page, const int32_t* table, int64_t table_ld,
                 const int32_t* kv_len, const int32_t* q_start, int B, rl_stream_t stream) {
  using namespace rl;
  const kv::Pool p{pool_k, pool_v, pool_ke, pool_ve, pages, kv_heads, page};
  const kv::Batch bt{table, table_ld, kv_len, q_start, B, T};
  int st;
  if ((st = kv::check_pool("rl_kv_append", p)) != RL_OK || (st = kv::check_batch("rl_kv_append", bt)) != RL_OK) return st;
  RL_REQUIRE(dtype == RL_F32 || dtype == RL_BF16, RL_ERR_ARGUMENT, "rl_kv_append: unknown dtype %d", dtype);
  RL_REQUIRE(T * kv_heads < (1ll << 35), RL_ERR_ARGUMENT, "rl_kv_append: %lld rows of %d heads", (long long)T, kv_heads);
  if (T == 0 || B == 0) return RL_OK;
  RL_REQUIRE(k && v && q_start, RL_ERR_ARGUMENT, "rl_kv_append: NULL pointer");
  const uintptr_t es = dtype == RL_F32 ? 4 : 2;
  RL_REQUIRE(aligned(k, es) && aligned(v, es), RL_ERR_ALIGNMENT, "rl_kv_append: k and v must be aligned to their type");
  RL_REQUIRE(device_is_sm100(), RL_ERR_UNSUPPORTED, "rl_kv_append: needs an sm_100 device");
  // one row per warp while all warps are resident at once (a decode step: every row leads a block of its own), else
  // 16 rows per warp, of which one or two lead
  const int rows = T * kv_heads * 2 <= static_cast<int64_t>(sm_count()) * 64 ? 1 : 16;
  const int64_t groups = (T + rows - 1) / rows;
  const int64_t ctas = (groups * kv_heads * 2 + 3) / 4;
  const kv::Source sk{k, k_st, k_sh, k_sd}, sv{v, v_st, v_sh, v_sd};
  auto wide = [](const kv::Source& s) { return s.sd == 1 && aligned(s.x, 16) && s.st % 8 == 0 && s.sh % 8 == 0; };
  const unsigned grid = static_cast<unsigned>(ctas) + 1;
  if (dtype == RL_BF16 && wide(sk) && wide(sv))
    kv::append_kernel<kv::WideBlock><<<grid, 128, 0, stream>>>(sk, sv, p, bt, rows, groups);
  else if (dtype == RL_BF16)
    kv::append_kernel<kv::AnyBlock<uint16_t>><<<grid, 128, 0, stream>>>(sk, sv, p, bt, rows, groups);
  else
    kv::append_kernel<kv::AnyBlock<float>><<<grid, 128, 0, stream>>>(sk, sv, p, bt, rows, groups);
  RL_TRY_CUDA(cudaGetLastError());
  return RL_OK;
}

int rl_kv_read(const uint8_t* pool_k, const uint8_t* pool_v, const uint8_t* pool_ke, const uint8_t* pool_ve,
               int64_t pages, int kv_heads, int page, const int32_t* table, int64_t table_ld, const int32_t* kv_len,
               const int32_t* start, int B, int64_t count, uint16_t* k_out, uint16_t* v_out, rl_stream_t stream) {
  using namespace rl;
  const kv::Pool p{const_cast<uint8_t*>(pool_k), const_cast<uint8_t*>(pool_v), const_cast<uint8_t*>(pool_ke),
                   const_cast<uint8_t*>(pool_ve), pages, kv_heads, page};
  const kv::Batch bt{table, table_ld, kv_len, nullptr, B, 0};
  int st;
  if ((st = kv::check_pool("rl_kv_read", p)) != RL_OK || (st = kv::check_batch("rl_kv_read", bt)) != RL_OK) return st;
  RL_REQUIRE(count >= 0 && count * kv_heads <= (1 << 27), RL_ERR_ARGUMENT, "rl_kv_read: count %lld of %d heads",
             (long long)count, kv_heads);
  if (count == 0 || B == 0) return RL_OK;
  RL_REQUIRE(start && k_out && v_out, RL_ERR_ARGUMENT, "rl_kv_read: NULL pointer");
  RL_REQUIRE(aligned(k_out, 16) && aligned(v_out, 16) && aligned(start, 4), RL_ERR_ALIGNMENT,
             "rl_kv_read: outputs must be 16-byte aligned");
  RL_REQUIRE(device_is_sm100(), RL_ERR_UNSUPPORTED, "rl_kv_read: needs an sm_100 device");
  const int64_t ctas = (count * kv_heads * (kv::HD / 16) + 255) / 256;
  const dim3 grid(static_cast<unsigned>(ctas), static_cast<unsigned>(B));
  kv::read_kernel<<<grid, 256, 0, stream>>>(p, table, table_ld, kv_len, start, static_cast<uint32_t>(count), k_out, v_out);
  RL_TRY_CUDA(cudaGetLastError());
  return RL_OK;
}

int rl_kv_copy_pages(uint8_t* pool_k, uint8_t* pool_v, uint8_t* pool_ke, uint8_t* pool_ve, int layers, int64_t pages,
                     int kv_heads, int page, const int32_t* src, const int32_t* dst, int64_t n, rl_stream_t stream) {
  using namespace rl;
  const kv::Pool p{pool_k, pool_v, pool_ke, pool_ve, pages, kv_heads, page};
  int st;
  if ((st = kv::check_pool("rl_kv_copy_pages", p)) != RL_OK) return st;
  RL_REQUIRE(layers > 0 && layers <= 65535, RL_ERR_ARGUMENT, "rl_kv_copy_pages: %d layers", layers);
  RL_REQUIRE(n >= 0 && n <= pages, RL_ERR_ARGUMENT, "rl_kv_copy_pages: %lld copies in %lld pages", (long long)n,
             (long long)pages);
  if (n == 0) return RL_OK;
  RL_REQUIRE(src && dst, RL_ERR_ARGUMENT, "rl_kv_copy_pages: NULL pointer");
  // The copies of one call run at once: a page may be copied to several others, but a page that is written must be
  // neither read nor written by another copy.
  uint8_t* seen = static_cast<uint8_t*>(std::calloc(static_cast<size_t>(pages), 1));
  RL_REQUIRE(seen, RL_ERR_ARGUMENT, "rl_kv_copy_pages: out of host memory");
  int64_t bad = -1;
  for (int64_t i = 0; i < n && bad < 0; ++i) {
    if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages || (seen[dst[i]] & 1)) bad = i;
    else seen[dst[i]] |= 1;
  }
  for (int64_t i = 0; i < n && bad < 0; ++i)
    if (seen[src[i]] & 1) bad = i;
  std::free(seen);
  RL_REQUIRE(bad < 0, RL_ERR_ARGUMENT,
             "rl_kv_copy_pages: copy %lld (page %d to %d): pages lie in [0, %lld), and a page that is written is neither "
             "read nor written by another copy of the call", (long long)bad, src[bad], dst[bad], (long long)pages);
  RL_REQUIRE(device_is_sm100(), RL_ERR_UNSUPPORTED, "rl_kv_copy_pages: needs an sm_100 device");
  const int64_t le = pages * kv_heads * (page / kv::BT), lc = pages * kv_heads * page * kv::HD;
  for (int64_t i = 0; i < n; i += 1024) {
    const int m = static_cast<int>(n - i < 1024 ? n - i : 1024);
    st = m <= 32 ? kv::copy_launch<32>(p, layers, lc, le, src + i, dst + i, m, stream)
                 : kv::copy_launch<1024>(p, layers, lc, le, src + i, dst + i, m, stream);
    if (st != RL_OK) return st;
  }
  return RL_OK;
}

int rl_kv_set(int32_t* dst, int64_t size, const int32_t* at, const int32_t* value, int64_t n, rl_stream_t stream) {
  using namespace rl;
  RL_REQUIRE(n >= 0 && size >= 0 && size <= INT32_MAX, RL_ERR_ARGUMENT, "rl_kv_set: %lld entries of %lld", (long long)n,
             (long long)size);
  if (n == 0) return RL_OK;
  RL_REQUIRE(dst && at && value, RL_ERR_ARGUMENT, "rl_kv_set: NULL pointer");
  RL_REQUIRE(aligned(dst, 4), RL_ERR_ALIGNMENT, "rl_kv_set: dst must be 4-byte aligned");
  for (int64_t i = 0; i < n; ++i)
    RL_REQUIRE(at[i] >= 0 && at[i] < size, RL_ERR_ARGUMENT, "rl_kv_set: entry %d of an array of %lld", at[i],
               (long long)size);
  RL_REQUIRE(device_is_sm100(), RL_ERR_UNSUPPORTED, "rl_kv_set: needs an sm_100 device");
  for (int64_t i = 0; i < n; i += 1024) {
    const int m = static_cast<int>(n - i < 1024 ? n - i : 1024);
    if (m <= 256) {
      kv::Pairs<256> a = {};
      for (int j = 0; j < m; ++j) a.src[j] = at[i + j], a.dst[j] = value[i + j];
      kv::set_kernel<256><<<1, 256, 0, stream>>>(dst, m, a);
    } else {
      kv::Pairs<1024> a = {};
      for (int j = 0; j < m; ++j) a.src[j] = at[i + j], a.dst[j] = value[i + j];
      kv::set_kernel<1024><<<1, 1024, 0, stream>>>(dst, m, a);
    }
    RL_TRY_CUDA(cudaGetLastError());
  }
  return RL_OK;
}

}  // extern "C"
