// C ABI of the attention over the paged cache: the choice between the split kernel (rl_kv_attn.cu) and the prompt kernel
// (rl_kv_prompt.cu).
#include "rl_common.cuh"
#include "rl_host.h"

namespace rl {
namespace kvattn {

inline int& path() {   // 0 = by the rules below, 1 = split kernel, 2 = prompt kernel, 3 = split kernel, in clusters
  static int v = 0;
  return v;
}

// The prompt kernel computes 256 rows x 128 keys in the time in which the split kernel, which runs on every SM whatever
// the shape, gets through about a quarter of them: it pays where its tiles are more than a quarter full of rows and
// the SMs more than a quarter full of tiles. (It scales row maxima, so it takes positive scales.)
// It goes by the call's averages: 63 sequences of one row and one of 1021 take the prompt kernel for all, 279 us, where the
// two kinds alone take 54 and 98; 63 without rows beside the same one fall to the split kernel, 424 us.
inline bool by_prompt(int64_t T, int B, int heads, int kv_heads, float scale_log2) {
  if (!(scale_log2 > 0.0f) || path() == 1 || path() == 3) return false;
  if (path() == 2) return true;
  const int64_t rows = T * (heads / kv_heads), each = (rows + B - 1) / B;
  const int64_t tiles = (each + kvprompt::ROWS - 1) / kvprompt::ROWS * B;
  const double full = static_cast<double>(rows) / (static_cast<double>(tiles) * kvprompt::ROWS);
  const double busy = static_cast<double>(tiles * kv_heads) / sm_count();
  return full * (busy < 1.0 ? busy : 1.0) > 0.25;
}

// The one-launch form splits every task in eight, whatever its length: it wins while the page table's width bounds the keys
// (the lengths are in device memory) and the tasks' CTAs fit the GPU at once. Device times, spread over the grid / in clusters
// (32 heads over 8, one row a sequence): 1 x 1024 keys 7.4 / 5.8 us, 1 x 4096 12.2 / 9.8, 1 x 8192 14.6 / 14.9, 2 x 8192 15.4 / 16.0, 8 x 4096 16.0 / 12.7,
// 8 x 8192 20.7 / 19.0, 16 x 8192 34.5 / 35.4, 64 x 1024 33 / 53; 16 x up to 5 rows, 4097 keys, 8 over 2: 19.0 / 13.9.
constexpr int64_t kShort = 6144;
inline bool by_cluster(int nt, int64_t T, int B, int group, int hkv, int64_t most_keys) {
  if (path() != 0) return path() == 3;
  const int64_t tiles = (T * group + 8 * nt - 1) / (8 * nt);
  return most_keys <= kShort && (tiles > B ? tiles : B) * hkv * kClusterCtas <= ctas_of(nt);
}

}  // namespace kvattn
}  // namespace rl

extern "C" {

int rl_set_kv_attention_path(int path) {
  const int prev = rl::kvattn::path();
  rl::kvattn::path() = path;
  return prev;
}

size_t rl_kv_attention_workspace(int64_t T, int B, int heads, int kv_heads) {
  using namespace rl;
  if (T <= 0 || B <= 0 || kv_heads <= 0 || heads <= 0) return 0;
  const int nt = kvattn::tile_n(T, B, heads / kv_heads);
  return kvattn::part_bytes(nt) + static_cast<size_t>(kvattn::ctas_of(nt)) * sizeof(kvattn::Record);
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
  RL_REQUIRE(T * heads < (1ll << 31), RL_ERR_ARGUMENT, "rl_kv_attention: %lld rows of %d heads", (long long)T, heads);
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
  a.o = o, a.ldo = ldo;
  a.group = kvattn::Div::of(heads / kv_heads), a.hkv = kvattn::Div::of(kv_heads);
  a.page_sh = __builtin_ctz(page);
  a.vec = aligned(o, 8) && ldo % 4 == 0;
  if (kvattn::by_prompt(T, B, heads, kv_heads, scale_log2)) {
    const kvprompt::Args p{q, q_st, q_sh, a.pool, a.batch, row_limit, scale_log2, o, ldo, a.group, a.hkv, a.page_sh,
                           aligned(o, 16) && ldo % 8 == 0};
    // at most this many: a sequence's last tile of 256 rows may be a part
    return kvprompt::launch((T * (heads / kv_heads) / kvprompt::ROWS + B) * kv_heads, p, stream);
  }
  const int nt = kvattn::tile_n(T, B, heads / kv_heads);
  a.part = static_cast<float*>(workspace);
  a.rec = reinterpret_cast<kvattn::Record*>(static_cast<uint8_t*>(workspace) + kvattn::part_bytes(nt));
  const int group = heads / kv_heads;
  if (kvattn::by_cluster(nt, T, B, group, kv_heads, table_ld * page)) {
    const int64_t tasks = kvattn::tasks_of(nt, T, B, group, kv_heads);
    switch (nt) {
      case 1: return kvattn::launch_cluster<1>(a, tasks, stream);
      case 2: return kvattn::launch_cluster<2>(a, tasks, stream);
      default: return kvattn::launch_cluster<4>(a, tasks, stream);
    }
  }
  switch (nt) {
    case 1: return kvattn::launch<1>(a, stream);
    case 2: return kvattn::launch<2>(a, stream);
    default: return kvattn::launch<4>(a, stream);
  }
}

}  // extern "C"
