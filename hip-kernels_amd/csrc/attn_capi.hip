// attn_capi.hip -- C ABI of the attention operators (include/gptoss_moe.h):
// argument checks, then one or two launches (for each 8192 sequences) on the
// caller's stream.
#include <cmath>

#include "attn_kernels.h"
#include "moe_status.h"

using namespace gxmoe;

namespace {

int ok() {
  clear_error();
  return GPTOSS_OK;
}

#define HIP_TRY(expr, what)                                                                                   \
  do {                                                                                                        \
    hipError_t _e = (expr);                                                                                   \
    if (_e != hipSuccess) return set_error(GPTOSS_ERR_HIP, "%s: %s", what, hipGetErrorString(_e));            \
  } while (0)

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Bytes from the first to past the last element of `rows` rows of `cols` bf16.
size_t extent(int rows, int64_t stride, int64_t cols) {
  return rows < 1 ? 0 : 2 * (static_cast<size_t>(rows - 1) * static_cast<size_t>(stride) + static_cast<size_t>(cols));
}

bool apart(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x + na <= y || y + nb <= x;
}

// Whether no row of a is one of b's: their spans are apart, or the rows of one lie
// between the other's, the same distance apart.
bool rows_apart(const void* a, int64_t a_stride, int64_t a_cols, const void* b, int64_t b_stride, int64_t b_cols, int rows) {
  if (apart(a, extent(rows, a_stride, a_cols), b, extent(rows, b_stride, b_cols))) return true;
  if (a_stride != b_stride) return false;
  const int64_t step = 2 * a_stride;
  int64_t from = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a)) % step;
  if (from < 0) from += step;  // where b's rows begin, of a step from a's rows on
  return from >= 2 * a_cols && from + 2 * b_cols <= step;
}

// Whether n bytes at p lie outside of what K's and V's pages span.
bool clear_of(const KvPages& kv, const void* p, size_t n) {
  typedef unsigned __int128 Wide;  // strides may be anything
  const Wide last = Wide(kv.num_blocks - 1) * static_cast<uint64_t>(kv.sb) + Wide(kv.kv_heads - 1) * static_cast<uint64_t>(kv.sh) +
                    ((Wide(1) << kv.bs_shift) - 1) * static_cast<uint64_t>(kv.st);
  const Wide span = (last + kv.head_dim) * (kv.e4m3 ? 1 : 2), x = reinterpret_cast<uintptr_t>(p);
  for (const void* pages : {kv.k, kv.v}) {
    const Wide y = reinterpret_cast<uintptr_t>(pages);
    if (x < y + span && y < x + n) return false;
  }
  return true;
}

constexpr int kMaxGroup = 128;  // query heads per kv head
constexpr int64_t kMaxRowHeads = 1 << 26, kMaxSeqHeads = 1 << 22;  // rows and sequences of a call, times heads

int check_cache(const gptoss_kv_cache* c, KvPages* kv) {
  if (c == nullptr) return set_error(GPTOSS_ERR_INVALID, "cache is NULL");
  if (c->dtype != GPTOSS_KV_BF16 && c->dtype != GPTOSS_KV_E4M3)
    return set_error(GPTOSS_ERR_INVALID, "cache dtype %d is neither GPTOSS_KV_BF16 nor GPTOSS_KV_E4M3", c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(GPTOSS_ERR_UNSUPPORTED, "head_dim=%d (64 or 128)", c->head_dim);
  if (c->block_size < 16 || c->block_size > 256 || (c->block_size & (c->block_size - 1)) != 0)
    return set_error(GPTOSS_ERR_UNSUPPORTED, "block_size=%d (16, 32, 64, 128 or 256)", c->block_size);
  if (c->num_kv_heads < 1 || c->num_blocks < 1)
    return set_error(GPTOSS_ERR_INVALID, "num_kv_heads=%d and num_blocks=%d must be positive", c->num_kv_heads,
                     c->num_blocks);
  if (c->num_blocks > 0x7fffffff / c->block_size)
    return set_error(GPTOSS_ERR_UNSUPPORTED, "%d pages of %d slots: more than 2^31 - 1 slots", c->num_blocks,
                     c->block_size);
  if (c->k == nullptr || c->v == nullptr) return set_error(GPTOSS_ERR_INVALID, "null cache");
  if (!aligned16(c->k) || !aligned16(c->v)) return set_error(GPTOSS_ERR_INVALID, "k and v must be 16-byte aligned");
  const bool e4m3 = c->dtype == GPTOSS_KV_E4M3;
  if (!e4m3 && (c->k_scale != nullptr || c->v_scale != nullptr))
    return set_error(GPTOSS_ERR_INVALID, "a bf16 cache has no scales");
  kv->k = c->k;
  kv->v = c->v;
  kv->k_scale = c->k_scale;
  kv->v_scale = c->v_scale;
  kv->sb = c->block_stride;
  kv->sh = c->head_stride;
  kv->st = c->token_stride;
  if (kv->sb == 0 && kv->sh == 0 && kv->st == 0) {
    kv->st = c->head_dim;
    kv->sh = kv->st * c->block_size;
    kv->sb = kv->sh * c->num_kv_heads;
  }
  const int64_t unit = e4m3 ? 16 : 8;
  for (const int64_t st : {kv->sb, kv->sh, kv->st})
    if (st < c->head_dim || st % unit != 0)
      return set_error(GPTOSS_ERR_INVALID, "cache strides %lld, %lld, %lld must be multiples of %d and at least head_dim",
                       static_cast<long long>(kv->sb), static_cast<long long>(kv->sh), static_cast<long long>(kv->st),
                       static_cast<int>(unit));
  if (kv->st > (1 << 24))
    return set_error(GPTOSS_ERR_UNSUPPORTED, "token_stride=%lld above 2^24", static_cast<long long>(kv->st));
  kv->num_blocks = c->num_blocks;
  kv->bs_shift = __builtin_ctz(static_cast<unsigned>(c->block_size));
  kv->kv_heads = c->num_kv_heads;
  kv->head_dim = c->head_dim;
  kv->e4m3 = e4m3;
  return GPTOSS_OK;
}

int check_heads(int heads, const KvPages& kv) {
  if (heads < 1 || heads % kv.kv_heads != 0)
    return set_error(GPTOSS_ERR_INVALID, "num_heads=%d is not a positive multiple of %d kv heads", heads, kv.kv_heads);
  if (heads / kv.kv_heads > kMaxGroup)
    return set_error(GPTOSS_ERR_UNSUPPORTED, "%d query heads per kv head (at most %d)", heads / kv.kv_heads, kMaxGroup);
  return GPTOSS_OK;
}

int check_rows(const char* name, const void* p, int64_t stride, int64_t cols) {
  if (p == nullptr) return set_error(GPTOSS_ERR_INVALID, "null %s", name);
  if (!aligned16(p)) return set_error(GPTOSS_ERR_INVALID, "%s must be 16-byte aligned", name);
  if (stride < cols || stride % 8 != 0)
    return set_error(GPTOSS_ERR_INVALID, "%s: rows %lld elements apart, a multiple of 8 and at least %lld are needed",
                     name, static_cast<long long>(stride), static_cast<long long>(cols));
  return GPTOSS_OK;
}

// The arguments that both attention calls share.
int check_attend(AttendArgs* a, const gptoss_kv_cache* cache, const gptoss_attention_config* cfg, int rows, int B,
                 const void* workspace, size_t workspace_bytes) {
  int rc = check_cache(cache, &a->kv);
  if (rc == GPTOSS_OK) rc = check_heads(a->heads, a->kv);
  if (rc != GPTOSS_OK) return rc;
  if (cfg == nullptr) return set_error(GPTOSS_ERR_INVALID, "cfg is NULL");
  a->scale_log2 = cfg->scale * 1.44269504088896340736f;
  if (!(cfg->scale > 0.0f) || std::isinf(a->scale_log2))
    return set_error(GPTOSS_ERR_INVALID, "scale=%g must be positive and below 2.3e38", static_cast<double>(cfg->scale));
  if (cfg->window < 0 || cfg->first_tokens < 0)
    return set_error(GPTOSS_ERR_INVALID, "window=%d and first_tokens=%d must not be negative", cfg->window,
                     cfg->first_tokens);
  if (rows == 0 || B == 0) return GPTOSS_OK;
  const int64_t cols = static_cast<int64_t>(a->heads) * a->kv.head_dim;
  rc = check_rows("q", a->q, a->q_stride, cols);
  if (rc == GPTOSS_OK) rc = check_rows("out", a->out, a->out_stride, cols);
  if (rc != GPTOSS_OK) return rc;
  if (!rows_apart(a->q, a->q_stride, cols, a->out, a->out_stride, cols, rows))
    return set_error(GPTOSS_ERR_INVALID, "out overlaps q");
  if (!clear_of(a->kv, a->out, extent(rows, a->out_stride, cols)))
    return set_error(GPTOSS_ERR_INVALID, "out overlaps the cache");
  if (a->tables == nullptr || a->lens == nullptr) return set_error(GPTOSS_ERR_INVALID, "null block_tables / seq_lens");
  if (a->max_blocks < 1 || a->table_stride < a->max_blocks)
    return set_error(GPTOSS_ERR_INVALID, "max_blocks=%d must be positive and at most table_stride=%lld", a->max_blocks,
                     static_cast<long long>(a->table_stride));
  // grids and counts of tiles stay within 32 bits
  if (static_cast<int64_t>(rows) * a->heads > kMaxRowHeads || static_cast<int64_t>(B) * a->heads > kMaxSeqHeads)
    return set_error(GPTOSS_ERR_UNSUPPORTED, "%d rows and %d sequences of %d heads in one call (at most 2^26 and 2^22)",
                     rows, B, a->heads);
  const int64_t cap = static_cast<int64_t>(a->max_blocks) << a->kv.bs_shift;
  if (cap > kMaxTokens || cap / 16 + 1 > 0x7fffffff / B)
    return set_error(GPTOSS_ERR_UNSUPPORTED, "tables of %d pages for %d sequences", a->max_blocks, B);
  const size_t need = gptoss_paged_attention_call_bytes(a->offsets == nullptr ? 0 : rows, B, a->heads, a->kv.kv_heads,
                                                        a->kv.head_dim, cap, cfg->window, cfg->first_tokens);
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need)
      return set_error(GPTOSS_ERR_INVALID, "workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : 0,
                       need);
    if (!aligned16(workspace)) return set_error(GPTOSS_ERR_INVALID, "workspace must be 16-byte aligned");
  }
  a->B = B;
  a->rows = rows;
  a->window = cfg->window < cap ? cfg->window : 0;  // one that holds every token is none
  a->first = cfg->first_tokens;
  a->sinks = cfg->sinks;
  return GPTOSS_OK;
}

}  // namespace

extern "C" {

int gptoss_rope_config_default(gptoss_rope_config* cfg) {
  if (cfg == nullptr) return set_error(GPTOSS_ERR_INVALID, "cfg is NULL");
  *cfg = gptoss_rope_config{64, 131072, 150000.0, 32.0, 4096.0, 32.0, 1.0};
  return ok();
}

int gptoss_rope_table(const gptoss_rope_config* cfg, float* table, void* stream) {
  if (cfg == nullptr) return set_error(GPTOSS_ERR_INVALID, "cfg is NULL");
  if (cfg->rotary_dim < 16 || cfg->rotary_dim % 16 != 0 || cfg->max_positions < 1)
    return set_error(GPTOSS_ERR_INVALID, "rotary_dim=%d (a positive multiple of 16), max_positions=%d (positive)",
                     cfg->rotary_dim, cfg->max_positions);
  if (!(cfg->theta > 1.0) || std::isinf(cfg->theta) || !(cfg->scaling_factor >= 1.0) || std::isinf(cfg->scaling_factor))
    return set_error(GPTOSS_ERR_INVALID, "theta=%g must be above 1, scaling_factor=%g at least 1", cfg->theta,
                     cfg->scaling_factor);
  if (cfg->scaling_factor != 1.0 && !(cfg->original_positions > 0.0 && cfg->beta_fast > 0.0 && cfg->beta_slow > 0.0))
    return set_error(GPTOSS_ERR_INVALID, "original_positions=%g, beta_fast=%g and beta_slow=%g must be positive",
                     cfg->original_positions, cfg->beta_fast, cfg->beta_slow);
  // (no dim turns that often, and a ramp from none has no slope)
  if (cfg->scaling_factor != 1.0 && !(cfg->original_positions / (cfg->beta_fast * 6.283185307179586) > 0.0))
    return set_error(GPTOSS_ERR_INVALID, "beta_fast=%g is too large for original_positions=%g", cfg->beta_fast,
                     cfg->original_positions);
  if (table == nullptr) return set_error(GPTOSS_ERR_INVALID, "null table");
  if (!aligned16(table)) return set_error(GPTOSS_ERR_INVALID, "table must be 16-byte aligned");
  RopeTableArgs a{};
  a.table = table;
  a.rotary = cfg->rotary_dim;
  a.max_positions = cfg->max_positions;
  a.theta = cfg->theta;
  a.factor = cfg->scaling_factor;
  a.original = cfg->original_positions;
  a.beta_fast = cfg->beta_fast;
  a.beta_slow = cfg->beta_slow;
  a.concentration = 0.1 * std::log(cfg->scaling_factor) + 1.0;
  HIP_TRY(launch_rope_table(a, static_cast<hipStream_t>(stream)), "rope table launch");
  return ok();
}

int gptoss_rope_kv_append(const uint16_t* qkv, int64_t qkv_stride, const int32_t* positions, const int32_t* slots,
                          const float* rope_table, int rotary_dim, int max_positions, int interleaved, int T, int H,
                          uint16_t* q_out, int64_t q_stride, const gptoss_kv_cache* cache, void* stream) {
  AppendArgs a{};
  int rc = check_cache(cache, &a.kv);
  if (rc == GPTOSS_OK) rc = check_heads(H, a.kv);
  if (rc != GPTOSS_OK) return rc;
  if (T < 0) return set_error(GPTOSS_ERR_INVALID, "num_tokens=%d < 0", T);
  const int D = a.kv.head_dim;
  if (rotary_dim < 16 || rotary_dim % 16 != 0 || rotary_dim > D)
    return set_error(GPTOSS_ERR_INVALID, "rotary_dim=%d must be a positive multiple of 16 and at most %d", rotary_dim, D);
  if (max_positions < 1) return set_error(GPTOSS_ERR_INVALID, "max_positions=%d must be positive", max_positions);
  if (T > 1 << 25) return set_error(GPTOSS_ERR_UNSUPPORTED, "%d rows in one call (at most 2^25)", T);  // a work-group each
  if (T == 0) return ok();
  const int64_t cols = (static_cast<int64_t>(H) + 2 * static_cast<int64_t>(a.kv.kv_heads)) * D, q_cols = static_cast<int64_t>(H) * D;
  rc = check_rows("qkv", qkv, qkv_stride, cols);
  if (rc == GPTOSS_OK) rc = check_rows("q_out", q_out, q_stride, q_cols);
  if (rc != GPTOSS_OK) return rc;
  if (positions == nullptr || slots == nullptr || rope_table == nullptr)
    return set_error(GPTOSS_ERR_INVALID, "null positions / slots / rope_table");
  if (!aligned16(rope_table)) return set_error(GPTOSS_ERR_INVALID, "rope_table must be 16-byte aligned");
  const bool in_place = q_out == qkv && q_stride == qkv_stride;
  if (!in_place && !rows_apart(qkv, qkv_stride, cols, q_out, q_stride, q_cols, T))
    return set_error(GPTOSS_ERR_INVALID, "q_out overlaps qkv without being its queries' place");
  if (!clear_of(a.kv, qkv, extent(T, qkv_stride, cols)) || !clear_of(a.kv, q_out, extent(T, q_stride, q_cols)))
    return set_error(GPTOSS_ERR_INVALID, "qkv or q_out overlaps the cache");
  a.qkv = qkv;
  a.qkv_stride = qkv_stride;
  a.positions = positions;
  a.slots = slots;
  a.table = rope_table;
  a.max_positions = max_positions;
  a.rotary = rotary_dim;
  a.interleaved = interleaved != 0;
  a.T = T;
  a.heads = H;
  a.q_out = q_out;
  a.q_stride = q_stride;
  HIP_TRY(launch_rope_append(a, static_cast<hipStream_t>(stream)), "rope append launch");
  return ok();
}

size_t gptoss_paged_attention_workspace_bytes(int num_tokens, int num_seqs, int num_heads, int num_kv_heads,
                                              int head_dim) {
  if (num_tokens < 1 || num_seqs < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || head_dim < 1) return 0;
  if (num_heads / num_kv_heads > kMaxGroup || num_heads > kMaxSeqHeads) return 0;  // no call takes these
  const size_t decode = decode_workspace_bytes(num_seqs, num_heads, num_kv_heads, head_dim);
  const size_t prefill = prefill_workspace_bytes(num_tokens, num_heads, num_kv_heads, head_dim);
  return decode > prefill ? decode : prefill;
}

size_t gptoss_paged_attention_call_bytes(int num_tokens, int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                         int64_t max_tokens, int window, int first_tokens) {
  if (num_tokens < 0 || num_seqs < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || head_dim < 1) return 0;
  if (num_heads / num_kv_heads > kMaxGroup || num_heads > kMaxSeqHeads) return 0;
  if (max_tokens < 1 || max_tokens > kMaxTokens || window < 0 || first_tokens < 0) return 0;
  const Reach r{max_tokens, window < max_tokens ? window : 0, first_tokens};
  return num_tokens == 0 ? decode_call_bytes(num_seqs, num_heads, num_kv_heads, head_dim, r)
                         : prefill_call_bytes(num_tokens, num_seqs, num_heads, num_kv_heads, head_dim, r);
}

int gptoss_paged_attention_decode(const uint16_t* q, int64_t q_stride, const gptoss_kv_cache* cache,
                                  const int32_t* block_tables, int64_t table_stride, int max_blocks,
                                  const int32_t* seq_lens, int num_seqs, int num_heads,
                                  const gptoss_attention_config* cfg, uint16_t* out, int64_t out_stride,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (num_seqs < 0) return set_error(GPTOSS_ERR_INVALID, "num_seqs=%d < 0", num_seqs);
  AttendArgs a{};
  a.q = q;
  a.q_stride = q_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.tables = block_tables;
  a.table_stride = table_stride;
  a.max_blocks = max_blocks;
  a.lens = seq_lens;
  a.heads = num_heads;
  const int rc = check_attend(&a, cache, cfg, num_seqs, num_seqs, workspace, workspace_bytes);
  if (rc != GPTOSS_OK) return rc;
  if (num_seqs == 0) return ok();
  HIP_TRY(launch_decode(a, workspace, static_cast<hipStream_t>(stream)), "paged attention decode launch");
  return ok();
}

int gptoss_paged_attention_prefill(const uint16_t* q, int64_t q_stride, const int32_t* query_offsets, int num_tokens,
                                   const gptoss_kv_cache* cache, const int32_t* block_tables, int64_t table_stride,
                                   int max_blocks, const int32_t* seq_lens, int num_seqs, int num_heads,
                                   const gptoss_attention_config* cfg, uint16_t* out, int64_t out_stride,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  if (num_tokens < 0 || num_seqs < 0)
    return set_error(GPTOSS_ERR_INVALID, "num_tokens=%d and num_seqs=%d must not be negative", num_tokens, num_seqs);
  AttendArgs a{};
  a.q = q;
  a.q_stride = q_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.tables = block_tables;
  a.table_stride = table_stride;
  a.max_blocks = max_blocks;
  a.lens = seq_lens;
  a.offsets = query_offsets;
  a.heads = num_heads;
  if (query_offsets == nullptr && num_tokens > 0 && num_seqs > 0)
    return set_error(GPTOSS_ERR_INVALID, "null query_offsets");
  const int rc = check_attend(&a, cache, cfg, num_tokens, num_seqs, workspace, workspace_bytes);
  if (rc != GPTOSS_OK) return rc;
  if (num_tokens == 0 || num_seqs == 0) return ok();
  HIP_TRY(launch_prefill(a, workspace, static_cast<hipStream_t>(stream)), "paged attention prefill launch");
  return ok();
}

}  // extern "C"
