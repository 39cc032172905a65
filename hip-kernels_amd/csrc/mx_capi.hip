// mx_capi.hip -- C ABI of the expert selection and of the MXFP4 operators
// (include/gptoss_moe.h): argument checks, then one launch on the caller's stream.
#include <cmath>

#include "moe_status.h"
#include "mx_kernels.h"

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

bool aligned(const void* p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

constexpr int kMaxRows = 1 << 26;     // rows of a call
constexpr int kMaxColumns = 1 << 24;  // K, N

// A span of memory: `rows` pieces of `bytes`, `step` bytes apart.
struct Span {
  const void* p;
  size_t rows, step, bytes;
};

bool apart(const Span& x, const Span& y) {
  if (x.p == nullptr || y.p == nullptr || x.rows == 0 || y.rows == 0) return true;
  const uintptr_t a = reinterpret_cast<uintptr_t>(x.p), b = reinterpret_cast<uintptr_t>(y.p);
  return a + (x.rows - 1) * x.step + x.bytes <= b || b + (y.rows - 1) * y.step + y.bytes <= a;
}

int check_shape(int rows, int K) {
  if (rows < 0 || K <= 0) return set_error(GPTOSS_ERR_INVALID, "MXFP4 matrix of %d x %d", rows, K);
  if (K % 32 != 0) return set_error(GPTOSS_ERR_INVALID, "MXFP4 K=%d is not a multiple of the 32-element block", K);
  if (rows > kMaxRows || K > kMaxColumns)
    return set_error(GPTOSS_ERR_UNSUPPORTED, "MXFP4 matrix of %d x %d (at most 2^26 x 2^24)", rows, K);
  return GPTOSS_OK;
}

int check_packed(const char* name, const void* packed, const void* scales) {
  if (packed == nullptr || scales == nullptr) return set_error(GPTOSS_ERR_INVALID, "null %s", name);
  if (!aligned(packed, 16)) return set_error(GPTOSS_ERR_INVALID, "%s: packed values must be 16-byte aligned", name);
  return GPTOSS_OK;
}

// Rows of `cols` values, `stride` elements of `size` bytes apart, on 16 bytes each.
int check_rows16(const char* name, const void* p, int64_t stride, int cols, int size) {
  if (p == nullptr) return set_error(GPTOSS_ERR_INVALID, "null %s", name);
  if (!aligned(p, 16)) return set_error(GPTOSS_ERR_INVALID, "%s must be 16-byte aligned", name);
  if (stride < cols || stride % (16 / size) != 0 || stride > (INT64_MAX >> 36))
    return set_error(GPTOSS_ERR_INVALID, "%s: rows %lld elements apart, a multiple of %d and at least %d are needed", name,
                     static_cast<long long>(stride), 16 / size, cols);
  return GPTOSS_OK;
}

Span span_of(const void* p, int rows, int64_t stride, int cols, int size) {
  return Span{p, static_cast<size_t>(rows), static_cast<size_t>(stride) * size, static_cast<size_t>(cols) * size};
}

Span flat(const void* p, size_t bytes) { return Span{p, bytes != 0, 0, bytes}; }

// One call's product, the dense one with E = 0.
int product(const uint8_t* a, const uint8_t* as, int a_rows, const int32_t* row_index, const int32_t* offsets, int E,
            int rows, const uint8_t* w, const uint8_t* ws, const uint16_t* bias, int N, int K,
            const gptoss_mxfp4_result* r, void* stream) {
  const bool grouped = E != 0;
  int rc = check_shape(a_rows, K);
  if (rc == GPTOSS_OK) rc = check_shape(N, K);
  if (rc != GPTOSS_OK) return rc;
  if (N <= 0 || N > kMaxColumns) return set_error(GPTOSS_ERR_INVALID, "N=%d (1 to 2^24)", N);
  if (rows < 0 || rows > kMaxRows) return set_error(GPTOSS_ERR_INVALID, "rows=%d (0 to 2^26)", rows);
  // the kernels count tiles in 32 bits
  if ((static_cast<int64_t>(rows) / 32 + E + 1) * (N / 64 + 1) > INT32_MAX)
    return set_error(GPTOSS_ERR_UNSUPPORTED, "%d rows of %d columns in one call (2^42 results)", rows, N);
  if (r == nullptr) return set_error(GPTOSS_ERR_INVALID, "result is NULL");
  const bool quantized = r->out_packed != nullptr || r->out_scales != nullptr;
  if (r->swiglu && N % 2 != 0) return set_error(GPTOSS_ERR_INVALID, "swiglu needs pairs of columns, N=%d", N);
  // (the kernels hold alpha / ln 2: an infinite one would make NaN of a gate of zero)
  if (r->swiglu && (!(std::fabs(r->alpha) <= 0x1p127f) || !(r->limit >= 0.0f)))
    return set_error(GPTOSS_ERR_INVALID, "swiglu: alpha=%g must be within 2^127, limit=%g not negative",
                     static_cast<double>(r->alpha), static_cast<double>(r->limit));
  const int cols = r->swiglu ? N / 2 : N;
  if (quantized && cols % 32 != 0)
    return set_error(GPTOSS_ERR_INVALID, "MXFP4 results of %d columns, not a multiple of the 32-element block", cols);
  if (quantized && r->out != nullptr) return set_error(GPTOSS_ERR_INVALID, "results as values and as MXFP4: one of them");
  if (rows == 0) return ok();
  if (row_index == nullptr && a_rows < rows)
    return set_error(GPTOSS_ERR_INVALID, "a has %d rows, %d are needed without row_index", a_rows, rows);
  if (a_rows == 0) return set_error(GPTOSS_ERR_INVALID, "a has no rows");
  rc = check_packed("a", a, as);
  if (rc == GPTOSS_OK) rc = check_packed("w", w, ws);
  if (rc != GPTOSS_OK) return rc;
  if (grouped && offsets == nullptr) return set_error(GPTOSS_ERR_INVALID, "null expert_offsets");
  if (!aligned(row_index, 4) || !aligned(offsets, 4) || !aligned(bias, 2))
    return set_error(GPTOSS_ERR_INVALID, "row_index, expert_offsets and bias must be aligned to their elements");
  const size_t nb = static_cast<size_t>(K) / 32, wrows = static_cast<size_t>(grouped ? E : 1) * static_cast<size_t>(N);
  const Span in[] = {flat(a, static_cast<size_t>(a_rows) * nb * 16), flat(as, static_cast<size_t>(a_rows) * nb),
                     flat(w, wrows * nb * 16), flat(ws, wrows * nb), flat(bias, wrows * 2),
                     flat(row_index, static_cast<size_t>(rows) * 4), flat(offsets, (static_cast<size_t>(E) + 1) * 4)};
  if (quantized) {
    if (!r->out_packed || !r->out_scales) return set_error(GPTOSS_ERR_INVALID, "null out_packed / out_scales");
    if (!aligned(r->out_packed, 16)) return set_error(GPTOSS_ERR_INVALID, "out_packed must be 16-byte aligned");
    const size_t blocks = static_cast<size_t>(rows) * static_cast<size_t>(cols / 32);
    const Span op = flat(r->out_packed, blocks * 16), os = flat(r->out_scales, blocks);
    if (!apart(op, os)) return set_error(GPTOSS_ERR_INVALID, "out_packed overlaps out_scales");
    for (const Span& x : in)
      if (!apart(x, op) || !apart(x, os)) return set_error(GPTOSS_ERR_INVALID, "the results overlap an input");
  } else {
    const int size = r->out_fp32 ? 4 : 2;
    if (r->out == nullptr) return set_error(GPTOSS_ERR_INVALID, "null out");
    if (!aligned(r->out, size)) return set_error(GPTOSS_ERR_INVALID, "out must be aligned to its elements");
    if (r->out_stride < cols || r->out_stride > (INT64_MAX >> 36))
      return set_error(GPTOSS_ERR_INVALID, "out: rows %lld elements apart, at least %d are needed",
                       static_cast<long long>(r->out_stride), cols);
    const Span o = span_of(r->out, rows, r->out_stride, cols, size);
    for (const Span& x : in)
      if (!apart(x, o)) return set_error(GPTOSS_ERR_INVALID, "out overlaps an input");
  }
  MxProductArgs p{};
  p.a = a;
  p.as = as;
  p.row_index = row_index;
  p.offsets = offsets;
  p.a_rows = a_rows;
  p.rows = rows;
  p.E = grouped ? E : 1;
  p.w = w;
  p.ws = ws;
  p.bias = bias;
  p.N = N;
  p.K = K;
  p.swiglu = r->swiglu != 0;
  p.alpha = r->alpha;
  p.limit = r->limit;
  p.out = quantized ? r->out_packed : r->out;
  p.stride = r->out_stride;
  p.out_fp32 = r->out_fp32 != 0;
  p.out_scales = r->out_scales;
  p.vec = aligned(r->out, 16) && r->out_stride % (r->out_fp32 ? 4 : 8) == 0;
  const hipError_t e = launch_mx_product(p, static_cast<hipStream_t>(stream));
  if (e == hipErrorInvalidConfiguration)
    return set_error(GPTOSS_ERR_UNSUPPORTED, "%d rows of %d columns in one call: more tiles than a launch holds", rows, N);
  HIP_TRY(e, "MXFP4 product launch");
  return ok();
}

}  // namespace

extern "C" {

int gptoss_moe_select_experts(const void* logits, int64_t logits_stride, int logits_fp32, const float* bias,
                              int num_tokens, int num_experts, const gptoss_routing_config* cfg,
                              int32_t* expert_indices, float* expert_weights, void* stream) {
  if (cfg == nullptr) return set_error(GPTOSS_ERR_INVALID, "cfg is NULL");
  if (num_tokens < 0) return set_error(GPTOSS_ERR_INVALID, "num_tokens=%d < 0", num_tokens);
  if (num_experts < 1 || num_experts > kSelectMaxExperts)
    return set_error(GPTOSS_ERR_UNSUPPORTED, "num_experts=%d outside [1, %d]", num_experts, kSelectMaxExperts);
  if (cfg->score != GPTOSS_SCORE_SOFTMAX && cfg->score != GPTOSS_SCORE_SIGMOID)
    return set_error(GPTOSS_ERR_INVALID, "score %d is neither GPTOSS_SCORE_SOFTMAX nor GPTOSS_SCORE_SIGMOID", cfg->score);
  if (cfg->num_groups < 1 || cfg->num_groups > kSelectMaxGroups || num_experts % cfg->num_groups != 0)
    return set_error(GPTOSS_ERR_INVALID, "num_groups=%d must divide num_experts=%d, 1 to %d", cfg->num_groups, num_experts,
                     kSelectMaxGroups);
  if (cfg->top_groups < 1 || cfg->top_groups > cfg->num_groups)
    return set_error(GPTOSS_ERR_INVALID, "top_groups=%d outside [1, num_groups=%d]", cfg->top_groups, cfg->num_groups);
  if (cfg->group_rank != 1 && cfg->group_rank != 2)
    return set_error(GPTOSS_ERR_INVALID, "group_rank=%d must be 1 or 2", cfg->group_rank);
  const int within = cfg->top_groups * (num_experts / cfg->num_groups);
  if (cfg->top_k < 1 || cfg->top_k > kSelectMaxTopK || cfg->top_k > within)
    return set_error(GPTOSS_ERR_INVALID, "top_k=%d outside [1, %d]", cfg->top_k,
                     within < kSelectMaxTopK ? within : kSelectMaxTopK);
  if (std::isnan(cfg->scale) || std::isinf(cfg->scale))
    return set_error(GPTOSS_ERR_INVALID, "scale=%g must be finite", static_cast<double>(cfg->scale));
  if (num_tokens > kMaxRows) return set_error(GPTOSS_ERR_UNSUPPORTED, "num_tokens=%d above 2^26", num_tokens);
  if (num_tokens == 0) return ok();
  if (!logits || !expert_indices || !expert_weights) return set_error(GPTOSS_ERR_INVALID, "null pointer");
  const int size = logits_fp32 ? 4 : 2;
  if (!aligned(logits, size) || !aligned(bias, 4) || !aligned(expert_indices, 4) || !aligned(expert_weights, 4))
    return set_error(GPTOSS_ERR_INVALID, "logits, bias, expert_indices and expert_weights must be aligned to their elements");
  if (logits_stride < num_experts || logits_stride > (INT64_MAX >> 36))
    return set_error(GPTOSS_ERR_INVALID, "logits: rows %lld elements apart, at least %d are needed",
                     static_cast<long long>(logits_stride), num_experts);
  const size_t slots = static_cast<size_t>(num_tokens) * static_cast<size_t>(cfg->top_k);
  const Span in[] = {span_of(logits, num_tokens, logits_stride, num_experts, size),
                     flat(bias, 4 * static_cast<size_t>(num_experts))};
  const Span idx = flat(expert_indices, 4 * slots), wts = flat(expert_weights, 4 * slots);
  if (!apart(idx, wts)) return set_error(GPTOSS_ERR_INVALID, "expert_indices overlaps expert_weights");
  for (const Span& x : in)
    if (!apart(x, idx) || !apart(x, wts)) return set_error(GPTOSS_ERR_INVALID, "the results overlap an input");
  SelectArgs a{};
  a.logits = logits;
  a.stride = logits_stride;
  a.bias = bias;
  a.idx = expert_indices;
  a.w = expert_weights;
  a.T = num_tokens;
  a.E = num_experts;
  a.k = cfg->top_k;
  a.groups = cfg->num_groups;
  a.top_groups = cfg->top_groups;
  a.group_rank = cfg->group_rank;
  a.fp32 = logits_fp32 != 0;
  a.sigmoid = cfg->score == GPTOSS_SCORE_SIGMOID;
  a.renormalize = cfg->renormalize != 0;
  a.scale = cfg->scale;
  HIP_TRY(launch_select_experts(a, static_cast<hipStream_t>(stream)), "expert selection launch");
  return ok();
}

int gptoss_mxfp4_quantize(const void* x, int64_t x_stride, int x_fp32, int rows, int K, uint8_t* packed, uint8_t* scales,
                          void* stream) {
  int rc = check_shape(rows, K);
  if (rc != GPTOSS_OK) return rc;
  if (rows == 0) return ok();
  const int size = x_fp32 ? 4 : 2;
  rc = check_rows16("x", x, x_stride, K, size);
  if (rc == GPTOSS_OK) rc = check_packed("result", packed, scales);
  if (rc != GPTOSS_OK) return rc;
  const size_t blocks = static_cast<size_t>(rows) * static_cast<size_t>(K / 32);
  const Span in = span_of(x, rows, x_stride, K, size), op = flat(packed, blocks * 16), os = flat(scales, blocks);
  if (!apart(in, op) || !apart(in, os) || !apart(op, os)) return set_error(GPTOSS_ERR_INVALID, "x, packed and scales overlap");
  HIP_TRY(launch_mx_quantize(x, x_stride, x_fp32 != 0, rows, K, packed, scales, static_cast<hipStream_t>(stream)),
          "MXFP4 quantisation launch");
  return ok();
}

int gptoss_mxfp4_dequantize(const uint8_t* packed, const uint8_t* scales, int rows, int K, void* out, int64_t out_stride,
                            int out_fp32, void* stream) {
  int rc = check_shape(rows, K);
  if (rc != GPTOSS_OK) return rc;
  if (rows == 0) return ok();
  const int size = out_fp32 ? 4 : 2;
  rc = check_packed("matrix", packed, scales);
  if (rc == GPTOSS_OK) rc = check_rows16("out", out, out_stride, K, size);
  if (rc != GPTOSS_OK) return rc;
  const size_t blocks = static_cast<size_t>(rows) * static_cast<size_t>(K / 32);
  const Span o = span_of(out, rows, out_stride, K, size);
  if (!apart(o, flat(packed, blocks * 16)) || !apart(o, flat(scales, blocks)))
    return set_error(GPTOSS_ERR_INVALID, "out overlaps the matrix");
  HIP_TRY(launch_mx_dequantize(packed, scales, rows, K, out, out_stride, out_fp32 != 0, static_cast<hipStream_t>(stream)),
          "MXFP4 read launch");
  return ok();
}

int gptoss_mxfp4_matmul(const uint8_t* a_packed, const uint8_t* a_scales, int M, const uint8_t* w_packed,
                        const uint8_t* w_scales, const uint16_t* bias, int N, int K, const gptoss_mxfp4_result* result,
                        void* stream) {
  return product(a_packed, a_scales, M, nullptr, nullptr, 0, M, w_packed, w_scales, bias, N, K, result, stream);
}

int gptoss_moe_grouped_mxfp4_matmul(const uint8_t* a_packed, const uint8_t* a_scales, int a_rows, const int32_t* row_index,
                                    const int32_t* expert_offsets, int num_experts, int rows, const uint8_t* w_packed,
                                    const uint8_t* w_scales, const uint16_t* bias, int N, int K,
                                    const gptoss_mxfp4_result* result, void* stream) {
  if (num_experts < 1 || num_experts > kMxMaxExperts)
    return set_error(GPTOSS_ERR_UNSUPPORTED, "num_experts=%d outside [1, %d]", num_experts, kMxMaxExperts);
  return product(a_packed, a_scales, a_rows, row_index, expert_offsets, num_experts, rows, w_packed, w_scales, bias, N, K,
                 result, stream);
}

}  // extern "C"
