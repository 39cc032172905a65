// attn_device.h -- device helpers of the attention kernels.
#pragma once

#include "attn_kernels.h"
#include "moe_device.h"

namespace gxmoe {

typedef uint32_t attn_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t attn_u32x2 __attribute__((ext_vector_type(2)));

constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;

// Tokens of sequence b: negative lengths read as 0, longer ones than its
// table holds are cut to that.
__device__ __forceinline__ int seq_len(const AttendArgs& a, int b) {
  const int64_t cap = static_cast<int64_t>(a.max_blocks) << a.kv.bs_shift;
  const int n = max(a.lens[b], 0);
  return cap < n ? static_cast<int>(cap) : n;
}

// Whether the token at position t is seen from position p: not a later one,
// and within the window or among the first tokens.
__device__ __forceinline__ bool sees(const AttendArgs& a, int p, int t) {
  return t <= p && (a.window == 0 || p - t < a.window || t < a.first);
}

}  // namespace gxmoe
