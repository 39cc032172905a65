// attn_device.h -- device helpers of the attention kernels.
#pragma once

#include "attn_kernels.h"
#include "moe_device.h"

namespace gxmoe {

typedef uint32_t attn_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t attn_u32x2 __attribute__((ext_vector_type(2)));

typedef const __attribute__((address_space(1))) uint8_t* GlobalBytes;

// A lane's offset as the block at hand sees it: 32 bits on a pointer in scalar
// registers.  (Hoisted out of the loop it would be a 64-bit sum per load.)
__device__ __forceinline__ uint32_t here(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A pointer that is the same in all lanes, kept apart from their offsets.
__device__ __forceinline__ GlobalBytes scalar(GlobalBytes p) {
  asm("" : "+s"(p));
  return p;
}

constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;

// The sum over this lane and those before it.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // from 1, 2, 4, 8 lanes before in the row of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row 0's sum to row 1, row 2's to row 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // the lower half's to the upper
  return v;
}

// acc + both bf16 of a dword.
__device__ __forceinline__ float add_two(uint32_t two, float acc) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two), __builtin_bit_cast(bf16x2, 0x3f803f80u), acc, false);
}

// The four e4m3 codes of a dword as bf16 (exact).
__device__ __forceinline__ void widen(uint32_t codes, uint32_t* out) {
  out[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, false));
  out[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, true));
}

// Tokens of sequence b: negative lengths read as 0, longer ones than its
// table holds are cut to that.
__device__ __forceinline__ int seq_len(const AttendArgs& a, int b) {
  const int64_t cap = static_cast<int64_t>(a.max_blocks) << a.kv.bs_shift;
  const int n = max(a.lens[b], 0);
  return cap < n ? static_cast<int>(cap) : n;
}

// What scores of a kv head are multiplied by.  Not 0 where the product underflows:
// a hidden token's -inf would become NaN (so small a scale gives every seen token
// the same weight, and the smallest number does too).
template <bool kE4m3>
__device__ __forceinline__ float score_scale(const AttendArgs& a, int kvh) {
  const float scale = a.scale_log2 * (kE4m3 && a.kv.k_scale ? a.kv.k_scale[kvh] : 1.0f);
  return scale == 0.0f ? 0x1p-149f : scale;
}

// Whether the token at position t is seen from position p: not a later one,
// and within the window or among the first tokens.
__device__ __forceinline__ bool sees(const AttendArgs& a, int p, int t) {
  return t <= p && (a.window == 0 || p - t < a.window || t < a.first);
}

}  // namespace gxmoe
