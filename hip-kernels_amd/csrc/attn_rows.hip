// attn_rows.hip -- attention of new tokens over the paged cache, one wave per
// (row, query head).
#include "attn_device.h"

namespace gxmoe {

namespace {

template <bool kE4m3>
__device__ __forceinline__ float kv_value(const void* p, int64_t i) {
  if constexpr (kE4m3)
    return __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(p)[i], 0);
  else
    return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
}

// Softmax over tiles of 64 tokens with a running maximum and sum: a lane
// takes the score of one token, then the wave's lanes take the dims and add
// the tile's values, weighted.
template <int D, bool kE4m3>
__global__ __launch_bounds__(64) void attend_rows_kernel(AttendArgs a) {
  const int row = blockIdx.x / a.heads, head = blockIdx.x % a.heads, lane = threadIdx.x;
  int b = row, new_tokens = 1, i = 0;
  if (a.offsets != nullptr) {
    b = -1;
    for (int b0 = 0; b0 < a.B && b < 0; b0 += 64) {
      const int c = min(b0 + lane, a.B - 1);
      const bool in = b0 + lane < a.B && a.offsets[c] <= row && row < a.offsets[c + 1];
      const uint64_t m = __ballot(in);
      if (m != 0) b = b0 + __builtin_ctzll(m);
    }
    if (b < 0) return;  // a row of no sequence
    new_tokens = a.offsets[b + 1] - a.offsets[b];
    i = row - a.offsets[b];
  }
  const int len = seq_len(a, b), p = len - new_tokens + i;
  const int h = head / (a.heads / a.kv.kv_heads);
  const uint16_t* q = a.q + row * a.q_stride + static_cast<int64_t>(head) * D;
  const float ks = kE4m3 && a.kv.k_scale ? a.kv.k_scale[h] : 1.0f;
  const float vs = kE4m3 && a.kv.v_scale ? a.kv.v_scale[h] : 1.0f;
  float m = a.sinks ? bf16_to_f32(a.sinks[head]) * kLog2e : kNegInf;
  float l = a.sinks ? 1.0f : 0.0f;
  float o[D / 64];
  for (int c = 0; c < D / 64; ++c) o[c] = 0.0f;
  bool any = false;
  for (int t0 = 0; t0 <= p; t0 += 64) {
    const int t = t0 + lane;
    bool seen = sees(a, p, t);
    int64_t at = 0;
    if (seen) {
      const int page = a.tables[b * a.table_stride + (t >> a.kv.bs_shift)];
      seen = page >= 0 && page < a.kv.num_blocks;
      at = page * a.kv.sb + h * a.kv.sh + (t & ((1 << a.kv.bs_shift) - 1)) * a.kv.st;
    }
    if (__ballot(seen) == 0) continue;
    any = true;
    float s = kNegInf;
    if (seen) {
      s = 0.0f;
      for (int d = 0; d < D; ++d) s = __builtin_fmaf(bf16_to_f32(q[d]), kv_value<kE4m3>(a.kv.k, at + d), s);
      s *= a.scale_log2 * ks;
    }
    float mt = s;
    for (int x = 32; x >= 1; x >>= 1) mt = __builtin_fmaxf(mt, __shfl_xor(mt, x));
    // a NaN score is passed over here and makes its weight, the sum and the row NaN
    const float mn = __builtin_fmaxf(m, mt);
    const float base = mn == kNegInf ? 0.0f : mn;
    const float pr = __builtin_amdgcn_exp2f(s - base);
    const float keep = __builtin_amdgcn_exp2f(m - base);
    l = l * keep + wave_butterfly_sum(pr);
    m = mn;
    for (int c = 0; c < D / 64; ++c) o[c] *= keep;
    for (int j = 0; j < 64; ++j) {
      const bool in = (__ballot(seen) >> j) & 1;
      if (!in) continue;
      const float w = __shfl(pr, j);
      const int64_t from = __shfl(at, j);
      for (int c = 0; c < D / 64; ++c)
        o[c] = __builtin_fmaf(w, kv_value<kE4m3>(a.kv.v, from + c * 64 + lane), o[c]);
    }
  }
  for (int c = 0; c < D / 64; ++c)
    a.out[row * a.out_stride + static_cast<int64_t>(head) * D + c * 64 + lane] = f32_to_bf16(any ? o[c] * vs / l : 0.0f);
}

}  // namespace

hipError_t launch_attend_rows(const AttendArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.rows) * a.heads);
#define GX_ROWS(D_, E_) hipLaunchKernelGGL((attend_rows_kernel<D_, E_>), grid, dim3(64), 0, s, a)
  if (a.kv.head_dim == 64) {
    if (a.kv.e4m3) GX_ROWS(64, true);
    else GX_ROWS(64, false);
  } else {
    if (a.kv.e4m3) GX_ROWS(128, true);
    else GX_ROWS(128, false);
  }
#undef GX_ROWS
  return hipGetLastError();
}

}  // namespace gxmoe
