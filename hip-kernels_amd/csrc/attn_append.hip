// attn_append.hip -- position rotation of queries and keys, and the append of
// keys and values to the paged cache (gfx950).
#include "attn_device.h"

namespace gxmoe {

namespace {

// cos and sin of every position, [position][cos, sin][rotary / 2], from the
// angle position * f_i in 64 bits (at position 131071 an angle in fp32 is off
// by up to 2^-8).  YaRN: a dimension that turns more than beta_fast times in
// the original context keeps its frequency, one that turns less than beta_slow
// times has it divided by the factor, with a linear ramp in between; cos and sin
// carry the concentration.
__global__ void rope_table_kernel(RopeTableArgs a) {
  const int half = a.rotary / 2;
  const size_t total = static_cast<size_t>(a.max_positions) * half;
  const double two_pi = 6.283185307179586476925286766559;
  const double log_theta = log(a.theta);
  for (size_t q = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; q < total;
       q += static_cast<size_t>(gridDim.x) * blockDim.x) {
    const int i = static_cast<int>(q % half);
    const size_t pos = q / half;
    double f = exp(-log_theta * (2.0 * i / a.rotary));
    if (a.factor != 1.0) {
      const double low = half * log(a.original / (a.beta_fast * two_pi)) / log_theta;
      const double high = half * log(a.original / (a.beta_slow * two_pi)) / log_theta;
      double ramp = high > low ? (i - low) / (high - low) : (i < low ? 0.0 : 1.0);
      ramp = ramp < 0.0 ? 0.0 : ramp > 1.0 ? 1.0 : ramp;
      f = (1.0 - ramp) * f + ramp * f / a.factor;
    }
    double s, c;
    sincos(static_cast<double>(pos) * f, &s, &c);
    a.table[(2 * pos) * half + i] = static_cast<float>(c * a.concentration);
    a.table[(2 * pos + 1) * half + i] = static_cast<float>(s * a.concentration);
  }
}

// e4m3 of x, past the largest finite value that value; NaN stays NaN.
__device__ __forceinline__ uint8_t to_e4m3(float x) {
  const float c = x != x ? x : __builtin_fminf(__builtin_fmaxf(x, -448.0f), 448.0f);
  return static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false));
}

// One thread per dim of a row: its value and its partner's, the table's cos
// and sin, one store.
template <bool kE4m3>
__global__ __launch_bounds__(256) void rope_append_kernel(AppendArgs a) {
  const int D = a.kv.head_dim, H = a.heads, Hk = a.kv.kv_heads, half = a.rotary / 2;
  const int cols = (H + 2 * Hk) * D;
  const size_t total = static_cast<size_t>(a.T) * cols;
  for (size_t q = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; q < total;
       q += static_cast<size_t>(gridDim.x) * blockDim.x) {
    const int t = static_cast<int>(q / cols), c = static_cast<int>(q % cols);
    const int head = c / D, d = c % D;
    const int pos = a.positions[t];
    if (pos < 0 || pos >= a.max_positions) continue;
    const uint16_t* row = a.qkv + t * a.qkv_stride + static_cast<int64_t>(head) * D;
    float v = bf16_to_f32(row[d]);
    if (head < H + Hk && d < a.rotary) {
      const bool second = a.interleaved ? (d & 1) != 0 : d >= half;
      const int i = a.interleaved ? d >> 1 : second ? d - half : d;
      const int partner = a.interleaved ? d ^ 1 : second ? d - half : d + half;
      const float cs = a.table[static_cast<size_t>(2) * pos * half + i];
      const float sn = a.table[(static_cast<size_t>(2) * pos + 1) * half + i];
      const float w = bf16_to_f32(row[partner]);
      v = second ? v * cs + w * sn : v * cs - w * sn;
    }
    if (head < H) {
      a.q_out[t * a.q_stride + static_cast<int64_t>(head) * D + d] = f32_to_bf16(v);
      continue;
    }
    const int slot = a.slots[t];
    if (slot < 0 || (slot >> a.kv.bs_shift) >= a.kv.num_blocks) continue;
    const bool is_k = head < H + Hk;
    const int h = is_k ? head - H : head - H - Hk;
    const int64_t at = (slot >> a.kv.bs_shift) * a.kv.sb + h * a.kv.sh + (slot & ((1 << a.kv.bs_shift) - 1)) * a.kv.st + d;
    void* base = is_k ? a.kv.k : a.kv.v;
    if constexpr (kE4m3) {
      const float* sc = is_k ? a.kv.k_scale : a.kv.v_scale;
      static_cast<uint8_t*>(base)[at] = to_e4m3(sc ? v / sc[h] : v);
    } else {
      static_cast<uint16_t*>(base)[at] = f32_to_bf16(v);
    }
  }
}

int grid_for(size_t total) {
  const size_t b = (total + 255) / 256;
  return static_cast<int>(b > 8192 ? 8192 : b < 1 ? 1 : b);
}

}  // namespace

hipError_t launch_rope_table(const RopeTableArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(rope_table_kernel, dim3(grid_for(static_cast<size_t>(a.max_positions) * (a.rotary / 2))), dim3(256),
                     0, s, a);
  return hipGetLastError();
}

hipError_t launch_rope_append(const AppendArgs& a, hipStream_t s) {
  const int grid = grid_for(static_cast<size_t>(a.T) * (a.heads + 2 * a.kv.kv_heads) * a.kv.head_dim);
  if (a.kv.e4m3)
    hipLaunchKernelGGL(rope_append_kernel<true>, dim3(grid), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(rope_append_kernel<false>, dim3(grid), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace gxmoe
