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

// Four e4m3 codes; past the largest finite value that value, NaN stays NaN.
__device__ __forceinline__ uint32_t to_e4m3x4(float x, float y, float z, float w) {
  auto clip = [](float v) { return v != v ? v : __builtin_fminf(__builtin_fmaxf(v, -448.0f), 448.0f); };
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(clip(x), clip(y), 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(clip(z), clip(w), lo, true));
}

// A wave takes a row: a lane has unit u = lane % U of heads lane / U, lane / U +
// 64 / U, ..., where a unit is 16 dims that turn by the same 8 angles (dims 8 u on
// and 8 u + rotary / 2 on, or 16 side by side), so that the angles are read once
// for all heads and every element moves in a 16-byte piece.  Bound by memory (the
// row in, the queries, keys and values out): 8192 rows of 64 + 8 + 8 heads of 64
// take 36 us, 4.7 TB/s, where a large copy reaches 4.95 (a thread per dim: 167 us).
// A wave is a work-group, so that few rows lie on as many CUs.
template <int D, bool kE4m3, bool kPairs>
__global__ __launch_bounds__(64) void rope_append_kernel(AppendArgs a) {
  constexpr int U = D / 16, kHeads = 64 / U;  // units of a head, heads of a pass
  constexpr int kPasses = 3;                  // whose loads are in flight together
  const int lane = threadIdx.x, u = lane % U, t = blockIdx.x;
  const int H = a.heads, Hk = a.kv.kv_heads, total = H + 2 * Hk;
  const int pos = a.positions[t], slot = a.slots[t];
  if (pos < 0 || pos >= a.max_positions) return;
  const bool stored = slot >= 0 && (slot >> a.kv.bs_shift) < a.kv.num_blocks;
  const bool turns = 16 * u < a.rotary;
  // the unit's two pieces: the halves of eight pairs, or dims side by side
  const int d0 = kPairs || !turns ? 16 * u : 8 * u;
  const int d1 = kPairs || !turns ? 16 * u + 8 : 8 * u + a.rotary / 2;
  float cs[8], sn[8];
  if (turns) {
    const float* at = a.table + static_cast<size_t>(pos) * a.rotary + 8 * u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 c = reinterpret_cast<const float4*>(at)[i], s = reinterpret_cast<const float4*>(at + a.rotary / 2)[i];
      cs[4 * i] = c.x, cs[4 * i + 1] = c.y, cs[4 * i + 2] = c.z, cs[4 * i + 3] = c.w;
      sn[4 * i] = s.x, sn[4 * i + 1] = s.y, sn[4 * i + 2] = s.z, sn[4 * i + 3] = s.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i] = 1.0f, sn[i] = 0.0f;
  }
  const uint16_t* row = a.qkv + t * a.qkv_stride;
  const int64_t place = (slot >> a.kv.bs_shift) * a.kv.sb + (slot & ((1 << a.kv.bs_shift) - 1)) * a.kv.st;
  for (int h0 = lane / U; h0 < total; h0 += kPasses * kHeads) {
    attn_u32x4 in[kPasses][2];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int h = h0 + p * kHeads;
      if (h >= total) continue;
      // values do not turn: their unit is 16 dims side by side
      const bool v = h >= H + Hk;
      in[p][0] = *reinterpret_cast<const attn_u32x4*>(row + static_cast<int64_t>(h) * D + (v ? 16 * u : d0));
      in[p][1] = *reinterpret_cast<const attn_u32x4*>(row + static_cast<int64_t>(h) * D + (v ? 16 * u + 8 : d1));
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int h = h0 + p * kHeads;
      if (h >= total || (h >= H && !stored)) continue;
      const bool v = h >= H + Hk;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(i & 1 ? in[p][i >> 3][(i & 7) >> 1] & 0xffff0000u : in[p][i >> 3][(i & 7) >> 1] << 16);
      if (!v && turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int lo = kPairs ? 2 * i : i, hi = kPairs ? 2 * i + 1 : i + 8;
          const float y = x[lo] * cs[i] - x[hi] * sn[i], z = x[hi] * cs[i] + x[lo] * sn[i];
          x[lo] = y, x[hi] = z;
        }
      }
      const int o0 = v ? 16 * u : d0, o1 = v ? 16 * u + 8 : d1;
      if (!kE4m3 || h < H) {
        uint16_t* to = h < H ? a.q_out + t * a.q_stride + static_cast<int64_t>(h) * D
                             : static_cast<uint16_t*>(v ? a.kv.v : a.kv.k) + place + (v ? h - H - Hk : h - H) * a.kv.sh;
        *reinterpret_cast<attn_u32x4*>(to + o0) =
            attn_u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
        *reinterpret_cast<attn_u32x4*>(to + o1) = attn_u32x4{pack_bf16x2(x[8], x[9]), pack_bf16x2(x[10], x[11]),
                                                             pack_bf16x2(x[12], x[13]), pack_bf16x2(x[14], x[15])};
      } else {
        const int hk = v ? h - H - Hk : h - H;
        const float* scales = v ? a.kv.v_scale : a.kv.k_scale;
        const float scale = scales ? scales[hk] : 1.0f;
        uint8_t* to = static_cast<uint8_t*>(v ? a.kv.v : a.kv.k) + place + hk * a.kv.sh;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = to_e4m3x4(x[4 * i] / scale, x[4 * i + 1] / scale, x[4 * i + 2] / scale, x[4 * i + 3] / scale);
        *reinterpret_cast<attn_u32x2*>(to + o0) = attn_u32x2{w[0], w[1]};
        *reinterpret_cast<attn_u32x2*>(to + o1) = attn_u32x2{w[2], w[3]};
      }
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
#define GX_APPEND(D_, E_, P_) hipLaunchKernelGGL((rope_append_kernel<D_, E_, P_>), dim3(a.T), dim3(64), 0, s, a)
#define GX_APPEND_P(D_, E_)               \
  do {                                    \
    if (a.interleaved) GX_APPEND(D_, E_, true); \
    else GX_APPEND(D_, E_, false);        \
  } while (0)
  if (a.kv.head_dim == 64) {
    if (a.kv.e4m3) GX_APPEND_P(64, true);
    else GX_APPEND_P(64, false);
  } else {
    if (a.kv.e4m3) GX_APPEND_P(128, true);
    else GX_APPEND_P(128, false);
  }
#undef GX_APPEND_P
#undef GX_APPEND
  return hipGetLastError();
}

}  // namespace gxmoe
