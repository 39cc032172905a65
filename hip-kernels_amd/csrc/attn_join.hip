// attn_join.hip -- joins the partial sums of rows whose tokens were cut into
// pieces (gfx950): attention's triples (reference m, sum l of 2^(s - m), weighted
// sum O of the values) over disjoint tokens, as attn_decode.hip has them, with the
// sink logit as one more token.  Bound by its launch and two dependent reads
// (4 us for 64 sequences of 64 heads).
#include "attn_device.h"

namespace gxmoe {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// T threads for each (row, head), 256 / T of these to a work-group.  A lane
// takes four dims of the pieces r, r + R, ..., with a reference of its own, so
// that nothing but the plan is waited for before they are read, U at a time.
template <int D, int T, int U>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a, JoinArgs j) {
  constexpr int kLanes = D / 4, R = T / kLanes;
  __shared__ f32x4 s_o[256 / kLanes][kLanes];
  __shared__ float s_m[256 / kLanes], s_l[256 / kLanes];
  __shared__ int s_any[256 / kLanes];
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (256 / T) + threadIdx.x / T;
  const int d = threadIdx.x % kLanes, row = threadIdx.x / kLanes, r0 = row / R * R;
  bool in = at < static_cast<int64_t>(a.rows) * a.heads;
  const int b = in ? static_cast<int>(at / a.heads) : 0, head = in ? static_cast<int>(at % a.heads) : 0;
  if (a.offsets != nullptr) in = in && b >= a.offsets[0] && b < a.offsets[a.B];  // rows of no sequence have no plan
  const int first = a.offsets != nullptr ? b : j.plan[2 * b];
  const int chunks = in ? min(j.plan[a.offsets != nullptr ? b : 2 * b + 1], j.max_pieces) : 0;
  const int64_t step = a.offsets != nullptr ? static_cast<int64_t>(a.rows) * a.heads : a.heads;
  const float sink = a.sinks ? bf16_to_f32(a.sinks[head]) * kLog2e : kNegInf;
  const float vs = a.kv.e4m3 && a.kv.v_scale ? a.kv.v_scale[head / (a.heads / a.kv.kv_heads)] : 1.0f;
  if (chunks > 1) {  // otherwise written by its only work-group
    const f32x4* ml = reinterpret_cast<const f32x4*>(j.part_ml) + static_cast<int64_t>(first) * a.heads + head;
    const f32x4* po = reinterpret_cast<const f32x4*>(j.part_o + (static_cast<int64_t>(first) * a.heads + head) * D) + d;
    float m = kNegInf, l = 0.0f;
    f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int any = 0;
    for (int c0 = row - r0; c0 < chunks; c0 += U * R) {
      f32x4 x[U], y[U];
      float top = m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t c = min(c0 + u * R, chunks - 1);
        x[u] = ml[c * step];
        y[u] = po[c * step * kLanes];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c0 + u * R >= chunks) x[u] = f32x4{kNegInf, 0.0f, 0.0f, 0.0f};
        top = __builtin_fmaxf(top, x[u][0]);
      }
      const float base = top == kNegInf ? 0.0f : top;
      const float keep = __builtin_amdgcn_exp2f(m - base);
      m = top;
      l *= keep;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c0 + u * R >= chunks) continue;
        const float f = __builtin_amdgcn_exp2f(x[u][0] - base);
        l = __builtin_fmaf(x[u][1], f, l);
        any |= x[u][2] != 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(y[u][e], f, o[e]);
      }
    }
    s_o[row][d] = o;
    if (d == 0) s_m[row] = m, s_l[row] = l, s_any[row] = any;
  }
  __syncthreads();
  if (chunks <= 1 || row != r0) return;
  float top = sink;
#pragma unroll
  for (int r = 0; r < R; ++r) top = __builtin_fmaxf(top, s_m[r0 + r]);
  const float base = top == kNegInf ? 0.0f : top;
  float sum = a.sinks ? __builtin_amdgcn_exp2f(sink - base) : 0.0f;
  f32x4 acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  int any = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float f = __builtin_amdgcn_exp2f(s_m[r0 + r] - base);
    sum = __builtin_fmaf(s_l[r0 + r], f, sum);
    any |= s_any[r0 + r];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(s_o[r0 + r][d][e], f, acc[e]);
  }
  const float f = vs / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = any ? acc[e] * f : 0.0f;
  *reinterpret_cast<attn_u32x2*>(a.out + b * a.out_stride + static_cast<int64_t>(head) * D + 4 * d) =
      attn_u32x2{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
}

// (row, head) pairs up to which a pair is a whole work-group
constexpr int kWide = 1024;

template <int D, int T>
hipError_t launch(const AttendArgs& a, const JoinArgs& j, int64_t mean, hipStream_t s) {
  constexpr int R = T / (D / 4);
  const int64_t pairs = static_cast<int64_t>(a.rows) * a.heads;
  const dim3 grid(static_cast<unsigned>((pairs + 256 / T - 1) / (256 / T)));
  // No more reads at a time than most rows have pieces, which a lane without
  // pieces waits for as well: 16384 pairs of four pieces of 128 dims 11 us, 16.5 with
  // 8 at a time; decode of 8 ragged sequences of up to 4000 10.6 / 11.4, of 4 of up to
  // 32000 with 128 dims, 17 pieces each, 38.6 / 37.4.
  if (mean <= 2 * R)
    hipLaunchKernelGGL((join_kernel<D, T, 2>), grid, dim3(256), 0, s, a, j);
  else
    hipLaunchKernelGGL((join_kernel<D, T, 8>), grid, dim3(256), 0, s, a, j);
  return hipGetLastError();
}

template <int D>
hipError_t launch(const AttendArgs& a, const JoinArgs& j, int64_t mean, hipStream_t s) {
  return static_cast<int64_t>(a.rows) * a.heads <= kWide ? launch<D, 256>(a, j, mean, s) : launch<D, 64>(a, j, mean, s);
}

}  // namespace

hipError_t launch_join(const AttendArgs& a, const JoinArgs& j, int64_t mean, hipStream_t s) {
  return a.kv.head_dim == 64 ? launch<64>(a, j, mean, s) : launch<128>(a, j, mean, s);
}

}  // namespace gxmoe
