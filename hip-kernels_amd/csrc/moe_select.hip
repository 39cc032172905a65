// moe_select.hip -- selection of a token's experts from the router's logits.
//
//   score   softmax over all experts, or sigmoid
//   choice  score + bias (a balance that steers the choice and not the weights)
//   groups  contiguous ones of E / groups experts; a group counts the sum of its
//           group_rank highest choices, and the top_groups best groups stay
//   k       highest choices of these, descending, ties to the lower index
//   weight  the score; over the sum of the chosen ones if renormalize; times scale
//
// An expert whose logit or choice is -inf or whose choice is NaN is switched off:
// it comes behind the others of the kept groups (lower index first), counts 0 in
// its group's sum and has weight 0.  (A NaN choice keeps its score as weight, so
// that NaN logits show.)
#include "mx_device.h"
#include "mx_kernels.h"

namespace gxmoe {

namespace {

constexpr int kSelectWaves = 4;

// Choices as integers of the same order; 1 is switched off, 0 not in a kept group.
__device__ __forceinline__ uint64_t choice_key(double c) {
  if (!(c > -__builtin_inf())) return 1u;  // NaN too
  c += 0.0;                                // -0 and +0 are equal
  const uint64_t u = __builtin_bit_cast(uint64_t, c);
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = __builtin_fmax(v, __shfl_xor(v, m, kWave));
  return v;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

// The largest key of the wave and the lowest expert that has it.
__device__ __forceinline__ void wave_best(uint64_t& key, int& e) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t k2 = __shfl_xor(key, m, kWave);
    const int e2 = __shfl_xor(e, m, kWave);
    if (k2 > key || (k2 == key && e2 < e)) {
      key = k2;
      e = e2;
    }
  }
}

// A wave per token, expert lane + 64 j in value j of a lane; everything in 64
// bits, so that the order is that of the exact values but for gaps of 1e-15.
template <int NV>
__global__ __launch_bounds__(kSelectWaves * kWave) void select_kernel(SelectArgs a) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int t = blockIdx.x * kSelectWaves + wave;
  if (t >= a.T) return;  // no barrier below
  const size_t row = static_cast<size_t>(t) * static_cast<size_t>(a.stride);
  const double inf = __builtin_inf();

  double score[NV];
  uint64_t key[NV];
  double x[NV], top = -inf;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = lane + kWave * j;
    x[j] = -inf;
    if (e < a.E)
      x[j] = a.fp32 ? static_cast<const float*>(a.logits)[row + e]
                    : bf16_to_f32(static_cast<const uint16_t*>(a.logits)[row + e]);
    top = __builtin_fmax(top, x[j]);
  }
  if (!a.sigmoid) {
    top = wave_max(top);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      score[j] = x[j] == top ? (top == -inf ? 0.0 : 1.0) : exp(x[j] - top);  // (inf - inf, and a row of -inf)
      sum += score[j];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < NV; ++j) score[j] = sum == 0.0 ? 0.0 : score[j] / sum;
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) score[j] = 1.0 / (1.0 + exp(-x[j]));
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = lane + kWave * j;
    double c = -inf;
    if (e < a.E) c = score[j] + (a.bias ? static_cast<double>(a.bias[e]) : 0.0);
    if (x[j] == -inf) c = -inf;
    if (c == -inf) score[j] = 0.0;
    key[j] = choice_key(c);
    x[j] = c;
  }

  if (a.groups > 1) {
    // group after group: its members of this lane's values, then the wave's best two
    const int size = a.E / a.groups;
    uint64_t mine = 0;  // lane g: the key of group g
    for (int g = 0; g < a.groups; ++g) {
      const int lo = g * size, hi = lo + size;
      double total = 0.0;
      bool any = false;
      int taken = -1;
      for (int r = 0; r < a.group_rank; ++r) {
        uint64_t best = 0;
        int at = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int e = lane + kWave * j;
          if (e >= lo && e < hi && e != taken && key[j] > best) {
            best = key[j];
            at = e;
          }
        }
        wave_best(best, at);
        if (best <= 1u) break;  // switched off, as all that follow
        taken = at;
        any = true;
        double c = 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (lane + kWave * j == at) c = x[j];
        total += __shfl(c, at & (kWave - 1), kWave);
      }
      const uint64_t gk = any ? choice_key(total) : 1u;
      if (lane == g) mine = gk;
    }
    uint64_t kept = 0;
    for (int r = 0; r < a.top_groups; ++r) {
      uint64_t best = mine;
      int at = lane;
      wave_best(best, at);
      kept |= 1ull << at;
      if (lane == at) mine = 0;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = lane + kWave * j;
      if (e < a.E && !((kept >> (e / size)) & 1u)) key[j] = 0;
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (lane + kWave * j >= a.E) key[j] = 0;

  int chosen = 0;     // lane s: the s-th choice
  double weight = 0.0;
  for (int s = 0; s < a.k; ++s) {
    uint64_t best = 0;
    int at = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (key[j] > best) {
        best = key[j];
        at = lane + kWave * j;
      }
    wave_best(best, at);
    double w = 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (lane + kWave * j == at) {
        w = score[j];
        key[j] = 0;
      }
    w = __shfl(w, at & (kWave - 1), kWave);
    if (lane == s) {
      chosen = at;
      weight = w;
    }
  }
  if (a.renormalize) {
    const double sum = wave_sum(weight);
    weight = sum == 0.0 ? 0.0 : weight / sum;
  }
  if (lane < a.k) {
    const size_t o = static_cast<size_t>(t) * static_cast<size_t>(a.k) + lane;
    a.idx[o] = chosen;
    a.w[o] = static_cast<float>(weight * static_cast<double>(a.scale));
  }
}

}  // namespace

hipError_t launch_select_experts(const SelectArgs& a, hipStream_t s) {
  const dim3 grid((a.T + kSelectWaves - 1) / kSelectWaves), block(kSelectWaves * kWave);
  if (a.E <= 64) hipLaunchKernelGGL(select_kernel<1>, grid, block, 0, s, a);
  else if (a.E <= 128) hipLaunchKernelGGL(select_kernel<2>, grid, block, 0, s, a);
  else if (a.E <= 256) hipLaunchKernelGGL(select_kernel<4>, grid, block, 0, s, a);
  else if (a.E <= 512) hipLaunchKernelGGL(select_kernel<8>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(select_kernel<16>, grid, block, 0, s, a);
  return hipGetLastError();
}

}  // namespace gxmoe
