// moe_select.hip -- selection of a token's experts from the router's logits.
//
//   score   softmax over all experts, or sigmoid
//   choice  score + bias (a balance that steers the choice and not the weights)
//   groups  contiguous ones of E / groups experts; a group counts the sum of its
//           group_rank highest choices, and the top_groups best groups stay
//   k       highest choices of these, descending, ties to the lower index
//   weight  the score; over the sum of the chosen ones if renormalize; times scale
//
// An expert whose logit or bias is -inf, or whose choice is NaN, is switched off:
// it comes behind the others of the kept groups (lower index first), counts 0 in
// its group's sum and has weight 0.  (A NaN choice without such a logit or bias keeps its
// score as weight, so that NaN logits show.)
//
// Bound by latency for few tokens (64 of 256 experts in 8 groups, 8 chosen: 5.7 us; one of 128, 4 chosen: 2.7) and
// by vector instructions for many (8192 of the same: 13 us, where reading the logits takes 1.6).
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

__device__ __forceinline__ double choice_of(uint64_t key) {  // key > 1
  return __builtin_bit_cast(double, (key >> 63) ? key & 0x7fffffffffffffffull : ~key);
}

// A lane's value with those of the lanes before it in its row of 16, then with the rows
// before: lane 63 ends with the wave's.  `none` stands for lanes that are not there.
template <int Ctrl, int Rows>
__device__ __forceinline__ uint32_t from_before(uint32_t v, uint32_t none) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(static_cast<int>(none), static_cast<int>(v), Ctrl, Rows, 0xf, false));
}

template <typename F>
__device__ __forceinline__ uint32_t wave_fold(uint32_t v, uint32_t none, F fold) {
  v = fold(v, from_before<0x111, 0xf>(v, none));  // row_shr 1, 2, 4, 8
  v = fold(v, from_before<0x112, 0xf>(v, none));
  v = fold(v, from_before<0x114, 0xf>(v, none));
  v = fold(v, from_before<0x118, 0xf>(v, none));
  v = fold(v, from_before<0x142, 0xa>(v, none));  // row_bcast 15 and 31
  v = fold(v, from_before<0x143, 0xc>(v, none));
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), kWave - 1));
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  return wave_fold(v, 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

__device__ __forceinline__ float wave_max(float v) {
  return __uint_as_float(wave_fold(__float_as_uint(v), 0xff800000u, [](uint32_t a, uint32_t b) {
    return __float_as_uint(__builtin_fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}

template <int Ctrl, int Rows>
__device__ __forceinline__ double add_before(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = from_before<Ctrl, Rows>(static_cast<uint32_t>(u), 0u);
  const uint32_t hi = from_before<Ctrl, Rows>(static_cast<uint32_t>(u >> 32), 0u);
  return v + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v)), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v >> 32)), lane);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

__device__ __forceinline__ double wave_sum(double v) {
  v = add_before<0x111, 0xf>(v);
  v = add_before<0x112, 0xf>(v);
  v = add_before<0x114, 0xf>(v);
  v = add_before<0x118, 0xf>(v);
  v = add_before<0x142, 0xa>(v);
  v = add_before<0x143, 0xc>(v);
  return __builtin_bit_cast(double, read_lane(__builtin_bit_cast(uint64_t, v), kWave - 1));
}

// The lowest lane that has the wave's largest key: the upper halves mostly tell.
__device__ __forceinline__ int best_lane(uint64_t key) {
  const uint32_t hi = static_cast<uint32_t>(key >> 32), top = wave_max(hi);
  uint64_t have = __ballot(hi == top);
  if (have & (have - 1)) {
    const uint32_t lo = hi == top ? static_cast<uint32_t>(key) : 0u, low = wave_max(lo);
    have &= __ballot(lo == low);
  }
  return __builtin_ctzll(have);
}

// How many of the wave's values are t or more.
template <int N>
__device__ __forceinline__ int count_from(const uint32_t (&v)[N], uint32_t t) {
  int n = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) n += __popcll(__ballot(v[j] >= t));
  return n;
}

// The upper halves of keys: a t that exactly k of the wave's are t or more of, found from the largest down
// in growing steps and then by halves.  False where there is none: equal halves on the border, or fewer than k
// that are not 0.
template <int N>
__device__ __forceinline__ bool find_border(const uint32_t (&v)[N], int k, uint32_t* t) {
  uint32_t most = v[0];
#pragma unroll
  for (int j = 1; j < N; ++j) most = max(most, v[j]);
  const uint32_t top = wave_max(most);
  if (top == 0u) return false;
  uint32_t up = top + 1, step = 1u << 18, lo = top > step ? top - step : 1u;  // (the largest is infinity's)
  int n = count_from(v, lo);
  while (n < k) {
    if (lo == 1u) return false;
    up = lo;
    step = step < 1u << 30 ? step << 2 : 0xffffffffu;
    lo = top > step ? top - step : 1u;
    n = count_from(v, lo);
  }
  while (n > k) {
    if (up - lo <= 1u) return false;
    const uint32_t mid = lo + (up - lo) / 2;
    const int m = count_from(v, mid);
    if (m >= k) {
      lo = mid;
      n = m;
    } else {
      up = mid;
    }
  }
  *t = lo;
  return true;
}

// A wave per token, experts NV lane to NV lane + NV - 1 a lane's own, so that of equal choices the
// lowest lane's first one counts.  Scores and choices are in 64 bits: the order is that of
// the exact values but for gaps of 1e-15, and a weight is rounded once.  Of four experts a lane and more, six or more
// chosen are told from the others by a border in the upper halves of their keys, found by
// counting, and then ranked among themselves; fewer, and where there is no such border, are taken one
// after the other.  (8192 tokens, 8 of 256: 13.3 us with the border, 15.1 one by one; 8 of 64: 5.8, 5.1; 4
// of 128 without a bias, where equal logits leave no border: 8.5, 6.9.)
template <int NV>
__global__ __launch_bounds__(kSelectWaves * kWave) void select_kernel(SelectArgs a) {
  __shared__ double scores[kSelectWaves][NV * kWave];
  __shared__ uint64_t few_keys[kSelectWaves][kSelectMaxTopK];
  __shared__ int few[kSelectWaves][kSelectMaxTopK];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int t = blockIdx.x * kSelectWaves + wave;
  if (t >= a.T) return;  // no barrier below
  const size_t row = static_cast<size_t>(t) * static_cast<size_t>(a.stride);
  const double inf = __builtin_inf();

  // (branches around all loads of a kind, so that these go out together)
  float x[NV], bias[NV];
  int at_e[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    at_e[j] = min(NV * lane + j, a.E - 1);
    bias[j] = 0.0f;
  }
  if (a.bias) {
#pragma unroll
    for (int j = 0; j < NV; ++j) bias[j] = a.bias[at_e[j]];
  }
  if (a.fp32) {
    const float* l = static_cast<const float*>(a.logits) + row;
#pragma unroll
    for (int j = 0; j < NV; ++j) x[j] = l[at_e[j]];
  } else {
    const uint16_t* l = static_cast<const uint16_t*>(a.logits) + row;
    uint32_t h[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) h[j] = l[at_e[j]];
#pragma unroll
    for (int j = 0; j < NV; ++j) x[j] = __uint_as_float(h[j] << 16);
  }
  double score[NV];
  uint64_t key[NV];
  if (!a.sigmoid) {
    float most = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < NV; ++j) most = __builtin_fmaxf(most, x[j]);
    const float top = wave_max(most);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      // (inf - inf, and a row of -inf)
      score[j] = x[j] == top ? (top == -__builtin_inff() ? 0.0 : 1.0) : exp(static_cast<double>(x[j]) - top);
      sum += NV * lane + j < a.E ? score[j] : 0.0;
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < NV; ++j) score[j] = sum == 0.0 ? 0.0 : score[j] / sum;
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) score[j] = 1.0 / (1.0 + exp(-static_cast<double>(x[j])));
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    double c = score[j] + static_cast<double>(bias[j]);
    if (x[j] == -__builtin_inff() || bias[j] == -__builtin_inff()) c = -inf;  // (the sum of NaN and -inf is NaN)
    if (c == -inf) score[j] = 0.0;
    key[j] = NV * lane + j < a.E ? choice_key(c) : 0u;
    scores[wave][NV * lane + j] = score[j];
  }

  __builtin_amdgcn_wave_barrier();

  if (a.groups > 1) {
    const int size = a.E / a.groups, lanes = size / NV;
    const bool pow2 = (lanes & (lanes - 1)) == 0;
    if (a.group_rank <= 2 && size % NV == 0 && (pow2 || lanes <= 16)) {
      // A group is lanes of its own: its best two by exchanges among them, or from one after the other (8192 tokens, 8
      // groups of 20: 16 us; group after group, as below, 27).
      uint64_t first = key[0], second = 0;
#pragma unroll
      for (int j = 1; j < NV; ++j) {
        second = max(second, min(first, key[j]));
        first = max(first, key[j]);
      }
      const int mine = lane / lanes;
      const auto join = [&](uint64_t f, uint64_t s) {
        second = max(max(second, s), min(first, f));
        first = max(first, f);
      };
      if (pow2) {
        for (int m = 1; m < lanes; m <<= 1) join(__shfl_xor(first, m, kWave), __shfl_xor(second, m, kWave));
      } else {
        const uint64_t own1 = first, own2 = second;
        int from = lane;
        for (int m = 1; m < lanes; ++m) {
          from = from + 1 < (mine + 1) * lanes ? from + 1 : mine * lanes;
          join(__shfl(own1, from, kWave), __shfl(own2, from, kWave));
        }
      }
      if (first > 1u) {  // (a group of switched off experts stays 1)
        double total = choice_of(first);
        if (a.group_rank == 2 && second > 1u) total += choice_of(second);
        first = choice_key(total);
      }
      // its place among the groups, those of equal sums in turn
      int before = 0;
      for (int g = 0; g < a.groups; ++g) {
        const uint64_t other = read_lane(first, g * lanes);
        before += other > first || (other == first && g < mine) ? 1 : 0;
      }
      if (before >= a.top_groups) {
#pragma unroll
        for (int j = 0; j < NV; ++j) key[j] = 0;
      }
    } else {
      // group after group
      uint64_t mine = 0;  // lane g: the key of group g
      for (int g = 0; g < a.groups; ++g) {
        const int lo = g * size, hi = lo + size;
        double total = 0.0;
        bool any = false;
        uint32_t taken = 0;  // of the lane's experts
        for (int r = 0; r < a.group_rank; ++r) {
          uint64_t best = 0;
          int at = 0;
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            const int e = NV * lane + j;
            if (e >= lo && e < hi && !((taken >> j) & 1u) && key[j] > best) {
              best = key[j];
              at = j;
            }
          }
          const int l = best_lane(best);
          const uint64_t k = read_lane(best, l);
          if (k <= 1u) break;  // switched off, as all that follow
          if (lane == l) taken |= 1u << at;
          any = true;
          total += choice_of(k);
        }
        if (lane == g) mine = any ? choice_key(total) : 1u;
      }
      uint64_t kept = 0;
      for (int r = 0; r < a.top_groups; ++r) {
        const int g = best_lane(mine);
        kept |= 1ull << g;
        if (lane == g) mine = 0;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e = NV * lane + j;
        if (e < a.E && !((kept >> (e / size)) & 1u)) key[j] = 0;
      }
    }
  }

  int chosen = 0;    // lane s: a choice
  int place = lane;  // and its place among them
  uint32_t high[NV], border;
#pragma unroll
  for (int j = 0; j < NV; ++j) high[j] = static_cast<uint32_t>(key[j] >> 32);
  if (NV >= 4 && a.k >= 6 && find_border(high, a.k, &border)) {
    int at = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint64_t in = __ballot(high[j] >= border);
      if (high[j] >= border) {
        const int i = at + static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(in >> 32),
                                                                      __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(in), 0)));
        few_keys[wave][i] = key[j];
        few[wave][i] = NV * lane + j;
      }
      at += __popcll(in);
    }
    __builtin_amdgcn_wave_barrier();
    const int mine = min(lane, a.k - 1);
    const uint64_t own = few_keys[wave][mine];
    chosen = few[wave][mine];
    place = 0;
    for (int i = 0; i < a.k; ++i) {
      const uint64_t other = few_keys[wave][i];
      place += other > own || (other == own && few[wave][i] < chosen) ? 1 : 0;
    }
  } else {
    uint64_t best = key[0];  // the lane's first of its largest
    int at = 0;
#pragma unroll
    for (int j = 1; j < NV; ++j)
      if (key[j] > best) {
        best = key[j];
        at = j;
      }
    for (int s = 0; s < a.k; ++s) {
      const int l = best_lane(best);
      const int e = NV * l + __builtin_amdgcn_readlane(at, l);
      chosen = lane == s ? e : chosen;
      if (lane == l) {
        best = 0;
        int next = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (j == at) key[j] = 0;
          if (key[j] > best) {
            best = key[j];
            next = j;
          }
        }
        at = next;
      }
    }
  }
  double weight = lane < a.k ? scores[wave][chosen] : 0.0;
  if (a.renormalize) {
    const double sum = wave_sum(weight);
    weight = sum == 0.0 ? 0.0 : weight / sum;
  }
  if (lane < a.k) {
    const size_t o = static_cast<size_t>(t) * static_cast<size_t>(a.k) + place;
    a.idx[o] = chosen;
    a.w[o] = static_cast<float>(weight * static_cast<double>(a.scale));
  }
}

}  // namespace

hipError_t launch_select_experts(const SelectArgs& a, hipStream_t s) {
  constexpr int kMost = 1 << 25;  // tokens of a launch, whose threads are below 2^32
  if (a.T > kMost) {
    SelectArgs part = a;
    part.T = kMost;
    const hipError_t e = launch_select_experts(part, s);
    if (e != hipSuccess) return e;
    const size_t row = static_cast<size_t>(a.stride) * (a.fp32 ? 4 : 2), slots = static_cast<size_t>(kMost) * a.k;
    part.logits = static_cast<const uint8_t*>(a.logits) + row * kMost;
    part.idx = a.idx + slots;
    part.w = a.w + slots;
    part.T = a.T - kMost;
    return launch_select_experts(part, s);
  }
  const dim3 grid((a.T + kSelectWaves - 1) / kSelectWaves), block(kSelectWaves * kWave);
  if (a.E <= 64) hipLaunchKernelGGL(select_kernel<1>, grid, block, 0, s, a);
  else if (a.E <= 128) hipLaunchKernelGGL(select_kernel<2>, grid, block, 0, s, a);
  else if (a.E <= 256) hipLaunchKernelGGL(select_kernel<4>, grid, block, 0, s, a);
  else if (a.E <= 512) hipLaunchKernelGGL(select_kernel<8>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(select_kernel<16>, grid, block, 0, s, a);
  return hipGetLastError();
}

}  // namespace gxmoe
