// mx_product.h -- what the MXFP4 product kernels share on the device.
//
// v_mfma_scale_f32_32x32x64_f8f6f4 takes both operands as they are stored: lane l
// gives row l % 32 of each, the 16 bytes of one block (l / 32 of two) and its scale
// byte.  The products of e2m1 values are exact in it and their sums have fp32's 24
// bits, across blocks of any scales and with the accumulator.  The weights are its
// first operand, so a lane ends with 16 results of one row (token) l % 32: columns
// 8 (i / 4) + 4 (l / 32) + i % 4 of the tile's 32.
//
// Blocks past a row's end (K of an odd number of blocks) are given the scale byte 0
// on both sides: whatever finite values they hold, their products are below 2^-240
// and vanish.
#pragma once

#include "mx_device.h"
#include "mx_kernels.h"

namespace gxmoe {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef gx_u32x4 u32x4_t;

__device__ __forceinline__ i32x8_t mx_operand(const u32x4_t& v) {
  return i32x8_t{static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]), static_cast<int>(v[3]), 0, 0, 0, 0};
}

// Rows [lo, hi) of expert e.
struct MTile {
  int e, lo, hi;
};

// The tile-th m-tile of `rows` rows each (the last of an expert has what is left), of
// the experts' in turn; e < 0 past the last one.  Every lane gets the same answer.
__device__ __forceinline__ MTile find_m_tile(const MxProductArgs& a, int tile, int rows, int lane) {
  if (!a.offsets) {
    const int lo = tile * rows;
    return lo < a.rows ? MTile{0, lo, min(lo + rows, a.rows)} : MTile{-1, 0, 0};
  }
  int before = 0;
  for (int base = 0; base < a.E; base += kWave) {
    const int e = base + lane;
    int lo = 0, hi = 0;
    if (e < a.E) {
      lo = min(max(a.offsets[e], 0), a.rows);  // whatever they hold, rows of the call
      hi = min(max(a.offsets[e + 1], lo), a.rows);
    }
    const int n = (hi - lo + rows - 1) / rows;
    int upto = n;
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
      const int v = __shfl_up(upto, m, kWave);
      if (lane >= m) upto += v;
    }
    const uint64_t past = __ballot(before + upto > tile);
    if (past != 0ull) {
      const int l = __builtin_ctzll(past);
      const int first = before + __shfl(upto - n, l, kWave);
      lo = __shfl(lo, l, kWave);
      hi = __shfl(hi, l, kWave);
      const int p = lo + (tile - first) * rows;
      return MTile{base + l, p, min(p + rows, hi)};
    }
    before += __shfl(upto, kWave - 1, kWave);
  }
  return MTile{-1, 0, 0};
}

// How many there are; whatever the offsets hold, not more than most_m_tiles().
__device__ __forceinline__ int count_m_tiles(const MxProductArgs& a, int rows, int lane) {
  if (!a.offsets) return (a.rows + rows - 1) / rows;
  const int most = a.rows / rows + min(a.E, a.rows);
  int n = 0;
  for (int e = lane; e < a.E; e += kWave) {
    const int lo = min(max(a.offsets[e], 0), a.rows), hi = min(max(a.offsets[e + 1], lo), a.rows);
    n += (hi - lo + rows - 1) / rows;
  }
  n = min(n, most);
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) n += __shfl_xor(n, m, kWave);
  return min(__builtin_amdgcn_readfirstlane(n), most);
}

// Row of a that result row p reads, -1 for one of zeros.
__device__ __forceinline__ int source_row(const MxProductArgs& a, int p) {
  const int src = a.row_index ? a.row_index[p] : p;
  return src >= 0 && src < a.a_rows ? src : -1;
}

// The same of several: their loads go out together.
template <int N>
__device__ __forceinline__ void source_rows(const MxProductArgs& a, int (&p)[N]) {
  if (a.row_index) {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = a.row_index[p[i]];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = p[i] >= 0 && p[i] < a.a_rows ? p[i] : -1;
}

// The lane's 16 results of a block of 32 columns (as both halves of the wave hold them)
// to MXFP4: eight of its 16 bytes each, and the scale byte.  kPairs: the lane's values
// are columns 4 q + 2 half + {0, 1} (after SwiGLU), otherwise 8 q + 4 half + {0 .. 3}.
template <bool kPairs>
__device__ __forceinline__ gx_u32x2 quantize_block(const float (&v)[16], uint32_t& code) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) top = max(top, mx_magnitude(v[j]));
  const auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);
  code = mx_scale_byte(max(both[0], both[1]));
  const float lo[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
  const float hi[8] = {v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]};
  // the lower lanes take what belongs to the first eight bytes, the upper the rest:
  // r[0] from the even (half 0) columns' lanes, r[1] from the odd ones'
  const auto r = __builtin_amdgcn_permlane32_swap(mx_pack8(lo, code), mx_pack8(hi, code), false, false);
  // v_perm_b32: bytes 0-3 of the second operand, 4-7 of the first
  if constexpr (kPairs)
    return gx_u32x2{__builtin_amdgcn_perm(r[1], r[0], 0x05010400u), __builtin_amdgcn_perm(r[1], r[0], 0x07030602u)};
  else
    return gx_u32x2{__builtin_amdgcn_perm(r[1], r[0], 0x05040100u), __builtin_amdgcn_perm(r[1], r[0], 0x07060302u)};
}

}  // namespace gxmoe
