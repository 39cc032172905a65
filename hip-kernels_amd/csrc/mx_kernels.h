// mx_kernels.h -- launchers of the expert selection and of the MXFP4 operators (internal).
//
// MXFP4 here is row-major: a matrix of [rows][K] values is packed [rows][K / 2]
// (low nibble = even k) and scales [rows][K / 32], value = e2m1 * 2^(scale - 127),
// a scale byte of 255 is NaN.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace gxmoe {

constexpr int kSelectMaxExperts = 1024;
constexpr int kSelectMaxTopK = 32;
constexpr int kSelectMaxGroups = 64;

struct SelectArgs {
  const void* logits;  // [T] rows of E, `stride` elements apart
  int64_t stride;
  const float* bias;   // [E] or null
  int32_t* idx;        // [T][k]
  float* w;            // [T][k]
  int T, E, k;
  int groups, top_groups, group_rank;
  bool fp32, sigmoid, renormalize;
  float scale;
};
hipError_t launch_select_experts(const SelectArgs& a, hipStream_t s);

// x: rows of K bf16 or fp32 values, `stride` elements apart.
hipError_t launch_mx_quantize(const void* x, int64_t stride, bool fp32, int rows, int K, uint8_t* packed, uint8_t* scales,
                              hipStream_t s);
hipError_t launch_mx_dequantize(const uint8_t* packed, const uint8_t* scales, int rows, int K, void* out, int64_t stride,
                                bool fp32, hipStream_t s);

constexpr int kMxMaxExperts = 1024;

// y[p][n] = sum_k a[row(p)][k] * w_e[n][k] + bias[e][n] for the rows p of expert
// e, [offsets[e], offsets[e + 1]); one expert of all rows without offsets.
struct MxProductArgs {
  const uint8_t* a;     // packed, [a_rows][K / 2]
  const uint8_t* as;    // scales, [a_rows][K / 32]
  const int32_t* row_index;  // [rows] or null: row(p) = p
  const int32_t* offsets;    // [E + 1] or null
  const uint8_t* w;     // [E][N][K / 2]
  const uint8_t* ws;    // [E][N][K / 32]
  const uint16_t* bias; // [E][N] or null
  // Values (bf16, or fp32), rows `stride` elements apart; or MXFP4, packed and scales.
  void* out;
  uint8_t* out_scales;
  int64_t stride;
  int a_rows, rows, E, N, K;
  float alpha, limit;  // of SwiGLU
  bool swiglu, out_fp32;
  bool vec;  // out's rows and their pieces of 16 bytes are on 16 bytes

  __host__ __device__ bool quantized() const { return out_scales != nullptr; }
};
// A launch whose arguments take 128 bytes or more, or that needs the hidden ones (gridDim),
// costs the host 3.5 us, a smaller one 2.7.
static_assert(sizeof(MxProductArgs) + sizeof(int) <= 116, "");
constexpr int kMxCus = 256;  // of the card

// m-tiles of `rows` rows that the call can have: each expert's last one may be a part.
inline int64_t most_m_tiles(const MxProductArgs& a, int rows) {
  return a.offsets ? a.rows / rows + (a.E < a.rows ? a.E : a.rows) : (static_cast<int64_t>(a.rows) + rows - 1) / rows;
}

// Tiles of 256 x 256, of 128 x 128 (rows x columns) or of 32 x 128.
enum class MxTile { large, middle, low };
hipError_t launch_mx_tile(const MxProductArgs& a, MxTile kind, hipStream_t s);
// 16 rows x 16 columns of a wave, 32 if `wide` (so for MXFP4 results); four waves along K if `split`.
constexpr int kStreamRows = 16;
hipError_t launch_mx_stream(const MxProductArgs& a, bool wide, bool split, hipStream_t s);
hipError_t launch_mx_product(const MxProductArgs& a, hipStream_t s);

}  // namespace gxmoe
