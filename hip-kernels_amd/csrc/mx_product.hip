// mx_product.hip -- products of MXFP4 rows with MXFP4 weights on the block-scaled
// matrix cores, dense and grouped by expert.
//
// v_mfma_scale_f32_32x32x64_f8f6f4 takes both operands as they are stored: lane l
// gives row l % 32 of each, the 16 bytes of one block (l / 32 of two) and its scale
// byte.  The products of e2m1 values are exact in it and their sums have fp32's 24
// bits, across blocks of any scales and with the accumulator.  The weights are its
// first operand, so a lane ends with 16 results of one row (token) l % 32: columns
// 8 (i / 4) + 4 (l / 32) + i % 4 of the tile's 32.
#include <cstdio>
#include <cstdlib>
#include "mx_device.h"
#include "mx_kernels.h"

namespace gxmoe {

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

constexpr int kTileM = 32;   // rows of a
constexpr int kTileN = 64;   // weight rows of a wave
constexpr int kWaves = 4;

// Rows [lo, hi) of expert e of m-tile `tile`, from the offsets; e < 0 past the last tile.
struct MTile {
  int e, lo, hi;
};

__device__ __forceinline__ MTile find_tile(const MxProductArgs& a, int tile, int lane) {
  if (!a.offsets) {
    const int lo = tile * kTileM;
    return lo < a.rows ? MTile{0, lo, min(lo + kTileM, a.rows)} : MTile{-1, 0, 0};
  }
  int before = 0;
  for (int base = 0; base < a.E; base += kWave) {
    const int e = base + lane;
    int lo = 0, hi = 0;
    if (e < a.E) {
      lo = min(max(a.offsets[e], 0), a.rows);  // whatever they hold, rows of the call
      hi = min(max(a.offsets[e + 1], lo), a.rows);
    }
    const int n = (hi - lo + kTileM - 1) / kTileM;
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
      const int p = lo + (tile - first) * kTileM;
      return MTile{base + l, p, min(p + kTileM, hi)};
    }
    before += __shfl(upto, kWave - 1, kWave);
  }
  return MTile{-1, 0, 0};
}

// A wave: 32 rows x 64 weight rows.
__global__ __launch_bounds__(kWaves * kWave) void product_kernel(MxProductArgs a, int n_groups) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const MTile mt = find_tile(a, blockIdx.x / n_groups, lane);
  const int n0 = ((blockIdx.x % n_groups) * kWaves + wave) * kTileN;
  if (mt.e < 0 || n0 >= a.N) return;  // no barrier below

  const int r = lane & 31, half = lane >> 5;
  const int nb = a.K / 32;
  const size_t row_bytes = static_cast<size_t>(a.K) / 2;
  const int p = mt.lo + r;
  const bool live = p < mt.hi;
  int src = live ? (a.row_index ? a.row_index[p] : p) : 0;
  const bool found = live && src >= 0 && src < a.a_rows;  // other rows are zeros
  src = found ? src : 0;
  const uint8_t* ap = a.a + static_cast<size_t>(src) * row_bytes;
  const uint8_t* asp = a.as + static_cast<size_t>(src) * nb;
  const uint8_t* wp[2];
  const uint8_t* wsp[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const size_t n = static_cast<size_t>(mt.e) * a.N + min(n0 + 32 * i + r, a.N - 1);
    wp[i] = a.w + n * row_bytes;
    wsp[i] = a.ws + n * nb;
  }

  f32x16_t acc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;

  for (int s = 0; 2 * s < nb; ++s) {
    const int b = 2 * s + half;
    const bool in = b < nb;
    const int bb = in ? b : nb - 1;  // a block past the end is one of zeros
    gx_u32x4 av = *reinterpret_cast<const gx_u32x4*>(ap + 16 * static_cast<size_t>(bb));
    int sa = asp[bb];
    if (!in || !found) {
      av = gx_u32x4{0u, 0u, 0u, 0u};
      sa = 127;
    }
    const i32x8_t ao{static_cast<int>(av[0]), static_cast<int>(av[1]), static_cast<int>(av[2]), static_cast<int>(av[3]),
                     0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const gx_u32x4 wv = *reinterpret_cast<const gx_u32x4*>(wp[i] + 16 * static_cast<size_t>(bb));
      const int sw = in ? wsp[i][bb] : 127;
      const i32x8_t wo{static_cast<int>(wv[0]), static_cast<int>(wv[1]), static_cast<int>(wv[2]),
                       static_cast<int>(wv[3]), 0, 0, 0, 0};
      acc[i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wo, ao, acc[i], 4, 4, 0, sw, 0, sa);
    }
  }

  // column of acc[i][4 q + j]: n0 + 32 i + 8 q + 4 half + j
  if (a.bias) {
    const uint16_t* bias = a.bias + static_cast<size_t>(mt.e) * a.N;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int n = n0 + 32 * i + 8 * (j / 4) + 4 * half + j % 4;
        acc[i][j] += bf16_to_f32(bias[min(n, a.N - 1)]);
      }
  }
  const int cols = a.swiglu ? a.N / 2 : a.N;
  if (a.swiglu) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = mx_swiglu(acc[i][2 * j], acc[i][2 * j + 1], a.alpha, a.limit);
  }

  if (a.out_packed) {
    // a block of 32 columns: those of both halves
    const size_t ob = static_cast<size_t>(p) * (cols / 32);
    auto block = [&](const float (&v)[16], int column) __attribute__((always_inline)) {  // lane's 16 of the block
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) top = max(top, mx_magnitude(v[j]));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, kWave)));
      const uint32_t code = mx_scale_byte(top);
      const float lo[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
      const float hi[8] = {v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]};
      const uint32_t c0 = mx_pack8(lo, code), c1 = mx_pack8(hi, code);
      if (live && column < cols) {
        uint8_t* o = a.out_packed + (ob + column / 32) * 16;
        if (a.swiglu) {  // the lane's values are columns 4 q + 2 half + {0, 1}, q = 0..7
#pragma unroll
          for (int q = 0; q < 8; ++q) o[2 * q + half] = static_cast<uint8_t>((q < 4 ? c0 : c1) >> (8 * (q & 3)));
        } else {  // columns 8 q + 4 half + {0 .. 3}, q = 0..3
#pragma unroll
          for (int q = 0; q < 4; ++q)
            reinterpret_cast<uint16_t*>(o)[2 * q + half] = static_cast<uint16_t>((q < 2 ? c0 : c1) >> (16 * (q & 1)));
        }
        if (half == 0) a.out_scales[ob + column / 32] = static_cast<uint8_t>(code);
      }
    };
    if (a.swiglu) {
      float v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = acc[j / 8][j % 8];
      block(v, n0 / 2);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = acc[i][j];
        block(v, n0 + 32 * i);
      }
    }
    return;
  }
  if (!live) return;
  const size_t row = static_cast<size_t>(p) * static_cast<size_t>(a.stride);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int n = a.swiglu ? n0 / 2 + 16 * i + 4 * (j / 2) + 2 * half + j % 2 : n0 + 32 * i + 8 * (j / 4) + 4 * half + j % 4;
      if (n < cols && (j < 8 || !a.swiglu)) {
        if (a.out_fp32) static_cast<float*>(a.out)[row + n] = acc[i][j];
        else static_cast<uint16_t*>(a.out)[row + n] = f32_to_bf16(acc[i][j]);
      }
    }
}

}  // namespace

hipError_t launch_mx_product(const MxProductArgs& a, hipStream_t s) {
  const char* f = getenv("MX_FORCE");
  if (f) {
    int nt, mt, ks;
    if (f[0] == 't') return launch_mx_tile(a, s);
    if (sscanf(f, "%d,%d,%d", &nt, &mt, &ks) == 3 && a.K >= 512) return launch_mx_stream(a, a.out_packed ? 2 : nt, mt, ks, s);
  }
  if (a.rows > 64) return launch_mx_tile(a, s);
  const int tiles = a.offsets ? a.rows / kTileM + (a.E < a.rows ? a.E : a.rows) : (a.rows + kTileM - 1) / kTileM;
  const int n_groups = (a.N + kWaves * kTileN - 1) / (kWaves * kTileN);
  hipLaunchKernelGGL(product_kernel, dim3(static_cast<uint32_t>(tiles) * static_cast<uint32_t>(n_groups)),
                     dim3(kWaves * kWave), 0, s, a, n_groups);
  return hipGetLastError();
}

}  // namespace gxmoe
