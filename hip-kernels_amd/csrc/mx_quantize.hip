// mx_quantize.hip -- rows to MXFP4 and back.
//
// A block of 32 values gets the power of two 2^e, e = max(floor(log2 of the largest magnitude) - 2, -126), taken
// from that magnitude's bits, and each value over it is rounded to the nearest e2m1 number by the
// hardware's conversion.  Four lanes hold a block, eight values each, so that loads are of 16 bytes and two exchanges
// give the largest.  Bound by memory: 46080 x 2880 from bf16 59 us (5.7 TB/s), from fp32 114 (5.3), back
// to bf16 65 (5.2); small ones by the launch: 8 x 2880 1.8.
#include "mx_device.h"
#include "mx_kernels.h"

namespace gxmoe {

namespace {

constexpr int kThreads = 256;

template <bool F32>
__device__ __forceinline__ void load8(const void* x, size_t at, float (&v)[8]) {
  if constexpr (F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + at);
    const float4 a = p[0], b = p[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const gx_u32x4 a = *reinterpret_cast<const gx_u32x4*>(static_cast<const uint16_t*>(x) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(a[i] << 16);
      v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
    }
  }
}

// Eight values per lane, a block per four lanes.  `step` threads are there (gridDim would be a hidden
// argument, for which the host takes 0.8 us more).
template <bool F32>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const void* x, size_t stride, size_t units, uint32_t per_row,
                                                            uint8_t* packed, uint8_t* scales, uint32_t step) {
  for (size_t u = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x; u < units; u += step) {
    const size_t row = u / per_row;
    float v[8];
    load8<F32>(x, row * stride + 8 * (u - row * per_row), v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, mx_magnitude(v[i]));
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1, kWave)));
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2, kWave)));
    const uint32_t code = mx_scale_byte(top);
    reinterpret_cast<uint32_t*>(packed)[u] = mx_pack8(v, code);
    if ((u & 3) == 0) scales[u >> 2] = static_cast<uint8_t>(code);
  }
}

// 16 bytes of results per lane: eight bf16 values, or four fp32 (with eight of those every store would
// leave half of each line to the next: 46080 x 2880 takes 135 us, with eight 157).
template <bool F32>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint8_t* packed, const uint8_t* scales, size_t units,
                                                              uint32_t per_row, void* out, size_t stride,
                                                              uint32_t step) {
  constexpr int kV = F32 ? 4 : 8;
  for (size_t u = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x; u < units; u += step) {
    const size_t row = u / per_row;
    uint32_t d;
    if constexpr (F32) d = reinterpret_cast<const uint16_t*>(packed)[u];
    else d = reinterpret_cast<const uint32_t*>(packed)[u];
    const uint32_t code = scales[u / (32 / kV)];
    // 2^-127 is a denormal number; 255 is NaN
    const float scale = __uint_as_float(code == 0u ? 0x00400000u : code == 255u ? 0x7fc00000u : code << 23);
    float v[8];
    fp4x2_to_f32<0>(d, 1.0f, v[0], v[1]);
    fp4x2_to_f32<1>(d, 1.0f, v[2], v[3]);
    if constexpr (!F32) {
      fp4x2_to_f32<2>(d, 1.0f, v[4], v[5]);
      fp4x2_to_f32<3>(d, 1.0f, v[6], v[7]);
    }
#pragma unroll
    for (int i = 0; i < kV; ++i) v[i] *= scale;
    const size_t at = row * stride + kV * (u - row * per_row);
    if constexpr (F32)
      *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = float4{v[0], v[1], v[2], v[3]};
    else
      *reinterpret_cast<gx_u32x4*>(static_cast<uint16_t*>(out) + at) = gx_u32x4{
          pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
  }
}

dim3 grid_of(size_t units) {
  const size_t n = (units + kThreads - 1) / kThreads;
  return dim3(static_cast<uint32_t>(n < 16384 ? n : 16384));
}

}  // namespace

hipError_t launch_mx_quantize(const void* x, int64_t stride, bool fp32, int rows, int K, uint8_t* packed, uint8_t* scales,
                              hipStream_t s) {
  const size_t units = static_cast<size_t>(rows) * static_cast<size_t>(K / 8);
  const dim3 grid = grid_of(units), block(kThreads);
  const uint32_t per_row = static_cast<uint32_t>(K / 8);
  if (fp32)
    hipLaunchKernelGGL(quantize_kernel<true>, grid, block, 0, s, x, static_cast<size_t>(stride), units, per_row, packed, scales,
                       grid.x * kThreads);
  else
    hipLaunchKernelGGL(quantize_kernel<false>, grid, block, 0, s, x, static_cast<size_t>(stride), units, per_row, packed, scales,
                       grid.x * kThreads);
  return hipGetLastError();
}

hipError_t launch_mx_dequantize(const uint8_t* packed, const uint8_t* scales, int rows, int K, void* out, int64_t stride,
                                bool fp32, hipStream_t s) {
  const uint32_t per_row = static_cast<uint32_t>(K / (fp32 ? 4 : 8));
  const size_t units = static_cast<size_t>(rows) * per_row;
  const dim3 grid = grid_of(units), block(kThreads);
  if (fp32)
    hipLaunchKernelGGL(dequantize_kernel<true>, grid, block, 0, s, packed, scales, units, per_row, out, static_cast<size_t>(stride),
                       grid.x * kThreads);
  else
    hipLaunchKernelGGL(dequantize_kernel<false>, grid, block, 0, s, packed, scales, units, per_row, out, static_cast<size_t>(stride),
                       grid.x * kThreads);
  return hipGetLastError();
}

}  // namespace gxmoe
