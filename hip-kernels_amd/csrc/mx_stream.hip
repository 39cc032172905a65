// mx_stream.hip -- MXFP4 products of few rows: the weights stream through LDS, wave by
// wave.
//
// A wave computes up to 16 MT rows x 16 NT columns over its share of K with
// v_mfma_scale_f32_16x16x128_f8f6f4 (lane l gives row l % 16 of each operand and block l / 16 of
// four; it ends with columns 4 (l / 16) + {0 .. 3} of row l % 16).  K goes in chunks of eight
// blocks: a line (128 bytes) of each of its weight rows reaches its own ring of D stages by direct
// global -> LDS loads, and comes out in the operands' order; no wave waits for another.  (Loads straight to
// the operands' registers take 64 bytes of a row at a time, and the memory then gives half: 64 tokens over
// 128 experts 453 us.)  The rows of a, few and read by all, go to registers D chunks ahead.
//
// A wave goes through a run of neighbouring tiles of the same rows, and the loads of the next
// tile's chunks follow those of the last without a pause.  A tile's K goes in spans of
// up to 128 blocks, whose weights' scales are loaded during the span before and put
// into LDS between the two.  Where tiles are few, KS waves share a tile's K, and their
// sums meet in LDS in a fixed order.
#include "mx_product.h"

namespace gxmoe {

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef u32x4_t __attribute__((aligned(1))) loose_u32x4;
typedef uint32_t __attribute__((aligned(1))) loose_u32;
typedef __attribute__((address_space(3))) void lds_void_t;

// Blocks whose scales are in LDS at a time: whole turns of the ring.
__host__ __device__ constexpr int span_blocks(int D) { return 16 / D * D * 8; }

template <int N>
__device__ __forceinline__ void wait_vm() {  // vmcnt(N), the other counters as they are
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0f70);
}

// Bytes between the scales of two rows: an odd number of 16, so that 16 rows meet all banks.
__host__ __device__ constexpr int scale_pitch(int nb, int D) {
  const int p = ((nb < span_blocks(D) ? nb : span_blocks(D)) + 15) / 16;
  return 16 * (p | 1);
}

// Of a wave: its ring, or its sums if more, and its scales.
template <int NT, int MT, int D>
__host__ __device__ constexpr int ring_bytes() {
  return D * NT * 2048 > NT * MT * 1024 ? D * NT * 2048 : NT * MT * 1024;
}

// The results of row p, columns n0 + 16 i + 4 (lane / 16) + {0 .. 3} of each lane: bias, SwiGLU and the store.
template <int NT>
__device__ __forceinline__ void write_rows(const MxProductArgs& a, const f32x4_t (&sum)[NT], int e, int n0, int p, bool live,
                                           bool zero, int lane) {
  const int r = lane & 15, g = lane >> 4;
  const int cols = a.swiglu ? a.N / 2 : a.N;
  f32x4_t bias[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) bias[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  if (a.bias) {
    const uint16_t* row = a.bias + static_cast<size_t>(e) * a.N;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) bias[i][q] = bf16_to_f32(row[min(n0 + 16 * i + 4 * g + q, a.N - 1)]);
  }
      float v[NT][4];
  #pragma unroll
      for (int i = 0; i < NT; ++i)
  #pragma unroll
        for (int q = 0; q < 4; ++q) v[i][q] = (zero ? 0.0f : sum[i][q]) + bias[i][q];
      if (a.swiglu) {
  #pragma unroll
        for (int i = 0; i < NT; ++i)
  #pragma unroll
          for (int q = 0; q < 2; ++q) v[i][q] = mx_swiglu(v[i][2 * q], v[i][2 * q + 1], a.alpha, a.limit);
      }
      if (a.out_packed) {
        const size_t ob = static_cast<size_t>(p) * (cols / 32);
        constexpr int kPer = 2;  // column tiles of a block without SwiGLU
        if (a.swiglu) {
          if constexpr (NT == 4) {  // the block of 32: columns 8 i + 2 g + {0, 1}, byte 4 i + g
            uint32_t top = 0;
  #pragma unroll
            for (int i = 0; i < NT; ++i) top = max(top, max(mx_magnitude(v[i][0]), mx_magnitude(v[i][1])));
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, kWave)));
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, kWave)));
            const uint32_t code = mx_scale_byte(top);
            const float x[8] = {v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
            const uint32_t mine = mx_pack8(x, code);  // byte i of the lane is byte 4 i + g of the block
            uint32_t d = 0;                           // dword g of the block
  #pragma unroll
            for (int q = 0; q < 4; ++q)
              d |= ((static_cast<uint32_t>(__shfl(static_cast<int>(mine), r + 16 * q, kWave)) >> (8 * g)) & 0xffu) << (8 * q);
            if (live && n0 / 2 < cols) {
              reinterpret_cast<uint32_t*>(a.out_packed)[4 * (ob + n0 / 64) + g] = d;
              if (g == 0) a.out_scales[ob + n0 / 64] = static_cast<uint8_t>(code);
            }
          }
        } else if constexpr (NT >= kPer) {
  #pragma unroll
          for (int i = 0; i < NT; i += kPer) {  // columns 16 i + 4 g + {0 .. 3} and 16 further on
            uint32_t top = 0;
  #pragma unroll
            for (int q = 0; q < 4; ++q) top = max(top, max(mx_magnitude(v[i][q]), mx_magnitude(v[i + 1][q])));
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, kWave)));
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, kWave)));
            const uint32_t code = mx_scale_byte(top);
            const float y[8] = {v[i][0], v[i][1], v[i][2], v[i][3], v[i + 1][0], v[i + 1][1], v[i + 1][2], v[i + 1][3]};
            const uint32_t d = mx_pack8(y, code);
            const int n = n0 + 16 * i;
            if (live && n < cols) {
              uint16_t* o = reinterpret_cast<uint16_t*>(a.out_packed + 16 * (ob + n / 32));
              o[g] = static_cast<uint16_t>(d);
              o[4 + g] = static_cast<uint16_t>(d >> 16);
              if (g == 0) a.out_scales[ob + n / 32] = static_cast<uint8_t>(code);
            }
          }
        }
        return;
      }
      if (!live) return;
      const size_t row = static_cast<size_t>(p) * static_cast<size_t>(a.stride);
  #pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (a.swiglu) {
          const int n = (n0 + 16 * i) / 2 + 2 * g;
          if (a.vec && n + 2 <= cols) {
            if (a.out_fp32) *reinterpret_cast<float2*>(static_cast<float*>(a.out) + row + n) = float2{v[i][0], v[i][1]};
            else *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + row + n) = pack_bf16x2(v[i][0], v[i][1]);
          } else {
  #pragma unroll
            for (int q = 0; q < 2; ++q)
              if (n + q < cols) {
                if (a.out_fp32) static_cast<float*>(a.out)[row + n + q] = v[i][q];
                else static_cast<uint16_t*>(a.out)[row + n + q] = f32_to_bf16(v[i][q]);
              }
          }
        } else {
          const int n = n0 + 16 * i + 4 * g;
          if (a.vec && n + 4 <= cols) {
            if (a.out_fp32)
              *reinterpret_cast<float4*>(static_cast<float*>(a.out) + row + n) = float4{v[i][0], v[i][1], v[i][2], v[i][3]};
            else
              *reinterpret_cast<gx_u32x2*>(static_cast<uint16_t*>(a.out) + row + n) =
                  gx_u32x2{pack_bf16x2(v[i][0], v[i][1]), pack_bf16x2(v[i][2], v[i][3])};
          } else {
  #pragma unroll
            for (int q = 0; q < 4; ++q)
              if (n + q < cols) {
                if (a.out_fp32) static_cast<float*>(a.out)[row + n + q] = v[i][q];
                else static_cast<uint16_t*>(a.out)[row + n + q] = f32_to_bf16(v[i][q]);
              }
          }
        }
      }
}

template <int NT, int MT, int KS, int D>
__device__ __forceinline__ void stream_tiles(const MxProductArgs& a, int n_tiles, uint8_t* lds) {
  constexpr int kM = 16 * MT, kN = 16 * NT, kSpan = span_blocks(D);
  constexpr int kLoads = 2 * NT + 4 * MT;  // of a chunk
  constexpr int kLanes = kWave / kN;       // per weight row, for its scales
  constexpr int kPieces = ((kSpan + 15) / 16 + kLanes - 1) / kLanes;
  static_assert((D - 1) * kLoads < 64, "vmcnt range");
  const int lane = threadIdx.x & (kWave - 1), k = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // this work-group's run of tiles, the columns of an m-tile in turn; XCD b % 8 has neighbouring runs
  const int m_tiles = count_m_tiles(a, kM, lane);
  const int64_t total = static_cast<int64_t>(m_tiles) * n_tiles;
  const int b = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  int id = static_cast<int>(total * b / gridDim.x);
  const int id_end = static_cast<int>(total * (b + 1) / gridDim.x);

  const int r = lane & 15, g = lane >> 4;
  const int nb = a.K / 32, chunks = (nb + 7) / 8;
  const int per = (chunks + KS - 1) / KS;
  const int first = k * per, last = min(first + per, chunks);  // this wave's chunks, maybe none
  const int begin = 8 * first, end = min(8 * last, nb);        // its blocks
  const size_t row_bytes = 16 * static_cast<size_t>(nb);
  const int pitch = scale_pitch(nb, D);
  uint8_t* const ring = lds + k * ring_bytes<NT, MT, D>();
  uint8_t* const scales = lds + KS * ring_bytes<NT, MT, D>() + k * (kN * pitch);
  // lane's piece of a load of eight weight rows: row lane / 8, and of the chunk's blocks the one that lies at
  // place lane % 8 (block b of row r: at b ^ (r / 2) % 8, so that 16 rows at one block meet all banks)
  const int place[2] = {(lane & 7) ^ (lane >> 4), (lane & 7) ^ (4 + (lane >> 4))};

  while (id < id_end) {
    const int m = id / n_tiles;
    int n0 = (id - m * n_tiles) * kN;
    int left = min(id_end, (m + 1) * n_tiles) - id;  // tiles of these rows
    id += left;
    const MTile mt = find_m_tile(a, m, kM, lane);
    const uint8_t *ap[MT], *asp[MT];
    bool zero[MT];
    {
      int src[MT];
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int p = min(mt.lo + 16 * j + r, mt.hi - 1);  // past the last row: that one
        src[j] = a.row_index ? a.row_index[p] : p;
      }
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        zero[j] = src[j] < 0 || src[j] >= a.a_rows;  // not a row of a: its result is replaced
        src[j] = zero[j] ? 0 : src[j];
        ap[j] = a.a + static_cast<size_t>(src[j]) * row_bytes;
        asp[j] = a.as + static_cast<size_t>(src[j]) * nb;
      }
    }
    const uint8_t* const w = a.w + static_cast<size_t>(mt.e) * a.N * row_bytes;
    const uint8_t* const ws = a.ws + static_cast<size_t>(mt.e) * a.N * nb;

    u32x4_t av[D][2][MT];
    uint32_t sa[D][2][MT];
    // Loads of the chunk at block `block` of the columns from n on.  Blocks past the end are the last one again: there are no
    // branches around loads, which would cost waits for all of them.
    auto issue = [&](int slot, int n, int block) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t at = min(block + 4 * q + g, end - 1);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          av[slot][q][j] = *reinterpret_cast<const u32x4_t*>(ap[j] + 16 * static_cast<size_t>(at));
          sa[slot][q][j] = asp[j][at];
        }
      }
      const uint8_t* from[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) from[i] = w + 16 * static_cast<size_t>(static_cast<uint32_t>(min(block + place[i], end - 1)));
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i) {
        const uint32_t row = min(n + 8 * i + (lane >> 3), a.N - 1);
        __builtin_amdgcn_global_load_lds(from[i & 1] + static_cast<uint64_t>(row) * static_cast<uint32_t>(row_bytes),
                                         (lds_void_t*)(ring + slot * (NT * 2048) + 1024 * i), 16, 0, 0);
      }
    };
    // Scales of the columns from n on, blocks from `span` on: 16 at a time, the last ones those at the row's end.
    u32x4_t sreg[kPieces];
    auto load_scales = [&](int n, int span) __attribute__((always_inline)) {
      const uint8_t* row = ws + static_cast<size_t>(static_cast<uint32_t>(min(n + lane / kLanes, a.N - 1))) * nb;
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        sreg[i] = *reinterpret_cast<const loose_u32x4*>(row + min(span + 16 * (i * kLanes + lane % kLanes), nb - 16));
    };
    auto put_scales = [&]() __attribute__((always_inline)) {
      uint8_t* row = scales + lane / kLanes * pitch;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int piece = i * kLanes + lane % kLanes;
        if (16 * piece < pitch) *reinterpret_cast<u32x4_t*>(row + 16 * piece) = sreg[i];
      }
    };

    f32x4_t acc[NT][MT];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    };
    clear();
    int span = begin;
    if (begin < end) {
      load_scales(n0, begin);
#pragma unroll
      for (int i = 0; i < D; ++i) issue(i, n0, begin + 8 * i);
      __builtin_amdgcn_sched_barrier(0);
      put_scales();
    }
    for (;;) {
      const bool ends = span + kSpan >= end;  // the tile's last span
      if (begin < end) {
        // The next span, of this tile or of the next one.  (Behind the last tile of the rows: the last one once more, for
        // nothing.)
        const int next_n = ends && left > 1 ? n0 + kN : n0, next_span = ends ? begin : span + kSpan;
        load_scales(next_n, next_span);
        __builtin_amdgcn_sched_barrier(0);
        const int upto = min(span + kSpan, end);
        const int turns = (upto - span + 8 * D - 1) / (8 * D);
        int c = 0;
        do {
          const bool next = c + 1 == turns;  // what is loaded belongs to the next span
          const int n_load = next ? next_n : n0, from = next ? next_span : span + 8 * D * (c + 1);
#pragma unroll
          for (int slot = 0; slot < D; ++slot) {
            wait_vm<(D - 1) * kLoads>();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int block = span + 8 * (D * c + slot) + 4 * q + g;
              const bool in = block < upto;  // blocks past the end are zeros of a
              const int at = min(block, upto - 1), piece = (at - span) >> 4;
              const int place_s = 16 * piece + at - min(span + 16 * piece, nb - 16);
              u32x4_t wv[NT], x[MT];
              uint32_t sw[NT];
#pragma unroll
              for (int i = 0; i < NT; ++i) {
                wv[i] = *reinterpret_cast<const u32x4_t*>(ring + slot * (NT * 2048) + (16 * i + r) * 128 +
                                                          16 * ((4 * q + g) ^ ((r >> 1) & 7)));
                sw[i] = scales[(16 * i + r) * pitch + place_s];
              }
#pragma unroll
              for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int d = 0; d < 4; ++d) x[j][d] = in ? av[slot][q][j][d] : 0u;
#pragma unroll
              for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < MT; ++j)
                  acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(wv[i]), mx_operand(x[j]), acc[i][j],
                                                                               4, 4, 0, static_cast<int>(sw[i]), 0,
                                                                               static_cast<int>(sa[slot][q][j]));
            }
            __builtin_amdgcn_s_waitcnt(0xc07f);  // the stage has been read
            __builtin_amdgcn_sched_barrier(0);
            issue(slot, n_load, from + 8 * slot);
            __builtin_amdgcn_sched_barrier(0);
          }
        } while (++c < turns);
        put_scales();
        span = next_span;
        if (!ends) continue;
      }
      if constexpr (KS > 1) {
        // Wave k sums row tile k of all waves, in turn.  (No load may still land in the rings.)
        wait_vm<0>();
        f32x4_t* const sums = reinterpret_cast<f32x4_t*>(lds);
        constexpr int kSums = ring_bytes<NT, MT, D>() / 16;  // between two waves'
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < MT; ++j) sums[k * kSums + (i * MT + j) * kWave + lane] = acc[i][j];
        __syncthreads();
        constexpr int kOwn = (MT + KS - 1) / KS;  // (of KS = 2 a wave has two of four row tiles)
#pragma unroll
        for (int o = 0; o < kOwn; ++o) {
          const int j = k + KS * o;
          if (j >= MT) break;
          f32x4_t v[NT];
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            v[i] = sums[(i * MT + j) * kWave + lane];
#pragma unroll
            for (int q = 1; q < KS; ++q) v[i] += sums[q * kSums + (i * MT + j) * kWave + lane];
          }
          const int p = mt.lo + 16 * j + r;
          write_rows<NT>(a, v, mt.e, n0, p, p < mt.hi, p < mt.hi && source_row(a, p) < 0, lane);
        }
        return;  // a work-group of several waves has one tile
      } else {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const int p = mt.lo + 16 * j + r;
          f32x4_t v[NT];
#pragma unroll
          for (int i = 0; i < NT; ++i) v[i] = acc[i][j];
          write_rows<NT>(a, v, mt.e, n0, p, p < mt.hi, zero[j], lane);
        }
        clear();
      }
      n0 += kN;
      if (--left == 0) break;
    }
    wait_vm<0>();  // no load may still land in the ring
  }
}

template <int NT, int MT, int KS, int D>
__global__ __launch_bounds__(KS * kWave) void stream_kernel(MxProductArgs a, int n_tiles) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  stream_tiles<NT, MT, KS, D>(a, n_tiles, lds);
}

template <int NT, int MT, int KS, int D>
hipError_t launch(const MxProductArgs& a, int cus, hipStream_t s) {
  constexpr int kM = 16 * MT, kN = 16 * NT;
  const int64_t m_tiles = a.offsets ? a.rows / kM + (a.E < a.rows ? a.E : a.rows) : (a.rows + kM - 1) / kM;
  const int n_tiles = (a.N + kN - 1) / kN;
  const size_t bytes = KS * (ring_bytes<NT, MT, D>() + static_cast<size_t>(kN) * scale_pitch(a.K / 32, D));
  int64_t grid = m_tiles * n_tiles;
  // one wave: as many as fit at once (two per SIMD with their registers), each with a run of tiles
  const int64_t fit = static_cast<int64_t>(cus) * (160 * 1024 / bytes < 8 ? 160 * 1024 / bytes : 8);
  if (KS == 1 && grid > fit) grid = fit;
  grid = (grid + 7) & ~int64_t(7);  // every XCD has as many work-groups
  hipLaunchKernelGGL((stream_kernel<NT, MT, KS, D>), dim3(static_cast<uint32_t>(grid)), dim3(KS * kWave), bytes, s, a, n_tiles);
  return hipGetLastError();
}

template <int NT, int MT, int D>
hipError_t launch_split(const MxProductArgs& a, int ks, hipStream_t s) {
  int dev = 0, cus = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e == hipSuccess) e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  if (e != hipSuccess) return e;
  if (ks >= 4) return launch<NT, MT, 4, D>(a, cus, s);
  if (ks >= 2) return launch<NT, MT, 2, D>(a, cus, s);
  return launch<NT, MT, 1, D>(a, cus, s);
}

}  // namespace

hipError_t launch_mx_stream(const MxProductArgs& a, int nt, int mt, int ks, hipStream_t s) {
  if (nt == 4) {
    if (mt == 4) return launch_split<4, 4, 3>(a, ks, s);
    if (mt == 2) return launch_split<4, 2, 3>(a, ks, s);
    return launch_split<4, 1, 3>(a, ks, s);
  }
  if (nt == 2) {
    if (mt == 4) return launch_split<2, 4, 4>(a, ks, s);
    if (mt == 2) return launch_split<2, 2, 4>(a, ks, s);
    return launch_split<2, 1, 4>(a, ks, s);
  }
  if (mt == 4) return launch_split<1, 4, 4>(a, ks, s);
  if (mt == 2) return launch_split<1, 2, 4>(a, ks, s);
  return launch_split<1, 1, 4>(a, ks, s);
}

}  // namespace gxmoe
