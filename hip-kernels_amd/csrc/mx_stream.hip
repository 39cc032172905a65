// mx_stream.hip -- MXFP4 products of few rows: the weights stream through LDS, wave by
// wave.
//
// A wave computes up to 16 rows x 16 NT columns over its share of K with
// v_mfma_scale_f32_16x16x128_f8f6f4 (lane l gives row l % 16 of each operand and block l / 16 of
// four; it ends with columns 4 (l / 16) + {0 .. 3} of row l % 16).  Its weight rows come line by
// line (128 bytes, eight blocks) into a ring of four lines each, by direct global -> LDS loads, and out
// of it in the operands' order; no wave waits for another.  The lines are the memory's: where rows
// do not begin on one (K = 2880: 1440 bytes), a row's blocks lie a few places further on, and a chunk of
// eight blocks needs two lines.  (Streaming alone, 5 to 8 waves on a CU: 128 bytes of each of 8 rows
// per load 6.9 TB/s where they are lines, 5.4 where they straddle two.  Loads straight to the
// operands' registers take 64 bytes of a row at a time: the whole kernel 3.1 TB/s.  Lines that no
// cache keeps, 6 to 8 % faster: 32 experts of a row each that were not read before, 54 us, without 59.)  The rows of a, few
// and read by all, go to registers four chunks ahead.
//
// A wave goes through a run of neighbouring tiles of the same rows, and the loads of the next
// tile's lines follow those of the last without a pause.  A tile's K goes in spans of 128
// blocks, whose weights' scales are loaded during the span before and put into LDS between
// the two.  Where tiles are few, KS waves share a tile's K, and their sums meet in LDS in
// a fixed order.
//
// Bound by the weights' bandwidth: one to six rows each of 107 experts, 5760 x 2880, 163 us (5.8 TB/s); one or two of 29
// experts 53 us (4.8); by latency where they are few: 1 x 5120 x 2880, weights in no cache, 7.5 us.
#include "mx_product.h"

namespace gxmoe {

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef u32x4_t __attribute__((aligned(1))) loose_u32x4;
typedef __attribute__((address_space(3))) void lds_void_t;

template <int N>
__device__ __forceinline__ void wait_vm() {  // vmcnt(N), the other counters as they are
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0f70);
}

constexpr int kRing = 4;    // lines (eight: 1 x 5120 x 2880 8.4 us for 7.3, whose 12 lines take two whole turns)
constexpr int kSpan = 128;  // blocks whose scales are in LDS at a time: whole turns of the ring

// Bytes between the scales of two rows: an odd number of 16, so that 16 rows meet all banks.
__host__ __device__ constexpr int scale_pitch(int nb) {
  const int p = ((nb < kSpan ? nb : kSpan) + 15) / 16;
  return 16 * (p | 1);
}

// LDS of a wave: its ring, its scales and, of several, its sums.
template <int NT, int KS>
__host__ __device__ constexpr int wave_bytes(int nb) {
  return kRing * NT * 2048 + 16 * NT * scale_pitch(nb) + (KS > 1 ? NT * 1024 : 0);
}

// Neighbouring results of a row from column n on: rounded to bf16 unless fp32, as one store
// where `vec` (the rows are on 16 bytes), and not past the last column.
template <int W>
__device__ __forceinline__ void store_few(const MxProductArgs& a, const float (&v)[W], size_t row, int n, int cols) {
  static_assert(W == 2 || W == 4, "");
  float* const f = static_cast<float*>(a.out) + row + n;
  uint16_t* const h = static_cast<uint16_t*>(a.out) + row + n;
  if (a.vec && n + W <= cols) {
    if constexpr (W == 2) {
      if (a.out_fp32) *reinterpret_cast<float2*>(f) = float2{v[0], v[1]};
      else *reinterpret_cast<uint32_t*>(h) = pack_bf16x2(v[0], v[1]);
    } else {
      if (a.out_fp32) *reinterpret_cast<float4*>(f) = float4{v[0], v[1], v[2], v[3]};
      else *reinterpret_cast<gx_u32x2*>(h) = gx_u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < W; ++q)
    if (n + q < cols) {
      if (a.out_fp32) f[q] = v[q];
      else h[q] = f32_to_bf16(v[q]);
    }
}

// The scale byte of a block that lanes l, l + 16, l + 32 and l + 48 hold, eight values each.
__device__ __forceinline__ uint32_t block_scale(const float (&x)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, mx_magnitude(x[i]));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, kWave)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, kWave)));
  return mx_scale_byte(top);
}

// The results of row p, columns n0 + 16 i + 4 (lane / 16) + {0 .. 3} of each lane: bias, SwiGLU and the store.
// A block of 32 after SwiGLU is two tiles of 32 columns: the first one's results wait in `held`.
template <int NT>
__device__ __forceinline__ void write_rows(const MxProductArgs& a, const f32x4_t (&sum)[NT], int e, int n0, int p, bool live,
                                           bool zero, int lane, f32x4_t& held) {
  const int r = lane & 15, g = lane >> 4;
  const int cols = a.swiglu ? a.N / 2 : a.N;
  float v[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) v[i][q] = zero ? 0.0f : sum[i][q];
  if (a.bias) {
    const uint16_t* bias = a.bias + static_cast<size_t>(e) * a.N;
    uint32_t x[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) x[i][q] = bias[min(n0 + 16 * i + 4 * g + q, a.N - 1)];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[i][q] += __uint_as_float(x[i][q] << 16);
  }
  if (a.swiglu) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q) v[i][q] = mx_swiglu(v[i][2 * q], v[i][2 * q + 1], a.alpha, a.limit);
  }
  if (a.quantized()) {
    if constexpr (NT == 2) {
      const size_t row = static_cast<size_t>(p) * (cols / 32);
      if (a.swiglu) {
        if ((n0 & 32) == 0) {
          held = f32x4_t{v[0][0], v[0][1], v[1][0], v[1][1]};
          return;
        }
        // of the 16-column tiles i, columns 8 i + 2 g + {0, 1}: byte 4 i + g of the block
        const float x[8] = {held[0], held[1], held[2], held[3], v[0][0], v[0][1], v[1][0], v[1][1]};
        const uint32_t code = block_scale(x), mine = mx_pack8(x, code);  // byte i
        uint32_t d = 0;                                                  // dword g of the block
#pragma unroll
        for (int q = 0; q < 4; ++q)
          d |= ((static_cast<uint32_t>(__shfl(static_cast<int>(mine), r + 16 * q, kWave)) >> (8 * g)) & 0xffu) << (8 * q);
        const int block = (n0 - 32) / 64;
        if (live && 32 * block < cols) {
          static_cast<uint32_t*>(a.out)[4 * (row + block) + g] = d;
          if (g == 0) a.out_scales[row + block] = static_cast<uint8_t>(code);
        }
      } else {  // columns 4 g + {0 .. 3} and 16 further on
        const float x[8] = {v[0][0], v[0][1], v[0][2], v[0][3], v[1][0], v[1][1], v[1][2], v[1][3]};
        const uint32_t code = block_scale(x), d = mx_pack8(x, code);
        if (live && n0 < cols) {
          uint16_t* o = static_cast<uint16_t*>(a.out) + 8 * (row + n0 / 32);
          o[g] = static_cast<uint16_t>(d);
          o[4 + g] = static_cast<uint16_t>(d >> 16);
          if (g == 0) a.out_scales[row + n0 / 32] = static_cast<uint8_t>(code);
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
      const float x[2] = {v[i][0], v[i][1]};
      store_few(a, x, row, (n0 + 16 * i) / 2 + 2 * g, cols);
    } else {
      store_few(a, v[i], row, n0 + 16 * i + 4 * g, cols);
    }
  }
}

template <int NT, int KS>
__device__ __forceinline__ void stream_tiles(const MxProductArgs& a, int grid, uint8_t* lds) {
  constexpr int kN = 16 * NT, kLine = NT * 2048;
  constexpr int kLoads = 2 * NT + 4;  // of a line of the rows, and a chunk of a's
  constexpr int kLanes = kWave / kN;       // per weight row, for its scales
  constexpr int kPieces = (kSpan / 16 + kLanes - 1) / kLanes;
  static_assert((kRing - 2) * kLoads < 64, "vmcnt range");
  const int lane = threadIdx.x & (kWave - 1), k = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // This work-group's run of tiles, the columns of an m-tile in turn: as long as all others' but the last, so that none
  // is left with a longer one (fewer waves hold the bandwidth too).  XCD b % 8 has neighbouring runs.  Tiles whose results
  // make one block go together.
  const int together = a.swiglu && a.quantized() ? 2 : 1;
  const int n_tiles = (a.N + kN * together - 1) / (kN * together) * together;
  const int m_tiles = count_m_tiles(a, kStreamRows, lane);
  const int64_t total = static_cast<int64_t>(m_tiles) * (n_tiles / together);
  const int64_t run = (total + grid - 1) / grid, runs = run ? (total + run - 1) / run : 0;
  const int xcd = blockIdx.x & 7, share = static_cast<int>(runs >> 3), more = static_cast<int>(runs & 7);
  if (static_cast<int>(blockIdx.x >> 3) >= share + (xcd < more ? 1 : 0)) return;
  const int64_t b = xcd * share + min(xcd, more) + static_cast<int>(blockIdx.x >> 3);
  int id = static_cast<int>(run * b) * together, id_end = static_cast<int>(min(run * (b + 1), total)) * together;
  if (run == 1) {
    // Without runs the m-tiles of the same columns are neighbours, whose weights come once to their L2.
    const int i = static_cast<int>(b);
    id = i % m_tiles * n_tiles + i / m_tiles * together;
    id_end = id + together;
  }

  const int r = lane & 15, g = lane >> 4;
  const int nb = a.K / 32, chunks = (nb + 7) / 8;
  const int per = (chunks + KS - 1) / KS;
  const int first = k * per, last = min(first + per, chunks);  // this wave's chunks, maybe none
  const int begin = 8 * first, end = min(8 * last, nb);        // its blocks
  const size_t row_bytes = 16 * static_cast<size_t>(nb);
  const int pitch = scale_pitch(nb);
  uint8_t* const ring = lds + k * wave_bytes<NT, KS>(nb);
  uint8_t* const scales = ring + kRing * kLine;

  while (id < id_end) {
    const int m = id / n_tiles;
    int n0 = (id - m * n_tiles) * kN;
    int left = min(id_end, (m + 1) * n_tiles) - id;  // tiles of these rows
    id += left;
    const MTile mt = find_m_tile(a, m, kStreamRows, lane);
    const int p = min(mt.lo + r, mt.hi - 1);  // past the last row: that one
    const int src = source_row(a, p);         // < 0: its result is replaced
    const uint8_t* const ap = a.a + static_cast<size_t>(max(src, 0)) * row_bytes;
    const uint8_t* const asp = a.as + static_cast<size_t>(max(src, 0)) * nb;
    const uint8_t* const w = a.w + static_cast<size_t>(mt.e) * a.N * row_bytes;
    const uint8_t* const ws = a.ws + static_cast<size_t>(mt.e) * a.N * nb;
    // Where a row begins in its first line, in blocks, and how many lines the wave's blocks can take; the ring goes
    // round whole.
    const uint32_t w16 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(w) >> 4);
    auto offset = [&](uint32_t row) __attribute__((always_inline)) { return static_cast<int>((w16 + row * nb) & 7u); };
    const int unit = nb & 1 ? 1 : nb & 2 ? 2 : nb & 4 ? 4 : 8;
    const int furthest = 8 - unit + static_cast<int>(w16 % unit);
    const int turns = ((end - 1 - begin + furthest) / 8 + kRing) / kRing;

    u32x4_t av[kRing][2];
    uint32_t sa[kRing][2];
    // Loads of line `line` of the columns from n on, and of a's chunk of that number.  Blocks past the end are the last one
    // again: there are no branches around loads, which would cost waits for all of them.
    auto issue = [&](int slot, int n, int line) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t at = min(begin + 8 * line + 4 * q + g, end - 1);
        av[slot][q] = *reinterpret_cast<const u32x4_t*>(ap + 16 * static_cast<size_t>(at));
        sa[slot][q] = asp[at];
      }
      // Row 8 i + lane / 8: place lane % 8 of its 128 bytes in LDS holds block (lane % 8) ^ (row / 2) % 8 of the line, so
      // that 16 rows meet all banks.
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i) {
        const uint32_t row = min(n + 8 * i + (lane >> 3), a.N - 1);
        const int place = (lane & 7) ^ (4 * (i & 1) + (lane >> 4));
        const uint32_t block = max(begin, min(begin + 8 * line + place - offset(row), end - 1));
        __builtin_amdgcn_global_load_lds(w + (static_cast<uint64_t>(row) * static_cast<uint32_t>(nb) + block) * 16,
                                         (lds_void_t*)(ring + slot * kLine + 1024 * i), 16, 0, 2);
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

    f32x4_t acc[NT], held = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    int from[NT];  // where the lane's rows begin
    auto open = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        from[i] = offset(min(n0 + 16 * i + r, a.N - 1));
        acc[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      }
    };
    open();
    int turn = 0;
    if (begin < end) {
      load_scales(n0, begin);
#pragma unroll
      for (int i = 0; i < kRing; ++i) issue(i, n0, i);
      __builtin_amdgcn_sched_barrier(0);
      put_scales();
    }
    for (;;) {
      bool ends = true;
      if (begin < end) {
        constexpr int kTurns = kSpan / 8 / kRing;  // of the ring, in a span
        ends = turn + kTurns >= turns;             // the tile's last span
        // The next span, of this tile or of the next one.  (Behind the last tile of the rows: the last one once more, for
        // nothing.)
        const int next_n = left > 1 ? n0 + kN : n0;
        const int span = begin + 8 * kRing * turn;
        load_scales(ends ? next_n : n0, ends ? begin : span + kSpan);
        __builtin_amdgcn_sched_barrier(0);
        const int upto = min(span + kSpan, end), stop = min(turn + kTurns, turns);
        do {
          const bool next = turn + 1 == turns;  // what is loaded belongs to the next tile
          const int n_load = next ? next_n : n0, line = next ? 0 : kRing * (turn + 1);
#pragma unroll
          for (int slot = 0; slot < kRing; ++slot) {
            wait_vm<(kRing - 2) * kLoads>();  // this line and the next one
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int rel = 8 * kRing * turn + 8 * slot + 4 * q + g;  // the lane's block of the wave's
              const bool in = begin + rel < upto;                      // past the end they are zeros of a
              const int at = min(begin + rel, upto - 1), piece = (at - span) >> 4;
              const int place = max(0, 16 * piece + at - min(span + 16 * piece, nb - 16));
              u32x4_t wv[NT], x;
              uint32_t sw[NT];
#pragma unroll
              for (int i = 0; i < NT; ++i) {
                const int pos = rel + from[i];
                wv[i] = *reinterpret_cast<const u32x4_t*>(ring + ((pos >> 3) & (kRing - 1)) * kLine + (16 * i + r) * 128 +
                                                          16 * ((pos & 7) ^ ((r >> 1) & 7)));
                sw[i] = scales[(16 * i + r) * pitch + place];
              }
#pragma unroll
              for (int d = 0; d < 4; ++d) x[d] = in ? av[slot][q][d] : 0u;
#pragma unroll
              for (int i = 0; i < NT; ++i)
                acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(wv[i]), mx_operand(x), acc[i], 4, 4, 0,
                                                                          static_cast<int>(sw[i]), 0,
                                                                          static_cast<int>(sa[slot][q]));
            }
            __builtin_amdgcn_s_waitcnt(0xc07f);  // the line has been read
            __builtin_amdgcn_sched_barrier(0);
            issue(slot, n_load, line + slot);
            __builtin_amdgcn_sched_barrier(0);
          }
        } while (++turn < stop);
        put_scales();
      }
      if (!ends) continue;
      const bool live = mt.lo + r < mt.hi;
      if constexpr (KS > 1) {
        // The first wave sums those of all, in turn.
        const int stride = wave_bytes<NT, KS>(nb) / 16;  // between two waves' sums
        f32x4_t* const sums = reinterpret_cast<f32x4_t*>(lds + kRing * kLine + kN * pitch);
#pragma unroll
        for (int i = 0; i < NT; ++i) sums[k * stride + i * kWave + lane] = acc[i];
        lds_barrier();
        if (k == 0) {
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int q = 1; q < KS; ++q) acc[i] += sums[q * stride + i * kWave + lane];
          write_rows<NT>(a, acc, mt.e, n0, mt.lo + r, live, src < 0, lane, held);
        }
        lds_barrier();  // before the next tile's sums
      } else {
        write_rows<NT>(a, acc, mt.e, n0, mt.lo + r, live, src < 0, lane, held);
      }
      n0 += kN;
      if (--left == 0) break;
      open();
      turn = 0;
    }
    wait_vm<0>();  // no load may still land in the ring
  }
}

template <int NT, int KS>
__global__ __launch_bounds__(KS * kWave) void stream_kernel(MxProductArgs a, int grid) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  stream_tiles<NT, KS>(a, grid, lds);
}

template <int NT, int KS>
hipError_t launch(const MxProductArgs& a, hipStream_t s) {
  constexpr int kN = 16 * NT;
  const int pieces = a.swiglu && a.quantized() ? 2 * kN : kN;  // columns that go together
  const size_t bytes = static_cast<size_t>(KS) * wave_bytes<NT, KS>(a.K / 32);
  // As many as fit at once, each with a run of tiles: eight waves on a CU, the two a SIMD that 32 columns' 203 and more
  // registers leave.  (16 columns' 143 and 146 would leave three; that was not measured.)
  const int64_t by_lds = 160 * 1024 / bytes, by_waves = 8 / KS, fit = kMxCus * (by_lds < by_waves ? by_lds : by_waves);
  int64_t grid = most_m_tiles(a, kStreamRows) * ((a.N + pieces - 1) / pieces);
  if (grid > fit) grid = fit;
  grid = (grid + 7) & ~int64_t(7);  // every XCD has as many work-groups
  hipLaunchKernelGGL((stream_kernel<NT, KS>), dim3(static_cast<uint32_t>(grid)), dim3(KS * kWave), bytes, s, a,
                     static_cast<int>(grid));
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_stream(const MxProductArgs& a, bool wide, bool split, hipStream_t s) {
  if (wide) return split ? launch<2, 4>(a, s) : launch<2, 1>(a, s);
  return split ? launch<1, 4>(a, s) : launch<1, 1>(a, s);
}

}  // namespace gxmoe
