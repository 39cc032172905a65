// mx_tile.hip -- MXFP4 products of many rows: tiles through LDS.
//
// A work-group computes 256 rows x 256 columns (fewer rows where an expert has no
// more), 128 x 128 or 32 x 128.  K goes in chunks of eight blocks: 128 bytes (a line) of each of
// the tile's rows and weight rows reach one of two LDS stages by direct global -> LDS loads, 16
// bytes a lane (such loads of 64 bytes of a row bring 14.6 TB/s over the chip, of whole
// lines 25.4); the 16-byte piece of block b of row r lies at b ^ (r / 2) % 8 of the row's 128
// bytes, so that the operand reads (one block of 16 rows at a time) meet all banks.  The scales
// come through registers into LDS, 32 blocks of a row at a time, since dwords of single
// rows would cost the address unit as much as the data.
//
// Per chunk a wave runs four steps of NT x MT products on operands that it read
// during the step before.  Before the last step, whose operands are in registers by then, it waits for
// its loads of the next chunk and meets the others, after which the chunk's
// stage is free for the loads of the chunk after the next.  These go out in three parts, in
// that step and the first two of the next chunk (8192^3: 274 us; all at once 279).
//
// Large tiles are bound by power: 8192 x 8192 x 8192 takes 270 us (4.1 PFLOP/s; the clock is
// 1.8 GHz), with operands of zeros 197; products alone, from registers, reach 6.2 to 6.7 PFLOP/s with random
// operands.  Each round of tiles takes 10 us beyond its chunks.  (Four waves of 128 x 128 each read a third less from
// LDS, but one wave a SIMD leaves gaps: 329 us.)  Smaller tiles stand two or three on a CU, so
// that one's first loads and last stores overlap another's chunks; their weights come at 4.2 TB/s
// with rows of 1440 bytes that straddle lines, at 5.3 where rows begin on them (128 experts of 16 rows
// each).  Four stages in place of two and fewer work-groups gave nothing (777 x 1001 x 2016: 13.4 us,
// with two 10.7).
#include <type_traits>

#include "mx_product.h"

namespace gxmoe {

namespace {

typedef __attribute__((address_space(3))) void lds_void_t;

constexpr int kBlocks = 8;  // of a chunk

// WN x WM waves, each NT x MT products of 32 columns x 32 rows, in a work-group of W waves:
// those that are left over load, and do another's products to no end.
template <int NT, int MT, int WN, int WM, int W = WN * WM>
struct Shape {
  static constexpr int kWaves = W, kThreads = kWaves * kWave;
  static constexpr int kTN = 32 * NT * WN, kTM = 32 * MT * WM;
  static constexpr int kRows = kTN + kTM;                         // the weights', then a's
  static constexpr int kPieces = kRows / 8;                       // of 1 KiB
  static constexpr int kLoads = (kPieces + kWaves - 1) / kWaves;  // per wave and chunk
  static constexpr int kStage = kRows * 16 * kBlocks;
  static constexpr int kScaleOff = 2 * kStage;                    // [2][4 chunks][kRows][8]
  static constexpr int kBytes = kScaleOff + 2 * 4 * kRows * 8;
  static_assert(kRows <= kThreads && kRows >= kThreads / 2 && kBytes <= 160 * 1024, "");
};

template <int N>
__device__ __forceinline__ void wait_vm() {  // vmcnt(N), the other counters as they are
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0f70);
}

typedef u32x4_t __attribute__((aligned(1))) loose_u32x4;

// 16 bytes of a row's scales from `from` on, zeros past the row's nb bytes: in two
// parts, so that the load is one that nothing waits for.  The load ends within the row
// (nb >= 16); what it holds too early is shifted out.
__device__ __forceinline__ u32x4_t shift_bytes(u32x4_t v, int n) {  // 0 < n < 16 bytes, uniform
  for (; n >= 4; n -= 4) v = u32x4_t{v[1], v[2], v[3], 0u};
  if (n > 0) {
    const int k = 8 * n;
    v = u32x4_t{v[0] >> k | v[1] << (32 - k), v[1] >> k | v[2] << (32 - k), v[2] >> k | v[3] << (32 - k), v[3] >> k};
  }
  return v;
}

__device__ __forceinline__ u32x4_t load_short_row(const uint8_t* row, int nb) {  // nb < 16
  u32x4_t v{0u, 0u, 0u, 0u};
  for (int i = 0; i < nb; ++i) {
    const uint32_t x = static_cast<uint32_t>(row[i]) << (8 * (i & 3));
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] |= (i >> 2) == j ? x : 0u;
  }
  return v;
}

// Up to 32 rows from LDS, `pitch` bytes apart, to rows `step` bytes apart: a T a lane, `across` lanes (a power of two) to a row, kBatch
// rows' reads ahead of their stores.  (A loop and not its copies: small calls would wait for their
// instructions.)  LDS is read through a type that may alias: the results were put there as others, two bf16 of SwiGLU
// as a dword, and nothing else holds the reads behind those stores.
template <typename T, int kBatch>
__device__ __forceinline__ void store_rows(const uint8_t* own, int pitch, int across, uint8_t* out, int64_t step, int rows, bool in,
                                           int lane) {
  typedef T __attribute__((may_alias)) any_t;
  const int log = __builtin_ctz(across), at_once = kWave >> log, row0 = lane >> log, off = sizeof(T) * (lane & (across - 1));
  const uint8_t* from = own + pitch * row0 + off;
  uint8_t* to = out + row0 * step + off;
  int left = in ? rows - row0 : 0;
  step *= at_once;
#pragma unroll 1
  for (int k = 0; k < 32; k += kBatch * at_once) {
    T d[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) d[u] = *reinterpret_cast<const any_t*>(from + pitch * at_once * u);
    from += kBatch * pitch * at_once;
    if (left > (kBatch - 1) * at_once) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) *reinterpret_cast<T*>(to + u * step) = d[u];
    } else {
#pragma unroll
      for (int u = 0; u < kBatch - 1; ++u)
        if (u * at_once < left) *reinterpret_cast<T*>(to + u * step) = d[u];
    }
    to += kBatch * step;
    left -= kBatch * at_once;
  }
}

template <int NT, int MT, int WN, int WM, int W = WN * WM>
__device__ __forceinline__ void tile(const MxProductArgs& a, const MTile& mt, int n0, uint8_t* lds) {
  typedef Shape<NT, MT, WN, WM, W> Sh;
  constexpr int kTileWaves = Sh::kWaves, kTileN = Sh::kTN, kRows = Sh::kRows;
  constexpr int kPieces = Sh::kPieces, L = Sh::kLoads, kStageBytes = Sh::kStage, kScaleOff = Sh::kScaleOff;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = w % WN, wm = w / WN % WM;
  const int r = lane & 31, half = lane >> 5;
  const int nb = a.K / 32, nch = (nb + kBlocks - 1) / kBlocks;
  const size_t row_bytes = static_cast<size_t>(a.K) / 2;
  const size_t wrow = static_cast<size_t>(mt.e) * a.N;

  // The lane's row of each piece that its wave loads.  A wave without a piece of its own
  // left loads its first one once more, so that all waves have as many loads in flight.
  const uint8_t* src[L];
  int piece[L], from[L + 1];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    piece[i] = w + kTileWaves * i < kPieces ? w + kTileWaves * i : w;
    from[i] = max(mt.lo, min(mt.lo + 8 * piece[i] + (lane >> 3) - kTileN, mt.hi - 1));
  }
  // The thread's row of the scales.  Threads that are left over do as the first ones: the same
  // bytes to the same place, where a branch would cost a wait for all loads.
  const int srow = tid < kRows ? tid : tid - kRows;
  from[L] = max(mt.lo, min(mt.lo + srow - kTileN, mt.hi - 1));
  source_rows(a, from);
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int row = 8 * piece[i] + (lane >> 3);
    src[i] = row < kTileN ? a.w + (wrow + min(n0 + row, a.N - 1)) * row_bytes
                          : a.a + static_cast<size_t>(max(from[i], 0)) * row_bytes;
  }
  const uint8_t* const ssrc = srow < kTileN ? a.ws + (wrow + min(n0 + srow, a.N - 1)) * nb
                                            : a.as + static_cast<size_t>(max(from[L], 0)) * nb;
  // (row / 2) % 8 of the lane's rows: all of its pieces are odd or all are even
  const int blk = (lane & 7) ^ (4 * (w & 1) + (lane >> 4));
  auto issue = [&](int c, auto from_piece, auto to_piece) __attribute__((always_inline)) {
    // blocks past the end: the last one again (its scale there is 0)
    const int b = min(kBlocks * c + blk, nb - 1);
    uint8_t* stage = lds + (c & 1) * kStageBytes;
#pragma unroll
    for (int i = decltype(from_piece)::value; i < decltype(to_piece)::value; ++i)
      __builtin_amdgcn_global_load_lds(src[i] + 16 * static_cast<size_t>(b), (lds_void_t*)(stage + 1024 * piece[i]), 16, 0, 0);
  };
  // A chunk's loads in three parts: the address unit takes one of a wave's in 16 cycles, and a
  // wave that waits for it gives no products meanwhile.
  const std::integral_constant<int, 0> part0{};
  const std::integral_constant<int, (3 * L + 7) / 8> part1{};
  const std::integral_constant<int, (6 * L + 7) / 8> part2{};
  const std::integral_constant<int, L> part3{};
  // Loads of 16 bytes with no branch around them: they end within the row, and where it has
  // fewer than 16 something is loaded that is not read.
  const uint8_t* sfrom = nb < 16 ? a.w : ssrc;
  const int slast = max(nb - 16, 0);
  u32x4_t sreg[2];
  auto load_scales = [&](int c) __attribute__((always_inline)) {  // of chunks c to c + 3
#pragma unroll
    for (int i = 0; i < 2; ++i) sreg[i] = *reinterpret_cast<const loose_u32x4*>(sfrom + min(kBlocks * c + 16 * i, slast));
  };
  auto put_scales = [&](int c) __attribute__((always_inline)) {
    gx_u32x2* to = reinterpret_cast<gx_u32x2*>(lds + kScaleOff) + ((c >> 2) & 1) * (4 * kRows) + srow;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int early = kBlocks * c + 16 * i + 16 - nb;
      if (early > 0) sreg[i] = early < 16 ? shift_bytes(sreg[i], early) : u32x4_t{0u, 0u, 0u, 0u};
      to[2 * kRows * i] = gx_u32x2{sreg[i][0], sreg[i][1]};
      to[2 * kRows * i + kRows] = gx_u32x2{sreg[i][2], sreg[i][3]};
    }
  };
  load_scales(0);
  issue(0, part0, part3);
  issue(1, part0, part1);
  if (nb < 16) {
    sreg[0] = load_short_row(ssrc, nb);
    sreg[1] = u32x4_t{0u, 0u, 0u, 0u};
    gx_u32x2* to = reinterpret_cast<gx_u32x2*>(lds + kScaleOff) + srow;
    to[0] = gx_u32x2{sreg[0][0], sreg[0][1]};
    to[kRows] = gx_u32x2{sreg[0][2], sreg[0][3]};
  } else {
    put_scales(0);
  }

  f32x16_t acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;

  const int wrow_l = 32 * NT * wn + r, arow_l = kTileN + 32 * MT * wm + r;
  const int piece0 = half ^ ((r >> 1) & 7);  // of step 0; of step s: ^ 2 s
  u32x4_t wv[2][NT], av[2][MT];
  gx_u32x2 sw[NT], sa[MT];
  auto read = [&](int c, int s, u32x4_t(&wo)[NT], u32x4_t(&ao)[MT]) __attribute__((always_inline)) {
    const uint8_t* stage = lds + (c & 1) * kStageBytes + 16 * (piece0 ^ (2 * s));
#pragma unroll
    for (int i = 0; i < NT; ++i) wo[i] = *reinterpret_cast<const u32x4_t*>(stage + 128 * wrow_l + 4096 * i);
#pragma unroll
    for (int j = 0; j < MT; ++j) ao[j] = *reinterpret_cast<const u32x4_t*>(stage + 128 * arow_l + 4096 * j);
  };
  auto read_scales = [&](int c) __attribute__((always_inline)) {
    const gx_u32x2* at = reinterpret_cast<const gx_u32x2*>(lds + kScaleOff) + kRows * (c & 7);
#pragma unroll
    for (int i = 0; i < NT; ++i) sw[i] = at[wrow_l + 32 * i];
#pragma unroll
    for (int j = 0; j < MT; ++j) sa[j] = at[arow_l + 32 * j];
  };

  wait_vm<decltype(part1)::value>();
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  read_scales(0);
  read(0, 0, wv[0], av[0]);

  // The products above stay above: without this the compiler gathers those of several
  // chunks behind the last one's barrier, and keeps all their operands.
  auto pin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) asm volatile("" : "+v"(acc[i][j]));
  };
  int c = 0;
  // Step s's products; the scale of block 2 s + half is byte 0 or 2 of what is left of the
  // row's dword s / 2 after a shift by the lane's half.
  uint32_t ow[NT], oa[MT];
  auto shift = [&](int d) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NT; ++i) ow[i] = sw[i][d] >> (8 * half);
#pragma unroll
    for (int j = 0; j < MT; ++j) oa[j] = sa[j][d] >> (8 * half);
  };
  auto products = [&](auto odd) __attribute__((always_inline)) {
    constexpr int kOdd = decltype(odd)::value;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(wv[kOdd][i]), mx_operand(av[kOdd][j]), acc[i][j],
                                                                    4, 4, 2 * kOdd, static_cast<int>(ow[i]), 2 * kOdd,
                                                                    static_cast<int>(oa[j]));
    pin();
  };
  // The next step's reads go out behind the first products of this one, then its loads.
  auto order = [&](auto from_piece, auto to_piece, auto more) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < (NT + MT + 1) / 2; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
#pragma unroll
    for (int i = 0; i < decltype(to_piece)::value - decltype(from_piece)::value + decltype(more)::value; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  const std::integral_constant<int, 0> p0{};
  const std::integral_constant<int, 1> p1{};
  const std::integral_constant<int, 2> p2{};
  const std::integral_constant<int, 3> p3{};
  auto chunk = [&](auto place) __attribute__((always_inline)) {
    constexpr int kPlace = decltype(place)::value;  // c % 4
    read(c, 1, wv[1], av[1]);
    issue(c + 1, part1, part2);
    shift(0);
    products(p0);
    order(part1, part2, p0);
    read(c, 2, wv[0], av[0]);
    issue(c + 1, part2, part3);
    products(p1);
    order(part2, part3, p0);
    read(c, 3, wv[1], av[1]);
    if constexpr (kPlace == 1) load_scales(c + 3);
    shift(1);
    products(p0);
    if constexpr (kPlace == 3) put_scales(c + 1);
    order(p0, p0, std::integral_constant<int, kPlace == 1 ? 2 : 0>{});
    wait_vm<kPlace == 1 ? 2 : 0>();      // this wave's loads of chunk c + 1
    __builtin_amdgcn_s_waitcnt(0xc07f);  // its reads of chunk c
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    read_scales(c + 1);
    read(c + 1, 0, wv[0], av[0]);
    issue(c + 2, part0, part1);
    products(p1);
    order(part0, part1, p0);
  };
  // (no way out between the chunks of four: it would cost a wait for all loads at the top)
  for (int left = nch >> 2; left > 0; --left) {
    chunk(p0), ++c;
    chunk(p1), ++c;
    chunk(p2), ++c;
    chunk(p3), ++c;
  }
  for (; c < nch; ++c) chunk(p2);  // up to three, whose scales are there
  // the ring becomes the waves' own room: no load may still land in it
  wait_vm<0>();
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_s_barrier();

  float* bias_all = reinterpret_cast<float*>(lds + kScaleOff);
  if (tid < kTileN) bias_all[tid] = a.bias ? bf16_to_f32(a.bias[wrow + min(n0 + tid, a.N - 1)]) : 0.0f;
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_s_barrier();
  if (w >= WN * WM) return;
  const float* bias = bias_all + 32 * NT * wn;
  uint8_t* own = lds + 2 * kStageBytes / kTileWaves * w;
  const int cols = a.swiglu ? a.N / 2 : a.N;
  constexpr int kG = NT < 2 ? NT : 2;  // column tiles that go together
  int reads[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) reads[j] = min(mt.lo + 32 * (MT * wm + j) + r, mt.hi - 1);
  source_rows(a, reads);
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int p = mt.lo + 32 * (MT * wm + j) + r;
    const bool live = p < mt.hi;
    const bool zero = reads[j] < 0;
#pragma unroll
    for (int g = 0; g < NT / kG; ++g) {
      const int n = n0 + 32 * (NT * wn + kG * g);  // the group's first column
      float v[kG][16];
#pragma unroll
      for (int i = 0; i < kG; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 b = *reinterpret_cast<const float4*>(bias + 32 * (kG * g + i) + 8 * q + 4 * half);
          const f32x16_t& x = acc[kG * g + i][j];
          v[i][4 * q + 0] = (zero ? 0.0f : x[4 * q + 0]) + b.x;
          v[i][4 * q + 1] = (zero ? 0.0f : x[4 * q + 1]) + b.y;
          v[i][4 * q + 2] = (zero ? 0.0f : x[4 * q + 2]) + b.z;
          v[i][4 * q + 3] = (zero ? 0.0f : x[4 * q + 3]) + b.w;
        }
      if (a.swiglu) {
#pragma unroll
        for (int i = 0; i < kG; ++i)
#pragma unroll
          for (int q = 0; q < 8; ++q) v[i][q] = mx_swiglu(v[i][2 * q], v[i][2 * q + 1], a.alpha, a.limit);
      }
      if (a.quantized()) {
        const size_t ob = static_cast<size_t>(p) * (cols / 32);
        uint32_t code;
        if (a.swiglu) {
          if constexpr (kG == 2) {
            const float x[16] = {v[0][0], v[0][1], v[0][2], v[0][3], v[0][4], v[0][5], v[0][6], v[0][7],
                                 v[1][0], v[1][1], v[1][2], v[1][3], v[1][4], v[1][5], v[1][6], v[1][7]};
            const gx_u32x2 d = quantize_block<true>(x, code);
            if (live && n / 2 < cols) {
              const size_t at = ob + n / 64;
              static_cast<gx_u32x2*>(a.out)[2 * at + half] = d;
              if (half == 0) a.out_scales[at] = static_cast<uint8_t>(code);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < kG; ++i) {
            const gx_u32x2 d = quantize_block<false>(v[i], code);
            if (live && n + 32 * i < cols) {
              const size_t at = ob + n / 32 + i;
              static_cast<gx_u32x2*>(a.out)[2 * at + half] = d;
              if (half == 0) a.out_scales[at] = static_cast<uint8_t>(code);
            }
          }
        }
        continue;
      }
      // through LDS, so that rows are written in whole pieces: 32 rows of `wide` bytes
      const int size = a.out_fp32 ? 4 : 2, have = 32 * kG >> (a.swiglu ? 1 : 0);
      const int wide = have * size, pitch = wide + 16;
#pragma unroll
      for (int i = 0; i < kG; ++i) {
        if (a.swiglu) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint8_t* at = own + pitch * r + size * (16 * i + 4 * q + 2 * half);
            if (a.out_fp32) *reinterpret_cast<float2*>(at) = float2{v[i][2 * q], v[i][2 * q + 1]};
            else *reinterpret_cast<uint32_t*>(at) = pack_bf16x2(v[i][2 * q], v[i][2 * q + 1]);
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint8_t* at = own + pitch * r + size * (32 * i + 8 * q + 4 * half);
            if (a.out_fp32)
              *reinterpret_cast<float4*>(at) = float4{v[i][4 * q], v[i][4 * q + 1], v[i][4 * q + 2], v[i][4 * q + 3]};
            else
              *reinterpret_cast<gx_u32x2*>(at) =
                  gx_u32x2{pack_bf16x2(v[i][4 * q], v[i][4 * q + 1]), pack_bf16x2(v[i][4 * q + 2], v[i][4 * q + 3])};
          }
        }
      }
      const int first = a.swiglu ? n / 2 : n;
      const int row = mt.lo + 32 * (MT * wm + j), rows = min(mt.hi - row, 32);
      uint8_t* to = static_cast<uint8_t*>(a.out) + (row * a.stride + first) * size;
      const int64_t step = a.stride * size;
      // 16 bytes a lane where rows lie on them and the group is whole; otherwise a column a lane, next to each other
      // (8008 x 4591 x 96 to bf16 40 us; with several columns of a lane's own 81)
      if (a.vec && first + have <= cols) store_rows<u32x4_t, 2>(own, pitch, wide / 16, to, step, rows, true, lane);
      else if (a.out_fp32) store_rows<uint32_t, 8>(own, pitch, have, to, step, rows, first + (lane & (have - 1)) < cols, lane);
      else store_rows<uint16_t, 8>(own, pitch, have, to, step, rows, first + (lane & (have - 1)) < cols, lane);
    }
  }
}

// Tiles are numbered four m-tiles x all n-tiles at a time, and every XCD (one of eight, in
// turn by work-group) takes a run of them, so that its L2 serves a tile's rows
// and weights to its neighbours.  The grid has room for every expert's last tile; how many there
// are is known here.
constexpr int kGroupM = 4;

struct Place {
  MTile m;
  int nt;
};

__device__ __forceinline__ bool find_place(const MxProductArgs& a, int rows, int n_tiles, Place* p) {
  const int lane = threadIdx.x & (kWave - 1);
  const int m_tiles = count_m_tiles(a, rows, lane);
  const int total = m_tiles * n_tiles, b = blockIdx.x;
  const int x = b & 7, share = total >> 3, more = total & 7;
  if ((b >> 3) >= share + (x < more ? 1 : 0)) return false;
  const int id = x * share + min(x, more) + (b >> 3);
  const int group = id / (kGroupM * n_tiles), in_group = id - group * (kGroupM * n_tiles);
  const int height = min(kGroupM, m_tiles - kGroupM * group);
  p->m = find_m_tile(a, kGroupM * group + in_group % height, rows, lane);
  p->nt = in_group / height;
  return true;
}

// 256 columns x 256 rows, fewer where an expert has no more.
__global__ __launch_bounds__(512, 2) void large_tile_kernel(MxProductArgs a, int n_tiles) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Shape<4, 2, 2, 4>::kBytes];
  Place p;
  if (!find_place(a, 256, n_tiles, &p)) return;
  const int rows = p.m.hi - p.m.lo;
  if (rows > 128) tile<4, 2, 2, 4>(a, p.m, p.nt * 256, lds);
  else if (rows > 64) tile<2, 2, 4, 2>(a, p.m, p.nt * 256, lds);
  else tile<2, 1, 4, 2>(a, p.m, p.nt * 256, lds);
}

// 128 columns x 128 or 64 rows, two work-groups on a CU.
__global__ __launch_bounds__(256, 2) void middle_tile_kernel(MxProductArgs a, int n_tiles) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Shape<2, 2, 2, 2>::kBytes];
  Place p;
  if (!find_place(a, 128, n_tiles, &p)) return;
  const int rows = p.m.hi - p.m.lo;
  if (rows > 64) tile<2, 2, 2, 2>(a, p.m, p.nt * 128, lds);
  else tile<2, 1, 2, 2>(a, p.m, p.nt * 128, lds);
}

// 128 columns x 32 rows, three work-groups on a CU.
__global__ __launch_bounds__(256, 3) void low_tile_kernel(MxProductArgs a, int n_tiles) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Shape<2, 1, 2, 1, 4>::kBytes];
  Place p;
  if (find_place(a, 32, n_tiles, &p)) tile<2, 1, 2, 1, 4>(a, p.m, p.nt * 128, lds);
}

}  // namespace

hipError_t launch_mx_tile(const MxProductArgs& a, MxTile kind, hipStream_t s) {
  const int rows = kind == MxTile::large ? 256 : kind == MxTile::middle ? 128 : 32;
  const int cols = kind == MxTile::large ? 256 : 128, n_tiles = (a.N + cols - 1) / cols;
  // a multiple of eight, so that every XCD has work-groups enough for its share
  const int64_t tiles = (most_m_tiles(a, rows) * n_tiles + 7) & ~int64_t(7);
  if (tiles * 512 > UINT32_MAX) return hipErrorInvalidConfiguration;  // a launch's threads
  const dim3 grid(static_cast<uint32_t>(tiles));
  if (kind == MxTile::large) hipLaunchKernelGGL(large_tile_kernel, grid, dim3(512), 0, s, a, n_tiles);
  else if (kind == MxTile::middle) hipLaunchKernelGGL(middle_tile_kernel, grid, dim3(256), 0, s, a, n_tiles);
  else hipLaunchKernelGGL(low_tile_kernel, grid, dim3(256), 0, s, a, n_tiles);
  return hipGetLastError();
}

}  // namespace gxmoe
