// attn_prefill.hip -- causal attention of prompt chunks over the paged cache
// (gfx950).
//
// Mathematics: the triples (reference m, sum l, weighted values O) of
// attn_decode.hip, for 128 or 256 rows at a time.  A row is one query head of one
// new token; the heads that share a kv head lie side by side, so that a
// work-group's rows are few tokens and what a window or the diagonal cuts off is
// cut off for all of them.
//
// A work-group is four waves of 32 or 64 rows (with few rows eight, see G) over
// tiles of 64 tokens.  The products are S^T = K Q^T and O^T = V^T P^T in
// 32 x 32 x 16 steps: S^T leaves a lane with its own row and the tokens that the
// second product wants from it, so the weights stay in registers.  K and V go
// through LDS, 16-byte pieces permuted by the token so that neither the row reads
// of K nor the transposing reads of V meet in a bank; the next tile is on its way
// to registers while one is worked on.
//
// The weights 2^(s - m) of a tile's half are formed, rounded to bf16 for the
// matrix cores (l sums them as rounded, so that what they share of the rounding
// leaves the result), while the products of the half before and the half after
// run.  m moves only when a lane's weights of a half sum to kMost or more: until
// then bf16 and fp32 lose nothing, and no maximum is looked for.
//
// Bound by the matrix cores with the vector and LDS work beside them, all 40 to 50 %
// busy, and for large calls by power (2.09 GHz then): a prompt of 8192 with 64
// heads of 64 takes 569 us, 966 TFLOP/s, where a matrix product of 8192^3 reaches
// 1250; 512 tokens over 16000 in e4m3 with 32 heads of 128 148 us, 923 TFLOP/s.  A
// short window is bound by the queries and results instead: a prompt of 8192 with a
// window of 128 64 us, of which these take 29.
// (Pairs of times beside the choices below are of one run each, and may be older.)
#include <type_traits>

#include "attn_device.h"

namespace gxmoe {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t* LdsBytes;

constexpr int kTile = 64;     // tokens of a step
constexpr int kMinTiles = 4;  // tiles of the smallest piece
constexpr float kMost = 4096.0f;  // a lane's sum of weights from which on the reference moves

// With few rows and a long context the tokens are cut too: piece p of a tile of
// rows takes its p-th part.
struct PieceArgs {
  int pieces;      // largest number
  float* part_o;   // as JoinArgs
  float* part_ml;
  int* plan;       // [rows] pieces
};

struct Chunk {
  int b, row0;     // sequence, its first row of q
  int tokens;      // new tokens of the tile
  int tok0;        // the first one, within the sequence's new ones
  int pos0;        // its position
  int len;
};

// Tile `at` of all tiles of `per` tokens, the last one first: the longest rows
// of a prompt begin earliest.  (64 sequences at a time, a lane each; what is read of
// the first 64 is read once, lengths and offsets together.)
__device__ __forceinline__ bool find_chunk(const AttendArgs& a, int at, int per, Chunk* c) {
  const int lane = threadIdx.x & 63;
  struct Span {
    int begin, n, len;  // new tokens of a sequence, within the rows that there are
  };
  auto span = [&](int b) {
    Span s{0, 0, 0};
    if (b < a.B) {
      const int lo = a.offsets[b], hi = a.offsets[b + 1];
      s.len = seq_len(a, b);
      s.begin = min(max(lo, 0), a.rows);
      s.n = max(0, min(hi, a.rows) - s.begin);
    }
    return s;
  };
  const Span mine = span(lane);
  int total = wave_scan((mine.n + per - 1) / per);
  for (int b0 = 64; b0 < a.B; b0 += 64) total += wave_scan((span(b0 + lane).n + per - 1) / per);
  at = __builtin_amdgcn_readlane(total, 63) - 1 - at;
  if (at < 0) return false;
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const Span s = b0 == 0 ? mine : span(b0 + lane);
    const int upto = before + wave_scan((s.n + per - 1) / per);
    const uint64_t reached = __ballot(at < upto);
    if (reached != 0) {
      const int who = __builtin_ctzll(reached);
      const int n = __builtin_amdgcn_readlane(s.n, who);
      const int first = __builtin_amdgcn_readlane(upto, who) - (n + per - 1) / per;
      c->b = b0 + who;
      c->row0 = __builtin_amdgcn_readlane(s.begin, who);
      c->tok0 = (at - first) * per;
      c->tokens = min(per, n - c->tok0);
      c->len = __builtin_amdgcn_readlane(s.len, who);
      c->pos0 = c->len - n + c->tok0;
      return true;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// The bits of the infinities and NaN among two bf16 or four e4m3.
template <bool kE4m3>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
  if constexpr (kE4m3) return (((x & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u) * 0xffu;
  return (((x & 0x7f807f80u) + 0x00800080u) >> 15 & 0x00010001u) * 0xffffu;
}

typedef attn_u32x4 __attribute__((may_alias)) Piece;
typedef attn_u32x2 __attribute__((may_alias)) HalfPiece;

// Orders a wave's LDS traffic: what its lanes wrote before is what they read
// behind it.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Where in its row of LDS a 16-byte piece of token t lies: the 16 tokens that
// take part in a read of K, and the four of a read of V, meet in no bank.
template <int D>
__device__ __forceinline__ int piece_at(int t, int piece) {
  if constexpr (D == 64) return piece ^ ((t >> 1 & 1) << 2 | (t >> 2 & 3));
  return piece ^ ((t & 3) << 2 | (t >> 2 & 3));
}

// kCols * 32 rows a wave.  G groups of four waves have the same rows and each its
// part of the tokens; the second one's sums join the first's through LDS.
template <int D, bool kE4m3, int kCols, int G>
__global__ __launch_bounds__(256 * G, D == 64 && kCols == 1 && G == 1 ? 3 : 2) void prefill_kernel(AttendArgs a, PieceArgs pa) {
  constexpr int kSize = kE4m3 ? 1 : 2;
  constexpr int kPieces = D * kSize / 16;      // 16-byte pieces of a token's row in memory
  constexpr int kLoads = 16 * kPieces / 64;    // loads of a wave for its 16 tokens of K, and of V
  constexpr int kRowBytes = 2 * D;             // of a token in LDS
  constexpr int kBytes = kTile * kRowBytes;
  constexpr int kSteps = D / 16, kDb = D / 32;
  constexpr int kOutRow = 144;                 // of a row's 128 bytes on their way out, in LDS
  // of each group K of two tiles, then V of two; the queries pass through the middle
  // half of it before, the results through its beginning afterwards
  __shared__ __attribute__((aligned(16))) uint8_t s_all[4 * G][kBytes];
  __shared__ uint32_t s_odd[2];  // the tiles (of 64 in turn) of which put() left out a value

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  const int part_of = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);  // its group
  uint8_t(*const s_kv)[kBytes] = s_all + 4 * part_of;
  uint8_t(*const s_k)[kBytes] = s_kv;
  uint8_t(*const s_v)[kBytes] = s_kv + 2;
  const int n = lane & 31, h = lane >> 5;
  const int group = a.heads / a.kv.kv_heads, per = 128 * kCols / group;
  const int kvh = __builtin_amdgcn_readfirstlane(blockIdx.x % a.kv.kv_heads);
  const int piece = __builtin_amdgcn_readfirstlane(blockIdx.x / a.kv.kv_heads % pa.pieces);
  Chunk c;
  if (!find_chunk(a, blockIdx.x / a.kv.kv_heads / pa.pieces, per, &c)) return;
  for (int* x : {&c.b, &c.row0, &c.tokens, &c.tok0, &c.pos0, &c.len}) *x = __builtin_amdgcn_readfirstlane(*x);

  // This lane's rows: 32 y + n of the wave's 32 kCols.  Rows move between memory
  // and LDS in 128-byte pieces, eight lanes to each (a lane to a row: 16 and 8
  // bytes of a line at a time, and the store of 8192 rows alone took 38 us).
  int head[kCols], pos[kCols];
  bool mine[kCols];
  int64_t qrow[kCols];
  attn_u32x4 qt[kCols][D / 64][4];
  bf16x8 q[kCols][kSteps];
#pragma unroll
  for (int y = 0; y < kCols; ++y) {
    const int r = 32 * (kCols * wave + y) + n, tok = r / group;
    head[y] = kvh * group + r % group;
    mine[y] = tok < c.tokens;
    pos[y] = mine[y] ? c.pos0 + tok : -1;
    qrow[y] = c.row0 + c.tok0 + (mine[y] ? tok : 0);
    const int64_t from = qrow[y] * a.q_stride + static_cast<int64_t>(head[y]) * D;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t* row = a.q + __shfl(from, 8 * i + (lane >> 3));
      const bool in = __shfl(static_cast<int>(mine[y]), 8 * i + (lane >> 3)) != 0;
#pragma unroll
      for (int g = 0; g < D / 64; ++g) {
        qt[y][g][i] = reinterpret_cast<const attn_u32x4*>(row + 64 * g)[lane & 7];
        if (!in) qt[y][g][i] = attn_u32x4{0, 0, 0, 0};
      }
    }
  }
  const float scale = score_scale<kE4m3>(a, kvh);

  const bool work = 32 * kCols * wave < c.tokens * group;  // whether any of the wave's rows is one
  // the tiles that the rows see: the first tokens', then the window's
  const int pmin = c.pos0, pmax = c.pos0 + c.tokens - 1;
  const int low = a.window > 0 ? max(0, pmin - a.window + 1) : 0;
  // (from a page's 16 tokens on, where no first tokens lie on the same grid)
  const int begin = a.first > 0 ? low & ~(kTile - 1) : low & ~15;
  const int nf = min((min(a.first, low) + kTile - 1) / kTile, begin / kTile);
  const int all_tiles = pmax < 0 ? 0 : nf + (pmax - begin) / kTile + 1;
  const int pieces = max(1, min(pa.pieces, all_tiles / (G * kMinTiles)));
  if (piece >= pieces) return;
  // the piece's tiles [t0, t1) go to the groups in equal parts, whose number of
  // steps is the same: what a group has past its last tile is hidden
  const int t0 = __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<int64_t>(all_tiles) * piece / pieces));
  const int t1 = __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<int64_t>(all_tiles) * (piece + 1) / pieces));
  const int steps = (t1 - t0 + G - 1) / G, first_tile = t0 + part_of * steps;
  const int tiles = max(0, min(steps, t1 - first_tile));
  auto tile_at = [&](int i) {
    const int t = first_tile + i;
    return t < nf ? t * kTile : begin + (t - nf) * kTile;
  };
  auto begin_of = [&](int i) { return __builtin_amdgcn_readfirstlane(tile_at(i)); };
  if (pa.pieces > 1 && piece == 0 && kvh == 0 && threadIdx.x < c.tokens) pa.plan[c.row0 + c.tok0 + threadIdx.x] = pieces;

  // Pages of 16 tiles at a time: lane 4 i + j has tokens 16 j on of tile i0 + i.
  auto load_pages = [&](int i0) {
    const int i = i0 + (lane >> 2);
    int page = -1;
    if (i < tiles) {
      const int t = tile_at(i) + 16 * (lane & 3);
      if (t < c.len) page = a.tables[c.b * a.table_stride + (t >> a.kv.bs_shift)];
    }
    return page;
  };
  const int mask = (1 << a.kv.bs_shift) - 1;
  const int st = static_cast<int>(a.kv.st) * kSize;
  int64_t off;     // where the lane's 16 tokens lie in K and in V
  uint64_t paged;  // which of them have a page
  auto locate = [&](int i0, int page) {
    const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.kv.num_blocks);
    const int t = tile_at(i0 + (lane >> 2)) + 16 * (lane & 3);
    off = (ok ? page : 0) * a.kv.sb * kSize + static_cast<int64_t>(t & mask) * st;
    paged = __ballot(ok);
  };
  int next = -1;
  // Tile i, in order: where this wave's part of it lies, and which of its pages
  // there are (past the last tile: the cache's first page, and none).
  auto fetch = [&](int i, uint32_t* pages) __attribute__((always_inline)) {
    if ((i & 15) == 0) {
      if (i == 0) next = load_pages(0);
      locate(i, next);
      next = load_pages(i + 16);
    }
    *pages = static_cast<uint32_t>(paged >> (4 * (i & 15))) & 15u;
    const int from = 4 * (i & 15) + wave;
    return static_cast<int64_t>(
        static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(off >> 32), from))) << 32 |
        static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(off), from)));
  };

  // staging: wave w brings tokens 16 w to 16 w + 15, load j the rows from
  // j * 64 / kPieces on
  GlobalBytes kb = (GlobalBytes)(static_cast<const uint8_t*>(a.kv.k) + kvh * a.kv.sh * kSize);
  GlobalBytes vb = (GlobalBytes)(static_cast<const uint8_t*>(a.kv.v) + kvh * a.kv.sh * kSize);
  const int srow = lane / kPieces, spiece = lane % kPieces;
  constexpr int kRowsPerLoad = 64 / kPieces;
  const uint32_t goff = srow * st + spiece * 16;
  attn_u32x4 kr[kLoads], vr[kLoads];
  auto load = [&](GlobalBytes base, int64_t at, attn_u32x4 (&r)[kLoads]) __attribute__((always_inline)) {
    const uint32_t go = here(goff);
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      r[j] = *reinterpret_cast<const __attribute__((address_space(1))) attn_u32x4*>(scalar(base + at + j * kRowsPerLoad * st) + go);
  };
  // whole: every row of the work-group sees every token of the tile
  auto is_whole = [&](int t, uint32_t pages) {
    return pages == 15u && t + kTile - 1 <= pmin && (a.window == 0 || t > pmax - a.window || t + kTile <= a.first);
  };
  // To LDS.  0 times an infinity or a NaN is not 0, so of a tile that not every
  // row sees whole such values become 0 here; the rows that do see one get it
  // at the end.
  auto put = [&](uint8_t* to, attn_u32x4 (&r)[kLoads]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int row = 16 * wave + j * kRowsPerLoad + srow;
      if constexpr (kE4m3) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          uint32_t w[4];
          widen(r[j][2 * p], w), widen(r[j][2 * p + 1], w + 2);
          *reinterpret_cast<attn_u32x4*>(to + row * kRowBytes + (piece_at<D>(row, 2 * spiece + p) << 4)) =
              attn_u32x4{w[0], w[1], w[2], w[3]};
        }
      } else {
        *reinterpret_cast<attn_u32x4*>(to + row * kRowBytes + (piece_at<D>(row, spiece) << 4)) = r[j];
      }
    }
  };
  auto put_values = [&](int buf, int tile, bool whole) __attribute__((always_inline)) {
    if (!whole) {
      uint32_t odd = 0;
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= not_finite<kE4m3>(vr[j][e]);
      if (__ballot(odd != 0) != 0) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) vr[j][e] &= ~not_finite<kE4m3>(vr[j][e]);
        if (lane == 0) atomicOr(&s_odd[tile >> 5 & 1], 1u << (tile & 31));
      }
    }
    put(s_v[buf], vr);
  };

  // The reference of a row, its negative as the scores' products take it (+inf: none
  // yet, so that the first score of the row leads to one), the sum.
  float m[kCols], less[kCols], l[kCols];
  bool any[kCols];
  f32x16 o[kCols][kDb];
#pragma unroll
  for (int y = 0; y < kCols; ++y) {
    m[y] = kNegInf, less[y] = mine[y] ? __builtin_inff() : 0.0f, l[y] = 0.0f, any[y] = false;
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[y][d][e] = 0.0f;
  }

  // LDS addresses.  K: token 32 b + n, piece 2 s + h.  V: the 16 lanes of a quarter
  // read 4 tokens x 16 dims and are left with 4 tokens of one dim each.
  const int vrow = 4 * h + ((lane & 15) >> 2);  // and vrow + 8 and so on
  const int vpiece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  int kat[kSteps], vat[kDb][2];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) kat[k] = n * kRowBytes + (piece_at<D>(n, 2 * k + h) << 4);
#pragma unroll
  for (int d = 0; d < kDb; ++d)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      vat[d][e] = (vrow + 8 * e) * kRowBytes + (piece_at<D>(vrow + 8 * e, 4 * d + vpiece) << 4) + 8 * (lane & 1);
  f32x16 s[2][kCols];   // scores of the two halves of a tile
  bf16x8 w[kCols][2];   // weights of a half
  // One of the kSteps products of the scores of half b of the tile in buffer buf.
  auto score = [&](int buf, int b, int k) __attribute__((always_inline)) {
    const bf16x8 x = *reinterpret_cast<const bf16x8*>(&s_k[buf][32 * b * kRowBytes + kat[k]]);
#pragma unroll
    for (int y = 0; y < kCols; ++y) s[b][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, q[y][k], s[b][y], 0, 0, 0);
  };
  auto clear = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int y = 0; y < kCols; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[b][y][e] = 0.0f;
  };
  // What the rows see of half b of the tile at t: a bit for each of its 32
  // tokens, the lane's own at the places that its scores have.
  auto hide = [&](int t, int b, uint32_t pages) __attribute__((always_inline)) {
    auto below = [](int x) { return x >= 32 ? ~0u : x <= 0 ? 0u : (1u << x) - 1u; };  // tokens 0 to x - 1
    const int at = t + 32 * b;
    const uint32_t there = (pages >> (2 * b) & 1u ? 0xffffu : 0u) | (pages >> (2 * b + 1) & 1u ? 0xffff0000u : 0u);
    const uint32_t first = below(min(a.first, 0x40000000) - at);
#pragma unroll
    for (int y = 0; y < kCols; ++y) {
      const int rel = pos[y] - at;
      const uint32_t old = a.window > 0 ? below(rel - a.window + 1) & ~first : 0u;
      const uint32_t in = (pos[y] < 0 ? 0u : below(rel + 1) & ~old & there) >> (4 * h);
      any[y] |= (in & 0x0f0f0f0fu) != 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t keep = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(in), 8 * (e >> 2) + (e & 3), 1));
        s[b][y][e] = __uint_as_float((__float_as_uint(s[b][y][e]) & keep) | (0xff800000u & ~keep));
      }
    }
  };
  // Weights number x to x + n - 1 of half b against 2^-off, and their sum.
  float part[kCols][2];
  uint32_t now[kCols][8];
  auto weigh = [&](int b, int y, float off, int x, int n) __attribute__((always_inline)) {
#pragma unroll
    for (int e = x; e < x + n; e += 2) {
      now[y][e / 2] = pack_bf16x2(__builtin_amdgcn_exp2f(__builtin_fmaf(s[b][y][e], scale, off)),
                                  __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][y][e + 1], scale, off)));
      part[y][e / 2 & 1] = add_two(now[y][e / 2], part[y][e / 2 & 1]);
    }
  };
  // One of the kSteps products of the weighted values of half b in buffer buf: 16
  // tokens, 32 dims, the dims in turn so that a sum is not waited for.
  auto add = [&](int buf, int b, int x) __attribute__((always_inline)) {
    const int d = x % kDb, k = x / kDb;
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      reinterpret_cast<s16x4*>(&v)[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)((LdsBytes)s_v[buf] + vat[d][e] + (32 * b + 16 * k) * kRowBytes));
#pragma unroll
    for (int y = 0; y < kCols; ++y) o[y][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, w[y][k], o[y][d], 0, 0, 0);
  };
  // Half b of the tile at t in buffer buf: its weights, beside the products of
  // the half before (values) and of the one after (scores).  These three do not
  // depend on each other, so that matrix and vector instructions run together.
  auto half = [&](int buf, int b, int t, uint32_t pages, bool whole) __attribute__((always_inline)) {
    if (!whole) hide(t, b, pages);
    clear(b ^ 1);
#pragma unroll
    for (int y = 0; y < kCols; ++y) any[y] |= whole, part[y][0] = part[y][1] = 0.0f;
#pragma unroll
    for (int x = 0; x < kSteps; ++x) {
      score(b == 0 ? buf : buf ^ 1, b ^ 1, x);
      add(b == 0 ? buf ^ 1 : buf, b ^ 1, x);
#pragma unroll
      for (int y = 0; y < kCols; ++y) weigh(b, y, less[y], 16 / kSteps * x, 16 / kSteps);
    }
    // The order to issue them in with 64 dims: LDS reads of a step ahead, or all
    // of them where two products share each, then every product with vector
    // instructions behind it.  (As the compiler has them: prompts of 1024 and 8192
    // 24.8 and 605 us, 23.0 and 584 so; with 128 dims its order is the best one.)
    if constexpr (D == 64) {
      __builtin_amdgcn_sched_group_barrier(0x100, kCols == 1 ? 3 : 12, 0);
#pragma unroll
      for (int x = 0; x < kSteps; ++x) {
#pragma unroll
        for (int y = 0; y < 2 * kCols; ++y) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, kCols == 1 ? 3 : 0, 0);
      }
    }
    // Only if the weights come out large (or there is no reference) the half's
    // maximum is looked for, and they are formed again.
    bool large = false;
#pragma unroll
    for (int y = 0; y < kCols; ++y) large |= !(part[y][0] + part[y][1] < kMost);
    if (__ballot(large) != 0) {
#pragma unroll
      for (int y = 0; y < kCols; ++y) {
        float top = s[b][y][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = __builtin_fmaxf(top, s[b][y][e]);
        top *= scale;
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float mn = __builtin_fmaxf(m[y], top), base = mn == kNegInf ? 0.0f : mn;
        const float keep = __builtin_amdgcn_exp2f(m[y] - base);
        m[y] = mn;
        less[y] = mn == kNegInf && mine[y] ? __builtin_inff() : -base;
        l[y] *= keep;
#pragma unroll
        for (int d = 0; d < kDb; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[y][d][e] *= keep;
        part[y][0] = part[y][1] = 0.0f;
        weigh(b, y, -base, 0, 16);
      }
    }
#pragma unroll
    for (int y = 0; y < kCols; ++y) {
      l[y] += part[y][0] + part[y][1];
      w[y][0] = __builtin_bit_cast(bf16x8, attn_u32x4{now[y][0], now[y][1], now[y][2], now[y][3]});
      w[y][1] = __builtin_bit_cast(bf16x8, attn_u32x4{now[y][4], now[y][5], now[y][6], now[y][7]});
    }
  };

  {
    uint8_t* mid = s_kv[1] + wave * 4096;  // the wave's own
#pragma unroll
    for (int y = 0; y < kCols; ++y)
#pragma unroll
      for (int g = 0; g < D / 64; ++g) {
        wave_order();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 8 * i + (lane >> 3);
          *reinterpret_cast<Piece*>(mid + row * 128 + (((lane & 7) ^ (row & 7)) << 4)) = qt[y][g][i];
        }
        wave_order();
#pragma unroll
        for (int k = 0; k < 4; ++k)
          q[y][4 * g + k] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const Piece*>(mid + n * 128 + (((2 * k + h) ^ (n & 7)) << 4)));
      }
  }

  if (threadIdx.x < 2) s_odd[threadIdx.x] = 0;
  __syncthreads();
  if (steps > 0) {
    // Tile i: K of tile i + 1 and V of tile i go to LDS, K of i + 2 and V of i + 1
    // are asked for; then its two halves, with the only barrier between them: it
    // shows what was put, and what is put next takes the place of K of tile i - 1
    // and V of i - 2, which no wave reads behind it.
    const bool two = pmax - begin_of(steps - 1) >= 32;  // whether any row sees the last tile's second half
    uint32_t pages, ahead;
    int64_t at = fetch(0, &pages);
    load(kb, at, kr);
    load(vb, at, vr);
    at = fetch(1, &ahead);
    put(s_k[0], kr);
    load(kb, at, kr);
    for (int x = threadIdx.x & 255; x < kBytes / 16; x += 256)  // taken with weights of 0 by the first half
      reinterpret_cast<attn_u32x4*>(s_v[1])[x] = attn_u32x4{0, 0, 0, 0};
    __syncthreads();
    clear(0);
#pragma unroll
    for (int x = 0; x < kSteps; ++x) score(0, 0, x);
#pragma unroll
    for (int y = 0; y < kCols; ++y) w[y][0] = w[y][1] = __builtin_bit_cast(bf16x8, attn_u32x4{0, 0, 0, 0});
    auto step = [&](auto B, int i) __attribute__((always_inline)) {
      constexpr int buf = decltype(B)::value;
      const int t = begin_of(i);
      const bool whole = is_whole(t, pages);
      put(s_k[buf ^ 1], kr);
      put_values(buf, first_tile + i, whole);
      uint32_t later;
      const int64_t to = fetch(i + 2, &later);
      load(vb, at, vr);
      load(kb, to, kr);
      at = to;
      if (work) half(buf, 0, t, pages, whole);
      __syncthreads();
      if (work && (i + 1 < steps || two)) half(buf, 1, t, pages, whole);
      pages = ahead;
      ahead = later;
    };
    for (int i = 0; i < steps; i += 2) {
      step(std::integral_constant<int, 0>{}, i);
      if (i + 1 < steps) step(std::integral_constant<int, 1>{}, i + 1);
    }
    // the values of the last half
#pragma unroll
    for (int x = 0; x < kSteps; ++x) {
      if (steps & 1) {
        if (two)
          add(0, 1, x);
        else
          add(0, 0, x);
      } else {
        if (two)
          add(1, 1, x);
        else
          add(1, 0, x);
      }
    }
  }
  if (work && (s_odd[0] | s_odd[1]) != 0) {
    // What put() left out, for the rows that see it.  Only tiles that it marked are
    // looked at, a lane to a token, and of these only tokens that do hold something:
    // most often it lies past the sequence's end (a prompt of 2048 with NaN there
    // 53 us, as without; 975 with every token of every tile looked at).
    for (int i = 0; i < tiles; ++i) {
      const int tile = first_tile + i, from = begin_of(i);
      if ((s_odd[tile >> 5 & 1] >> (tile & 31) & 1) == 0) continue;
      const int mine_t = from + lane;
      int page = mine_t < c.len ? a.tables[c.b * a.table_stride + (mine_t >> a.kv.bs_shift)] : -1;
      const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.kv.num_blocks);
      const uint64_t there = __ballot(ok);
      uint32_t all = 0;  // as fetch() has them
#pragma unroll
      for (int j = 0; j < 4; ++j) all |= static_cast<uint32_t>(there >> (16 * j) & 1) << j;
      if (is_whole(from, all)) continue;
      uint32_t odd = 0;
      if (ok && mine_t <= pmax) {
        GlobalBytes v = vb + page * a.kv.sb * kSize + static_cast<int64_t>(mine_t & mask) * st;
#pragma unroll 2
        for (int k = 0; k < kPieces; ++k) {
          const attn_u32x4 x = *reinterpret_cast<const __attribute__((address_space(1))) attn_u32x4*>(v + 16 * k);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= not_finite<kE4m3>(x[e]);
        }
      }
      for (uint64_t left = __ballot(odd != 0); left != 0; left &= left - 1) {
        const int x = __builtin_ctzll(left), t = from + x;
        GlobalBytes v = vb + __builtin_amdgcn_readlane(page, x) * a.kv.sb * kSize + static_cast<int64_t>(t & mask) * st + 4 * h * kSize;
#pragma unroll
        for (int y = 0; y < kCols; ++y) {
          if (pos[y] < 0 || !sees(a, pos[y], t)) continue;
#pragma unroll
          for (int d = 0; d < kDb; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t w[2];
              if constexpr (kE4m3) {
                widen(*reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(v + 32 * d + 8 * k), w);
              } else {
                const attn_u32x2 x = *reinterpret_cast<const __attribute__((address_space(1))) attn_u32x2*>(v + 64 * d + 16 * k);
                w[0] = x[0], w[1] = x[1];
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float x = bf16_to_f32(static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1))));
                o[y][d][4 * k + e] += (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? x : 0.0f;
              }
            }
        }
      }
    }
  }

  // A 128-byte piece of 32 rows from the wave's part of LDS: row r to at(r) bytes
  // from `to`, rows of no token left out.
  __syncthreads();
  if constexpr (G == 2) {
    // the second group's sums to the first, lane by lane
    static_assert(kCols == 1, "32 rows a wave");
    Piece* at = reinterpret_cast<Piece*>(s_all[4 + wave]) + lane;
    float* ml = reinterpret_cast<float*>(s_all[3]) + 192 * wave + lane;
    if (part_of == 1) {
#pragma unroll
      for (int d = 0; d < kDb; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          at[64 * (4 * d + k)] = __builtin_bit_cast(attn_u32x4, f32x4{o[0][d][4 * k], o[0][d][4 * k + 1], o[0][d][4 * k + 2], o[0][d][4 * k + 3]});
      ml[0] = m[0], ml[64] = l[0], ml[128] = any[0] ? 1.0f : 0.0f;
    }
    __syncthreads();
    if (part_of == 1) return;
    const float m1 = ml[0], top = __builtin_fmaxf(m[0], m1), base = top == kNegInf ? 0.0f : top;
    const float f0 = __builtin_amdgcn_exp2f(m[0] - base), f1 = __builtin_amdgcn_exp2f(m1 - base);
    m[0] = top;
    l[0] = __builtin_fmaf(ml[64], f1, l[0] * f0);
    any[0] |= ml[128] != 0.0f;
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x4 x = __builtin_bit_cast(f32x4, at[64 * (4 * d + k)]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[0][d][4 * k + e] = __builtin_fmaf(x[e], f1, o[0][d][4 * k + e] * f0);
      }
    wave_order();
  }
  uint8_t* mid = s_kv[0] + wave * 32 * kOutRow;
  auto emit = [&](void* to, int64_t at, bool in) __attribute__((always_inline)) {
    wave_order();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 8 * i + (lane >> 3);
      const Piece x = *reinterpret_cast<const Piece*>(mid + row * kOutRow + 16 * (lane & 7));
      const int64_t there = __shfl(at, row);
      // (past the caches, where the next kernel would not find it on another die:
      // 64 tokens over 8000 32.0 us, 30.2 so)
      if (__shfl(static_cast<int>(in), row) != 0)
        __builtin_nontemporal_store(static_cast<attn_u32x4>(x), reinterpret_cast<attn_u32x4*>(static_cast<uint8_t*>(to) + there + 16 * (lane & 7)));
    }
    wave_order();
  };
  const float vs = kE4m3 && a.kv.v_scale ? a.kv.v_scale[kvh] : 1.0f;
#pragma unroll
  for (int y = 0; y < kCols; ++y) {
    float sum = l[y] + __shfl_xor(l[y], 32);
    const bool seen = any[y] | (__shfl_xor(static_cast<int>(any[y]), 32) != 0);
    if (pieces > 1) {
      const int64_t at = (static_cast<int64_t>(piece) * a.rows + qrow[y]) * a.heads + head[y];
#pragma unroll
      for (int d = 0; d < kDb; ++d) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<Piece*>(mid + n * kOutRow + 32 * k + 16 * h) =
              __builtin_bit_cast(attn_u32x4, f32x4{o[y][d][4 * k], o[y][d][4 * k + 1], o[y][d][4 * k + 2], o[y][d][4 * k + 3]});
        emit(pa.part_o, (at * D + 32 * d) * 4, mine[y]);
      }
      if (h == 0 && mine[y]) reinterpret_cast<f32x4*>(pa.part_ml)[at] = f32x4{m[y], sum, seen ? 1.0f : 0.0f, 0.0f};
      continue;
    }
    float f = vs / sum;
    if (a.sinks) {
      const float sink = bf16_to_f32(a.sinks[head[y]]) * kLog2e;
      const float top = __builtin_fmaxf(m[y], sink), base = top == kNegInf ? 0.0f : top;
      const float keep = __builtin_amdgcn_exp2f(m[y] - base);
      f = keep * (vs / (sum * keep + __builtin_amdgcn_exp2f(sink - base)));
    }
#pragma unroll
    for (int g = 0; g < D / 64; ++g) {
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = seen ? o[y][2 * g + d][4 * k + e] * f : 0.0f;
          *reinterpret_cast<HalfPiece*>(mid + n * kOutRow + 64 * d + 16 * k + 8 * h) =
              attn_u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
        }
      emit(a.out, (qrow[y] * a.out_stride + static_cast<int64_t>(head[y]) * D + 64 * g) * 2, mine[y]);
    }
  }
}

// Rows of a wave: 64 where the registers allow it and there are rows to fill the
// chip with, else 32 (a prompt of 8192 573 / 618 us, of 2048 60.7 / 54.3).
constexpr int kTwoCols = 2048;
int cols_of(int rows, int heads, int head_dim) {
  return head_dim == 64 && static_cast<int64_t>(rows) * heads >= 256 * kTwoCols ? 2 : 1;
}

// Pieces: no more than fill the chip (work-groups that it holds at once: three on a
// CU with heads of 64 dims, two with 128) when the tiles of rows alone do not.
constexpr int kCus = 256;
int fill_of(int head_dim) { return head_dim == 64 ? 768 : 512; }

// Where that gives more than one work-group to a CU and most rows of the tiles are
// there, two groups of waves in one work-group do what two pieces would, with half
// the partial sums or none and no join (one group and two: 512 tokens 21.6 / 13.8
// us, 430 over 2889 52.6 / 43.2, 64 over 8000 30.0 / 27.7, five of up to 200 over
// 634 with 128 dims in e4m3 31.2 / 23.0).  With tiles hardly filled or a CU to each
// piece the pieces are better (eight of up to 24 over 2000 19.1 / 22.3, 1055 with 4
// heads of 128 21.0 / 27.0), and with many tiles, where work-groups of four waves
// follow each other (1024 tokens 23.2 / 25.3; two of up to 1117 with 128 dims, the
// shorter chain for once, 34 / 28.5).  Nor for several sequences whose lengths may
// be very different, which fewer work-groups balance worse: kAlike is the tiles by
// which one may miss the longest, and half of those by which all together may
// (seven of up to 39 over up to 10753 62 / 117 us, two of up to 200 over up to 8000
// 64.5 / 90.5, eight of up to 128 over up to 4000 38 / 51, eight of up to 60 over up to
// 1900 23.4 / 29.2; eight of up to 128 over up to 900 23.8 / 19.7, two of up to 256 over
// up to 1800 34.5 / 30.6, three of up to 258 over up to 4563 with a window 56.3 / 49.0).
constexpr int64_t kAlike = 80;

// How long a tile of 64 dims takes a work-group, a join, and a partial sum's float on
// its way to it and back: a piece more has to save more than it costs (680 tokens in
// two pieces 27.2 us, in one 16.4; four of up to 120 over up to 1000 20.7 / 19.2).
constexpr double kTileUs = 1.2, kJoinUs = 4.0, kPartUs = 2e-6;

// No more tiles than the longest sequence, or the window over a tile's rows and the
// first tokens, has.
int64_t most_tiles(const Reach& r, int rows, int heads, int kv_heads, int head_dim) {
  const int per = 128 * cols_of(rows, heads, head_dim) / (heads / kv_heads);
  const int64_t all = (r.tokens + kTile - 1) / kTile;
  return r.window == 0 ? all : min(all, (r.window + per + kTile - 3) / kTile + 1 + (r.first + kTile - 1) / kTile);
}

struct Split {
  int groups, pieces;
};

Split split_of(int rows, int B, int heads, int kv_heads, int head_dim, int64_t most) {
  if (cols_of(rows, heads, head_dim) == 2) return {1, 1};
  const int per = 128 / (heads / kv_heads);
  const int64_t tiles = (static_cast<int64_t>(rows) + per - 1) / per + (B < rows ? B : rows) - 1;
  const int64_t wgs = tiles * kv_heads;
  auto top = [&](int64_t fill, int groups) { return max(int64_t{1}, min(fill / wgs, most / (groups * kMinTiles))); };
  const bool few = wgs <= kCus || (head_dim == 128 && wgs <= 2 * kCus && most >= 2 * kMinTiles);
  const bool even = B == 1 || (most <= kAlike && (B - 1) * most <= 2 * kAlike);
  const bool two = few && even && wgs * top(fill_of(head_dim), 1) > kCus && 2 * static_cast<int64_t>(rows) >= tiles * per;
  Split s{two ? 2 : 1, 1};
  double least = 0.0;
  for (int p = 1; p <= top(two ? kCus : fill_of(head_dim), s.groups); ++p) {
    const double chain = kTileUs * head_dim / 64 * static_cast<double>(most) / (s.groups * p);
    const double join = p == 1 ? 0.0 : kJoinUs + kPartUs * p * rows * heads * (head_dim + 4);
    if (p == 1 || chain + join < least) s.pieces = p, least = chain + join;
  }
  return s;
}

}  // namespace

size_t prefill_call_bytes(int rows, int B, int heads, int kv_heads, int head_dim, const Reach& r) {
  const int pieces = split_of(rows, B, heads, kv_heads, head_dim, most_tiles(r, rows, heads, kv_heads, head_dim)).pieces;
  if (pieces == 1) return 0;
  return static_cast<size_t>(pieces) * rows * heads * (head_dim + 4) * sizeof(float) +
         ((static_cast<size_t>(rows) * sizeof(int) + 15) & ~size_t{15});
}

// For any call of up to `rows` rows: with t tiles there are at most fill / (t
// kv_heads) pieces of at most t * per rows.
size_t prefill_workspace_bytes(int rows, int heads, int kv_heads, int head_dim) {
  const int per = 128 / (heads / kv_heads);
  const size_t pieces = fill_of(head_dim) / kv_heads;
  if (pieces < 2) return 0;
  const size_t part_rows = min(static_cast<size_t>(rows) * pieces, static_cast<size_t>(per) * fill_of(head_dim) / kv_heads);
  return part_rows * heads * (head_dim + 4) * sizeof(float) + ((static_cast<size_t>(rows) * sizeof(int) + 15) & ~size_t{15});
}

hipError_t launch_prefill(const AttendArgs& a, void* workspace, hipStream_t s) {
  const int cols = cols_of(a.rows, a.heads, a.kv.head_dim), per = 128 * cols / (a.heads / a.kv.kv_heads);
  PieceArgs pa{};
  const Split split = split_of(a.rows, a.B, a.heads, a.kv.kv_heads, a.kv.head_dim,
                               most_tiles(reach_of(a), a.rows, a.heads, a.kv.kv_heads, a.kv.head_dim));
  pa.pieces = split.pieces;
  const size_t parts = static_cast<size_t>(pa.pieces) * a.rows * a.heads;
  pa.part_o = static_cast<float*>(workspace);
  pa.part_ml = pa.part_o + parts * a.kv.head_dim;
  pa.plan = reinterpret_cast<int*>(pa.part_ml + parts * 4);
  AttendArgs x = a;  // kSearch of its sequences at a time
#define GX_PREFILL(D_, E_, C_, G_) \
  hipLaunchKernelGGL((prefill_kernel<D_, E_, C_, G_>), grid, dim3(256 * G_), 0, s, x, pa)
#define GX_PREFILL_E(D_, C_, G_)               \
  do {                                         \
    if (a.kv.e4m3) GX_PREFILL(D_, true, C_, G_); \
    else GX_PREFILL(D_, false, C_, G_);        \
  } while (0)
  for (int b = 0; b < a.B; b += kSearch) {
    x.B = min(kSearch, a.B - b);
    x.offsets = a.offsets + b;
    x.lens = a.lens + b;
    x.tables = a.tables + b * a.table_stride;
    // sum of ceil(new tokens / per), at most one tile more for each sequence that has rows
    const int64_t tiles = (static_cast<int64_t>(a.rows) + per - 1) / per + min(x.B, a.rows);
    const dim3 grid(static_cast<unsigned>(tiles * a.kv.kv_heads * pa.pieces));
    if (a.kv.head_dim == 64 && cols == 2) GX_PREFILL_E(64, 2, 1);
    else if (a.kv.head_dim == 64 && split.groups == 1) GX_PREFILL_E(64, 1, 1);
    else if (a.kv.head_dim == 64) GX_PREFILL_E(64, 1, 2);
    else if (split.groups == 1) GX_PREFILL_E(128, 1, 1);
    else GX_PREFILL_E(128, 1, 2);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
#undef GX_PREFILL_E
#undef GX_PREFILL
  if (pa.pieces == 1) return hipSuccess;
  JoinArgs j{};
  j.part_o = pa.part_o;
  j.part_ml = pa.part_ml;
  j.plan = pa.plan;
  j.max_pieces = pa.pieces;
  return launch_join(a, j, pa.pieces, s);
}

}  // namespace gxmoe
