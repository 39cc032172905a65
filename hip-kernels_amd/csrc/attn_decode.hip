// attn_decode.hip -- attention of one new token per sequence over the paged
// cache (gfx950).
//
// Mathematics.  With base-2 scores s = (q . k) scale log2(e), a wave keeps for
// each head a reference m, the sum l of 2^(s - m) and the weighted sum O of
// the values; two such triples over disjoint tokens join as
//   M = max(m1, m2), l = l1 2^(m1 - M) + l2 2^(m2 - M), O likewise,
// so tokens are split over tiles, waves and work-groups in any way.
//
// Bound by reading K and V once: 8 heads on a kv head take 8 flops per byte in
// bf16, 16 in e4m3.
// Everything else is laid out so that nothing but the loads is slow: K and V go
// from memory to registers, whole 128-byte rows, and from there into the
// matrix cores without passing through LDS.
//   S^T = K Q^T   (16 tokens x 16 heads a product): a lane holds one token's
//                 quarter of the dims, the same quarter of its head's query.
//   O^T = V^T P^T (16 dims x 16 heads): the lane that S^T leaves with head
//                 l % 16 and tokens 4 (l / 16) + i is the one that holds these as
//                 the second operand, so the weights stay where they are; V's
//                 rows are read 16 lanes to a row and interleaved by byte
//                 permutes (the order of dims and tokens inside a product is free
//                 as long as both operands agree).
// The reference m of a head moves only when a score exceeds it by 2^8: until
// then weights up to 256 lose nothing in bf16 or fp32, and the tile needs no
// exchange between lanes.  The weights meet the values as two bf16 each.
//
// With 64 heads on 8 of 64 dims in bf16, joins included: one sequence of 131072 51
// us, 5.3 TB/s (a kernel that only reads the same, 44 us and 6.1); four of them 6.3
// TB/s; 64 of 4000 96 us, 5.5 TB/s; 64 of very different lengths up to 8192 27.4 us,
// 3.7 TB/s, of which the join takes 4.  With 32 heads on 8 of 128 one of 131072 88.6
// us, 6.1 TB/s; with 64 dims in e4m3 31.2 us, 4.3 TB/s.
// (Pairs of times beside the choices below are of one run each, and may be older.)
#include "attn_device.h"

namespace gxmoe {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;      // tokens per step of a wave
constexpr int kClasses = 2;     // of a piece's length
constexpr int kWholeTiles = 32;  // tiles up to which many sequences are not cut
constexpr float kSlack = 8.0f;  // how far a score may exceed the reference, in powers of two

// The tiles of a sequence that its new token sees: the first nf tiles (first
// tokens of a windowed sequence), then all from tile `main` on.
struct Seen {
  int len, low;  // tokens from `low` on are inside the window
  int nf, main, tiles;
};

__device__ __forceinline__ Seen seen_tiles(const AttendArgs& a, int len) {
  Seen s;
  s.len = len;
  s.low = a.window > 0 && len > a.window ? len - a.window : 0;
  s.main = s.low / kTile;
  s.nf = min((min(a.first, s.low) + kTile - 1) / kTile, s.main);
  s.tiles = s.nf + (len + kTile - 1) / kTile - s.main;
  return s;
}

struct SplitArgs {
  int slots, min_tiles;  // pieces aimed at (0: one per sequence), smallest piece
  int max_slots;         // no more pieces
  bool same_die;         // all heads of a piece on one of the eight dies
  bool whole_ok;         // sequences of about the same length need not be cut
  float* part_o;         // [piece][heads][D] sums of the cut sequences' pieces
  float* part_ml;        // [piece][heads][4] reference, sum, whether any token was seen
  int* plan;             // [B][2] first piece and number of pieces
};

// What a work-group does: tiles [t0, t1) of sequence b, piece `slot` of all.
struct Piece {
  int b, t0, t1, chunks, first_slot;
  Seen seen;
};

// Sequences are cut into pieces of `size` tiles, the size chosen from all
// lengths so that the pieces of one kv head are about sp.slots in number; every
// wave works it out from the lengths, which only the device knows (64 kSeqs at a
// time, kSeqs to a lane, with scans over the lanes' registers).  The pieces are
// numbered by classes of their length, the longest first: late in the grid they
// would run when little else does.
template <int kSeqs>
__device__ __forceinline__ bool find_piece(const AttendArgs& a, const SplitArgs& sp, int slot, Piece* p) {
  const int lane = threadIdx.x & 63;
  int len[kSeqs], tiles[kSeqs];  // -1: no sequence
  auto read = [&](int b0) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kSeqs; ++j) len[j] = b0 + 64 * j + lane < a.B ? seq_len(a, b0 + 64 * j + lane) : -1;
#pragma unroll
    for (int j = 0; j < kSeqs; ++j) tiles[j] = len[j] < 0 ? -1 : seen_tiles(a, len[j]).tiles;
  };
  int total = 0, longest = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64 * kSeqs) {
    read(b0);
#pragma unroll
    for (int j = 0; j < kSeqs; ++j) total += max(tiles[j], 0), longest = max(longest, tiles[j]);
  }
  total = __builtin_amdgcn_readlane(wave_scan(total), 63);
  int size = max(sp.min_tiles, (total + sp.slots - 1) / sp.slots);
  if (sp.whole_ok) {
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) longest = max(longest, __shfl_xor(longest, x));
    if (longest <= 2 * kWholeTiles && 2 * static_cast<int64_t>(longest) * a.B <= 3 * static_cast<int64_t>(total)) size = max(size, longest);
  }
  const float per_size = 1.0f / static_cast<float>(size);  // (all waves divide alike: no more is asked of it)
  int cuts[kSeqs];
  auto cut = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kSeqs; ++j) cuts[j] = max(1, static_cast<int>(__builtin_fmaf(static_cast<float>(tiles[j]), per_size, 0.5f)));
  };
  cut();
  int before = 0;
  for (int k = 0; k < kClasses; ++k) {
    // tiles of a sequence of class k: at least `least`, and less than the class before
    const int least = k == kClasses - 1 ? 0 : size >> (2 * k + 1), below = k == 0 ? 0x7fffffff : size >> (2 * k - 1);
    for (int b0 = 0; b0 < a.B; b0 += 64 * kSeqs) {
      if (a.B > 64 * kSeqs) read(b0), cut();
      int mine[kSeqs], sum = 0;
#pragma unroll
      for (int j = 0; j < kSeqs; ++j) {
        mine[j] = tiles[j] >= least && tiles[j] < below ? cuts[j] : 0;
        sum += mine[j];
      }
      const int upto = wave_scan(sum);
      const int all = __builtin_amdgcn_readlane(upto, 63);
      if (slot < before + all) {
        const int at = slot - before;
        const int who = __builtin_ctzll(__ballot(at < upto));
        int first = __builtin_amdgcn_readlane(upto, who) - __builtin_amdgcn_readlane(sum, who);
#pragma unroll
        for (int j = 0; j < kSeqs; ++j) {
          const int n = __builtin_amdgcn_readlane(mine[j], who);
          if (at >= first && at < first + n) {
            p->b = b0 + 64 * j + who;
            p->chunks = n;
            p->first_slot = before + first;
            p->seen = seen_tiles(a, __builtin_amdgcn_readlane(len[j], who));
            p->t0 = static_cast<int>(static_cast<int64_t>(p->seen.tiles) * (at - first) / n);
            p->t1 = static_cast<int>(static_cast<int64_t>(p->seen.tiles) * (at - first + 1) / n);
          }
          first += n;
        }
        return true;
      }
      before += all;
    }
  }
  return false;
}

// One tile's K and V as a lane holds them.  Half j: of token 16 j + l % 16 the
// 16 bytes from 64 c + 16 (l / 16) on, for every c, so that a load takes 64
// bytes of a row.  Row i: token 16 (i / 4) + 4 (l / 16) + i % 4, dims
// (l % 16) D/16 on.
template <int D, bool kE4m3>
struct TileRegs {
  static constexpr int kKd = D / 16 * (kE4m3 ? 1 : 2);  // dwords of K per half
  static constexpr int kVd = D / 64 * (kE4m3 ? 1 : 2);  // dwords of a row of V
  uint32_t k[2][kKd];
  uint32_t v[8][kVd];
};

// N dwords, 16 bytes at a time `step` bytes apart.
template <int N>
__device__ __forceinline__ void load_dwords(GlobalBytes p, uint32_t (&d)[N], int step = 16) {
  if constexpr (N == 1) {
    d[0] = __builtin_nontemporal_load(reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(p));
  } else if constexpr (N == 2) {
    const attn_u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const __attribute__((address_space(1))) attn_u32x2*>(p));
    d[0] = x[0], d[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const attn_u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const __attribute__((address_space(1))) attn_u32x4*>(p + i * step));
#pragma unroll
      for (int c = 0; c < 4; ++c) d[4 * i + c] = x[c];
    }
  }
}

template <int D, bool kE4m3, int W>
__global__ __launch_bounds__(64 * W, 2) void decode_kernel(AttendArgs a, SplitArgs sp) {
  typedef TileRegs<D, kE4m3> Regs;
  constexpr int kSteps = D / 32;             // products of 32 dims per half
  constexpr int kDt = D / 16;                // tiles of 16 dims of the output
  constexpr int kSize = kE4m3 ? 1 : 2;       // bytes per element
  constexpr int kRow = D + 4;                // floats of a head's partial result in LDS
  __shared__ float s_o[W][16][kRow];
  __shared__ float s_m[W][16], s_l[W][16];
  __shared__ int s_any[W];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int group = a.heads / a.kv.kv_heads;
  const int parts = (group + 15) / 16;  // tiles of 16 heads per kv head
  // the tiles of heads of a piece side by side: the pieces that there are come
  // first in the grid and lie on all CUs (piece-minor, 128 of 1032 work-groups
  // shared a few CUs: one sequence of 4000, 17.9 us)
  const int th = a.kv.kv_heads * parts;
  int piece = blockIdx.x / th, tile_of_heads = blockIdx.x % th;
  if (sp.same_die) {
    piece = blockIdx.x / (8 * th) * 8 + blockIdx.x % 8;
    tile_of_heads = blockIdx.x / 8 % th;
    if (piece >= sp.max_slots) return;
  }
  const int kvh = tile_of_heads / parts, h0 = kvh * group + (tile_of_heads % parts) * 16;
  const int nh = min(16, (kvh + 1) * group - h0);

  Piece p;
  if (sp.slots > 0) {
    if (!(a.B <= 64 ? find_piece<1>(a, sp, piece, &p) : find_piece<4>(a, sp, piece, &p))) return;
    for (int* x : {&p.b, &p.t0, &p.t1, &p.chunks, &p.first_slot, &p.seen.len, &p.seen.low, &p.seen.nf, &p.seen.main,
                   &p.seen.tiles})
      *x = __builtin_amdgcn_readfirstlane(*x);  // the same in all lanes: addresses in scalar registers
  } else {
    p.b = piece;
    p.chunks = 1;
    p.first_slot = 0;
    p.seen = seen_tiles(a, __builtin_amdgcn_readfirstlane(seq_len(a, p.b)));
    p.t0 = 0;
    p.t1 = p.seen.tiles;
  }
  if (sp.slots > 0 && p.t0 == 0 && tile_of_heads == 0 && threadIdx.x == 0) {
    sp.plan[2 * p.b] = p.first_slot;
    sp.plan[2 * p.b + 1] = p.chunks;
  }

  // queries: head h0 + n, the dims that K's loads bring for step s (a load of
  // 16 bytes is one step of bf16 and two of e4m3)
  bf16x8 q[kSteps];
  {
    const uint16_t* row = a.q + p.b * a.q_stride + static_cast<int64_t>(h0 + min(n, nh - 1)) * D;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = kE4m3 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
      attn_u32x4 x = *reinterpret_cast<const attn_u32x4*>(row + d);
      if (n >= nh) x = attn_u32x4{0, 0, 0, 0};
      q[s] = __builtin_bit_cast(bf16x8, x);
    }
  }
  const float scale = score_scale<kE4m3>(a, kvh);

  // Pages of 32 of this wave's tiles at a time: lane 2 i + j has half j of
  // the i-th (tile t0 + wave + W i).
  const int mine = max(0, (p.t1 - p.t0 - wave + W - 1) / W);
  auto tile_of = [&](int i) {  // where the wave's i-th tile begins
    const int t = p.t0 + wave + W * i;
    return (t < p.seen.nf ? t : p.seen.main + t - p.seen.nf) * kTile;
  };
  auto load_pages = [&](int i0) {
    const int i = i0 + (lane >> 1);
    int page = -1;
    if (i < mine) {
      const int t = tile_of(i) + 16 * (lane & 1);
      if (t < p.seen.len) page = a.tables[p.b * a.table_stride + (t >> a.kv.bs_shift)];
    }
    return page;
  };
  GlobalBytes kb = (GlobalBytes)(static_cast<const uint8_t*>(a.kv.k) + kvh * a.kv.sh * kSize);
  GlobalBytes vb = (GlobalBytes)(static_cast<const uint8_t*>(a.kv.v) + kvh * a.kv.sh * kSize);
  const int st = static_cast<int>(a.kv.st) * kSize;
  const uint32_t koff = n * st + g * 16, voff = 4 * g * st + n * (D / 16) * kSize;
  const int mask = (1 << a.kv.bs_shift) - 1;

  // where their halves lie in K and V (the cache's first page where there is
  // none: what is read there is hidden), and which have a page
  int64_t off;
  uint64_t paged;
  auto locate = [&](int i0, int page) {
    const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.kv.num_blocks);
    const int t = tile_of(i0 + (lane >> 1)) + 16 * (lane & 1);
    off = (ok ? page : 0) * a.kv.sb * kSize + static_cast<int64_t>(t & mask) * st;
    paged = __ballot(ok);
  };
  locate(0, load_pages(0));
  int next_pages = -1;
  auto load = [&](int i, Regs& r) {
    const uint32_t ko = here(koff), vo = here(voff);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int from = 2 * (i & 31) + j;
      const int64_t at =
          static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(
                                   __builtin_amdgcn_readlane(static_cast<int>(off >> 32), from)))
                               << 32) |
          static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(off), from));
      GlobalBytes ks = scalar(kb + at);
      GlobalBytes vs = vb + at;
      load_dwords(ks + ko, r.k[j], 64);
#pragma unroll
      for (int c = 0; c < 4; ++c) load_dwords(scalar(vs + c * st) + vo, r.v[4 * j + c]);
    }
  };

  float m = kNegInf, l = 0.0f;
  bool any = false;  // whether the wave saw a token (its scores may all be -inf)
  f32x4 o[kDt];
#pragma unroll
  for (int d = 0; d < kDt; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  auto compute = [&](int i, bool have0, bool have1, Regs& r) {
    const int t = tile_of(i);
    f32x4 s[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t kd[D / 8];
      if constexpr (kE4m3) {
#pragma unroll
        for (int c = 0; c < Regs::kKd; ++c) widen(r.k[j][c], kd + 2 * c);
      } else {
#pragma unroll
        for (int c = 0; c < Regs::kKd; ++c) kd[c] = r.k[j][c];
      }
      s[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < kSteps; ++c)
        s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, attn_u32x4{kd[4 * c], kd[4 * c + 1], kd[4 * c + 2], kd[4 * c + 3]}), q[c], s[j], 0,
            0, 0);
    }
    uint32_t vd[8][D / 32];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      if constexpr (kE4m3) {
#pragma unroll
        for (int x = 0; x < Regs::kVd; ++x) widen(r.v[c][x], vd[c] + 2 * x);
      } else {
#pragma unroll
        for (int x = 0; x < Regs::kVd; ++x) vd[c][x] = r.v[c][x];
      }
    }
    const bool whole = have0 && have1 && t + kTile <= p.seen.len && (t >= p.seen.low || t + kTile <= a.first);
    if (whole) {
      any = true;
    } else {
      // hidden tokens: no score, and a value of zero, whatever the page holds
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int at = t + 16 * (c >> 2) + 4 * g + (c & 3);
        const bool in = (c < 4 ? have0 : have1) && at < p.seen.len && (at >= p.seen.low || at < a.first);
        any |= __ballot(in) != 0;
        s[c >> 2][c & 3] = in ? s[c >> 2][c & 3] : kNegInf;
#pragma unroll
        for (int x = 0; x < D / 32; ++x) vd[c][x] = in ? vd[c][x] : 0u;
      }
    }
    float top = __builtin_fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int c = 1; c < 4; ++c) top = __builtin_fmaxf(top, __builtin_fmaxf(s[0][c], s[1][c]));
    top *= scale;
    if (__ballot(top > m + kSlack) != 0) {
      top = __builtin_fmaxf(top, __shfl_xor(top, 16));
      top = __builtin_fmaxf(top, __shfl_xor(top, 32));
      const float mn = __builtin_fmaxf(m, top);
      const float keep = __builtin_amdgcn_exp2f(m - (mn == kNegInf ? 0.0f : mn));
      m = mn;
      l *= keep;
#pragma unroll
      for (int d = 0; d < kDt; ++d)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[d][c] *= keep;
    }
    const float base = m == kNegInf ? 0.0f : m;
    float w[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) w[c] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c >> 2][c & 3], scale, -base));
    l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    // The weights as two bf16 each, cut off and what that leaves: 16 bits of them
    // count, for a product that the loads hide.  The second is not 0 where the weight
    // is not, or 0 times an infinite value would be NaN: it is at least 2^-17 of the
    // weight, which is less than these bits, and bf16's smallest number.  A weight of
    // 0, one below 2^-126, stays 0: a large value of such a token counts for nothing.
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float rest[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = w[2 * c + e];
        rest[e] = __builtin_fmaxf(x - __uint_as_float(__float_as_uint(x) & 0xffff0000u),
                                 __builtin_fmaxf(x * 0x1p-17f, __builtin_fminf(x, 0x1p-133f)));
      }
      hi[c] = __builtin_amdgcn_perm(__float_as_uint(w[2 * c + 1]), __float_as_uint(w[2 * c]), 0x07060302u);
      lo[c] = pack_bf16x2(rest[0], rest[1]);
    }
    const bf16x8 wb = __builtin_bit_cast(bf16x8, attn_u32x4{hi[0], hi[1], hi[2], hi[3]});
    const bf16x8 wl = __builtin_bit_cast(bf16x8, attn_u32x4{lo[0], lo[1], lo[2], lo[3]});
#pragma unroll
    for (int d = 0; d < kDt; ++d) {
      const uint32_t sel = d & 1 ? 0x07060302u : 0x05040100u;  // the high or the low halves of two dwords
      attn_u32x4 x;
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = __builtin_amdgcn_perm(vd[2 * c + 1][d >> 1], vd[2 * c][d >> 1], sel);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), wb, o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), wl, o[d], 0, 0, 0);
    }
  };

  // Two tiles in turn: the next one is on its way while one is worked on (two on
  // their way: 32 of 2000 28.6 / 27.6 us, 256 of 1000 23.7 / 29.2).  The
  // loads stand outside of any branch, since a wait counts the loads behind it
  // and a branch would make that number the smaller one (a wave's last load is
  // its last tile again).
  auto have = [&](int i, int j) { return (paged >> (2 * (i & 31) + j) & 1) != 0; };
  if (mine > 0) {
    Regs ra, rb;
    load(0, ra);
    int i = 0;
    for (; i + 1 < mine; i += 2) {
      const bool a0 = have(i, 0), a1 = have(i, 1), b0 = have(i + 1, 0), b1 = have(i + 1, 1);
      if ((i & 31) == 0) next_pages = load_pages(i + 32);
      load(i + 1, rb);
      compute(i, a0, a1, ra);
      if ((i & 31) == 30 && i + 2 < mine) locate(i + 2, next_pages);
      load(min(i + 2, mine - 1), ra);
      compute(i + 1, b0, b1, rb);
    }
    if (i < mine) compute(i, have(i, 0), have(i, 1), ra);
  }

  // the wave's sum, then the waves'
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (lane == 0) s_any[wave] = any;
  if (n < nh) {
    if (g == 0) s_m[wave][n] = m, s_l[wave][n] = l;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int d = 0; d < kDt; d += 4)  // row 4 g + c of tile d is dim (4 g + c) D/16 + d
        *reinterpret_cast<f32x4*>(&s_o[wave][n][(4 * g + c) * kDt + d]) = f32x4{o[d][c], o[d + 1][c], o[d + 2][c], o[d + 3][c]};
  }
  __syncthreads();
  const float vs = kE4m3 && a.kv.v_scale ? a.kv.v_scale[kvh] : 1.0f;
  any = false;
#pragma unroll
  for (int w = 0; w < W; ++w) any |= s_any[w] != 0;
  for (int e = threadIdx.x; e < nh * (D / 4); e += 64 * W) {
    const int h = e / (D / 4), d = e % (D / 4) * 4, head = h0 + h;
    const bool last = p.chunks == 1;
    float top = last && a.sinks ? bf16_to_f32(a.sinks[head]) * kLog2e : kNegInf;
    const float sink = top;
#pragma unroll
    for (int w = 0; w < W; ++w) top = __builtin_fmaxf(top, s_m[w][h]);
    const float base = top == kNegInf ? 0.0f : top;
    float sum = last && a.sinks ? __builtin_amdgcn_exp2f(sink - base) : 0.0f;
    f32x4 acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_m[w][h] - base);
      sum += s_l[w][h] * f;
      const f32x4 x = *reinterpret_cast<const f32x4*>(&s_o[w][h][d]);
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c] = __builtin_fmaf(x[c], f, acc[c]);
    }
    if (last) {
      const float f = any ? vs / sum : 0.0f;
      uint32_t* to = reinterpret_cast<uint32_t*>(a.out + p.b * a.out_stride + static_cast<int64_t>(head) * D + d);
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c] = any ? acc[c] * f : 0.0f;
      *reinterpret_cast<attn_u32x2*>(to) = attn_u32x2{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
    } else {
      const int64_t at = static_cast<int64_t>(piece) * a.heads + head;
      *reinterpret_cast<f32x4*>(sp.part_o + at * D + d) = acc;
      if (d == 0) reinterpret_cast<f32x4*>(sp.part_ml)[at] = f32x4{top, sum, any ? 1.0f : 0.0f, 0.0f};
    }
  }
}

// A work-group has two waves, which leaves more of them to a CU and suits short and
// ragged sequences; four (or one) would be better for many long ones of the same
// length.  us with 2 and 4 waves: 64 ragged of up to 2000 18.3 / 19.8, of up to 8192
// 28.4 / 30.3, 256 of 1000 23.6 / 27.3, 64 of 4000 96.4 / 88.1, one of 131072 54 / 53;
// 185 of two tokens 9.2 / 12.6; 32 of 1000 15.1 / 15.5, and 22.8 with one.  Where the
// chip is not filled and nothing is cut it has four (one of 1000 11.4 / 10.1, of
// 500 7.9 / 7.5; 8 with a window of 128 4.6 / 4.8, so not for the shortest).
// Tiles of the smallest piece of a cut sequence (of 128 dims a tile has twice the
// work; us with 6 and 4: one of 1000 with 128 dims 10.7 / 9.4, 32 ragged of up to
// 1500 with 64 13.9 / 15.3).
int min_tiles(int head_dim) { return head_dim == 64 ? 6 : 4; }
// Work-groups from which on, one to a CU, sequences of up to 2 kWholeTiles whose
// mean is two thirds of the longest are not cut either (cut or whole, join
// included: 32 of 2000 31.6 / 28.4 us, 64 of 2000 56.2 / 53; 40 of 3000 55 / 65).
constexpr int kFull = 256;
// Where the table or the window holds no more than kWholeTiles (1024 tokens), or
// with 128 dims and few work-groups half of that, the call is one launch of a piece
// to each sequence.  us cut (where the table would hold more) and whole, in a graph:
//   64 dims: one of 1000 10.7 / 9.6, of 500 9.9 / 7.0; 64 of 1000 28.6 / 25.9; 16 of
//   1000 16.2 / 14.1, 8 of 1000 13.7 / 11.8, 8 ragged of up to 1000 10.5 / 11.0, 8 with
//   a window of 512 10 / 8; one of 1000 launched by the host 13.8 / 9.5
//   128 dims: 4 of 900 12 / 16.5; 8 of 500 10.5 / 12.4, launched by the host 13.7 /
//   12.4
constexpr int kMany = 128;

struct Cut {
  int slots;          // pieces aimed at for each tile of 16 heads; 0: none is cut
  int64_t max_slots;  // and their largest number
  int waves;          // of a work-group
};

// Work-groups aimed at: three for each CU with heads of 64 dims, two with 128.
// The registers hold twice as many, and one sequence of 131072 takes 58.0 us so
// against 54.8 (fewer partial sums, and a CU's loads are enough in flight).
Cut cut_of(int B, int64_t most_tiles, int tiles_of_heads, int head_dim) {
  const bool many = static_cast<int64_t>(B) * tiles_of_heads >= kMany;
  if (most_tiles <= (many || head_dim == 64 ? kWholeTiles : kWholeTiles / 2)) return Cut{0, B, !many && most_tiles > 8 ? 4 : 2};
  const int work_groups = head_dim == 64 ? 768 : 512;
  const int slots = (work_groups + tiles_of_heads - 1) / tiles_of_heads;
  // sum of max(1, (tiles + size / 2) / size) <= B + slots
  const int64_t pieces = static_cast<int64_t>(B) * ((most_tiles + min_tiles(head_dim) - 1) / min_tiles(head_dim));
  const int64_t most = static_cast<int64_t>(B) + slots;
  return Cut{slots, pieces < most ? pieces : most, 2};
}

// No more tiles than the longest sequence, or its window and first tokens, has.
int64_t most_tiles(const Reach& r) {
  const int64_t all = (r.tokens + kTile - 1) / kTile;
  return r.window == 0 ? all : min(all, (r.window + kTile - 2) / kTile + 1 + (r.first + kTile - 1) / kTile);
}

int tiles_of_heads(int heads, int kv_heads) { return kv_heads * ((heads / kv_heads + 15) / 16); }

}  // namespace

size_t decode_call_bytes(int B, int heads, int kv_heads, int head_dim, const Reach& r) {
  const Cut c = cut_of(B, most_tiles(r), tiles_of_heads(heads, kv_heads), head_dim);
  if (c.slots == 0) return 0;
  const size_t pieces = static_cast<size_t>(c.max_slots) * heads;
  return pieces * (head_dim + 4) * sizeof(float) + ((static_cast<size_t>(B) * 2 * sizeof(int) + 15) & ~size_t{15});
}

size_t decode_workspace_bytes(int B, int heads, int kv_heads, int head_dim) {
  return decode_call_bytes(B, heads, kv_heads, head_dim, Reach{kMaxTokens, 0, 0});
}

namespace {

// The sequences of `a`, cut as c says, in one launch and the join behind it.
hipError_t launch(const AttendArgs& a, const Cut& c, void* workspace, hipStream_t s) {
  const int th = tiles_of_heads(a.heads, a.kv.kv_heads);
  SplitArgs sp{};
  sp.slots = c.slots;
  sp.min_tiles = min_tiles(a.kv.head_dim);
  sp.whole_ok = static_cast<int64_t>(a.B) * th >= kFull;
  const size_t pieces = static_cast<size_t>(c.max_slots) * a.heads;
  sp.part_o = static_cast<float*>(workspace);
  sp.part_ml = sp.part_o + pieces * a.kv.head_dim;
  sp.plan = reinterpret_cast<int*>(sp.part_ml + pieces * 4);
  // Rows of neighbouring heads share a line: it is read once if one die's L2 serves
  // them (e4m3, 64 dims, token-major: 125 sequences of 1952 95 / 77 us, one of 74359
  // 35.7 / 28.1; rows of whole lines the same either way).
  sp.same_die = a.kv.sh * (a.kv.e4m3 ? 1 : 2) < 128;
  sp.max_slots = static_cast<int>(c.max_slots);
  const dim3 grid(static_cast<unsigned>((sp.same_die ? (c.max_slots + 7) / 8 * 8 : c.max_slots) * th));
#define GX_DECODE(D_, E_, W_) hipLaunchKernelGGL((decode_kernel<D_, E_, W_>), grid, dim3(64 * W_), 0, s, a, sp)
#define GX_DECODE_W(D_, E_)               \
  do {                                    \
    if (c.waves == 4) GX_DECODE(D_, E_, 4); \
    else GX_DECODE(D_, E_, 2);            \
  } while (0)
  if (a.kv.head_dim == 64) {
    if (a.kv.e4m3) GX_DECODE_W(64, true);
    else GX_DECODE_W(64, false);
  } else {
    if (a.kv.e4m3) GX_DECODE_W(128, true);
    else GX_DECODE_W(128, false);
  }
#undef GX_DECODE_W
#undef GX_DECODE
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || c.slots == 0) return e;
  JoinArgs j{};
  j.part_o = sp.part_o;
  j.part_ml = sp.part_ml;
  j.plan = sp.plan;
  j.max_pieces = static_cast<int>(c.max_slots);
  return launch_join(a, j, c.max_slots / a.B, s);
}

}  // namespace

hipError_t launch_decode(const AttendArgs& a, void* workspace, hipStream_t s) {
  const int th = tiles_of_heads(a.heads, a.kv.kv_heads);
  const int64_t most = most_tiles(reach_of(a));
  const Cut c = cut_of(a.B, most, th, a.kv.head_dim);
  if (c.slots == 0 || a.B <= kSearch) return launch(a, c, workspace, s);
  const int parts = (a.B + kSearch - 1) / kSearch, per = (a.B + parts - 1) / parts;
  for (int b = 0; b < a.B; b += per) {
    AttendArgs x = a;
    x.B = x.rows = min(per, a.B - b);
    x.q += b * a.q_stride;
    x.out += b * a.out_stride;
    x.tables += b * a.table_stride;
    x.lens += b;
    const hipError_t e = launch(x, cut_of(x.B, most, th, a.kv.head_dim), workspace, s);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace gxmoe
