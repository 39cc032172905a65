// attn_kernels.h -- arguments and host launchers of the attention kernels
// (internal): the position rotation with the append to the paged key-value
// cache, and attention of new tokens over that cache.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gxmoe {

// A paged cache: element (page, kv head, slot, dim) of K and of V lies at
// page * sb + head * sh + slot * st + dim.  Pages hold 1 << bs_shift slots.
struct KvPages {
  void* k;
  void* v;
  const float* k_scale;  // [kv_heads], e4m3 only; null = 1
  const float* v_scale;
  int64_t sb, sh, st;
  int num_blocks, bs_shift, kv_heads, head_dim;
  bool e4m3;
};

struct AppendArgs {
  const uint16_t* qkv;  // [T][(heads + 2 kv_heads) head_dim]
  int64_t qkv_stride;
  const int32_t* positions;  // [T]
  const int32_t* slots;      // [T], outside the cache: not stored
  const float* table;        // [max_positions][2][rotary / 2]
  int max_positions, rotary, interleaved;
  int T, heads;
  uint16_t* q_out;
  int64_t q_stride;
  KvPages kv;
};

struct AttendArgs {
  const uint16_t* q;  // [rows][heads head_dim]
  int64_t q_stride;
  uint16_t* out;
  int64_t out_stride;
  KvPages kv;
  const int32_t* tables;  // [B][table_stride], max_blocks entries used
  int64_t table_stride;
  int max_blocks;
  const int32_t* lens;     // [B], tokens of the sequence, the new ones included
  const int32_t* offsets;  // [B + 1] first row of each sequence; null: one row each
  int B, rows, heads;
  float scale_log2;  // scale * log2(e): softmax runs on powers of two
  int window, first;
  const uint16_t* sinks;  // [heads] or null
};

// Partial sums of rows that were cut into pieces.  Decode: piece c of row b is
// number plan[2 b] + c of plan[2 b + 1].  Prefill (offsets set): piece c of row r
// is number c * rows + r of plan[r].  One piece: the row is already written.
struct JoinArgs {
  const float* part_o;   // [piece][heads][head_dim] weighted sums
  const float* part_ml;  // [piece][heads][4] reference, sum, whether any token was seen
  const int* plan;
  int max_pieces;  // no row has more
};

struct RopeTableArgs {
  float* table;
  int rotary, max_positions;
  double theta, factor, original, beta_fast, beta_slow, concentration;
};

hipError_t launch_rope_table(const RopeTableArgs& a, hipStream_t s);
hipError_t launch_rope_append(const AppendArgs& a, hipStream_t s);
hipError_t launch_join(const AttendArgs& a, const JoinArgs& j, int64_t mean, hipStream_t s);  // mean: pieces of a row
constexpr int64_t kMaxTokens = 1 << 30;  // of a sequence

// Every work-group finds its part among the lengths of all sequences of its launch,
// in a time that grows with them.  Calls of more go in several launches (65536
// sequences of 8 heads in one and in eight: decode 19.1 / 3.2 ms, prefill 50.9 / 8.3).
constexpr int kSearch = 8192;

// What a sequence of a call can hold and a query of it see, as the host knows it.
struct Reach {
  int64_t tokens, window, first;  // window 0: all
};

inline Reach reach_of(const AttendArgs& a) {
  return Reach{static_cast<int64_t>(a.max_blocks) << a.kv.bs_shift, a.window, a.first};
}

// Bytes for one call, and for any of at most its counts.
size_t decode_call_bytes(int B, int heads, int kv_heads, int head_dim, const Reach& r);
size_t prefill_call_bytes(int rows, int B, int heads, int kv_heads, int head_dim, const Reach& r);
size_t decode_workspace_bytes(int B, int heads, int kv_heads, int head_dim);
hipError_t launch_decode(const AttendArgs& a, void* workspace, hipStream_t s);
size_t prefill_workspace_bytes(int rows, int heads, int kv_heads, int head_dim);
hipError_t launch_prefill(const AttendArgs& a, void* workspace, hipStream_t s);

}  // namespace gxmoe
