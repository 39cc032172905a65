/*
 * gptoss_moe.h -- C ABI of the MI355X (gfx950) GPT-OSS MoE block.
 *
 * Drop-in boundary for the MoE hot path of the reference engine
 * (Jayluci4/hip-kernels).  Every entry point takes plain pointers and sizes;
 * device pointers are HIP device memory of the current device, `stream` is
 * a hipStream_t (NULL = the null stream).  Every call returns a status code
 * (GPTOSS_OK = 0) and records a message readable with gptoss_last_error() on
 * the calling thread; nothing aborts the process (the reference aborts on
 * every HIP error, include/cuda_utils.h:17-35).
 *
 * Numerics: fp32 accumulation; bf16 rounding at the reference's points
 * (logits, gate_up, SwiGLU output, expert output, layer output); expert
 * indices chosen by (logit desc, index asc) as topk_softmax.cu:60-72.
 *
 * bf16 values are passed as uint16_t bit patterns.
 */
#ifndef GPTOSS_MOE_H
#define GPTOSS_MOE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GPTOSS_MOE_ABI_VERSION 7

enum {
  GPTOSS_OK = 0,
  GPTOSS_ERR_INVALID = 1,      /* bad argument (shape, null pointer, k > 8, ...) */
  GPTOSS_ERR_UNSUPPORTED = 2,  /* valid but not supported by this build (shape limits) */
  GPTOSS_ERR_HIP = 3,          /* a HIP runtime call failed */
  GPTOSS_ERR_STATE = 4,        /* object not initialised / already initialised */
  GPTOSS_ERR_OOM = 5,          /* device allocation failed */
  GPTOSS_ERR_NOT_FOUND = 6,    /* checkpoint tensor or shard file not found */
  GPTOSS_ERR_IO = 7            /* checkpoint file unreadable or not valid safetensors */
};

/* Message of the last failing call on this thread ("" if none); UTF-8, with
 * any byte of a quoted name or path that is not well-formed UTF-8 as '?'. */
const char* gptoss_last_error(void);
int gptoss_abi_version(void);

/* MoE shape and constants.  Replaces the compile-time ModelConfig MoE fields
 * (include/config.h:20-23, 40-43, 53, 57): E and k are runtime values here, so
 * the 20B (E=32) and 120B (E=128) shapes run from one library. */
typedef struct gptoss_moe_config {
  int hidden_size;        /* H (2880) */
  int num_experts;        /* E (128 for 120B, 32 for 20B) */
  int top_k;              /* k (4); 1, 2, 4 or 8 */
  int intermediate_size;  /* I (2880); gate_up rows = 2I, interleaved gate/up */
  float swiglu_alpha;     /* 1.702 (config.h:43) */
  float swiglu_limit;     /* 7.0   (config.h:42) */
  float rms_norm_eps;     /* 1e-5  (config.h:39), used by forward() only */
  int logits_fp32;        /* 0: bf16 router logits (reference), 1: fp32 logits */
  int max_tokens;         /* largest T a forward call may pass (scratch sizing) */
  /* Forwards of at least this many tokens run the expert products as grouped
   * GEMMs on the matrix cores (fp32 accumulation in the matrix core's order:
   * within one bf16 rounding step of the canonical result, not bit-identical).
   * 0 = never.  Default 128. */
  int prefill_min_tokens;
  /* Smaller forwards (decode) stream the expert weights once per step.
   * 0 (default): on the matrix cores, fp32 accumulation in the matrix core's
   * order (like prefill).  1: through the exact VALU kernels, whose results
   * are bit-identical to the canonical order (one ascending fma chain per
   * K-part, parts added in order), at a lower streaming rate.  The
   * matrix-core decode kernels take at most 1024 slots (T * top_k); larger
   * forwards below prefill_min_tokens (only when it is 0 or above 256 at
   * top-4) run the exact kernels, about 5 ms for 1024 GPT-OSS-120B tokens
   * against 0.47 ms on the prefill path. */
  int decode_exact;
  /* Prefill expert products (T >= prefill_min_tokens).  0 (default): the
   * bf16 matrix core with the weights decoded in registers; fp32 accumulation.
   * 1: the block-scaled matrix core (v_mfma_scale_f32_16x16x128_f8f6f4): the
   * fp4 weights with their e8m0 scales as stored, times the activations split
   * into two e4m3 parts per 32-element block (hi + lo/32, exact for every
   * value above 2^-13 of its block's largest), two products each.  2: the
   * same with the hi part alone (each activation rounded to four significant
   * bits).  The block-scaled product sums inside each instruction at less
   * than fp32 precision, so 1 and 2 fall outside the north-star tolerance at
   * GPT-OSS-120B's K = 2880, and on gfx950 neither is faster than 0: they
   * are kept as measured alternatives, not as the default. */
  int prefill_block_scaled;
} gptoss_moe_config;

/* Fill `cfg` with the GPT-OSS constants for `num_experts` experts. */
int gptoss_moe_config_default(gptoss_moe_config* cfg, int num_experts, int max_tokens);

/* ---- MXFP4 weight layout (src/memory) ----------------------------------
 * Reference layout of one expert matrix [N rows, K inputs]
 * (weight_loader.cu:782-842, fused_mxfp4_gemv.cu:13-15): packed [N][K/2]
 * bytes, low nibble = even k; scales [N][K/32] e8m0 bytes.
 * The kernels read a tiled layout: per 64-row tile, K/32 blocks of one KiB
 * holding the 64 rows' 16-byte blocks as dwords ordered for the matrix
 * cores (slot 16g + r%16, dword r/16 = bytes 4g..4g+3 of row r); scales
 * twice, per (tile, K-part, row) and per (tile, block) in slot order. */
int gptoss_mxfp4_tiled_size(int N, int K, size_t* nibble_bytes, size_t* scale_bytes);
int gptoss_mxfp4_pack_tiled(const uint8_t* packed, const uint8_t* scales, int N, int K,
                            uint8_t* tiled_nibbles, uint8_t* tiled_scales, void* stream);

/* ---- Layer object: replaces gptoss::MoELayer and moe_layer_* -------------
 * (src/model/moe_layer.cu:1556-1615). */
typedef struct gptoss_moe_layer gptoss_moe_layer;

typedef struct gptoss_moe_weights {
  const uint16_t* moe_norm_weight;  /* [H] bf16, used by forward() (may be NULL otherwise) */
  const uint16_t* router_weight;    /* [E][H] bf16 (mlp.router.weight) */
  const uint16_t* router_bias;      /* [E] bf16 or NULL */
  const uint16_t* gate_up_bias;     /* [E][2I] bf16 or NULL */
  const uint16_t* down_bias;        /* [E][H] bf16 or NULL */
  /* Either: reference-layout experts, host arrays of E device pointers
   * (MXFP4Weight tables of moe_layer.cu:585-589); the layer packs them into
   * its own tiled copy at init. */
  const uint8_t* const* mlp1_packed;  /* [E] -> [2I][H/2] */
  const uint8_t* const* mlp1_scales;  /* [E] -> [2I][H/32] */
  const uint8_t* const* mlp2_packed;  /* [E] -> [H][I/2] */
  const uint8_t* const* mlp2_scales;  /* [E] -> [H][I/32] */
  /* Or: already tiled, expert-major contiguous buffers (borrowed, not copied):
   * E x gptoss_mxfp4_tiled_size(2I, H) and E x gptoss_mxfp4_tiled_size(H, I). */
  const uint8_t* mlp1_tiled_nibbles;
  const uint8_t* mlp1_tiled_scales;
  const uint8_t* mlp2_tiled_nibbles;
  const uint8_t* mlp2_tiled_scales;
} gptoss_moe_weights;

gptoss_moe_layer* gptoss_moe_layer_create(void);                    /* moe_layer_create */
/* moe_layer_init: the layer allocates its per-forward scratch for
 * cfg->max_tokens tokens (gptoss_moe_layer_workspace_bytes bytes). */
int gptoss_moe_layer_init(gptoss_moe_layer* layer, const gptoss_moe_config* cfg, int device_id,
                          const gptoss_moe_weights* weights);       /* moe_layer_init */
/* Bytes of per-forward scratch (routing plan, SwiGLU activations, expert
 * outputs, norm output) of a layer of this config, sized for
 * cfg->max_tokens; 0 for an invalid config. */
size_t gptoss_moe_layer_workspace_bytes(const gptoss_moe_config* cfg);
/* moe_layer_init with the per-forward scratch in a caller-owned device buffer
 * of device_id (at least gptoss_moe_layer_workspace_bytes(cfg) bytes,
 * 256-byte aligned), as the reference engine hands every layer the same
 * scratch buffers (engine.cu:975-1000, moe_layer.cu:1585-1600).  Layers whose
 * forwards are ordered on one stream may share one workspace, whatever their
 * configs (each needs the bytes of its own); forwards that can overlap in time
 * need separate workspaces.  The first 1152 bytes hold a work queue that must
 * read zero whenever no forward is running: init zeroes it (after waiting for
 * all work already queued on the device, so a forward in flight on another
 * stream is not disturbed) and every forward leaves it zero, so nothing else
 * may write there; a forward enqueued on it by another host thread while an
 * init runs races with that zeroing.  The workspace must
 * outlive the layer; a trace (gptoss_moe_layer_trace) then shows the last
 * forward of any layer on it. */
int gptoss_moe_layer_init_with_workspace(gptoss_moe_layer* layer, const gptoss_moe_config* cfg, int device_id,
                                         const gptoss_moe_weights* weights, void* workspace,
                                         size_t workspace_bytes);
/* out = input + MoE(RMSNorm(input))  (moe_layer_forward, moe_layer.cu:982-1005) */
int gptoss_moe_layer_forward(gptoss_moe_layer* layer, const uint16_t* input, uint16_t* output,
                             int num_tokens, void* stream);
/* The decode step's residual add + RMSNorm and the MoE in one call: it
 * replaces fused_residual_rmsnorm_forward(residual, delta, moe_norm_weight,
 * normed, sum) followed by moe_layer_forward_prenormed(normed, sum, out)
 * (transformer.cu:696-715, rmsnorm.cu:224-337).  sum = residual + delta is
 * formed in fp32; residual_out (may be NULL) receives bf16(sum); out =
 * bf16(sum) + MoE(RMSNorm(sum)).  Up to 4 tokens the norm runs inside the
 * router's launch (one launch fewer), above in a launch of its own.  Needs
 * moe_norm_weight.  residual_out must not overlap residual or delta (the
 * reference double-buffers the residual stream, transformer.cu:697-701;
 * GPTOSS_ERR_INVALID otherwise); out may equal residual, residual_out or
 * neither, but must not partially overlap residual_out. */
int gptoss_moe_layer_forward_residual(gptoss_moe_layer* layer, const uint16_t* residual,
                                      const uint16_t* delta, uint16_t* residual_out, uint16_t* output,
                                      int num_tokens, void* stream);
/* out = residual + MoE(normed)  (moe_layer_forward_prenormed, moe_layer.cu:960-980);
 * residual may be NULL (out = MoE(normed)). */
int gptoss_moe_layer_forward_prenormed(gptoss_moe_layer* layer, const uint16_t* normed,
                                       const uint16_t* residual, uint16_t* output,
                                       int num_tokens, void* stream);
/* The layer's expert half with the routing given: out = residual +
 * sum_k w[t,k] * FFN_{idx[t,k]}(normed[t]).  This is forward_core's
 * permute / experts / combine (moe_layer.cu:1196-1549) entered after its
 * single-GPU top-k (moe_layer.cu:1188), for callers that route elsewhere (or inject a routing, as prefill
 * benchmarks with skewed expert popularity do).  Indices must lie in
 * [0, num_experts) and be distinct per token; weights are used as given. */
int gptoss_moe_layer_forward_routed(gptoss_moe_layer* layer, const uint16_t* normed,
                                    const uint16_t* residual, const int32_t* expert_indices,
                                    const float* expert_weights, uint16_t* output, int num_tokens,
                                    void* stream);
/* forward_prenormed with no allocation and no use of the layer's own scratch:
 * no counterpart in the reference.  For callers that cannot allocate device
 * memory (code under hipGraph capture, tight serving loops, harnesses that
 * forbid hipMalloc): the forward scratch is a static device array of 8 MiB
 * that the library holds on every GPU it runs on until the process ends, so
 * num_tokens is limited to 64 and to configs whose scratch fits (the
 * GPT-OSS-120B layer at 64 tokens takes about 3.7 MiB); larger calls return
 * GPTOSS_ERR_INVALID.  The layer's max_tokens does not bound it.  Calls on one
 * GPU share that array: calls that overlap in time on one GPU (other streams,
 * other threads) race, and the layer's trace does not show these calls.
 * Results are those of gptoss_moe_layer_forward_prenormed. */
int gptoss_moe_layer_forward_prenormed_noalloc(gptoss_moe_layer* layer, const uint16_t* normed,
                                               const uint16_t* residual, uint16_t* output, int num_tokens,
                                               void* stream);
const uint16_t* gptoss_moe_layer_get_ffn_norm_weight(const gptoss_moe_layer* layer);
/* The config and device the layer was initialised with. */
int gptoss_moe_layer_get_config(const gptoss_moe_layer* layer, gptoss_moe_config* cfg, int* device_id);
void gptoss_moe_layer_destroy(gptoss_moe_layer* layer);           /* moe_layer_destroy */

/* ---- Checkpoints (src/memory/weight_loader.cu) ---------------------------
 * A safetensors checkpoint: every `*.safetensors` file of a directory in
 * name order (weight_loader.cu:456-482), or one file, mapped read-only
 * (:488-537).  The index maps names to tensors; a name present in several
 * shards resolves to the last shard in name order (:546-555). */
typedef struct gptoss_checkpoint gptoss_checkpoint;

typedef struct gptoss_tensor_info {
  const char* name;   /* valid while the checkpoint is open */
  const char* dtype;  /* as in the header: "BF16", "F32", "U8", ... */
  int ndim;           /* at most 8 */
  int64_t shape[8];
  uint64_t nbytes;    /* data_offsets end - begin */
  const void* data;   /* host address inside the read-only mapping */
  int shard;          /* shard index in name order */
} gptoss_tensor_info;

/* WeightLoader::init's shard scan, mmap and header parse
 * (weight_loader.cu:297-345, 456-540).  Malformed files return
 * GPTOSS_ERR_IO instead of aborting. */
int gptoss_checkpoint_open(const char* path, gptoss_checkpoint** out);
void gptoss_checkpoint_close(gptoss_checkpoint* ckpt);              /* WeightLoader::destroy */
int gptoss_checkpoint_num_tensors(const gptoss_checkpoint* ckpt);
int gptoss_checkpoint_tensor_at(const gptoss_checkpoint* ckpt, int i, gptoss_tensor_info* info);
/* has_tensor / get_tensor_data (weight_loader.cu:556-575): GPTOSS_ERR_NOT_FOUND
 * when absent. */
int gptoss_checkpoint_find(const gptoss_checkpoint* ckpt, const char* name, gptoss_tensor_info* info);
/* Size of each of the two pinned host and two device staging slots that
 * gptoss_moe_layer_init_from_checkpoint streams experts through (default
 * 32 MiB; a slot always holds at least one expert matrix).  The checkpoint
 * keeps the staging of each device it has loaded a layer onto until it is
 * closed, so the layers of a model reuse one pinned allocation. */
int gptoss_checkpoint_set_staging_bytes(gptoss_checkpoint* ckpt, size_t bytes);

/* One MoE layer from a checkpoint: WeightLoader::load_layer_weights' MoE part
 * (weight_loader.cu:1083-1165) with load_packed_experts (:818-842) or
 * load_per_expert_weights (:847-895), then moe_layer_init.  Names under
 * "model.layers.<layer_index>.": mlp.gate|router.{weight,bias},
 * post_attention_layernorm.weight, mlp.experts.{gate_up,down}_proj_{blocks,
 * scales,bias} or mlp.experts.<e>.{mlp1|gate_up_proj|w1, mlp2|down_proj|w2}
 * .weight[_scale].  bf16 tensors stored as F32 or F16 are rounded to bf16
 * (nearest even).  The layer owns one device allocation holding every
 * weight, the experts already tiled; names, shapes and dtypes are checked
 * against cfg before any device work.  Loads from one checkpoint run one at
 * a time (they share its staging). */
int gptoss_moe_layer_init_from_checkpoint(gptoss_moe_layer* layer, const gptoss_moe_config* cfg,
                                          int device_id, const gptoss_checkpoint* ckpt, int layer_index);

/* ---- Layer stack: the MoE half of the engine's decode step ----------------
 * The engine's decode step (transformer.cu:653-753) runs, per layer,
 * attention (a delta), fused_residual_rmsnorm_forward and
 * moe_layer_forward_prenormed, and is never graph-captured because the
 * reference MoE synchronises the host (engine.cu:309-320).  A stack runs the
 * same per-layer sequence over its layers, in place on a residual buffer it
 * owns:
 *     hook(layer, residual, delta[layer])            (optional: attention)
 *     residual = bf16(residual + delta[layer]) + MoE_layer(RMSNorm(...))
 * and, since nothing in it synchronises the host, can capture the whole step
 * in one hipGraph per token count, kept and replayed by later steps. */
typedef struct gptoss_moe_stack gptoss_moe_stack;

/* Writes layer `layer`'s delta [T][H] from the current residual [T][H] with
 * launches on `stream` (the engine's attention).  With graph replay the hook
 * runs once, while its step is captured: its launches are replayed as
 * captured, so they must not synchronise the host or change pointers. */
typedef void (*gptoss_layer_hook)(void* user, int layer, const uint16_t* residual, uint16_t* delta,
                                  int num_tokens, void* stream);

/* num_layers layers from first_layer on, each loaded as
 * gptoss_moe_layer_init_from_checkpoint does (needs
 * post_attention_layernorm.weight). */
int gptoss_moe_stack_create(const gptoss_moe_config* cfg, int device_id, const gptoss_checkpoint* ckpt,
                            int first_layer, int num_layers, gptoss_moe_stack** out);
/* Over initialised layers (borrowed; one device, one shape, each with
 * moe_norm_weight). */
int gptoss_moe_stack_create_from_layers(gptoss_moe_layer* const* layers, int num_layers,
                                        gptoss_moe_stack** out);
/* The stack's device buffers: residual [max_tokens][H] and deltas
 * [num_layers][max_tokens][H], bf16.  Any output may be NULL. */
int gptoss_moe_stack_io(gptoss_moe_stack* stack, uint16_t** residual, uint16_t** deltas, int* max_tokens,
                        int* num_layers);
/* Step on caller-owned buffers of the same shapes instead (NULL: back to the
 * stack's own); waits for the device, then drops the captured graphs, which
 * hold the old pointers. */
int gptoss_moe_stack_bind(gptoss_moe_stack* stack, uint16_t* residual, uint16_t* deltas);
int gptoss_moe_stack_layer(gptoss_moe_stack* stack, int index, gptoss_moe_layer** layer);
/* One step over every layer, ordered on `stream`.  use_graph = 1: replay
 * the step's graph for num_tokens (captured on first use, and again when
 * hook or user change). */
int gptoss_moe_stack_decode_step(gptoss_moe_stack* stack, int num_tokens, gptoss_layer_hook hook, void* user,
                                 int use_graph, void* stream);
void gptoss_moe_stack_destroy(gptoss_moe_stack* stack);

/* Device views of the layer's scratch after the last forward on `stream`
 * (valid until the next forward): routing and per-slot intermediates in the
 * permuted (expert-sorted) order.  Any output pointer may be NULL. */
typedef struct gptoss_moe_trace {
  const void* logits;         /* [T][E] bf16 or fp32 (cfg.logits_fp32) */
  const int32_t* expert_indices;  /* [T][k] */
  const float* expert_weights;    /* [T][k] */
  const int32_t* expert_counts;   /* [E] */
  const int32_t* expert_offsets;  /* [E+1] */
  const int32_t* gather_map;      /* [T*k] slot -> permuted row, -1 if dropped */
  const int32_t* perm_token;      /* [T*k] permuted row -> token */
  const int32_t* active_experts;  /* [E] ascending, first n_active valid */
  const int32_t* n_active;        /* [1] */
  const uint16_t* gate_up;        /* [T*k][2I] bf16 (only if trace_gate_up was enabled) */
  const uint16_t* act;            /* [T*k][I] bf16 SwiGLU output */
  const uint16_t* expert_out;     /* [T*k][H] bf16 */
} gptoss_moe_trace;
int gptoss_moe_layer_trace(const gptoss_moe_layer* layer, gptoss_moe_trace* trace);
/* Also write the bf16 gate_up intermediate on the next forwards (debug). */
int gptoss_moe_layer_set_trace_gate_up(gptoss_moe_layer* layer, int enable);

/* Per-launch timing, the role of the reference's PROF regions
 * (include/profiler.h:20-30, src/engine/profiler.cu:106-360): with
 * max_forwards > 0 the next max_forwards forwards time their route (or plan,
 * for forward_routed), gate_up (W1), down (W2) and combine launches with HIP
 * events stamped by each dispatch itself (hipExtLaunchKernelGGL: the
 * kernel's execution alone).  Forwards captured into a hipGraph are not
 * timed and use no slot.  profile_read waits for the events and returns the
 * summed milliseconds per launch and the count of recorded forwards (any
 * output pointer may be NULL).  Calling set_profiling again re-arms;
 * max_forwards = 0 turns recording off. */
int gptoss_moe_layer_set_profiling(gptoss_moe_layer* layer, int max_forwards);
int gptoss_moe_layer_profile_read(gptoss_moe_layer* layer, float* route_ms, float* w1_ms,
                                  float* w2_ms, float* combine_ms, int* n_forwards);
/* One recorded forward, for per-launch traces and summaries (the records
 * behind the reference's profiler_save_chrome_trace / _summary_json,
 * src/engine/profiler.cu:215-360): host_us is the host steady-clock time
 * (microseconds) at which the forward was enqueued; launch i (0 route, or the
 * plan for forward_routed; 1 gate_up; 2 down; 3 combine) started start_ms[i]
 * after launch 0 and ran dur_ms[i]. */
typedef struct gptoss_moe_prof_record {
  double host_us;
  int num_tokens;
  int prefill;       /* 1: the grouped prefill kernels ran (num_tokens >= prefill_min_tokens) */
  float start_ms[4];
  float dur_ms[4];
} gptoss_moe_prof_record;
/* Waits for the events of the first min(capacity, recorded) forwards since the
 * last set_profiling and writes their records; *n_records (may be NULL) gets
 * the number recorded. */
int gptoss_moe_layer_profile_records(gptoss_moe_layer* layer, gptoss_moe_prof_record* records,
                                     int capacity, int* n_records);

/* ---- Stage entry points (the reference's kernel launchers) --------------- */

/* Router + top-k softmax: replaces gemv_bf16_forward (T == 1,
 * gemv_bf16.cu:236-247) / gemm_bf16_lt (T > 1, cuda_utils.h:226-308) plus
 * topk_softmax_forward (topk_softmax.cu:380).  logits: [T][E] bf16 if
 * logits_fp32 == 0 else fp32 (the router output, rounded as the reference's
 * bf16 logits or kept in fp32).  `scratch` is reserved: it must be non-NULL
 * (gptoss_moe_route_scratch_bytes bytes of device memory, 256 today) and is
 * neither read nor written; routing exchanges no values between
 * work-groups, so no workspace is needed.
 * Up to 64 tokens every logit follows the reference's gemv_bf16 tree (its
 * T = 1 path, gemv_bf16.cu:57-129), bit-exact against the oracle.  Above 64
 * (when hidden % 32 == 0) the logits come from the matrix cores: fp32 sums of
 * exact bf16 products, four chains per logit (32-element blocks j, j + 4, ...
 * in block order), added pairwise, then the bias, as the reference's
 * hipBLASLt path for T > 1 sums in its own order; within the fp32 error bound
 * of the exact sum, deterministic, and independent of the other tokens in the
 * call.  router_b may be NULL (zero bias).  Logits need no alignment beyond
 * their element size. */
size_t gptoss_moe_route_scratch_bytes(int num_tokens, int num_experts, int top_k);
int gptoss_moe_route(const uint16_t* x, const uint16_t* router_w, const uint16_t* router_b,
                     int num_tokens, int num_experts, int hidden, int top_k, int logits_fp32,
                     void* logits, int32_t* expert_indices, float* expert_weights,
                     void* scratch, void* stream);

/* topk_softmax_forward (topk_softmax.cu:380-432) on given logits; bf16 logits
 * unless logits_fp32.  tokens_per_expert may be NULL (atomic histogram). */
int gptoss_topk_softmax_forward(const void* logits, int logits_fp32, int32_t* expert_indices,
                                float* expert_weights, int32_t* tokens_per_expert,
                                int num_tokens, int num_experts, int top_k, void* stream);

/* moe_permute_classify + moe_compute_gather_map_cpu (moe_permute.cu:129-236)
 * on the device: per-expert counts, offsets[E+1], stable gather map,
 * permuted token list, active expert list and its length. */
int gptoss_moe_permute_plan(const int32_t* expert_indices, int num_tokens, int top_k,
                            int num_experts, int32_t* counts, int32_t* offsets,
                            int32_t* gather_map, int32_t* perm_token, int32_t* active_experts,
                            int32_t* n_active, void* stream);

/* moe_scatter_tokens (moe_permute.cu:241-259): permuted[gather_map[s]] = x[s/k]. */
int gptoss_moe_scatter_tokens(const uint16_t* x, const int32_t* gather_map, uint16_t* permuted,
                              int num_tokens, int hidden, int top_k, void* stream);

/* fused_mxfp4_gemv_forward (fused_mxfp4_gemv.cu:452-464) generalised to M rows:
 * y[m][n] = bf16(sum_k x[m][k] * W[n][k] + bias[n]) with W in the tiled layout. */
int gptoss_mxfp4_gemv_forward(const uint16_t* x, int M, const uint8_t* tiled_nibbles,
                              const uint8_t* tiled_scales, const uint16_t* bias, uint16_t* y,
                              int N, int K, void* stream);

/* fused_residual_rmsnorm_forward (rmsnorm.cu:224-337): s = residual + delta
 * (fp32), sum_out = bf16(s) (may be NULL), normed = bf16((s * inv) * weight)
 * with inv = 1/sqrt(mean(s^2) + eps); the sum of squares follows the
 * router's gemv_bf16 tree and sqrt / divide are IEEE (the reference uses
 * rsqrtf). */
int gptoss_fused_residual_rmsnorm_forward(const uint16_t* residual, const uint16_t* delta,
                                          const uint16_t* weight, uint16_t* normed, uint16_t* sum_out,
                                          int num_tokens, int hidden, float eps, void* stream);

/* swiglu_forward (swiglu.cu:178-211): interleaved [T][2I] -> [T][I]. */
int gptoss_swiglu_forward(const uint16_t* gate_up, uint16_t* out, int num_tokens,
                          int intermediate, float alpha, float limit, void* stream);

/* moe_combine_forward (moe_combine.cu:175-204), single GPU (no remote rows):
 * out[t] = bf16(sum_k w[t,k] * expert_out[gather_map[t,k]] + residual[t]). */
int gptoss_moe_combine_forward(uint16_t* out, const uint16_t* expert_out,
                               const int32_t* gather_map, const float* expert_weights,
                               const uint16_t* residual, int num_tokens, int hidden,
                               int top_k, void* stream);

/* The prefill expert products: per active expert, mxfp4_dequant_batched
 * (mxfp4_dequant.cu:353-375) + CublasHandle::gemm_bf16_lt (cuda_utils.h:
 * 226-308) + bias_add_rows (moe_layer.cu:171-194) [+ swiglu_forward] as issued
 * by moe_layer.cu:1389-1487, in one grouped launch on the matrix cores:
 *   y[p][n] = bf16(sum_k x[row(p)][k] * W_e[n][k] + bias[e][n])
 * for every expert e and permuted row p in [offsets[e], offsets[e+1]), with
 * row(p) = row_index[p] (a gather from token rows, e.g. the plan's
 * perm_token) or p when row_index is NULL.  W_e is expert e of an
 * expert-major tiled array (E x gptoss_mxfp4_tiled_size(N, K)).
 * swiglu == 0: out[p][n] = y[p][n] ([rows][N]).  swiglu != 0: out[p][i] =
 * bf16(SwiGLU(y[p][2i], y[p][2i+1])) ([rows][N/2], interleaved gate/up rows),
 * and gate_up (may be NULL) receives y.  offsets (device, [E+1]) must be
 * nondecreasing from 0 with offsets[E] <= rows.  fp32 accumulation in the
 * matrix core's order (see prefill_min_tokens). */
int gptoss_moe_grouped_mxfp4_gemm(const uint16_t* x, const int32_t* row_index,
                                  const int32_t* expert_offsets, int num_experts, int rows,
                                  const uint8_t* tiled_nibbles, const uint8_t* tiled_scales,
                                  const uint16_t* bias, int N, int K, int swiglu, float alpha,
                                  float limit, uint16_t* out, uint16_t* gate_up, void* stream);

/* mxfp4_dequant_batched (mxfp4_dequant.cu:353-375) for one tiled matrix:
 * out[n][k] = bf16(e2m1 * 2^(scale-127)), row-major [N][K]. */
int gptoss_mxfp4_dequant(const uint8_t* tiled_nibbles, const uint8_t* tiled_scales, int N, int K,
                         uint16_t* out, void* stream);

/* ---- Attention over a paged key-value cache ------------------------------
 * The attention half of a layer (src/model/attention.cu:635-959) between its
 * two projections.  A decode step calls, on the rows of the QKV projection, gptoss_rope_kv_append and then
 * gptoss_paged_attention_decode; a prompt chunk the same with
 * gptoss_paged_attention_prefill.  None of these calls synchronises the host or
 * allocates, so a layer hook (gptoss_moe_stack_decode_step) may capture them;
 * lengths, positions, slots and page tables are read on the device, so a
 * replayed graph follows the values that those buffers hold then.
 * These entry points are additions: the ABI version stays. */

enum { GPTOSS_KV_BF16 = 0, GPTOSS_KV_E4M3 = 1 };

/* Where the cache lies.  Element (page, kv head, slot, dim) of K is at
 * page * block_stride + head * head_stride + slot * token_stride + dim
 * elements from k, and of V from v.  All three strides 0: the reference's
 * [num_blocks][kv_heads][block_size][head_dim] without gaps.  Strides are
 * multiples of 16 bytes and at least head_dim, k and v are 16-byte aligned, so
 * token-major pages and K / V interleaved by page are covered.  head_dim is 64
 * or 128, block_size a power of two from 16 to 256.  E4M3 (OCP, gfx950's own)
 * elements stand for code * scale[kv head], scales positive; a null scale is 1,
 * and bf16 caches have none. */
typedef struct gptoss_kv_cache {
  void* k;
  void* v;
  const float* k_scale;  /* device [num_kv_heads] or NULL */
  const float* v_scale;
  int64_t block_stride, head_stride, token_stride; /* elements */
  int dtype;             /* GPTOSS_KV_BF16 or GPTOSS_KV_E4M3 */
  int num_blocks, block_size, num_kv_heads, head_dim;
} gptoss_kv_cache;

/* YaRN rotary positions (rope.cu:42-512): rotary_dim dims of a head turn, dim
 * pair i at frequency theta^(-2i/rotary_dim), or that over scaling_factor
 * where it turns less than beta_slow times within original_positions, with a
 * linear ramp from the dims that turn beta_fast times.  cos and sin carry the
 * concentration 0.1 ln(scaling_factor) + 1.  scaling_factor 1: plain rotary
 * positions. */
typedef struct gptoss_rope_config {
  int rotary_dim;      /* a positive multiple of 16 */
  int max_positions;
  double theta;        /* > 1 */
  double scaling_factor; /* >= 1 */
  double original_positions, beta_fast, beta_slow; /* > 0, original_positions / beta_fast too; unused at factor 1 */
} gptoss_rope_config;

/* GPT-OSS: rotary_dim 64, 131072 positions, theta 150000, factor 32 over 4096,
 * beta 32 / 1 (include/config.h:29-36). */
int gptoss_rope_config_default(gptoss_rope_config* cfg);

/* table: [max_positions][2][rotary_dim / 2] fp32, the cosines of a position and
 * then its sines; angles are formed in 64 bits. */
int gptoss_rope_table(const gptoss_rope_config* cfg, float* table, void* stream);

/* Position rotation, and the append to the cache (the reference's pieces of it:
 * attention.cu:105-380, kv_cache_manager.cu:32).  Row t of qkv holds the
 * num_heads queries, the kv heads' keys and their values, head_dim each, rows
 * qkv_stride elements apart (a multiple of 8).  Queries and keys are turned by
 * positions[t] (pair i is dims i and i + rotary_dim / 2, or 2i and 2i + 1 if
 * interleaved != 0; dims from rotary_dim on are kept): products and their sum
 * are fp32 operations, rounded once.  Queries go to q_out as bf16 (rows q_stride
 * apart, a multiple of 8); keys and values to slot slots[t] = page *
 * block_size + place of the cache, as bf16 or as e4m3 of value / scale, those
 * past +-448 as +-448.  A row whose slot is not in the cache (as -1) stores no
 * key or value; one whose position is not in the table [0, max_positions)
 * writes nothing at all.  Slots of one call are distinct: of rows that share
 * one, any may be found there, in pieces.  q_out may be the queries' place in
 * qkv (same pointer and stride) and otherwise lies apart from qkv (or its rows
 * between qkv's, at the same stride); both lie
 * outside of what the cache's pages span.
 * qkv, q_out and rope_table are 16-byte aligned; rotary_dim <= head_dim;
 * num_tokens is at most 2^25. */
int gptoss_rope_kv_append(const uint16_t* qkv, int64_t qkv_stride, const int32_t* positions,
                          const int32_t* slots, const float* rope_table, int rotary_dim, int max_positions,
                          int interleaved, int num_tokens, int num_heads, uint16_t* q_out, int64_t q_stride,
                          const gptoss_kv_cache* cache, void* stream);

/* What a query at position p sees: the tokens t <= p, and with window > 0 of
 * those only the last `window` (its own among them) and the first
 * first_tokens of the sequence.  sinks (device bf16 [num_heads], may be NULL)
 * adds exp(sinks[head]) to the softmax's sum, as a token without a value.  A
 * query that sees nothing gives zeros. */
typedef struct gptoss_attention_config {
  float scale;       /* of the scores; > 0, below 2.3e38 */
  int window;        /* 0: no window */
  int first_tokens;
  const uint16_t* sinks;
} gptoss_attention_config;

/* Sequence b's token t lies in page block_tables[b * table_stride +
 * t / block_size] at place t % block_size.  Tokens of a page number outside
 * [0, num_blocks) (as -1 for a page given back once it left the window) are not
 * seen.  seq_lens[b] counts the tokens in the cache, the new ones included;
 * negative ones are 0, and those past max_blocks pages are cut to that.  What
 * pages hold past a sequence's end, or outside of what is seen, has no effect,
 * NaN included.
 *
 * Decode (the reference's: paged_attention.cu:112-717): one new token per
 * sequence, at position seq_lens[b] - 1; q and out are [num_seqs][num_heads *
 * head_dim] bf16, rows q_stride and out_stride elements apart (multiples of
 * 8), apart from each other (rows of one may lie between the other's, at the
 * same stride), 16-byte aligned; out lies outside of what the
 * cache's pages span.  num_heads is a multiple of the
 * kv heads, at most 128 per kv head.  Scores and sums are fp32; the softmax's
 * weights meet the values with 16 significant bits here and rounded to bf16 in
 * the prefill call; one below 2^-126 of the largest is 0.  Values are summed
 * before the division, weights reaching 2^12: bf16 values whose magnitude times
 * the number of tokens is past 2^115 may give infinities.
 * workspace: gptoss_paged_attention_workspace_bytes bytes, 16-byte aligned,
 * that no call running at the same time uses (two graphs that may overlap need
 * two); nothing is kept in it between calls.  The bytes for num_tokens rows and
 * num_seqs sequences are enough for calls of fewer, whatever their lengths (rows
 * of any call: a decode call has num_seqs of them, and 0 rows need 0 bytes).
 * What one call needs is less, and 0 where nothing is split (workspace may be NULL
 * then): gptoss_paged_attention_call_bytes, with max_tokens = max_blocks *
 * block_size and num_tokens = 0 for decode.
 * The host knows of the lengths only that they fit into max_blocks pages, and
 * cuts sequences into pieces (a second launch joins these) where that many tokens
 * would want it.  Tables no wider than the longest sequence needs are faster for
 * short ones: one token over 1000 9.6 us, with a table of 131072 10.7; a prompt of
 * 680 17 and 27.
 * Limits of a call (GPTOSS_ERR_UNSUPPORTED): num_tokens * num_heads 2^26, num_seqs
 * * num_heads 2^22, max_blocks * block_size 2^30, num_seqs * max_blocks *
 * block_size 2^35, token_stride 2^24.  More than 8192 sequences go in several
 * launches. */
size_t gptoss_paged_attention_workspace_bytes(int num_tokens, int num_seqs, int num_heads, int num_kv_heads,
                                              int head_dim);
size_t gptoss_paged_attention_call_bytes(int num_tokens, int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                         int64_t max_tokens, int window, int first_tokens);
int gptoss_paged_attention_decode(const uint16_t* q, int64_t q_stride, const gptoss_kv_cache* cache,
                                  const int32_t* block_tables, int64_t table_stride, int max_blocks,
                                  const int32_t* seq_lens, int num_seqs, int num_heads,
                                  const gptoss_attention_config* cfg, uint16_t* out, int64_t out_stride,
                                  void* workspace, size_t workspace_bytes, void* stream);
/* Prompt chunks (the reference's: flash_attention.cu:100-447, there without a
 * cache): rows query_offsets[b] to query_offsets[b + 1] - 1 of q and out (num_tokens
 * rows) are the last tokens of sequence b, already appended, so row i of n is
 * at position seq_lens[b] - n + i; rows at negative positions give zeros.
 * query_offsets is [num_seqs + 1], nondecreasing; rows outside
 * [query_offsets[0], query_offsets[num_seqs]) are left as they were. */
int gptoss_paged_attention_prefill(const uint16_t* q, int64_t q_stride, const int32_t* query_offsets,
                                   int num_tokens, const gptoss_kv_cache* cache, const int32_t* block_tables,
                                   int64_t table_stride, int max_blocks, const int32_t* seq_lens, int num_seqs,
                                   int num_heads, const gptoss_attention_config* cfg, uint16_t* out,
                                   int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream);

/* ---- Routing of other models, and products of MXFP4 with MXFP4 ------------
 * None of these calls synchronises the host, allocates or needs a workspace;
 * routing, offsets and row numbers are read on the device.  They are additions:
 * the ABI version stays.  The reference has no counterpart: it routes by the
 * top logits (topk_softmax.cu:47-432), only reads MXFP4
 * (mxfp4_dequant.cu:32-71) and multiplies bf16 with it
 * (fused_mxfp4_gemv.cu:76-310). */

enum { GPTOSS_SCORE_SOFTMAX = 0, GPTOSS_SCORE_SIGMOID = 1 };

/* How a token's experts are chosen.  score: the softmax over all experts, or the
 * sigmoid of each.  choice: score + bias.  groups: num_groups contiguous ones of
 * equal size; a group counts the sum of its group_rank (1 or 2) highest choices,
 * and the top_groups highest groups stay (num_groups 1: no groups).  Of their
 * experts the top_k highest choices are taken, in descending order.  Equal ones:
 * the lower index.  Weights are the scores, without the bias; over the sum of the
 * chosen ones if renormalize (0 where that sum is 0); times scale.
 * Scores, choices and sums are those of 64 bits (choices that are closer
 * than that may come in either order), weights rounded once.
 * An expert whose logit or bias is -inf is switched off: it counts 0 in
 * its group's sum (a group of these alone comes last), is chosen only where the
 * kept groups have no other left, lower index first, and has weight 0 (whatever
 * its score is), so indices are distinct and valid in any case.  A choice of NaN is last
 * too, with its score as the weight; a NaN logit makes a softmax row's weights NaN.
 * Over a sum that is NaN all of a token's weights are. */
typedef struct gptoss_routing_config {
  int score;        /* GPTOSS_SCORE_SOFTMAX or GPTOSS_SCORE_SIGMOID */
  int top_k;        /* 1 to 32, at most the experts of top_groups groups */
  int num_groups;   /* 1 to 64, divides num_experts */
  int top_groups;   /* 1 to num_groups */
  int group_rank;   /* 1 or 2 */
  int renormalize;
  float scale;      /* finite */
} gptoss_routing_config;

/* logits: num_tokens rows of num_experts (1 to 1024) bf16 or fp32 values,
 * logits_stride elements apart, as gptoss_moe_route writes them.  bias: device fp32
 * [num_experts] or NULL.  expert_indices and expert_weights ([num_tokens][top_k])
 * are what gptoss_moe_permute_plan, gptoss_moe_layer_forward_routed and
 * gptoss_moe_combine_forward take, within their limits (256 experts and 8 of a token for
 * the plan). */
int gptoss_moe_select_experts(const void* logits, int64_t logits_stride, int logits_fp32, const float* bias,
                              int num_tokens, int num_experts, const gptoss_routing_config* cfg,
                              int32_t* expert_indices, float* expert_weights, void* stream);

/* Rows to MXFP4 in the reference layout (packed [rows][K/2], low nibble = even k;
 * scales [rows][K/32]), which gptoss_mxfp4_pack_tiled and the layer's expert
 * tables take.  A block of 32 values has the scale byte e + 127,
 * e = max(floor(log2(largest magnitude)) - 2, -126), and each value over 2^e
 * rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with its sign (half way: the
 * even code; above 6: 6).  A block with an infinity or NaN has the byte 255 and zero
 * nibbles: NaN throughout.  x: bf16 or fp32 rows, x_stride elements apart, a multiple
 * of 16 bytes; x and packed are 16-byte aligned; K is a multiple of 32. */
int gptoss_mxfp4_quantize(const void* x, int64_t x_stride, int x_fp32, int rows, int K, uint8_t* packed, uint8_t* scales,
                          void* stream);

/* The values of such a matrix, e2m1 * 2^(scale byte - 127), exact in bf16 and in fp32
 * (past the types' range: infinity; below 2^-133 rounded in bf16); NaN for a byte of 255.  out:
 * rows out_stride elements apart, a multiple of 16 bytes; 16-byte aligned.  (Of a
 * tiled matrix: gptoss_mxfp4_dequant.) */
int gptoss_mxfp4_dequantize(const uint8_t* packed, const uint8_t* scales, int rows, int K, void* out, int64_t out_stride,
                            int out_fp32, void* stream);

/* Where a product's results go.  swiglu: columns 2i (gate) and 2i + 1 (up) give
 * column i, (clamp(up, -limit, limit) + 1) * g * sigmoid(alpha * g),
 * g = min(gate, limit); NaN is kept; alpha is finite and at most 2^127 in magnitude, limit
 * is not negative.  Then either values, bf16 or fp32 in rows out_stride
 * elements apart, or (out NULL) MXFP4 as gptoss_mxfp4_quantize makes it of the
 * fp32 results, a multiple of 32 columns, out_packed 16-byte aligned.  Nothing is rounded in between; a sigmoid
 * below 2^-126 counts as 0. */
typedef struct gptoss_mxfp4_result {
  int swiglu;
  float alpha, limit;
  int out_fp32;
  void* out;
  int64_t out_stride;
  uint8_t* out_packed;
  uint8_t* out_scales;
} gptoss_mxfp4_result;

/* y[m][n] = sum_k a[m][k] * w[n][k] + bias[n], a [M][K] and w [N][K] in MXFP4, row-major
 * (16-byte aligned packed values), bias bf16 or NULL.  Products are exact and summed in
 * fp32 on the block-scaled matrix cores; a scale byte of 255 makes its row's
 * results NaN, and byte 0 is 2^-127. */
int gptoss_mxfp4_matmul(const uint8_t* a_packed, const uint8_t* a_scales, int M, const uint8_t* w_packed,
                        const uint8_t* w_scales, const uint16_t* bias, int N, int K, const gptoss_mxfp4_result* result,
                        void* stream);

/* The same for each expert e's rows p in [expert_offsets[e], expert_offsets[e + 1]), as
 * gptoss_moe_permute_plan sorts them: result row p is that of row row_index[p] of
 * a (perm_token; NULL: row p) with w_e and bias_e, w [num_experts][N][K],
 * bias [num_experts][N].  expert_offsets (device, [num_experts + 1], at most 1024
 * experts) is nondecreasing within [0, rows]; result rows outside of it are left as they
 * were.  A row number outside [0, a_rows) stands for a row of zeros: its sums are 0, also with
 * weights that are NaN, and its results those of the bias alone. */
int gptoss_moe_grouped_mxfp4_matmul(const uint8_t* a_packed, const uint8_t* a_scales, int a_rows, const int32_t* row_index,
                                    const int32_t* expert_offsets, int num_experts, int rows, const uint8_t* w_packed,
                                    const uint8_t* w_scales, const uint16_t* bias, int N, int K,
                                    const gptoss_mxfp4_result* result, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* GPTOSS_MOE_H */
