// klp_launch.h — kernel parameter blocks and launcher declarations shared by
// the kernel translation units and the C-ABI dispatcher (klp_abi.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/kernel_opt_hip.h"
#include "klp_device.h"

namespace klp {

// Depth of the forward's register ring: chunks are loaded kFwdRing - 1
// ahead of their use (klp_forward.hip).
constexpr int kFwdRing = 3;

struct FwdParams {
    const void* logits;
    RowMap rm;
    int64_t n_rows;
    int64_t vocab;
    const int64_t* targets;
    float* logprob;
    float* entropy;
    float* lse;
    // Split rows (splits > 1): [n_rows * splits] float4 (m, z, t, target
    // logit or 0) piece states and [n_rows] arrival counters, all zero
    // before the launch and left zero by it.
    float* partials;
    unsigned int* counters;
    int splits;
    float scale;      // 1 / temperature; logits are multiplied by it on load
    // Vocabulary shards (splits == 1 only): the row holds columns
    // [target_offset, target_offset + vocab) of the full vocabulary, and with
    // `state` non-null each row's float4 (m, z, t, target logit or 0) is
    // written there instead of the outputs.
    int64_t target_offset;
    float* state;
    // Last vocabulary chunk of klp_fwd_chunk (splits == 1, state null): the
    // earlier chunks' row states, [merge_count][n_rows] float4, merged in
    // chunk order with this launch's own before the outputs are written.
    // Null for every other launch.
    const float* merge_states;
    int64_t merge_count;
};

// Merge of per-shard row states (klp_fwd_shard_merge).
struct ShardMergeParams {
    const float* states;     // [n_shards][n_rows] float4
    int64_t n_shards;
    int64_t n_rows;
    const int64_t* targets;  // [n_rows], indices into the full vocabulary
    int64_t shard_vocab;     // columns per shard (the last may hold fewer)
    int64_t vocab;           // full vocabulary
    float* logprob;
    float* entropy;
    float* lse;
};

struct NaiveParams {
    const void* logits;
    RowMap rm;
    int64_t n_rows;
    int64_t vocab;
    const int64_t* targets;
    float* logprob;
    float* entropy;
    float* lse;
};

struct BwdParams {
    const void* logits;
    RowMap rm;
    int64_t n_rows;
    int64_t vocab;
    const int64_t* targets;
    const float* lse;
    const float* entropy;
    const float* g_logp;  // nullable
    const float* g_ent;   // nullable
    const float* g_lse;   // nullable
    void* d_logits;       // dense [n_rows, vocab]
    int splits;
    float scale;          // 1 / temperature (gradient is w.r.t. the unscaled logits)
    // klp_bwd_top: the alternatives and the gradients of their
    // log-probabilities, [n_rows, k]; null for every other call.
    const int64_t* top_ids;
    const float* g_top;
    int k;
};

// Launch shape: `waves` wave64s per workgroup, `unroll` 16-byte loads per
// thread per iteration, `splits` workgroups per row.  `flags` selects kernel
// variants: bit 0 (backward only) = non-temporal gradient stores.  The
// forward reads logits with non-temporal loads, the backward with ordinary
// ones.
struct FwdConfig {
    int waves;
    int unroll;
    int splits;
    int flags;
};
typedef FwdConfig BwdConfig;
constexpr int kFlagNtStore = 1;

template <typename... KArgs, typename... Args>
inline hipError_t launch_kernel(void (*kernel)(KArgs...), dim3 grid, dim3 block,
                                hipStream_t stream, Args... args) {
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, args...);
    return hipGetLastError();
}

// GRPO loss (klp_grpo.hip).  Arrays are float32 [B, S] unless noted.
struct GrpoParams {
    const float* logp;
    const float* old_logp;
    const float* ref_logp;   // nullable
    const float* adv;        // [B], or [B, S] when adv_per_token
    const void* mask;        // nullable (all ones), of mask_dtype
    int mask_dtype;          // KLP_MASK_BOOL / _U8 / _I32 / _I64, or kMaskF32
    float* mask_out;         // forward: the mask in float32, nullable
    int64_t B;
    int64_t S;
    float eps_low;
    float eps_high;
    float beta;
    float norm_const;
    int loss_type;           // klp_grpo_loss_type
    int level;               // klp_grpo_level
    int adv_per_token;
    float* ws;               // [B * kGrpoRowWords + 1]
    float* loss;             // forward: [1]
    float* stats;            // forward: [4], nullable
    const float* grad_loss;  // backward: device scalar, nullable (1)
    float* d_logp;           // backward: [B, S]
};
constexpr int kMaskF32 = -1;
// Workspace words per row of the GRPO loss (5 used, padded).
constexpr int kGrpoRowWords = 8;

// Token weights of the GRPO step (klp_grpo_token_weights): a bool / uint8,
// int32 or int64 mask (or none: all ones) divided by the loss type's
// normaliser.
struct TokenWeightsParams {
    const void* mask;  // nullable (all ones)
    int mask_dtype;    // KLP_MASK_U8 / KLP_MASK_I32 / KLP_MASK_I64
    int kind;          // 0 "grpo", 1 "bnpo", 2 fixed (scale)
    int64_t B;
    int64_t S;
    float scale;       // kind 2: the normaliser's float32 reciprocal
    float* weights;    // [B, S]
    int64_t* partial;  // kind 1: one mask sum per workgroup (kGrpoWeightsMaxBlocks)
};
// Workgroups of the token-weights kernels' grid-wide passes at most; kind 1
// keeps one 64-bit partial sum per workgroup in the caller's workspace.
constexpr int kGrpoWeightsMaxBlocks = 1024;

// Row counter of the persistent GRPO step kernel (klp_grpo_step's `sched`):
// zero before a launch, and left zero by it.
struct StepSched {
    unsigned long long next;  // rows handed out after the first gridDim.x
    unsigned int done;        // workgroups past the last row
    unsigned int unused;
};

// Fused GRPO step (klp_grpo_step.hip): the row held in the registers of one
// workgroup.  Rows are token rows of a [B, S] batch (n_rows = B * S).
struct GrpoStepParams {
    const void* logits;
    RowMap rm;
    int64_t n_rows;
    int64_t vocab;
    const int64_t* targets;
    float scale;              // 1 / temperature
    const float* old_logp;    // [n_rows]
    const float* ref_logp;    // [n_rows], nullable
    const float* adv;         // [n_rows / seq_len], or [n_rows] when adv_per_token
    const float* tok_weight;  // [n_rows]: d batch-loss / d token-loss (mask / normaliser)
    int64_t seq_len;
    float eps_low;
    float eps_high;
    float beta;
    int adv_per_token;
    float grad_scale;         // multiplies every token's gradient (not its loss)
    float* logprob;           // [n_rows]
    float* entropy;           // [n_rows]
    float* lse;               // [n_rows], nullable
    float* loss_tok;          // [n_rows]: tok_weight * token loss
    void* d_logits;           // dense [n_rows, vocab], logits dtype
    StepSched* sched;         // nullable: one workgroup per row
};
// Most 16-byte vectors one thread of the step kernel holds (1024 threads).
constexpr int kGrpoStepMaxVec = 19;
constexpr int kGrpoStepThreads = 1024;
hipError_t launch_grpo_step(int dtype, const GrpoStepParams& p, hipStream_t stream);
// Rows from which launch_grpo_step runs the persistent kernel (given a
// counter) on the current device; -1 if unknown, 0 for unsupported rows.
int64_t grpo_step_persistent_min_rows(int dtype, int64_t vocab, bool scaled);

// In-place scaling by a device scalar (klp_scale_inplace): elements
// [0, head) and [head + nvec * per-vector, n) one by one, the nvec 16-byte
// vectors from element `head` (16-byte aligned) in between.
struct ScaleParams {
    void* data;
    int64_t n;
    int64_t head;
    int64_t nvec;
    const float* scale;       // device scalar g
    float applied;            // data holds values already scaled by this; factor g / applied
};

hipError_t launch_scale(int dtype, const ScaleParams& p, hipStream_t stream);

// Fused LM head (klp_lmhead.hip).
struct LmhParams {
    const uint16_t* hidden;  // [n_tokens, ld_hidden], first `dim` columns used
    int64_t ld_hidden;
    const uint16_t* weight;  // [vocab, ld_weight]
    int64_t ld_weight;
    int64_t n_tokens;
    int64_t vocab;
    int64_t dim;             // K, a multiple of 64
    const int64_t* targets;  // [n_tokens]; row targets[n] - target_offset of the weight
    int64_t target_offset;
    float scale;             // 1 / temperature
    float* partials;         // [n_chunks, n_tokens] float4 (m, z, t, unused)
    float* target_logit;     // [n_tokens], behind the partials; written where a target is valid
    bool far;                // a row stride above kLmhMaxStride: bf16, float32 logits
    int block_tokens;        // tokens per workgroup: 256, 192 or 128
    int64_t n_tblocks;       // ceil(n_tokens / block_tokens)
    int64_t n_vtiles;        // ceil(vocab / 256)
    int64_t tiles_per_chunk;
    int64_t n_chunks;        // ceil(n_vtiles / tiles_per_chunk)
    float* logprob;
    float* entropy;
    float* lse;
    // d_logits (backward) only:
    const float* g_logp;     // nullable
    const float* g_ent;      // nullable
    const float* g_lse;      // nullable
    const float* saved_lse;  // [n_tokens], as the forward wrote it
    const float* saved_entropy;
    // d_logits and logits: [n_tokens, ld_out], columns vocab .. n_out - 1
    // written with zeros; out_align: alignment of every row, 16, 8 or 2 bytes.
    uint16_t* out;
    int64_t ld_out;
    int64_t n_out;
    int out_align;
};
int64_t lmh_vocab_tiles(int64_t vocab);
// The longest row stride whose 256 rows 32-bit byte offsets reach.
constexpr int64_t kLmhMaxStride = INT32_MAX / 512;
// `rounded`: logits rounded once to `dtype` (bf16 or fp16); otherwise bf16
// operands and float32 logits.
hipError_t launch_lmh_fwd(int dtype, bool rounded, const LmhParams& p, hipStream_t stream);
hipError_t launch_lmh_dlogits(int dtype, bool rounded, const LmhParams& p, hipStream_t stream);
hipError_t launch_lmh_logits(int dtype, const LmhParams& p, hipStream_t stream);

// The LM head's backward products (klp_head_gemm.hip): out[n, m] (or, with
// `slabs`, float32 slab[split][n, m]) = sum_k a[k, m] * b, b = b[k, n] for
// 16-bit output and b[n, k] for slabs.  16-bit a, b; strides in elements,
// multiples of 8; m a multiple of 64; K-contiguous b: k a multiple of 8.
struct HeadGemmParams {
    const uint16_t* a;
    int64_t ld_a;
    const uint16_t* b;
    int64_t ld_b;
    int64_t m, n, k;
    int64_t m_tiles, n_tiles;  // of 256
    int64_t k_per_split;       // a multiple of 64 (k without splits)
    int64_t n_items;           // m_tiles * n_tiles * splits
    int64_t group;             // row blocks taken together
    uint16_t* out;             // [n, ld_out]
    int64_t ld_out;
    float* slabs;              // [splits][n][m], nullable
};
struct HeadSumParams {
    const float* slabs;
    int n_slabs;
    int accumulate;            // add to acc
    int64_t n_vec;             // n * m / 4
    float* acc;                // float32 result, and addend with `accumulate`
    uint16_t* out;             // 16-bit result instead, nullable
};
// Workgroups at once: one per CU.
constexpr int64_t kHeadGemmCus = 256;
// Row blocks taken together, at most: 6 x 5 tiles are an XCD's 32 at a time.
constexpr int64_t kHeadGemmGroup = 6;
hipError_t launch_head_gemm(int dtype, const HeadGemmParams& p, hipStream_t stream);
hipError_t launch_head_sum(int dtype, const HeadSumParams& p, hipStream_t stream);

// Root-mean-square norm (klp_norm.hip).  Rows of x, residual at row strides;
// every other array dense.
constexpr int kScaleBlock = 128;        // elements along a row that share an e4m3 scale
constexpr int64_t kNormMaxDim = 65536;  // a row is held by one workgroup
struct NormParams {
    const void* x;         // [rows, ld_x]
    int64_t ld_x;
    const void* residual;  // [rows, ld_r], nullable
    int64_t ld_r;
    const void* weight;    // [dim], float32 with weight_f32, else of the rows' dtype
    int weight_f32;
    int64_t rows;
    int64_t dim;
    float eps;
    void* h;               // [rows, dim]: written with a residual
    void* y;               // [rows, dim]
    float* rstd;           // [rows], nullable
    uint8_t* q;            // [rows, dim] e4m3 codes, instead of y; nullable
    float* scales;         // [rows, n_blocks]
    int64_t n_blocks;      // ceil(dim / kScaleBlock)
};
struct NormBwdParams {
    const void* h;         // [rows, ld_h]
    int64_t ld_h;
    const void* weight;
    int weight_f32;
    const float* rstd;     // [rows]
    const void* g_y;       // [rows, dim]
    const void* g_h;       // [rows, dim], nullable
    int64_t rows;
    int64_t dim;
    int64_t groups;        // norm_bwd_groups(rows, dim)
    void* d_x;             // [rows, dim]
    float* partials;       // [groups, dim], nullable: no d_weight
    void* d_weight;        // [dim]
};
// Threads of the backward's grid: 1024 a CU.
constexpr int64_t kNormBwdThreads = 256 * 1024;
int64_t norm_threads(int64_t dim);  // of a row
int64_t norm_bwd_groups(int64_t rows, int64_t dim);
hipError_t launch_norm(int dtype, const NormParams& p, hipStream_t stream);
hipError_t launch_norm_bwd(int dtype, const NormBwdParams& p, hipStream_t stream);
hipError_t launch_norm_dw(int weight_dtype, const NormBwdParams& p, hipStream_t stream);

// The norms around a block (klp_block.hip).  Rows of x and residual at row
// strides; every other array dense.
constexpr int64_t kBlockMaxDim = 16384;
struct BlockParams {
    const void* x;         // [rows, ld_x]
    int64_t ld_x;
    const void* residual;  // [rows, ld_r]
    int64_t ld_r;
    const void* post;      // [dim], nullable: no norm behind the block
    const void* weight;    // [dim]; both float32 with weight_f32, else of the rows' dtype
    int weight_f32;
    const void* gate;      // [ceil(rows / per_gate), dim], nullable
    int gate_f32;
    int64_t per_gate;      // consecutive rows that share a gate
    float scale;
    int64_t rows;
    int64_t dim;
    float eps;
    void* h;               // [rows, dim]
    void* y;               // [rows, dim]
    float* rstd_x;         // [rows], nullable; with `post`
    float* rstd_h;         // [rows], nullable
    uint8_t* q;            // [rows, dim] e4m3 codes, instead of y; nullable
    float* scales;         // [rows, n_blocks]
    uint8_t* x_codes;      // checkpoints of x and h: codes [rows, dim], nullable,
    float* x_scales;       // and scales [rows, n_blocks]
    uint8_t* h_codes;
    float* h_scales;
    int64_t n_blocks;      // ceil(dim / kScaleBlock)
    int whole;             // dim a multiple of 8, every row at one of 16 bytes
};
struct BlockBwdParams {
    const void* x;         // [rows, ld_x], or x_codes and x_scales; null: not needed
    int64_t ld_x;
    const uint8_t* x_codes;
    const float* x_scales;
    const void* h;         // [rows, dim], or h_codes and h_scales
    const uint8_t* h_codes;
    const float* h_scales;
    int64_t n_blocks;
    const void* post;
    const void* weight;
    int weight_f32;
    const void* gate;
    int gate_f32;
    int64_t per_gate;
    float scale;
    const float* rstd_x;
    const float* rstd_h;
    const void* g_y;       // [rows, dim], nullable
    const void* g_h;       // [rows, dim], nullable
    int64_t rows;
    int64_t dim;
    int64_t groups;        // block_shape(rows, dim): of per_group consecutive rows
    int64_t per_group;
    int whole;             // as BlockParams'
    void* d_x;             // [rows, dim], nullable
    void* d_r;             // [rows, dim], nullable
    void* d_post;          // [dim], nullable
    void* d_weight;        // [dim], nullable
    void* d_gate;          // as gate, nullable
    // Float32 sums of the workgroups (of their groups' rows) for d_post,
    // d_weight and a gate that all rows share, [BlockShape::shares][dim] each;
    // and of the first and last gate of every group, [2 groups][dim].
    float* post_shares;
    float* weight_shares;
    float* gate_shares;
};
struct BlockShape {
    int64_t groups, per_group, shares;
};
BlockShape block_shape(int64_t rows, int64_t dim);
hipError_t launch_block(int dtype, const BlockParams& p, hipStream_t stream);
hipError_t launch_block_bwd(int dtype, const BlockBwdParams& p, hipStream_t stream);

// e4m3 codes and scales (klp_fp8.hip): 128 elements of a row share a scale,
// or 128 x 128 elements do.
struct QuantizeParams {
    const void* x;      // [rows, ld_x]
    int64_t ld_x;
    int64_t rows;
    int64_t dim;
    int64_t n_blocks;   // ceil(dim / kScaleBlock)
    int block_rows;     // 1 or 128
    uint8_t* q;         // [rows, dim]
    float* scales;      // [ceil(rows / block_rows), n_blocks]
};
hipError_t launch_quantize(int dtype, const QuantizeParams& p, hipStream_t stream);

// Product of e4m3 matrices with a scale for each 128 of K (klp_fp8_gemm.hip):
// out[m, n] = sum_b xs[m, b] ws[n / 128, b] sum_{k in b} x[m, k] w[n, k].
struct Fp8LinearParams {
    const uint8_t* x;   // [m, ld_x]
    int64_t ld_x;
    const float* xs;    // [m, n_blocks]
    const uint8_t* w;   // [n, ld_w]
    int64_t ld_w;
    const float* ws;    // [ceil(n / 128), n_blocks]
    int64_t m, n, k;
    int64_t n_blocks;   // ceil(k / 128)
    void* out;          // [m, ld_out]
    int64_t ld_out;
    // Epilogue: out = act(product + bias) + residual.
    int epilogue;          // any of the following
    const void* bias;      // [n], nullable; float32 with bias_f32, else of out's dtype
    int bias_f32;
    int act;               // klp_activation
    float cap;             // KLP_ACT_SOFTCAP
    const void* residual;  // [m, ld_res] of out's dtype, nullable
    int64_t ld_res;
    int res_aligned;       // 4 consecutive elements at a multiple of their size
};
hipError_t launch_fp8_linear(int out_dtype, const Fp8LinearParams& p, hipStream_t stream);

// Sampling (klp_sample.hip).
constexpr int64_t kSampleMaxVocab = int64_t{1} << 26;
struct SampleParams {
    const void* logits;
    RowMap rm;
    int64_t n_rows;
    int64_t vocab;
    const float* uniform;       // [n_rows]
    // A parameter of every row, or an array of one per row where non-null.
    float temperature, top_p, min_p;
    int top_k;
    const float* temperatures;
    const float* top_ps;
    const float* min_ps;
    const int32_t* top_ks;
    int64_t* tokens;            // [n_rows]
    float* logp;                // [n_rows]
    float* sample_logp;         // [n_rows]
};
hipError_t launch_sample(int dtype, const SampleParams& p, hipStream_t stream);

// Log-probabilities with alternatives (klp_top.hip).
constexpr int64_t kTopMaxVocab = int64_t{1} << 26;
constexpr int kTopMax = 256;            // alternatives of a row at most
constexpr int kTopMergeKeys = 4096;     // splits * k at most
constexpr int kTopCounterStride = 16;   // a row's counter has 64 bytes
// Rows of up to this many logits stay in a workgroup's registers.
constexpr int64_t kTopShort = 4096;
struct TopParams {
    const void* logits;
    RowMap rm;
    int64_t n_rows;
    int64_t vocab;
    const int64_t* targets;
    int k;
    float factor;          // log2(e) / temperature
    float inv_t;           // 1 / temperature
    int waves;             // of a workgroup: 4 or 8
    int splits;            // workgroups of a row, at most 64
    // Pieces (splits > 1): arrival counters, kTopCounterStride words a row,
    // zero before the launch and left zero by it, and [n_rows, splits, k + 2]
    // words of any contents: a piece's state and its keys.
    unsigned int* counters;
    unsigned long long* words;
    float* logprob;
    float* entropy;
    float* lse;
    int64_t* rank;
    int64_t* top_ids;      // [n_rows, k]
    float* top_logprob;    // [n_rows, k]
};
hipError_t launch_top(int dtype, const TopParams& p, hipStream_t stream);

// Calibration kernels (klp_ceiling.hip): rows of `row_bytes` (a multiple of
// 16) at `src` (and `dst`), 16-byte aligned and contiguous; `splits`
// workgroups per row.  Modes: the forward's ring read, and the backward's
// loop as a copy, its loads alone and its stores alone.
enum : int { kCeilRead = 0, kCeilCopy = 1, kCeilReadPieces = 2, kCeilWrite = 3 };
struct CeilingParams {
    const void* src;     // all modes but kCeilWrite
    void* dst;           // kCeilCopy, kCeilWrite
    int64_t n_rows;
    int64_t row_bytes;
    int64_t splits;
    uint32_t* sink;      // reads: [n_rows * splits], written when fold == magic
    uint32_t magic;
};
hipError_t launch_ceiling(int mode, const CeilingParams& p, int waves, int unroll,
                          hipStream_t stream);

hipError_t launch_fwd(int dtype, const FwdParams& p, const FwdConfig& c, hipStream_t stream);
hipError_t launch_shard_merge(const ShardMergeParams& p, hipStream_t stream);
hipError_t launch_fwd_naive(int dtype, const NaiveParams& p, hipStream_t stream);
hipError_t launch_bwd(int dtype, const BwdParams& p, const BwdConfig& c, hipStream_t stream);
hipError_t launch_grpo_fwd(const GrpoParams& p, hipStream_t stream);
hipError_t launch_grpo_bwd(const GrpoParams& p, hipStream_t stream);
hipError_t launch_grpo_token_weights(const TokenWeightsParams& p, hipStream_t stream);
bool fwd_config_supported(const FwdConfig& c);
bool bwd_config_supported(const BwdConfig& c);

}  // namespace klp
