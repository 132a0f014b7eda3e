/*
 * wisp_b200.h -- C ABI of libwisp_b200.so, the B200-native (sm_100a)
 * routed-expert int4 FFN hot path for the WISP engine.
 *
 * Part 1 re-exports the reference engine's GPU launcher ABI with identical
 * names and signatures, so the reference C engine links against this
 * library in place of its csrc/cuda/*.cu objects.
 * Part 2 adds the fused entry points the reference's gpu_expert_ffn /
 * run_moe would call instead of the dequant -> gemv -> scale_accum chain.
 *
 * No entry point allocates device memory per call: the caller passes every
 * buffer (workspace sizes come from the *_workspace_bytes queries). All
 * pointers named d_* are device pointers; launches are asynchronous on the
 * given stream.
 */
#ifndef WISP_B200_H
#define WISP_B200_H

#include <stddef.h>
#include <stdint.h>
#include <cuda_runtime.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* --------------------------------------------------------------------------
 * Engine types shared with the reference ABI. A translation unit that has
 * already included the reference's csrc/core/wisp_engine.h defines
 * WISP_B200_NO_ENGINE_TYPES before including this header.
 * Layouts are identical to csrc/core/wisp_engine.h:32-40, 50-64, 214-251.
 * ------------------------------------------------------------------------ */
#ifndef WISP_B200_NO_ENGINE_TYPES
typedef uint16_t wisp_half; /* raw fp16 bits (the reference's C view) */

typedef enum {
    WISP_OK = 0,
    WISP_ERR_OOM = 1,
    WISP_ERR_IO = 2,
    WISP_ERR_CUDA = 3,
    WISP_ERR_INVALID_ARG = 4,
    WISP_ERR_EXPERT_MISS = 5,
    WISP_ERR_MODEL = 6,
    WISP_ERR_TIMEOUT = 7,
} WispError;

typedef struct {
    WispError code;
    char message[512];
    const char* file;
    int line;
} WispErrCtx;

#define WISP_EXPERT_MAGIC 0x57455850u
#define WISP_EXPERT_VERSION 1u
#define WISP_EXPERT_NMATS 3

#pragma pack(push, 1)
typedef struct {
    uint32_t rows;
    uint32_t cols;
    uint64_t packed_bytes;
    uint64_t scales_bytes;
    uint64_t zeros_bytes;
} WispExpertMat;

typedef struct {
    uint32_t magic;
    uint32_t version;
    uint32_t layer_id;
    uint32_t expert_id;
    uint32_t group_size;
    uint32_t n_mats;
    WispExpertMat mats[WISP_EXPERT_NMATS];
} WispExpertHeader; /* exactly 120 bytes */
#pragma pack(pop)

typedef struct {
    size_t packed_off[WISP_EXPERT_NMATS];
    size_t scales_off[WISP_EXPERT_NMATS];
    size_t zeros_off[WISP_EXPERT_NMATS];
    uint32_t rows[WISP_EXPERT_NMATS];
    uint32_t cols[WISP_EXPERT_NMATS];
    uint32_t group_size;
    size_t total_bytes;
    int valid;
} WispExpertMeta;
#endif /* WISP_B200_NO_ENGINE_TYPES */

/* ==========================================================================
 * Part 1 -- reference launcher ABI (drop-in)
 * ======================================================================== */

/* Replaces csrc/cuda/expert_loader.cu:46-63 (declared at
 * csrc/core/wisp_engine.h:545-550). cudaErrorInvalidValue when
 * n_elements <= 0 or group_size <= 0, else the launch status. */
cudaError_t launch_dequant_expert(const uint8_t* d_packed, const wisp_half* d_scales,
                                  const wisp_half* d_zeros, wisp_half* d_output,
                                  int n_elements, int group_size, cudaStream_t stream);

/* Replaces csrc/cuda/expert_loader.cu:67-97 (wisp_engine.h:551-559). */
cudaError_t async_load_expert(const uint8_t* h_packed, const wisp_half* h_scales,
                              const wisp_half* h_zeros, uint8_t* d_packed_tmp,
                              wisp_half* d_scales_tmp, wisp_half* d_zeros_tmp,
                              wisp_half* d_output, int n_elements, int group_size,
                              cudaStream_t stream);

/* Replaces csrc/cuda/matmul.cu:58-65 (wisp_engine.h:499-500): y = W x. */
void wisp_gpu_gemv_f16(const wisp_half* W, const float* x, float* y, int rows, int cols,
                       cudaStream_t s);

/* Replaces csrc/cuda/matmul.cu:141-148 (wisp_engine.h:507-508). */
void wisp_gpu_swiglu(const float* gate, const float* up, float* out, int n, cudaStream_t s);

/* Replaces csrc/cuda/matmul.cu:198-205 (wisp_engine.h:509-511):
 * h[r] = silu(Wg[r].x) * (Wu[r].x). */
void wisp_gpu_swiglu_ffn(const wisp_half* Wg, const wisp_half* Wu, const float* x, float* h,
                         int inter, int cols, cudaStream_t s);

/* Replaces csrc/cuda/matmul.cu:156-161 (wisp_engine.h:512-513): acc += w x. */
void wisp_gpu_scale_accum(float* acc, const float* x, float w, int n, cudaStream_t s);

/* Replaces csrc/cuda/router.cu:140-171 (wisp_engine.h:534-537). Softmax
 * top-k with renormalised weights; ties go to the lower expert index.
 * out_idx / out_w are host (pinned) buffers filled by async copies on `s`;
 * the caller synchronises `s` before reading them. top_k is clamped to 64;
 * any n_experts (logits_scratch [n_experts] is working memory, as in the
 * reference: it holds exp(logit - max) afterwards). */
void wisp_gpu_router_topk(const wisp_half* W, const wisp_half* bias, const float* x,
                          float* logits_scratch, int n_experts, int hidden, int top_k,
                          int* out_idx, float* out_w, cudaStream_t s);

/* ==========================================================================
 * Part 2 -- fused entry points
 * ======================================================================== */

/* Parse an expert blob header held in HOST memory. Same contract as the
 * reference's wisp_expert_parse_header (csrc/core/wisp_engine.c:268-303):
 * WISP_ERR_MODEL on a bad magic/version/n_mats or a truncated blob. */
WispError wisp_b200_parse_expert_header(const void* blob, size_t blob_size,
                                        WispExpertMeta* meta, WispErrCtx* err);

/* One token, several experts, reference precision (fp32 activations):
 *   d_acc[hidden] += sum_j weights[j] * down_j(silu(gate_j x) * up_j x)
 * Replaces the per-expert loop of gpu_expert_ffn (csrc/core/wisp_engine.c:
 * 1507-1531) as called from run_moe (:1666-1670), plus an int4 shared
 * expert passed as one more blob with weight 1.0. d_blobs[j] is the device
 * address of blob j (header at offset 0; the packed weights must be at least
 * 8-byte aligned). weights is a HOST array. 1 <= n_blobs <= 16. The scratch
 * holds the intermediate activations; its size comes from
 * wisp_b200_expert_ffn_scratch_bytes. */
size_t wisp_b200_expert_ffn_scratch_bytes(const WispExpertMeta* meta, int n_blobs);
WispError wisp_b200_expert_ffn(const WispExpertMeta* meta, const void* const* d_blobs,
                               const float* weights, int n_blobs, const float* d_x,
                               float* d_acc, void* d_scratch, size_t scratch_bytes,
                               cudaStream_t stream, WispErrCtx* err);

/* The same computation for callers that cannot allocate device memory (an
 * engine whose VRAM budget is fully committed to the expert cache, or a
 * host callback where cudaMalloc would synchronise the device). No
 * counterpart in the reference. The intermediate activations use a fixed
 * 227 KB array per device compiled into the library, so n_blobs * inter must
 * be <= 58112 (else WISP_ERR_INVALID_ARG). The first call on a device looks
 * up that array's device address in the device's primary context; make it
 * before any stream capture, and do not use this entry after a
 * cudaDeviceReset or from another driver context. Calls share the array:
 * calls that overlap on the GPU race on it. */
WispError wisp_b200_expert_ffn_noalloc(const WispExpertMeta* meta, const void* const* d_blobs,
                                       const float* weights, int n_blobs, const float* d_x,
                                       float* d_acc, cudaStream_t stream, WispErrCtx* err);

/* --------------------------------------------------------------------------
 * Batched MoE layer (T tokens, bf16 activations).
 * ------------------------------------------------------------------------ */
enum { WISP_SCORE_SOFTMAX = 0, WISP_SCORE_SIGMOID_GROUPED = 1 };

typedef struct {
    int tokens;        /* T */
    int hidden;        /* M: multiple of 128 */
    int inter;         /* I: multiple of 128 */
    int n_experts;     /* routed experts E (<= 1024) */
    int top_k;         /* <= min(32, n_experts) */
    int group_size;    /* int4 quantisation group along K: 64 or 128 */
    int scoring;       /* WISP_SCORE_* */
    int n_groups;      /* sigmoid scoring: expert groups (E % n_groups == 0) */
    int topk_groups;   /* sigmoid scoring: groups kept */
    float routed_scaling; /* sigmoid scoring: weight multiplier */
    int has_shared;    /* 1: an always-on shared expert of the same shape */
    int router_fp16;   /* router weight dtype: 0 = bf16, 1 = fp16 (the
                          reference's router ABI, wisp_engine.h:534-537) */
    int deterministic; /* wisp_b200_moe_forward only (other entry points
                          ignore it). 0: expert outputs meet in fp32 atomics,
                          so results may differ in the last bits from run to
                          run. 1: the expert outputs are written as rows and
                          each token's are summed in a fixed order, so every
                          run gives the same bits; costs a (T x (top_k +
                          shared)) x hidden fp32 buffer in the workspace and
                          the single-token decode fast path. */
} WispMoeConfig;

/* One int4 matrix in the reference's packing (low nibble = even index,
 * value = (nibble - 8) * scale + zero, groups along K). zeros may be NULL
 * (symmetric). packed / scales / zeros must be 16-byte aligned. */
typedef struct {
    const uint8_t* packed;
    const wisp_half* scales;
    const wisp_half* zeros;
} WispInt4Mat;

/* gate [I x M], up [I x M], down [M x I]. */
typedef struct {
    WispInt4Mat gate, up, down;
} WispInt4Expert;

typedef struct {
    const uint16_t* router_w;       /* bf16 or fp16 [E x M] (cfg->router_fp16) */
    const float* router_bias;       /* fp32 [E], added before scoring; may be NULL */
    const WispInt4Expert* experts;  /* DEVICE array: E routed experts, then the
                                       shared expert when cfg->has_shared */
    const void* prepared;           /* from wisp_b200_prepare_experts over the
                                       same E (+1) entries */
} WispMoeWeights;

/* One-time preparation of a weight set for the tensor-core kernels (once per
 * layer when the weights are loaded, or when an expert blob is promoted into
 * the VRAM tier): per matrix a TMA descriptor of its packed nibbles, and its
 * scales / zero points transposed to [128-row tile][group][row] so each
 * stage's scales are one contiguous run. The packed nibbles stay where they
 * are and must stay valid. d_experts is a DEVICE array of n_entries; the call
 * copies it to the host, so it synchronises `stream`. */
size_t wisp_b200_prepared_bytes(const WispMoeConfig* cfg, int n_entries);
WispError wisp_b200_prepare_experts(const WispMoeConfig* cfg, const WispInt4Expert* d_experts,
                                    int n_entries, void* d_prepared, size_t prepared_bytes,
                                    cudaStream_t stream, WispErrCtx* err);

/* Re-prepares entry `slot` (0 <= slot < n_entries) of a prepared set in
 * place from a HOST copy of its expert-table entry and leaves every other
 * entry as it is: the hook for an expert blob that has just been promoted
 * into a VRAM slot (csrc/core/wisp_engine.c:1164-1203 copies the blob into
 * VRAM; this call then builds that slot's TMA descriptors and transposed
 * scales). The bytes it writes equal those wisp_b200_prepare_experts writes
 * for the same entry. The packed nibbles are used where they lie, in the
 * blob's own layout. Asynchronous on `stream`, with no host staging (the
 * descriptors travel as kernel parameters); updating the device expert
 * table entry itself is the caller's part. */
WispError wisp_b200_prepare_expert_slot(const WispMoeConfig* cfg, int n_entries, int slot,
                                        const WispInt4Expert* entry, void* d_prepared,
                                        size_t prepared_bytes, cudaStream_t stream,
                                        WispErrCtx* err);

/* The expert-table entry of a reference expert blob that lies at device
 * address d_blob: pointers to its gate, up and down packed nibbles, scales
 * and (when the blob carries them) zero points, at the offsets of the
 * parsed header (csrc/core/wisp_engine.c:268-303). Host-only pointer
 * arithmetic: d_blob is never dereferenced. WISP_ERR_INVALID_ARG when meta
 * is invalid or a matrix's packed data or scales would not be 16-byte
 * aligned (a blob placed at an address = 8 mod 16 has both aligned, since
 * its packed data starts at offset 120). */
WispError wisp_b200_blob_expert(const WispExpertMeta* meta, const void* d_blob,
                                WispInt4Expert* out, WispErrCtx* err);

size_t wisp_b200_moe_workspace_bytes(const WispMoeConfig* cfg);

/* out[T x M] (fp32) = sum_k w[t,k] * expert_{idx[t,k]}(x_t) + shared(x_t).
 * x: bf16 [T x M]. topk_idx / topk_w ([T x k], int32 / fp32) receive the
 * routing and may be NULL. */
WispError wisp_b200_moe_forward(const WispMoeConfig* cfg, const WispMoeWeights* w,
                                const uint16_t* d_x, float* d_out, int* d_topk_idx,
                                float* d_topk_w, void* d_workspace, size_t workspace_bytes,
                                cudaStream_t stream, WispErrCtx* err);

/* Dense int4 MLP over T tokens (the MLP of the first dense layers of
 * DeepSeek/GLM models, csrc/core/wisp_engine.c:1676-1686, and any
 * always-on MLP quantised to int4):
 *   d_out[T x M] (fp32) = down(silu(gate x) * up x), x bf16 [T x M].
 * d_mlp is a DEVICE array holding the MLP's one WispInt4Expert entry and
 * d_prepared its prepared set (wisp_b200_prepare_experts over that entry).
 * Uses cfg's tokens, hidden, inter and group_size only. The output rows are
 * written, not accumulated. d_error_flag as for wisp_b200_grouped_ffn (may
 * be NULL). One call at a time per workspace. */
size_t wisp_b200_dense_mlp_workspace_bytes(const WispMoeConfig* cfg);
WispError wisp_b200_dense_mlp(const WispMoeConfig* cfg, const void* d_prepared,
                              const WispInt4Expert* d_mlp, const uint16_t* d_x, float* d_out,
                              void* d_workspace, size_t workspace_bytes, int* d_error_flag,
                              cudaStream_t stream, WispErrCtx* err);

/* --------------------------------------------------------------------------
 * Building blocks (used by the expert-parallel path and by tests).
 * ------------------------------------------------------------------------ */

/* Router only: d_idx / d_w [T x k]; d_logits (fp32 [T x E]) receives the
 * logits, bias included. */
WispError wisp_b200_route(const WispMoeConfig* cfg, const WispMoeWeights* w, const uint16_t* d_x,
                          float* d_logits, int* d_idx, float* d_w, cudaStream_t stream,
                          WispErrCtx* err);

/* The same routing with the logits summed over K splits, so that a few
 * tokens still spread over the SMs (wisp_b200_route computes each token
 * tile's logits in one pass over K). d_workspace holds the split partial
 * sums (wisp_b200_route_workspace_bytes, 16-byte aligned; one call at a
 * time per workspace); d_logits may be NULL. Same results as
 * wisp_b200_route within fp32 summation order. */
size_t wisp_b200_route_workspace_bytes(const WispMoeConfig* cfg);
WispError wisp_b200_route_ws(const WispMoeConfig* cfg, const WispMoeWeights* w,
                             const uint16_t* d_x, float* d_logits, int* d_idx, float* d_w,
                             void* d_workspace, size_t workspace_bytes, cudaStream_t stream,
                             WispErrCtx* err);

/* A contiguous run of activation rows that all go through one expert. */
typedef struct {
    int32_t expert;    /* index into the expert table */
    int32_t row_begin; /* first row in the activation buffer */
    int32_t rows;      /* number of rows (0 allowed) */
    int32_t reserved;
} WispSegment;

/* Grouped expert FFN over pre-permuted rows. d_prepared / d_experts /
 * n_entries: a prepared weight set and its device expert table (segment
 * experts index its entries). Segments of at most 32 rows (decode) run on
 * the register-fed integer tensor-core kernel, larger ones on the tcgen05
 * kernel.
 *   d_xp:   fp16 [R x M] activation rows in interleaved K order (within each
 *           8 K: 0,4,1,5,2,6,3,7) -- produced by wisp_b200_pack_rows.
 *   d_segs: DEVICE array of n_segs segments.
 *   d_h:    [R x I] scratch of 2 bytes per element (the SwiGLU output: fp16
 *           rows for tensor-core segments, 16-bit integer rows with
 *           per-128-K scales in the workspace for register-path segments).
 *   mode 0: d_out[row_token[p] * M + m] += row_weight[p] * y[p, m] (atomic fp32)
 *   mode 1: d_y[p * M + m] = y[p, m] (fp32 rows, no weighting)
 * d_workspace: wisp_b200_grouped_workspace_bytes(cfg, n_segs, rows_capacity)
 *          bytes, 256-byte aligned (tile and unit plans, the register path's
 *          integer activation rows and their scales, and ~33.5 MB for the
 *          partial sums of a K-split gate/up); one call at a time per
 *          workspace.
 * d_error_flag: device int set to nonzero if a bounded wait gave up (may be
 * NULL); check it with wisp_b200_check_error_flag. */
size_t wisp_b200_grouped_workspace_bytes(const WispMoeConfig* cfg, int n_segs, int rows_capacity);
WispError wisp_b200_grouped_ffn(const WispMoeConfig* cfg, const void* d_prepared,
                                const WispInt4Expert* d_experts, int n_entries,
                                const WispSegment* d_segs, int n_segs, int rows_capacity,
                                const uint16_t* d_xp, uint16_t* d_h, int mode,
                                const int* d_row_token, const float* d_row_weight,
                                float* d_out, void* d_workspace, size_t workspace_bytes,
                                int* d_error_flag, cudaStream_t stream, WispErrCtx* err);

/* Dispatch plan from a routing: one segment per expert (then the shared
 * expert with every token when cfg->has_shared), rows sorted by (token,
 * slot) inside each expert. d_counts [V], d_segs [V], d_row_token /
 * d_row_weight [T*k (+T)], V = E (+1). Deterministic. */
WispError wisp_b200_dispatch_plan(const WispMoeConfig* cfg, const int* d_idx, const float* d_w,
                                  int* d_counts, WispSegment* d_segs, int* d_row_token,
                                  float* d_row_weight, cudaStream_t stream, WispErrCtx* err);

/* d_out[row_token[p]] += row_weight[p] * d_y[p] for p < n_rows (fp32 rows;
 * atomic adds): the combine step of the expert-parallel path. */
WispError wisp_b200_combine_rows(const float* d_y, const int* d_row_token, const float* d_row_weight,
                                 int n_rows, int hidden, float* d_out, cudaStream_t stream,
                                 WispErrCtx* err);

/* --------------------------------------------------------------------------
 * Expert-parallel exchange (no counterpart in the reference, which runs on one
 * GPU). Experts are sharded in contiguous blocks of e_loc = n_experts/world.
 * Each rank pair exchanges one fixed-size block per direction, so all counts
 * stay on the device; a token travels to an owner rank once, whatever the
 * number of its experts there. cap = the most tokens any rank holds. Block
 * layout (wisp_b200_ep_block_bytes bytes, 16-byte aligned parts):
 *   int32 n_rows, 3 pad; int32 cnt[e_loc]           header
 *   int32 ent_row[cap*top_k]; float ent_w[cap*top_k] entries, expert-major
 *   fp16 rows[cap][hidden]                           interleaved K order
 * ------------------------------------------------------------------------ */
size_t wisp_b200_ep_block_bytes(int hidden, int e_loc, int cap, int top_k);

/* Send side: d_send [world blocks] from this rank's routing (d_topk_idx
 * [tokens x top_k], global experts) and its dispatch plan over the n_experts
 * routed experts (d_plan_segs, d_row_token, d_row_weight from
 * wisp_b200_dispatch_plan with has_shared = 0). d_slot [tokens x world]
 * receives the row of each token in each block (-1: not sent there). d_own
 * (may be NULL) receives the same rows for this rank's own tokens [tokens x
 * hidden] (fp16, interleaved K order), the shared expert's input. */
WispError wisp_b200_ep_dispatch(const uint16_t* d_x, int tokens, int hidden, const int* d_topk_idx,
                                int top_k, const WispSegment* d_plan_segs, const int* d_row_token,
                                const float* d_row_weight, int n_experts, int world, int cap,
                                uint8_t* d_send, int* d_slot, uint16_t* d_own,
                                cudaStream_t stream, WispErrCtx* err);

/* Receive side, from the received blocks d_recv [world blocks] (world * e_loc
 * <= 1024): the entries are gathered expert-contiguous (expert, then source)
 * so each local expert is one segment: d_segs [e_loc] over the gathered
 * rows, d_src_pos[j] = receive row (source * cap + block row) and
 * d_weight[j] = routing weight of gathered row j, *d_total = entries.
 * own_rows > 0 (<= cap) appends this rank's own own_rows token rows as
 * segment e_loc (the shared expert's entry of the local table), with
 * d_src_pos = world * cap + t and weight 1, so the shared expert runs in the
 * same grouped call as the routed experts. d_src_pos and d_weight hold
 * world * cap * top_k + own_rows entries, d_segs e_loc (+1). */
WispError wisp_b200_ep_recv_plan(const uint8_t* d_recv, int world, int e_loc, int cap, int top_k,
                                 int hidden, int own_rows, WispSegment* d_segs, int* d_src_pos,
                                 float* d_weight, int* d_total, cudaStream_t stream,
                                 WispErrCtx* err);

/* d_sorted[j] = receive row d_src_pos[j] for j < *d_total + own_rows (fp16
 * rows; a d_src_pos of world * cap + t reads row t of d_own, this rank's own
 * token rows packed with wisp_b200_pack_rows; max_rows bounds the launch,
 * normally world * cap * top_k + own_rows). The grouped FFN then runs in
 * mode 0 with row_token = d_src_pos and row_weight = d_weight into fp32 rows
 * [(world * cap + own_rows) x hidden] (zeroed first): one row per received
 * token, which the return exchange sends back, then the shared expert's
 * output for each own token. */
WispError wisp_b200_ep_gather_rows(const uint8_t* d_recv, int world, int e_loc, int cap, int top_k,
                                   int hidden, const int* d_src_pos, const int* d_total,
                                   const uint16_t* d_own, int own_rows, int max_rows,
                                   uint16_t* d_sorted, cudaStream_t stream, WispErrCtx* err);

/* d_out[t] += d_yback[q * cap + d_slot[t * world + q]] over q = 0..world-1
 * with a slot >= 0, in rank order (fp32 rows; one block per token). */
WispError wisp_b200_ep_combine(const float* d_yback, const int* d_slot, int tokens, int world,
                               int cap, int hidden, float* d_out, cudaStream_t stream,
                               WispErrCtx* err);

/* The return exchange in fp16 (half the bytes of fp32 rows): the owner
 * rounds its fp32 return rows to fp16 (d_y16[i] = fp16(d_y[i]) for rows x
 * hidden values), the rows travel, and the home rank adds them in rank
 * order with wisp_b200_ep_combine_f16 (wisp_b200_ep_combine's contract with
 * fp16 rows; with d_local non-NULL, fp32 [tokens x hidden], the result is
 * d_out[t] = d_local[t] + the returned rows, written rather than added). */
WispError wisp_b200_ep_return_rows(const float* d_y, int rows, int hidden, uint16_t* d_y16,
                                   cudaStream_t stream, WispErrCtx* err);
WispError wisp_b200_ep_combine_f16(const uint16_t* d_yback, const int* d_slot,
                                   const float* d_local, int tokens, int world, int cap,
                                   int hidden, float* d_out, cudaStream_t stream,
                                   WispErrCtx* err);

/* --------------------------------------------------------------------------
 * 4-bit block-scaled operands ("fp4"): rows of e2m1 values (+-{0, 0.5, 1, 1.5,
 * 2, 3, 4, 6}), two per byte along the row (low nibble = even index), and one
 * scale byte per block of consecutive values. No counterpart in the reference,
 * whose 4-bit format is integer (wisp/converter/quantizer.py:1-17).
 *   WISP_FP4_MX: blocks of 32, scale = 2^(byte - 127) (byte 255: NaN)
 *   WISP_FP4_NV: blocks of 16, scale = e4m3(byte) * tensor_scale, where
 *                tensor_scale is one positive fp32 on the device per matrix
 * Rows are contiguous: cols/2 code bytes and cols/block scale bytes each, at
 * most 2^31 - 256 rows a call.
 * ------------------------------------------------------------------------ */
enum { WISP_FP4_MX = 0, WISP_FP4_NV = 1 };
enum { WISP_DT_F32 = 0, WISP_DT_BF16 = 1, WISP_DT_F16 = 2 };

/* Quantises rows: row p of the result is row d_src[p] of d_x (d_src NULL:
 * row p; an index outside [0, x_rows) gives a row of zeros). d_x has x_rows
 * rows of cols values of x_type, ld elements apart. cols is a multiple of the
 * block. Per block, with a = max|x|:
 *   MX: scale = 2^(floor(log2 a) - 2), at least 2^-127
 *   NV: scale byte = e4m3(a / (6 tensor_scale)) rounded to nearest even and
 *       saturated at 448
 * and each code is the e2m1 value nearest to x / scale (ties to the even
 * code, saturated at 6), decided as if by exact arithmetic. A zero scale
 * gives zero codes; a block holding an infinity or a NaN, or a tensor_scale
 * that is not positive and finite, gives the NaN scale byte and zero codes.
 * d_tensor_scale is not read for MX.
 * rows = 0 is allowed and launches nothing. */
WispError wisp_b200_fp4_quantize(const void* d_x, int x_type, int64_t ld, int x_rows,
                                 const int* d_src, int rows, int cols, int format,
                                 const float* d_tensor_scale, uint8_t* d_codes,
                                 uint8_t* d_scales, cudaStream_t stream, WispErrCtx* err);

/* The values of quantised rows, rounded once to out_type (ld elements
 * between output rows). d_tensor_scale: one fp32 or NULL (1), for NV rows; MX
 * rows have none, and one given for them is refused (here and in
 * wisp_b200_fp4_product). */
WispError wisp_b200_fp4_dequantize(const uint8_t* d_codes, const uint8_t* d_scales, int rows,
                                   int cols, int format, const float* d_tensor_scale, void* d_out,
                                   int out_type, int64_t ld, cudaStream_t stream,
                                   WispErrCtx* err);

/* A set of n_entries matrices [n x k] (one per expert), used by one product. */
typedef struct {
    int format;    /* WISP_FP4_* (weights and rows) */
    int n_entries;
    int n;         /* output features, any n >= 1 */
    int k;         /* multiple of 32 */
    int swiglu;    /* 1: silu(gate x) * up x over two sets, 0: one set */
    int out_type;  /* WISP_DT_* */
} WispFp4Config;

/* codes: [n_entries x n x k/2] contiguous, 16-byte aligned, used where they
 * lie. prepared: from wisp_b200_fp4_prepare over the set's scale bytes.
 * tensor_scale: [n_entries] fp32 or NULL (all 1). */
typedef struct {
    const uint8_t* codes;
    const void* prepared;
    const float* tensor_scale;
} WispFp4Mats;

/* Activation rows from wisp_b200_fp4_quantize; tensor_scale: one fp32 or NULL
 * (1), NULL for MX. codes 16-byte aligned. */
typedef struct {
    const uint8_t* codes;
    const uint8_t* scales;
    const float* tensor_scale;
    int rows;
} WispFp4Rows;

/* One-time layout of a set's scale bytes [n_entries x n x k/block] as the
 * tensor cores take them (128 features x 256 k per run). d_prepared: 256-byte
 * aligned, wisp_b200_fp4_prepared_bytes bytes. */
size_t wisp_b200_fp4_prepared_bytes(const WispFp4Config* cfg);
WispError wisp_b200_fp4_prepare(const WispFp4Config* cfg, const uint8_t* d_scales,
                                void* d_prepared, size_t prepared_bytes, cudaStream_t stream,
                                WispErrCtx* err);

/* out[p, f] = sum_k x[p, k] w_e[f, k] (fp32 accumulation, rounded once to
 * out_type; with swiglu silu(w x) * (up x)) for every row p of every segment,
 * e = the segment's expert. d_segs: DEVICE array of n_segs <= 1025 segments
 * over the rows, which must not overlap; NULL: all rows through entry 0. Rows
 * in no segment are left as they are. A segment whose expert or rows lie
 * outside the set or the rows is skipped and sets bit 2 of *d_error_flag. ld:
 * elements between output rows. up is NULL unless swiglu. d_out overlaps none of the
 * inputs. d_error_flag as for wisp_b200_grouped_ffn (may be NULL; the call
 * does not clear it). rows = 0 is allowed and launches nothing. */
WispError wisp_b200_fp4_product(const WispFp4Config* cfg, const WispFp4Mats* w,
                                const WispFp4Mats* up, const WispFp4Rows* x,
                                const WispSegment* d_segs, int n_segs, void* d_out, int64_t ld,
                                int* d_error_flag, cudaStream_t stream, WispErrCtx* err);

/* The MoE layer of wisp_b200_moe_forward over fp4 experts: route, dispatch
 * plan, quantise the gathered rows, gate/up product with SwiGLU (bf16 rows),
 * quantise, down product (bf16 rows), each token's rows summed in fp32 in a
 * fixed order with the routing weights. d_out 16-byte aligned. gate, up: sets
 * of E (+1 shared) entries [inter x hidden], down: [hidden x inter], all
 * prepared. cfg->group_size, cfg->deterministic are ignored (every run gives
 * the same bits). x_scale,
 * h_scale: the NV tensor scales of the layer's input and of the SwiGLU output
 * (device, from calibration; NULL for MX). */
typedef struct {
    const uint16_t* router_w;  /* as in WispMoeWeights */
    const float* router_bias;
    WispFp4Mats gate, up, down;
    const float* x_scale;
    const float* h_scale;
    int format;
} WispFp4MoeWeights;

size_t wisp_b200_fp4_moe_workspace_bytes(const WispMoeConfig* cfg, int format);
WispError wisp_b200_fp4_moe_forward(const WispMoeConfig* cfg, const WispFp4MoeWeights* w,
                                    const uint16_t* d_x, float* d_out, int* d_topk_idx,
                                    float* d_topk_w, void* d_workspace, size_t workspace_bytes,
                                    int* d_error_flag, cudaStream_t stream, WispErrCtx* err);

/* --------------------------------------------------------------------------
 * 8-bit block-scaled operands ("fp8"): e4m3 values (largest 448, codes 0x7f and
 * 0xff NaN) with fp32 scales, one per 128 consecutive values of an activation
 * row and one per 128 x 128 block of a weight matrix; the last blocks may be
 * shorter. No counterpart in the reference.
 * Code rows are contiguous and 16-byte aligned, their length a multiple of 16, at
 * most 2^27; a call takes at most 2^31 - 256 rows. The scale of row p and block b
 * lies at scales[p * scale_row + b * scale_block] (scale_row = 1 and scale_block =
 * the rows or more suit the product: a block's scales are then read together).
 * ------------------------------------------------------------------------ */

/* Quantises rows: row p of the result is row d_src[p] of d_x (d_src NULL: row p;
 * an index outside [0, x_rows) gives a row of zeros). d_x has x_rows rows of cols
 * values of x_type, ld elements apart. Per block, with a = max|x|:
 *   scale = fp32(a / 448), or with pow2 the least power of two that is not below
 *           a / 448, at least 2^-126; 0 for a = 0
 * and each code is the e4m3 value nearest to x / scale (ties to the even code,
 * saturated at 448), decided as if by exact arithmetic. A zero scale gives zero
 * codes; a block holding an infinity or a NaN gives a NaN scale and zero codes.
 * rows = 0 is allowed and launches nothing. */
WispError wisp_b200_fp8_quantize(const void* d_x, int x_type, int64_t ld, int x_rows,
                                 const int* d_src, int rows, int cols, int pow2,
                                 uint8_t* d_codes, float* d_scales, int64_t scale_row,
                                 int64_t scale_block, cudaStream_t stream, WispErrCtx* err);

/* The values of quantised rows: code * scale in fp32, rounded to out_type (ld
 * elements between output rows). */
WispError wisp_b200_fp8_dequantize(const uint8_t* d_codes, const float* d_scales,
                                   int64_t scale_row, int64_t scale_block, int rows, int cols,
                                   void* d_out, int out_type, int64_t ld, cudaStream_t stream,
                                   WispErrCtx* err);

/* Activation rows from wisp_b200_fp8_quantize. */
typedef struct {
    const uint8_t* codes;
    const float* scales;
    int64_t scale_row, scale_block;
    int rows;
} WispFp8Rows;

/* Copies quantised rows: row p of the result is row d_src[p] of x, codes and scales as
 * they are, or a row of zeros (codes and scales) for an index outside [0, x->rows).
 * What quantising the gathered rows gives, where each row is wanted several times. The
 * result lies nowhere in x. rows = 0 is allowed and launches nothing. */
WispError wisp_b200_fp8_gather(const WispFp8Rows* x, const int* d_src, int rows, int cols,
                               uint8_t* d_codes, float* d_scales, int64_t scale_row,
                               int64_t scale_block, cudaStream_t stream, WispErrCtx* err);

/* Quantises matrices d_w [n_entries x n x k] of w_type (contiguous) to codes of
 * the same shape and scales [n_entries x ceil(n / 128) x ceil(k / 128)], by the
 * rule above over blocks of 128 x 128. At most 65535 matrices and 65535 * 128
 * rows each. */
WispError wisp_b200_fp8_quantize_weights(const void* d_w, int w_type, int n_entries, int n, int k,
                                         uint8_t* d_codes, float* d_scales, cudaStream_t stream,
                                         WispErrCtx* err);

/* A set of n_entries matrices [n x k] (one per expert), used by one product. */
typedef struct {
    int n_entries;
    int n;         /* output features, any n >= 1 */
    int k;         /* multiple of 16, at most 2^27 */
    int swiglu;    /* 1: silu(gate x) * up x over two sets, 0: one set */
    int out_type;  /* WISP_DT_* */
} WispFp8Config;

/* codes [n_entries x n x k], 16-byte aligned; scales [n_entries x ceil(n / 128) x
 * ceil(k / 128)]. Both contiguous and used where they lie. */
typedef struct {
    const uint8_t* codes;
    const float* scales;
} WispFp8Mats;

/* out[p, f] = sum_k x[p, k] w_e[f, k] for every row p of every segment, e = the
 * segment's expert (with swiglu silu(w x) * (up x)). Each block of 128 k is summed
 * on the tensor cores in fp32, scaled by the product of its two scales (in fp32, whose
 * range that product has to stay in) and added up in fp32; the sum is rounded once to
 * out_type. d_segs, n_segs, ld, up, the rows in no segment
 * and d_error_flag as for wisp_b200_fp4_product. rows = 0 is allowed and launches
 * nothing. */
WispError wisp_b200_fp8_product(const WispFp8Config* cfg, const WispFp8Mats* w,
                                const WispFp8Mats* up, const WispFp8Rows* x,
                                const WispSegment* d_segs, int n_segs, void* d_out, int64_t ld,
                                int* d_error_flag, cudaStream_t stream, WispErrCtx* err);

/* --------------------------------------------------------------------------
 * Routing from logits, with a bias for balance.
 *   score  = softmax(logits) over the token's experts, or sigmoid(logit)
 *   choice = score + bias                     (the bias chooses, it does not weigh)
 *   of n_groups groups of consecutive experts the topk_groups best are kept, by the
 *   sum of their group_top largest choices; of the kept groups' experts the top_k
 *   of largest choice are taken, in that order
 *   weight = score (renormalize: / the sum over the token's top_k) * scaling
 * Scores, choices and weights are computed in fp64 and the weights rounded once;
 * equal choices go to the lower expert, equal groups to the lower group. An expert
 * whose choice is NaN or -infinity is never taken and adds nothing to its group's
 * sum (a NaN or +infinite logit makes all of a token's softmax scores NaN); where
 * fewer than top_k are left, the remaining slots have index -1 and weight 0, which
 * wisp_b200_dispatch_plan routes nowhere. (wisp_b200_route, whose bias enters before
 * the scores, is the other form.)
 * ------------------------------------------------------------------------ */
enum { WISP_ROUTE_SOFTMAX = 0, WISP_ROUTE_SIGMOID = 1 };

typedef struct {
    int scoring;        /* WISP_ROUTE_* */
    int n_groups;       /* 1..32, n_experts % n_groups == 0 */
    int topk_groups;    /* 1..n_groups */
    int group_top;      /* 1 or 2 */
    int renormalize;
    float scaling;
} WispRouting;

/* d_logits: tokens rows of n_experts (<= 1024) values of logits_type, ld elements
 * apart. d_bias: fp32 [n_experts] or NULL. d_idx, d_w: [tokens x top_k], top_k <=
 * min(32, the kept groups' experts). tokens = 0 is allowed and launches nothing. */
WispError wisp_b200_select_experts(const WispRouting* routing, const void* d_logits,
                                   int logits_type, int64_t ld, int tokens, int n_experts,
                                   int top_k, const float* d_bias, int* d_idx, float* d_w,
                                   cudaStream_t stream, WispErrCtx* err);

/* The MoE layer of wisp_b200_moe_forward over fp8 experts: route, dispatch plan,
 * quantise the rows, gate/up product with SwiGLU (bf16 rows), quantise, down
 * product (bf16 rows), each token's rows summed in fp32 in a fixed order with the
 * routing weights. gate, up: sets of E (+1 shared) entries [inter x hidden], down:
 * [hidden x inter]. routing NULL: cfg's scoring, as the other layers route; else
 * the logits (router_bias added) are routed as wisp_b200_select_experts does, with
 * score_bias as its bias, and cfg's scoring, n_groups, topk_groups and
 * routed_scaling are ignored, as group_size and deterministic always are (every run
 * gives the same bits). d_x, router_w and d_out 16-byte aligned, the workspace
 * 256-byte, the other arrays to their types: what the layer refuses, it refuses before it
 * launches anything. One call at a time per workspace. */
typedef struct {
    const uint16_t* router_w;   /* as in WispMoeWeights */
    const float* router_bias;   /* added to the logits; may be NULL */
    const float* score_bias;    /* added to the scores for the choice; may be NULL */
    WispFp8Mats gate, up, down;
    int pow2;                   /* scales of the quantised rows are powers of two */
} WispFp8MoeWeights;

size_t wisp_b200_fp8_moe_workspace_bytes(const WispMoeConfig* cfg, const WispRouting* routing);
WispError wisp_b200_fp8_moe_forward(const WispMoeConfig* cfg, const WispRouting* routing,
                                    const WispFp8MoeWeights* w, const uint16_t* d_x, float* d_out,
                                    int* d_topk_idx, float* d_topk_w, void* d_workspace,
                                    size_t workspace_bytes, int* d_error_flag,
                                    cudaStream_t stream, WispErrCtx* err);

/* --------------------------------------------------------------------------
 * Norms around a block, with its gate and its residual (the reference runs
 * them as op_rmsnorm, op_residual and op_rmsnorm over fp32,
 * csrc/core/wisp_engine.c:1715-1722):
 *   p  = post_norm ? y / rms(y) * (weight_offset + post_w) : y
 *   x' = residual_scale * x + gate * p          (without y: x' = x)
 *   n  = x' / rms(x') * (weight_offset + pre_w) (when d_n is not NULL)
 * rms(v) = sqrt(mean(v^2) + eps). All in fp32; n is taken from x' before x'
 * is rounded to x_type, so each output is rounded once.
 * ------------------------------------------------------------------------ */
enum { WISP_GATE_NONE = 0, WISP_GATE_CHANNEL = 1, WISP_GATE_TOKEN = 2, WISP_GATE_ELEMENT = 3 };

typedef struct {
    int tokens;            /* at most 2^31 - 256; 0 allowed: launches nothing */
    int hidden;            /* 1 .. 32768 */
    int x_type, y_type;    /* WISP_DT_*: residual stream, block output */
    int w_type, gate_type; /* norm weights, gate */
    int n_type;            /* normalised output */
    int post_norm;         /* 0: y enters without a norm */
    int gate_kind;         /* WISP_GATE_*: [hidden], [tokens] or [tokens x hidden] */
    float residual_scale;
    float eps;             /* >= 0 */
    float weight_offset;   /* 0, or 1 for weights stored around 0 */
    int64_t ld_x, ld_y, ld_gate, ld_x_out, ld_n; /* elements between rows */
} WispBlockNorm;

/* d_y NULL: no block output (d_x_out, if given, is left as it is). d_post_w /
 * d_pre_w NULL: ones. d_x_out NULL: x' is not stored; it may equal d_x (with
 * the same row stride). d_n NULL: no norm after. No other buffers may overlap. */
WispError wisp_b200_block_norm(const WispBlockNorm* cfg, const void* d_x, const void* d_y,
                               const void* d_gate, const void* d_post_w, const void* d_pre_w,
                               void* d_x_out, void* d_n, cudaStream_t stream, WispErrCtx* err);

/* Device error word of wisp_b200_block_norm on the current device, for
 * wisp_b200_check_error_flag: set when a wait for a row gave up (that row and
 * some after it are then NaN); cleared by nobody but its reader. NULL without a
 * device. */
int* wisp_b200_block_norm_error_word(void);

/* Between stacked layers: d_out[t] = bf16(d_in[t] / rms(d_in[t])), fp32 in. */
WispError wisp_b200_rms_rescale(const float* d_in, uint16_t* d_out, int tokens, int hidden,
                                float eps, cudaStream_t stream, WispErrCtx* err);

/* Copy bf16 rows into fp16 interleaved-K rows: xp[p] = x[src[p]] for
 * p < n_rows (src may be NULL: identity). */
WispError wisp_b200_pack_rows(const uint16_t* d_x, const int* d_src, int n_rows, int hidden,
                              uint16_t* d_xp, cudaStream_t stream, WispErrCtx* err);

/* Device error word, of two bits that kernels set beside what the word holds.
 * 1: a bounded wait gave up (the results of that launch are invalid), reported
 * as WISP_ERR_TIMEOUT whatever else is set. 2, from wisp_b200_fp4_product and
 * wisp_b200_fp8_product: a segment was skipped, WISP_ERR_INVALID_ARG. The word is not cleared
 * here. */
WispError wisp_b200_check_error_flag(const int* d_error_flag, cudaStream_t stream,
                                     WispErrCtx* err);

/* Address of the device error word inside a wisp_b200_moe_forward
 * workspace (cleared at the start of every forward). */
int* wisp_b200_moe_error_word(const WispMoeConfig* cfg, void* d_workspace);

/* Diagnostics: when d_counters (38 uint64, zeroed by the caller) is
 * non-NULL, the grouped kernels accumulate the clock cycles each role spends
 * in each of its waits: the tensor-core gate/up kernel in [0,15), its down
 * kernel in [15,30), the register-path gate/up kernel in [30,34) and its
 * down kernel in [34,38). Pass NULL to switch off. Not thread-safe; for
 * profiling runs only. */
void wisp_b200_debug_set_counters(unsigned long long* d_counters);

/* Largest segment (rows) routed to the register-fed kernel, which takes any
 * segment in chunks of 16 rows; 0 sends every segment to the tcgen05 kernel,
 * a negative value restores the default. Process-wide; for tests and
 * tuning. */
void wisp_b200_set_skinny_max_rows(int rows);

/* Library version string. */
const char* wisp_b200_version(void);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif

#endif /* WISP_B200_H */
