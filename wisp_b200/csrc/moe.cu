// moe.cu -- host orchestration of the batched MoE layer and the small
// host-side pieces of the ABI (blob header parsing, error word, version).
//
// wisp_b200_moe_forward runs, on one stream and without any host sync:
//   route (logits + top-k) -> dispatch plan (segments, row -> token map)
//   -> pack rows (q16 rows for register-path segments, fp16 interleaved
//      rows for tensor-core ones) -> zero out
//   -> grouped gate/up + SwiGLU -> grouped down + weighted scatter-combine
//      (fp32 atomics into out), each on the register-path kernel for
//      segments of up to 32 rows and on the tcgen05 kernel for larger ones.
// Decode batches of at most 4 tokens take a shorter chain: router logits,
// one planner launch (top-k, plan, q16 rows, zeroing, unit plans), then the
// register-path gate/up and down launches.
// It is the batched counterpart of run_moe (csrc/core/wisp_engine.c:
// 1563-1674), which the reference can only run one token at a time.
#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace wb {
size_t router_splits(int T, int E, int M);
int launch_logits(const WispMoeConfig* c, const uint16_t* x, const uint16_t* W, float* part,
                  size_t splits, cudaStream_t st);
WispError launch_route(const WispMoeConfig* c, const uint16_t* x, const uint16_t* W,
                       const float* bias, float* part, size_t splits, float* logits_out, int* idx,
                       float* w, cudaStream_t st, WispErrCtx* err);
WispError launch_plan(const WispMoeConfig* c, const int* idx, const float* w, int* counts,
                      WispSegment* segs, int* row_token, float* row_weight, cudaStream_t st,
                      WispErrCtx* err, int* scratch);
size_t plan_scratch_ints(const WispMoeConfig* c);
WispError launch_pack(const uint16_t* x, const int* src, int n_rows, int M, uint16_t* xp,
                      cudaStream_t st, WispErrCtx* err);
WispError launch_pack_q16(const uint16_t* x, const int* src, int n_rows, int M, uint16_t* xp,
                          uint8_t* xq, const WispSegment* segs, int nseg, int sk_rows,
                          cudaStream_t st, WispErrCtx* err);
int grouped_sk_rows(int n_segs, int n_entries);
uint8_t* grouped_xq(void* d_workspace, int n_segs, int rows_capacity, int M, int I);
WispError grouped_ffn_impl(const WispMoeConfig* cfg, const void* d_prepared,
                           const WispInt4Expert* d_experts, int n_entries,
                           const WispSegment* d_segs, int n_segs, int rows_capacity,
                           const uint16_t* d_xp, uint16_t* d_h, int mode, const int* d_row_token,
                           const float* d_row_weight, float* d_out, void* d_workspace,
                           size_t workspace_bytes, int* d_error_flag, bool xq_ready,
                           int max_seg_rows, cudaStream_t stream, WispErrCtx* err,
                           bool plans_ready = false);
void decode_units(const WispMoeConfig* cfg, int n_segs, int n_entries, int rows_capacity, int mode,
                  void* d_workspace, DecodeUnits* du);
WispError launch_router_gemv(const WispMoeConfig* c, const uint16_t* x, const uint16_t* W,
                             float* logits, cudaStream_t st, WispErrCtx* err);
bool decode_plan_fits(const WispMoeConfig* c, int sk_rows);
WispError launch_decode_plan(const WispMoeConfig* c, const float* logits, const float* bias,
                             int* idx, float* w, int* counts, WispSegment* segs, int* row_token,
                             float* row_weight, const uint16_t* x, float* out, int* error_flag,
                             const DecodeUnits& du, cudaStream_t st, WispErrCtx* err);
}  // namespace wb

namespace {

struct Carve {
  size_t off = 0;
  template <typename T>
  T* take(void* base, size_t count) {
    off = (off + 255) & ~(size_t)255;
    T* p = base ? reinterpret_cast<T*>(static_cast<uint8_t*>(base) + off) : nullptr;
    off += count * sizeof(T);
    return p;
  }
};

struct Workspace {
  float* part;
  int* plan_scratch;
  int* idx;
  float* w;
  int* counts;
  WispSegment* segs;
  int* row_token;
  float* row_weight;
  void* grouped;
  size_t grouped_bytes;
  int* error_flag;
  uint16_t* xp;
  uint16_t* h;
  // deterministic layers only: the expert outputs, one fp32 row per routed
  // row, and each token's rows
  float* y;
  int* tok_cnt;
  int* tok_list;
  int lanes;   // rows per token: top_k (+ 1 with a shared expert)
  size_t bytes;
  size_t splits;
  int rows;
};

Workspace carve(const WispMoeConfig* c, void* base) {
  Workspace ws;
  Carve cv;
  const int T = c->tokens, E = c->n_experts, k = c->top_k, M = c->hidden, I = c->inter;
  const int V = E + (c->has_shared ? 1 : 0);
  ws.rows = T * k + (c->has_shared ? T : 0);
  ws.splits = wb::router_splits(T, E, M);
  ws.part = cv.take<float>(base, ws.splits * (size_t)T * E);
  ws.plan_scratch = cv.take<int>(base, std::max<size_t>(1, wb::plan_scratch_ints(c)));
  ws.idx = cv.take<int>(base, (size_t)T * k);
  ws.w = cv.take<float>(base, (size_t)T * k);
  ws.counts = cv.take<int>(base, V);
  ws.segs = cv.take<WispSegment>(base, V);
  ws.row_token = cv.take<int>(base, ws.rows);
  ws.row_weight = cv.take<float>(base, ws.rows);
  ws.grouped_bytes = wisp_b200_grouped_workspace_bytes(c, V, ws.rows);
  ws.grouped = cv.take<uint8_t>(base, ws.grouped_bytes);
  ws.error_flag = cv.take<int>(base, 1);
  ws.xp = cv.take<uint16_t>(base, (size_t)ws.rows * M);
  ws.h = cv.take<uint16_t>(base, (size_t)ws.rows * I);
  ws.lanes = k + (c->has_shared ? 1 : 0);
  ws.y = nullptr;
  ws.tok_cnt = ws.tok_list = nullptr;
  if (c->deterministic) {
    ws.y = cv.take<float>(base, (size_t)ws.rows * M);
    ws.tok_cnt = cv.take<int>(base, T);
    ws.tok_list = cv.take<int>(base, (size_t)T * ws.lanes);
  }
  ws.bytes = (cv.off + 255) & ~(size_t)255;
  return ws;
}

// Deterministic combine (WispMoeConfig.deterministic). The expert outputs
// arrive as plain fp32 rows (grouped FFN mode 1: no weights, no atomics, no
// K split of the down projection); each token's output is then the sum of
// its rows in ascending row order -- routed experts by index, then the
// shared expert -- so every run produces the same bits, where the atomics
// of the fused combine add in whatever order the hardware picks.
// Step 1: each token's rows into a per-token list (in any order).
__global__ void token_rows_kernel(const int* __restrict__ row_token,
                                  const WispSegment* __restrict__ segs, int V, int cap, int lanes,
                                  int* __restrict__ cnt, int* __restrict__ list) {
  const int total = min(cap, segs[V - 1].row_begin + segs[V - 1].rows);
  for (int p = blockIdx.x * blockDim.x + threadIdx.x; p < total; p += gridDim.x * blockDim.x) {
    const int t = row_token[p];
    const int j = atomicAdd(cnt + t, 1);
    if (j < lanes) list[(size_t)t * lanes + j] = p;
  }
}

// Step 2: one block per (token, 1024 columns): the token's rows sorted by
// position, then out[t][m] = sum over them, in that order, of weight * y.
constexpr int kDetMaxLanes = 64;
__global__ void combine_ordered_kernel(const float* __restrict__ y,
                                       const float* __restrict__ row_weight,
                                       const int* __restrict__ cnt, const int* __restrict__ list,
                                       int lanes, int M, float* __restrict__ out) {
  __shared__ int s_p[kDetMaxLanes];
  __shared__ float s_w[kDetMaxLanes];
  __shared__ int s_n;
  const int t = blockIdx.x;
  if (threadIdx.x == 0) {
    const int n = min(cnt[t], lanes);
    for (int i = 0; i < n; i++) {   // insertion sort of at most 33 positions
      const int v = list[(size_t)t * lanes + i];
      int j = i;
      while (j > 0 && s_p[j - 1] > v) {
        s_p[j] = s_p[j - 1];
        j--;
      }
      s_p[j] = v;
    }
    for (int i = 0; i < n; i++) s_w[i] = row_weight[s_p[i]];
    s_n = n;
  }
  __syncthreads();
  const int n = s_n;
  const int m1 = min(M, (int)(blockIdx.y + 1) * 1024);
  for (int m = (int)blockIdx.y * 1024 + threadIdx.x; m < m1; m += blockDim.x) {
    float acc = 0.f;
    for (int i = 0; i < n; i++) acc = fmaf(s_w[i], y[(size_t)s_p[i] * M + m], acc);
    out[(size_t)t * M + m] = acc;
  }
}

WispError validate(const WispMoeConfig* c, WispErrCtx* err) {
  if (!c) return WB_FAIL(WISP_ERR_INVALID_ARG, "moe: null config");
  if (c->tokens <= 0 || c->n_experts <= 0 || c->n_experts > 1024)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "moe: tokens=%d n_experts=%d (1..1024)", c->tokens, c->n_experts);
  if (c->top_k <= 0 || c->top_k > 32 || c->top_k > c->n_experts)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "moe: top_k=%d (1..min(32, n_experts))", c->top_k);
  if (c->hidden <= 0 || c->inter <= 0 || c->hidden % 128 || c->inter % 128)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "moe: hidden=%d inter=%d must be multiples of 128", c->hidden, c->inter);
  if (c->group_size != 64 && c->group_size != 128)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "moe: group_size=%d (64 or 128)", c->group_size);
  if (c->scoring == WISP_SCORE_SIGMOID_GROUPED) {
    if (c->n_groups <= 0 || c->n_groups > 32 || c->n_experts % c->n_groups ||
        c->topk_groups <= 0 || c->topk_groups > c->n_groups ||
        c->top_k > c->topk_groups * (c->n_experts / c->n_groups))
      return WB_FAIL(WISP_ERR_INVALID_ARG, "moe: bad group routing (E=%d groups=%d keep=%d k=%d)",
                     c->n_experts, c->n_groups, c->topk_groups, c->top_k);
  } else if (c->scoring != WISP_SCORE_SOFTMAX) {
    return WB_FAIL(WISP_ERR_INVALID_ARG, "moe: unknown scoring %d", c->scoring);
  }
  return WISP_OK;
}

}  // namespace

extern "C" size_t wisp_b200_moe_workspace_bytes(const WispMoeConfig* cfg) {
  if (validate(cfg, nullptr) != WISP_OK) return 0;
  return carve(cfg, nullptr).bytes;
}

extern "C" WispError wisp_b200_route(const WispMoeConfig* cfg, const WispMoeWeights* w,
                                     const uint16_t* d_x, float* d_logits, int* d_idx, float* d_w,
                                     cudaStream_t stream, WispErrCtx* err) {
  WispError e = validate(cfg, err);
  if (e != WISP_OK) return e;
  if (!w || !w->router_w || !d_x || !d_logits || !d_idx || !d_w)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "route: null pointer argument");
  // d_logits serves as the (single-split) partial buffer and then receives
  // the final logits (bias included); each token's row is read before it
  // is rewritten by the same thread.
  return wb::launch_route(cfg, d_x, w->router_w, w->router_bias, d_logits, 1, d_logits, d_idx, d_w,
                          stream, err);
}

namespace {
// wisp_b200_route_ws workspace: the split partial sums.
size_t route_part_bytes(const WispMoeConfig* cfg) {
  const size_t n = wb::router_splits(cfg->tokens, cfg->n_experts, cfg->hidden) *
                   (size_t)cfg->tokens * cfg->n_experts * sizeof(float);
  return (n + 255) & ~(size_t)255;
}
}  // namespace

extern "C" size_t wisp_b200_route_workspace_bytes(const WispMoeConfig* cfg) {
  if (validate(cfg, nullptr) != WISP_OK) return 0;
  return route_part_bytes(cfg);
}

extern "C" WispError wisp_b200_route_ws(const WispMoeConfig* cfg, const WispMoeWeights* w,
                                        const uint16_t* d_x, float* d_logits, int* d_idx,
                                        float* d_w, void* d_workspace, size_t workspace_bytes,
                                        cudaStream_t stream, WispErrCtx* err) {
  WispError e = validate(cfg, err);
  if (e != WISP_OK) return e;
  if (!w || !w->router_w || !d_x || !d_idx || !d_w || !d_workspace)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "route_ws: null pointer argument");
  const size_t splits = wb::router_splits(cfg->tokens, cfg->n_experts, cfg->hidden);
  const size_t need = wisp_b200_route_workspace_bytes(cfg);
  if (workspace_bytes < need)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "route_ws: workspace %zu < required %zu", workspace_bytes,
                   need);
  if (((uintptr_t)d_x | (uintptr_t)w->router_w | (uintptr_t)d_workspace) & 15)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "route_ws: x, router_w and workspace must be 16-byte aligned");
  return wb::launch_route(cfg, d_x, w->router_w, w->router_bias, static_cast<float*>(d_workspace),
                          splits, d_logits, d_idx, d_w, stream, err);
}

extern "C" WispError wisp_b200_moe_forward(const WispMoeConfig* cfg, const WispMoeWeights* w,
                                           const uint16_t* d_x, float* d_out, int* d_topk_idx,
                                           float* d_topk_w, void* d_workspace,
                                           size_t workspace_bytes, cudaStream_t stream,
                                           WispErrCtx* err) {
  WispError e = validate(cfg, err);
  if (e != WISP_OK) return e;
  if (!w || !w->router_w || !w->prepared || !d_x || !d_out || !d_workspace)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "moe_forward: null pointer argument (router_w, prepared, x, out, workspace)");
  if (((uintptr_t)d_x | (uintptr_t)w->router_w | (uintptr_t)d_workspace) & 15)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "moe_forward: x, router_w and workspace must be 16-byte aligned");
  Workspace ws = carve(cfg, d_workspace);
  if (workspace_bytes < ws.bytes)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "moe_forward: workspace %zu < required %zu", workspace_bytes, ws.bytes);
  int* idx = d_topk_idx ? d_topk_idx : ws.idx;
  float* wt = d_topk_w ? d_topk_w : ws.w;
  const int V = cfg->n_experts + (cfg->has_shared ? 1 : 0);
  if (!w->experts) return WB_FAIL(WISP_ERR_INVALID_ARG, "moe_forward: null expert table");

  // Decode batches (T <= 4): router logits, then one planner launch for
  // top-k, dispatch plan, q16 rows, output zeroing and the register path's
  // unit plans, then the register-path gate/up and down launches.
  const bool det = cfg->deterministic != 0;
  if (!det && wb::decode_plan_fits(cfg, wb::grouped_sk_rows(V, V))) {
    // ws.part holds splits * T * E floats, splits >= 1: room for the logits
    e = wb::launch_router_gemv(cfg, d_x, w->router_w, ws.part, stream, err);
    if (e != WISP_OK) return e;
    wb::DecodeUnits du;
    wb::decode_units(cfg, V, V, ws.rows, 0, ws.grouped, &du);
    e = wb::launch_decode_plan(cfg, ws.part, w->router_bias, idx, wt, ws.counts, ws.segs,
                               ws.row_token, ws.row_weight, d_x, d_out, ws.error_flag, du, stream,
                               err);
    if (e != WISP_OK) return e;
    return wb::grouped_ffn_impl(cfg, w->prepared, w->experts, V, ws.segs, V, ws.rows, ws.xp, ws.h,
                                0, ws.row_token, ws.row_weight, d_out, ws.grouped,
                                ws.grouped_bytes, ws.error_flag, true, cfg->tokens, stream, err,
                                true);
  }

  e = wb::launch_route(cfg, d_x, w->router_w, w->router_bias, ws.part, ws.splits, nullptr, idx, wt,
                       stream, err);
  if (e != WISP_OK) return e;
  e = wb::launch_plan(cfg, idx, wt, ws.counts, ws.segs, ws.row_token, ws.row_weight, stream, err,
                      ws.plan_scratch);
  if (e != WISP_OK) return e;
  // The gathered rows in the operand form of the kernel their segment runs
  // on: fp16 for the tensor-core kernel, q16 (into the grouped workspace) for
  // the register path.
  e = wb::launch_pack_q16(d_x, ws.row_token, ws.rows, cfg->hidden, ws.xp,
                          wb::grouped_xq(ws.grouped, V, ws.rows, cfg->hidden, cfg->inter), ws.segs,
                          V, wb::grouped_sk_rows(V, V), stream, err);
  if (e != WISP_OK) return e;
  WB_CUDA_CHECK(cudaMemsetAsync(ws.error_flag, 0, sizeof(int), stream));
  if (det) {
    // expert outputs as rows, then the fixed-order combine
    e = wb::grouped_ffn_impl(cfg, w->prepared, w->experts, V, ws.segs, V, ws.rows, ws.xp, ws.h, 1,
                             ws.row_token, ws.row_weight, ws.y, ws.grouped, ws.grouped_bytes,
                             ws.error_flag, true, cfg->tokens, stream, err);
    if (e != WISP_OK) return e;
    WB_CUDA_CHECK(cudaMemsetAsync(ws.tok_cnt, 0, (size_t)cfg->tokens * sizeof(int), stream));
    wb::launch_k(token_rows_kernel, (ws.rows + 255) / 256, 256, 0, stream, ws.row_token, ws.segs, V,
                 ws.rows, ws.lanes, ws.tok_cnt, ws.tok_list);
    wb::launch_k(combine_ordered_kernel, dim3(cfg->tokens, (cfg->hidden + 1023) / 1024), 256, 0,
                 stream, ws.y, ws.row_weight, ws.tok_cnt, ws.tok_list, ws.lanes, cfg->hidden, d_out);
    WB_CUDA_CHECK(cudaGetLastError());
    return WISP_OK;
  }
  WB_CUDA_CHECK(cudaMemsetAsync(d_out, 0, (size_t)cfg->tokens * cfg->hidden * sizeof(float), stream));
  // A routed expert gets at most one row per token and the shared expert T
  // rows, so no segment exceeds T rows.
  return wb::grouped_ffn_impl(cfg, w->prepared, w->experts, V, ws.segs, V, ws.rows, ws.xp, ws.h, 0,
                              ws.row_token, ws.row_weight, d_out, ws.grouped, ws.grouped_bytes,
                              ws.error_flag, true, cfg->tokens, stream, err);
}

// ---------------------------------------------------------------------------
// Dense int4 MLP: the MLP as the one segment of a one-entry weight set, run
// through the grouped kernels in mode 1 (plain fp32 row stores, no weights,
// no atomics). The reference runs this MLP in fp16 through op_swiglu_ffn +
// op_gemv (csrc/core/wisp_engine.c:1676-1686).
// ---------------------------------------------------------------------------
namespace {

__global__ void one_segment_kernel(WispSegment* s, int rows) {
  WispSegment v;
  v.expert = 0;
  v.row_begin = 0;
  v.rows = rows;
  v.reserved = 0;
  *s = v;
}

struct DenseWs {
  WispSegment* seg;
  void* grouped;
  size_t grouped_bytes;
  uint16_t* xp;
  uint16_t* h;
  size_t bytes;
};

DenseWs carve_dense(const WispMoeConfig* c, void* base) {
  DenseWs ws;
  Carve cv;
  const int T = c->tokens;
  ws.seg = cv.take<WispSegment>(base, 1);
  ws.grouped_bytes = wisp_b200_grouped_workspace_bytes(c, 1, T);
  ws.grouped = cv.take<uint8_t>(base, ws.grouped_bytes);
  ws.xp = cv.take<uint16_t>(base, (size_t)T * c->hidden);
  ws.h = cv.take<uint16_t>(base, (size_t)T * c->inter);
  ws.bytes = (cv.off + 255) & ~(size_t)255;
  return ws;
}

WispError validate_dense(const WispMoeConfig* c, WispErrCtx* err) {
  if (!c) return WB_FAIL(WISP_ERR_INVALID_ARG, "dense_mlp: null config");
  if (c->tokens <= 0 || c->hidden <= 0 || c->inter <= 0 || c->hidden % 128 || c->inter % 128)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "dense_mlp: tokens=%d hidden=%d inter=%d (hidden, inter multiples of 128)",
                   c->tokens, c->hidden, c->inter);
  if (c->group_size != 64 && c->group_size != 128)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "dense_mlp: group_size=%d (64 or 128)", c->group_size);
  return WISP_OK;
}

}  // namespace

extern "C" size_t wisp_b200_dense_mlp_workspace_bytes(const WispMoeConfig* cfg) {
  if (validate_dense(cfg, nullptr) != WISP_OK) return 0;
  return carve_dense(cfg, nullptr).bytes;
}

extern "C" WispError wisp_b200_dense_mlp(const WispMoeConfig* cfg, const void* d_prepared,
                                         const WispInt4Expert* d_mlp, const uint16_t* d_x,
                                         float* d_out, void* d_workspace, size_t workspace_bytes,
                                         int* d_error_flag, cudaStream_t stream, WispErrCtx* err) {
  WispError e = validate_dense(cfg, err);
  if (e != WISP_OK) return e;
  if (!d_prepared || !d_mlp || !d_x || !d_out || !d_workspace)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "dense_mlp: null pointer argument");
  if (((uintptr_t)d_x | (uintptr_t)d_workspace) & 15)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "dense_mlp: x and workspace must be 16-byte aligned");
  const DenseWs ws = carve_dense(cfg, d_workspace);
  if (workspace_bytes < ws.bytes)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "dense_mlp: workspace %zu < required %zu",
                   workspace_bytes, ws.bytes);
  const int T = cfg->tokens;
  one_segment_kernel<<<1, 1, 0, stream>>>(ws.seg, T);
  WB_CUDA_CHECK(cudaGetLastError());
  e = wb::launch_pack_q16(d_x, nullptr, T, cfg->hidden, ws.xp,
                          wb::grouped_xq(ws.grouped, 1, T, cfg->hidden, cfg->inter), ws.seg, 1,
                          wb::grouped_sk_rows(1, 1), stream, err);
  if (e != WISP_OK) return e;
  return wb::grouped_ffn_impl(cfg, d_prepared, d_mlp, 1, ws.seg, 1, T, ws.xp, ws.h, 1, nullptr,
                              nullptr, d_out, ws.grouped, ws.grouped_bytes, d_error_flag, true, T,
                              stream, err);
}

// ---------------------------------------------------------------------------
// The same layer over fp4 experts: route and dispatch plan as above, then the
// products of fp4_product.cu with the rows quantised before each, and a
// fixed-order combine.
// ---------------------------------------------------------------------------
namespace {

// out[t] = sum over the token's rows, in ascending row order, of weight * y: the
// fixed order of combine_ordered_kernel over bf16 rows. (fp32 rows would double
// the traffic of the down product's output and of this sum, 2.1 GB of 2.9 at
// 4096 tokens; one rounding of 2^-9 per expert's output is a fiftieth of what
// its 4-bit operands cost. Of 8-bit ones it is a 26th: normal values through an
// expert of 2 x 2048 x 7168 are 4.3 % off by quantising both its inputs to e4m3, 0.17 %
// by the rounding; with the SwiGLU rows in bf16 too 4.33 % in place of 4.32.)
// One block per token and 2048 columns, 8 per thread.
// SCAN: the token's rows are found by reading all of row_token, else they come
// from token_rows_kernel.
constexpr int kScanRows = 1024;
template <bool SCAN>
__global__ void __launch_bounds__(256)
combine_bf16_kernel(const uint16_t* __restrict__ y, const float* __restrict__ row_weight,
                    const int* __restrict__ row_token, const WispSegment* __restrict__ segs, int V,
                    int cap, const int* __restrict__ cnt, const int* __restrict__ list, int lanes,
                    int M, float* __restrict__ out) {
  __shared__ int s_n, s_any[kDetMaxLanes], s_p[kDetMaxLanes];
  __shared__ float s_w[kDetMaxLanes];
  const int t = blockIdx.x, tid = threadIdx.x;
  if (SCAN) {
    if (tid == 0) s_n = 0;
    __syncthreads();
    const int total = min(cap, segs[V - 1].row_begin + segs[V - 1].rows);
    for (int p = tid; p < total; p += 256)
      if (row_token[p] == t) {
        const int j = atomicAdd(&s_n, 1);
        if (j < lanes) s_any[j] = p;
      }
  } else {
    if (tid == 0) s_n = cnt[t];
    if (tid < lanes) s_any[tid] = list[(size_t)t * lanes + tid];
  }
  __syncthreads();
  const int n = min(s_n, lanes);
  if (tid < n) {
    int rank = 0;
    for (int i = 0; i < n; i++) rank += s_any[i] < s_any[tid];
    s_p[rank] = s_any[tid];
    s_w[rank] = row_weight[s_any[tid]];
  }
  __syncthreads();
  const int m = (blockIdx.y * 256 + tid) * 8;
  if (m >= M) return;
  float acc[8] = {};
  for (int i0 = 0; i0 < n; i0 += 4) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i0 + i < n) v[i] = __ldg(reinterpret_cast<const uint4*>(y + (size_t)s_p[i0 + i] * M + m));
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (i0 + i < n) {
        const float w = s_w[i0 + i];
        const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
          acc[2 * j] = fmaf(w, __uint_as_float(u[j] << 16), acc[2 * j]);
          acc[2 * j + 1] = fmaf(w, __uint_as_float(u[j] & 0xffff0000u), acc[2 * j + 1]);
        }
      }
    }
  }
  float4* o = reinterpret_cast<float4*>(out + (size_t)t * M + m);
  o[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  o[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
}

// Each token's bf16 expert outputs summed with their weights.
WispError combine_bf16(const Workspace& b, const uint16_t* y, int V, int T, int M, float* out,
                       cudaStream_t stream, WispErrCtx* err) {
  const dim3 grid(T, (M + 2047) / 2048);
  if (b.rows <= kScanRows) {
    wb::launch_k(combine_bf16_kernel<true>, grid, 256, 0, stream, y, b.row_weight, b.row_token,
                 b.segs, V, b.rows, nullptr, nullptr, b.lanes, M, out);
  } else {
    WB_CUDA_CHECK(cudaMemsetAsync(b.tok_cnt, 0, (size_t)T * sizeof(int), stream));
    wb::launch_k(token_rows_kernel, (b.rows + 255) / 256, 256, 0, stream, b.row_token, b.segs, V,
                 b.rows, b.lanes, b.tok_cnt, b.tok_list);
    wb::launch_k(combine_bf16_kernel<false>, grid, 256, 0, stream, y, b.row_weight, b.row_token,
                 b.segs, V, b.rows, b.tok_cnt, b.tok_list, b.lanes, M, out);
  }
  WB_CUDA_CHECK(cudaGetLastError());
  return WISP_OK;
}

// dst row p = src row row_token[p], for quantised rows: codes in 16-byte and
// scales in 4-byte words. A token without a valid logit is routed nowhere, so
// the plan may fill fewer rows than there are; what row_token holds behind them
// is no index.
__global__ void __launch_bounds__(256)
gather_fp4_kernel(const uint4* __restrict__ codes, const uint32_t* __restrict__ scales,
                  const int* __restrict__ row_token, int tokens, int code_words, int scale_words,
                  uint4* __restrict__ out_codes, uint32_t* __restrict__ out_scales) {
  const size_t p = blockIdx.x;
  const int src = row_token[p];
  if (src < 0 || src >= tokens) return;
  const size_t t = src;
  for (int i = threadIdx.x; i < code_words; i += 256)
    out_codes[p * code_words + i] = __ldg(codes + t * code_words + i);
  for (int i = threadIdx.x; i < scale_words; i += 256)
    out_scales[p * scale_words + i] = __ldg(scales + t * scale_words + i);
}

// Rows from which the layer quantises its tokens once and copies the codes to
// their rows, instead of quantising every row (36,864 rows of 4096 tokens: 72
// us MX, 99 NV against 40): one launch more.
constexpr int kGatherRows = 2048;

struct Fp4Ws {
  Workspace base;      // routing, plan, token lists
  float* part;
  uint16_t* y;         // bf16 expert outputs
  uint8_t* tc;         // the tokens' codes and scales (copy_fp8_rows)
  uint8_t* ts;
  uint8_t* xc;
  uint8_t* xs;
  uint16_t* h;
  uint8_t* hc;
  uint8_t* hs;
  size_t bytes;
};

Fp4Ws carve_fp4(const WispMoeConfig* c, int format, void* base) {
  Fp4Ws ws;
  Carve cv;
  const int T = c->tokens, E = c->n_experts, k = c->top_k, M = c->hidden, I = c->inter;
  const int V = E + (c->has_shared ? 1 : 0);
  const int block = format == WISP_FP4_NV ? 16 : 32;
  Workspace& b = ws.base;
  b.lanes = k + (c->has_shared ? 1 : 0);
  b.rows = T * b.lanes;
  b.splits = wb::router_splits(T, E, M);
  ws.part = cv.take<float>(base, b.splits * (size_t)T * E);
  b.plan_scratch = cv.take<int>(base, std::max<size_t>(1, wb::plan_scratch_ints(c)));
  b.idx = cv.take<int>(base, (size_t)T * k);
  b.w = cv.take<float>(base, (size_t)T * k);
  b.counts = cv.take<int>(base, V);
  b.segs = cv.take<WispSegment>(base, V);
  b.row_token = cv.take<int>(base, b.rows);
  b.row_weight = cv.take<float>(base, b.rows);
  b.y = nullptr;
  ws.y = cv.take<uint16_t>(base, (size_t)b.rows * M);
  b.tok_cnt = cv.take<int>(base, T);
  b.tok_list = cv.take<int>(base, (size_t)T * b.lanes);
  const size_t tokens = b.rows >= kGatherRows ? T : 0;
  ws.tc = cv.take<uint8_t>(base, tokens * (M / 2));
  ws.ts = cv.take<uint8_t>(base, tokens * (M / block));
  ws.xc = cv.take<uint8_t>(base, (size_t)b.rows * (M / 2));
  ws.xs = cv.take<uint8_t>(base, (size_t)b.rows * (M / block));
  ws.h = cv.take<uint16_t>(base, (size_t)b.rows * I);
  ws.hc = cv.take<uint8_t>(base, (size_t)b.rows * (I / 2));
  ws.hs = cv.take<uint8_t>(base, (size_t)b.rows * (I / block));
  ws.bytes = (cv.off + 255) & ~(size_t)255;
  return ws;
}

// group_size is the int4 layer's; any valid value passes its check.
WispError validate_fp4(const WispMoeConfig* c, int format, WispErrCtx* err) {
  if (!c) return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_moe: null config");
  if (format != WISP_FP4_MX && format != WISP_FP4_NV)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_moe: unknown format %d", format);
  WispMoeConfig v = *c;
  v.group_size = 128;
  return validate(&v, err);
}

}  // namespace

extern "C" size_t wisp_b200_fp4_moe_workspace_bytes(const WispMoeConfig* cfg, int format) {
  if (validate_fp4(cfg, format, nullptr) != WISP_OK) return 0;
  return carve_fp4(cfg, format, nullptr).bytes;
}

extern "C" WispError wisp_b200_fp4_moe_forward(const WispMoeConfig* cfg, const WispFp4MoeWeights* w,
                                               const uint16_t* d_x, float* d_out, int* d_topk_idx,
                                               float* d_topk_w, void* d_workspace,
                                               size_t workspace_bytes, int* d_error_flag,
                                               cudaStream_t stream, WispErrCtx* err) {
  if (!w) return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_moe_forward: null weights");
  WispError e = validate_fp4(cfg, w->format, err);
  if (e != WISP_OK) return e;
  if (!w->router_w || !d_x || !d_out || !d_workspace)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp4_moe_forward: null pointer argument (router_w, x, out, workspace)");
  if (((uintptr_t)d_x | (uintptr_t)w->router_w | (uintptr_t)d_out) & 15 ||
      (uintptr_t)d_workspace & 255)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp4_moe_forward: x, out and router_w must be 16-byte, workspace 256-byte aligned");
  if (w->format == WISP_FP4_NV && (!w->x_scale || !w->h_scale))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_moe_forward: NV needs x_scale and h_scale");
  const Fp4Ws ws = carve_fp4(cfg, w->format, d_workspace);
  if (workspace_bytes < ws.bytes)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_moe_forward: workspace %zu < required %zu",
                   workspace_bytes, ws.bytes);
  const Workspace& b = ws.base;
  const int T = cfg->tokens, M = cfg->hidden, I = cfg->inter;
  const int V = cfg->n_experts + (cfg->has_shared ? 1 : 0);
  int* idx = d_topk_idx ? d_topk_idx : b.idx;
  float* wt = d_topk_w ? d_topk_w : b.w;
  const bool nv = w->format == WISP_FP4_NV;
  const float* xsc = nv ? w->x_scale : nullptr;
  const float* hsc = nv ? w->h_scale : nullptr;

  e = wb::launch_route(cfg, d_x, w->router_w, w->router_bias, ws.part, b.splits, nullptr, idx, wt,
                       stream, err);
  if (e != WISP_OK) return e;
  e = wb::launch_plan(cfg, idx, wt, b.counts, b.segs, b.row_token, b.row_weight, stream, err,
                      b.plan_scratch);
  if (e != WISP_OK) return e;
  if (b.rows >= kGatherRows) {
    const int block = nv ? 16 : 32;
    e = wisp_b200_fp4_quantize(d_x, WISP_DT_BF16, M, T, nullptr, T, M, w->format, xsc, ws.tc, ws.ts,
                               stream, err);
    if (e != WISP_OK) return e;
    wb::launch_k(gather_fp4_kernel, b.rows, 256, 0, stream, reinterpret_cast<const uint4*>(ws.tc),
                 reinterpret_cast<const uint32_t*>(ws.ts), b.row_token, T, M / 32, M / block / 4,
                 reinterpret_cast<uint4*>(ws.xc), reinterpret_cast<uint32_t*>(ws.xs));
    WB_CUDA_CHECK(cudaGetLastError());
  } else {
    e = wisp_b200_fp4_quantize(d_x, WISP_DT_BF16, M, T, b.row_token, b.rows, M, w->format, xsc,
                               ws.xc, ws.xs, stream, err);
    if (e != WISP_OK) return e;
  }
  WispFp4Config gu = {w->format, V, I, M, 1, WISP_DT_BF16};
  const WispFp4Rows xr = {ws.xc, ws.xs, xsc, b.rows};
  e = wisp_b200_fp4_product(&gu, &w->gate, &w->up, &xr, b.segs, V, ws.h, I, d_error_flag, stream,
                            err);
  if (e != WISP_OK) return e;
  e = wisp_b200_fp4_quantize(ws.h, WISP_DT_BF16, I, b.rows, nullptr, b.rows, I, w->format, hsc,
                             ws.hc, ws.hs, stream, err);
  if (e != WISP_OK) return e;
  WispFp4Config dn = {w->format, V, M, I, 0, WISP_DT_BF16};
  const WispFp4Rows hr = {ws.hc, ws.hs, hsc, b.rows};
  e = wisp_b200_fp4_product(&dn, &w->down, nullptr, &hr, b.segs, V, ws.y, M, d_error_flag, stream,
                            err);
  if (e != WISP_OK) return e;
  return combine_bf16(b, ws.y, V, T, M, d_out, stream, err);
}

namespace {

// Whether the layer quantises its tokens once and copies codes and scales to their rows,
// instead of quantising every row: one launch more and the codes read and written again,
// against the reading and the arithmetic of rows wanted `lanes` times. Powers of two need
// little arithmetic, so that copying them pays later. us, every row / copied, 7168 columns:
// one lane of 2048 tokens 12.2 / 17.3 (powers of two 7.7 / 12.9), two 20.7 / 21.1 (11.6 /
// 17.6), three 28.7 / 23.1 (16.0 / 18.9), four 37.2 / 27.2 (21.4 / 23.8), five 45.6 / 30.3
// (26.1 / 27.2), nine 79.1 / 42.4 (45.0 / 40.4); nine of 512 22.5 / 15.5 (12.6 / 14.0).
// 2048 columns: three lanes of 2048 11.3 / 10.4 (6.7 / 8.5), of 1024 6.7 / 7.4, five of 512
// 6.2 / 6.5, of 1024 10.0 / 8.2 (6.1 / 7.5), of 4096 27.0 / 18.0 (15.6 / 15.2).
bool copy_fp8_rows(int tokens, int lanes, int cols, bool pow2) {
  return lanes >= (pow2 ? 5 : 4) && (int64_t)tokens * lanes * cols >= (pow2 ? 1 << 25 : 1 << 23);
}

struct Fp8Ws {
  Workspace base;      // routing, plan, token lists
  float* part;
  uint16_t* y;         // bf16 expert outputs
  uint8_t* tc;         // the tokens' codes and scales (copy_fp8_rows)
  float* ts;
  uint8_t* xc;
  float* xs;
  uint16_t* h;
  uint8_t* hc;
  float* hs;
  size_t bytes;
};

Fp8Ws carve_fp8(const WispMoeConfig* c, void* base) {
  Fp8Ws ws;
  Carve cv;
  const int T = c->tokens, E = c->n_experts, k = c->top_k, M = c->hidden, I = c->inter;
  const int V = E + (c->has_shared ? 1 : 0);
  Workspace& b = ws.base;
  b.lanes = k + (c->has_shared ? 1 : 0);
  b.rows = T * b.lanes;
  b.splits = wb::router_splits(T, E, M);
  ws.part = cv.take<float>(base, b.splits * (size_t)T * E);
  b.plan_scratch = cv.take<int>(base, std::max<size_t>(1, wb::plan_scratch_ints(c)));
  b.idx = cv.take<int>(base, (size_t)T * k);
  b.w = cv.take<float>(base, (size_t)T * k);
  b.counts = cv.take<int>(base, V);
  b.segs = cv.take<WispSegment>(base, V);
  b.row_token = cv.take<int>(base, b.rows);
  b.row_weight = cv.take<float>(base, b.rows);
  b.y = nullptr;
  ws.y = cv.take<uint16_t>(base, (size_t)b.rows * M);
  b.tok_cnt = cv.take<int>(base, T);
  b.tok_list = cv.take<int>(base, (size_t)T * b.lanes);
  // (what the scales are is not known here; of the two, copying powers of two pays later)
  const size_t tokens = copy_fp8_rows(T, b.lanes, M, false) ? T : 0;
  ws.tc = cv.take<uint8_t>(base, tokens * M);
  ws.ts = cv.take<float>(base, tokens * (M / 128));
  ws.xc = cv.take<uint8_t>(base, (size_t)b.rows * M);
  ws.xs = cv.take<float>(base, (size_t)b.rows * (M / 128));
  ws.h = cv.take<uint16_t>(base, (size_t)b.rows * I);
  ws.hc = cv.take<uint8_t>(base, (size_t)b.rows * I);
  ws.hs = cv.take<float>(base, (size_t)b.rows * (I / 128));
  ws.bytes = (cv.off + 255) & ~(size_t)255;
  return ws;
}

// group_size is the int4 layer's, and with a routing of its own the layer does not
// use the config's: any valid values pass those checks.
WispError validate_fp8(const WispMoeConfig* c, const WispRouting* r, WispErrCtx* err) {
  if (!c) return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_moe: null config");
  WispMoeConfig v = *c;
  v.group_size = 128;
  if (r) v.scoring = WISP_SCORE_SOFTMAX;
  WispError e = validate(&v, err);
  if (e != WISP_OK) return e;
  // the products' limits
  const int V = c->n_experts + (c->has_shared ? 1 : 0);
  const WispFp8Config gu = {V, c->inter, c->hidden, 1, WISP_DT_BF16};
  const WispFp8Config dn = {V, c->hidden, c->inter, 0, WISP_DT_BF16};
  if ((e = wb::fp8_validate(&gu, "fp8_moe", err)) != WISP_OK) return e;
  if ((e = wb::fp8_validate(&dn, "fp8_moe", err)) != WISP_OK) return e;
  // rows are counted in 32 bits
  if ((int64_t)c->tokens * (c->top_k + (c->has_shared ? 1 : 0)) > 0x7fffff00LL)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_moe: %d tokens of %d experts are more than 2^31 - 256 "
                   "rows", c->tokens, c->top_k);
  return r ? wb::routing_validate(r, c->tokens, c->n_experts, c->top_k, "fp8_moe", err) : WISP_OK;
}

}  // namespace

extern "C" size_t wisp_b200_fp8_moe_workspace_bytes(const WispMoeConfig* cfg,
                                                    const WispRouting* routing) {
  if (validate_fp8(cfg, routing, nullptr) != WISP_OK) return 0;
  return carve_fp8(cfg, nullptr).bytes;
}

extern "C" WispError wisp_b200_fp8_moe_forward(const WispMoeConfig* cfg, const WispRouting* routing,
                                               const WispFp8MoeWeights* w, const uint16_t* d_x,
                                               float* d_out, int* d_topk_idx, float* d_topk_w,
                                               void* d_workspace, size_t workspace_bytes,
                                               int* d_error_flag, cudaStream_t stream,
                                               WispErrCtx* err) {
  WispError e = validate_fp8(cfg, routing, err);
  if (e != WISP_OK) return e;
  if (!w || !w->router_w || !d_x || !d_out || !d_workspace)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp8_moe_forward: null pointer argument (weights, router_w, x, out, workspace)");
  if (((uintptr_t)d_x | (uintptr_t)w->router_w | (uintptr_t)d_out) & 15 ||
      (uintptr_t)d_workspace & 255)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp8_moe_forward: x, out and router_w must be 16-byte, workspace 256-byte aligned");
  if (w->score_bias && !routing)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_moe_forward: score_bias without a routing");
  const Fp8Ws ws = carve_fp8(cfg, d_workspace);
  if (workspace_bytes < ws.bytes)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_moe_forward: workspace %zu < required %zu",
                   workspace_bytes, ws.bytes);
  // (all that the steps below would refuse, before the first of them is launched)
  if (((uintptr_t)w->router_bias | (uintptr_t)w->score_bias | (uintptr_t)d_topk_idx |
       (uintptr_t)d_topk_w | (uintptr_t)d_error_flag) & 3)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp8_moe_forward: router_bias, score_bias, topk_idx, topk_w and the error word must "
                   "be 4-byte aligned");
  if ((e = wb::fp8_check_mats(&w->gate, "fp8_moe_forward", "gate", err)) != WISP_OK) return e;
  if ((e = wb::fp8_check_mats(&w->up, "fp8_moe_forward", "up", err)) != WISP_OK) return e;
  if ((e = wb::fp8_check_mats(&w->down, "fp8_moe_forward", "down", err)) != WISP_OK) return e;
  const Workspace& b = ws.base;
  const int T = cfg->tokens, M = cfg->hidden, I = cfg->inter;
  const int V = cfg->n_experts + (cfg->has_shared ? 1 : 0);
  int* idx = d_topk_idx ? d_topk_idx : b.idx;
  float* wt = d_topk_w ? d_topk_w : b.w;

  if (routing) {
    const int parts = wb::launch_logits(cfg, d_x, w->router_w, ws.part, b.splits, stream);
    WB_CUDA_CHECK(cudaGetLastError());
    e = wb::launch_select(routing, ws.part, parts, w->router_bias, w->score_bias, T, cfg->n_experts,
                          cfg->top_k, idx, wt, stream, err);
  } else {
    e = wb::launch_route(cfg, d_x, w->router_w, w->router_bias, ws.part, b.splits, nullptr, idx, wt,
                         stream, err);
  }
  if (e != WISP_OK) return e;
  e = wb::launch_plan(cfg, idx, wt, b.counts, b.segs, b.row_token, b.row_weight, stream, err,
                      b.plan_scratch);
  if (e != WISP_OK) return e;
  if (copy_fp8_rows(T, b.lanes, M, w->pow2)) {
    e = wisp_b200_fp8_quantize(d_x, WISP_DT_BF16, M, T, nullptr, T, M, w->pow2, ws.tc, ws.ts, 1, T,
                               stream, err);
    if (e != WISP_OK) return e;
    const WispFp8Rows tr = {ws.tc, ws.ts, 1, T, T};
    e = wisp_b200_fp8_gather(&tr, b.row_token, b.rows, M, ws.xc, ws.xs, 1, b.rows, stream, err);
    if (e != WISP_OK) return e;
  } else {
    e = wisp_b200_fp8_quantize(d_x, WISP_DT_BF16, M, T, b.row_token, b.rows, M, w->pow2, ws.xc,
                               ws.xs, 1, b.rows, stream, err);
    if (e != WISP_OK) return e;
  }
  const WispFp8Config gu = {V, I, M, 1, WISP_DT_BF16};
  const WispFp8Rows xr = {ws.xc, ws.xs, 1, b.rows, b.rows};
  e = wisp_b200_fp8_product(&gu, &w->gate, &w->up, &xr, b.segs, V, ws.h, I, d_error_flag, stream,
                            err);
  if (e != WISP_OK) return e;
  e = wisp_b200_fp8_quantize(ws.h, WISP_DT_BF16, I, b.rows, nullptr, b.rows, I, w->pow2, ws.hc,
                             ws.hs, 1, b.rows, stream, err);
  if (e != WISP_OK) return e;
  const WispFp8Config dn = {V, M, I, 0, WISP_DT_BF16};
  const WispFp8Rows hr = {ws.hc, ws.hs, 1, b.rows, b.rows};
  e = wisp_b200_fp8_product(&dn, &w->down, nullptr, &hr, b.segs, V, ws.y, M, d_error_flag, stream,
                            err);
  if (e != WISP_OK) return e;
  return combine_bf16(b, ws.y, V, T, M, d_out, stream, err);
}

// Pointers into a reference blob (header at offset 0) from its parsed meta.
extern "C" WispError wisp_b200_blob_expert(const WispExpertMeta* meta, const void* d_blob,
                                           WispInt4Expert* out, WispErrCtx* err) {
  if (!meta || !d_blob || !out) return WB_FAIL(WISP_ERR_INVALID_ARG, "blob_expert: null pointer");
  if (!meta->valid) return WB_FAIL(WISP_ERR_INVALID_ARG, "blob_expert: meta not valid");
  const uint8_t* base = static_cast<const uint8_t*>(d_blob);
  WispInt4Mat* mats[3] = {&out->gate, &out->up, &out->down};
  for (int m = 0; m < 3; m++) {
    const uint8_t* packed = base + meta->packed_off[m];
    const uint8_t* scales = base + meta->scales_off[m];
    // Zero points are present when bytes remain between zeros_off and the
    // next matrix's packed data (the end of the blob for down).
    const size_t end = m < 2 ? meta->packed_off[m + 1] : meta->total_bytes;
    const uint8_t* zeros = end > meta->zeros_off[m] ? base + meta->zeros_off[m] : nullptr;
    if (((uintptr_t)packed | (uintptr_t)scales | (uintptr_t)zeros) & 15)
      return WB_FAIL(WISP_ERR_INVALID_ARG,
                     "blob_expert: matrix %d data not 16-byte aligned (place the blob at an "
                     "address = 8 mod 16)", m);
    mats[m]->packed = packed;
    mats[m]->scales = reinterpret_cast<const wisp_half*>(scales);
    mats[m]->zeros = reinterpret_cast<const wisp_half*>(zeros);
  }
  return WISP_OK;
}

extern "C" int* wisp_b200_moe_error_word(const WispMoeConfig* cfg, void* d_workspace) {
  if (validate(cfg, nullptr) != WISP_OK || !d_workspace) return nullptr;
  return carve(cfg, d_workspace).error_flag;
}

extern "C" WispError wisp_b200_check_error_flag(const int* d_error_flag, cudaStream_t stream,
                                                WispErrCtx* err) {
  if (!d_error_flag) return WB_FAIL(WISP_ERR_INVALID_ARG, "check_error_flag: null pointer");
  int h = 0;
  WB_CUDA_CHECK(cudaMemcpyAsync(&h, d_error_flag, sizeof(int), cudaMemcpyDeviceToHost, stream));
  WB_CUDA_CHECK(cudaStreamSynchronize(stream));
  if (h == wb::kErrorSkipped)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "a segment lay outside its weights or rows and was skipped (device error word 2)");
  if (h)
    return WB_FAIL(WISP_ERR_TIMEOUT, "a kernel gave up waiting%s (device error word %d)",
                   h & wb::kErrorSkipped ? ", and a segment was skipped" : "", h);
  return WISP_OK;
}

// Header parse on host memory; semantics of csrc/core/wisp_engine.c:268-303.
extern "C" WispError wisp_b200_parse_expert_header(const void* blob, size_t blob_size,
                                                   WispExpertMeta* meta, WispErrCtx* err) {
  if (!blob || !meta) return WB_FAIL(WISP_ERR_OOM, "NULL pointer: expert_parse_header: blob");
  if (blob_size < sizeof(WispExpertHeader))
    return WB_FAIL(WISP_ERR_MODEL, "expert blob too small: %zu bytes", blob_size);
  WispExpertHeader h;
  memcpy(&h, blob, sizeof h);
  if (h.magic != WISP_EXPERT_MAGIC || h.version != WISP_EXPERT_VERSION || h.n_mats != WISP_EXPERT_NMATS)
    return WB_FAIL(WISP_ERR_MODEL, "expert blob corrupt: magic=%08x version=%u n_mats=%u", h.magic,
                   h.version, h.n_mats);
  size_t off = sizeof(WispExpertHeader);
  for (int m = 0; m < WISP_EXPERT_NMATS; m++) {
    meta->rows[m] = h.mats[m].rows;
    meta->cols[m] = h.mats[m].cols;
    meta->packed_off[m] = off;
    off += h.mats[m].packed_bytes;
    meta->scales_off[m] = off;
    off += h.mats[m].scales_bytes;
    meta->zeros_off[m] = off;
    off += h.mats[m].zeros_bytes;
  }
  meta->group_size = h.group_size;
  meta->total_bytes = off;
  meta->valid = 1;
  if (off > blob_size) {
    meta->valid = 0;
    return WB_FAIL(WISP_ERR_MODEL, "expert blob truncated: needs %zu, have %zu", off, blob_size);
  }
  return WISP_OK;
}

extern "C" const char* wisp_b200_version(void) { return "wisp_b200 0.1.0 (sm_100a)"; }
