// select.cu -- which experts each token goes to, and with what weight, from the
// router's logits: softmax or sigmoid scores, a bias that takes part in the choice
// and not in the weights, groups of experts of which the best are kept, top-k.
#include <cuda_bf16.h>

#include "common.cuh"
#include "internal.h"
#include "numeric.cuh"

namespace {

using namespace wb;

constexpr int kWarps = 4;          // tokens per CTA

struct Params {
  const void* logits;
  int type;
  int64_t ld;
  int splits;                      // fp32 partial sums to add, `split` values apart
  int64_t split;
  const float* logit_bias;         // added to the logits
  const float* bias;
  int T, E, k;
  int scoring, groups, kept, group_top, renorm;
  float scaling;
  int* idx;
  float* w;
};

// A double as an unsigned integer in the same order; 0 for what cannot be chosen
// (NaN and -infinity).
WB_DEV uint64_t order_key(double v) {
  if (!(v > -INFINITY)) return 0;
  if (v == 0.0) v = 0.0;           // -0 and +0 are equal
  const int64_t b = __double_as_longlong(v);
  return (uint64_t)(b ^ ((b >> 63) | INT64_MIN));
}

WB_DEV double shfl_xor(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// One warp per token; lane l holds experts l + 32 j, j < PER. Scores and choice
// are 64-bit: two experts whose choices lie closer than fp32 resolves still come
// out in their order, and only equal choices are ties, which go to the lower
// expert.
template <int PER>
__global__ void __launch_bounds__(kWarps * 32) select_kernel(const Params p) {
  extern __shared__ double choices[];       // [kWarps][E], with groups
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kWarps + warp;
  if (t >= p.T) return;
  const int E = p.E;
  double score[PER];
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int e = lane + 32 * j;
    score[j] = -INFINITY;
    if (e < E) {
      float v = load_one(p.logits, p.type, t * p.ld + e);
      for (int z = 1; z < p.splits; z++)
        v += static_cast<const float*>(p.logits)[z * p.split + t * p.ld + e];
      if (p.logit_bias) v += p.logit_bias[e];
      score[j] = (double)v;
    }
  }
  if (p.scoring == WISP_ROUTE_SOFTMAX) {
    // (a NaN logit makes every score NaN, as does +infinity)
    double mx = -INFINITY, sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; j++) mx = fmax(mx, score[j]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmax(mx, shfl_xor(mx, o));
#pragma unroll
    for (int j = 0; j < PER; j++) {
      score[j] = lane + 32 * j < E ? exp(score[j] - mx) : 0.0;
      sum += score[j];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += shfl_xor(sum, o);
#pragma unroll
    for (int j = 0; j < PER; j++) score[j] /= sum;
  } else {
#pragma unroll
    for (int j = 0; j < PER; j++) score[j] = 1.0 / (1.0 + exp(-score[j]));
  }
  uint64_t key[PER];
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int e = lane + 32 * j;
    key[j] = 0;
    if (e < E) {
      const double c = p.bias ? score[j] + (double)p.bias[e] : score[j];
      key[j] = order_key(c);
      if (p.kept < p.groups) choices[warp * E + e] = c;
    }
  }
  if (p.kept < p.groups) {
    // lanes g L .. g L + L - 1 read group g's choices, and find its best two
    __syncwarp();
    const int gsz = E / p.groups;
    int L = 1;
    while (2 * L * p.groups <= 32) L *= 2;
    const int g = lane / L;
    double a = -INFINITY, b = -INFINITY;
    if (g < p.groups) {
      for (int i = lane % L; i < gsz; i += L) {
        const double c = choices[warp * E + g * gsz + i];
        if (c > a) {
          b = a;
          a = c;
        } else if (c > b) {
          b = c;
        }
      }
    }
    for (int o = 1; o < L; o <<= 1) {
      const double oa = shfl_xor(a, o), ob = shfl_xor(b, o);
      b = fmax(fmin(a, oa), fmax(b, ob));
      a = fmax(a, oa);
    }
    // choices that cannot be made (-infinity, NaN) count nothing; a group of
    // those alone is never kept
    const double s = p.group_top > 1 && b > -INFINITY ? a + b : a;
    int rank = 0;
    for (int h = 0; h < p.groups; h++) {
      const double o = __shfl_sync(0xffffffffu, s, h * L);
      rank += o > s || (o == s && h < g);
    }
    const uint32_t keep = __ballot_sync(
        0xffffffffu, g < p.groups && lane % L == 0 && rank < p.kept && s > -INFINITY);
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const int e = lane + 32 * j;
      if (e < E && !(keep >> (e / gsz * L) & 1u)) key[j] = 0;
    }
  }
  // k rounds of the largest key, the lowest expert among equal ones
  int mine = -1;
  double weight = 0.0, total = 0.0;
  for (int r = 0; r < p.k; r++) {
    uint64_t best = 0;
    int at = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      if (key[j] > best) {
        best = key[j];
        at = j;
      }
    }
    const uint32_t hi = (uint32_t)(best >> 32), lo = (uint32_t)best;
    const uint32_t mhi = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t mlo = __reduce_max_sync(0xffffffffu, hi == mhi ? lo : 0u);
    if (!(mhi | mlo)) break;       // nothing is left to choose
    const uint32_t e = __reduce_min_sync(
        0xffffffffu, hi == mhi && lo == mlo ? (uint32_t)(lane + 32 * at) : 0xffffffffu);
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      if ((int)e == lane + 32 * j) {
        key[j] = 0;
        s = score[j];
      }
    }
    s = __shfl_sync(0xffffffffu, s, e & 31);
    if (lane == r) {
      mine = (int)e;
      weight = s;
    }
    total += s;
  }
  if (lane < p.k) {
    if (p.renorm) weight = total > 0.0 ? weight / total : 0.0;
    p.idx[t * p.k + lane] = mine;
    p.w[t * p.k + lane] = (float)(weight * (double)p.scaling);
  }
}

WispError launch(const Params& p, cudaStream_t st, WispErrCtx* err) {
  auto kernel = p.E <= 32 ? select_kernel<1> : p.E <= 64 ? select_kernel<2>
              : p.E <= 128 ? select_kernel<4> : p.E <= 256 ? select_kernel<8>
              : p.E <= 512 ? select_kernel<16> : select_kernel<32>;
  const size_t smem = p.kept < p.groups ? sizeof(double) * kWarps * p.E : 0;
  wb::launch_k(kernel, (unsigned)(((int64_t)p.T + kWarps - 1) / kWarps), kWarps * 32, smem, st, p);
  WB_CUDA_CHECK(cudaGetLastError());
  return WISP_OK;
}

}  // namespace

WispError wb::routing_validate(const WispRouting* r, int tokens, int n_experts, int top_k,
                               const char* who, WispErrCtx* err) {
  if (!r) return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: null routing", who);
  if (tokens < 0 || tokens > wb::kMaxRows || n_experts <= 0 || n_experts > 1024)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: tokens=%d n_experts=%d (0..2^31 - 256, 1..1024)", who,
                   tokens, n_experts);
  if (r->scoring != WISP_ROUTE_SOFTMAX && r->scoring != WISP_ROUTE_SIGMOID)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: unknown scoring %d", who, r->scoring);
  if (r->n_groups <= 0 || r->n_groups > 32 || n_experts % r->n_groups || r->topk_groups <= 0 ||
      r->topk_groups > r->n_groups)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "%s: n_groups=%d topk_groups=%d (1..32 equal groups of %d experts, of which as "
                   "many are kept at most)",
                   who, r->n_groups, r->topk_groups, n_experts);
  if (r->group_top != 1 && r->group_top != 2)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: group_top=%d (1 or 2)", who, r->group_top);
  if (top_k <= 0 || top_k > 32 || top_k > r->topk_groups * (n_experts / r->n_groups))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: top_k=%d (1..32, and within the kept groups' experts)",
                   who, top_k);
  return WISP_OK;
}

WispError wb::launch_select(const WispRouting* r, const float* part, int splits,
                            const float* logit_bias, const float* bias, int tokens, int n_experts,
                            int top_k, int* idx, float* w, cudaStream_t st, WispErrCtx* err) {
  Params p;
  p.logits = part;
  p.type = WISP_DT_F32;
  p.ld = n_experts;
  p.splits = splits;
  p.split = (int64_t)tokens * n_experts;
  p.logit_bias = logit_bias;
  p.bias = bias;
  p.T = tokens;
  p.E = n_experts;
  p.k = top_k;
  p.scoring = r->scoring;
  p.groups = r->n_groups;
  p.kept = r->topk_groups;
  p.group_top = r->group_top;
  p.renorm = r->renormalize;
  p.scaling = r->scaling;
  p.idx = idx;
  p.w = w;
  return launch(p, st, err);
}

extern "C" WispError wisp_b200_select_experts(const WispRouting* routing, const void* d_logits,
                                              int logits_type, int64_t ld, int tokens,
                                              int n_experts, int top_k, const float* d_bias,
                                              int* d_idx, float* d_w, cudaStream_t stream,
                                              WispErrCtx* err) {
  WispError e = wb::routing_validate(routing, tokens, n_experts, top_k, "select_experts", err);
  if (e != WISP_OK) return e;
  if (!dt_valid(logits_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "select_experts: unknown logits_type %d", logits_type);
  if (ld < n_experts)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "select_experts: ld=%lld < n_experts=%d", (long long)ld,
                   n_experts);
  if (tokens == 0) return WISP_OK;
  if (!d_logits || !d_idx || !d_w)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "select_experts: null pointer argument (logits, idx, w)");
  if ((uintptr_t)d_logits % dt_size(logits_type) ||
      (((uintptr_t)d_bias | (uintptr_t)d_idx | (uintptr_t)d_w) & 3))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "select_experts: an argument is not aligned to its type");
  Params p;
  p.logits = d_logits;
  p.type = logits_type;
  p.ld = ld;
  p.splits = 1;
  p.split = 0;
  p.logit_bias = nullptr;
  p.bias = d_bias;
  p.T = tokens;
  p.E = n_experts;
  p.k = top_k;
  p.scoring = routing->scoring;
  p.groups = routing->n_groups;
  p.kept = routing->topk_groups;
  p.group_top = routing->group_top;
  p.renorm = routing->renormalize;
  p.scaling = routing->scaling;
  p.idx = d_idx;
  p.w = d_w;
  return launch(p, stream, err);
}
