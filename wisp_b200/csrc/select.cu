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
  int gsz, lanes;                  // experts of a group, lanes that look at them
  uint32_t by_gsz;                 // 2^32 / gsz rounded up
  float scaling;
  int* idx;
  float* w;
};

// A double, a float as an unsigned integer in the same order; 0 for what cannot be
// chosen (NaN and -infinity).
WB_DEV uint64_t order_key(double v) {
  if (!(v > -INFINITY)) return 0;
  if (v == 0.0) v = 0.0;           // -0 and +0 are equal
  const int64_t b = __double_as_longlong(v);
  return (uint64_t)(b ^ ((b >> 63) | INT64_MIN));
}
WB_DEV uint32_t order_key(float v) {
  const int32_t b = __float_as_int(v + 0.f);
  return (uint32_t)(b ^ ((b >> 31) | INT32_MIN));
}
WB_DEV float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

WB_DEV float to_float(float v) { return v; }
WB_DEV float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
WB_DEV float to_float(__half v) { return __half2float(v); }

WB_DEV double shfl_xor(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }
WB_DEV float shfl_xor(float v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

WB_DEV int group_of(const Params& p, int e) { return p.gsz == 1 ? e : (int)__umulhi(e, p.by_gsz); }

// The best two of a lane's group (-infinity where there are fewer), from the choices
// in shared memory: lanes g L .. g L + L - 1 look at group g's.
template <typename R>
WB_DEV void best_two(const Params& p, const R* choices, int lane, R& a, R& b) {
  a = b = -INFINITY;
  const int gsz = p.gsz, L = p.lanes, g = lane / L;
  if (g < p.groups) {
    for (int i = lane % L; i < gsz; i += L) {
      const R c = choices[g * gsz + i];
      if (c > a) {
        b = a;
        a = c;
      } else if (c > b) {
        b = c;
      }
    }
  }
  for (int o = 1; o < L; o <<= 1) {
    const R oa = shfl_xor(a, o), ob = shfl_xor(b, o);
    b = fmax(fmin(a, oa), fmax(b, ob));
    a = fmax(a, oa);
  }
}

// The weights of a token's choices: lane r < k holds expert `mine` (-1: none), its
// score and its place in the row.
WB_DEV void put_weights(const Params& p, int64_t t, int lane, int mine, double score, double total) {
  if (lane < p.k) {
    if (p.renorm) score = total > 0.0 ? score / total : 0.0;
    p.idx[t * p.k + lane] = mine;
    p.w[t * p.k + lane] = (float)(score * (double)p.scaling);
  }
}

// The routing of one token in 64 bits. v: the logits of experts lane + 32 j,
// -infinity where there is none.
template <int PER>
WB_DEV void route_exact(const Params& p, int64_t t, const float (&v)[PER], int lane, double* choices) {
  const int E = p.E;
  double score[PER];
#pragma unroll
  for (int j = 0; j < PER; j++) score[j] = (double)v[j];
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
  __syncwarp();                      // the choices in 32 bits have been read
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int e = lane + 32 * j;
    key[j] = 0;
    if (e < E) {
      const double c = p.bias ? score[j] + (double)p.bias[e] : score[j];
      key[j] = order_key(c);
      if (p.kept < p.groups) choices[e] = c;
    }
  }
  if (p.kept < p.groups) {
    __syncwarp();
    const int L = p.lanes, g = lane / L;
    double a, b;
    best_two(p, choices, lane, a, b);
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
      if (e < E && !(keep >> (group_of(p, e) * L) & 1u)) key[j] = 0;
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
  put_weights(p, t, lane, mine, weight, total);
}

// The same out of line, for logits in shared memory: a rare path whose registers the
// usual one does without.
template <int PER>
__device__ __noinline__ void route_exact_from(const Params& p, int64_t t, const float* logits,
                                              int lane, double* choices) {
  float v[PER];
#pragma unroll
  for (int j = 0; j < PER; j++) v[j] = logits[32 * j];
  route_exact<PER>(p, t, v, lane, choices);
}

// A token's logits; past the experts -infinity. (One branch on the type for all loads,
// none on the experts that there are: what is read past them is the last one's.)
template <int PER>
WB_DEV void load_logits(const Params& p, int64_t t, int lane, float (&v)[PER]) {
  auto load = [&](auto* q) {
#pragma unroll
    for (int j = 0; j < PER; j++) v[j] = to_float(q[min(lane + 32 * j, p.E - 1)]);
  };
  if (p.type == WISP_DT_F32)
    load(static_cast<const float*>(p.logits) + t * p.ld);
  else if (p.type == WISP_DT_BF16)
    load(static_cast<const __nv_bfloat16*>(p.logits) + t * p.ld);
  else
    load(static_cast<const __half*>(p.logits) + t * p.ld);
  for (int z = 1; z < p.splits; z++) {
    const float* q = static_cast<const float*>(p.logits) + z * p.split + t * p.ld;
#pragma unroll
    for (int j = 0; j < PER; j++) v[j] += q[min(lane + 32 * j, p.E - 1)];
  }
  if (p.logit_bias) {
#pragma unroll
    for (int j = 0; j < PER; j++) v[j] += p.logit_bias[min(lane + 32 * j, p.E - 1)];
  }
#pragma unroll
  for (int j = 0; j < PER; j++)
    if (lane + 32 * j >= p.E) v[j] = -INFINITY;
}

// One warp per token, all in 64 bits.
template <int PER>
__global__ void __launch_bounds__(kWarps * 32) select_exact_kernel(const Params p) {
  extern __shared__ double choices64[];       // [kWarps][E], with groups
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kWarps + warp;
  if (t >= p.T) return;
  float v[PER];
  load_logits<PER>(p, t, lane, v);
  route_exact<PER>(p, t, v, lane, choices64 + (p.kept < p.groups ? warp * p.E : 0));
}

// The largest of a warp's keys and the lowest expert that has it.
template <int PER>
WB_DEV uint32_t take_best(uint32_t (&key)[PER], int lane, uint32_t& expert) {
  uint32_t best = 0;
#pragma unroll
  for (int j = 0; j < PER; j++) best = max(best, key[j]);
  best = __reduce_max_sync(0xffffffffu, best);
  uint32_t e = 0xffffffffu;
#pragma unroll
  for (int j = PER - 1; j >= 0; j--)
    if (key[j] == best) e = lane + 32 * j;
  e = __reduce_min_sync(0xffffffffu, e);
#pragma unroll
  for (int j = 0; j < PER; j++)
    if (e == (uint32_t)(lane + 32 * j)) key[j] = 0;
  expert = e;
  return best;
}

// One warp per token; lane l holds experts l + 32 j, j < PER.
//
// The result is that of 64-bit scores and choices (route_exact), found in 32 bits
// where that decides it. With u = 2^-24, half a step of fp32 at most: the quick exponential
// of x is off by 2 + 1.2 |x| steps, (4 + 2.4 |x|) u of itself. A sigmoid s takes s (1 - s) of
// that, at most 1.3 u (at |x| = 0.8), and with the sum in its divisor (1 u) and
// the quick reciprocal (2 u) it is off by less than 5 u: 2^-21 covers it. A softmax, d
// below the largest logit, has an exponential off by (4 + 3.4 d) u of itself, d u of it
// from rounding the argument: e^-d times that is at most 4 u of the largest. Their sum is
// off by their errors' mean, at most 20 u of it (1023 of them at d = 5.4 beside the
// largest: 19.1), by 36 roundings (31 in a lane, 5 across) and the reciprocal's 2 u: 58 u.
// With the last product's rounding a score is off by at most 4 + 58 + 1 = 63 u of the
// largest score: 2^-18. Adding the bias rounds by u of the choice, the sum of two choices
// by as much, and the comparison again: 2^-22 of each choice. Without a bias the scores
// are in the logits' order, which needs no scores at all: equal logits are ties, and
// those 2^-20 apart have different 64-bit scores as long as these are not near 1 (logits above
// 16) or 0 (logits, from the largest on for softmax, below -700). Only a token with a
// closer pair where it matters, or with a value that is not finite, goes the 64-bit
// way. (A softmax whose weights are not renormalised needs the 64-bit sum over all
// experts, and goes that way at once: 12.6 us where this takes 15.6.) 256 experts with
// bias and groups, us a launch, in 64 bits alone and so: one token 7.9 and 4.6, 4096
// 14.3 and 11.7, 16,384 47 and 34; bound by its instructions, 1700 a token.
template <int PER>
__global__ void __launch_bounds__(kWarps * 32) select_kernel(const Params p) {
  extern __shared__ double choices64[];       // [kWarps][E], with groups
  __shared__ float logits[kWarps][32 * PER];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kWarps + warp;
  if (t >= p.T) return;
  const int E = p.E;
  const bool softmax = p.scoring == WISP_ROUTE_SOFTMAX, grouped = p.kept < p.groups;
  float v[PER], mx = -INFINITY, span = 0.f;
  load_logits<PER>(p, t, lane, v);
#pragma unroll
  for (int j = 0; j < PER; j++) {
    if (lane + 32 * j < E) span += v[j] - v[j];       // NaN where a value is not finite
    mx = fmaxf(mx, v[j]);
  }
#pragma unroll
  for (int j = 0; j < PER; j++) logits[warp][lane + 32 * j] = v[j];
  const float* mine_v = logits[warp] + lane;
  double* choices = choices64 + (grouped ? warp * E : 0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, shfl_xor(mx, o));
  // what the experts are ordered by, as keys
  const bool scores = p.bias || (grouped && p.group_top > 1);
  float top = 1.f;                   // the largest score of a softmax
  uint32_t key[PER];
  if (scores) {
    float s[PER], sum = 0.f;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      s[j] = __expf(softmax ? v[j] - mx : -v[j]);      // (softmax: 0 past the experts)
      sum += s[j];
    }
    if (softmax) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += shfl_xor(sum, o);
      sum = top = rcp_approx(sum);
    }
#pragma unroll
    for (int j = 0; j < PER; j++) s[j] = softmax ? s[j] * sum : rcp_approx(1.f + s[j]);
    if (p.bias) {
#pragma unroll
      for (int j = 0; j < PER; j++) {
        s[j] += p.bias[min(lane + 32 * j, E - 1)];
        span += s[j] - s[j];
      }
    }
#pragma unroll
    for (int j = 0; j < PER; j++) {
      key[j] = lane + 32 * j < E ? order_key(s[j]) : 0u;
      if (grouped && lane + 32 * j < E) reinterpret_cast<float*>(choices)[lane + 32 * j] = s[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < PER; j++) {
      key[j] = lane + 32 * j < E ? order_key(v[j]) : 0u;
      if (grouped && lane + 32 * j < E) reinterpret_cast<float*>(choices)[lane + 32 * j] = v[j];
    }
  }
  bool sure = __all_sync(0xffffffffu, span == 0.f) && (scores || softmax || mx <= 16.f);
  // How far a choice may be off (with scores), see above.
  const float off = softmax ? 3.814697265625e-6f * top : 4.76837158203125e-7f;   // 2^-18, 2^-21
  auto err = [&](float c) { return off + 2.384185791015625e-7f * fabsf(c); };
  const float least = softmax ? mx - 700.f : -700.f;
  // Whether a > b is beyond doubt, or (without scores) both are the same for certain.
  auto apart = [&](float a, float b) {
    const float d = a - b;
    if (scores) return d > err(a) + err(b);
    return a >= least && (d >= 9.5367431640625e-7f * fmaxf(1.f, fabsf(a)) || d == 0.f);   // 2^-20
  };
  if (grouped && sure) {
    __syncwarp();
    const int L = p.lanes, g = lane / L;
    float a, b;
    best_two(p, reinterpret_cast<const float*>(choices), lane, a, b);
    const float s = p.group_top > 1 && p.gsz > 1 ? a + b : a;
    int rank = 0;
    for (int h = 0; h < p.groups; h++) {
      const float o = __shfl_sync(0xffffffffu, s, h * L);
      rank += o > s || (o == s && h < g);
    }
    const bool head = g < p.groups && lane % L == 0, kept = head && rank < p.kept;
    const uint32_t keep = __ballot_sync(0xffffffffu, kept);
    // the worst that is kept, at its lowest, against the best that is not, at its highest
    // (two choices of opposite signs leave a sum that is smaller than what they are off by)
    const float e = !scores ? 0.f : p.group_top > 1 && p.gsz > 1 ? err(a) + err(b) : err(a);
    const float worst = key_value(__reduce_min_sync(0xffffffffu, kept ? order_key(s - e) : 0xffffffffu));
    const float next = key_value(__reduce_max_sync(0xffffffffu, head && !kept ? order_key(s + e) : 0u));
    sure = scores ? worst > next : apart(worst, next);
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const int e = lane + 32 * j;
      if (e < E && !(keep >> (group_of(p, e) * L) & 1u)) key[j] = 0;
    }
  }
  int mine = -1;
  float last = INFINITY;
  for (int r = 0; r <= p.k && sure; r++) {       // one round more, for the last one's distance
    uint32_t e;
    const uint32_t best = take_best(key, lane, e);
    if (best == 0) break;          // (all of the kept groups' experts are taken)
    const float c = key_value(best);
    if (r > 0) sure = apart(last, c);
    last = c;
    if (lane == r && r < p.k) mine = (int)e;
  }
  if (!sure) {
    route_exact_from<PER>(p, t, mine_v, lane, choices);
    return;
  }
  // the weights, of these experts alone: the sum over all of a softmax cancels
  __syncwarp();
  const double l = mine >= 0 ? (double)logits[warp][mine] : 0.0;
  double score = 0.0, total = 0.0;
  if (mine >= 0) score = softmax ? exp(l - (double)mx) : 1.0 / (1.0 + exp(-l));
  if (p.renorm) {
    total = score;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += shfl_xor(total, o);
  }
  put_weights(p, t, lane, mine, score, total);
}

WispError launch(Params& p, cudaStream_t st, WispErrCtx* err) {
  p.gsz = p.E / p.groups;
  p.by_gsz = (uint32_t)(((1ull << 32) + p.gsz - 1) / p.gsz);
  p.lanes = 1;
  while (2 * p.lanes * p.groups <= 32) p.lanes *= 2;
  const bool exact = p.scoring == WISP_ROUTE_SOFTMAX && !p.renorm;
  auto of = [&](auto usual, auto all64) { return exact ? all64 : usual; };
  auto kernel = p.E <= 32 ? of(select_kernel<1>, select_exact_kernel<1>)
              : p.E <= 64 ? of(select_kernel<2>, select_exact_kernel<2>)
              : p.E <= 128 ? of(select_kernel<4>, select_exact_kernel<4>)
              : p.E <= 256 ? of(select_kernel<8>, select_exact_kernel<8>)
              : p.E <= 512 ? of(select_kernel<16>, select_exact_kernel<16>)
                           : of(select_kernel<32>, select_exact_kernel<32>);
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
