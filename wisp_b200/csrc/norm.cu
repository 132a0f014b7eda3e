// norm.cu -- the norms after and before a block with its gate and residual:
//   p = y / rms(y) * (o + w_post),  x' = rs * x + gate * p,
//   n = x' / rms(x') * (o + w_pre)
// One CTA per row; a row's x and y stay in registers (8 values per vector, at
// most V vectors per thread), so each input is read once and each output
// written once and the bound is HBM (and, for a few rows, the latency of one
// load, two block sums and one store). n is taken from the fp32 x'.
#include "common.cuh"
#include "internal.h"
#include "numeric.cuh"

namespace {

using namespace wb;

struct NormParams {
  WispBlockNorm c;
  const void* x;
  const void* y;
  const void* gate;
  const void* post_w;
  const void* pre_w;
  void* x_out;
  void* n;
  // whether rows start on 16-byte boundaries and hold whole vectors
  int wide_x, wide_y, wide_g, wide_post, wide_pre, wide_xo, wide_n;
};

// Sum over the block, the same bits in every thread.
WB_DEV float block_sum(float v, float* buf) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = (blockDim.x + 31) >> 5, lane = threadIdx.x & 31;
  if (lane == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? buf[lane] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int V>
__global__ void __launch_bounds__(1024) block_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float buf[2][32];
  const WispBlockNorm& c = p.c;
  const int64_t t = blockIdx.x;
  const int M = c.hidden;
  float x[V][8], y[V][8];
#pragma unroll
  for (int k = 0; k < V; k++) {
    const int i = (k * blockDim.x + threadIdx.x) * 8, n = M - i;
    if (n > 0) {
      if (p.y) load8(p.y, c.y_type, t * c.ld_y + i, p.wide_y && n >= 8, n, y[k]);
      load8(p.x, c.x_type, t * c.ld_x + i, p.wide_x && n >= 8, n, x[k]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) x[k][j] = y[k][j] = 0.f;
    }
  }
  if (p.y) {
    float r = 1.f;
    if (c.post_norm) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < V; k++)
#pragma unroll
        for (int j = 0; j < 8; j++) s = fmaf(y[k][j], y[k][j], s);
      r = 1.f / sqrtf(block_sum(s, buf[0]) / (float)M + c.eps);
    }
    const float gt = c.gate_kind == WISP_GATE_TOKEN ? load_one(p.gate, c.gate_type, t) : 1.f;
#pragma unroll
    for (int k = 0; k < V; k++) {
      const int i = (k * blockDim.x + threadIdx.x) * 8, n = M - i;
      if (n <= 0) continue;
      float w[8];
      if (c.post_norm) {
        if (p.post_w) {
          load8(p.post_w, c.w_type, i, p.wide_post && n >= 8, n, w);
#pragma unroll
          for (int j = 0; j < 8; j++) y[k][j] = y[k][j] * r * (c.weight_offset + w[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) y[k][j] *= r;
        }
      }
      if (c.gate_kind == WISP_GATE_CHANNEL || c.gate_kind == WISP_GATE_ELEMENT) {
        const int64_t g0 = c.gate_kind == WISP_GATE_ELEMENT ? t * c.ld_gate : 0;
        load8(p.gate, c.gate_type, g0 + i, p.wide_g && n >= 8, n, w);
#pragma unroll
        for (int j = 0; j < 8; j++) y[k][j] *= w[j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) y[k][j] *= gt;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) x[k][j] = fmaf(c.residual_scale, x[k][j], y[k][j]);
      if (p.x_out)
        store8(p.x_out, c.x_type, t * c.ld_x_out + i, p.wide_xo && n >= 8, n, x[k]);
    }
  }
  if (p.n) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < V; k++) {
      const int n = M - (int)(k * blockDim.x + threadIdx.x) * 8;
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (j < n) s = fmaf(x[k][j], x[k][j], s);
    }
    const float r = 1.f / sqrtf(block_sum(s, buf[1]) / (float)M + c.eps);
#pragma unroll
    for (int k = 0; k < V; k++) {
      const int i = (k * blockDim.x + threadIdx.x) * 8, n = M - i;
      if (n <= 0) continue;
      float w[8];
      if (p.pre_w) {
        load8(p.pre_w, c.w_type, i, p.wide_pre && n >= 8, n, w);
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = x[k][j] * r * (c.weight_offset + w[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = x[k][j] * r;
      }
      store8(p.n, c.n_type, t * c.ld_n + i, p.wide_n && n >= 8, n, w);
    }
  }
}

}  // namespace

extern "C" WispError wisp_b200_block_norm(const WispBlockNorm* cfg, const void* d_x,
                                          const void* d_y, const void* d_gate,
                                          const void* d_post_w, const void* d_pre_w,
                                          void* d_x_out, void* d_n, cudaStream_t stream,
                                          WispErrCtx* err) {
  if (!cfg) return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: null config");
  const WispBlockNorm& c = *cfg;
  if (c.tokens < 0 || c.hidden <= 0 || c.hidden > 32768)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: tokens=%d hidden=%d (1..32768)", c.tokens,
                   c.hidden);
  if (!dt_valid(c.x_type) || !dt_valid(c.y_type) || !dt_valid(c.w_type) ||
      !dt_valid(c.gate_type) || !dt_valid(c.n_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: unknown type");
  if (c.gate_kind < WISP_GATE_NONE || c.gate_kind > WISP_GATE_ELEMENT)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: unknown gate_kind %d", c.gate_kind);
  if (!(c.eps >= 0.f)) return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: eps must be >= 0");
  if (d_y ? (!d_x_out && !d_n) : !d_n)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: no output (x_out, n)");
  if (!d_y && (c.post_norm || c.gate_kind != WISP_GATE_NONE || d_post_w))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: post norm or gate without y");
  if (d_post_w && !c.post_norm)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: post_w without post_norm");
  if (d_pre_w && !d_n) return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: pre_w without n");
  if ((c.gate_kind != WISP_GATE_NONE) != (d_gate != nullptr))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: gate and gate_kind disagree");
  if (c.ld_x < c.hidden || (d_y && c.ld_y < c.hidden) || (d_x_out && d_y && c.ld_x_out < c.hidden) ||
      (d_n && c.ld_n < c.hidden) || (c.gate_kind == WISP_GATE_ELEMENT && c.ld_gate < c.hidden))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: a row stride is less than hidden=%d", c.hidden);
  if (c.tokens == 0) return WISP_OK;
  if (!d_x) return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: null pointer argument (x)");
  if ((uintptr_t)d_x % dt_size(c.x_type) || (uintptr_t)d_y % dt_size(c.y_type) ||
      (uintptr_t)d_x_out % dt_size(c.x_type) || (uintptr_t)d_n % dt_size(c.n_type) ||
      (uintptr_t)d_post_w % dt_size(c.w_type) || (uintptr_t)d_pre_w % dt_size(c.w_type) ||
      (uintptr_t)d_gate % dt_size(c.gate_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: a buffer is not aligned to its type");
  NormParams p;
  p.c = c;
  p.x = d_x;
  p.y = d_y;
  p.gate = d_gate;
  p.post_w = d_post_w;
  p.pre_w = d_pre_w;
  p.x_out = d_x_out;
  p.n = d_n;
  auto wide = [](const void* q, int type, int64_t ld) {
    return (int)(!((uintptr_t)q & 15) && ld * dt_size(type) % 16 == 0);
  };
  p.wide_x = wide(d_x, c.x_type, c.ld_x);
  p.wide_y = wide(d_y, c.y_type, c.ld_y);
  p.wide_g = wide(d_gate, c.gate_type, c.gate_kind == WISP_GATE_ELEMENT ? c.ld_gate : 0);
  p.wide_post = wide(d_post_w, c.w_type, 0);
  p.wide_pre = wide(d_pre_w, c.w_type, 0);
  p.wide_xo = wide(d_x_out, c.x_type, c.ld_x_out);
  p.wide_n = wide(d_n, c.n_type, c.ld_n);
  const int vecs = (c.hidden + 7) / 8;
  if (vecs <= 1024 && c.tokens <= 296) {
    wb::launch_k(block_norm_kernel<1>, c.tokens, (vecs + 31) / 32 * 32, 0, stream, p);
  } else {
    const int threads = ((vecs + 3) / 4 + 31) / 32 * 32;
    wb::launch_k(block_norm_kernel<4>, c.tokens, threads, 0, stream, p);
  }
  WB_CUDA_CHECK(cudaGetLastError());
  return WISP_OK;
}
