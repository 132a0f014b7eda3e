// norm.cu -- the norms after and before a block with its gate and residual:
//   p = y / rms(y) * (o + w_post),  x' = rs * x + gate * p,
//   n = x' / rms(x') * (o + w_pre)
// A row's x and y are held by one CTA, so each input is read once and each
// output written once and the bound is HBM (and, for a few rows, the latency
// of one load, two block sums and one store). n is taken from the fp32 x'.
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
  float inv_m;     // 1 / hidden
};

// 1 / rms from the mean square (rsqrt: 2 ulp at most, under the sum's own error).
WB_DEV float inv_rms(float mean_sq, float eps) { return rsqrtf(mean_sq + eps); }

// Sums of N values over the block, the same bits in every thread.
template <int N>
WB_DEV void block_sum(float (&v)[N], float (*buf)[32]) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  const int warps = (blockDim.x + 31) >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; i++) buf[i][threadIdx.x >> 5] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = lane < warps ? buf[i][lane] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
}

WB_DEV float square_sum(const float (&v)[8], float s) {
#pragma unroll
  for (int j = 0; j < 8; j++) s = fmaf(v[j], v[j], s);
  return s;
}

// A row's values over nt threads, vectors of 8: thread i of `VEC` kernels holds
// elements 8 (k nt + i) .. + 7; otherwise (a row that does not start on 16
// bytes) elements (8 k + j) nt + i, so that a warp's single loads are
// consecutive.
template <typename T>
WB_DEV void load_strided(const T* q, int M, int e, int nt, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j++, e += nt) v[j] = e < M ? (float)q[e] : 0.f;
}
template <typename T>
WB_DEV void store_strided(T* q, int M, int e, int nt, const float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j++, e += nt)
    if (e < M) q[e] = (T)v[j];        // (the 16-bit types round to nearest even)
}

template <bool VEC>
WB_DEV void load_row(const void* q, int type, int64_t base, int k, int M, int i, int nt,
                     float (&v)[8]) {
  if (VEC) {
    const int e = (k * nt + i) * 8;
    if (e < M) {
      load8(q, type, base + e, true, 8, v);
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = 0.f;
  } else {
    const int e = 8 * k * nt + i;
    if (type == WISP_DT_F32)
      load_strided(static_cast<const float*>(q) + base, M, e, nt, v);
    else if (type == WISP_DT_BF16)
      load_strided(static_cast<const __nv_bfloat16*>(q) + base, M, e, nt, v);
    else
      load_strided(static_cast<const __half*>(q) + base, M, e, nt, v);
  }
}

template <bool VEC>
WB_DEV void store_row(void* q, int type, int64_t base, int k, int M, int i, int nt,
                      const float (&v)[8]) {
  if (VEC) {
    const int e = (k * nt + i) * 8;
    if (e < M) store8(q, type, base + e, true, 8, v);
  } else {
    const int e = 8 * k * nt + i;
    if (type == WISP_DT_F32)
      store_strided(static_cast<float*>(q) + base, M, e, nt, v);
    else if (type == WISP_DT_BF16)
      store_strided(static_cast<__nv_bfloat16*>(q) + base, M, e, nt, v);
    else
      store_strided(static_cast<__half*>(q) + base, M, e, nt, v);
  }
}

// One row over nt threads; `sum` adds a value over them (round: 0, then 1).
template <int V, bool VEC, typename Sum>
WB_DEV void norm_row(const NormParams& p, int64_t t, int i, int nt, Sum sum) {
  const WispBlockNorm& c = p.c;
  const int M = c.hidden;
  float x[V][8], y[V][8];
#pragma unroll
  for (int k = 0; k < V; k++) {
    if (p.y) load_row<VEC>(p.y, c.y_type, t * c.ld_y, k, M, i, nt, y[k]);
    load_row<VEC>(p.x, c.x_type, t * c.ld_x, k, M, i, nt, x[k]);
  }
  if (p.y) {
    float r = 1.f;
    if (c.post_norm) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < V; k++) s = square_sum(y[k], s);
      r = inv_rms(sum(s, 0) * p.inv_m, c.eps);
    }
    if (c.gate_kind == WISP_GATE_TOKEN) r *= load_one(p.gate, c.gate_type, t);
#pragma unroll
    for (int k = 0; k < V; k++) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; j++) y[k][j] *= r;
      if (p.post_w) {
        load_row<VEC>(p.post_w, c.w_type, 0, k, M, i, nt, w);
#pragma unroll
        for (int j = 0; j < 8; j++) y[k][j] *= c.weight_offset + w[j];
      }
      if (c.gate_kind == WISP_GATE_CHANNEL || c.gate_kind == WISP_GATE_ELEMENT) {
        load_row<VEC>(p.gate, c.gate_type, c.gate_kind == WISP_GATE_ELEMENT ? t * c.ld_gate : 0, k,
                      M, i, nt, w);
#pragma unroll
        for (int j = 0; j < 8; j++) y[k][j] *= w[j];
      }
#pragma unroll
      for (int j = 0; j < 8; j++) x[k][j] = fmaf(c.residual_scale, x[k][j], y[k][j]);
      if (p.x_out) store_row<VEC>(p.x_out, c.x_type, t * c.ld_x_out, k, M, i, nt, x[k]);
    }
  }
  if (p.n) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < V; k++) s = square_sum(x[k], s);
    const float r = inv_rms(sum(s, 1) * p.inv_m, c.eps);
#pragma unroll
    for (int k = 0; k < V; k++) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; j++) x[k][j] *= r;
      if (p.pre_w) {
        load_row<VEC>(p.pre_w, c.w_type, 0, k, M, i, nt, w);
#pragma unroll
        for (int j = 0; j < 8; j++) x[k][j] *= c.weight_offset + w[j];
      }
      store_row<VEC>(p.n, c.n_type, t * c.ld_n, k, M, i, nt, x[k]);
    }
  }
}

// Rows of at most 512: one per warp, no barrier (65,536 rows of 64: 59 us with
// the ring below, 26 so; 16,384 of 1024 the other way round, 35 and 47). At 64
// columns 8 of the 32 lanes hold values: four times the copy rate's 6.4 us.
constexpr int kNormWarps = 8;
template <int V, bool VEC>
__global__ void __launch_bounds__(32 * kNormWarps)
block_norm_warp_kernel(const __grid_constant__ NormParams p) {
  const int64_t t = (int64_t)blockIdx.x * kNormWarps + (threadIdx.x >> 5);
  if (t >= p.c.tokens) return;
  norm_row<V, VEC>(p, t, threadIdx.x & 31, 32, [](float s, int) {
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  });
}

// One row per CTA, V vectors of 8 a thread: as few as 1024 threads allow, since
// 64 registers hold two of x and y and spill four. (bf16 x, fp32 y, by two
// instead of four: 4096 x 8200 113 -> 82 us, 2048 x 16384 100 -> 88, 16 x 16384
// 14.3 -> 10.2. Above 16384 four remain: 1024 x 32768 109 to 114 us = 3.0 TB/s.)
template <int V, int THREADS, bool VEC>
__global__ void __launch_bounds__(THREADS) block_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float buf[2][1][32];
  norm_row<V, VEC>(p, blockIdx.x, threadIdx.x, blockDim.x, [&](float s, int round) {
    float v[1] = {s};
    block_sum(v, buf[round]);
    return v[0];
  });
}

template <bool VEC>
void launch_rows(const NormParams& p, cudaStream_t st) {
  const int T = p.c.tokens, vecs = (p.c.hidden + 7) / 8;
  const int blocks = (T + kNormWarps - 1) / kNormWarps;
  if (vecs <= 32)
    wb::launch_k(block_norm_warp_kernel<1, VEC>, blocks, 32 * kNormWarps, 0, st, p);
  else if (vecs <= 64)
    wb::launch_k(block_norm_warp_kernel<2, VEC>, blocks, 32 * kNormWarps, 0, st, p);
  else if (vecs <= 1024)
    wb::launch_k(block_norm_kernel<1, 1024, VEC>, T, (vecs + 31) / 32 * 32, 0, st, p);
  else if (vecs <= 2048)
    wb::launch_k(block_norm_kernel<2, 1024, VEC>, T, ((vecs + 1) / 2 + 31) / 32 * 32, 0, st, p);
  else
    wb::launch_k(block_norm_kernel<4, 1024, VEC>, T, ((vecs + 3) / 4 + 31) / 32 * 32, 0, st, p);
}

// Many rows: persistent CTAs that take rows blockIdx.x, + gridDim.x, ..., whose
// x and y arrive through a ring of bulk copies, so that the memory stays busy
// while a row's sums go round the CTA. A thread holds 8 columns, and their
// weights and channel gate for good. The sum of a row's x'^2 goes round
// together with the sum of the next row's y^2: one barrier per row. (At 4096 x
// 7168, 10 bytes a value, one row per CTA took 117 us, this ring with two sums
// after one another 64, with one 59 to 61 with L2 flushed, 55 = 5.3 TB/s back to
// back; 45 us are the copy rate. What is left is the issue of 28 warps'
// arithmetic between two barriers. Rows that start anywhere, whose values are
// read and written one by one: 3952 x 3373 44 to 51 us, copy rate 20.)
constexpr int kNormStages = 8;
__device__ int norm_error;     // kErrorTimeout: a copy never landed
struct RingShape {
  int stages, x_bytes, y_bytes;
};

// Rows that do not start on 16 bytes (VEC false) come as the 16-byte words
// around them, and a thread then has columns tid, + threads, ...
WB_DEV int64_t word_start(const void* q, int64_t byte) {
  return (int64_t)((uintptr_t)q + byte) & ~(int64_t)15;
}

template <bool VEC>
__global__ void __launch_bounds__(1024, 1)
block_norm_stream_kernel(const __grid_constant__ NormParams p, const RingShape rs) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ uint64_t full[kNormStages];
  __shared__ float buf[2][2][32];
  __shared__ int abort, late;
  const WispBlockNorm& c = p.c;
  const int M = c.hidden, tid = threadIdx.x, nt = blockDim.x, T = c.tokens;
  const int stage = rs.x_bytes + rs.y_bytes;
  const int64_t sx = c.ld_x * dt_size(c.x_type), sy = c.ld_y * dt_size(c.y_type);
  // bytes of a row in its words
  auto words = [&](const void* q, int64_t at, int type) {
    return (uint32_t)(word_start(q, at + M * dt_size(type) + 15) - word_start(q, at));
  };
  auto issue = [&](int s, int64_t t) {
    uint32_t bx = rs.x_bytes, by = rs.y_bytes;
    if (!VEC) {
      bx = words(p.x, t * sx, c.x_type);
      if (by) by = words(p.y, t * sy, c.y_type);
    }
    mbar_arrive_expect_tx(&full[s], bx + by);
    bulk_load(ring + s * stage, reinterpret_cast<const void*>(word_start(p.x, t * sx)), bx, &full[s]);
    if (by)
      bulk_load(ring + s * stage + rs.x_bytes,
                reinterpret_cast<const void*>(word_start(p.y, t * sy)), by, &full[s]);
  };
  int issued = 0;      // rows (thread 0)
  if (tid == 0) {
    abort = late = 0;
    for (int i = 0; i < rs.stages; i++) mbar_init(&full[i], 1);
    fence_barrier_init();
    for (int i = 0; i < rs.stages; i++) {
      const int64_t t = blockIdx.x + (int64_t)i * gridDim.x;
      if (t < T) {
        issue(i, t);
        issued++;
      }
    }
  }
  // A thread has columns if it has a first one. (VEC: all eight are there then,
  // and the accesses check nothing; with a check in each, 4096 x 7168 took 63.5
  // us instead of 59.4.)
  const bool in = (VEC ? tid * 8 : tid) < M;
  auto load_cols = [&](const void* q, int type, int64_t base, float (&v)[8]) {
    if (VEC)
      load8(q, type, base + tid * 8, true, 8, v);
    else
      load_row<false>(q, type, base, 0, M, tid, nt, v);
  };
  auto store_cols = [&](void* q, int type, int64_t base, const float (&v)[8]) {
    if (VEC)
      store8(q, type, base + tid * 8, true, 8, v);
    else
      store_row<false>(q, type, base, 0, M, tid, nt, v);
  };
  // columns' factors: a of y / rms(y), b of x' / rms(x')
  float a[8], b[8], w[8];
#pragma unroll
  for (int j = 0; j < 8; j++) a[j] = b[j] = 1.f;
  if (p.post_w) {
    load_row<VEC>(p.post_w, c.w_type, 0, 0, M, tid, nt, w);
#pragma unroll
    for (int j = 0; j < 8; j++) a[j] = c.weight_offset + w[j];
  }
  if (c.gate_kind == WISP_GATE_CHANNEL) {
    load_row<VEC>(p.gate, c.gate_type, 0, 0, M, tid, nt, w);
#pragma unroll
    for (int j = 0; j < 8; j++) a[j] *= w[j];
  }
  if (p.pre_w) {
    load_row<VEC>(p.pre_w, c.w_type, 0, 0, M, tid, nt, w);
#pragma unroll
    for (int j = 0; j < 8; j++) b[j] = c.weight_offset + w[j];
  }
  int s = 0, flip = 0;
  uint32_t ph = 0;
  float x[8], y[8];
  // The ring's next row into x and y. A copy that never lands (the wait is
  // bounded) makes its row and later ones NaN: a thread that has given up waits
  // no more, since a slot's parity could then stand for an older phase, and
  // thread 0 then issues no more (while it has seen a slot's copy land, the slot
  // is free, whatever other threads saw). The slot may be refilled after the
  // next barrier.
  bool ok = true;
  auto take = [&](int64_t t) {
    ok = ok && mbar_wait(&full[s], ph, &abort);
    const uint8_t* st = ring + s * stage;
    const float none = ok ? 0.f : __uint_as_float(0x7fffffffu);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = y[j] = none;
    if (in && ok) {
      const int ox = VEC ? 0 : (int)((uintptr_t)p.x + t * sx) & 15;
      load_cols(st + ox, c.x_type, 0, x);
      if (p.y) {
        const int oy = VEC ? 0 : (int)((uintptr_t)p.y + t * sy) & 15;
        load_cols(st + rs.x_bytes + oy, c.y_type, 0, y);
      }
    }
  };
  auto refill = [&](int64_t t) {      // the slot row t was taken from
    if (tid == 0) {
      const int64_t next = t + (int64_t)rs.stages * gridDim.x;
      if (next < T && ok) {
        issue(s, next);
        issued++;
      }
    }
    if (++s == rs.stages) {
      s = 0;
      ph ^= 1;
    }
  };
#pragma unroll
  for (int j = 0; j < 8; j++) y[j] = 0.f;
  __syncthreads();
  int64_t t = blockIdx.x;
  take(t);
  float q[2] = {0.f, square_sum(y, 0.f)};
  block_sum(q, buf[flip]);
  refill(t);
  for (; t < T; t += gridDim.x) {
    flip ^= 1;
    if (p.y) {
      float r = c.post_norm ? inv_rms(q[1] * p.inv_m, c.eps) : 1.f;
      if (c.gate_kind == WISP_GATE_TOKEN) r *= load_one(p.gate, c.gate_type, t);
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] *= r * a[j];
      if (c.gate_kind == WISP_GATE_ELEMENT && in) {
        float w[8];
        load_cols(p.gate, c.gate_type, t * c.ld_gate, w);
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] *= w[j];
      }
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = fmaf(c.residual_scale, x[j], y[j]);
      if (p.x_out && in) store_cols(p.x_out, c.x_type, t * c.ld_x_out, x);
    }
    float xp[8];
#pragma unroll
    for (int j = 0; j < 8; j++) xp[j] = x[j];
    q[0] = square_sum(x, 0.f);
    const int64_t tn = t + gridDim.x;
    if (tn < T) take(tn);
    q[1] = square_sum(y, 0.f);
    block_sum(q, buf[flip]);
    if (tn < T) refill(tn);
    if (p.n && in) {
      const float r = inv_rms(q[0] * p.inv_m, c.eps);
#pragma unroll
      for (int j = 0; j < 8; j++) xp[j] *= r * b[j];
      store_cols(p.n, c.n_type, t * c.ld_n, xp);
    }
  }
  // (every wait lies before the last barrier)
  if (tid == 0 && *static_cast<volatile int*>(&abort)) {
    atomicOr(&norm_error, kErrorTimeout);
    // let the copies in flight land before the CTA's memory goes away
    for (int i = max(issued - rs.stages, 0); i < issued; i++)
      mbar_wait(&full[i % rs.stages], i / rs.stages & 1, &late, 20000000LL);
  }
}

}  // namespace

extern "C" int* wisp_b200_block_norm_error_word(void) {
  void* p = nullptr;
  return cudaGetSymbolAddress(&p, norm_error) == cudaSuccess ? static_cast<int*>(p) : nullptr;
}

extern "C" WispError wisp_b200_block_norm(const WispBlockNorm* cfg, const void* d_x,
                                          const void* d_y, const void* d_gate,
                                          const void* d_post_w, const void* d_pre_w,
                                          void* d_x_out, void* d_n, cudaStream_t stream,
                                          WispErrCtx* err) {
  if (!cfg) return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: null config");
  const WispBlockNorm& c = *cfg;
  if (c.tokens < 0 || c.tokens > wb::kMaxRows || c.hidden <= 0 || c.hidden > 32768)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "block_norm: tokens=%d (at most 2^31 - 256) hidden=%d (1..32768)", c.tokens,
                   c.hidden);
  if (!dt_valid(c.x_type) || !dt_valid(c.y_type) || !dt_valid(c.w_type) ||
      !dt_valid(c.gate_type) || !dt_valid(c.n_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: unknown type");
  if (c.gate_kind < WISP_GATE_NONE || c.gate_kind > WISP_GATE_ELEMENT)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: unknown gate_kind %d", c.gate_kind);
  if (!(c.eps >= 0.f)) return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: eps must be >= 0");
  if (c.tokens == 0) return WISP_OK;     // (buffers of no rows may have no address)
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
  if (!d_x) return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: null pointer argument (x)");
  if (d_y && d_x_out == d_x && c.ld_x_out != c.ld_x && c.tokens > 1)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "block_norm: x_out in place with another row stride");
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
  p.inv_m = 1.f / (float)c.hidden;
  auto wide = [](const void* q, int type, int64_t ld) {
    return !((uintptr_t)q & 15) && ld * dt_size(type) % 16 == 0;
  };
  const bool vec =
      c.hidden % 8 == 0 && wide(d_x, c.x_type, c.ld_x) && (!d_y || wide(d_y, c.y_type, c.ld_y)) &&
      wide(d_gate, c.gate_type, c.gate_kind == WISP_GATE_ELEMENT ? c.ld_gate : 0) &&
      wide(d_post_w, c.w_type, 0) && wide(d_pre_w, c.w_type, 0) &&
      (!p.x_out || wide(d_x_out, c.x_type, c.ld_x_out)) && (!d_n || wide(d_n, c.n_type, c.ld_n));
  const int threads1 = (c.hidden + 255) / 256 * 32, T = c.tokens;    // a vector of 8 each
  int dev = 0, sms = 0;
  WB_CUDA_CHECK(wb::device_sms(&dev, &sms));
  if (threads1 > 64 && threads1 <= 1024 && T > 2 * sms) {
    RingShape rs;
    auto room = [&](int type) {     // the words of a row that starts anywhere
      const int bytes = c.hidden * dt_size(type);
      return vec ? bytes : (bytes + 15) / 16 * 16 + 16;
    };
    rs.x_bytes = room(c.x_type);
    rs.y_bytes = d_y ? room(c.y_type) : 0;
    // as many CTAs per SM as make 1024 threads, which share its memory
    const int ctas = 1024 / threads1 < 8 ? 1024 / threads1 : 8;
    const int budget = 200 * 1024 / ctas, stage = rs.x_bytes + rs.y_bytes;
    rs.stages = budget / stage < kNormStages ? budget / stage : kNormStages;
    const int grid = ctas * sms < T ? ctas * sms : T;
    auto kernel = vec ? block_norm_stream_kernel<true> : block_norm_stream_kernel<false>;
    static std::atomic<uint64_t> raised[2];
    WB_CUDA_CHECK(wb::raise_smem(kernel, 200 * 1024, dev, raised[vec]));
    wb::launch_k(kernel, grid, threads1, (size_t)rs.stages * stage, stream, p, rs);
  } else if (vec) {
    launch_rows<true>(p, stream);
  } else {
    launch_rows<false>(p, stream);
  }
  WB_CUDA_CHECK(cudaGetLastError());
  return WISP_OK;
}
