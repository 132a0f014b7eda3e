// fp4.cu -- rows to 4-bit block-scaled codes and back, and the one-time
// layout of a weight set's scales for the product (fp4_product.cu).
//
// A block's codes are e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), so
// seven borders 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5 decide them. The result is
// the one exact arithmetic gives, so that codes do not depend on how a scale
// was divided out:
//   MX: the scale is a power of two; x / scale is exact in fp32.
//   NV: the scale is e4m3 * tensor_scale (4 + 24 significant bits). q = x times
//       the fp32 reciprocal is within 3 roundings (2^-22.4 relative) of the
//       quotient, so the code is certain unless 4 q is within 2^-16 of an
//       integer (every border is a multiple of 0.25, and q <= 6.5 wherever
//       the border matters); those few values are decided by comparing |x|
//       with border * scale in fp64, where both are exact (31 bits).
#include <cuda_fp8.h>

#include "common.cuh"
#include "internal.h"
#include "numeric.cuh"

namespace {

using namespace wb;

constexpr int kUnit = 16;   // values per thread: one NV block, half an MX block

// Codes of (a, b): a in the low nibble. Round to nearest even, saturating.
WB_DEV uint32_t e2m1x2(float a, float b) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}"
      : "=r"(r) : "f"(a), "f"(b));
  return r;
}

// Exact code (sign excluded) of |x| over the scale s * g.
__device__ __noinline__ uint32_t e2m1_exact(float ax, float s, float g) {
  const double t = (double)s * (double)g, a = (double)ax;
  uint32_t c = a > 0.25 * t;
  c += a >= 0.75 * t;
  c += a > 1.25 * t;
  c += a >= 1.75 * t;
  c += a > 2.5 * t;
  c += a >= 3.5 * t;
  c += a > 5.0 * t;
  return c;
}

// e4m3 of a / (6 g), nearest even, saturating; exact like the codes. The
// quotient goes to fp32 by rounding to odd (truncate, then set the last bit
// when anything was cut off), so that the rounding to 4 significant bits
// decides as it would on the exact quotient.
WB_DEV uint32_t nv_scale_byte(float a, float g) {
  const double d = 6.0 * (double)g;
  float t = __double2float_rz((double)a / d);
  if (t < 512.f) {
    const double r = fma(-(double)t, d, (double)a);
    if (r < 0.0) t = __uint_as_float(__float_as_uint(t) - 1);
    if (r != 0.0) t = __uint_as_float(__float_as_uint(t) | 1u);
  }
  return __nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3);
}

WB_DEV float e4m3_value(uint32_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}

struct QuantParams {
  const void* x;
  int type;
  int64_t ld;
  int x_rows;
  const int* src;
  int cols;
  const float* ts;
  uint8_t* codes;
  uint8_t* scales;
  int wide;   // rows of x start on 16-byte boundaries
};

// grid (rows, ceil(cols / 16 / blockDim)): one thread per 16 values, 32 (bf16)
// or 64 (fp32) bytes read and 8 written.
template <bool NV>
__global__ void __launch_bounds__(256) quantize_kernel(const QuantParams p) {
  const int64_t row = blockIdx.x;
  const int u = blockIdx.y * blockDim.x + threadIdx.x;
  const int units = p.cols / kUnit;
  const bool in = u < units;
  const int64_t sr = p.src ? (int64_t)p.src[row] : row;
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; j++) v[j] = 0.f;
  if (in && sr >= 0 && sr < p.x_rows) {
    const int64_t i = sr * p.ld + (int64_t)u * kUnit;
    float a[8], b[8];
    load8(p.x, p.type, i, p.wide, 8, a);
    load8(p.x, p.type, i + 8, p.wide, 8, b);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      v[j] = a[j];
      v[8 + j] = b[j];
    }
  }
  // as integers, so that a NaN is the largest of all
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 16; j++) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  uint32_t code[2] = {0u, 0u};
  if (NV) {
    if (!in) return;
    const float g = *p.ts;
    const int64_t o = row * units + u;
    const bool bad = top >= 0x7f800000u || !(g > 0.f && g <= 3.402823466e38f);
    uint32_t sb = 0x7f;
    if (!bad) {
      sb = nv_scale_byte(__uint_as_float(top), g);
      const float s = e4m3_value(sb);
      const float t = s * g;
      if (t >= 1.1754943508e-38f) {
        const float r = __frcp_rn(t);
        float near = 1.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float q0 = v[2 * j] * r, q1 = v[2 * j + 1] * r;
          const float f0 = 4.f * q0, f1 = 4.f * q1;
          // distance to the nearest integer (the sum rounds to one); values
          // near 0 are code 0 whatever they are
          const float d0 = fabsf(f0) < 0.5f ? 1.f : fabsf(f0 - ((f0 + 12582912.f) - 12582912.f));
          const float d1 = fabsf(f1) < 0.5f ? 1.f : fabsf(f1 - ((f1 + 12582912.f) - 12582912.f));
          near = fminf(near, fminf(d0, d1));
          code[j >> 2] |= e2m1x2(q0, q1) << (8 * (j & 3));
        }
        // r itself overflows for the very smallest scales: 1 / t of a t below
        // 2^-126 never gets here, above it r <= 2^126
        if (near < 1.52587890625e-5f) {
          code[0] = code[1] = 0u;
#pragma unroll
          for (int j = 0; j < 16; j++) {
            const uint32_t c = e2m1_exact(fabsf(v[j]), s, g) |
                               (__float_as_uint(v[j]) >> 28 & 8u);
            code[j >> 3] |= c << (4 * (j & 7));
          }
        }
      } else if (s > 0.f) {
#pragma unroll
        for (int j = 0; j < 16; j++) {
          const uint32_t c = e2m1_exact(fabsf(v[j]), s, g) | (__float_as_uint(v[j]) >> 28 & 8u);
          code[j >> 3] |= c << (4 * (j & 7));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; j++)
          code[j >> 3] |= (__float_as_uint(v[j]) >> 28 & 8u) << (4 * (j & 7));
      }
    }
    p.scales[o] = (uint8_t)sb;
    *reinterpret_cast<uint2*>(p.codes + o * 8) = make_uint2(code[0], code[1]);
  } else {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    if (!in) return;
    const int64_t o = row * units + u;
    uint32_t sb = 255;
    if (top < 0x7f800000u) {
      const uint32_t e = top >> 23;
      sb = e > 2 ? e - 2 : 0;
      const float inv = __uint_as_float((254u - sb) << 23);   // 2^(127 - sb)
#pragma unroll
      for (int j = 0; j < 8; j++)
        code[j >> 2] |= e2m1x2(v[2 * j] * inv, v[2 * j + 1] * inv) << (8 * (j & 3));
    }
    if (!(u & 1)) p.scales[o >> 1] = (uint8_t)sb;
    *reinterpret_cast<uint2*>(p.codes + o * 8) = make_uint2(code[0], code[1]);
  }
}

struct DequantParams {
  const uint8_t* codes;
  const uint8_t* scales;
  int cols;
  const float* ts;
  void* out;
  int type;
  int64_t ld;
  int wide;
};

WB_DEV float2 e2m1_values(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(byte));
  return __half22float2(u2h2(h));
}

// grid (rows, ceil(cols / 8 / blockDim)): one thread per 8 values. code *
// scale is exact in fp32 (2 x 4 significant bits); the tensor scale and the
// output type round once each.
template <bool NV>
__global__ void __launch_bounds__(256) dequantize_kernel(const DequantParams p) {
  const int64_t row = blockIdx.x;
  const int u = blockIdx.y * blockDim.x + threadIdx.x;
  const int units = p.cols / 8;
  if (u >= units) return;
  const int64_t o = row * units + u;
  const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(p.codes) + o);
  const uint32_t sb = __ldg(p.scales + (NV ? o >> 1 : o >> 2));
  float s, g = 1.f;
  if (NV) {
    s = e4m3_value(sb);
    if (p.ts) g = __ldg(p.ts);
  } else {
    // 2^(sb - 127): 2^-127 is subnormal, 255 is NaN
    s = __uint_as_float(sb == 255 ? 0x7fffffffu : sb == 0 ? 0x00400000u : sb << 23);
  }
  float v[8];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float2 f = e2m1_values((c >> (8 * j)) & 255u);
    v[2 * j] = f.x * s * g;
    v[2 * j + 1] = f.y * s * g;
  }
  store8(p.out, p.type, row * p.ld + (int64_t)u * 8, p.wide, 8, v);
}

// Scale bytes [entries x n x kb] to runs of one 128-feature x 256-k stage:
// per 4 consecutive scales of a row ("word") a 512-byte tile in which row r's
// word lies at 16 (r % 32) + 4 (r / 32), the order in which tcgen05.cp
// (32x128b) spreads it over the tensor memory's lanes and columns. Rows and
// scales past the end are 0.
__global__ void __launch_bounds__(256) prepare_scales_kernel(const uint8_t* __restrict__ in, int n,
                                                             int kb, int ftiles, int nk, int words,
                                                             uint32_t* __restrict__ out,
                                                             int64_t total) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int q = (int)(i & 127);           // word within the tile
    const int64_t tile = i >> 7;
    const int w = (int)(tile % words);
    const int64_t t2 = tile / words;
    const int kk = (int)(t2 % nk);
    const int64_t t3 = t2 / nk;
    const int ft = (int)(t3 % ftiles);
    const int64_t e = t3 / ftiles;
    const int f = ft * 128 + (q >> 2) + 32 * (q & 3);
    const int k0 = (kk * words + w) * 4;
    uint32_t v = 0;
    if (f < n) {
      const uint8_t* src = in + (e * n + f) * (int64_t)kb;
#pragma unroll
      for (int b = 0; b < 4; b++)
        if (k0 + b < kb) v |= (uint32_t)src[k0 + b] << (8 * b);
    }
    out[i] = v;
  }
}

int block_of(int format) { return format == WISP_FP4_NV ? 16 : 32; }

}  // namespace

extern "C" WispError wisp_b200_fp4_quantize(const void* d_x, int x_type, int64_t ld, int x_rows,
                                            const int* d_src, int rows, int cols, int format,
                                            const float* d_tensor_scale, uint8_t* d_codes,
                                            uint8_t* d_scales, cudaStream_t stream,
                                            WispErrCtx* err) {
  if (format != WISP_FP4_MX && format != WISP_FP4_NV)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_quantize: unknown format %d", format);
  if (!dt_valid(x_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_quantize: unknown x_type %d", x_type);
  if (rows < 0 || x_rows < 0 || cols <= 0 || cols % block_of(format) || ld < cols)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp4_quantize: rows=%d x_rows=%d cols=%d ld=%lld (cols a multiple of %d, ld >= cols)",
                   rows, x_rows, cols, (long long)ld, block_of(format));
  if (!d_src && rows > x_rows)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_quantize: rows=%d > x_rows=%d without d_src", rows,
                   x_rows);
  if (rows == 0) return WISP_OK;
  if ((!d_x && x_rows > 0) || !d_codes || !d_scales || (format == WISP_FP4_NV && !d_tensor_scale))
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp4_quantize: null pointer argument (x, codes, scales, the NV tensor scale)");
  if ((uintptr_t)d_codes & 7)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_quantize: codes must be 8-byte aligned");
  if ((uintptr_t)d_x % dt_size(x_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_quantize: x not aligned to its type");
  QuantParams p;
  p.x = d_x;
  p.type = x_type;
  p.ld = ld;
  p.x_rows = x_rows;
  p.src = d_src;
  p.cols = cols;
  p.ts = d_tensor_scale;
  p.codes = d_codes;
  p.scales = d_scales;
  p.wide = !((uintptr_t)d_x & 15) && (ld * dt_size(x_type)) % 16 == 0;
  const int units = cols / kUnit;
  const int threads = units >= 256 ? 256 : (units + 31) / 32 * 32;
  const dim3 grid(rows, (units + threads - 1) / threads);
  if (format == WISP_FP4_NV)
    wb::launch_k(quantize_kernel<true>, grid, threads, 0, stream, p);
  else
    wb::launch_k(quantize_kernel<false>, grid, threads, 0, stream, p);
  WB_CUDA_CHECK(cudaGetLastError());
  return WISP_OK;
}

extern "C" WispError wisp_b200_fp4_dequantize(const uint8_t* d_codes, const uint8_t* d_scales,
                                              int rows, int cols, int format,
                                              const float* d_tensor_scale, void* d_out,
                                              int out_type, int64_t ld, cudaStream_t stream,
                                              WispErrCtx* err) {
  if (format != WISP_FP4_MX && format != WISP_FP4_NV)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_dequantize: unknown format %d", format);
  if (!dt_valid(out_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_dequantize: unknown out_type %d", out_type);
  if (rows < 0 || cols <= 0 || cols % block_of(format) || ld < cols)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp4_dequantize: rows=%d cols=%d ld=%lld (cols a multiple of %d, ld >= cols)",
                   rows, cols, (long long)ld, block_of(format));
  if (rows == 0) return WISP_OK;
  if (!d_codes || !d_scales || !d_out)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_dequantize: null pointer argument");
  if ((uintptr_t)d_codes & 3)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_dequantize: codes must be 4-byte aligned");
  if ((uintptr_t)d_out % dt_size(out_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_dequantize: out not aligned to its type");
  DequantParams p;
  p.codes = d_codes;
  p.scales = d_scales;
  p.cols = cols;
  p.ts = d_tensor_scale;
  p.out = d_out;
  p.type = out_type;
  p.ld = ld;
  p.wide = !((uintptr_t)d_out & 15) && (ld * dt_size(out_type)) % 16 == 0;
  const int units = cols / 8;
  const int threads = units >= 256 ? 256 : (units + 31) / 32 * 32;
  const dim3 grid(rows, (units + threads - 1) / threads);
  if (format == WISP_FP4_NV)
    wb::launch_k(dequantize_kernel<true>, grid, threads, 0, stream, p);
  else
    wb::launch_k(dequantize_kernel<false>, grid, threads, 0, stream, p);
  WB_CUDA_CHECK(cudaGetLastError());
  return WISP_OK;
}

namespace {

// 32-bit words of one prepared set.
int64_t prepared_words(const WispFp4Config* c) {
  const int64_t ft = ((int64_t)c->n + 127) / 128, nk = ((int64_t)c->k + 255) / 256;
  return c->n_entries * ft * nk * (c->format == WISP_FP4_NV ? 4 : 2) * 128;
}

}  // namespace

WispError wb::fp4_validate(const WispFp4Config* c, const char* who, WispErrCtx* err) {
  if (!c) return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: null config", who);
  if (c->format != WISP_FP4_MX && c->format != WISP_FP4_NV)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: unknown format %d", who, c->format);
  if (c->n_entries <= 0 || c->n <= 0 || c->k <= 0 || c->k % 32)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: n_entries=%d n=%d k=%d (k a multiple of 32)", who,
                   c->n_entries, c->n, c->k);
  // the tensor map's row index (entries x n, plus one tile) is 32-bit
  if ((int64_t)c->n_entries * c->n > 0x7fffff00LL)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: n_entries * n = %lld exceeds 2^31", who,
                   (long long)c->n_entries * c->n);
  if (!dt_valid(c->out_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: unknown out_type %d", who, c->out_type);
  return WISP_OK;
}

extern "C" size_t wisp_b200_fp4_prepared_bytes(const WispFp4Config* cfg) {
  if (wb::fp4_validate(cfg, "fp4_prepared_bytes", nullptr) != WISP_OK) return 0;
  return (size_t)prepared_words(cfg) * 4;
}

extern "C" WispError wisp_b200_fp4_prepare(const WispFp4Config* cfg, const uint8_t* d_scales,
                                           void* d_prepared, size_t prepared_bytes,
                                           cudaStream_t stream, WispErrCtx* err) {
  WispError e = wb::fp4_validate(cfg, "fp4_prepare", err);
  if (e != WISP_OK) return e;
  if (!d_scales || !d_prepared)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_prepare: null pointer argument");
  if ((uintptr_t)d_prepared & 255)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_prepare: prepared must be 256-byte aligned");
  const int64_t total = prepared_words(cfg);
  if (prepared_bytes < (size_t)total * 4)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_prepare: prepared buffer %zu < required %zu",
                   prepared_bytes, (size_t)total * 4);
  const int64_t blocks = (total + 255) / 256;
  wb::launch_k(prepare_scales_kernel, (unsigned)(blocks < 148 * 32 ? blocks : 148 * 32), 256, 0,
               stream, d_scales, cfg->n, cfg->k / block_of(cfg->format), (cfg->n + 127) / 128,
               (cfg->k + 255) / 256, cfg->format == WISP_FP4_NV ? 4 : 2,
               static_cast<uint32_t*>(d_prepared), total);
  WB_CUDA_CHECK(cudaGetLastError());
  return WISP_OK;
}
