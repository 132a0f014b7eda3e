// fp4.cu -- rows to 4-bit block-scaled codes and back, and the one-time
// layout of a weight set's scales for the product (fp4_product.cu).
//
// A block's codes are e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), so
// seven borders 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5 decide them. The result is
// the one exact arithmetic gives, so that codes do not depend on how a scale
// was divided out:
//   MX: the scale is a power of two; x / scale is exact in fp32.
//   NV: the scale is e4m3 * tensor_scale (4 + 24 significant bits). x times
//       the fp32 reciprocal of that product, made 2^-21 smaller or larger, is
//       within 2^-21.7 relative of where exact arithmetic has it (three
//       roundings and the reciprocal's ulp), so the codes of the two enclose
//       the right one. Where they differ (one value in about 800 for bf16 rows
//       under the tensor scale of their own maximum), |x| is compared with
//       border * scale by the sign of one fused multiply-add: border * e4m3 has
//       7 bits, so the difference is rounded once and its sign is right. The
//       scale byte itself is found in the same way.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "numeric.cuh"

namespace {

using namespace wb;

constexpr int kUnit = 16;   // values per thread: one NV block, half an MX block

// A row of `units` threads split over equal blocks of at most 256.
int row_threads(int units) {
  const int blocks = (units + 255) / 256;
  return ((units + blocks - 1) / blocks + 31) / 32 * 32;
}

// Codes of eight values, the first in the low nibble. Round to nearest even,
// saturating.
WB_DEV uint32_t e2m1x8(const float* v, float r) {
  uint32_t o;
  float q[8];
#pragma unroll
  for (int j = 0; j < 4; j++)     // two products per instruction
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\t"
        "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(q[2 * j]), "=f"(q[2 * j + 1])
        : "f"(v[2 * j]), "f"(v[2 * j + 1]), "f"(r));
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(o)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return o;
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

WB_DEV float e4m3_value(uint32_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}

// e4m3 of a / (6 g), nearest even, saturating. The quotient goes to fp32 by
// rounding to odd (truncate, then set the last bit when anything was cut
// off), so that the rounding to 4 significant bits decides as it would on the
// exact quotient.
__device__ __noinline__ uint32_t nv_scale_exact(float a, float g) {
  const double d = 6.0 * (double)g;
  float t = __double2float_rz((double)a / d);
  if (t < 512.f) {
    const double r = fma(-(double)t, d, (double)a);
    if (r < 0.0) t = __uint_as_float(__float_as_uint(t) - 1);
    if (r != 0.0) t = __uint_as_float(__float_as_uint(t) | 1u);
  }
  return __nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3);
}

// Tensor scales for which nothing in the fp32 decisions overflows or drops
// below fp32's last subnormal bit (the least product compared is 2^-111, of 31
// significant bits).
WB_DEV bool nv_plain_range(float g) { return g >= 1e-30f && g <= 1e30f; }

constexpr float kBelow = 1.f - 4.76837158203125e-7f, kAbove = 1.f + 4.76837158203125e-7f;  // 2^-21

// The same for a plain g: the byte of the scaled-down and scaled-up fp32
// quotient, or where those differ by the sign of border * 6 g - a.
WB_DEV uint32_t nv_scale_byte(float a, float g) {
  const float t = a * rcp_approx(6.f * g);
  const uint32_t both =
      __nv_cvt_float2_to_fp8x2(make_float2(t * kBelow, t * kAbove), __NV_SATFINITE, __NV_E4M3);
  const uint32_t lo = both & 255u, hi = both >> 8;
  if (lo == hi) return lo;
  const float border = 0.5f * (e4m3_value(lo) + e4m3_value(hi));
  const float d = fmaf(6.f * border, g, -a);
  return d < 0.f || (d == 0.f && !(hi & 1)) ? hi : lo;
}

struct QuantParams {
  const void* x;
  int64_t ld;
  int x_rows;
  const int* src;
  int rows, cols;
  const float* ts;
  uint8_t* codes;
  uint8_t* scales;
  int wide;   // rows of x start on 32-byte boundaries
};

// 16 values of one thread as they lie in memory.
template <typename T>
struct Raw {
  uint32_t u[4 * sizeof(T)];
};

template <typename T>
WB_DEV void load_raw(const T* x, bool wide, Raw<T>& r) {
  constexpr int W = 4 * sizeof(T);
  if (wide) {
#pragma unroll
    for (int j = 0; j < W / 8; j++) load32(reinterpret_cast<const uint8_t*>(x) + 32 * j, r.u + 8 * j);
  } else if (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < W; j++) r.u[j] = __ldg(reinterpret_cast<const uint32_t*>(x) + j);
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(x);
#pragma unroll
    for (int j = 0; j < W; j++) r.u[j] = __ldg(q + 2 * j) | (uint32_t)__ldg(q + 2 * j + 1) << 16;
  }
}

// Their values, and the largest magnitude's bits in fp32 (found on integers,
// so that a NaN is the largest of all).
template <typename T>
WB_DEV uint32_t unpack_raw(const Raw<T>& r, float (&v)[16]) {
  uint32_t top = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 16; j++) {
      v[j] = __uint_as_float(r.u[j]);
      top = max(top, r.u[j] & 0x7fffffffu);
    }
    return top;
  } else {
    constexpr int type = std::is_same<T, __half>::value ? WISP_DT_F16 : WISP_DT_BF16;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float2 f = unpack2(r.u[j], type);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
      top = __vmaxu2(top, r.u[j] & 0x7fff7fffu);
    }
    return __float_as_uint(unpack2(max(top & 0xffffu, top >> 16), type).x);
  }
}

// Codes and scale byte of one NV block for any g and x: every decision in
// fp64.
__device__ __noinline__ uint32_t nv_block_exact(const float (&v)[16], uint32_t top, float g,
                                                uint32_t (&code)[2]) {
  const uint32_t sb = nv_scale_exact(__uint_as_float(top), g);
  const float s = e4m3_value(sb);
  for (int j = 0; j < 16; j++) {
    const uint32_t c = (s > 0.f ? e2m1_exact(fabsf(v[j]), s, g) : 0u) |
                       (__float_as_uint(v[j]) >> 28 & 8u);
    code[j >> 3] |= c << (4 * (j & 7));
  }
  return sb;
}

// Decides the values among eight whose two candidate codes differ.
WB_DEV uint32_t nv_settle(const float* v, uint32_t lo, uint32_t hi, float r, float s, float g) {
  const uint32_t diff = lo ^ hi;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    if (diff >> (4 * j) & 15u) {
      const float ax = fabsf(v[j]);
      const float border = 0.25f * rintf(4.f * ax * r);   // borders are multiples of 1/4
      const float d = fmaf(border * s, g, -ax);
      const uint32_t even = !(hi >> (4 * j) & 1u);
      if (d < 0.f || (d == 0.f && even)) lo = (lo & ~(15u << (4 * j))) | (hi & 15u << (4 * j));
    }
  }
  return lo;
}

WB_DEV uint32_t nv_block(const float (&v)[16], uint32_t top, float g, uint32_t (&code)[2]) {
  code[0] = code[1] = 0u;
  if (top >= 0x7f800000u || !(g > 0.f && g <= 3.402823466e38f)) return 0x7f;
  if (!nv_plain_range(g)) {
    float w[16];
#pragma unroll
    for (int j = 0; j < 16; j++) w[j] = v[j];
    return nv_block_exact(w, top, g, code);
  }
  const uint32_t sb = nv_scale_byte(__uint_as_float(top), g);
  const float s = e4m3_value(sb);
  // a zero scale: zero codes with the values' signs
  const float r = sb ? rcp_approx(s * g) : 0.f;
  const float rl = r * kBelow, rh = r * kAbove;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    code[i] = e2m1x8(v + 8 * i, rl);
    const uint32_t hi = e2m1x8(v + 8 * i, rh);
    if (code[i] != hi) code[i] = nv_settle(v + 8 * i, code[i], hi, r, s, g);
  }
  return sb;
}

// grid (ceil(rows / R), ceil(cols / 16 / blockDim)): one thread per 16 values
// of R rows, 32 (16-bit types) or 64 (fp32) bytes read and 8 written for each;
// the R rows' loads are issued together. 32,768 gathered bf16 rows of 7168: MX
// 71 us (their reads, 470 MB from L2, bound it), NV 100 to 107 us (its ~190
// instructions per block do; six CTAs per SM instead of four gave 6 us).
template <bool NV, typename T, int R>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 6 : 4) quantize_kernel(const QuantParams p) {
  const int64_t row0 = (int64_t)blockIdx.x * R;
  const int u = blockIdx.y * blockDim.x + threadIdx.x;
  const int units = p.cols / kUnit;
  const bool in = u < units;
  const float g = NV ? __ldg(p.ts) : 1.f;
  Raw<T> raw[R];
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int64_t row = row0 + i;
    int64_t sr = -1;
    if (row < p.rows) sr = p.src ? (int64_t)__ldg(p.src + row) : row;
#pragma unroll
    for (int j = 0; j < 4 * (int)sizeof(T); j++) raw[i].u[j] = 0;
    if (in && sr >= 0 && sr < p.x_rows)
      load_raw(static_cast<const T*>(p.x) + sr * p.ld + (int64_t)u * kUnit, p.wide, raw[i]);
  }
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int64_t row = row0 + i, o = row * units + u;
    float v[16];
    uint32_t top = unpack_raw(raw[i], v);
    uint32_t code[2] = {0u, 0u};
    if (NV) {
      const uint32_t sb = nv_block(v, top, g, code);
      if (in && row < p.rows) {
        p.scales[o] = (uint8_t)sb;
        *reinterpret_cast<uint2*>(p.codes + o * 8) = make_uint2(code[0], code[1]);
      }
    } else {
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      uint32_t sb = 255;
      if (top < 0x7f800000u) {
        const uint32_t e = top >> 23;
        sb = e > 2 ? e - 2 : 0;
        const float inv = __uint_as_float((254u - sb) << 23);   // 2^(127 - sb)
        code[0] = e2m1x8(v, inv);
        code[1] = e2m1x8(v + 8, inv);
      }
      if (in && row < p.rows) {
        if (!(u & 1)) p.scales[o >> 1] = (uint8_t)sb;
        *reinterpret_cast<uint2*>(p.codes + o * 8) = make_uint2(code[0], code[1]);
      }
    }
  }
}

template <bool NV, typename T>
void launch_quantize_t(const QuantParams& p, cudaStream_t st) {
  const int units = p.cols / kUnit, threads = row_threads(units);
  const int gy = (units + threads - 1) / threads;
  constexpr int R = NV || sizeof(T) == 4 ? 2 : 4;
  // Several rows per thread once there are enough to fill the GPU all the same.
  if ((int64_t)p.rows * gy >= 148 * 8 * R)
    wb::launch_k(quantize_kernel<NV, T, R>, dim3((p.rows + R - 1) / R, gy), threads, 0, st, p);
  else
    wb::launch_k(quantize_kernel<NV, T, 1>, dim3(p.rows, gy), threads, 0, st, p);
}

template <bool NV>
void launch_quantize(const QuantParams& p, int type, cudaStream_t st) {
  if (type == WISP_DT_F32)
    launch_quantize_t<NV, float>(p, st);
  else if (type == WISP_DT_BF16)
    launch_quantize_t<NV, __nv_bfloat16>(p, st);
  else
    launch_quantize_t<NV, __half>(p, st);
}

struct DequantParams {
  const uint8_t* codes;
  const uint8_t* scales;
  int rows, cols;
  const float* ts;
  void* out;
  int64_t ld;
  int wide;
};

WB_DEV float2 e2m1_values(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(byte));
  return __half22float2(u2h2(h));
}

WB_DEV float scale_value(uint32_t sb, bool nv) {
  // MX 2^(sb - 127): 2^-127 is subnormal, 255 is NaN
  return nv ? e4m3_value(sb)
            : __uint_as_float(sb == 255 ? 0x7fffffffu : sb == 0 ? 0x00400000u : sb << 23);
}

// grid (ceil(rows / R), ceil(cols / 16 / blockDim)): 16 values of R rows per
// thread. fp32: in four chunks of 16 bytes blockDim apart, so that a warp's
// stores are 512 consecutive bytes (14336 x 4096: 63 -> 45 to 48 us); 16-bit types:
// 16 neighbours, read with one load and written as one sector. code * scale is
// exact in fp32 (2 x 4 significant bits); the tensor scale and the output type
// round once each.
template <bool NV, int TYPE, int R>
__global__ void __launch_bounds__(256) dequantize_kernel(const DequantParams p) {
  const int64_t row = (int64_t)blockIdx.x * R;
  const int tid = threadIdx.x;
  const float g = p.ts ? __ldg(p.ts) : 1.f;
  const uint8_t* codes = p.codes + row * (p.cols / 2);
  const uint8_t* scales = p.scales + row * (p.cols / (NV ? 16 : 32));
  if (TYPE == WISP_DT_F32) {
    const int first = blockIdx.y * blockDim.x * 4 + tid, chunks = p.cols / 4;
    uint32_t c[4];
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int u = first + i * blockDim.x;
      if (u < chunks) {
        c[i] = __ldg(reinterpret_cast<const uint16_t*>(codes) + u);
        s[i] = scale_value(__ldg(scales + (NV ? u >> 2 : u >> 3)), NV);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int u = first + i * blockDim.x;
      if (u < chunks) {
        float* q = static_cast<float*>(p.out) + row * p.ld + (int64_t)u * 4;
        const float2 f0 = e2m1_values(c[i] & 255u), f1 = e2m1_values(c[i] >> 8);
        const float4 v = make_float4(f0.x * s[i] * g, f0.y * s[i] * g, f1.x * s[i] * g, f1.y * s[i] * g);
        if (p.wide) {
          *reinterpret_cast<float4*>(q) = v;
        } else {
          q[0] = v.x;
          q[1] = v.y;
          q[2] = v.z;
          q[3] = v.w;
        }
      }
    }
  } else {
    const int u = blockIdx.y * blockDim.x + tid;
    if (u >= p.cols / kUnit) return;
    uint32_t c[R][2];
    float s[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (row + r < p.rows) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(codes + (int64_t)r * (p.cols / 2));
        c[r][0] = __ldg(q + 2 * u);
        c[r][1] = __ldg(q + 2 * u + 1);
        s[r] = scale_value(__ldg(scales + (int64_t)r * (p.cols / (NV ? 16 : 32)) + (NV ? u : u >> 1)), NV);
      }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (row + r < p.rows) {
        float v[16];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float2 f = e2m1_values((c[r][j >> 2] >> (8 * (j & 3))) & 255u);
          v[2 * j] = f.x * s[r] * g;
          v[2 * j + 1] = f.y * s[r] * g;
        }
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = pack2(v[2 * j], v[2 * j + 1], TYPE);
        uint16_t* q = static_cast<uint16_t*>(p.out) + (row + r) * p.ld + (int64_t)u * kUnit;
        if (p.wide) {
          store32(q, o);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) {
            q[2 * j] = (uint16_t)o[j];
            q[2 * j + 1] = (uint16_t)(o[j] >> 16);
          }
        }
      }
    }
  }
}

template <bool NV, int TYPE>
void launch_dequantize_t(const DequantParams& p, cudaStream_t st) {
  const int units = p.cols / kUnit, threads = row_threads(units);
  const int gy = (units + threads - 1) / threads;
  constexpr int R = TYPE == WISP_DT_F32 ? 1 : 2;
  if ((int64_t)p.rows * gy >= 148 * 8 * R)
    wb::launch_k(dequantize_kernel<NV, TYPE, R>, dim3((p.rows + R - 1) / R, gy), threads, 0, st, p);
  else
    wb::launch_k(dequantize_kernel<NV, TYPE, 1>, dim3(p.rows, gy), threads, 0, st, p);
}

template <bool NV>
void launch_dequantize(const DequantParams& p, int type, cudaStream_t st) {
  if (type == WISP_DT_F32)
    launch_dequantize_t<NV, WISP_DT_F32>(p, st);
  else if (type == WISP_DT_BF16)
    launch_dequantize_t<NV, WISP_DT_BF16>(p, st);
  else
    launch_dequantize_t<NV, WISP_DT_F16>(p, st);
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
  if (rows < 0 || rows > wb::kMaxRows || x_rows < 0 || cols <= 0 || cols % block_of(format) ||
      ld < cols)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp4_quantize: rows=%d x_rows=%d cols=%d ld=%lld (at most 2^31 - 256 rows, cols a "
                   "multiple of %d, ld >= cols)",
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
  p.ld = ld;
  p.x_rows = x_rows;
  p.src = d_src;
  p.rows = rows;
  p.cols = cols;
  p.ts = d_tensor_scale;
  p.codes = d_codes;
  p.scales = d_scales;
  p.wide = !((uintptr_t)d_x & 31) && (ld * dt_size(x_type)) % 32 == 0;
  if (format == WISP_FP4_NV)
    launch_quantize<true>(p, x_type, stream);
  else
    launch_quantize<false>(p, x_type, stream);
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
  if (rows < 0 || rows > wb::kMaxRows || cols <= 0 || cols % block_of(format) || ld < cols)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp4_dequantize: rows=%d cols=%d ld=%lld (at most 2^31 - 256 rows, cols a "
                   "multiple of %d, ld >= cols)",
                   rows, cols, (long long)ld, block_of(format));
  if (rows == 0) return WISP_OK;
  if (!d_codes || !d_scales || !d_out)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_dequantize: null pointer argument");
  if ((uintptr_t)d_codes & 3)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_dequantize: codes must be 4-byte aligned");
  if ((uintptr_t)d_out % dt_size(out_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_dequantize: out not aligned to its type");
  if (format == WISP_FP4_MX && d_tensor_scale)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_dequantize: MX rows have no tensor scale");
  DequantParams p;
  p.codes = d_codes;
  p.scales = d_scales;
  p.rows = rows;
  p.cols = cols;
  p.ts = d_tensor_scale;
  p.out = d_out;
  p.ld = ld;
  const int align = out_type == WISP_DT_F32 ? 16 : 32;
  p.wide = (uintptr_t)d_out % align == 0 && ld * dt_size(out_type) % align == 0;
  if (format == WISP_FP4_NV)
    launch_dequantize<true>(p, out_type, stream);
  else
    launch_dequantize<false>(p, out_type, stream);
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
