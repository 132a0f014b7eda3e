// fp8.cu -- rows to e4m3 codes with one fp32 scale per 128 values and back, and
// matrices to codes with one per block of 128 x 128.
//
// scale = fp32(max|x| / 448) or the least power of two that is not below max|x| /
// 448; a code is the e4m3 value nearest to x / scale, ties to the even code. The
// result is the one exact arithmetic gives, so that codes do not depend on how the
// scale was divided out: x times the fp32 reciprocal of the scale, made 2^-21
// smaller or larger, is within 2^-22 relative of where exact arithmetic has it (a
// reciprocal's ulp and two roundings), so the codes of the two enclose the right
// one. Where they differ, |x| is compared with border * scale by the sign of one
// fused multiply-add: a border has 5 significant bits, so the difference is rounded
// once and its sign is right. (For 16-bit rows that is no rare event: the quotient of
// two 8-bit significands by 7 * 64 lies on a border for one value in a few hundred.)
// With a power of two as the scale the first product is exact.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "numeric.cuh"

namespace {

using namespace wb;

constexpr int kUnit = 16;      // values per thread; 8 threads hold a block of 128
constexpr int kBlock = 128;
constexpr int kLanes = kBlock / kUnit;
constexpr int kMaxCols = 1 << 27;    // what a launch's grid holds, with room
constexpr float kTop = 448.f;
// Below this, products and remainders of fp32 may lose bits to its range.
constexpr float kTiny = 1e-30f, kRaise = 1.2676506002282294e30f;     // 2^100
constexpr float kBelow = 1.f - 4.76837158203125e-7f, kAbove = 1.f + 4.76837158203125e-7f;  // 2^-21

constexpr int kSms = 148;      // a B200's; layouts depend on it, results do not

// How `rows` rows of `cols` values lie over the grid, at R rows per thread: a row's
// threads over equal CTAs of at most 256, or, of short rows, several in one CTA as long as
// that leaves four CTAs an SM (100,000 bf16 rows of 64, us: quantise 23.6 -> 9.6, back 27.3 ->
// 4.6; 65,536 of 128: 17.3 -> 8.0, 18.5 -> 4.1).
struct Layout {
  dim3 grid, block;
};
Layout layout_rows(int rows, int cols, int R) {
  const int units = (cols + kBlock - 1) / kBlock * kLanes;
  for (int k = 256 / units; k > 1; k--)
    if (units * k % 32 == 0 && rows >= (int64_t)kSms * 4 * R * k)
      return {dim3(((int64_t)rows + R * k - 1) / (R * k)), dim3(units, k)};
  const int parts = (units + 255) / 256;
  const int threads = ((units + parts - 1) / parts + 31) / 32 * 32;
  return {dim3(((int64_t)rows + R - 1) / R, (units + threads - 1) / threads), dim3(threads)};
}
// Several rows per thread once there are enough to fill the GPU all the same.
bool many_rows(int rows, int cols, int R) {
  return (int64_t)rows * layout_rows(1, cols, 1).grid.y >= kSms * 8 * R;
}

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

// The bits of the largest magnitude in fp32 (found on integers, so that a NaN is
// the largest of all).
template <typename T>
WB_DEV uint32_t top_of(const Raw<T>& r) {
  uint32_t top = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 16; j++) top = max(top, r.u[j] & 0x7fffffffu);
    return top;
  } else {
    constexpr int type = std::is_same<T, __half>::value ? WISP_DT_F16 : WISP_DT_BF16;
#pragma unroll
    for (int j = 0; j < 8; j++) top = __vmaxu2(top, r.u[j] & 0x7fff7fffu);
    return __float_as_uint(unpack2(max(top & 0xffffu, top >> 16), type).x);
  }
}

template <typename T>
WB_DEV float2 pair_of(const Raw<T>& r, int j) {
  if constexpr (sizeof(T) == 4)
    return make_float2(__uint_as_float(r.u[2 * j]), __uint_as_float(r.u[2 * j + 1]));
  else
    return unpack2(r.u[j], std::is_same<T, __half>::value ? WISP_DT_F16 : WISP_DT_BF16);
}

// The scale of a block whose largest magnitude has the bits `top`. An infinity or
// a NaN in the block: NaN.
template <bool POW2>
WB_DEV float scale_of(uint32_t top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  if (!POW2) {
    // a / 448 rounded to nearest: the quotient by the rounded reciprocal, corrected
    // once by its exact remainder (Markstein 1990: the correction by a correctly
    // rounded reciprocal gives the correctly rounded quotient). Where the remainder
    // would drop below fp32's last bit, the same in fp64. (A division is a call, which
    // keeps registers of what comes after it.)
    const float a = __uint_as_float(top);
    if (a < kTiny) {
      constexpr double r = 1.0 / kTop;
      const double q = a * r;
      return (float)fma(fma(-q, (double)kTop, (double)a), r, q);
    }
    constexpr float r = 1.f / kTop;
    const float q = a * r;
    return fmaf(fmaf(-q, kTop, a), r, q);
  }
  // top = m 2^e, 448 = 1.75 2^8: 2^(e - 8), one more where m > 1.75
  if (top == 0) return 0.f;
  const int e = (int)((top + 0x1fffffu) >> 23) - 8;
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// Codes of four values, the first in the low byte. Round to nearest even,
// saturating.
WB_DEV uint32_t e4m3x4(float2 a, float2 b, float r) {
  uint32_t o;
  asm("{\n\t.reg .b64 x, y, z;\n\t.reg .b16 p, q;\n\t.reg .f32 f, g;\n\t"
      "mov.b64 z, {%5, %5};\n\tmov.b64 x, {%1, %2};\n\tmov.b64 y, {%3, %4};\n\t"
      "mul.rn.f32x2 x, x, z;\n\tmul.rn.f32x2 y, y, z;\n\t"
      "mov.b64 {f, g}, x;\n\tcvt.rn.satfinite.e4m3x2.f32 p, g, f;\n\t"
      "mov.b64 {f, g}, y;\n\tcvt.rn.satfinite.e4m3x2.f32 q, g, f;\n\t"
      "mov.b32 %0, {p, q};\n\t}"
      : "=r"(o) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(r));
  return o;
}

// The codes of a thread's 16 values, which lie at x.
template <bool POW2, typename T>
WB_DEV void codes_of(Raw<T> raw, const T* x, float s, uint32_t (&c)[4]) {
  c[0] = c[1] = c[2] = c[3] = 0u;
  if (!(s > 0.f)) return;           // a zero block, or NaN
  float raise = 1.f;
  if (!POW2 && !std::is_same<T, __half>::value && s < kTiny) {
    // the same quotients from values and scale times 2^100, which is exact (fp16 has
    // no values as small)
    raise = kRaise;
    s *= kRaise;
#pragma unroll
    for (int j = 0; j < (int)(4 * sizeof(T)); j++) {
      if constexpr (sizeof(T) == 4) {
        raw.u[j] = __float_as_uint(__uint_as_float(raw.u[j]) * kRaise);
      } else {
        const float2 v = pair_of(raw, j);
        raw.u[j] = pack2(v.x * kRaise, v.y * kRaise, WISP_DT_BF16);
      }
    }
  }
  const float r = POW2 ? __uint_as_float(0x7f000000u - __float_as_uint(s)) : rcp_approx(s);
  uint32_t hi[4], differ = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 a = pair_of(raw, 2 * i), b = pair_of(raw, 2 * i + 1);
    c[i] = e4m3x4(a, b, POW2 ? r : r * kBelow);
    if (!POW2) {
      hi[i] = e4m3x4(a, b, r * kAbove);
      differ |= c[i] ^ hi[i];
    }
  }
  if (!POW2 && differ) {
    // One value of each lane after the other.
    uint32_t left = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)      // a bit per byte that differs
      left |= ((__vcmpne4(c[i], hi[i]) & 0x08040201u) * 0x01010101u >> 24) << 4 * i;
#pragma unroll 1
    do {
      const int j = __ffs(left) - 1, i = j >> 2, at = 8 * (j & 3);
      left &= left - 1;
      const uint32_t cl = i < 2 ? (i < 1 ? c[0] : c[1]) : (i < 3 ? c[2] : c[3]);
      const uint32_t ch = i < 2 ? (i < 1 ? hi[0] : hi[1]) : (i < 3 ? hi[2] : hi[3]);
      float ax;
      if constexpr (sizeof(T) == 4) {
        ax = fabsf(x[j]) * raise;       // (rare: read again)
      } else {
        const int w = j >> 1;
        const uint32_t w0 = w & 1 ? raw.u[1] : raw.u[0], w1 = w & 1 ? raw.u[3] : raw.u[2];
        const uint32_t w2 = w & 1 ? raw.u[5] : raw.u[4], w3 = w & 1 ? raw.u[7] : raw.u[6];
        const uint32_t lo = w & 2 ? w1 : w0, up = w & 2 ? w3 : w2;
        const float2 v = unpack2(w & 4 ? up : lo,
                                 std::is_same<T, __half>::value ? WISP_DT_F16 : WISP_DT_BF16);
        ax = fabsf(j & 1 ? v.y : v.x);
      }
      // the border: the quotient, which is next to it, to 5 significant bits
      const float border = __uint_as_float((__float_as_uint(ax * r) + 0x40000u) & 0xfff80000u);
      const float d = fmaf(border, s, -ax);
      if (d < 0.f || (d == 0.f && !(ch >> at & 1u))) {
        const uint32_t m = 255u << at, v = (cl & ~m) | (ch & m);
        if (i == 0) c[0] = v;
        if (i == 1) c[1] = v;
        if (i == 2) c[2] = v;
        if (i == 3) c[3] = v;
      }
    } while (left);
  }
}

struct QuantParams {
  const void* x;
  int64_t ld;
  int x_rows;
  const int* src;
  int rows, cols;
  uint8_t* codes;
  float* scales;
  int64_t s_row, s_block;
  int wide;   // rows of x start on 32-byte boundaries
};

// layout_rows: one thread per 16 values of R rows, 32 (16-bit types) or 64 (fp32)
// bytes read and 16 written for each; the R
// rows' loads are issued together. Lane i of a block's eight writes the scale of
// row i, so that scales stored block by block go out 4 R bytes at a time.
template <bool POW2, typename T, int R>
__global__ void __launch_bounds__(256) quantize_kernel(const QuantParams p) {
  const int64_t row0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * R;
  const int u = blockIdx.y * blockDim.x + threadIdx.x;
  const int units = p.cols / kUnit;
  const bool in = u < units;
  Raw<T> raw[R];
  const T* x[R];
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int64_t row = row0 + i;
    int64_t sr = -1;
    if (row < p.rows) sr = p.src ? (int64_t)__ldg(p.src + row) : row;
    x[i] = static_cast<const T*>(p.x) + sr * p.ld + (int64_t)u * kUnit;
#pragma unroll
    for (int j = 0; j < 4 * (int)sizeof(T); j++) raw[i].u[j] = 0;
    if (in && sr >= 0 && sr < p.x_rows) load_raw(x[i], p.wide, raw[i]);
  }
  float mine = 0.f;
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int64_t row = row0 + i;
    uint32_t top = top_of(raw[i]);
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float s = scale_of<POW2>(top);
    if ((u & (kLanes - 1)) == i) mine = s;
    uint32_t c[4];
    codes_of<POW2>(raw[i], x[i], s, c);
    if (in && row < p.rows)
      *reinterpret_cast<uint4*>(p.codes + row * p.cols + (int64_t)u * kUnit) =
          make_uint4(c[0], c[1], c[2], c[3]);
  }
  // (the last block of a row may have fewer lanes than R rows)
  const int i = u & (kLanes - 1), b = u / kLanes;
  if (i < R && b * kBlock < p.cols && row0 + i < p.rows)
    p.scales[(row0 + i) * p.s_row + b * p.s_block] = mine;
}

template <bool POW2, typename T>
void launch_quantize(const QuantParams& p, cudaStream_t st) {
  constexpr int R = sizeof(T) == 4 ? 2 : 4;
  const bool many = many_rows(p.rows, p.cols, R);
  const Layout l = layout_rows(p.rows, p.cols, many ? R : 1);
  wb::launch_k(many ? quantize_kernel<POW2, T, R> : quantize_kernel<POW2, T, 1>, l.grid, l.block, 0,
               st, p);
}

template <bool POW2>
void launch_quantize(const QuantParams& p, int type, cudaStream_t st) {
  if (type == WISP_DT_F32)
    launch_quantize<POW2, float>(p, st);
  else if (type == WISP_DT_BF16)
    launch_quantize<POW2, __nv_bfloat16>(p, st);
  else
    launch_quantize<POW2, __half>(p, st);
}

struct BlockParams {
  const void* x;
  int n, k, kb, nb;
  uint8_t* codes;
  float* scales;
  int wide;
};

// One CTA per block of 128 x 128 (grid kb x nb x entries): a thread holds 16
// values of four rows.
template <typename T>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const BlockParams p) {
  __shared__ uint32_t tops[8];
  const int tid = threadIdx.x, c0 = blockIdx.x * kBlock + (tid & 7) * kUnit;
  const int64_t first = (int64_t)blockIdx.z * p.n;
  const T* x = static_cast<const T*>(p.x) + first * p.k + c0;
  Raw<T> raw[4];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = blockIdx.y * kBlock + (tid >> 3) + 32 * i;
#pragma unroll
    for (int j = 0; j < 4 * (int)sizeof(T); j++) raw[i].u[j] = 0;
    if (r < p.n && c0 < p.k) load_raw(x + (int64_t)r * p.k, p.wide, raw[i]);
    top = max(top, top_of(raw[i]));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) tops[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; i++) top = max(top, tops[i]);
  const float s = scale_of<false>(top);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = blockIdx.y * kBlock + (tid >> 3) + 32 * i;
    if (r < p.n && c0 < p.k) {
      uint32_t c[4];
      codes_of<false>(raw[i], x + (int64_t)r * p.k, s, c);
      *reinterpret_cast<uint4*>(p.codes + (first + r) * p.k + c0) =
          make_uint4(c[0], c[1], c[2], c[3]);
    }
  }
  if (tid == 0) p.scales[((int64_t)blockIdx.z * p.nb + blockIdx.y) * p.kb + blockIdx.x] = s;
}

struct DequantParams {
  const uint8_t* codes;
  const float* scales;
  int64_t s_row, s_block;
  int rows, cols;
  void* out;
  int64_t ld;
  int wide;
};

WB_DEV float2 e4m3_values(uint32_t two) {
  uint32_t h;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(h) : "r"(two));
  return __half22float2(u2h2(h));
}

// layout_rows: 16 values of R rows per thread. code * scale is rounded to fp32, then to
// the output's type.
template <int TYPE, int R>
__global__ void __launch_bounds__(256) dequantize_kernel(const DequantParams p) {
  const int64_t row0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * R;
  const int u = blockIdx.y * blockDim.x + threadIdx.x;
  const bool in = u < p.cols / kUnit;
  const int lane = u & (kLanes - 1), b = u / kLanes;
  // lane i of a block's eight reads the scale of row i
  float mine = 0.f;
  if (lane < R && b * kBlock < p.cols && row0 + lane < p.rows)
    mine = __ldg(p.scales + (row0 + lane) * p.s_row + b * p.s_block);
  uint4 c[R];
#pragma unroll
  for (int i = 0; i < R; i++) {
    c[i] = make_uint4(0u, 0u, 0u, 0u);
    if (in && row0 + i < p.rows)
      c[i] = __ldg(reinterpret_cast<const uint4*>(p.codes + (row0 + i) * p.cols) + u);
  }
  float scale[R];
#pragma unroll
  for (int i = 0; i < R; i++) scale[i] = __shfl_sync(0xffffffffu, mine, i, kLanes);
#pragma unroll
  for (int i = 0; i < R; i++) {
    if (!in || row0 + i >= p.rows) continue;
    const float s = scale[i];
    const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
    float v[16];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float2 f = e4m3_values(w[j >> 1] >> (16 * (j & 1)) & 0xffffu);
      v[2 * j] = f.x * s;
      v[2 * j + 1] = f.y * s;
    }
    const int64_t at = (row0 + i) * p.ld + (int64_t)u * kUnit;
    if constexpr (TYPE == WISP_DT_F32) {
      float* q = static_cast<float*>(p.out) + at;
      if (p.wide) {
        uint32_t o[16];
#pragma unroll
        for (int j = 0; j < 16; j++) o[j] = __float_as_uint(v[j]);
        store32(q, o);
        store32(q + 8, o + 8);
      } else {
#pragma unroll
        for (int j = 0; j < 16; j++) q[j] = v[j];
      }
    } else {
      uint16_t* q = static_cast<uint16_t*>(p.out) + at;
      uint32_t o[8];
#pragma unroll
      for (int j = 0; j < 8; j++) o[j] = pack2(v[2 * j], v[2 * j + 1], TYPE);
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

template <int TYPE>
void launch_dequantize(const DequantParams& p, cudaStream_t st) {
  constexpr int R = 2;
  const bool many = many_rows(p.rows, p.cols, R);
  const Layout l = layout_rows(p.rows, p.cols, many ? R : 1);
  wb::launch_k(many ? dequantize_kernel<TYPE, R> : dequantize_kernel<TYPE, 1>, l.grid, l.block, 0,
               st, p);
}

struct GatherParams {
  const uint8_t* codes;
  const float* scales;
  int64_t s_row, s_block;
  int x_rows;
  const int* src;
  int rows, cols;
  uint8_t* out;
  float* out_scales;
  int64_t o_row, o_block;
  int past_l2;       // the result is larger than the L2 cache
};

// layout_rows: 16 codes of R rows per thread.
// Lane i of a block's eight moves the scale of row i, so that scales stored block by
// block go out 4 R bytes at a time. 32,768 of 4096 rows of 7168 take 49 us, of which
// the 242 MB that are written are 37 at the copy rate (without the hint that what the L2
// cannot hold need not stay there: 55).
template <int R>
__global__ void __launch_bounds__(256) gather_kernel(const GatherParams p) {
  const int64_t row0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * R;
  const int u = blockIdx.y * blockDim.x + threadIdx.x;
  const bool in = u < p.cols / kUnit;
  uint4 c[R];
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int64_t sr = row0 + i < p.rows ? (int64_t)__ldg(p.src + row0 + i) : -1;
    c[i] = make_uint4(0u, 0u, 0u, 0u);
    if (in && sr >= 0 && sr < p.x_rows)
      c[i] = __ldg(reinterpret_cast<const uint4*>(p.codes + sr * p.cols) + u);
  }
  const int lane = u & (kLanes - 1), b = u / kLanes;
  if (lane < R && b * kBlock < p.cols && row0 + lane < p.rows) {
    const int64_t sr = __ldg(p.src + row0 + lane);
    p.out_scales[(row0 + lane) * p.o_row + b * p.o_block] =
        sr >= 0 && sr < p.x_rows ? __ldg(p.scales + sr * p.s_row + b * p.s_block) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < R; i++)
    if (in && row0 + i < p.rows) {
      uint4* o = reinterpret_cast<uint4*>(p.out + (row0 + i) * p.cols) + u;
      if (p.past_l2)
        __stcs(o, c[i]);
      else
        *o = c[i];
    }
}

void launch_gather(const GatherParams& p, cudaStream_t st) {
  constexpr int R = 8;
  const bool many = many_rows(p.rows, p.cols, R);
  const Layout l = layout_rows(p.rows, p.cols, many ? R : 1);
  wb::launch_k(many ? gather_kernel<R> : gather_kernel<1>, l.grid, l.block, 0, st, p);
}

}  // namespace

extern "C" WispError wisp_b200_fp8_quantize(const void* d_x, int x_type, int64_t ld, int x_rows,
                                            const int* d_src, int rows, int cols, int pow2,
                                            uint8_t* d_codes, float* d_scales, int64_t scale_row,
                                            int64_t scale_block, cudaStream_t stream,
                                            WispErrCtx* err) {
  if (!dt_valid(x_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_quantize: unknown x_type %d", x_type);
  if (rows < 0 || rows > wb::kMaxRows || x_rows < 0 || cols <= 0 || cols > kMaxCols ||
      cols % kUnit || ld < cols)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp8_quantize: rows=%d x_rows=%d cols=%d ld=%lld (at most 2^31 - 256 rows, cols a "
                   "multiple of 16 up to 2^27, ld >= cols)",
                   rows, x_rows, cols, (long long)ld);
  if (!d_src && rows > x_rows)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_quantize: rows=%d > x_rows=%d without d_src", rows,
                   x_rows);
  if (scale_row < 1 || scale_block < 1)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_quantize: scale strides %lld, %lld (at least 1)",
                   (long long)scale_row, (long long)scale_block);
  if (rows == 0) return WISP_OK;
  if ((!d_x && x_rows > 0) || !d_codes || !d_scales)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_quantize: null pointer argument (x, codes, scales)");
  if (((uintptr_t)d_codes & 15) || ((uintptr_t)d_scales & 3))
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp8_quantize: codes must be 16-byte, scales 4-byte aligned");
  if ((uintptr_t)d_x % dt_size(x_type) || ((uintptr_t)d_src & 3))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_quantize: x or d_src not aligned to its type");
  QuantParams p;
  p.x = d_x;
  p.ld = ld;
  p.x_rows = x_rows;
  p.src = d_src;
  p.rows = rows;
  p.cols = cols;
  p.codes = d_codes;
  p.scales = d_scales;
  p.s_row = scale_row;
  p.s_block = scale_block;
  p.wide = !((uintptr_t)d_x & 31) && (ld * dt_size(x_type)) % 32 == 0;
  if (pow2)
    launch_quantize<true>(p, x_type, stream);
  else
    launch_quantize<false>(p, x_type, stream);
  WB_CUDA_CHECK(cudaGetLastError());
  return WISP_OK;
}

extern "C" WispError wisp_b200_fp8_dequantize(const uint8_t* d_codes, const float* d_scales,
                                              int64_t scale_row, int64_t scale_block, int rows,
                                              int cols, void* d_out, int out_type, int64_t ld,
                                              cudaStream_t stream, WispErrCtx* err) {
  if (!dt_valid(out_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_dequantize: unknown out_type %d", out_type);
  if (rows < 0 || rows > wb::kMaxRows || cols <= 0 || cols > kMaxCols ||
      cols % kUnit || ld < cols)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp8_dequantize: rows=%d cols=%d ld=%lld (at most 2^31 - 256 rows, cols a "
                   "multiple of 16 up to 2^27, ld >= cols)",
                   rows, cols, (long long)ld);
  if (rows == 0) return WISP_OK;
  if (!d_codes || !d_scales || !d_out)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_dequantize: null pointer argument");
  if (((uintptr_t)d_codes & 15) || ((uintptr_t)d_scales & 3))
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp8_dequantize: codes must be 16-byte, scales 4-byte aligned");
  if ((uintptr_t)d_out % dt_size(out_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_dequantize: out not aligned to its type");
  DequantParams p;
  p.codes = d_codes;
  p.scales = d_scales;
  p.s_row = scale_row;
  p.s_block = scale_block;
  p.rows = rows;
  p.cols = cols;
  p.out = d_out;
  p.ld = ld;
  p.wide = !((uintptr_t)d_out & 31) && ld * dt_size(out_type) % 32 == 0;
  if (out_type == WISP_DT_F32)
    launch_dequantize<WISP_DT_F32>(p, stream);
  else if (out_type == WISP_DT_BF16)
    launch_dequantize<WISP_DT_BF16>(p, stream);
  else
    launch_dequantize<WISP_DT_F16>(p, stream);
  WB_CUDA_CHECK(cudaGetLastError());
  return WISP_OK;
}

extern "C" WispError wisp_b200_fp8_gather(const WispFp8Rows* x, const int* d_src, int rows, int cols,
                                          uint8_t* d_codes, float* d_scales, int64_t scale_row,
                                          int64_t scale_block, cudaStream_t stream,
                                          WispErrCtx* err) {
  if (!x || x->rows < 0 || rows < 0 || rows > wb::kMaxRows || cols <= 0 || cols > kMaxCols ||
      cols % kUnit)
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp8_gather: x=%p rows=%d cols=%d (at most 2^31 - 256 rows, cols a multiple of 16 "
                   "up to 2^27)",
                   (const void*)x, rows, cols);
  if (scale_row < 1 || scale_block < 1)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_gather: scale strides %lld, %lld (at least 1)",
                   (long long)scale_row, (long long)scale_block);
  if (rows == 0) return WISP_OK;
  if (((!x->codes || !x->scales) && x->rows > 0) || !d_src || !d_codes || !d_scales)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_gather: null pointer argument");
  if (((uintptr_t)x->codes & 15) || ((uintptr_t)x->scales & 3) || ((uintptr_t)d_src & 3) ||
      ((uintptr_t)d_codes & 15) || ((uintptr_t)d_scales & 3))
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp8_gather: codes must be 16-byte, scales and d_src 4-byte aligned");
  launch_gather({x->codes, x->scales, x->scale_row, x->scale_block, x->rows, d_src, rows, cols,
                 d_codes, d_scales, scale_row, scale_block, (int64_t)rows * cols > 1 << 27},
                stream);
  WB_CUDA_CHECK(cudaGetLastError());
  return WISP_OK;
}

WispError wb::fp8_validate(const WispFp8Config* c, const char* who, WispErrCtx* err) {
  if (!c) return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: null config", who);
  if (c->n_entries <= 0 || c->n <= 0 || c->k <= 0 || c->k > kMaxCols || c->k % kUnit)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: n_entries=%d n=%d k=%d (k a multiple of 16 up to 2^27)",
                   who, c->n_entries, c->n, c->k);
  // the tensor map's row index (entries x n, plus one tile) is 32-bit
  if ((int64_t)c->n_entries * c->n > wb::kMaxRows)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: n_entries * n = %lld exceeds 2^31 - 256", who,
                   (long long)c->n_entries * c->n);
  if (!dt_valid(c->out_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: unknown out_type %d", who, c->out_type);
  return WISP_OK;
}

WispError wb::fp8_check_mats(const WispFp8Mats* m, const char* who, const char* what,
                             WispErrCtx* err) {
  if (!m || !m->codes || !m->scales)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: null pointer argument (%s)", who, what);
  if (((uintptr_t)m->codes & 15) || ((uintptr_t)m->scales & 3))
    return WB_FAIL(WISP_ERR_INVALID_ARG, "%s: %s codes must be 16-byte, scales 4-byte aligned", who,
                   what);
  return WISP_OK;
}

extern "C" WispError wisp_b200_fp8_quantize_weights(const void* d_w, int w_type, int n_entries,
                                                    int n, int k, uint8_t* d_codes,
                                                    float* d_scales, cudaStream_t stream,
                                                    WispErrCtx* err) {
  const WispFp8Config c = {n_entries, n, k, 0, w_type};
  WispError e = wb::fp8_validate(&c, "fp8_quantize_weights", err);
  if (e != WISP_OK) return e;
  BlockParams p;
  p.kb = (k + kBlock - 1) / kBlock;
  p.nb = (int)(((int64_t)n + kBlock - 1) / kBlock);
  if (n_entries > 65535 || p.nb > 65535)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_quantize_weights: n_entries=%d n=%d (65535 matrices "
                   "or blocks of rows at most)", n_entries, n);
  if (!d_w || !d_codes || !d_scales)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_quantize_weights: null pointer argument");
  if (((uintptr_t)d_codes & 15) || ((uintptr_t)d_scales & 3) ||
      (uintptr_t)d_w % dt_size(w_type))
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp8_quantize_weights: codes must be 16-byte, scales and weights aligned to "
                   "their types");
  p.x = d_w;
  p.n = n;
  p.k = k;
  p.codes = d_codes;
  p.scales = d_scales;
  // (16 values are 32 bytes or more, so every row start is as aligned as the first)
  p.wide = !((uintptr_t)d_w & 31);
  const dim3 grid(p.kb, p.nb, n_entries);
  if (w_type == WISP_DT_F32)
    wb::launch_k(quantize_blocks_kernel<float>, grid, 256, 0, stream, p);
  else if (w_type == WISP_DT_BF16)
    wb::launch_k(quantize_blocks_kernel<__nv_bfloat16>, grid, 256, 0, stream, p);
  else
    wb::launch_k(quantize_blocks_kernel<__half>, grid, 256, 0, stream, p);
  WB_CUDA_CHECK(cudaGetLastError());
  return WISP_OK;
}
