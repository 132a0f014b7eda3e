// numeric.cuh -- loads and stores of runs of values in any of the ABI's types
// (WISP_DT_*), for the operators that take several. The type is a launch-wide
// run-time value: every thread takes the same branch, and the operators are
// bound by memory, so the branch costs less than a kernel per combination.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "wisp_b200.h"

namespace wb {

__host__ __device__ inline int dt_size(int t) { return t == WISP_DT_F32 ? 4 : 2; }
// Rows of one call at most: counts rounded up to a tile or a block stay below
// 2^31.
constexpr int kMaxRows = 0x7fffff00;
inline bool dt_valid(int t) { return t == WISP_DT_F32 || t == WISP_DT_BF16 || t == WISP_DT_F16; }

// 1 / x to 1 ulp, for normal x and 1 / x.
WB_DEV float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

WB_DEV float load_one(const void* p, int type, int64_t i) {
  if (type == WISP_DT_F32) return static_cast<const float*>(p)[i];
  if (type == WISP_DT_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

WB_DEV void store_one(void* p, int type, int64_t i, float v) {
  if (type == WISP_DT_F32)
    static_cast<float*>(p)[i] = v;
  else if (type == WISP_DT_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Two 16-bit values of a 32-bit word.
WB_DEV float2 unpack2(uint32_t u, int type) {
  if (type == WISP_DT_BF16) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  return __half22float2(u2h2(u));
}
WB_DEV uint32_t pack2(float a, float b, int type) {
  if (type == WISP_DT_BF16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  return h22u(__floats2half2_rn(a, b));
}

// 32 bytes per thread in one instruction (32-byte aligned): a warp's access is
// then 1 KB of whole sectors, where two 16-byte accesses each touch half of
// every sector.
WB_DEV void load32(const void* p, uint32_t* u) {
  asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]),
                 "=r"(u[6]), "=r"(u[7])
               : "l"(p));
}
WB_DEV void store32(void* p, const uint32_t* u) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(u[0]), "r"(u[1]),
               "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}

// Eight consecutive values from element i. `wide`: p + i is 16-byte aligned
// (32-byte runs for fp32 are two 16-byte loads) and all eight exist; else the
// first n are read one by one and the rest are 0.
WB_DEV void load8(const void* p, int type, int64_t i, bool wide, int n, float (&v)[8]) {
  if (wide) {
    if (type == WISP_DT_F32) {
      const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      const float4 a = q[0], b = q[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
      const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float2 f = unpack2(u[j], type);
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = j < n ? load_one(p, type, i + j) : 0.f;
  }
}

WB_DEV void store8(void* p, int type, int64_t i, bool wide, int n, const float (&v)[8]) {
  if (wide) {
    if (type == WISP_DT_F32) {
      float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
      q[0] = make_float4(v[0], v[1], v[2], v[3]);
      q[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 a;
      a.x = pack2(v[0], v[1], type);
      a.y = pack2(v[2], v[3], type);
      a.z = pack2(v[4], v[5], type);
      a.w = pack2(v[6], v[7], type);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = a;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (j < n) store_one(p, type, i + j, v[j]);
  }
}

}  // namespace wb
