// tiles.cuh -- how the rows of a product with expert matrices (one expert per
// segment of rows) are cut into tiles, and how the roles of a persistent CTA
// walk them. Shared by the 4-bit and the 8-bit product.
//
// Params is the kernel's own parameter block; used here are its members segs,
// nseg, rows, V (matrices), cap (rows per tile at most) and error_flag. Cut
// gives the rows per tile of a segment, Cut::rows(rows, cap), a multiple of the
// MMA's granularity.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "numeric.cuh"
#include "wisp_b200.h"

namespace wb {

constexpr int kMaxSegs = 1025;

struct Tile {
  int expert, row0, cnt;   // rows row0 .. row0 + cnt - 1
  int ft;                  // features 128 ft ..
};

// As many tiles as at most `cap` rows each demand, of equal size up to the
// MMA's granularity UNIT (16; 32 in a pair, 16 rows per CTA).
template <int UNIT>
struct EvenCut {
  WB_DEV static int rows(int rows, int cap) {
    int per = rows;
    if (rows > cap) {
      const int t = (rows - 1) / cap + 1;      // (rows + t may pass 2^31)
      per = (rows - 1) / t + 1;
    }
    return (per + UNIT - 1) & ~(UNIT - 1);
  }
};

template <typename Params>
WB_DEV WispSegment segment(const Params& p, int s) {
  if (p.segs) return p.segs[s];
  WispSegment v;
  v.expert = 0;
  v.row_begin = 0;
  v.rows = p.rows;
  v.reserved = 0;
  return v;
}

template <typename Params>
WB_DEV bool segment_ok(const Params& p, const WispSegment& v) {
  return v.rows >= 0 && v.row_begin >= 0 && (int64_t)v.row_begin + v.rows <= p.rows &&
         (v.rows == 0 || (v.expert >= 0 && v.expert < p.V));
}

// The work: each token tile has `fitems` items (feature tiles, or pairs of
// them). Segments of one token tile and those of several are listed apart, in
// order (the second list from the end of the arrays); pref holds the tiles
// before a segment within its list. A single tile's weights come from memory
// while the tiles after the first of a larger segment find theirs in the L2
// cache, so the items of the two lists are dealt out evenly over the launch,
// each list in its order.
struct Plan {
  const int* pref;
  const uint16_t* order;
  int singles, multis, multi_tiles;     // segments of one, of several tiles; tiles of these
  int fitems;
};

// The lists of segments and the largest tile, by all THREADS threads of the CTA: a
// scan over (segments of one tile | segments of several << 16, tiles of these),
// THREADS segments at a time. (Loops are not unrolled: this runs once, from cold
// instructions.) pref, order: [kMaxSegs], warp_tot: [THREADS / 32], in shared
// memory; the caller puts a barrier before their first use. The first of the
// barriers here also orders the caller's tensor memory allocation and is followed
// by the arrival on the cluster's barrier. `first(segment, ft)`, called by one
// thread, hands out item it0 where every segment is one tile and all are seen in
// one round: first_done says whether it was.
template <typename Cut, int THREADS, typename Params, typename First>
WB_DEV Plan make_plan(const Params& p, int fitems, int it0, int* pref, uint16_t* order,
                      int4* warp_tot, int& max_cnt, bool& first_done, First&& first) {
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  Plan plan;
  plan.pref = pref;
  plan.order = order;
  plan.singles = plan.multis = plan.multi_tiles = 0;
  plan.fitems = fitems;
  max_cnt = 0;
  first_done = false;
  const int nseg = p.segs ? p.nseg : 1;
#pragma unroll 1
  for (int s0 = 0; s0 < nseg; s0 += THREADS) {
    WispSegment v;
    v.rows = 0;
    int n = 0, per = 0;
    if (s0 + tid < nseg) {
      v = segment(p, s0 + tid);
      if (!segment_ok(p, v)) {
        if (p.error_flag && blockIdx.x == 0) atomicOr(p.error_flag, kErrorSkipped);
      } else if (v.rows > 0) {
        per = Cut::rows(v.rows, p.cap);
        n = v.rows <= p.cap ? 1 : (v.rows - 1) / per + 1;
      }
    }
    const int most = __reduce_max_sync(0xffffffffu, min(per, v.rows));
    const int kind = n == 0 ? 0 : n == 1 ? 1 : 1 << 16, many = n > 1 ? n : 0;
    int x = kind, z = many;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int y0 = __shfl_up_sync(0xffffffffu, x, o), y1 = __shfl_up_sync(0xffffffffu, z, o);
      if (lane >= o) {
        x += y0;
        z += y1;
      }
    }
    if (s0 > 0) __syncthreads();          // the last round's totals have been read
    if (lane == 31) warp_tot[warp] = make_int4(x, z, most, 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (s0 == 0) cluster_arrive();
    // every warp scans the warps' totals
    const int4 w = lane < THREADS / 32 ? warp_tot[lane] : make_int4(0, 0, 0, 0);
    int wx = w.x, wz = w.y;
#pragma unroll 1
    for (int o = 1; o < 16; o <<= 1) {
      const int y0 = __shfl_up_sync(0xffffffffu, wx, o), y1 = __shfl_up_sync(0xffffffffu, wz, o);
      if (lane >= o) {
        wx += y0;
        wz += y1;
      }
    }
    max_cnt = max(max_cnt, __reduce_max_sync(0xffffffffu, w.z));
    const int bx = __shfl_sync(0xffffffffu, wx - w.x, warp) + x - kind;
    const int bz = __shfl_sync(0xffffffffu, wz - w.y, warp) + z - many;
    if (n == 1) {
      const int at = plan.singles + (bx & 0xffff);
      order[at] = (uint16_t)(s0 + tid);
    } else if (n > 1) {
      const int at = kMaxSegs - 1 - (plan.multis + (bx >> 16));
      order[at] = (uint16_t)(s0 + tid);
      pref[at] = plan.multi_tiles + bz;
    }
    // The first tile, when every segment is one tile and this thread has it.
    const int tx = __shfl_sync(0xffffffffu, wx, 15);
    first_done = nseg <= THREADS && tx > 0 && tx < (1 << 16) && it0 < tx * fitems;
    if (first_done && n == 1) {
      const int ft = it0 - (bx & 0xffff) * fitems;
      if (ft >= 0 && ft < fitems) first(v, ft);
    }
    plan.singles += tx & 0xffff;
    plan.multis += tx >> 16;
    plan.multi_tiles += __shfl_sync(0xffffffffu, wz, 15);
  }
  return plan;
}

template <typename Cut, typename Params>
__device__ __noinline__ Tile find_tile(const Params& p, const Plan& q, int it) {
  const int fitems = q.fitems, single = q.singles * fitems;
  const int items = single + q.multi_tiles * fitems;
  int i = it;
  bool one = q.multi_tiles == 0;
  if (q.multi_tiles > 0 && single > 0) {
    const int before = (int)((int64_t)it * single / items);     // singles among the items before
    const int after = (int)((int64_t)(it + 1) * single / items);
    one = after > before;
    i = one ? before : it - before;
  }
  int tt = i / fitems;
  Tile t;
  t.ft = i - tt * fitems;
  int at = tt;                  // its place in the list
  if (!one) {
    int lo = 0, hi = q.multis;       // the last segment with pref <= tt
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (q.pref[kMaxSegs - 1 - m] <= tt)
        lo = m;
      else
        hi = m;
    }
    at = kMaxSegs - 1 - lo;
    tt -= q.pref[at];
  } else {
    tt = 0;
  }
  const WispSegment v = segment(p, q.order[at]);
  const int per = Cut::rows(v.rows, p.cap);
  t.expert = v.expert;
  t.row0 = v.row_begin + tt * per;
  t.cnt = min(per, v.rows - tt * per);
  return t;
}

// A position in the ring of stages.
struct Ring {
  int s = 0;
  uint32_t ph = 0;     // parity of the slot's current use
  WB_DEV void next(int S) {
    if (++s == S) {
      s = 0;
      ph ^= 1;
    }
  }
};

// A role's walk through the tiles that the scheduler warp puts into a ring of
// SLOTS: Bars has tile_full and tile_empty barriers and the tiles (expert (-1: no
// more), first row, rows, feature tile).
template <int SLOTS>
struct TileWalk {
  int s = 0;
  uint32_t ph = 0;
  // Every lane gets the tile; false: no more, or the wait was given up.
  template <typename Bars>
  WB_DEV bool next(Bars& bars, Tile& t, volatile int* abort) {
    const bool ok = mbar_wait(&bars.tile_full[s], ph, abort);
    if (!__all_sync(0xffffffffu, ok)) return false;
    const int4 v = bars.tile[s];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&bars.tile_empty[s]);
    if (++s == SLOTS) {
      s = 0;
      ph ^= 1;
    }
    t.expert = __shfl_sync(0xffffffffu, v.x, 0);
    t.row0 = __shfl_sync(0xffffffffu, v.y, 0);
    t.cnt = __shfl_sync(0xffffffffu, v.z, 0);
    t.ft = __shfl_sync(0xffffffffu, v.w, 0);
    return t.expert >= 0;
  }
};

// Arrive on a barrier (of both CTAs of a pair) when the MMAs and copies issued
// so far have completed.
template <bool PAIR>
WB_DEV void commit(uint64_t* bar) {
  if constexpr (PAIR)
    mma_commit_pair(bar);
  else
    mma_commit(bar);
}

WB_DEV void put_out(float* q, float v) { *q = v; }
WB_DEV void put_out(__nv_bfloat16* q, float v) { *q = __float2bfloat16_rn(v); }
WB_DEV void put_out(__half* q, float v) { *q = __float2half_rn(v); }

// silu(g) * u, with h = exp(-|g| / 2): g / (1 + h^2), or g h^2 / (1 + h^2) for a
// negative g. Nothing overflows, and the divisor lies in [1, 2]. (With
// g / (1 + exp(-g)) and a quick quotient, which is 0 for divisors above 2^126,
// the result is 0 from g = -87.4 down, where silu is still 1e-36; the time is
// the same.) 16-bit outputs take the quick power of two for the exponential,
// whose error, about |g| 2^-23 relative, is far below theirs.
template <typename T>
WB_DEV float swiglu(float g, float u) {
  float h;
  if (sizeof(T) == 4)
    h = expf(-0.5f * fabsf(g));
  else     // exp(-|g| / 2) = 2^(-|g| / (2 ln 2)); 0 below 2^-126, where g h^2 is 0 too
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(fabsf(g) * -0.72134752f));
  return (g < 0.f ? g * h * h : g) * rcp_approx(fmaf(h, h, 1.f)) * u;
}

}  // namespace wb
