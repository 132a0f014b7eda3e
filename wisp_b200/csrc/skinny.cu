// skinny.cu -- grouped int4 expert FFN for small token groups (decode).
//
// When an expert sees a few tokens (batch decode: ~5 per expert in the
// 256-token / 384-expert configuration), the work per weight is one int4
// conversion plus a handful of multiply-adds, and the kernel's only job is
// to stream the packed weights at HBM speed. A tcgen05.mma (M=128, K=16)
// costs a fixed ~60-95 SM cycles whatever N <= 128 is (measured on B200), so
// at small N the 5th-generation path tops out far below HBM speed; this
// kernel feeds register-operand integer MMAs instead.
//
// Arithmetic. Each packed weight byte holds two nibbles n; the MMA's A
// operand is the signed byte 16 (n - 8), which one LOP3 produces for the
// high nibbles of a 32-bit word ((q ^ 0x88888888) & 0xF0F0F0F0: n ^ 8 is
// the two's-complement nibble of n - 8) and a shift plus one LOP3 for the
// low ones -- three instructions per eight weights, against nine for an
// exact int4 -> fp16 conversion, which made the fp16 form of this kernel
// instruction-issue bound. The activations are 16-bit integers with one
// scale per (row, 128-K block) (see skinny.h), split into a signed high
// byte and an unsigned low byte; m16n8k32 s8 x s8 and s8 x u8 MMAs (the
// same issue rate as m16n8k16 fp16 on B200, twice the K) give exact int32
// sums per scale group, and the fold adds
//     w_scale * a_scale / 16 * float(256 * D_hi + D_lo)
// (+ zero point * activation sum) into fp32 accumulators. A token's result
// is therefore bit-identical whatever chunk of the segment it lands in,
// and the 16-bit activations carry more precision than fp16.
//
// One persistent CTA per SM, warp-specialised:
//   producer    (the last warp) per 256-K stage four copies into a 4-deep
//               shared-memory ring of 46 KB stages: one TMA box of packed
//               nibbles per 128-row weight block (128 rows x 128 bytes,
//               128-byte swizzle), one 3D TMA box of the unit's q16 token rows
//               (five 128-byte lines per row: the stage's values and the rows'
//               block scales), and one bulk copy of the stage's run of weight
//               scales (zero points: one more) from the prepared per-unit
//               copy. Each extra small copy per stage measurably cut the
//               streaming rate (a probe of this ring: 7.2 TB/s with the two
//               weight boxes alone, 3.5 TB/s with six more small copies), so
//               everything else a stage needs rides in these four. Up to
//               128 KB of weights are in flight per SM. Units are looked up
//               in a shared-memory copy of the unit prefix; the next unit's
//               segment record is fetched one unit ahead.
//   consumers   8 warps with two 16-row MMA tiles each (by default; see
//               WB_SK_TILES_PER_WARP -- sixteen one-tile warps measured
//               slower: their 96-register cap spilled and every warp
//               re-reads the token fragments). All shared-memory reads are
//               a per-thread offset plus a compile-time constant from the
//               stage base. Per 128-K group a thread reads 2 x 8 bytes of each
//               of its weight rows (packed words 2t, 2t+1 and 8+2t, 9+2t of
//               the group; MMA row g lives in box row sigma(g) = 2(g%4) + g/4
//               (mod 8), so each half-warp's rows fall in distinct swizzle
//               chunks) and one 16-byte chunk of each token row per MMA step
//               (conflict-free: step s of thread t reads packed word 8(s/2) +
//               2t + s%2, whose chunk parity alternates between neighbouring
//               token rows), runs four k32 steps of high/low MMAs and folds
//               them. Units of at most 8 tokens read a whole stage into
//               registers and release it before any arithmetic, and issue the
//               two groups' MMA chains side by side.
//
// Work unit = (segment, weight row block, chunk of up to 16 tokens, and for
// a weighted down projection with fewer than two units per SM a part of a K
// split, whose partial sums the epilogue adds atomically):
//   GATEUP: 128 intermediate rows i of gate and of up; warp w takes rows
//           8w..8w+7 of both (gate as MMA rows 0-7, up as rows 8-15) ->
//           h = silu(g) * u, quantised per token over the unit's 128 rows
//           (one q16 block of H: the warps exchange their column maxima and
//           sums through shared memory) and written as q16 rows of H with
//           their block metadata.
//   DOWN:   256 output rows m (two 128-row blocks); warp w takes 16 rows ->
//           out[token] += w * y (mode 0, fp32 atomics) or y rows (mode 1).
// Chunks of one row block are consecutive units, so CTAs that run them at
// the same time share the weight tile through L2. Segments larger than the
// routing threshold go to the tcgen05 kernel (grouped.cu), which keeps
// fp16 activation rows; the two kernels work on disjoint rows.
//
// Fragment mapping (m16n8k32, 8-bit operands). Thread (g = lane/4, t =
// lane%4) holds A bytes (row g, k 4t..4t+3) and (row g, k 16+4t..16+4t+3)
// and the same for row g+8; B bytes (k 4t..4t+3, col g) and (k 16+4t..,
// col g); D (row g, cols 2t, 2t+1) and (row g+8, same). The logical k of
// one MMA may map to any physical K as long as A and B agree: in step s,
// thread t's k 4t+i is physical K 2i and k 16+4t+i is K 2i+1 of packed word
// 8(s/2) + 2t + s%2 of the 128-K group, so A is (even nibbles, odd nibbles)
// of that word and B is the (evens, odds) byte quads of its q16 chunk.
#include "common.cuh"
#include "internal.h"
#include "skinny.h"

using namespace wb;

namespace {

// Consumer warps x 16-row MMA tiles per warp = 16 tiles per 256-K stage.
#ifndef WB_SK_TILES_PER_WARP
#define WB_SK_TILES_PER_WARP 2
#endif
constexpr int kTPW = WB_SK_TILES_PER_WARP;
constexpr int kCW = 16 / kTPW;
static_assert(kTPW == 1 || kTPW == 2, "one or two tiles per consumer warp");
constexpr int kThreads = (kCW + 1) * 32;      // + one producer warp
constexpr int kStages = 4;
constexpr int kCols = 16;                     // tokens per unit
// Default routing threshold: segments of up to 32 rows run here (two 16-row
// chunks, the second reading the weight tile through L2), larger ones on the
// tcgen05 kernel. Measured on B200 with the layer's CUDA graph and L2 flushed
// between steps: Mixtral b64 (segments of 12-21 rows) 449 us at 16 -> 342 us
// at 24-128; DeepSeek prefill (4096 skewed tokens) best at 32 (7.60 ms
// against 7.86 ms at 16 and 7.77 ms at 64).
constexpr int kSkMaxRows = 32;
constexpr int kBalanceMaxPer = 12;            // units per CTA up to which the grid is balanced
constexpr int kKS = kQ16StageK;               // K per stage (256)
constexpr int kAG = kKS / kQ16Block;          // 128-K activation groups per stage
constexpr int kBoxRows = 128;
constexpr int kBoxBytes = kBoxRows * 128;     // one weight block of a stage
constexpr int kTokBytes = kQ16Lines * kCols * kQ16LineBytes;  // one stage of 16 q16 rows
constexpr int kScRun = 4 * kBoxRows * 2;      // up to 4 scale groups x 128 rows per block
// Stage layout (bytes): [weights 2 blocks][token rows: 5 lines x rows x 128 B]
// [scales 2 blocks][zeros 2 blocks]; the stage headers live apart, so a stage
// is a whole number of KB and every TMA box keeps 1024-byte alignment.
constexpr int kOffB = 2 * kBoxBytes;
constexpr int kOffS = kOffB + kTokBytes;
constexpr int kOffZ = kOffS + 2 * kScRun;
constexpr int kStageBytes = kOffZ + 2 * kScRun;
static_assert(kStageBytes % 1024 == 0, "stages must keep 1024-byte alignment");
constexpr int kMaxSegs = 1040;                // segments per launch (experts + shared)
constexpr int kMaxEntries = 1536;             // prepared expert entries
enum { SK_GATEUP = 0, SK_DOWN = 1 };
enum { HF_HZ0 = 1, HF_HZ1 = 2, HF_V1 = 4 };

struct __align__(16) StageHdr {
  int prow0;  // first activation row of the unit
  int n;      // tokens in the unit (1..16)
  int row0;   // first weight row of the unit
  int flags;  // HF_*: zero points of block 0 / 1, block 1 inside the matrix
  int kg0;    // first 256-K stage of the unit's K range
  int nst;    // stages in the unit (the whole K, or one part of a K split)
  int pad[2];
};

struct SkSmem {
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t epi[2];        // GATEUP epilogue: column maxima, then column sums
  StageHdr hdr[kStages];
  float red_max[kCW][kCols];
  int red_sum[kCW][kCols];
  int abort;
  uint32_t zbits[kMaxEntries * 3 / 32];  // zero-point flag per matrix entry
  int32_t units[kMaxSegs + 2];           // unit prefix per segment, then the K split
};

struct SkParams {
  CUtensorMap act_map[2];  // q16 token rows, boxes {128 bytes, 8/16 rows, 5 lines}, 128-byte swizzle
  const uint8_t* prepared;
  size_t p_maps_sk, p_zbits, p_sk_scales, p_sk_zeros, sk_gu_bytes, sk_dn_bytes;
  const WispSegment* segs;
  const int32_t* units;  // [0, S]: unit prefix per segment; [S + 1]: K split
  int nseg;
  int n_entries;
  int M, I, gs;
  uint8_t* hq;      // q16 H rows
  const int* row_token;
  const float* row_weight;
  float* out;
  int mode;
  int* error_flag;
  unsigned long long* counters;  // optional wait-cycle counters (diagnostics)
  int tok_row0;                  // gate/up token rows from row 0 (see SkLaunch)
};

// Diagnostic counters (cycles summed over warps): consumers' waits for a
// full stage and their total time, the producer's waits for a free stage
// and its total time.
enum { SC_FULL_WAIT, SC_CONS_TOTAL, SC_EMPTY_WAIT, SC_PROD_TOTAL, SC_COUNT };

// ---------------------------------------------------------------------------
// Integer MMAs and operand preparation.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void imma_ss(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void imma_ss_z(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void imma_su(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void imma_su_z(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}

// (a ^ b) & c in one LOP3 (immediate LUT 0x28).
__device__ __forceinline__ uint32_t lop_xor_and(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x28;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// Signed bytes 16 (n - 8) of the even (K 0,2,4,6) and odd (K 1,3,5,7)
// nibbles of a packed word.
__device__ __forceinline__ uint32_t w_even(uint32_t q) {
  return lop_xor_and(q << 4, 0x88888888u, 0xF0F0F0F0u);
}
__device__ __forceinline__ uint32_t w_odd(uint32_t q) {
  return lop_xor_and(q, 0x88888888u, 0xF0F0F0F0u);
}

// Waits without the abort shortcut: used to let issued copies land before
// the CTA exits.
__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity, long long limit) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity))
    if (clock64() - t0 > limit) return;
}

// Shared-memory loads on 32-bit shared addresses (base + per-thread offset
// + a compile-time constant, which the assembler folds into the instruction).
__device__ __forceinline__ uint2 lds_v2(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint4 lds_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ float lds_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ float lds_h2f(uint32_t a) {
  unsigned short h;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(a));
  return __half2float(__ushort_as_half(h));
}

// Where a warp's MMA tiles sit in a stage. Tile 0's MMA row g is box row
// rg0 of weight block bg0; the other rows differ by compile-time steps:
//   GATEUP, two tiles: tile ti = block ti (gate, up), rows rg0 and rg0 + 8;
//           one tile: MMA row g = gate row rg0, row g+8 = the same up row
//           (block 1) -- either way a thread holds the gate and up sums of
//           its intermediate rows;
//   DOWN:   two tiles: rows rg0 (+8) and rg0 + 16 (+8); one tile: rg0 (+8).
// Byte steps of (tile, MMA row g / g+8) in the weight boxes and in the
// stage's run of scales (G scale groups per block and stage).
template <int MODE>
__device__ __forceinline__ constexpr uint32_t box_step(int ti, int rr) {
  return MODE == SK_GATEUP ? (kTPW == 2 ? 16384u * ti + 1024u * rr : 16384u * rr)
                           : (kTPW == 2 ? 2048u * ti + 1024u * rr : 1024u * rr);
}
template <int MODE, int G>
__device__ __forceinline__ constexpr uint32_t scale_step(int ti, int rr) {
  return MODE == SK_GATEUP ? (kTPW == 2 ? (uint32_t)G * 256u * ti + 16u * rr : (uint32_t)G * 256u * rr)
                           : (kTPW == 2 ? 32u * ti + 16u * rr : 16u * rr);
}
// Weight block of (tile, row): GATEUP two tiles -> ti, one tile -> rr; DOWN -> bg0.
template <int MODE>
__device__ __forceinline__ constexpr int block_of(int ti, int rr) {
  return MODE == SK_GATEUP ? (kTPW == 2 ? ti : rr) : 0;
}

// Per-thread stage offsets (bytes from the stage base), fixed for a warp.
struct ThreadOffs {
  uint32_t a[2][2];   // [group j][words 2t,2t+1 / 8+2t,9+2t] of tile 0's row g
  uint32_t sc;        // tile 0 row g's scale in the stage's run
  uint32_t b[2];      // [s % 2]: token row g's chunk 2t + s%2 (before the line offset)
  uint32_t m[2][2];   // [c][j]: metadata of token row 2t + c for group j (before the line offset)
  int bg0, rg0;
};

template <int MODE>
__device__ __forceinline__ ThreadOffs thread_offs(int warp, int lane, int G) {
  const int g = lane >> 2, t = lane & 3;
  const int sig = ((g & 3) << 1) | (g >> 2);  // box row (mod 8) of MMA row g
  ThreadOffs o;
  if (MODE == SK_GATEUP) {
    o.bg0 = 0;
    o.rg0 = (kTPW == 2 ? 16 : 8) * warp + sig;
  } else {
    o.bg0 = warp / (kCW / 2);
    o.rg0 = 16 * kTPW * (warp % (kCW / 2)) + sig;
  }
#pragma unroll
  for (int j = 0; j < 2; j++)
#pragma unroll
    for (int h = 0; h < 2; h++)
      o.a[j][h] = o.bg0 * kBoxBytes + o.rg0 * 128 + 8 * (t & 1) +
                  ((((4 * j + 2 * h + (t >> 1)) ^ sig) & 7) << 4);
  o.sc = (uint32_t)(o.bg0 * G * kBoxRows + o.rg0) * 2;
#pragma unroll
  for (int u = 0; u < 2; u++) o.b[u] = g * 128 + (((2 * t + u) ^ g) << 4);
#pragma unroll
  for (int c = 0; c < 2; c++)
#pragma unroll
    for (int j = 0; j < 2; j++) o.m[c][j] = (2 * t + c) * 128 + ((j ^ (2 * t + c)) << 4);
  return o;
}

// Everything one 128-K activation group of a stage contributes to a warp's
// tiles, in registers. GPS = weight scale groups per activation group (1:
// group size 128, 2: group size 64, folded per 64-K half).
template <int NT, int GPS, bool HZ>
struct GroupIn {
  uint2 a[kTPW][2][2];        // [tile][MMA row g / g+8][words 2t,2t+1 / 8+2t,9+2t]
  uint4 b[4][NT];             // [step][n8 tile]: hi evens, hi odds, lo evens, lo odds
  float ws[kTPW][2][GPS];     // weight scale [tile][row][scale group]
  float as[NT][2];            // activation scale / 16 of columns 2t, 2t+1
  float wz[kTPW][2][HZ ? GPS : 1];       // zero points
  float asum[NT][2][HZ ? GPS : 1];       // activation sums over each scale group
};

// Loads activation group j of the stage at shared address st. The stage's
// token rows are [5 lines][8 NT rows][128 bytes] (lines 2j, 2j+1: group j's
// values; line 4: the rows' block metadata).
template <int MODE, int NT, int GPS, bool HZ>
__device__ __forceinline__ void load_group(GroupIn<NT, GPS, HZ>& in, uint32_t st, int j,
                                           const ThreadOffs& o, bool hz0, bool hz1) {
  constexpr int G = 2 * GPS;  // weight scale groups per 256-K stage
  constexpr int BR = 8 * NT;  // token rows in the box
#pragma unroll
  for (int ti = 0; ti < kTPW; ti++)
#pragma unroll
    for (int rr = 0; rr < 2; rr++) {
      const uint32_t bs = box_step<MODE>(ti, rr);
      in.a[ti][rr][0] = lds_v2(st + o.a[j][0] + bs);
      in.a[ti][rr][1] = lds_v2(st + o.a[j][1] + bs);
      const uint32_t ss = scale_step<MODE, G>(ti, rr);
#pragma unroll
      for (int h = 0; h < GPS; h++) {
        in.ws[ti][rr][h] = lds_h2f(st + kOffS + o.sc + ss + (j * GPS + h) * 256);
        if (HZ) {
          const bool hz = (MODE == SK_GATEUP ? block_of<MODE>(ti, rr) : o.bg0) ? hz1 : hz0;
          in.wz[ti][rr][HZ ? h : 0] = hz ? lds_h2f(st + kOffZ + o.sc + ss + (j * GPS + h) * 256) : 0.f;
        }
      }
    }
#pragma unroll
  for (int s = 0; s < 4; s++)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
      in.b[s][nt] = lds_v4(st + o.b[s & 1] + kOffB + ((2 * j + (s >> 1)) * BR + 8 * nt) * 128);
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const uint32_t m = st + o.m[c][j] + kOffB + ((kQ16Lines - 1) * BR + 8 * nt) * 128;
      in.as[nt][c] = lds_f32(m);
      if (HZ) {
        if (GPS == 1) in.asum[nt][c][0] = lds_f32(m + 4) + lds_f32(m + 8);
        else
#pragma unroll
          for (int h = 0; h < GPS; h++) in.asum[nt][c][HZ ? h : 0] = lds_f32(m + 4 + 4 * h);
      }
    }
}

// acc += the group's contribution (K order: scale group by scale group).
template <int NT, int GPS, bool HZ>
__device__ __forceinline__ void compute_group(float (&acc)[kTPW][NT][4],
                                              const GroupIn<NT, GPS, HZ>& in) {
  constexpr int SPG = 4 / GPS;  // MMA steps per scale group
#pragma unroll
  for (int h = 0; h < GPS; h++) {
    int dh[kTPW][NT][4], dl[kTPW][NT][4];
#pragma unroll
    for (int ss = 0; ss < SPG; ss++) {
      const int s = h * SPG + ss;
#pragma unroll
      for (int ti = 0; ti < kTPW; ti++) {
        const uint2 wg = in.a[ti][0][s >> 1], w8 = in.a[ti][1][s >> 1];
        const uint32_t qg = (s & 1) ? wg.y : wg.x, q8 = (s & 1) ? w8.y : w8.x;
        const uint32_t a0 = w_even(qg), a2 = w_odd(qg), a1 = w_even(q8), a3 = w_odd(q8);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const uint4 b = in.b[s][nt];
          if (ss == 0) {
            imma_ss_z(dh[ti][nt], a0, a1, a2, a3, b.x, b.y);
            imma_su_z(dl[ti][nt], a0, a1, a2, a3, b.z, b.w);
          } else {
            imma_ss(dh[ti][nt], a0, a1, a2, a3, b.x, b.y);
            imma_su(dl[ti][nt], a0, a1, a2, a3, b.z, b.w);
          }
        }
      }
    }
#pragma unroll
    for (int ti = 0; ti < kTPW; ti++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int rr = e >> 1, c = e & 1;
          const float f = (float)(dh[ti][nt][e] * 256 + dl[ti][nt][e]);
          acc[ti][nt][e] = fmaf(in.ws[ti][rr][h] * in.as[nt][c], f, acc[ti][nt][e]);
          if (HZ)
            acc[ti][nt][e] = fmaf(in.wz[ti][rr][HZ ? h : 0], in.asum[nt][c][HZ ? h : 0], acc[ti][nt][e]);
        }
  }
}

// Both activation groups of a full stage, group size 128: the MMA chains
// of the two groups are issued step by step side by side (twice the
// independent work between dependent MMAs), then folded in K order (group
// 0, then group 1), which is the same arithmetic as two compute_group calls.
template <int NT, bool HZ>
__device__ __forceinline__ void compute_stage(float (&acc)[kTPW][NT][4],
                                              const GroupIn<NT, 1, HZ> (&in)[kAG]) {
  int dh[kAG][kTPW][NT][4], dl[kAG][kTPW][NT][4];
#pragma unroll
  for (int s = 0; s < 4; s++)
#pragma unroll
    for (int j = 0; j < kAG; j++)
#pragma unroll
      for (int ti = 0; ti < kTPW; ti++) {
        const uint2 wg = in[j].a[ti][0][s >> 1], w8 = in[j].a[ti][1][s >> 1];
        const uint32_t qg = (s & 1) ? wg.y : wg.x, q8 = (s & 1) ? w8.y : w8.x;
        const uint32_t a0 = w_even(qg), a2 = w_odd(qg), a1 = w_even(q8), a3 = w_odd(q8);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const uint4 b = in[j].b[s][nt];
          if (s == 0) {
            imma_ss_z(dh[j][ti][nt], a0, a1, a2, a3, b.x, b.y);
            imma_su_z(dl[j][ti][nt], a0, a1, a2, a3, b.z, b.w);
          } else {
            imma_ss(dh[j][ti][nt], a0, a1, a2, a3, b.x, b.y);
            imma_su(dl[j][ti][nt], a0, a1, a2, a3, b.z, b.w);
          }
        }
      }
#pragma unroll
  for (int j = 0; j < kAG; j++)
#pragma unroll
    for (int ti = 0; ti < kTPW; ti++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int rr = e >> 1, c = e & 1;
          const float f = (float)(dh[j][ti][nt][e] * 256 + dl[j][ti][nt][e]);
          acc[ti][nt][e] = fmaf(in[j].ws[ti][rr][0] * in[j].as[nt][c], f, acc[ti][nt][e]);
          if (HZ) acc[ti][nt][e] = fmaf(in[j].wz[ti][rr][0], in[j].asum[nt][c][0], acc[ti][nt][e]);
        }
}

// ---------------------------------------------------------------------------
// Producer warp.
// ---------------------------------------------------------------------------
// The segment of unit u: the last segment at or after `lo` whose first unit
// is <= u (units is the prefix, units[lo] <= u < units[nseg]; empty
// segments share the next one's start). A binary search: at batch 1 the
// touched experts lie scattered among hundreds of empty segments, and a
// linear scan over them cost each CTA microseconds before its first copy.
__device__ __forceinline__ int unit_segment(const int32_t* units, int lo, int nseg, int u) {
  int hi = nseg;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (units[mid] <= u) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int MODE>
__device__ void sk_producer(const SkParams& p, uint8_t* ring, SkSmem* L, int total, int stride,
                            int lane) {
  volatile int* abort = &L->abort;
  const int K = MODE == SK_GATEUP ? p.M : p.I;
  const int nk = (K + kKS - 1) / kKS;
  const uint32_t scb = 2u * (kKS / p.gs) * kBoxRows * 2;   // one stage's run of scales
  const int ksplit = L->units[p.nseg + 1];
  if (lane < 2) tma_prefetch_desc(&p.act_map[lane]);
  int slot = 0, item = 0;
  uint32_t phase = 0;
  const long long t_start = p.counters ? clock64() : 0;
  long long wait_cycles = 0;
  bool ok = true;
  // Units are resolved from the unit prefix (ascending); the segment record
  // of the next unit is requested one unit ahead so its latency hides behind
  // the current unit's stages.
  int seg = unit_segment(L->units, 0, p.nseg, blockIdx.x);
  WispSegment sg_next = p.segs[seg];
  int seg_next = seg;
  for (int u = blockIdx.x; u < total && ok; u += stride) {
    const WispSegment sg = sg_next;
    seg = seg_next;
    const int un = u + stride;
    if (un < total) {
      // a few steps forward (dense segments), else a binary search
      for (int hop = 0; hop < 4 && L->units[seg_next + 1] <= un; hop++) seg_next++;
      if (L->units[seg_next + 1] <= un) seg_next = unit_segment(L->units, seg_next + 1, p.nseg, un);
      sg_next = p.segs[seg_next];
    }
    const int chunks = (sg.rows + kCols - 1) / kCols;
    const int l = u - L->units[seg];
    // l = (row block * ksplit + K part) * chunks + chunk: the chunks of one
    // weight tile are consecutive units
    const int ch = l % chunks, rest = l / chunks;
    const int ks = rest % ksplit, rbk = rest / ksplit;
    const int kg0 = ks * nk / ksplit, kg1 = (ks + 1) * nk / ksplit;
    const int col0 = ch * kCols;
    const int n = min(kCols, sg.rows - col0);
    const int mi = n <= 8 ? 0 : 1;               // token box of 8 / 16 rows
    const uint32_t tb = (uint32_t)kQ16Lines * (8u << mi) * kQ16LineBytes;   // bytes of the token box
    const int row0 = rbk * (MODE == SK_GATEUP ? kBoxRows : 2 * kBoxRows);
    const int row1 = MODE == SK_GATEUP ? row0 : row0 + kBoxRows;
    const bool v1 = MODE == SK_GATEUP || row1 < p.M;
    const int e0 = sg.expert * 3 + (MODE == SK_GATEUP ? 0 : 2);
    const int e1 = MODE == SK_GATEUP ? e0 + 1 : e0;
    const bool hz0 = (L->zbits[e0 >> 5] >> (e0 & 31)) & 1;
    const bool hz1 = v1 && ((L->zbits[e1 >> 5] >> (e1 & 31)) & 1);
    const CUtensorMap* map0 =
        reinterpret_cast<const CUtensorMap*>(p.prepared + p.p_maps_sk + (size_t)e0 * sizeof(CUtensorMap));
    const CUtensorMap* map1 =
        reinterpret_cast<const CUtensorMap*>(p.prepared + p.p_maps_sk + (size_t)e1 * sizeof(CUtensorMap));
    // the unit's runs of weight scales (and zero points), one per stage
    const size_t run0 = (size_t)sg.expert * (p.sk_gu_bytes + p.sk_dn_bytes) +
                        (MODE == SK_GATEUP ? 0 : p.sk_gu_bytes) + (size_t)rbk * nk * scb;
    const uint8_t* sc = p.prepared + p.p_sk_scales + run0;
    const uint8_t* zr = p.prepared + p.p_sk_zeros + run0;
    StageHdr hdr;
    hdr.prow0 = sg.row_begin + col0;
    hdr.n = n;
    hdr.row0 = row0;
    hdr.flags = (hz0 ? HF_HZ0 : 0) | (hz1 ? HF_HZ1 : 0) | (v1 ? HF_V1 : 0);
    hdr.kg0 = kg0;
    hdr.nst = kg1 - kg0;
    if (lane == 0) {
      tma_prefetch_desc(map0);
      if (MODE == SK_GATEUP) tma_prefetch_desc(map1);
    }
    for (int kg = kg0; kg < kg1; kg++, item++) {
      const uint32_t bytes = (v1 ? 2 : 1) * kBoxBytes + tb + scb * ((hz0 || hz1) ? 2 : 1);
      if (lane == 0 && item >= kStages) {
        const long long tw = p.counters ? clock64() : 0;
        ok = mbar_wait(&L->empty[slot], phase ^ 1, abort);
        if (p.counters) wait_cycles += clock64() - tw;
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      uint8_t* st = ring + slot * kStageBytes;
      uint64_t* fb = &L->full[slot];
      if (lane == 0) {
        L->hdr[slot] = hdr;
        mbar_arrive_expect_tx(fb, bytes);
      }
      __syncwarp();
      if (lane < 2) {
        if (lane == 0 || v1)
          tma_load_2d(st + lane * kBoxBytes, lane ? map1 : map0, fb, kg * (kKS / 2),
                      lane ? row1 : row0);
      } else if (lane == 2) {
        tma_load_3d(st + kOffB, &p.act_map[mi], fb, 0,
                    (MODE == SK_GATEUP && p.tok_row0) ? 0 : hdr.prow0, kg * kQ16Lines);
      } else if (lane == 3) {
        bulk_load(st + kOffS, sc + (size_t)kg * scb, scb, fb);
      } else if (lane == 4) {
        if (hz0 || hz1) bulk_load(st + kOffZ, zr + (size_t)kg * scb, scb, fb);
      }
      if (++slot == kStages) { slot = 0; phase ^= 1; }
    }
  }
  // Let every issued copy land before the CTA can exit: slot i was last
  // filled by item j = the largest j < item with j % kStages == i.
  if (lane == 0)
    for (int i = 0; i < kStages && i < item; i++) {
      const int j = i + (item - 1 - i) / kStages * kStages;
      drain_wait(&L->full[i], (uint32_t)((j / kStages) & 1), 200000000LL);
    }
  if (p.counters && lane == 0) {
    atomicAdd(p.counters + SC_EMPTY_WAIT, (unsigned long long)wait_cycles);
    atomicAdd(p.counters + SC_PROD_TOTAL, (unsigned long long)(clock64() - t_start));
  }
}

// One warp's arrival on an epilogue exchange barrier, then a bounded wait
// for all kCW consumer warps.
__device__ __forceinline__ bool epi_sync(SkSmem* L, int which, uint32_t parity, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(&L->epi[which]);
  return mbar_wait(&L->epi[which], parity, &L->abort);
}

// ---------------------------------------------------------------------------
// Consumer warps: one unit with NT n8 token tiles.
// ---------------------------------------------------------------------------
template <int MODE, int NT, int GPS, bool HZ>
__device__ bool sk_unit(const SkParams& p, uint8_t* ring, SkSmem* L, const StageHdr& hdr,
                        int warp, int lane, int& slot, uint32_t& phase, uint32_t& epi_phase,
                        long long& wait_cycles) {
  volatile int* abort = &L->abort;
  const int g = lane >> 2, t = lane & 3;
  const int sig = ((g & 3) << 1) | (g >> 2);  // box row (mod 8) of MMA row g
  const int K = MODE == SK_GATEUP ? p.M : p.I;
  const ThreadOffs o = thread_offs<MODE>(warp, lane, 2 * GPS);
  const bool hz0 = hdr.flags & HF_HZ0, hz1 = hdr.flags & HF_HZ1;
  const bool active = MODE == SK_GATEUP || o.bg0 == 0 || (hdr.flags & HF_V1);

  float acc[kTPW][NT][4];
#pragma unroll
  for (int ti = 0; ti < kTPW; ti++)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[ti][nt][e] = 0.f;

  // The down epilogue's token indices and router weights, requested now so
  // that their latency hides behind the unit's stages.
  int tok[NT][2];
  float wgt[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int col = nt * 8 + 2 * t + j;
      const bool need = MODE == SK_DOWN && p.mode == 0 && active && col < hdr.n;
      tok[nt][j] = need ? __ldg(p.row_token + hdr.prow0 + col) : 0;
      wgt[nt][j] = need ? __ldg(p.row_weight + hdr.prow0 + col) : 0.f;
    }

  for (int kk = 0; kk < hdr.nst; kk++) {
    if (kk > 0) {
      const long long tw = p.counters ? clock64() : 0;
      if (!mbar_wait(&L->full[slot], phase, abort)) return false;
      if (p.counters) wait_cycles += clock64() - tw;
    }
    const uint32_t st = smem_u32(ring) + slot * kStageBytes;
    const int ng = min(kAG, (K - (hdr.kg0 + kk) * kKS) / kQ16Block);
    if (active && NT == 1 && ng == kAG) {
      // Whole stage into registers, release, then the arithmetic.
      GroupIn<NT, GPS, HZ> in[kAG];
#pragma unroll
      for (int j = 0; j < kAG; j++) load_group<MODE>(in[j], st, j, o, hz0, hz1);
      __syncwarp();
      if (lane == 0) mbar_arrive(&L->empty[slot]);
      if constexpr (GPS == 1) {
        compute_stage(acc, in);
      } else {
#pragma unroll
        for (int j = 0; j < kAG; j++) compute_group(acc, in[j]);
      }
    } else if (active) {
#pragma unroll
      for (int j = 0; j < kAG; j++) {
        if (j < ng) {
          GroupIn<NT, GPS, HZ> in;
          load_group<MODE>(in, st, j, o, hz0, hz1);
          if (j == ng - 1) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&L->empty[slot]);
          }
          compute_group(acc, in);
        }
      }
    } else {
      __syncwarp();
      if (lane == 0) mbar_arrive(&L->empty[slot]);
    }
    if (++slot == kStages) { slot = 0; phase ^= 1; }
  }
  if (!active) return true;

  // Epilogue. acc[tile][nt][0..1]: MMA row g, columns 2t, 2t+1; [2..3]: row g+8.
  if (MODE == SK_GATEUP) {
    // h = silu(gate) * up for the thread's kTPW intermediate rows
    // (i = row0 + hrow[q]) and its columns.
    constexpr int NH = kTPW;
    float hv[NH][NT][2];
    int hrow[NH];
#pragma unroll
    for (int q = 0; q < NH; q++) {
      hrow[q] = o.rg0 + 8 * q;
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++)
          hv[q][nt][c] = kTPW == 2 ? silu(acc[0][nt][2 * q + c]) * acc[kTPW - 1][nt][2 * q + c]
                                   : silu(acc[0][nt][c]) * acc[0][nt][2 + c];
    }
    // Column maxima over the unit's 128 rows: the warp's, then all warps
    // through shared memory.
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float m = 0.f;
#pragma unroll
        for (int q = 0; q < NH; q++) m = fmaxf(m, fabsf(hv[q][nt][c]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        if (g == 0) L->red_max[warp][nt * 8 + 2 * t + c] = m;
      }
    if (!epi_sync(L, 0, epi_phase, lane)) return false;
    float mx[NT][2];
    int vq[NH][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float m = 0.f;
#pragma unroll
        for (int w = 0; w < kCW; w++) m = fmaxf(m, L->red_max[w][nt * 8 + 2 * t + c]);
        mx[nt][c] = m;
        const float inv = m > 0.f ? 32767.f / m : 0.f;
        int s = 0;
#pragma unroll
        for (int q = 0; q < NH; q++) {
          vq[q][nt][c] = max(-32767, min(32767, __float2int_rn(hv[q][nt][c] * inv)));
          s += vq[q][nt][c];
        }
        // the warp's 8 * NH rows lie in one 64-K half of the block
        s += __shfl_xor_sync(0xffffffffu, s, 4);
        s += __shfl_xor_sync(0xffffffffu, s, 8);
        s += __shfl_xor_sync(0xffffffffu, s, 16);
        if (g == 0) L->red_sum[warp][nt * 8 + 2 * t + c] = s;
      }
    if (!epi_sync(L, 1, epi_phase, lane)) return false;
    epi_phase ^= 1;
    const int rbk = hdr.row0 / kQ16Block;          // the unit's q16 block of H
    const size_t rbytes = q16_row_bytes(p.I);
    size_t hb[NH];                                 // byte of each row's K index
#pragma unroll
    for (int q = 0; q < NH; q++) {
      const int i = hdr.row0 + hrow[q];
      hb[q] = q16_word_offset(i >> 3) + (sig & 1) * 4 + (sig >> 1);
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int col = nt * 8 + 2 * t + c;
        if (col >= hdr.n) continue;
        uint8_t* hr = p.hq + (size_t)(hdr.prow0 + col) * rbytes;
#pragma unroll
        for (int q = 0; q < NH; q++) {
          const int v = vq[q][nt][c];
          hr[hb[q]] = (uint8_t)((v >> 8) & 0xFF);
          hr[hb[q] + 8] = (uint8_t)(v & 0xFF);
        }
        if (warp == 0 && g == 0) {
          int s0 = 0, s1 = 0;
#pragma unroll
          for (int w = 0; w < kCW / 2; w++) {
            s0 += L->red_sum[w][col];
            s1 += L->red_sum[kCW / 2 + w][col];
          }
          const float sc = mx[nt][c] / 32767.f;
          *reinterpret_cast<float4*>(hr + q16_meta_offset(rbk)) =
              make_float4(sc * 0.0625f, sc * (float)s0, sc * (float)s1, 0.f);
        }
      }
  } else {
#pragma unroll
    for (int ti = 0; ti < kTPW; ti++) {
      const int mg = hdr.row0 + o.bg0 * kBoxRows + o.rg0 + 16 * ti;   // output row of MMA row g
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int j = e & 1, col = nt * 8 + 2 * t + j;
          if (col >= hdr.n) continue;
          const int m = mg + 8 * (e >> 1);
          if (p.mode == 0)
            red_add_f32(p.out + (size_t)tok[nt][j] * p.M + m, wgt[nt][j] * acc[ti][nt][e]);
          else
            p.out[(size_t)(hdr.prow0 + col) * p.M + m] = acc[ti][nt][e];
        }
      }
    }
  }
  return true;
}

// Units of experts with zero points or a 64-K scale group (neither occurs
// in the benchmark configurations) run out of line, so their extra
// registers do not raise the pressure on the common path.
template <int MODE, int NT, int GPS, bool HZ>
__device__ __noinline__ bool sk_unit_cold(const SkParams& p, uint8_t* ring, SkSmem* L,
                                          const StageHdr& hdr, int warp, int lane, int& slot,
                                          uint32_t& phase, uint32_t& epi_phase,
                                          long long& wait_cycles) {
  return sk_unit<MODE, NT, GPS, HZ>(p, ring, L, hdr, warp, lane, slot, phase, epi_phase, wait_cycles);
}

template <int MODE, int GPS>
__device__ __forceinline__ bool sk_unit_any(const SkParams& p, uint8_t* ring, SkSmem* L,
                                            const StageHdr& hdr, int warp, int lane, int& slot,
                                            uint32_t& phase, uint32_t& epi_phase,
                                            long long& wait_cycles) {
  const bool hz = hdr.flags & (HF_HZ0 | HF_HZ1);
  if (GPS == 1 && !hz) {
    if (hdr.n <= 8)
      return sk_unit<MODE, 1, GPS, false>(p, ring, L, hdr, warp, lane, slot, phase, epi_phase, wait_cycles);
    return sk_unit<MODE, 2, GPS, false>(p, ring, L, hdr, warp, lane, slot, phase, epi_phase, wait_cycles);
  }
  if (hdr.n <= 8)
    return hz ? sk_unit_cold<MODE, 1, GPS, true>(p, ring, L, hdr, warp, lane, slot, phase, epi_phase, wait_cycles)
              : sk_unit_cold<MODE, 1, GPS, false>(p, ring, L, hdr, warp, lane, slot, phase, epi_phase, wait_cycles);
  return hz ? sk_unit_cold<MODE, 2, GPS, true>(p, ring, L, hdr, warp, lane, slot, phase, epi_phase, wait_cycles)
            : sk_unit_cold<MODE, 2, GPS, false>(p, ring, L, hdr, warp, lane, slot, phase, epi_phase, wait_cycles);
}

template <int MODE>
__device__ void sk_consumer(const SkParams& p, uint8_t* ring, SkSmem* L, int total, int stride,
                            int warp, int lane) {
  volatile int* abort = &L->abort;
  int slot = 0;
  uint32_t phase = 0, epi_phase = 0;
  const long long t_start = p.counters ? clock64() : 0;
  long long wait_cycles = 0;
  for (int u = blockIdx.x; u < total; u += stride) {
    const long long tw = p.counters ? clock64() : 0;
    if (!mbar_wait(&L->full[slot], phase, abort)) return;
    if (p.counters) wait_cycles += clock64() - tw;
    const StageHdr hdr = L->hdr[slot];
    const bool ok = p.gs == 128
        ? sk_unit_any<MODE, 1>(p, ring, L, hdr, warp, lane, slot, phase, epi_phase, wait_cycles)
        : sk_unit_any<MODE, 2>(p, ring, L, hdr, warp, lane, slot, phase, epi_phase, wait_cycles);
    if (!ok) return;
  }
  if (p.counters && lane == 0) {
    atomicAdd(p.counters + SC_FULL_WAIT, (unsigned long long)wait_cycles);
    atomicAdd(p.counters + SC_CONS_TOTAL, (unsigned long long)(clock64() - t_start));
  }
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1) skinny_ffn_kernel(const __grid_constant__ SkParams p) {
  extern __shared__ uint8_t smem_raw[];
  const int total = __ldg(p.units + p.nseg);
  // With a few units per CTA, units go round-robin to the fewest CTAs that
  // keep the same number per CTA (the others exit), so no SM sits out the
  // last round while the others stream. Measured on B200: Mixtral b1 71.7 ->
  // 69.6 us, the 8-rank expert-parallel layer 5.7 % faster; with many units
  // per CTA (the one-GPU stack: 42) keeping every CTA was 1.7 % faster.
  const int per = (total + (int)gridDim.x - 1) / (int)gridDim.x;
  const int stride = (per > 0 && per <= kBalanceMaxPer) ? (total + per - 1) / per : (int)gridDim.x;
  if ((int)blockIdx.x >= min(stride, total)) return;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  SkSmem* L = reinterpret_cast<SkSmem*>(ring + kStages * kStageBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; i++) {
      mbar_init(&L->full[i], 1);
      mbar_init(&L->empty[i], kCW);
    }
    mbar_init(&L->epi[0], kCW);
    mbar_init(&L->epi[1], kCW);
    L->abort = 0;
    fence_barrier_init();
  }
  const uint32_t* zb = reinterpret_cast<const uint32_t*>(p.prepared + p.p_zbits);
  for (int w = threadIdx.x; w < (p.n_entries * 3 + 31) / 32; w += blockDim.x) L->zbits[w] = __ldg(zb + w);
  for (int i = threadIdx.x; i <= p.nseg + 1; i += blockDim.x) L->units[i] = __ldg(p.units + i);
  __syncthreads();
  if (warp == kCW)
    sk_producer<MODE>(p, ring, L, total, stride, lane);
  else
    sk_consumer<MODE>(p, ring, L, total, stride, warp, lane);
  __syncthreads();
  if (threadIdx.x == 0 && L->abort && p.error_flag) atomicOr(p.error_flag, kErrorTimeout);
}

constexpr size_t kSmemBytes = 1024 + (size_t)kStages * kStageBytes + sizeof(SkSmem);
static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");

}  // namespace

namespace wb {

int skinny_max_rows() { return kSkMaxRows; }
int skinny_max_segs() { return kMaxSegs; }
int skinny_max_entries() { return kMaxEntries; }
int skinny_cols() { return kCols; }
int skinny_stages(int K) { return (K + kKS - 1) / kKS; }
int skinny_units_gateup(int I) { return I / kBoxRows; }
int skinny_units_down(int M) { return (M + 2 * kBoxRows - 1) / (2 * kBoxRows); }

cudaError_t launch_skinny(const SkLaunch& L, int phase, int grid, cudaStream_t st) {
  // The attribute belongs to the current device's context: set it per launch.
  cudaError_t ce = phase == 0
      ? cudaFuncSetAttribute(skinny_ffn_kernel<SK_GATEUP>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes)
      : cudaFuncSetAttribute(skinny_ffn_kernel<SK_DOWN>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
  if (ce != cudaSuccess) return ce;
  SkParams p;
  memset(&p, 0, sizeof p);
  p.prepared = L.prepared;
  p.p_maps_sk = L.p_maps_sk;
  p.p_zbits = L.p_zbits;
  p.p_sk_scales = L.p_sk_scales;
  p.p_sk_zeros = L.p_sk_zeros;
  p.sk_gu_bytes = L.sk_gu_bytes;
  p.sk_dn_bytes = L.sk_dn_bytes;
  p.segs = L.segs;
  p.nseg = L.nseg;
  p.n_entries = L.n_entries;
  p.M = L.M;
  p.I = L.I;
  p.gs = L.gs;
  p.hq = L.hq;
  p.row_token = L.row_token;
  p.row_weight = L.row_weight;
  p.out = L.out;
  p.mode = L.mode;
  p.error_flag = L.error_flag;
  p.tok_row0 = L.tok_row0;
  p.counters = L.counters ? L.counters + phase * SC_COUNT : nullptr;
  const CUtensorMap* maps = phase == 0 ? L.xq_maps : L.hq_maps;
  for (int i = 0; i < 2; i++) p.act_map[i] = maps[i];
  if (phase == 0) {
    p.units = L.units_gu;
    wb::launch_k(skinny_ffn_kernel<SK_GATEUP>, grid, kThreads, kSmemBytes, st, p);
  } else {
    p.units = L.units_dn;
    wb::launch_k(skinny_ffn_kernel<SK_DOWN>, grid, kThreads, kSmemBytes, st, p);
  }
  return cudaGetLastError();
}

}  // namespace wb
