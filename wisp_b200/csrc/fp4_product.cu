// fp4_product.cu -- out[p, f] = sum_k x[p, k] w_e[f, k] over 4-bit
// block-scaled rows and expert matrices (one expert per segment of rows), on
// the tensor cores' block-scaled 4-bit instructions.
//
// The features are the MMA's M (128 per tile, so that a weight matrix streams
// through shared memory once per token tile), the rows its N: any multiple of
// 16 (32 in a pair) up to kMaxN, set per tile in the instruction descriptor, so
// one kernel serves single tokens and prefill. An accumulator lane is then one
// feature and a column one row: an epilogue warp stores 32 consecutive features
// of a row at a time, and SwiGLU pairs the gate and up accumulators lane by lane.
//
// Two forms. CTA pairs (cta_group::2, M = 256) take two feature tiles of one
// token tile, and each loads its own weights but only half of the row codes,
// which halves what the rows cost in L2 traffic, shared memory and power; the
// even CTA issues all MMAs, the odd CTA's MMA warp only passes on that its
// stages are full. (At 4096 tokens over 257 experts 4 to 6 % faster than single
// CTAs, at 40 tokens 3 %, dense 8192^3 12 %.) Single CTAs (cta_group::1) take matrices of one
// feature tile; and when there are few tiles, clusters of 2 or 4 of them take
// one tile each and split K: their partial sums meet in shared memory and are
// added in the order of K.
//
// Warps of a persistent CTA: 0 issues the TMA copies (weights, their prepared
// scales, row codes; 128-byte swizzle, 256 k per stage), 2, 3 (and 13 for NV)
// copy the rows' scale bytes into the layout tcgen05.cp spreads over tensor
// memory (in a pair the even CTA's do, and send the odd one a copy), 1 issues the scale copies and MMAs, 4-11 are the epilogue, 12 hands
// out the tiles. tcgen05.mma after tcgen05.cp of one thread are ordered; the
// reverse is not documented, so the scales in tensor memory have several
// buffers, and one is refilled only when the MMAs that read it have completed.
//
// Measured on one B200 (64 experts of 2 x 2048 x 7168, MX, L2 flushed): one row
// per expert 152 us = 6.6 TB/s, 128 rows 170 us = 6.3 TB/s, 224 rows 199 us =
// 4.2 PFLOP/s; a dense 8192^3 product 209 to 215 us = 5.1 to 5.3 PFLOP/s (NV 281
// us = 3.9). The weights' bytes bound it up to ~200 rows per expert. Above that
// the copies into an SM do more than the MMAs: the MMA warp waits a quarter (one
// matrix) to 45 % (gate/up) of its cycles for a full stage and 10 to 17 % for a
// scale buffer, with the ring full of copies in flight; and under steady load the
// power limit lowers the clock (1.27 to 1.45 GHz at prefill).
#include "common.cuh"
#include "internal.h"
#include "numeric.cuh"
#include "tiles.cuh"

namespace {

using namespace wb;

constexpr int kEpiWarp = 4;       // first of 8 epilogue warps
constexpr int kSchedWarp = 12;    // then the scale warps after 2 and 3
constexpr int kABytes = 128 * 128;
constexpr int kMaxStages = 8;
constexpr int kRingBytes = 218 * 1024;
constexpr int kTileRing = kMaxStages;

template <bool NV, bool SWIGLU>
struct Shape {
  static constexpr int kWords = NV ? 4 : 2;           // 4-scale words per row and stage
  static constexpr int kMats = SWIGLU ? 2 : 1;
  // The row scales' warps take turns at 16 bytes a row; from the last stage
  // of a warp's turn to the first of its next are kTurn stages at most, and
  // the ring must hold as many (see there).
  static constexpr int kUnitStages = 4 / kWords, kScaleWarps = NV ? 3 : 2;
  static constexpr int kTurn = (kScaleWarps - 1) * kUnitStages + 1;
  static constexpr int kThreads = 32 * (kSchedWarp + 1 + kScaleWarps - 2);
  // Tensor memory: accumulators in two halves of as many columns as the
  // launch's largest tile has rows (gate and up, or two tiles of one matrix),
  // then two buffers of scales or more.
  static constexpr int kMaxN = NV ? 192 : 224;
  static constexpr int kSfCols = kWords * (4 * kMats + 8);
  static_assert(2 * kMaxN + 2 * kSfCols <= 512, "tensor memory");
  static constexpr int kSfaBytes = kWords * 512;
  // A stage: weights (gate, up), their scales, the row scales (a 512-byte
  // tile per word and 128 rows), then as many 32-row boxes of row codes as
  // the launch's largest tile has.
  static constexpr int kOffSfa = kMats * kABytes;
  static constexpr int kOffSfb = kOffSfa + kMats * kSfaBytes;
  static_assert((kOffSfb + kWords * 512) % 1024 == 0, "128-byte swizzle atoms");
};

struct Bars {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t red_full, red_empty;     // partial sums of a cluster's CTAs
  uint64_t tile_full[kTileRing];
  uint64_t tile_empty[kTileRing];
  int4 tile[kTileRing];     // expert (-1: no more), first row, rows, feature tile
  uint32_t tmem;
  int abort;
};

struct alignas(64) Params {
  CUtensorMap tm_w, tm_up, tm_x;
  const uint8_t* sf_w;
  const uint8_t* sf_up;
  const float* ts_w;
  const float* ts_up;
  const float* ts_x;
  const uint8_t* xs;      // row scales, xs_ld bytes per row
  int xs_ld;
  int rows;
  const WispSegment* segs;
  int nseg;
  int V, N, nk, ftiles;
  int cap;                // rows per tile at most: a multiple of 32, <= kMaxN
  void* out;
  int64_t ld;
  int out_type;
  int* error_flag;
};

// Instruction descriptor of the block-scaled 4-bit MMAs: A and B e2m1, both
// K-major, M = 128 (256 for a pair); scale type bit 23 (0: e4m3, 1: e8m0); the
// scale bytes used within each 32-bit word at bits 29 (A) and 4 (B).
template <bool NV, bool PAIR>
WB_DEV uint32_t idesc_fp4(int n) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((NV ? 0u : 1u) << 23) |
         ((uint32_t)((PAIR ? 256 : 128) >> 4) << 24);
}

#define WB_MMA_FP4(GROUP, KIND)                                                              \
  asm volatile(                                                                              \
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                        \
      "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" \
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc) : "memory")

template <bool NV, bool PAIR>
WB_DEV void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                    uint32_t acc) {
  if constexpr (NV && PAIR)
    WB_MMA_FP4("2", "mxf4nvf4.block_scale.scale_vec::4X");
  else if constexpr (NV)
    WB_MMA_FP4("1", "mxf4nvf4.block_scale.scale_vec::4X");
  else if constexpr (PAIR)
    WB_MMA_FP4("2", "mxf4.block_scale.scale_vec::2X");
  else
    WB_MMA_FP4("1", "mxf4.block_scale.scale_vec::2X");
}
#undef WB_MMA_FP4

// 32 rows x 16 bytes of shared memory into 4 columns of every warp's lanes (in
// a pair, each CTA's shared memory into its own tensor memory).
template <bool PAIR>
WB_DEV void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
                 : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
                 : "memory");
}

// Shared-memory descriptor of a 512-byte scale tile: no swizzle, 8-row groups
// of 16-byte rows 128 bytes apart.
WB_DEV uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1u << 16) |
         ((uint64_t)(128u >> 4) << 32) | ((uint64_t)1u << 46);
}

// The accumulators: two halves of `cols` columns. A tile of one matrix, or a
// gate/up tile of at most cols / 2 rows (up cols / 2 columns after gate), takes
// one half, so its epilogue overlaps the next tile's MMAs; a larger
// gate/up tile takes both (gate, up). MMA and epilogue warps walk the tiles in
// the same order and so agree on the halves and their phases.
template <bool SWIGLU>
struct Acc {
  int cols;
  int h = 0;                       // the tile's (first) half
  bool both = false;
  int nxt = 0;
  uint32_t uses0 = 0, uses1 = 0;   // of each half, before this tile
  WB_DEV void take(int n) {      // n: the MMA's columns
    both = SWIGLU && n > cols / 2;
    h = both ? 0 : nxt;
  }
  WB_DEV uint32_t uses() const { return h ? uses1 : uses0; }
  WB_DEV uint32_t up_offset() const { return both ? cols : cols / 2; }
  WB_DEV void done() {
    if (both || h == 0) uses0++;
    if (both || h == 1) uses1++;
    if (!both) nxt ^= 1;
  }
};

// One warp's part of a tile: its lane's feature f, rows 16 half + 32 i ...
// Everything is fp32 until the one rounding to the output type.
template <bool SWIGLU, typename T>
WB_DEV void store_tile(const Params& p, const Tile& t, uint32_t d, uint32_t du, int half, int f,
                       float ag, float au) {
  const int64_t ld = p.ld;
  T* out = static_cast<T*>(p.out) + (t.row0 + half * 16) * ld + f;
  for (int c = half * 16; c < t.cnt; c += 32, out += 32 * ld) {
    uint32_t g[16], u[16];
    tmem_ld16(d + c, g);
    if (SWIGLU) tmem_ld16(du + c, u);
    tmem_wait_ld();
    const int left = t.cnt - c;
    if (f < p.N) {
      T* q = out;
      if (left >= 16) {
#pragma unroll
        for (int i = 0; i < 16; i++, q += ld) {
          float v = __uint_as_float(g[i]) * ag;
          if (SWIGLU) v = swiglu<T>(v, __uint_as_float(u[i]) * au);
          put_out(q, v);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; i++, q += ld) {
          if (i < left) {
            float v = __uint_as_float(g[i]) * ag;
            if (SWIGLU) v = swiglu<T>(v, __uint_as_float(u[i]) * au);
            put_out(q, v);
          }
        }
      }
    }
    __syncwarp();
  }
}

// The epilogue of a cluster that splits K. 16 rows at a time, every CTA puts its
// partial sums into its shared memory (four warps the gate's or the only ones,
// four the up's), and CTA kp adds those of all, in the order of K, for the rows
// kp, kp + ks, ... (a warp per row, 4 features per lane).
constexpr int kRedRows = 16;
template <bool SWIGLU>
struct Reduce {
  float* buf;        // [gate, up][kRedRows][128 features]
  Bars* bars;
  int ks, kp;
  uint32_t uses = 0;

  WB_DEV void arrive_all(uint64_t* bar) const {
    __syncwarp();
    const int j = threadIdx.x & 31;
    if (j < ks) mbar_arrive_remote_release(cluster_addr(bar, j));
  }

  // w: 0..7, the warp's place among the epilogue's
  template <typename T>
  WB_DEV bool store(const Params& p, const Tile& t, uint32_t d, uint32_t du, int w, float ag,
                    float au, volatile int* abort) {
    const int lane = threadIdx.x & 31, half = w >> 2, quad = threadIdx.x >> 5 & 3;
    for (int c = 0; c < t.cnt; c += kRedRows, uses++) {
      bool ok = uses == 0 || mbar_wait_cluster(&bars->red_empty, (uses - 1) & 1, abort);
      if (!__all_sync(0xffffffffu, ok)) return false;
      if (half == 0 || SWIGLU) {
        uint32_t g[16];
        tmem_ld16((half ? du : d) + c, g);
        tmem_wait_ld();
        float* q = buf + half * kRedRows * 128 + quad * 32 + lane;
#pragma unroll
        for (int i = 0; i < 16; i++) q[i * 128] = __uint_as_float(g[i]);
      }
      arrive_all(&bars->red_full);
      ok = mbar_wait_cluster(&bars->red_full, uses & 1, abort);
      if (!__all_sync(0xffffffffu, ok)) return false;
      for (int r = kp + ks * w; r < min(kRedRows, t.cnt - c); r += ks * 8) {
        float v[4] = {0.f, 0.f, 0.f, 0.f}, x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int j = 0; j < ks; j++) {
          const uint32_t a = cluster_addr(buf + r * 128 + lane * 4, j);
          const float4 y = ld_cluster_f4(a);
          v[0] += y.x;
          v[1] += y.y;
          v[2] += y.z;
          v[3] += y.w;
          if (SWIGLU) {
            const float4 z = ld_cluster_f4(a + kRedRows * 128 * 4);
            x[0] += z.x;
            x[1] += z.y;
            x[2] += z.z;
            x[3] += z.w;
          }
        }
        const int f = t.ft * 128 + lane * 4;
        T* out = static_cast<T*>(p.out) + (int64_t)(t.row0 + c + r) * p.ld + f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float o = v[i] * ag;
          if (SWIGLU) o = swiglu<T>(o, x[i] * au);
          if (f + i < p.N) put_out(out + i, o);
        }
      }
      arrive_all(&bars->red_empty);
    }
    return true;
  }
};

template <bool NV, bool SWIGLU, bool PAIR>
__global__ void __launch_bounds__(Shape<NV, SWIGLU>::kThreads, 1)
fp4_product_kernel(const __grid_constant__ Params p) {
  using C = Shape<NV, SWIGLU>;
  constexpr int kThreads = C::kThreads;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ Bars bars;
  __shared__ int pref[kMaxSegs];
  __shared__ uint16_t order[kMaxSegs];
  __shared__ int4 warp_tot[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  volatile int* abort = &bars.abort;
  constexpr int kUnit = PAIR ? 32 : 16;
  using Cut = EvenCut<kUnit>;
  constexpr int kBox = PAIR ? 16 : 32;            // rows per copy of row codes
  // pair: this CTA's place in it; else the K split: kp of ks
  const int rank = PAIR ? (int)cluster_rank() : 0;
  const int ks = PAIR ? 1 : (int)cluster_size(), kp = PAIR ? 0 : (int)cluster_rank();
  const int fitems = PAIR ? (p.ftiles + 1) / 2 : p.ftiles;

  if (warp == 0 && elect_sync()) {
    tma_prefetch_desc(&p.tm_w);
    tma_prefetch_desc(&p.tm_x);
    if (SWIGLU) tma_prefetch_desc(&p.tm_up);
  }
  __syncwarp();
  // The prologue is most of a single token's time, so its parts overlap: the
  // barriers are initialised by as many threads, the cluster barrier is waited
  // for only where another CTA's barriers are used, and the thread that holds
  // the first tile's segment hands that tile out itself.
  if (tid < kMaxStages) {
    // the copies, a scale warp, the odd CTA's word; in the odd CTA all comes by
    // copies
    mbar_init(&bars.full[tid], !PAIR ? 2 : rank == 0 ? 3 : 1);
    mbar_init(&bars.empty[tid], 1);
    mbar_init(&bars.tile_full[tid], 1);
    // all warps that walk the tiles
    mbar_init(&bars.tile_empty[tid], 10 + (rank == 0 ? C::kScaleWarps : 0));
    if (tid < 2) {
      mbar_init(&bars.acc_full[tid], 1);
      mbar_init(&bars.acc_empty[tid], PAIR ? 16 : 8);
    } else if (tid == 2) {
      mbar_init(&bars.red_full, 8 * ks);
      mbar_init(&bars.red_empty, 8 * ks);
      bars.abort = 0;
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    if (PAIR)
      tmem_alloc_pair(&bars.tmem, 512);
    else
      tmem_alloc(&bars.tmem, 512);
  }
  const int group = PAIR ? 2 : ks;                   // CTAs that share a tile
  const int it0 = blockIdx.x / group, it_step = gridDim.x / group;
  int max_cnt;
  bool first_done;
  const Plan plan = make_plan<Cut, kThreads>(
      p, fitems, it0, pref, order, warp_tot, max_cnt, first_done,
      [&](const WispSegment& v, int ft) {
        bars.tile[0] = make_int4(v.expert, v.row_begin, v.rows, PAIR ? 2 * ft + rank : ft);
        mbar_arrive(&bars.tile_full[0]);
      });
  // the scheduler warp reads pref and order
  __syncwarp();
  if (warp == kSchedWarp)
    asm volatile("barrier.cta.sync.aligned 1, %0;" ::"n"(kThreads) : "memory");
  else
    asm volatile("barrier.cta.arrive.aligned 1, %0;" ::"n"(kThreads) : "memory");
  const uint32_t tmem = bars.tmem;
  const int k0 = p.nk * kp / ks, k1 = p.nk * (kp + 1) / ks;     // this CTA's stages
  // Few rows leave room for more stages in flight, which is what hides the
  // memory's latency when the weights are most of the traffic.
  const int row_tiles = max_cnt > 128 ? 2 : 1;     // of 128 rows' scales
  const int sfb_bytes = C::kWords * 512 * row_tiles, off_b = C::kOffSfb + sfb_bytes;
  // a pair's CTA holds half of the tile's rows, in boxes of 16
  const int stage_bytes = off_b + ((max_cnt + 31) >> 5) * (PAIR ? 2048 : 4096);
  constexpr int kRedBytes = C::kMats * kRedRows * 128 * 4;     // a cluster's partial sums
  // S >= kTurn even for the largest stages (kMaxN rows in one CTA)
  static_assert(kRingBytes - kRedBytes >= C::kTurn * (C::kOffSfb + C::kWords * 1024 + C::kMaxN * 128),
                "ring");
  const int S = min(kMaxStages, (kRingBytes - (ks > 1 ? kRedBytes : 0)) / stage_bytes);
  // columns of an accumulator half (two sets of the largest tile's, where a
  // half can hold gate and up), buffers of scales
  const int cols = min(max((max_cnt + 31) & ~31, 32) * C::kMats, C::kMaxN);
  const int sf_bufs = min(S, (512 - 2 * cols) / C::kSfCols);
  TileWalk<kTileRing> tiles;
  Tile t;

  if (warp == 0) {
    Ring r;
    bool first = true, ok = true;
    while (ok && tiles.next(bars, t, abort)) {
      const int wrow = t.expert * p.N + t.ft * 128;
      // (an odd number of feature tiles leaves a pair's second without one)
      const int64_t sf =
          ((int64_t)t.expert * p.ftiles + min(t.ft, p.ftiles - 1)) * p.nk * C::kSfaBytes;
      const uint8_t* sfw = p.sf_w + sf;
      const uint8_t* sfu = p.sf_up + sf;
      const int nb = (t.cnt + 31) >> 5;           // (in a pair: half of the rows each)
      const int xrow = t.row0 + rank * nb * 16;
      const uint32_t bytes = C::kMats * (kABytes + C::kSfaBytes) + nb * kBox * 128 +
                             (rank == 1 ? sfb_bytes : 0);     // the even CTA's copy
      for (int kk = k0; kk < k1; kk++) {
        if (!first && !mbar_wait(&bars.empty[r.s], r.ph ^ 1, abort)) { ok = false; break; }
        uint8_t* st = smem + r.s * stage_bytes;
        uint64_t* full = &bars.full[r.s];
        if (elect_sync()) {
          mbar_arrive_expect_tx(full, bytes);
          tma_load_2d(st, &p.tm_w, full, kk * 128, wrow);
          if (SWIGLU) tma_load_2d(st + kABytes, &p.tm_up, full, kk * 128, wrow);
          bulk_load(st + C::kOffSfa, sfw + kk * C::kSfaBytes, C::kSfaBytes, full);
          if (SWIGLU)
            bulk_load(st + C::kOffSfa + C::kSfaBytes, sfu + kk * C::kSfaBytes, C::kSfaBytes, full);
          for (int b = 0; b < nb; b++)
            tma_load_2d(st + off_b + b * kBox * 128, &p.tm_x, full, kk * 128, xrow + b * kBox);
        }
        __syncwarp();
        r.next(S);
        if (r.s == 0) first = false;
      }
    }
    if (*abort) {
      // let the copies in flight land before the CTA's memory goes away
      for (int i = 0; i < S; i++) {
        const int s = (r.s + i) % S;
        const bool wrapped = s >= r.s;
        if (first && wrapped) continue;      // never used
        mbar_wait(&bars.full[s], wrapped ? r.ph ^ 1 : r.ph, abort, 20000000LL);
      }
    }
  } else if (warp == 1 && rank == 1) {
    cluster_wait();
    Ring r;
    bool ok = true;
    while (ok && tiles.next(bars, t, abort)) {
      for (int kk = k0; kk < k1; kk++) {
        // All of the odd CTA's stage came by asynchronous copies, whose completion
        // the barrier reports at cluster scope; the word to the even CTA has no
        // scope of its own. (Were there plain stores among them, as the scale
        // warps' once were, it would need cluster-scope release, a fence of about
        // a microsecond each under load: one token per expert 154 -> 254 us,
        // dense 8192^3 207 -> 467, with four warps taking turns 162 and 240.)
        if (!mbar_wait_cluster(&bars.full[r.s], r.ph, abort)) { ok = false; break; }
        if (lane == 0) mbar_arrive_remote(cluster_addr(&bars.full[r.s], 0));
        __syncwarp();
        r.next(S);
      }
    }
  } else if (warp == 1) {
    cluster_wait();
    Ring r;
    Acc<SWIGLU> acc;
    acc.cols = cols;
    int uses = 0;       // stages so far, up to sf_bufs
    int buf = 0;
    bool ok = true;
    const int dsb_word = 32 * row_tiles;       // descriptor units of 16 bytes
    while (ok && tiles.next(bars, t, abort)) {
      const int n = (t.cnt + kUnit - 1) / kUnit * kUnit;
      const uint32_t idesc = idesc_fp4<NV, PAIR>(n);
      acc.take(n);
      if (acc.uses() && !mbar_wait(&bars.acc_empty[acc.h], (acc.uses() - 1) & 1, abort)) break;
      if (acc.both && acc.uses1 && !mbar_wait(&bars.acc_empty[1], (acc.uses1 - 1) & 1, abort)) break;
      tc_fence_after();
      const uint32_t d = tmem + acc.h * cols, du = d + acc.up_offset();
      for (int kk = k0; kk < k1; kk++) {
        if (PAIR ? !mbar_wait_cluster(&bars.full[r.s], r.ph, abort)
                 : !mbar_wait(&bars.full[r.s], r.ph, abort)) { ok = false; break; }
        // The scale buffer's last readers are the MMAs of the stage sf_bufs
        // before. (With as many buffers as stages they have completed: their
        // slot has been filled again.)
        if (uses < sf_bufs) {
          uses++;
        } else if (sf_bufs < S) {
          const int s2 = r.s - sf_bufs;
          if (!mbar_wait(&bars.empty[s2 < 0 ? s2 + S : s2], s2 < 0 ? r.ph ^ 1 : r.ph, abort)) {
            ok = false;
            break;
          }
        }
        tc_fence_after();
        const uint32_t st = smem_u32(smem) + r.s * stage_bytes;
        const uint32_t sfa = tmem + 2 * cols + buf * C::kSfCols;
        const uint32_t sfb = sfa + C::kMats * C::kWords * 4;
        if (elect_sync()) {
          const uint64_t dsa = scale_desc(st + C::kOffSfa), dsb = scale_desc(st + C::kOffSfb);
#pragma unroll
          for (int w = 0; w < C::kMats * C::kWords; w++) tmem_cp_scales<PAIR>(sfa + w * 4, dsa + w * 32);
#pragma unroll
          for (int w = 0; w < C::kWords; w++) tmem_cp_scales<PAIR>(sfb + w * 8, dsb + w * dsb_word);
          if (n > 128) {
#pragma unroll
            for (int w = 0; w < C::kWords; w++) tmem_cp_scales<PAIR>(sfb + w * 8 + 4, dsb + w * dsb_word + 32);
          }
          const uint64_t da = smem_desc_sw128(st), db = smem_desc_sw128(st + off_b);
#pragma unroll
          for (int j = 0; j < 4; j++) {          // 64 k (32 bytes) each
            const int w = NV ? j : j >> 1;
            const uint32_t id = NV ? 0u : (uint32_t)(j & 1) * 2;
            const uint32_t ids = idesc | (id << 29) | (id << 4);
            const uint32_t add = kk > k0 || j ? 1u : 0u;
            mma_fp4<NV, PAIR>(d, da + j * 2, db + j * 2, ids, sfa + w * 4, sfb + w * 8, add);
            if (SWIGLU)
              mma_fp4<NV, PAIR>(du, da + (kABytes >> 4) + j * 2, db + j * 2, ids,
                          sfa + (C::kWords + w) * 4, sfb + w * 8, add);
          }
          commit<PAIR>(&bars.empty[r.s]);
          if (kk == k1 - 1) {
            commit<PAIR>(&bars.acc_full[acc.h]);
            if (acc.both) commit<PAIR>(&bars.acc_full[1]);
          }
        }
        __syncwarp();
        r.next(S);
        if (++buf == sf_bufs) buf = 0;
      }
      acc.done();
    }
    if (*abort) {
      // MMAs in flight read shared memory: wait for the last stages issued
      for (int i = 0; i < uses; i++) {
        const int s = (r.s + 2 * S - 1 - i) % S;
        mbar_wait(&bars.empty[s], s < r.s ? r.ph : r.ph ^ 1, abort, 20000000LL);
      }
    }
  } else if (rank == 0 && (warp < kEpiWarp || warp > kSchedWarp)) {
    // Row scales. The warps take turns at units of 16 scale bytes per row (two
    // stages of MX, one of NV). In a pair both CTAs' MMAs take the scales of all
    // rows: the even CTA's warps put them down here and copy them into the odd
    // one's stage, so that no plain store of one CTA is handed to a thread of the
    // other. (Each CTA for itself is up to 4 % faster, and not in order by the
    // memory model.) A lane reads the one or two 16-byte words
    // around the bytes of rows lane + 32 i (rows may start anywhere), while the
    // warp's last unit waits for its slots, and puts the four rows whose words
    // lie side by side in the layout down at once. (Measured and dropped: every
    // warp at every stage with 32 rows each, where four proxy fences a stage
    // made dense NV products 28 % slower; narrower reads, whose sectors bound a
    // stage of 224 unaligned rows at ~2000 cycles.)
    constexpr int R = (C::kMaxN + 31) / 32, W = C::kWords, U = C::kUnitStages;
    const int wi = warp < kEpiWarp ? warp - 2 : warp - kSchedWarp + 1;
    struct Pos {
      int kk;
      bool more;
      Tile t;
    };
    Pos q;
    q.kk = k0;
    q.more = tiles.next(bars, q.t, abort);
    auto step = [&]() {      // one unit on; the stages of the one left behind
      const int n = min(U, k1 - q.kk);
      q.kk += U;
      if (q.kk >= k1) {
        q.kk = k0;
        q.more = tiles.next(bars, q.t, abort);
      }
      return n;
    };
    auto skip = [&](int units) {
      int n = 0;
      for (int i = 0; i < units && q.more; i++) n += step();
      return n;
    };
    uint4 v[R][2];
    auto fetch = [&]() {
      const int at = q.kk * W * 4, nb = min(p.xs_ld - at, 16);
#pragma unroll
      for (int i = 0; i < R; i++) {
        v[i][0] = v[i][1] = make_uint4(0u, 0u, 0u, 0u);
        if (q.more && lane + 32 * i < q.t.cnt) {
          const uint8_t* g = p.xs + (int64_t)(q.t.row0 + lane + 32 * i) * p.xs_ld + at;
          const int off = (int)((uintptr_t)g & 15);
          const uint4* a = reinterpret_cast<const uint4*>(g - off);
          v[i][0] = __ldg(a);
          if (16 < off + nb) v[i][1] = __ldg(a + 1);     // never without a byte of the row
        }
      }
    };
    Ring r;
    int use = 0;            // stages so far, up to S
    bool ok = true;
    // Waits for the slot of the next stage, i, in the ring: for the MMAs of
    // stage i - S. The parity would take those of i - 3 S for them, were i - 2 S
    // not complete. But this warp has put down stage i - kTurn, or a later one,
    // and so seen stage i - kTurn - S complete, which is i - 2 S or later as
    // long as S >= kTurn.
    auto slot = [&]() {
      ok = use < S || mbar_wait(&bars.empty[r.s], r.ph ^ 1, abort);
      ok = __all_sync(0xffffffffu, ok);
    };
    auto leave = [&]() {
      r.next(S);
      use = min(use + 1, S);
    };
    int ahead = skip(wi);   // stages of the other warps before this one's next
    fetch();
    cluster_wait();
    while (q.more && ok) {
      const int n = min(U, k1 - q.kk), at = q.kk * W * 4, nb = min(p.xs_ld - at, 16);
      uint32_t w[4][8];     // [word][row / 32]
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (i < R) {
          const uint32_t off =
              (uint32_t)((uintptr_t)p.xs + (q.t.row0 + lane + 32 * i) * (int64_t)p.xs_ld + at) & 15u;
          uint32_t u[8] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w,
                           v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w};
#pragma unroll
          for (int j = 0; j < 7; j++) u[j] = off & 4u ? u[j + 1] : u[j];
#pragma unroll
          for (int j = 0; j < 5; j++) u[j] = off & 8u ? u[j + 2] : u[j];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int valid = nb - 4 * j;       // bytes past the row count as 0
            const uint32_t x = __funnelshift_r(u[j], u[j + 1], 8 * (off & 3u));
            w[j][i] = valid >= 4 ? x : valid > 0 ? x & ((1u << (8 * valid)) - 1u) : 0u;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++) w[j][i] = 0u;
        }
      }
      step();
      const int others = skip(C::kScaleWarps - 1);
      fetch();
      for (int i = 0; i < ahead; i++) leave();
      ahead = others;
#pragma unroll
      for (int st = 0; st < U; st++) {
        if (st < n && ok) {
          slot();
          if (ok) {
            uint4* dst = reinterpret_cast<uint4*>(smem + r.s * stage_bytes + C::kOffSfb) + lane;
#pragma unroll
            for (int j = 0; j < W; j++) {
              const uint32_t* x = w[st * W + j];
              dst[j * 32 * row_tiles] = make_uint4(x[0], x[1], x[2], x[3]);
              if (row_tiles == 2) dst[j * 64 + 32] = make_uint4(x[4], x[5], x[6], x[7]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              if (PAIR) {       // (the MMAs of stage i - S have released both CTAs' slots)
                const uint8_t* sfb = smem + r.s * stage_bytes + C::kOffSfb;
                bulk_copy_cluster(cluster_addr(sfb, 1), sfb, sfb_bytes,
                                  cluster_addr(&bars.full[r.s], 1));
              }
              mbar_arrive(&bars.full[r.s]);
            }
            leave();
          }
        }
      }
    }
  } else if (warp >= kEpiWarp && warp < kSchedWarp) {
    cluster_wait();
    // Epilogue: warp % 4 is the lane quadrant, the two warps of a quadrant
    // take alternate groups of 16 rows.
    const int quad = warp & 3, half = (warp - kEpiWarp) >> 2;
    Reduce<SWIGLU> red;
    red.buf = reinterpret_cast<float*>(smem + kRingBytes - kRedBytes);
    red.bars = &bars;
    red.ks = ks;
    red.kp = kp;
    const float tx = p.ts_x ? __ldg(p.ts_x) : 1.f;
    Acc<SWIGLU> acc;
    acc.cols = cols;
    while (tiles.next(bars, t, abort)) {
      const int n = (t.cnt + kUnit - 1) / kUnit * kUnit;
      const int f = t.ft * 128 + quad * 32 + lane;
      const float ag = tx * (p.ts_w ? __ldg(p.ts_w + t.expert) : 1.f);
      const float au = SWIGLU ? tx * (p.ts_up ? __ldg(p.ts_up + t.expert) : 1.f) : 0.f;
      acc.take(n);
      bool ok = mbar_wait(&bars.acc_full[acc.h], acc.uses() & 1, abort);
      if (acc.both) ok = ok && mbar_wait(&bars.acc_full[1], acc.uses1 & 1, abort);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t d = tmem + acc.h * cols + ((uint32_t)(quad * 32) << 16);
      const uint32_t du = d + acc.up_offset();
      if (!PAIR && ks > 1) {
        if (p.out_type == WISP_DT_F32)
          ok = red.template store<float>(p, t, d, du, warp - kEpiWarp, ag, au, abort);
        else if (p.out_type == WISP_DT_BF16)
          ok = red.template store<__nv_bfloat16>(p, t, d, du, warp - kEpiWarp, ag, au, abort);
        else
          ok = red.template store<__half>(p, t, d, du, warp - kEpiWarp, ag, au, abort);
        if (!ok) break;
      } else if (p.out_type == WISP_DT_F32) {
        store_tile<SWIGLU, float>(p, t, d, du, half, f, ag, au);
      } else if (p.out_type == WISP_DT_BF16) {
        store_tile<SWIGLU, __nv_bfloat16>(p, t, d, du, half, f, ag, au);
      } else {
        store_tile<SWIGLU, __half>(p, t, d, du, half, f, ag, au);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) {
          mbar_arrive_remote(cluster_addr(&bars.acc_empty[acc.h], 0));
          if (acc.both) mbar_arrive_remote(cluster_addr(&bars.acc_empty[1], 0));
        } else {
          mbar_arrive(&bars.acc_empty[acc.h]);
          if (acc.both) mbar_arrive(&bars.acc_empty[1]);
        }
      }
      acc.done();
    }
  } else if (warp == kSchedWarp && lane == 0) {
    // Scheduler: finding a tile (a search, a segment read from memory, a
    // division) takes ~1 us, which cost the MMA warp 5 to 24 % of its time.
    const int items = (plan.singles + plan.multi_tiles) * fitems;
    int s = first_done ? 1 : 0;
    uint32_t ph = 0;
    bool first = true;
    for (int it = first_done ? it0 + it_step : it0;; it += it_step) {
      Tile v;
      v.expert = -1;
      v.row0 = v.cnt = v.ft = 0;
      if (it < items) {
        v = find_tile<Cut>(p, plan, it);
        if (PAIR) v.ft = 2 * v.ft + rank;
      }
      if (!first && !mbar_wait(&bars.tile_empty[s], ph ^ 1, abort)) break;
      bars.tile[s] = make_int4(v.expert, v.row0, v.cnt, v.ft);
      mbar_arrive(&bars.tile_full[s]);
      if (++s == kTileRing) {
        s = 0;
        ph ^= 1;
        first = false;
      }
      if (it >= items) break;
    }
  }
  __syncwarp();
  // (the others have waited before their first use of the other CTA's barriers)
  const bool scale_warp = (warp > 1 && warp < kEpiWarp) || warp > kSchedWarp;
  if (warp == 0 || warp == kSchedWarp || (scale_warp && rank == 1)) cluster_wait();
  tc_fence_before();
  cluster_sync();      // no CTA's memory goes away while another uses it
  tc_fence_after();
  if (warp == 1) {
    if (PAIR) {
      tmem_relinquish_pair();
      tmem_dealloc_pair(tmem, 512);
    } else {
      tmem_relinquish();
      tmem_dealloc(tmem, 512);
    }
  }
  if (tid == 0 && bars.abort && p.error_flag) atomicOr(p.error_flag, kErrorTimeout);
}

// Code rows [rows x k/2 bytes] as a 2D tensor; one box = box_rows x 128 bytes
// (256 k), 128-byte swizzle. Bytes past a row and rows past the end read 0.
bool encode_codes(CUtensorMap* m, const void* base, int64_t rows, int k, int box_rows) {
  wb::TensorMapEncodeFn fn = wb::tensor_map_encoder();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)k / 2, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)k / 2};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// grid CTAs in clusters of `cluster`.
template <bool NV, bool SWIGLU, bool PAIR>
WispError launch_product(const Params& p, int dev, unsigned grid, int cluster, cudaStream_t stream,
                         WispErrCtx* err) {
  const int smem = kRingBytes + 1024;
  auto kernel = fp4_product_kernel<NV, SWIGLU, PAIR>;
  static std::atomic<uint64_t> raised{0};
  WB_CUDA_CHECK(wb::raise_smem(kernel, smem, dev, raised));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(Shape<NV, SWIGLU>::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  WB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
  return WISP_OK;
}

template <bool PAIR>
WispError launch_product(bool nv, bool swiglu, const Params& p, int dev, unsigned grid,
                         int cluster, cudaStream_t stream, WispErrCtx* err) {
  if (nv)
    return swiglu ? launch_product<true, true, PAIR>(p, dev, grid, cluster, stream, err)
                  : launch_product<true, false, PAIR>(p, dev, grid, cluster, stream, err);
  return swiglu ? launch_product<false, true, PAIR>(p, dev, grid, cluster, stream, err)
                : launch_product<false, false, PAIR>(p, dev, grid, cluster, stream, err);
}

WispError check_mats(const WispFp4Mats* m, const char* what, WispErrCtx* err) {
  if (!m || !m->codes || !m->prepared)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_product: null pointer argument (%s)", what);
  if (((uintptr_t)m->codes & 15) || ((uintptr_t)m->prepared & 255) ||
      ((uintptr_t)m->tensor_scale & 3))
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp4_product: %s codes must be 16-byte, prepared 256-byte aligned", what);
  return WISP_OK;
}

}  // namespace

extern "C" WispError wisp_b200_fp4_product(const WispFp4Config* cfg, const WispFp4Mats* w,
                                           const WispFp4Mats* up, const WispFp4Rows* x,
                                           const WispSegment* d_segs, int n_segs, void* d_out,
                                           int64_t ld, int* d_error_flag, cudaStream_t stream,
                                           WispErrCtx* err) {
  WispError e = wb::fp4_validate(cfg, "fp4_product", err);
  if (e != WISP_OK) return e;
  if ((e = check_mats(w, "weights", err)) != WISP_OK) return e;
  if (cfg->swiglu && (e = check_mats(up, "up weights", err)) != WISP_OK) return e;
  if (!cfg->swiglu && up)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_product: up weights without swiglu");
  if (!x || x->rows < 0 || x->rows > wb::kMaxRows)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_product: bad rows (0 .. 2^31 - 256)");
  if (d_segs ? (n_segs < 0 || n_segs > kMaxSegs) : n_segs != 0)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_product: n_segs=%d (0..%d, 0 without segments)",
                   n_segs, kMaxSegs);
  if (ld < cfg->n)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_product: ld=%lld < n=%d", (long long)ld, cfg->n);
  if (x->rows == 0 || (d_segs && n_segs == 0)) return WISP_OK;
  if (!x->codes || !x->scales || !d_out)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_product: null pointer argument (rows, out)");
  if (((uintptr_t)x->codes & 15) || ((uintptr_t)x->tensor_scale & 3) ||
      ((uintptr_t)d_out % dt_size(cfg->out_type)) || ((uintptr_t)d_segs & 3) ||
      ((uintptr_t)d_error_flag & 3))
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp4_product: row codes must be 16-byte aligned, segments and error word 4-byte, "
                   "out to its type");
  const bool nv = cfg->format == WISP_FP4_NV;
  if (!nv && x->tensor_scale)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp4_product: MX rows have no tensor scale");
  int dev = 0, sms = 0;
  WB_CUDA_CHECK(wb::device_sms(&dev, &sms));
  // Token tiles of at most `cap` rows, an upper bound: at most one per row, and
  // per segment one more than its rows fill.
  int cap = nv ? Shape<true, false>::kMaxN : Shape<false, false>::kMaxN;
  auto tiles_of = [&](int rows_per_tile) {
    const int64_t most = (int64_t)x->rows / rows_per_tile + (d_segs ? n_segs : 1);
    return most < x->rows ? most : x->rows;
  };
  const int64_t tiles = tiles_of(cap);
  const int ftiles = (cfg->n + 127) / 128, nk = (cfg->k + 255) / 256;
  // Pairs, unless there are few rows and all tiles together could use at most
  // 3/8 of the SMs as single CTAs: then clusters of 4 (2) of these split K, as
  // long as they fill at most 3/4 of the SMs (GPCs of an odd number of SMs hold
  // fewer clusters) and have two stages of K each. One row, warm L2, us a call,
  // as pairs / split by 2 / by 4: 2048 x 7168 11.6 / 10.4 / 8.6, with gate and
  // up 13.1 / 11.9 / 9.6, 2048 x 2048 7.3 / 7.5 / 7.0, 7168 x 2048 7.6 / 7.8 /
  // 14.0 (two waves). More rows pay a cluster round per 16.
  const int64_t items = tiles * ftiles;
  const int split = nk < 8 || x->rows > 64              ? 1
                    : items * 16 <= 3 * (int64_t)sms ? 4
                    : items * 8 <= 3 * (int64_t)sms  ? 2
                                                     : 1;
  // With one feature tile a pair's second CTA would have none: single CTAs.
  const bool single = split == 1 && ftiles == 1;
  if (split == 1) {
    // Smaller tiles when the largest would leave pairs without work: as many
    // rows as give every pair one tile if the rows lay in one segment, at least
    // 64 (what the MMA's fixed cost per weight is paid for anyway). 666 rows in
    // 11 ragged segments, 1000 x 2080 with gate and up: 15.0 -> 13.0 us.
    const int64_t width = single ? 1 : (ftiles + 1) / 2 * 2;
    const int64_t per = ((int64_t)x->rows * width + sms - 1) / sms;
    const int fit = per < 64 ? 64 : per > cap ? cap : (int)((per + 31) & ~31);
    if (fit < cap) cap = fit;
  }
  Params p;
  memset(&p, 0, sizeof p);
  p.cap = cap;
  const int64_t wrows = (int64_t)cfg->n_entries * cfg->n;
  if (!encode_codes(&p.tm_w, w->codes, wrows, cfg->k, 128) ||
      (cfg->swiglu && !encode_codes(&p.tm_up, up->codes, wrows, cfg->k, 128)) ||
      !encode_codes(&p.tm_x, x->codes, x->rows, cfg->k, split > 1 || single ? 32 : 16))
    return WB_FAIL(WISP_ERR_CUDA, "fp4_product: cuTensorMapEncodeTiled failed");
  p.sf_w = static_cast<const uint8_t*>(w->prepared);
  p.ts_w = w->tensor_scale;
  if (cfg->swiglu) {
    p.sf_up = static_cast<const uint8_t*>(up->prepared);
    p.ts_up = up->tensor_scale;
  }
  p.ts_x = x->tensor_scale;
  p.xs = x->scales;
  p.xs_ld = cfg->k / (nv ? 16 : 32);
  p.rows = x->rows;
  p.segs = d_segs;
  p.nseg = n_segs;
  p.V = cfg->n_entries;
  p.N = cfg->n;
  p.nk = nk;
  p.ftiles = ftiles;
  p.out = d_out;
  p.ld = ld;
  p.out_type = cfg->out_type;
  p.error_flag = d_error_flag;
  if (split > 1)
    return launch_product<false>(nv, cfg->swiglu, p, dev, (unsigned)(items * split), split, stream,
                                 err);
  if (single) {
    const int64_t want = tiles_of(cap);
    return launch_product<false>(nv, cfg->swiglu, p, dev, (unsigned)(want < sms ? want : sms), 1,
                                 stream, err);
  }
  const int64_t want = tiles_of(cap) * ((ftiles + 1) / 2) * 2;
  return launch_product<true>(nv, cfg->swiglu, p, dev,
                              (unsigned)(want < (sms & ~1) ? want : sms & ~1), 2, stream, err);
}
