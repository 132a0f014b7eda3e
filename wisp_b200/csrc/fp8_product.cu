// fp8_product.cu -- out[p, f] = sum_b xs[p, b] ws_e[f / 128, b] sum_{k in b} x[p, k] w_e[f, k]
// over e4m3 rows with one fp32 scale per block b of 128 k and e4m3 expert
// matrices with one per block of 128 x 128 (one expert per segment of rows).
//
// The scales are no powers of two, so the tensor cores cannot apply them: each
// block of 128 k is an MMA accumulation of its own in tensor memory (four
// tcgen05.mma of 32 k), which the epilogue warps scale and add to fp32 sums in
// registers while the MMAs of the next blocks fill other buffers.
//
// Two forms of tile, for one CTA pair (cta_group::2, M = 256) or a single CTA
// (cta_group::1, M = 128):
//   narrow (at most 128 rows): the features are the MMA's M (128 per CTA), the
//     rows its N, any multiple of 16 (32 in a pair), so that a weight matrix
//     streams through once and few rows cost little. An accumulator lane is one
//     feature; the rows' scales run over the columns and are read from shared
//     memory.
//   wide (129 to 256 rows, pairs only): the rows are M (128 per CTA), N is 256
//     features, one block of 128 in either CTA's shared memory: two of one
//     matrix, or gate in the even and up in the odd CTA. A lane is one row: its
//     scale is one register, where the narrow form would read 4 bytes of shared
//     memory per accumulator and block (and take two passes over the weights).
//
// What a buffer of accumulators waits for bounds a product of many rows: from its
// MMAs' issue to the next ones' into it pass their own time, 400 cycles until the
// barriers have reported them, the loads into registers, and 160 until the MMA
// warp has seen it free. So one barrier stands for a whole block (gate and up, or
// both blocks of features: groups of 128 columns with barriers of their own have
// twice the waits, and a wide tile's MMAs then read the rows twice from shared
// memory), and a buffer is free as soon as it has been read, before the last of it is
// added.
//
// Measured (us; L2 flushed by writes, whose way back to memory costs ~20): 64 experts of
// 2 x 2048 x 7168 with 1 / 64 / 128 / 256 rows each 289 / 302 / 334 / 444, where the
// weights take 287 at the copy rate (on another B200 297 / 308 / 344 / 455); 64 of 7168 x
// 2048, fp32 outputs, 171 / 192 / 233 / 281 (143): bound by HBM up to ~100 rows. 8192 x 8192 x
// 7168 373 = 2.58 PFLOP/s; without a pause between calls 470, as the power limit lowers
// the clock. A block of a wide tile takes 0.44 (0.27 at the MMAs' nominal rate), a change of
// tiles 2.5 more.
//
// Warps of a persistent CTA: 0 issues the TMA copies (128 k per stage, 128-byte
// swizzle), 1 the MMAs, 2 hands out the tiles, 3 multiplies the scales, 4-11 are the
// epilogue, with the registers that the first four give up. An epilogue warp's work
// on a block is a chain of dependent steps (wait, load, release, add) that its one
// companion on the scheduler cannot hide, so the steps around the additions are kept
// few: one wait a block, no branch by lane, no addresses to work out.
#include "common.cuh"
#include "internal.h"
#include "numeric.cuh"
#include "tiles.cuh"

namespace {

using namespace wb;

constexpr int kThreads = 384;
constexpr int kSchedWarp = 2;
constexpr int kEpiWarp = 4;       // first of 8 epilogue warps
constexpr int kABytes = 128 * 128;
constexpr int kNarrow = 128;      // rows of a narrow tile at most
constexpr int kWide = 256;
constexpr int kMaxStages = 12;
constexpr int kMaxBufs = 8;
constexpr int kRingBytes = 206 * 1024;
constexpr int kStoreBytes = 8 * 4096;     // of these, where wide tiles' outputs change places
// Blocks whose scales are held or on their way; scales of a block: of the CTA's rows,
// then the weights' two.
constexpr int kRawSlots = 8, kRawFloats = 132;
constexpr int kTileRing = 8;
static_assert(kMaxStages > kMaxBufs && kMaxStages >= kTileRing, "threads that initialise barriers");
// Registers: launch 168 x 384 = 64,512; 256 x 232 + 128 x 40 = 64,512.
constexpr int kEpiRegs = 232, kOtherRegs = 40;
struct Bars {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full[kMaxBufs];
  uint64_t acc_empty[kMaxBufs];
  uint64_t scale_empty[kMaxBufs];
  uint64_t red_full, red_empty;     // partial sums of a cluster's CTAs
  uint64_t tile_full[kTileRing];
  uint64_t tile_empty[kTileRing];
  int4 tile[kTileRing];     // expert (-1: no more), first row, rows, feature tile
  uint32_t tmem;
  int abort;
};

struct alignas(64) Params {
  CUtensorMap tm_w, tm_up, tm_x, tm_x128;     // tm_x: boxes of 16 rows, tm_x128 of 128
  const float* ws_w;
  const float* ws_up;
  const float* xs;        // scale of row p, block b: xs[p * xs_row + b * xs_block]
  int64_t xs_row, xs_block;
  int rows;
  const WispSegment* segs;
  int nseg;
  int V, N, nk, ftiles;
  int cap;                // rows per tile at most: a multiple of 32 up to kNarrow, or kWide
  void* out;
  int64_t ld;
  int wide_out, even_out;   // output rows start on 32-byte, 4-byte boundaries
  int* error_flag;
};

// kWide: whole wide tiles and a rest, so that the rest can be a narrow one.
template <int UNIT>
struct Cut8 {
  WB_DEV static int rows(int rows, int cap) {
    return cap == kWide && rows > kWide ? kWide : EvenCut<UNIT>::rows(rows, cap);
  }
};

// Instruction descriptor of kind::f8f6f4: A and B e4m3, both K-major, fp32 sums.
WB_DEV uint32_t idesc_fp8(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <bool PAIR>
WB_DEV void mma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}

// Registers that a wait for loads has covered: as operands, they cannot be read
// before it.
WB_DEV void waited(uint32_t (&v)[32]) {
  asm volatile(""
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]),
                 "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                 "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]),
                 "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                 "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                 "+r"(v[30]), "+r"(v[31])
               :
               : "memory");
}
// Arrivals of one lane without a branch.
WB_DEV void arrive_one(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\t"
      "@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(smem_u32(bar)) : "memory");
}
WB_DEV void arrive_one_remote(uint32_t cluster_bar) {
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\t"
      "@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}" ::"r"(cluster_bar) : "memory");
}

WB_DEV void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
}

// Two sums of products per instruction.
WB_DEV void fma2(float2& c, float2 a, float2 b) {
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mov.b64 z, {%0, %1};\n\tfma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "+f"(c.x), "+f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
}

// The sums of one thread.
//   wide:   features [half 64 ..][64] of the first block of 128, then of the second
//   narrow: [matrix][chunk j: rows (2 j + half) 32 ..][32]; one matrix uses the
//           first 32
struct Sums {
  float2 v[64];
};

// A warp of the epilogue.
struct Warp {
  int lane, quad, half, rank;
};

// sums += accumulators * a scale each, of 32 columns.
WB_DEV void add32(float2* v, const uint32_t (&u)[32], float y) {
#pragma unroll
  for (int q = 0; q < 16; q++)
    fma2(v[q], make_float2(__uint_as_float(u[2 * q]), __uint_as_float(u[2 * q + 1])),
         make_float2(y, y));
}
WB_DEV void add32(float2* v, const uint32_t (&u)[32], const float* s) {
#pragma unroll
  for (int q = 0; q < 16; q += 2) {
    const float4 y = *reinterpret_cast<const float4*>(s + 2 * q);
    fma2(v[q], make_float2(__uint_as_float(u[2 * q]), __uint_as_float(u[2 * q + 1])),
         make_float2(y.x, y.y));
    fma2(v[q + 1], make_float2(__uint_as_float(u[2 * q + 2]), __uint_as_float(u[2 * q + 3])),
         make_float2(y.z, y.w));
  }
}

// The scale warp: of a tile's scales, block by block, the products of each row's
// with the weights' two (gate and up, or a wide tile's blocks of features). The
// scales come by cp.async (4 bytes, so that rows' scales may lie anywhere)
// kRawSlots - 1 blocks ahead; the products go where the block's buffer of
// accumulators has its place. Rows past the tile's have none: what their lanes and
// columns hold is not stored.
template <bool SWIGLU>
WB_DEV bool multiply_scales(const Params& p, const Tile& t, bool wide, int rank, int k0, int k1,
                            Bars& bars, float (*raw)[kRawFloats], float (*products)[256], Ring& r,
                            bool& first, int bufs, volatile int* abort) {
  const int lane = threadIdx.x & 31;
  const int row = (wide ? rank * 128 : 0) + lane, left = t.cnt - row;
  const float* x = p.xs + (t.row0 + (int64_t)row) * p.xs_row + k0 * p.xs_block;
  const int fb = wide && !SWIGLU ? (t.ft & ~1) + lane : t.ft;
  const float* w = (SWIGLU && lane ? p.ws_up : p.ws_w) +
                   ((int64_t)t.expert * p.ftiles + min(fb, p.ftiles - 1)) * p.nk + k0;
  const bool two = SWIGLU || wide, has_w = lane < (two ? 2 : 1);
  int in = 0;
  auto fetch = [&](int kk) {
    if (kk < k1) {
      float* s = raw[in] + lane;
      if (left > 0) cp_async_4(s, x);
      if (left > 32) cp_async_4(s + 32, x + 32 * p.xs_row);
      if (left > 64) cp_async_4(s + 64, x + 64 * p.xs_row);
      if (left > 96) cp_async_4(s + 96, x + 96 * p.xs_row);
      if (has_w) cp_async_4(s + 128, w);
      x += p.xs_block;
      w++;
    }
    cp_async_commit();
    in = (in + 1) % kRawSlots;
  };
#pragma unroll 1
  for (int i = 0; i < kRawSlots - 1; i++) fetch(k0 + i);
  for (int kk = k0; kk < k1; kk++) {
    __syncwarp();                // the slot that is filled next has been read
    const float* s = raw[(in + 1) % kRawSlots];
    fetch(kk + kRawSlots - 1);
    cp_async_wait<kRawSlots - 1>();
    __syncwarp();                // every lane's copies of this block have landed
    // four rows a lane, ready before the place they go to
    const float4 v = reinterpret_cast<const float4*>(s)[lane];
    const float w0 = s[128], w1 = s[129];
    const bool ok = first || mbar_wait(&bars.scale_empty[r.s], r.ph ^ 1, abort);
    if (!__all_sync(0xffffffffu, ok)) return false;
    float4* o = reinterpret_cast<float4*>(products[r.s]) + lane;
    o[0] = make_float4(v.x * w0, v.y * w0, v.z * w0, v.w * w0);
    if (two) o[32] = make_float4(v.x * w1, v.y * w1, v.z * w1, v.w * w1);
    __syncwarp();
    // (its last reads being over, so is the barrier's last phase)
    arrive_one(&bars.acc_full[r.s]);
    r.next(bufs);
    if (r.s == 0) first = false;
  }
  return true;
}

// A wide tile's outputs: a lane holds a row. 128 bytes of each row at a time change
// places in the warp's 4 KB of shared memory (16-byte words, swizzled), so that eight
// lanes write a line of one row, or the whole warp where rows start anywhere. (Straight
// from the registers, 32 bytes or one value of 32 rows per instruction, the lines pass one
// a cycle: 8192 x 8192 x 7168 385 us, so 375; 64 experts of 7168 x 2048 with 256 rows and
// fp32 outputs 300 and 282; 31 experts of 2 x 3754 x 224 with ~150 rows, whose rows start
// on 4 bytes, 263 and 64.)
template <bool SWIGLU, typename T>
WB_DEV void store_wide(const Params& p, const Sums& a, const Tile& t, const Warp& me, uint4* stage) {
  const int row0 = me.rank * 128 + me.quad * 32, rows = min(t.cnt - row0, 32);
  if (rows <= 0) return;
  constexpr int kWord = 16 / (int)sizeof(T), kLine = 8 * kWord;      // values
  constexpr int kType = sizeof(T) == 4 ? WISP_DT_F32
                                       : std::is_same<T, __half>::value ? WISP_DT_F16 : WISP_DT_BF16;
  T* out = static_cast<T*>(p.out) + (t.row0 + (int64_t)row0) * p.ld;
#pragma unroll
  for (int q = 0; q < (SWIGLU ? 1 : 2); q++) {
#pragma unroll
    for (int l = 0; l < 64; l += kLine) {
      __syncwarp();                      // the last line has been read
#pragma unroll
      for (int w = 0; w < 8; w++) {
        float o[kWord];
#pragma unroll
        for (int j = 0; j < kWord; j++) {
          const int i = l + w * kWord + j;
          const float2 g = a.v[q * 32 + i / 2], u = a.v[32 + i / 2];
          o[j] = i & 1 ? g.y : g.x;
          if (SWIGLU) o[j] = swiglu<T>(o[j], i & 1 ? u.y : u.x);
        }
        uint32_t v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if constexpr (sizeof(T) == 4)
            v[j] = __float_as_uint(o[j]);
          else
            v[j] = pack2(o[2 * j], o[2 * j + 1], kType);
        }
        stage[me.lane * 8 + (w ^ (me.lane & 7))] = make_uint4(v[0], v[1], v[2], v[3]);
      }
      __syncwarp();
      const int f = (SWIGLU ? t.ft : (t.ft & ~1) + q) * 128 + me.half * 64 + l;
      if (f >= p.N) return;
      const int left = p.N - f;          // values of the line that there are
      if (p.wide_out && left >= kLine) {
        const int r = me.lane >> 3, c = me.lane & 7;
        T* o = out + f + r * p.ld + c * kWord;
#pragma unroll
        for (int i = 0; i < 32; i += 4, o += 4 * p.ld)
          if (r + i < rows)
            *reinterpret_cast<uint4*>(o) = stage[(r + i) * 8 + (c ^ ((r + i) & 7))];
      } else {
        using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
        const bool pairs = sizeof(T) == 2 && p.even_out;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(stage) + (me.lane & 3);
        Bits* o = reinterpret_cast<Bits*>(out + f);
#pragma unroll 4
        for (int i = 0; i < rows; i++, o += p.ld) {
          const uint32_t v = words[i * 32 + 4 * (me.lane / 4 ^ (i & 7))];
          if constexpr (sizeof(T) == 4) {
            if (me.lane < left) o[me.lane] = v;
          } else if (pairs && 2 * me.lane + 1 < left) {
            *reinterpret_cast<uint32_t*>(o + 2 * me.lane) = v;
          } else {
            if (2 * me.lane < left) o[2 * me.lane] = (Bits)v;
            if (2 * me.lane + 1 < left) o[2 * me.lane + 1] = (Bits)(v >> 16);
          }
        }
      }
    }
  }
}

// The same for silu(gate) * up on rows that start on 32 bytes, straight from the
// registers: half the values, and the shared memory is a stage of the ring (64 experts
// of 2 x 2048 x 7168 with 256 rows 457 us; through it 467).
template <typename T>
WB_DEV void store_wide_swiglu(const Params& p, const Sums& a, const Tile& t, const Warp& me) {
  const int r = me.rank * 128 + me.quad * 32 + me.lane;
  if (r >= t.cnt) return;
  T* row = static_cast<T*>(p.out) + (t.row0 + (int64_t)r) * p.ld;
  constexpr int kRun = 32 / (int)sizeof(T);      // values of a 32-byte store
  const int f = t.ft * 128 + me.half * 64;
#pragma unroll
  for (int i = 0; i < 64; i += kRun) {
    float o[kRun];
#pragma unroll
    for (int j = 0; j < kRun; j++) {
      const float2 g = a.v[(i + j) / 2], u = a.v[32 + (i + j) / 2];
      o[j] = swiglu<T>(j & 1 ? g.y : g.x, j & 1 ? u.y : u.x);
    }
    if (f + i + kRun <= p.N) {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if constexpr (sizeof(T) == 4)
          w[j] = __float_as_uint(o[j]);
        else
          w[j] = pack2(o[2 * j], o[2 * j + 1],
                       std::is_same<T, __half>::value ? WISP_DT_F16 : WISP_DT_BF16);
      }
      store32(row + f + i, w);
    } else {
#pragma unroll
      for (int j = 0; j < kRun; j++)
        if (f + i + j < p.N) put_out(row + f + i + j, o[j]);
    }
  }
}

template <bool SWIGLU, typename T>
WB_DEV void store_narrow(const Params& p, const Sums& a, const Tile& t, const Warp& me) {
  const int64_t ld = p.ld;
  const int f = t.ft * 128 + me.quad * 32 + me.lane;
  if (f >= p.N) return;
  T* out = static_cast<T*>(p.out) + (int64_t)t.row0 * ld + f;
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const int c = (2 * j + me.half) * 32;
    if (c < t.cnt) {
      T* q = out + c * ld;
#pragma unroll
      for (int i = 0; i < 32; i++, q += ld) {
        // (out of the unrolled code at once: walking past it, from cold instructions, is
        // 1 us of a call with one row: gate/up 2048 x 1024 10.3, so 9.3)
        if (c + i >= t.cnt) break;
        const float2 g = a.v[j * 16 + i / 2];
        float o = i & 1 ? g.y : g.x;
        if (SWIGLU) {
          const float2 u = a.v[32 + j * 16 + i / 2];
          o = swiglu<T>(o, i & 1 ? u.y : u.x);
        }
        put_out(q, o);
      }
    }
  }
}

// The join of a cluster whose CTAs split K (tiles of at most 64 rows).
// 16 rows of each half at a time, every CTA puts its sums into its shared memory, and CTA kp
// adds those of all, in the order of K, for the rows kp, kp + ks, ... (a warp per
// row, 4 features per lane).
constexpr int kRedRows = 32, kSplitRows = 64;
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

  template <typename T>
  WB_DEV bool store(const Params& p, const Sums& a, const Tile& t, const Warp& me,
                    volatile int* abort) {
    const int lane = me.lane, w = me.half * 4 + me.quad;
#pragma unroll
    for (int j = 0; j < kSplitRows / kRedRows; j++) {
      // rows 16 j + (0 .. 15) and 32 + 16 j + (0 .. 15)
      if (16 * j >= t.cnt) break;
      bool ok = uses == 0 || mbar_wait_cluster(&bars->red_empty, (uses - 1) & 1, abort);
      if (!__all_sync(0xffffffffu, ok)) return false;
      if (me.half * 32 + 16 * j < t.cnt) {
        float* q = buf + me.half * 16 * 128 + me.quad * 32 + lane;
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float2 g = a.v[j * 8 + i / 2];
          q[i * 128] = i & 1 ? g.y : g.x;
          if (SWIGLU) {
            const float2 u = a.v[32 + j * 8 + i / 2];
            q[(kRedRows + i) * 128] = i & 1 ? u.y : u.x;
          }
        }
      }
      arrive_all(&bars->red_full);
      ok = mbar_wait_cluster(&bars->red_full, uses & 1, abort);
      if (!__all_sync(0xffffffffu, ok)) return false;
      for (int r = kp + ks * w; r < kRedRows; r += ks * 8) {
        const int row = (r & 16) * 2 + 16 * j + (r & 15);
        if (row >= t.cnt) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f}, x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < ks; i++) {
          const uint32_t at = cluster_addr(buf + r * 128 + lane * 4, i);
          const float4 y = ld_cluster_f4(at);
          v[0] += y.x;
          v[1] += y.y;
          v[2] += y.z;
          v[3] += y.w;
          if (SWIGLU) {
            const float4 z = ld_cluster_f4(at + kRedRows * 128 * 4);
            x[0] += z.x;
            x[1] += z.y;
            x[2] += z.z;
            x[3] += z.w;
          }
        }
        const int f = t.ft * 128 + lane * 4;
        T* out = static_cast<T*>(p.out) + (t.row0 + (int64_t)row) * p.ld + f;
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (f + i < p.N) put_out(out + i, SWIGLU ? swiglu<T>(v[i], x[i]) : v[i]);
      }
      arrive_all(&bars->red_empty);
      uses++;
    }
    return true;
  }
};

// DIRECT: wide tiles' outputs leave by store_wide_swiglu. (Both forms in one kernel: the
// 457 us above became 467.)
template <typename T, bool SWIGLU, bool PAIR, bool DIRECT>
__global__ void __launch_bounds__(kThreads, 1)
fp8_product_kernel(const __grid_constant__ Params p) {
  constexpr int kMats = SWIGLU ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ Bars bars;
  __shared__ alignas(16) float raw[kRawSlots][kRawFloats];
  __shared__ alignas(16) float products[kMaxBufs][256];      // of scales
  __shared__ int pref[kMaxSegs];
  __shared__ uint16_t order[kMaxSegs];
  __shared__ int4 warp_tot[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  volatile int* abort = &bars.abort;
  constexpr int kUnit = PAIR ? 32 : 16;
  using Cut = Cut8<kUnit>;
  // pair: this CTA's place in it; else the K split: kp of ks
  const int rank = PAIR ? (int)cluster_rank() : 0;
  const int ks = PAIR ? 1 : (int)cluster_size(), kp = PAIR ? 0 : (int)cluster_rank();
  const int fitems = PAIR ? (p.ftiles + 1) / 2 : p.ftiles;

  if (warp == 0 && elect_sync()) {
    tma_prefetch_desc(&p.tm_w);
    tma_prefetch_desc(&p.tm_x);
    if (SWIGLU) tma_prefetch_desc(&p.tm_up);
    if (PAIR && p.cap > kNarrow) tma_prefetch_desc(&p.tm_x128);
  }
  __syncwarp();
  if (tid < kMaxStages) {
    // the copies; the odd CTA's word
    mbar_init(&bars.full[tid], PAIR && rank == 0 ? 2 : 1);
    mbar_init(&bars.empty[tid], 1);
    if (tid < kTileRing) {
      mbar_init(&bars.tile_full[tid], 1);
      mbar_init(&bars.tile_empty[tid], 11);     // all warps that walk the tiles
    }
    if (tid < kMaxBufs) {
      mbar_init(&bars.acc_full[tid], 2);        // the MMAs, the products of scales
      mbar_init(&bars.scale_empty[tid], 8);
      mbar_init(&bars.acc_empty[tid], PAIR ? 16 : 8);
    } else if (tid == kMaxBufs) {
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
  // a wide item of gate and up is two tiles, which only the scheduler hands out
  const bool two_tiles = PAIR && SWIGLU && p.cap > kNarrow;
  int max_cnt;
  bool first_done;
  const Plan plan = make_plan<Cut, kThreads>(
      p, fitems, it0, pref, order, warp_tot, max_cnt, first_done,
      [&](const WispSegment& v, int ft) {
        if (two_tiles) return;
        bars.tile[0] = make_int4(v.expert, v.row_begin, v.rows, PAIR ? 2 * ft + rank : ft);
        mbar_arrive(&bars.tile_full[0]);
      });
  if (two_tiles) first_done = false;
  const bool wides = PAIR && max_cnt > kNarrow;
  // the scheduler warp reads pref and order
  __syncthreads();
  const uint32_t tmem = bars.tmem;
  const int k0 = PAIR ? 0 : p.nk * kp / ks, k1 = PAIR ? p.nk : p.nk * (kp + 1) / ks;     // this CTA's stages
  // A stage: weights (in narrow tiles gate and up), then rows: of a narrow tile n
  // (a pair's CTA half of them), of a wide one 128. Few rows leave room for more
  // stages, which is what hides the memory's latency when the weights are most of
  // the traffic.
  const int narrow_n = (min(max_cnt, kNarrow) + kUnit - 1) / kUnit * kUnit;
  const int narrow_bytes = kMats * kABytes + narrow_n / (PAIR ? 2 : 1) * 128;
  const int stage_bytes = wides ? max(narrow_bytes, 2 * kABytes) : narrow_bytes;
  constexpr int kRedBytes = kMats * kRedRows * 128 * 4;     // a cluster's partial sums
  const int S = min(kMaxStages, (kRingBytes - (ks > 1 ? kRedBytes : wides && !DIRECT ? kStoreBytes : 0)) / stage_bytes);
  // accumulators: buffers of `cols` columns, one for a block of k (gate, then up)
  const int up_offset = (narrow_n + 31) & ~31;
  const int cols = wides ? kWide : up_offset * kMats;
  const int bufs = min(kMaxBufs, 512 / cols);
  TileWalk<kTileRing> tiles;
  Tile t;

  // (within each role, so that the compiler knows what the role may use)
  if (warp == 0) {
    give_registers();
    Ring r;
    bool first = true, ok = true;
    while (ok && tiles.next(bars, t, abort)) {
      const bool wide = PAIR && t.cnt > kNarrow;
      const int wrow = t.expert * p.N + t.ft * 128;
      const bool second = SWIGLU && wide && rank == 1;      // this CTA's block is up's
      const int nb = ((t.cnt + kUnit - 1) / kUnit);         // boxes of 16 rows
      const int xrow = t.row0 + rank * (wide ? 128 : nb * 16);
      const uint32_t bytes = wide ? 2 * kABytes : kMats * kABytes + nb * 2048;
      for (int kk = k0; kk < k1; kk++) {
        if (!first && !mbar_wait(&bars.empty[r.s], r.ph ^ 1, abort)) { ok = false; break; }
        uint8_t* st = smem + r.s * stage_bytes;
        uint64_t* full = &bars.full[r.s];
        if (elect_sync()) {
          mbar_arrive_expect_tx(full, bytes);
          if (wide) {
            tma_load_2d(st, second ? &p.tm_up : &p.tm_w, full, kk * 128, wrow);
            tma_load_2d(st + kABytes, &p.tm_x128, full, kk * 128, xrow);
          } else {
            tma_load_2d(st, &p.tm_w, full, kk * 128, wrow);
            if (SWIGLU) tma_load_2d(st + kABytes, &p.tm_up, full, kk * 128, wrow);
            for (int b = 0; b < nb; b++)
              tma_load_2d(st + kMats * kABytes + b * 2048, &p.tm_x, full, kk * 128, xrow + b * 16);
          }
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
    cluster_wait();
  } else if (warp == 1 && rank == 1) {
    give_registers();
    cluster_wait();
    Ring r;
    bool ok = true;
    while (ok && tiles.next(bars, t, abort)) {
      for (int kk = k0; kk < k1; kk++) {
        // All of the odd CTA's stage came by asynchronous copies, whose completion
        // the barrier reports at cluster scope; the word to the even CTA has no
        // scope of its own.
        if (!mbar_wait_cluster(&bars.full[r.s], r.ph, abort)) { ok = false; break; }
        if (lane == 0) mbar_arrive_remote(cluster_addr(&bars.full[r.s], 0));
        __syncwarp();
        r.next(S);
      }
    }
  } else if (warp == 1) {
    give_registers();
    cluster_wait();
    Ring r, b;                    // stages, accumulators
    int uses = 0;                 // stages so far, up to S
    bool fresh = true, ok = true;
    while (ok && tiles.next(bars, t, abort)) {
      const bool wide = PAIR && t.cnt > kNarrow;
      const int n = (t.cnt + kUnit - 1) / kUnit * kUnit;
      const uint32_t idesc = idesc_fp8(PAIR ? 256 : 128, wide ? kWide : n);
      for (int kk = k0; kk < k1; kk++) {
        if (PAIR ? !mbar_wait_cluster(&bars.full[r.s], r.ph, abort)
                 : !mbar_wait(&bars.full[r.s], r.ph, abort)) { ok = false; break; }
        // A, B: rows and weights of a wide tile, weights and rows of a narrow one.
        const uint32_t st = smem_u32(smem) + r.s * stage_bytes;
        const uint64_t dw = smem_desc_sw128(st);
        const uint64_t dx = smem_desc_sw128(st + (wide ? kABytes : kMats * kABytes));
        const uint32_t d = tmem + b.s * cols;
        if (!fresh && !mbar_wait(&bars.acc_empty[b.s], b.ph ^ 1, abort)) { ok = false; break; }
        tc_fence_after();
        if (elect_sync()) {
#pragma unroll
          for (int j = 0; j < 4; j++) {          // 32 k (32 bytes) each
            mma_fp8<PAIR>(d, (wide ? dx : dw) + j * 2, (wide ? dw : dx) + j * 2, idesc, j ? 1u : 0u);
            if (SWIGLU && !wide)
              mma_fp8<PAIR>(d + up_offset, dw + (kABytes >> 4) + j * 2, dx + j * 2, idesc, j ? 1u : 0u);
          }
          commit<PAIR>(&bars.acc_full[b.s]);
          commit<PAIR>(&bars.empty[r.s]);
        }
        __syncwarp();
        b.next(bufs);
        if (b.s == 0) fresh = false;
        r.next(S);
        uses = min(uses + 1, S);
      }
    }
    if (*abort) {
      // MMAs in flight read shared memory: wait for the last stages issued
      for (int i = 0; i < uses; i++) {
        const int s = (r.s + 2 * S - 1 - i) % S;
        mbar_wait(&bars.empty[s], s < r.s ? r.ph : r.ph ^ 1, abort, 20000000LL);
      }
    }
  } else if (warp >= kEpiWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    cluster_wait();
    // warp % 4 is the lane quadrant; the two warps of a quadrant take alternate
    // groups of 32 rows of a narrow tile, a half of each 128 features of a wide one
    const Warp me = {lane, warp & 3, (warp - kEpiWarp) >> 2, rank};
    Reduce<SWIGLU> red;
    red.buf = reinterpret_cast<float*>(smem + kRingBytes - kRedBytes);
    red.bars = &bars;
    red.ks = ks;
    red.kp = kp;
    uint4* stage = reinterpret_cast<uint4*>(smem + kRingBytes - kStoreBytes) + (warp - kEpiWarp) * 256;
    Ring b;
    const uint32_t base = tmem + ((uint32_t)(me.quad * 32) << 16);
    const uint32_t empty0 = cluster_addr(&bars.acc_empty[0], PAIR ? 0 : kp);
    bool ok = true;
    // The next block's accumulators and products of scales are there, and have been
    // read.
    auto full = [&]() {
      ok = __all_sync(0xffffffffu, mbar_wait(&bars.acc_full[b.s], b.ph, abort));
      tc_fence_after();
      return ok;
    };
    auto release = [&]() {
      tc_fence_before();
      __syncwarp();
      if (PAIR)
        arrive_one_remote(empty0 + b.s * 8);
      else
        arrive_one(&bars.acc_empty[b.s]);
    };
    auto release_scales = [&]() {
      __syncwarp();
      arrive_one(&bars.scale_empty[b.s]);
      b.next(bufs);
    };
    while (ok && tiles.next(bars, t, abort)) {
      const bool wide = PAIR && t.cnt > kNarrow;
      Sums a;
#pragma unroll
      for (int i = 0; i < 64; i++) a.v[i] = make_float2(0.f, 0.f);
      if (wide) {
        for (int kk = k0; kk < k1; kk++) {
          if (!full()) break;
          uint32_t u[2][32];
          const uint32_t d = base + b.s * cols + me.half * 64;
          tmem_ld32(d, u[0]);
          tmem_ld32(d + 32, u[1]);
          const float* s = products[b.s] + me.quad * 32 + lane;
          const float y0 = s[0], y1 = s[128];
          tmem_wait_ld();
          waited(u[0]);
          add32(a.v, u[0], y0);
          tmem_ld32(d + 128, u[0]);
          waited(u[1]);
          add32(a.v + 16, u[1], y0);
          tmem_ld32(d + 160, u[1]);
          tmem_wait_ld();
          waited(u[0]);
          waited(u[1]);
          release();
          release_scales();
          add32(a.v + 32, u[0], y1);
          add32(a.v + 48, u[1], y1);
        }
      } else {
        const uint32_t c = me.half * 32;
        const int chunks = t.cnt > (int)c + 64 ? 2 : t.cnt > (int)c ? 1 : 0;
        for (int kk = k0; kk < k1; kk++) {
          if (!full()) break;
          uint32_t u[2][32];
          const uint32_t d = base + b.s * cols + c, du = d + up_offset;
          const float* s = products[b.s] + c;
          if (chunks > 0) tmem_ld32(d, u[0]);
          if (SWIGLU && chunks == 1) tmem_ld32(du, u[1]);
          if (chunks == 2) tmem_ld32(d + 64, u[1]);
          tmem_wait_ld();
          if (!SWIGLU || chunks < 2) release();
          if (chunks > 0) {
            waited(u[0]);
            add32(a.v, u[0], s);
          }
          if (SWIGLU && chunks == 1) {
            waited(u[1]);
            add32(a.v + 32, u[1], s + 128);
          }
          if (chunks == 2) {
            if (SWIGLU) tmem_ld32(du, u[0]);
            waited(u[1]);
            add32(a.v + 16, u[1], s + 64);
            if (SWIGLU) {
              tmem_ld32(du + 64, u[1]);
              tmem_wait_ld();
              release();
              waited(u[0]);
              waited(u[1]);
              add32(a.v + 32, u[0], s + 128);
              add32(a.v + 48, u[1], s + 192);
            }
          }
          release_scales();
        }
      }
      if (!ok) break;
      if (!PAIR && ks > 1) {
        ok = red.template store<T>(p, a, t, me, abort);
      } else if (wide) {
        if constexpr (DIRECT)
          store_wide_swiglu<T>(p, a, t, me);
        else
          store_wide<SWIGLU, T>(p, a, t, me, stage);
      } else {
        store_narrow<SWIGLU, T>(p, a, t, me);
      }
      __syncwarp();
    }
  } else if (warp == kSchedWarp) {
    give_registers();
    if (lane == 0) {
      const int items = (plan.singles + plan.multi_tiles) * fitems;
      int s = first_done ? 1 : 0;
      uint32_t ph = 0;
      bool first = true, ok = true;
      for (int it = first_done ? it0 + it_step : it0; ok; it += it_step) {
        Tile v;
        v.expert = -1;
        v.row0 = v.cnt = v.ft = 0;
        int n = 1;
        if (it < items) {
          v = find_tile<Cut>(p, plan, it);
          if (PAIR && SWIGLU && v.cnt > kNarrow) {
            // both feature tiles, one after the other, each by the whole pair
            v.ft *= 2;
            n = min(2, p.ftiles - v.ft);
          } else if (PAIR) {
            v.ft = 2 * v.ft + rank;
          }
        }
        for (int i = 0; i < n; i++) {
          if (!first && !mbar_wait(&bars.tile_empty[s], ph ^ 1, abort)) { ok = false; break; }
          bars.tile[s] = make_int4(v.expert, v.row0, v.cnt, v.ft + i);
          mbar_arrive(&bars.tile_full[s]);
          if (++s == kTileRing) {
            s = 0;
            ph ^= 1;
            first = false;
          }
        }
        if (it >= items) break;
      }
    }
    __syncwarp();
    cluster_wait();
  } else {
    give_registers();
    Ring r;
    bool first = true;
    while (tiles.next(bars, t, abort))
      if (!multiply_scales<SWIGLU>(p, t, PAIR && t.cnt > kNarrow, rank, k0, k1, bars, raw, products,
                                   r, first, bufs, abort))
        break;
    cp_async_wait_all();
    cluster_wait();
  }
  __syncwarp();
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

// e4m3 rows [rows x k bytes] as a 2D tensor; one box = box_rows x 128 bytes (one
// block of k), 128-byte swizzle. Bytes past a row and rows past the end read 0.
bool encode_codes(CUtensorMap* m, const void* base, int64_t rows, int k, int box_rows) {
  wb::TensorMapEncodeFn fn = wb::tensor_map_encoder();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)k};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// grid CTAs in clusters of `cluster`.
template <typename T, bool SWIGLU, bool PAIR, bool DIRECT>
WispError launch_kernel(const Params& p, int dev, unsigned grid, int cluster, cudaStream_t stream,
                        WispErrCtx* err) {
  const int smem = kRingBytes + 1024;
  auto kernel = fp8_product_kernel<T, SWIGLU, PAIR, DIRECT>;
  static std::atomic<uint64_t> raised{0};
  WB_CUDA_CHECK(wb::raise_smem(kernel, smem, dev, raised));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
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

template <typename T, bool PAIR>
WispError launch_typed(bool swiglu, const Params& p, int dev, unsigned grid, int cluster,
                       cudaStream_t stream, WispErrCtx* err) {
  if constexpr (PAIR) {
    if (swiglu && p.wide_out && p.cap > kNarrow)
      return launch_kernel<T, true, true, true>(p, dev, grid, cluster, stream, err);
  }
  return swiglu ? launch_kernel<T, true, PAIR, false>(p, dev, grid, cluster, stream, err)
                : launch_kernel<T, false, PAIR, false>(p, dev, grid, cluster, stream, err);
}

template <bool PAIR>
WispError launch_product(const WispFp8Config* c, const Params& p, int dev, unsigned grid,
                         int cluster, cudaStream_t stream, WispErrCtx* err) {
  if (c->out_type == WISP_DT_F32)
    return launch_typed<float, PAIR>(c->swiglu, p, dev, grid, cluster, stream, err);
  if (c->out_type == WISP_DT_BF16)
    return launch_typed<__nv_bfloat16, PAIR>(c->swiglu, p, dev, grid, cluster, stream, err);
  return launch_typed<__half, PAIR>(c->swiglu, p, dev, grid, cluster, stream, err);
}

// Clusters of `size` single CTAs that run at once on device dev. (Asked once per device
// and size; the kernel's forms all take the same registers and shared memory.)
WispError cluster_room(int dev, int size, int* room, WispErrCtx* err) {
  static std::atomic<int> known[64][9];
  const bool keep = dev >= 0 && dev < 64;
  if (keep && (*room = known[dev][size].load(std::memory_order_relaxed)) > 0) return WISP_OK;
  auto kernel = fp8_product_kernel<__nv_bfloat16, false, false, false>;
  const int smem = kRingBytes + 1024;
  static std::atomic<uint64_t> raised{0};
  WB_CUDA_CHECK(wb::raise_smem(kernel, smem, dev, raised));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  WB_CUDA_CHECK(cudaOccupancyMaxActiveClusters(room, kernel, &cfg));
  if (keep) known[dev][size].store(*room, std::memory_order_relaxed);
  return WISP_OK;
}

}  // namespace

extern "C" WispError wisp_b200_fp8_product(const WispFp8Config* cfg, const WispFp8Mats* w,
                                           const WispFp8Mats* up, const WispFp8Rows* x,
                                           const WispSegment* d_segs, int n_segs, void* d_out,
                                           int64_t ld, int* d_error_flag, cudaStream_t stream,
                                           WispErrCtx* err) {
  WispError e = wb::fp8_validate(cfg, "fp8_product", err);
  if (e != WISP_OK) return e;
  if ((e = wb::fp8_check_mats(w, "fp8_product", "weights", err)) != WISP_OK) return e;
  if (cfg->swiglu && (e = wb::fp8_check_mats(up, "fp8_product", "up weights", err)) != WISP_OK)
    return e;
  if (!cfg->swiglu && up)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_product: up weights without swiglu");
  if (!x || x->rows < 0 || x->rows > wb::kMaxRows)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_product: bad rows (0 .. 2^31 - 256)");
  if (d_segs ? (n_segs < 0 || n_segs > kMaxSegs) : n_segs != 0)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_product: n_segs=%d (0..%d, 0 without segments)",
                   n_segs, kMaxSegs);
  if (ld < cfg->n)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_product: ld=%lld < n=%d", (long long)ld, cfg->n);
  if (x->rows == 0 || (d_segs && n_segs == 0)) return WISP_OK;
  if (!x->codes || !x->scales || !d_out)
    return WB_FAIL(WISP_ERR_INVALID_ARG, "fp8_product: null pointer argument (rows, out)");
  if (((uintptr_t)x->codes & 15) || ((uintptr_t)x->scales & 3) ||
      ((uintptr_t)d_out % dt_size(cfg->out_type)) || ((uintptr_t)d_segs & 3) ||
      ((uintptr_t)d_error_flag & 3))
    return WB_FAIL(WISP_ERR_INVALID_ARG,
                   "fp8_product: row codes must be 16-byte aligned, segments and error word 4-byte, "
                   "scales and out to their types");
  int dev = 0, sms = 0;
  WB_CUDA_CHECK(wb::device_sms(&dev, &sms));
  auto tiles_of = [&](int rows_per_tile) {     // an upper bound: at most one per row, and
    // per segment one more than its rows fill
    const int64_t most = (int64_t)x->rows / rows_per_tile + (d_segs ? n_segs : 1);
    return most < x->rows ? most : x->rows;
  };
  const int ftiles = (cfg->n + 127) / 128, nk = (cfg->k + 127) / 128;
  const int64_t items = tiles_of(kSplitRows) * ftiles;
  // Few tiles: clusters of up to 8 CTAs split K, the largest that all run at once (one CTA
  // an SM; a GPC's SMs past the last whole cluster hold none: 74, 45, 33, 26, 22, 15 and 15
  // clusters of 2 to 8) with at least four blocks each. One row, us, as pairs / split:
  // 7168 x 7168 21.1 / 14.2 (by two); by half as many or fewer / so: 2048 x 7168 10.2 / 9.5
  // (six), 4096 x 7168 14.0 / 10.7 (four), 7168 x 2048 10.1 / 8.8 (two). 100 rows as pairs / as
  // tiles of 64: 256 x 7168 23.7 / 12.8, 2048 x 7168 24.1 / 14.9, gate/up 1536 x 2048 15.9 /
  // 13.8; 3000 rows of 128 x 7168 23.9 / 19.0. From 16 blocks on: of 8 to 15 one row gains
  // and 32 to 128 lose, whose join costs more than the blocks (n 2048, one row / 64 / 128, as
  // it is 7.3 / 8.1 / 9.3 with k 1024, 9.5 / 10.4 / 11.5 with k 1920; by two or three 7.2 / 10.1 /
  // 11.3, 7.8 / 11.2 / 12.6). (Where many segments make the bound on tiles
  // too large it may be too few: 8 of 512 x 2048 with 64 rows 11.0 as pairs, 11.8 by two.)
  int split = 1;
  if (nk >= 16) {
    for (int k = 8; k > 1 && split == 1; k--) {
      int room = 0;
      if (nk >= 4 * k && items * k <= sms) {
        if ((e = cluster_room(dev, k, &room, err)) != WISP_OK) return e;
        if (items <= room) split = k;
      }
    }
  }
  // With one feature tile a pair's second CTA would have none: single CTAs.
  const bool single = split == 1 && ftiles == 1;
  int cap = split > 1 ? kSplitRows : single ? kNarrow : kWide;
  if (split == 1) {
    // Smaller tiles when the largest would leave SMs without work: as many rows
    // as give every CTA one tile if the rows lay in one segment, at least 64.
    const int64_t width = single ? 1 : (ftiles + 1) / 2 * 2;
    const int64_t per = ((int64_t)x->rows * width + sms - 1) / sms;
    if (per <= kNarrow) cap = per < 64 ? 64 : (int)((per + 31) & ~31);
  }
  Params p;
  memset(&p, 0, sizeof p);
  p.cap = cap;
  const int64_t wrows = (int64_t)cfg->n_entries * cfg->n;
  if (!encode_codes(&p.tm_w, w->codes, wrows, cfg->k, 128) ||
      (cfg->swiglu && !encode_codes(&p.tm_up, up->codes, wrows, cfg->k, 128)) ||
      !encode_codes(&p.tm_x, x->codes, x->rows, cfg->k, 16) ||
      (cap > kNarrow && !encode_codes(&p.tm_x128, x->codes, x->rows, cfg->k, 128)))
    return WB_FAIL(WISP_ERR_CUDA, "fp8_product: cuTensorMapEncodeTiled failed");
  p.ws_w = w->scales;
  p.ws_up = cfg->swiglu ? up->scales : nullptr;
  p.xs = x->scales;
  p.xs_row = x->scale_row;
  p.xs_block = x->scale_block;
  p.rows = x->rows;
  p.segs = d_segs;
  p.nseg = n_segs;
  p.V = cfg->n_entries;
  p.N = cfg->n;
  p.nk = nk;
  p.ftiles = ftiles;
  p.out = d_out;
  p.ld = ld;
  p.wide_out = !((uintptr_t)d_out & 31) && ld * dt_size(cfg->out_type) % 32 == 0;
  p.even_out = !((uintptr_t)d_out & 3) && ld * dt_size(cfg->out_type) % 4 == 0;
  p.error_flag = d_error_flag;
  if (split > 1)
    return launch_product<false>(cfg, p, dev, (unsigned)(items * split), split, stream, err);
  if (single) {
    const int64_t want = tiles_of(cap);
    return launch_product<false>(cfg, p, dev, (unsigned)(want < sms ? want : sms), 1,
                                 stream, err);
  }
  const int64_t want = tiles_of(cap) * ((ftiles + 1) / 2) * 2;
  return launch_product<true>(cfg, p, dev,
                              (unsigned)(want < (sms & ~1) ? want : sms & ~1), 2, stream, err);
}
