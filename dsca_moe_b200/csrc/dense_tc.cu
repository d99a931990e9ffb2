// The products of dense.cuh on the tensor cores: CTA pairs, tcgen05 cta_group::2, TMA-fed.
//
// A tile is 256 rows of one operand (the MMA's A, 128 a CTA) by up to 256 of the other (its B, half a CTA), so an
// SM streams 32 KB for every 64-wide slice of k in 16 bits (128-wide in 8); the even CTA issues the MMAs into both
// CTAs' tensor memory.  Two orientations:
//   rows      A is the operand of the output's rows (tokens; rows of a weight's gradient): TMEM lane = row,
//             columns = consecutive values of that row, which a thread stores as they lie.
//   columns   A is the weight, B the tokens: a tile of 20 tokens costs 32 columns, not 256 rows; the epilogue turns
//             32 x 32 blocks in shared memory.  For up to 128 rows of output, and for rows off 16-byte boundaries, whose
//             single values it stores side by side.
//   warp 0      TMA producer, 128-byte swizzle, three stages of two 128-byte k boxes
//   warp 1      TMEM (512 columns: two accumulators); in the even CTA the MMA issuer
//   warps 4-11  epilogue: two warps to a lane quarter, alternate chunks of 32 TMEM columns
// Operands: a K-major one is loaded as boxes of 128 bytes of k by its rows; an MN-major one as boxes of 64
// rows of k by 64 values of m or n, which the MMA reads transposed, so that the gradients' products take
// weights and activations as they lie.
//
// Gated products (kGlu).  Rows: the even CTA loads the gate rows of B and the odd one the up rows of the same
// channels, so that each thread finds a token's gate and up values in its own lane, half a tile apart.  Columns: a
// CTA's 128 rows of A are 64 gate rows and the up rows of the same channels; the warps of lane quarters q and
// q + 2 hold the two, and for each chunk of 32 tokens the gate warp forms the products of the first 16 and the up
// warp those of the last, after handing each other the other half through shared memory.
// Saved for the backward pass in 16 bits: g and u as fp16 with one power of two for a token's 32 channels (11 bits of
// significand for every value within 2^29 of the largest), half of fp32's bytes, which the backward pass reads
// against the clock of its first product.
//
// 32-bit inputs (kF32): every value is split into three bf16 terms (8 + 8 + 8 bits, dense_split.cu); a stage holds the
// three planes of both operands' slice of k (72 KB, two stages), and six products are taken of them: hi.hi into one
// accumulator, hi.mid, mid.hi, hi.lo, mid.mid and lo.hi into another.  What is left out is 2^-24 of the product's
// terms.  The tensor cores' fp32 additions truncate, half a step of the running sum each, always towards zero: chains
// over all of k = 1408 were off by 4e-6.  So every 256 of k the epilogue warps take the sums into registers and
// add them there, rounding to nearest.
//
// Long k with few tiles: the k boxes are split over several pairs, each stores its fp32 tile to the workspace,
// and for every warp's part the last one to arrive adds the parts in the order of k: the result does not
// depend on who is last.
//
// Bound by the tensor pipe where tiles are many: 4096 x 2048 x 5632 bf16, pipe active 84 % (gate and up, 120 us, 1575
// TFLOP/s), 87 % (down, 69 us), 62 % (first backward product, 86 us, beside 220 MB of g, u and their gradients) and 94 %
// (the other gradients, 300 us) of the cycles; 8-bit 71 to 73 %.  Under the power cap the clock gives way: loops of the
// forward pass hold 1288 TFLOP/s at 1365 MHz.  Small products are bound by their 6 us of set-up, first loads and last
// epilogue; fp32 by six MMAs for one.
//
// Every wait is bounded (2 s); on a timeout the kernel records DSCA_ERR_WAIT_TIMEOUT, drains what it can
// observe, waits a grace period for copies into the pair, frees TMEM and returns.
#include "dense.cuh"

#include <algorithm>
#include <type_traits>

namespace dsca {
namespace dense {
namespace tc {

constexpr int kMaxStages = 3;
constexpr int kBoxBytes = 128 * 128;             // A's part of one k box (slice of k); B's, but for kF32
constexpr int kRingBytes = 12 * kBoxBytes;       // all stages
constexpr int kEpiWarps = 8;
constexpr int kFirstEpi = 4;                       // warps 0 producer, 1 MMA issuer, 2 and 3 idle
constexpr int kThreads = 32 * (kFirstEpi + kEpiWarps);
// Registers a thread after the set-up: the launch's 168 x 384 are dealt out anew (168 would spill what an epilogue has
// on its way from memory, which waits for it there).
constexpr int kRegsFew = 56, kRegsEpi = 224;
static_assert(128 * kRegsFew + 32 * kEpiWarps * kRegsEpi <= 168 * kThreads, "registers of the launch");
constexpr int kStgBytes = 2 * 32 * 32 * 2;       // per epilogue warp: two 32 x 32 blocks of bf16
constexpr int kSmemBytes = kRingBytes + kEpiWarps * kStgBytes + 1024;
static_assert(kSmemBytes <= 227 * 1024, "shared memory of a CTA");

enum In { kBf16 = 0, kI8 = 1, kF32 = 2 };

// A stage's layout by the inputs: two boxes of A and two of B; kF32: one slice, three planes of A and of B (whose
// tiles have at most 128 rows, half a box).
template <int IN>
struct Ring {
  static constexpr bool F = IN == kF32;
  static constexpr int kSub = F ? 1 : 2;     // slices of a stage
  static constexpr int kPlanes = F ? 3 : 1;
  static constexpr int kStages = F ? 2 : 3;
  static constexpr int kBBytes = F ? kBoxBytes / 2 : kBoxBytes;
  static constexpr int kB = kSub * kPlanes * kBoxBytes;                  // offset of B in a stage
  static constexpr int kStageBytes = kB + kSub * kPlanes * kBBytes;
  static constexpr int kChunk = 4;           // kF32: slices between two takings of the sums
  static_assert(kStages * kStageBytes <= kRingBytes && kStages <= kMaxStages, "ring");
};

struct Prob {
  int rows, cols, K;     // of the output [rows, cols]
  int row;               // orientation: rows (1) or columns (0)
  int nseg, kb;          // segments; k boxes of each
  int boxes;             // nseg * kb
  int a_mn, b_mn;        // majors of the MMA's A and B
  int tiles_m, tiles_n, tn;
  int splits, per;       // k splits and boxes of each
  int first;             // the problem's first unit of work
  int a_plane, b_plane;  // kF32: rows between the planes of three terms
  int vec;               // output rows start on 16-byte (1) or 32-byte (2) boundaries
  int64_t part;          // splits > 1: offset of the partial tiles in floats
  int counter;           // ... and of the arrival counters
  void* out;
  int64_t ldo;
};

struct Params {
  CUtensorMap a[kMaxProblems][2], b[kMaxProblems][2];
  Prob prob[kMaxProblems];
  int nprob, total, act;
  void* save_g;   // fp16 codes (16-bit inputs) or fp32
  void* save_u;
  uint8_t* save_e;  // fp16: the exponents, [2][rows][exp_groups(cols)]
  void* out2;
  const float* row_scale;  // CLOSE: row_max
  const float* col_scale[2];
  const void* bias;
  int vec_cols;  // col_scale on 16-byte boundaries
  float* parts;
  uint32_t* counters;
  int32_t* err;
};

struct Ctl {
  uint64_t full[kMaxStages], empty[kMaxStages], tmem_full[2], tmem_empty[2], mma_done;
  uint32_t tmem_base;
  int abort_flag;
  int pair_ok[2][kEpiWarps], pair_old[kEpiWarps];
};

struct Tile {
  int p, m0, n0, nval, box0, box1, split;  // first row of A, of B and how many of B (kGlu rows: of channels)
  int64_t tile;                            // within the problem
};

__device__ __forceinline__ Tile decode(const Params& P, int unit, int am, int bn) {
  Tile t;
  t.p = 0;
  while (t.p + 1 < P.nprob && unit >= P.prob[t.p + 1].first) ++t.p;
  const Prob& q = P.prob[t.p];
  int l = unit - q.first;
  t.split = l % q.splits;
  l /= q.splits;
  t.tile = l;
  // groups of eight m tiles, n by n inside: the pairs that run at one time share both operands' rows in L2
  const int g = l / (8 * q.tiles_n), r = l - g * 8 * q.tiles_n;
  const int gm = min(8, q.tiles_m - 8 * g);
  t.m0 = (8 * g + r % gm) * (q.row ? 256 : am);
  const int step = q.row ? q.tn / bn : q.tn;
  t.n0 = (r / gm) * step;
  t.nval = min(step, (q.row ? q.cols : q.rows) - t.n0);
  t.box0 = t.split * q.per;
  t.box1 = min(q.boxes, t.box0 + q.per);
  return t;
}

// MMA N of a tile: each CTA holds half of B's rows, whole 8-row groups (64 rows if MN-major); the rows form of a
// gated product always takes the whole tile.  A pair's 8-bit MMAs of 256 rows have N in steps of 32, its 16-bit ones of
// 16; every tile's width (and with it the boxes that land) is a multiple of 32, so the rounded N stays inside it.
template <int IN>
__host__ __device__ __forceinline__ int mma_n(const Prob& q, int nval, bool glu) {
  constexpr int kStep = IN == kI8 ? 32 : 16;
  if (glu && q.row) return q.tn;
  return q.b_mn ? (nval + 127) & ~127 : (nval + kStep - 1) & ~(kStep - 1);
}

__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - t0 > kWaitLimitNs) return;
}

// MN-major tile written by TMA with 128-byte swizzle: 64 values of m or n a row, rows of k; 8 KB to the next
// 64 values, 1 KB to the next eight rows of k.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)(8192 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// The producer and the MMA issuer are whole warps, of which one lane (`one`, a predicate in the instruction and no
// branch) issues: their loops stay uniform over the warp, so that addresses, coordinates and descriptors are computed
// in uniform registers, where these instructions take them.  Loops of a single lane moved every operand there by
// itself, an MMA took 160 to 190 cycles to issue and 128 to run.
__device__ __forceinline__ void umma_pair(uint32_t one, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t one, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void commit_both(uint32_t one, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
      "h"((unsigned short)3), "r"(one)
      : "memory");
}
__device__ __forceinline__ void load_pair(uint32_t one, uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster, int32_t c0,
                                          int32_t c1) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(c0), "r"(c1), "r"(one)
      : "memory");
}
__device__ __forceinline__ void expect_tx(uint32_t one, uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes), "r"(one)
      : "memory");
}
// mbar_wait() with one verdict for the warp
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* err) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err)) != 0;
}

// Where box b of a problem lies: slice k of a segment.
struct BoxAt {
  int seg, k;
  __device__ __forceinline__ BoxAt(const Prob& q, int b) : seg(b >= q.kb ? 1 : 0), k(b - seg * q.kb) {}
  __device__ __forceinline__ void next(int kb) {
    if (++k == kb) {
      k = 0;
      ++seg;
    }
  }
};

// The two warps (64 threads) that exchange gate and up values.
__device__ __forceinline__ void pair_barrier(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.4028234663852886e38f ? a : 0.0f;
}

// h = act(g) u, in place of g; dg = dh u act'(g) and du = dh act(g), in place of g and u.  One loop for each gate, so
// that the choice is made once.
template <bool kFast, int N>
__device__ __forceinline__ void gate_all(float (&g)[N], const float (&u)[N], int act) {
  if (act == DSCA_GATE_SILU) {
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] = gate<kFast>(g[j], DSCA_GATE_SILU) * u[j];
  } else if (act == DSCA_GATE_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] = gate<kFast>(g[j], DSCA_GATE_RELU) * u[j];
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] = gate<kFast>(g[j], DSCA_GATE_GELU) * u[j];
  }
}
template <bool kFast, int ACT, int N>
__device__ __forceinline__ void gate_grad_loop(const float (&dh)[N], float (&g)[N], float (&u)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float a, da;
    gate_grad<kFast>(g[j], ACT, &a, &da);
    g[j] = dh[j] * u[j] * da;
    u[j] = dh[j] * a;
  }
}
template <bool kFast, int N>
__device__ __forceinline__ void gate_grad_all(const float (&dh)[N], float (&g)[N], float (&u)[N], int act) {
  if (act == DSCA_GATE_SILU) gate_grad_loop<kFast, DSCA_GATE_SILU>(dh, g, u);
  else if (act == DSCA_GATE_RELU) gate_grad_loop<kFast, DSCA_GATE_RELU>(dh, g, u);
  else gate_grad_loop<kFast, DSCA_GATE_GELU>(dh, g, u);
}

// ---- rows form: 32 consecutive values of one output row from column n on.  vec: rows start on 16-byte (1) or
// 32-byte (2) boundaries; a whole 32-byte sector a store where they do, half a sector costs L2 twice the writes.
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
template <typename O>
__device__ __forceinline__ void store_row(O* row, int n, int cols, int vec, const float (&v)[32]) {
  constexpr int PER = 32 / sizeof(O);  // values of 32 bytes
#pragma unroll
  for (int i = 0; i < 32 / PER; ++i) {
    const int at = n + i * PER;
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (sizeof(O) == 2) w[k] = pack_bf16x2(v[i * PER + 2 * k], v[i * PER + 2 * k + 1]);
      else w[k] = __float_as_uint(v[i * PER + k]);
    }
    if (vec == 2 && at + PER <= cols) {
      store32(row + at, w);
    } else if (vec && at + PER <= cols) {
      *reinterpret_cast<uint4*>(row + at) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(row + at + PER / 2) = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (at + k < cols) {
          if constexpr (sizeof(O) == 2) row[at + k] = __float2bfloat16_rn(v[i * PER + k]);
          else row[at + k] = v[i * PER + k];
        }
    }
  }
}
// 32 floats from column n on (zeros past cols); the same for every lane or a row of its own
__device__ __forceinline__ void load_row(const float* row, int n, int cols, bool vec, float (&v)[32]) {
  if (vec && n + 32 <= cols) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(row + n + 4 * i));
      v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = n + j < cols ? __ldg(row + n + j) : 0.0f;
}
// Saved rows start on 16-byte boundaries and hold a multiple of eight values (ld_h), so pieces of eight are whole.
__device__ __forceinline__ void save_row_f16(const Params& P, const Prob& q, int up, int64_t row, int n, const float (&v)[32]) {
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < 32; ++j) m = fmaxf(m, finite_abs(v[j]));
  const uint32_t e = f16_exp(m);
  const float s = f16_factor(e);
  __half* at = reinterpret_cast<__half*>(up ? P.save_u : P.save_g) + row * q.ldo + n;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const __half2 h2 = __floats2half2_rn(v[16 * i + 2 * k] * s, v[16 * i + 2 * k + 1] * s);
      w[k] = *reinterpret_cast<const uint32_t*>(&h2);
    }
    if (q.vec == 2 && n + 16 * i + 16 <= q.cols) {
      store32(at + 16 * i, w);
    } else {
      if (n + 16 * i < q.cols) *reinterpret_cast<uint4*>(at + 16 * i) = make_uint4(w[0], w[1], w[2], w[3]);
      if (n + 16 * i + 8 < q.cols) *reinterpret_cast<uint4*>(at + 16 * i + 8) = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  *reinterpret_cast<uint32_t*>(P.save_e + ((int64_t)up * q.rows + row) * exp_groups(q.cols) + n / 8) = e * 0x01010101u;
}
// g and u of a chunk, loaded while the one before it is in work: 32 bytes a load where rows start on such boundaries.
// Every lane has a row of its own, and what these loads and the stores leave in L1 only pushes one another out: without
// it 4096 x 2048 x 5632's first backward product takes 86 us instead of 103.
__device__ __forceinline__ void load32(const void* p, uint32_t* w) {
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
struct Ahead {
  uint32_t v[2][16];
  uint32_t e[2];
  __device__ __forceinline__ void load(const Params& P, const Prob& q, int64_t row, int n, int nend) {
    const bool live = row < q.rows && n < nend;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half* p = reinterpret_cast<const __half*>(i == 0 ? P.save_g : P.save_u) + row * q.ldo + n;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!live || n + 16 * h >= q.cols) {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[i][8 * h + k] = 0u;
        } else if (q.vec == 2) {
          load32(p + 16 * h, v[i] + 8 * h);
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint4 x = n + 16 * h + 8 * k < q.cols ? __ldg(reinterpret_cast<const uint4*>(p + 16 * h + 8 * k))
                                                        : make_uint4(0u, 0u, 0u, 0u);
            v[i][8 * h + 4 * k] = x.x; v[i][8 * h + 4 * k + 1] = x.y;
            v[i][8 * h + 4 * k + 2] = x.z; v[i][8 * h + 4 * k + 3] = x.w;
          }
        }
      }
      e[i] = live ? *reinterpret_cast<const uint32_t*>(P.save_e + ((int64_t)i * q.rows + row) * exp_groups(q.cols) + n / 8) : 0u;
    }
  }
  __device__ __forceinline__ void get(int i, float (&o)[32]) const {
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float s = f16_back(e[i] >> (8 * (k / 4)) & 255u);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[i][k]));
      o[2 * k] = f.x * s;
      o[2 * k + 1] = f.y * s;
    }
  }
};

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
}

// CLOSE: gated 8-bit products by close_h.
template <int EPI, int IN, typename O, bool CLOSE = false>
__global__ void __launch_bounds__(kThreads, 1) dense_kernel(const __grid_constant__ Params P) {
  constexpr bool kGluE = EPI == kGlu;
  using R = Ring<IN>;
  constexpr int kSub = R::kSub, kStages = R::kStages, kStageBytes = R::kStageBytes;
  constexpr int kAM = kGluE ? 128 : 256;     // channels or columns of a tile in the columns form
  constexpr int kBN = kGluE ? 2 : 1;         // rows of B to a channel in the rows form
  constexpr int KE = IN == kI8 ? 128 : 64;   // k elements of a box
  constexpr int KS = IN == kI8 ? 32 : 16;    // ... and of one MMA
  constexpr bool kFast = IN != kF32;
  constexpr bool kBigI8 = EPI == kStore && sizeof(O) == 4;  // order of an 8-bit sum's scales
  static_assert(!CLOSE || (kGluE && IN == kI8), "gated 8-bit products");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ Ctl ctl;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_a = smem_u32(smem), smem_b = smem_a + R::kB;  // of stage 0
  const int warp = __shfl_sync(0xffffffffu, warp_id(), 0), lane = lane_id();  // uniform for the compiler too
  const uint32_t one = lane == 0;
  volatile int* abort_flag = &ctl.abort_flag;
  const uint32_t rank = cluster_ctarank();
  const int unit0 = (int)(blockIdx.x >> 1), units = (int)(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&ctl.full[s]), 1);
      mbar_init(smem_u32(&ctl.empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctl.tmem_full[i]), 1);
      mbar_init(smem_u32(&ctl.tmem_empty[i]), 2 * kEpiWarps);
    }
    mbar_init(smem_u32(&ctl.mma_done), 1);
    ctl.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0)
    for (int i = 0; i < P.nprob; ++i) {
      prefetch_tmap(&P.a[i][0]);
      prefetch_tmap(&P.b[i][0]);
    }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&ctl.tmem_base), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before any signal between them
  tc_fence_after();
  const uint32_t tmem_base = ctl.tmem_base;
  pdl_launch_dependents();
  pdl_wait();  // the launch before this one (when it is its programmatic dependent) has written its results

  if (warp < kFirstEpi) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
    if (warp == 0) {
      // ---------------- TMA producer
      const uint32_t full0 = smem_u32(&ctl.full[0]), empty0 = smem_u32(&ctl.empty[0]), full0_even = mapa_shared(full0, 0);
      const uint32_t even = rank == 0;
      int s = 0;
      uint32_t ph = 0;
      uint32_t armed = 0, parity = 0;  // stages with copies under way since, and the phase of each
      bool ok = true;
      for (int unit = unit0; ok && unit < P.total; unit += units) {
        const Tile t = decode(P, unit, kAM, kBN);
        const Prob& q = P.prob[t.p];
        const bool glu_rows = kGluE && q.row;
        const int b_row = glu_rows ? t.n0 : t.n0 + mma_n<IN>(q, t.nval, kGluE) / 2 * (int)rank;
        const int a_row = kGluE && !q.row ? t.m0 + 64 * (int)rank : t.m0 + 128 * (int)rank;
        const uint32_t b_bytes = (uint32_t)(q.tn / 2) * 128u;  // a whole box lands; rows past the tile are not used
        const int kb = q.kb, a_mn = q.a_mn, b_atoms = q.b_mn ? q.tn / 128 : 0, a_plane = q.a_plane, b_plane = q.b_plane;
        const CUtensorMap *ma = P.a[t.p], *mb = glu_rows ? P.b[t.p] + rank : P.b[t.p];
        BoxAt at(q, t.box0);
        for (int b = t.box0; b < t.box1; b += kSub) {
          if (!wait_warp(empty0 + 8 * s, ph ^ 1u, abort_flag, P.err)) { ok = false; break; }
          const uint32_t fb0 = full0_even + 8 * s;
          const int nb = min(kSub, t.box1 - b);
          expect_tx(one & even, full0 + 8 * s, 2u * (uint32_t)(nb * R::kPlanes) * ((uint32_t)kBoxBytes + b_bytes));
          for (int h = 0; h < nb; ++h, at.next(kb)) {
            const int kx = at.k * KE;
#pragma unroll
            for (int pl = 0; pl < R::kPlanes; ++pl) {
              const uint32_t da = smem_a + s * kStageBytes + (h + pl) * kBoxBytes, db = smem_b + s * kStageBytes + (h + pl) * R::kBBytes;
              const int pa = pl * a_plane, pb = pl * b_plane;
              if (kGluE && !glu_rows) {
                load_pair(one, da, ma, fb0, kx, a_row + pa);
                load_pair(one, da + 8192, ma + 1, fb0, kx, a_row + pa);
              } else if (a_mn) {
                load_pair(one, da, ma + at.seg, fb0, a_row, kx + pa);
                load_pair(one, da + 8192, ma + at.seg, fb0, a_row + 64, kx + pa);
              } else {
                load_pair(one, da, ma + at.seg, fb0, kx, a_row + pa);
              }
              if (b_atoms) {
                load_pair(one, db, mb + at.seg, fb0, b_row, kx + pb);
                if (b_atoms > 1) load_pair(one, db + 8192, mb + at.seg, fb0, b_row + 64, kx + pb);
              } else {
                load_pair(one, db, mb + at.seg, fb0, kx, b_row + pb);
              }
            }
          }
          armed |= 1u << s;
          parity = (parity & ~(1u << s)) | ph << s;
          if (++s == kStages) { s = 0; ph ^= 1u; }
        }
      }
      if (!ok && rank == 0)
        for (int i = 0; i < kStages; ++i)
          if (armed >> i & 1u) drain(full0 + 8 * i, parity >> i & 1u);
    } else if (warp == 1) {
      // ---------------- MMA issuer (even CTA)
      if (rank == 0) {
        const uint32_t full0 = smem_u32(&ctl.full[0]), empty0 = smem_u32(&ctl.empty[0]);
        const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
        int s = 0, it = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int unit = unit0; ok && unit < P.total; unit += units) {
          const Tile t = decode(P, unit, kAM, kBN);
          const Prob& q = P.prob[t.p];
          // D f32 (1) or s32 (2); A, B bf16 (1) or signed 8-bit (1); majors; N; M = 256
          const uint32_t idesc = ((IN == kI8 ? 2u : 1u) << 4) | (1u << 7) | (1u << 10) | ((uint32_t)q.a_mn << 15) |
                                 ((uint32_t)q.b_mn << 16) | ((uint32_t)(mma_n<IN>(q, t.nval, kGluE) >> 3) << 17) | (16u << 24);
          // descriptors but for the stage, and their steps of one MMA (in 16 bytes: 2 KB or 32 bytes)
          const uint64_t ad0 = q.a_mn ? sw128_mnmajor_desc(smem_a) : sw128_kmajor_desc(smem_a);
          const uint64_t bd0 = q.b_mn ? sw128_mnmajor_desc(smem_b) : sw128_kmajor_desc(smem_b);
          const uint64_t astep = q.a_mn ? 128u : 2u, bstep = q.b_mn ? 128u : 2u;
          const int kb = q.kb, last_steps = (q.K - (kb - 1) * KE + KS - 1) / KS;
          BoxAt at(q, t.box0);
          // an accumulator takes the whole tile, kF32: a chunk of it
          for (int c0 = t.box0; ok && c0 < t.box1; ++it) {
            const int c1 = IN == kF32 ? min(t.box1, c0 + R::kChunk) : t.box1;
            const int acc = it & 1;
            if (!wait_warp(smem_u32(&ctl.tmem_empty[acc]), (uint32_t)(((it >> 1) & 1) ^ 1), abort_flag, P.err)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t d = tmem + (uint32_t)(acc * 256);
            uint32_t used = 0u;
            for (int b = c0; b < c1; b += kSub) {
              if (!wait_warp(full0 + 8 * s, ph, abort_flag, P.err)) { ok = false; break; }
              tc_fence_after();
              const int nb = min(kSub, c1 - b);
#pragma unroll
              for (int h = 0; h < kSub; ++h) {
                if (h < nb) {
                  const uint64_t ad = ad0 + (uint64_t)((s * kStageBytes + h * kBoxBytes) >> 4);
                  const uint64_t bd = bd0 + (uint64_t)((s * kStageBytes + h * R::kBBytes) >> 4);
                  const int steps = at.k == kb - 1 ? last_steps : 4;
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    if (i < steps) {
                      const uint64_t ai = ad + astep * i, bi = bd + bstep * i;
                      if constexpr (IN == kI8) {
                        umma_i8_pair(one, d, ai, bi, idesc, used);
                      } else {
                        umma_pair(one, d, ai, bi, idesc, used);
                        if constexpr (IN == kF32) {
                          constexpr uint64_t PA = kBoxBytes >> 4, PB = R::kBBytes >> 4;
                          umma_pair(one, d + 128u, ai, bi + PB, idesc, used);
                          umma_pair(one, d + 128u, ai + PA, bi, idesc, 1u);
                          umma_pair(one, d + 128u, ai, bi + 2 * PB, idesc, 1u);
                          umma_pair(one, d + 128u, ai + PA, bi + PB, idesc, 1u);
                          umma_pair(one, d + 128u, ai + 2 * PA, bi, idesc, 1u);
                        }
                      }
                      used = 1u;
                    }
                  at.next(kb);
                }
              }
              commit_both(one, empty0 + 8 * s);
              if (++s == kStages) { s = 0; ph ^= 1u; }
            }
            if (!ok) break;
            commit_both(one, smem_u32(&ctl.tmem_full[acc]));
            c0 = c1;
          }
        }
        if (!ok) {  // every MMA issued has completed before TMEM is freed
          if (lane == 0) umma_commit_pair(mapa_shared(smem_u32(&ctl.mma_done), 0));
          drain(smem_u32(&ctl.mma_done), 0);
        }
      }
    }
  } else {
    // ---------------- epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    const int q4 = warp & 3, ew = warp - kFirstEpi, eh = ew >> 2;
    uint8_t* stg = smem + kRingBytes + ew * kStgBytes;
    const int pair_id = 1 + (ew & 1) + 2 * eh;  // barrier of an exchange
    int it = 0, xb = 0, round = 0;
    Ahead ahead;
    for (int unit = unit0; unit < P.total; unit += units) {
      const Tile t = decode(P, unit, kAM, kBN);
      const Prob& q = P.prob[t.p];
      const int64_t lrow = t.m0 + 128 * (int)rank + 32 * q4 + lane;  // rows form: this lane's output row
      if constexpr (EPI == kDGlu && IN == kBf16)
        if (q.row) ahead.load(P, q, lrow, t.n0 + 32 * eh, t.n0 + t.nval);
      const int ncol = mma_n<IN>(q, t.nval, kGluE);
      uint32_t taddr = 0;
      float fs[2][32];  // kF32: the sums of this warp's two chunks of columns
      if constexpr (IN == kF32) {
#pragma unroll
        for (int j = 0; j < 32; ++j) fs[0][j] = fs[1][j] = 0.0f;
      }
      int w_ok = 1;
      for (int c0 = t.box0; c0 < t.box1; c0 += IN == kF32 ? R::kChunk : t.box1 - t.box0) {
        const int acc = it & 1;
        w_ok = 1;
        if (lane == 0) w_ok = mbar_wait(smem_u32(&ctl.tmem_full[acc]), (uint32_t)((it >> 1) & 1), abort_flag, P.err) ? 1 : 0;
        w_ok = __shfl_sync(0xffffffffu, w_ok, 0);
        if (!w_ok) break;
        tc_fence_after();
        taddr = tmem_base + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * 256);
        if constexpr (IN == kF32) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (32 * eh + 64 * h < ncol) {
              uint32_t v[32], w[32];
              tmem_ld32(taddr + 32 * eh + 64 * h, v);
              tmem_ld32(taddr + 128 + 32 * eh + 64 * h, w);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) fs[h][j] += __uint_as_float(v[j]) + __uint_as_float(w[j]);
            }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&ctl.tmem_empty[acc]), 0));
          ++it;
        }
      }
      if constexpr (kGluE) {
        // the two warps of an exchange go on or leave together (two verdicts in turn: a warp may give its next one
        // before the other has read this one)
        if (lane == 0) ctl.pair_ok[round & 1][ew] = w_ok;
        pair_barrier(pair_id);
        w_ok = *reinterpret_cast<volatile int*>(&ctl.pair_ok[round & 1][ew ^ 2]) & w_ok;
        ++round;
      }
      if (!w_ok) break;
      // 32 columns of the accumulator from c on
      auto chunk = [&](int c, uint32_t (&v)[32]) {
        if constexpr (IN == kF32) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(c >= 64 ? fs[1][j] : fs[0][j]);
        } else {
          tmem_ld32(taddr + c, v);
          tmem_wait_ld();
        }
      };
      bool mine = true;
      float* part = nullptr;  // [split][rank][column / 4][lane][4]
      const int tnp = (q.tn + 31) & ~31;  // whole chunks
      const int64_t part_step = (int64_t)2 * tnp * 128;
      if (q.splits > 1) {
        part = P.parts + q.part + t.tile * q.splits * part_step + (int64_t)rank * tnp * 128 + (q4 * 32 + lane) * 4;
        for (int c = 32 * eh; c < ncol; c += 64) {
          uint32_t v[32];
          chunk(c, v);
          float* at = part + t.split * part_step + (int64_t)c * 128;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(at + j * 512) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
        __threadfence();
        __syncwarp();
        uint32_t old = 0;
        uint32_t* counter = P.counters + q.counter + (t.tile * 2 + rank) * kEpiWarps + ew;
        if constexpr (kGluE) {
          // one count for the two warps of an exchange, which finish a tile together
          pair_barrier(pair_id);
          if (!(q4 >> 1) && lane == 0) {
            __threadfence();
            ctl.pair_old[ew] = (int)atomicAdd(counter, 1u);
          }
          pair_barrier(pair_id);
          old = (uint32_t)*reinterpret_cast<volatile int*>(&ctl.pair_old[ew & ~2]);  // the gate warps are 0, 1, 4, 5
        } else {
          if (lane == 0) old = atomicAdd(counter, 1u);
          old = __shfl_sync(0xffffffffu, old, 0);
        }
        mine = old == (uint32_t)q.splits - 1u;
        if (mine) __threadfence();
      }
      // the finished product's 32 columns from c on: parts in the order of k (8-bit: int32 sums)
      auto finished = [&](int c, uint32_t (&r)[32]) {
        if (q.splits == 1) {
          chunk(c, r);
          return;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = 0u;
#pragma unroll 2
        for (int s = 0; s < q.splits; ++s) {
          const float* at = part + s * part_step + (int64_t)c * 128;
          uint4 x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = __ldcg(reinterpret_cast<const uint4*>(at + j * 512));
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if constexpr (IN == kI8) r[4 * j + k] += w[k];
              else r[4 * j + k] = __float_as_uint(__uint_as_float(r[4 * j + k]) + __uint_as_float(w[k]));
            }
          }
        }
      };
      // sixteen columns, of 8-bit operands
      auto finished16 = [&](int c, uint32_t (&r)[16]) {
        if (q.splits == 1) {
          tmem_ld16(taddr + c, r);
          return;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = 0u;
        for (int s = 0; s < q.splits; ++s) {
          const float* at = part + s * part_step + (int64_t)c * 128;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 x = __ldcg(reinterpret_cast<const uint4*>(at + j * 512));
            r[4 * j] += x.x; r[4 * j + 1] += x.y; r[4 * j + 2] += x.z; r[4 * j + 3] += x.w;
          }
        }
      };
      if constexpr (CLOSE) {
        // ------------ 16 values of a row (rows) or of a column (columns) at a time, which keeps the code short
        if (mine && q.row) {
          const bool live = lrow < q.rows;
          const Two xs = scale_two(live ? __ldg(P.row_scale + lrow) : 0.0f);
          float* out = reinterpret_cast<float*>(q.out) + lrow * q.ldo;
#pragma unroll 1
          for (int c = 32 * eh; c < t.nval; c += c % 32 == 16 ? 48 : 16) {  // alternate chunks of 32
            const int n = t.n0 + c;
            uint32_t g[16], u[16];
            __syncwarp();
            finished16(c, g);
            finished16(c + q.tn / 2, u);
            float gs[16], us[16], h[16];
            Two x16[16];
            if (P.vec_cols && n + 16 <= q.cols) {
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                const float4 a = __ldg(reinterpret_cast<const float4*>(P.col_scale[0] + n + j));
                const float4 b = __ldg(reinterpret_cast<const float4*>(P.col_scale[1] + n + j));
                gs[j] = a.x; gs[j + 1] = a.y; gs[j + 2] = a.z; gs[j + 3] = a.w;
                us[j] = b.x; us[j + 1] = b.y; us[j + 2] = b.z; us[j + 3] = b.w;
              }
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const int at = min(n + j, q.cols - 1);
                gs[j] = __ldg(P.col_scale[0] + at);
                us[j] = __ldg(P.col_scale[1] + at);
              }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) x16[j] = xs;
            tmem_wait_ld();
            close_all(h, reinterpret_cast<const int(&)[16]>(g), reinterpret_cast<const int(&)[16]>(u), gs, us, x16, P.act);
            if (live) {
#pragma unroll
              for (int i = 0; i < 16; i += 8) {
                if (q.vec == 2 && n + i + 8 <= q.cols) {
                  uint32_t w[8];
#pragma unroll
                  for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(h[i + j]);
                  store32(out + n + i, w);
                } else {
#pragma unroll
                  for (int j = 0; j < 8; ++j)
                    if (n + i + j < q.cols) out[n + i + j] = h[i + j];
                }
              }
            }
          }
        } else if (mine) {
          const int ch = t.m0 + 64 * (int)rank + 32 * (q4 & 1) + lane, up = q4 >> 1;
          const bool in = ch < q.cols;
          const float gs = in ? __ldg(P.col_scale[0] + ch) : 0.0f, us = in ? __ldg(P.col_scale[1] + ch) : 0.0f;
          float gs16[16], us16[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) gs16[j] = gs, us16[j] = us;
#pragma unroll 1
          for (int c = 32 * eh; c < t.nval; c += 64) {
            uint32_t r[32];
            finished(c, r);
            const Two mine2 = scale_two(c + lane < t.nval ? __ldg(P.row_scale + t.n0 + c + lane) : 0.0f);  // of token c + lane
            // the gate warp forms the first 16 tokens, the up warp the others (two buffers: one barrier a chunk)
            uint32_t* mine_x = reinterpret_cast<uint32_t*>(stg) + xb * 512;
            const uint32_t* other_x = reinterpret_cast<const uint32_t*>(smem + kRingBytes + (ew ^ 2) * kStgBytes) + xb * 512;
            xb ^= 1;
#pragma unroll
            for (int j = 0; j < 16; ++j) mine_x[j * 32 + lane] = up ? r[j] : r[16 + j];
            pair_barrier(pair_id);
            int g[16], u[16];
            float h[16];
            Two xs[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const uint32_t got = other_x[j * 32 + lane];
              g[j] = (int)(up ? got : r[j]);
              u[j] = (int)(up ? r[16 + j] : got);
              xs[j] = {__shfl_sync(0xffffffffu, mine2.hi, 16 * up + j), __shfl_sync(0xffffffffu, mine2.lo, 16 * up + j)};
            }
            close_all(h, g, u, gs16, us16, xs, P.act);
            float* out = reinterpret_cast<float*>(q.out) + (int64_t)(t.n0 + c + 16 * up) * q.ldo + ch;
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (in && c + 16 * up + j < t.nval) out[j * q.ldo] = h[j];
          }
        }
      } else if (mine && q.row) {
        // ------------ rows: this lane's row, 32 of its values at a time
        const bool live = lrow < q.rows;
        O* out = reinterpret_cast<O*>(q.out) + lrow * q.ldo;
        float rs = 1.0f;
        if constexpr (IN == kI8) rs = live ? __ldg(P.row_scale + lrow) : 0.0f;
        const int span = kGluE ? q.tn / 2 : ncol;  // columns of the tile's output
#pragma unroll 1
        for (int c = 32 * eh; c < span; c += 64) {
          if (c >= t.nval) break;
          const int n = t.n0 + c;
          float v[32];
          {
            uint32_t r[32];
            finished(c, r);
            if constexpr (IN == kI8) {
              float cs[32];
              load_row(P.col_scale[0], n, q.cols, P.vec_cols, cs);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = scaled<kBigI8>((int)r[j], cs[j], rs);
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
            }
          }
          if constexpr (kGluE) {
            float u[32];
            {
              uint32_t r[32];
              finished(c + q.tn / 2, r);
              if constexpr (IN == kI8) {
                float cs[32];
                load_row(P.col_scale[1], n, q.cols, P.vec_cols, cs);
#pragma unroll
                for (int j = 0; j < 32; ++j) u[j] = scaled<kBigI8>((int)r[j], cs[j], rs);
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) u[j] = __uint_as_float(r[j]);
              }
            }
            if (P.save_g != nullptr && live) {
              if constexpr (IN == kBf16) {
                save_row_f16(P, q, 0, lrow, n, v);
                save_row_f16(P, q, 1, lrow, n, u);
              } else {
                store_row(reinterpret_cast<float*>(P.save_g) + lrow * q.ldo, n, q.cols, 1, v);
                store_row(reinterpret_cast<float*>(P.save_u) + lrow * q.ldo, n, q.cols, 1, u);
              }
            }
            gate_all<kFast>(v, u, P.act);
            if (live) store_row(out, n, q.cols, q.vec, v);
          } else if constexpr (EPI == kDGlu) {
            float g[32], u[32];
            if constexpr (IN == kBf16) {
              ahead.get(0, g);
              ahead.get(1, u);
              ahead.load(P, q, lrow, n + 64, t.n0 + t.nval);
            } else if (live) {
              load_row(reinterpret_cast<const float*>(P.save_g) + lrow * q.ldo, n, q.cols, true, g);
              load_row(reinterpret_cast<const float*>(P.save_u) + lrow * q.ldo, n, q.cols, true, u);
            }
            if (live) {
              gate_grad_all<kFast>(v, g, u, P.act);
              store_row(out, n, q.cols, q.vec, g);
              store_row(reinterpret_cast<O*>(P.out2) + lrow * q.ldo, n, q.cols, q.vec, u);
            }
          } else {
            if constexpr (IN == kI8) {
              if (P.bias != nullptr) {
                const O* b = reinterpret_cast<const O*>(P.bias);
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (n + j < q.cols) {
                    if constexpr (sizeof(O) == 2) v[j] += __bfloat162float(b[n + j]);
                    else v[j] += b[n + j];
                  }
              }
            }
            if (live) store_row(out, n, q.cols, q.vec, v);
          }
        }
      } else if (mine) {
        // ------------ columns: this lane's output column, 32 tokens at a time
        const int ch = kGluE ? t.m0 + 64 * (int)rank + 32 * (q4 & 1) + lane : (int)lrow;
        const int up = kGluE ? q4 >> 1 : 0;  // kGlu: a warp of gate or up values
        const bool whole = q.vec && (ch & ~31) + 32 <= q.cols;
        float cs = 1.0f, bias = 0.0f;
        if constexpr (IN == kI8) cs = ch < q.cols ? __ldg((up ? P.col_scale[1] : P.col_scale[0]) + ch) : 0.0f;
        if constexpr (EPI == kStore && IN == kI8) {
          if (P.bias != nullptr && ch < q.cols) {
            if constexpr (sizeof(O) == 2) bias = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(P.bias)[ch]);
            else bias = reinterpret_cast<const float*>(P.bias)[ch];
          }
        }
        // 32 or 16 tokens of the block o (lane = column) from token tok0 of the tile on, through `st`
        const int64_t ldo = q.ldo;
        const int cols = q.cols;
        auto put = [&](O* base, const auto& o, int tok0, __nv_bfloat16* st) {
          constexpr int N = sizeof(o) / sizeof(o[0]);
          const int left = t.nval - tok0;  // tokens
          if constexpr (sizeof(O) == 2) {
            if (whole) {
#pragma unroll
              for (int j = 0; j < N; ++j) st[j * 32 + lane] = __float2bfloat16_rn(o[j]);
              __syncwarp();
              O* at = base + (int64_t)(t.n0 + tok0 + (lane >> 2)) * ldo + (ch & ~31) + 8 * (lane & 3);
#pragma unroll
              for (int rr = 0; rr < N / 8; ++rr, at += 8 * ldo)
                if (rr * 8 + (lane >> 2) < left)
                  *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(st + (rr * 8 + (lane >> 2)) * 32 + 8 * (lane & 3));
              __syncwarp();
              return;
            }
          }
          if (ch < cols) {
            O* at = base + (int64_t)(t.n0 + tok0) * ldo + ch;
            auto one = [&](float x) {
              if constexpr (sizeof(O) == 2) *at = __float2bfloat16_rn(x);
              else *at = x;
              at += ldo;
            };
            if (left >= N) {
#pragma unroll
              for (int j = 0; j < N; ++j) one(o[j]);
            } else {
#pragma unroll
              for (int j = 0; j < N; ++j)
                if (j < left) one(o[j]);
            }
          }
        };
#pragma unroll 1
        for (int c = 32 * eh; c < ncol; c += 64) {
          if (c >= t.nval) break;
          float v[32];
          {
            uint32_t r[32];
            finished(c, r);
            if constexpr (IN == kI8) {
              const float rs = c + lane < t.nval ? __ldg(P.row_scale + t.n0 + c + lane) : 0.0f;
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = scaled<kBigI8>((int)r[j], cs, __shfl_sync(0xffffffffu, rs, j));
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
            }
          }
          const int64_t tok = t.n0 + c;
          if constexpr (kGluE) {
            if (P.save_g != nullptr) {
              if constexpr (IN == kBf16) {
                uint32_t el = 0;  // lane j's: the exponent of token j
                __half* at = reinterpret_cast<__half*>(up ? P.save_u : P.save_g) + tok * q.ldo + ch;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  const float a = ch < q.cols ? finite_abs(v[j]) : 0.0f;
                  const uint32_t e = f16_exp(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a))));
                  if (lane == j) el = e;
                  if (ch < q.cols && c + j < t.nval) at[j * q.ldo] = __float2half_rn(v[j] * f16_factor(e));
                }
                if (c + lane < t.nval && (ch & ~31) < q.cols)
                  *reinterpret_cast<uint32_t*>(P.save_e + ((int64_t)up * q.rows + tok + lane) * exp_groups(q.cols) +
                                               (ch & ~31) / 8) = el * 0x01010101u;
              } else if (ch < q.cols) {
                float* at = reinterpret_cast<float*>(up ? P.save_u : P.save_g) + tok * q.ldo + ch;
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (c + j < t.nval) at[j * q.ldo] = v[j];
              }
            }
            // two buffers, so that one barrier a chunk is enough
            float* mine_x = reinterpret_cast<float*>(stg) + xb * 512;
            float* other_x = reinterpret_cast<float*>(smem + kRingBytes + (ew ^ 2) * kStgBytes) + xb * 512;
            xb ^= 1;
#pragma unroll
            for (int j = 0; j < 16; ++j) mine_x[j * 32 + lane] = up ? v[j] : v[16 + j];
            pair_barrier(pair_id);
            float g[16], u[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float got = other_x[j * 32 + lane];
              g[j] = up ? got : v[j];
              u[j] = up ? v[16 + j] : got;
            }
            gate_all<kFast>(g, u, P.act);
            // staged where the other warp's values lay, which this warp alone reads
            __syncwarp();
            put(reinterpret_cast<O*>(q.out), g, c + 16 * up, reinterpret_cast<__nv_bfloat16*>(other_x));
          } else if constexpr (EPI == kDGlu) {
            float g[32], u[32];
            if constexpr (IN == kBf16) {
              uint32_t ex[2] = {0u, 0u};  // lane j's: the exponents of token j
              if (c + lane < t.nval && (ch & ~31) < q.cols) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                  ex[i] = *reinterpret_cast<const uint32_t*>(P.save_e + ((int64_t)i * q.rows + tok + lane) * exp_groups(q.cols) +
                                                             (ch & ~31) / 8);
              }
              const __half *pg = reinterpret_cast<const __half*>(P.save_g), *pu = reinterpret_cast<const __half*>(P.save_u);
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const bool in = ch < q.cols && c + j < t.nval;
                const int64_t at = (tok + j) * q.ldo + ch;
                g[j] = in ? __half2float(pg[at]) : 0.0f;
                u[j] = in ? __half2float(pu[at]) : 0.0f;
              }
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                // of this lane's eight channels
                g[j] *= f16_back(__shfl_sync(0xffffffffu, ex[0], j) >> (lane & 24) & 255u);
                u[j] *= f16_back(__shfl_sync(0xffffffffu, ex[1], j) >> (lane & 24) & 255u);
              }
            } else {
              const float *pg = reinterpret_cast<const float*>(P.save_g), *pu = reinterpret_cast<const float*>(P.save_u);
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const bool in = ch < q.cols && c + j < t.nval;
                const int64_t at = (tok + j) * q.ldo + ch;
                g[j] = in ? __ldg(pg + at) : 0.0f;
                u[j] = in ? __ldg(pu + at) : 0.0f;
              }
            }
            gate_grad_all<kFast>(v, g, u, P.act);
            put(reinterpret_cast<O*>(q.out), g, c, reinterpret_cast<__nv_bfloat16*>(stg));
            put(reinterpret_cast<O*>(P.out2), u, c, reinterpret_cast<__nv_bfloat16*>(stg));
          } else {
            if constexpr (IN == kI8) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] += bias;
            }
            put(reinterpret_cast<O*>(q.out), v, c, reinterpret_cast<__nv_bfloat16*>(stg));
          }
        }
      }
      if constexpr (IN != kF32) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&ctl.tmem_empty[it & 1]), 0));
        ++it;
      }
    }
  }

  __syncthreads();
  if (*abort_flag) {
    // the odd CTA's loads complete on the even CTA's barriers: a grace period for copies in flight
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- host side
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  EncodeFn f = __atomic_load_n(&fn, __ATOMIC_ACQUIRE);
  if (f == nullptr) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      return nullptr;
    f = reinterpret_cast<EncodeFn>(ptr);
    __atomic_store_n(&fn, f, __ATOMIC_RELEASE);
  }
  return f;
}

// rows x cols elements, rows ld apart; boxes of 128 bytes by box_rows
int make_map(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld, int es, int box_rows) {
  EncodeFn enc = encode_fn();
  if (enc == nullptr) return DSCA_ERR_CUDA;
  if (reinterpret_cast<uintptr_t>(base) % 16 != 0 || ld * es % 16 != 0) return DSCA_ERR_BAD_ARG;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(ld * es)};
  cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  auto encode = [&] {
    return enc(m, es == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
               const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {
    // a thread that has made no CUDA call yet (autograd's worker): bind its device's context
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = encode();
  }
  return r == CUDA_SUCCESS ? DSCA_OK : DSCA_ERR_CUDA;
}

template <int EPI, int IN, typename O, bool CLOSE = false>
int launch(const Params& P, int pairs, bool pdl, cudaStream_t stream) {
  static PerDeviceOnce once;
  auto kern = dense_kernel<EPI, IN, O, CLOSE>;
  if (once.run([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes); }) !=
      cudaSuccess)
    return DSCA_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min(pairs, P.total)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, P) == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

// Pairs that can be resident at once (a pair needs two free SMs of one cluster of SMs).
int resident_pairs() {
  static volatile int cache[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return current_device_sms() / 2;
  int n = __atomic_load_n(&cache[dev], __ATOMIC_ACQUIRE);
  if (n > 0) return n;
  auto kern = dense_kernel<kStore, kBf16, __nv_bfloat16>;
  const int sms = current_device_sms();
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sms & ~1));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) n = 0;
  }
  cudaGetLastError();
  n = n > 0 ? std::min(n, sms / 2) : std::max(1, sms / 2);
  __atomic_store_n(&cache[dev], n, __ATOMIC_RELEASE);
  return n;
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Boxes of 16-bit operands that one accumulator takes, 65536 of k: the tensor cores' additions truncate, always towards
// zero, and a sum of one sign loses 3e-4 to 5e-4 of itself over these (12 million tokens in 8 accumulators: a weight's gradient
// off by 9.5e-3, now 5e-4).  Longer sums are split, their parts added in rounded fp32.
constexpr int kMaxChain = 1024;

// The tiling of a job: fills everything of P but the maps and pointers.  Returns the units of work, or -1 when they
// pass 2^31.
int64_t plan(const Job& j, Params& P, int pairs, size_t* floats, size_t* counters) {
  const bool f32 = !j.i8 && j.dtype == DSCA_F32;
  const int ke = j.i8 ? 128 : 64;
  const int most = f32 ? 128 : 256;  // two accumulators of 128 columns share a buffer
  int64_t total = 0;
  *floats = *counters = 0;
  P.nprob = j.nprob;
  for (int i = 0; i < j.nprob; ++i) {
    const Problem& s = j.prob[i];
    Prob& q = P.prob[i];
    q = Prob{};
    const bool glu = j.epi == kGlu;
    q.rows = s.N; q.cols = s.M; q.K = s.K;
    const int oes = j.dtype == DSCA_BF16 ? 2 : 4;
    auto on = [&](const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
    auto rows_on = [&](int64_t n) {
      return s.ldo * oes % n == 0 && on(s.out, n) && on(j.out2, n) && on(j.save_g, n) && on(j.save_u, n);
    };
    q.vec = rows_on(32) ? 2 : rows_on(16) ? 1 : 0;
    // Rows need wide stores: a thread's single values would lie a row apart (2-byte stores of 901-wide rows, training
    // 333 x 1021 x 901: 53 us against 21 for the last product)
    q.row = s.N > 128 && q.vec;
    q.nseg = glu ? 1 : s.nseg;
    q.kb = ceil_div(s.K, ke);
    q.boxes = q.nseg * q.kb;
    q.a_mn = q.row ? s.b[0].mn : s.a[0].mn;
    q.b_mn = q.row ? s.a[0].mn : s.b[0].mn;
    // Tile width and k splits by an estimate of the time: waves of tiles, each its boxes' time and a fixed part.  A box
    // costs 0.38 us at 256 rows of B, 0.28 at 128 (4096 x 2048 x 5632); an fp32 slice three times that.
    const int whole = f32 ? 1 : 2;  // boxes of a stage
    const double slice = f32 ? 3.0 : 1.0;  // a box's time against 16 bits'
    double best = -1;
    auto consider = [&](int tn, int splits) {
      const int per_tile = q.row && glu ? tn / 2 : tn;
      const int tm = q.row ? ceil_div(q.rows, 256) : ceil_div(q.cols, glu ? 128 : 256);
      const int tiles_n = ceil_div(q.row ? q.cols : q.rows, per_tile);
      const int64_t tiles = (int64_t)tm * tiles_n;
      const int per = ceil_div(ceil_div(q.boxes, splits), whole) * whole;
      splits = ceil_div(q.boxes, per);
      if (splits > 1 && tiles * splits > 2 * pairs) return;  // bounds the partial tiles
      const double box = slice * (0.2 + 0.09 * tn / 128.0);          // us
      // the last tile's epilogue is not hidden: its chunks of 32 columns, two warps a lane quarter, and the pieces'
      // sums if the tile is split
      const double chunks = (tn + 63) / 64;
      const double last = chunks + (splits > 1 ? 2.0 + 0.4 * splits * chunks : 0.0);
      const double waves = j.nprob == 1 ? (double)ceil_div(tiles * splits, pairs) : std::max(1.0, (double)(tiles * splits) / pairs);
      const double cost = waves * (box * per + 0.5) + last;
      if (best < 0 || cost < best * 0.98) {
        best = cost;
        q.tn = tn; q.tiles_m = tm; q.tiles_n = tiles_n;
        q.splits = splits; q.per = per;
      }
    };
    for (int splits = 1; splits <= (j.nprob == 1 ? 8 : 1) && (splits == 1 || q.boxes >= (f32 ? 2 : 8) * splits); ++splits) {
      if (q.row || q.b_mn) {
        // a gated tile's gate and up chunks of 32 belong to one warp only from 64 channels on
        for (int tn = most; tn >= (q.b_mn || glu ? 128 : 64); tn /= 2) consider(tn, splits);
      } else {
        for (int nt = ceil_div(q.rows, most), e = nt + std::min(nt + 4, 12); nt <= e; ++nt)  // tokens in equal tiles
          consider(std::max(32, ceil_div(ceil_div(q.rows, nt), 32) * 32), splits);
      }
    }
  }
  // Several problems: one whose tiles take long against the whole launch's share of a pair is split (training
  // 640 x 768 x 2048: dx has nine tiles of 64 boxes beside 72 of ten)
  if (j.nprob > 1) {
    double work = 0;
    auto time = [](const Prob& q) { return (0.2 + 0.09 * q.tn / 128.0) * q.boxes; };
    for (int i = 0; i < j.nprob; ++i) work += time(P.prob[i]) * P.prob[i].tiles_m * P.prob[i].tiles_n;
    for (int i = 0; i < j.nprob; ++i) {
      Prob& q = P.prob[i];
      const int whole = f32 ? 1 : 2;
      int want = (int)std::min(8.0, time(q) / (0.6 * work / pairs));
      want = std::min(want, q.boxes / (f32 ? 2 : 8));
      if (want < 2 || (int64_t)q.tiles_m * q.tiles_n * want > 2 * pairs) continue;
      q.per = ceil_div(ceil_div(q.boxes, want), whole) * whole;
      q.splits = ceil_div(q.boxes, q.per);
    }
  }
  for (int i = 0; i < j.nprob; ++i) {
    Prob& q = P.prob[i];
    const int64_t tiles = (int64_t)q.tiles_m * q.tiles_n;
    if (!j.i8 && !f32 && q.per > kMaxChain) {
      q.per = kMaxChain;
      q.splits = ceil_div(q.boxes, q.per);
    }
    if (q.splits > 1) {
      if ((int64_t)*counters + tiles * 2 * kEpiWarps > 0x7fffffff) return -1;
      q.part = (int64_t)*floats;
      q.counter = (int)*counters;
      *floats += (size_t)tiles * q.splits * 2 * ((q.tn + 31) / 32 * 32) * 128;
      *counters += (size_t)tiles * 2 * kEpiWarps;
    }
    q.first = (int)total;
    total += tiles * q.splits;
    if (total > 0x7fffffff - 65536) return -1;
  }
  P.total = (int)total;
  return total;
}

}  // namespace tc

int tc_workspace(const Job& j, size_t* parts, size_t* counters) {
  tc::Params P;
  size_t floats, n;
  if (tc::plan(j, P, tc::resident_pairs(), &floats, &n) < 0) return DSCA_ERR_CAPACITY;
  *parts = floats * 4;
  *counters = n * 4;
  return DSCA_OK;
}

int launch_tc(const Job& j, void* parts, void* counts, int32_t* err, bool pdl, cudaStream_t stream) {
  tc::Params P = {};
  const int pairs = tc::resident_pairs();
  size_t floats, counters;
  if (tc::plan(j, P, pairs, &floats, &counters) < 0) return DSCA_ERR_CAPACITY;
  if (P.total == 0) return DSCA_OK;
  const bool f32 = !j.i8 && j.dtype == DSCA_F32;
  const int es = j.i8 ? 1 : 2;
  for (int i = 0; i < j.nprob; ++i) {
    const Problem& s = j.prob[i];
    tc::Prob& q = P.prob[i];
    q.out = s.out;
    q.ldo = s.ldo;
    const int planes = f32 ? 3 : 1;
    const Operand *A = q.row ? s.b : s.a, *B = q.row ? s.a : s.b;  // the MMA's operands
    const int a_ext = q.row ? s.N : s.M, b_ext = q.row ? s.M : s.N;
    q.a_plane = (int)A[0].plane;
    q.b_plane = (int)B[0].plane;
    const bool glu = j.epi == kGlu;
    const int na = glu ? (q.row ? 1 : 2) : s.nseg, nb = glu ? (q.row ? 2 : 1) : s.nseg;
    // fp32: three planes of rows (an MN-major plane ends on a whole MMA step of zeros)
    auto map = [&](CUtensorMap* m, const Operand& o, int ext, int box) {
      const int64_t rows = f32 ? planes * o.plane : (int64_t)(o.mn ? s.K : ext);
      return tc::make_map(m, o.p, rows, o.mn ? ext : s.K, o.ld, es, o.mn ? 64 : box);
    };
    for (int g = 0; g < na; ++g)
      if (int rc = map(&P.a[i][g], A[g], a_ext, glu && !q.row ? 64 : 128)) return rc;
    for (int g = 0; g < nb; ++g)
      if (int rc = map(&P.b[i][g], B[g], b_ext, q.tn / 2)) return rc;
  }
  P.act = j.act;
  P.save_g = j.save_g; P.save_u = j.save_u; P.save_e = j.save_e; P.out2 = j.out2;
  P.row_scale = j.row_max != nullptr ? j.row_max : j.row_scale; P.col_scale[0] = j.col_scale[0]; P.col_scale[1] = j.col_scale[1]; P.bias = j.bias;
  P.vec_cols = (reinterpret_cast<uintptr_t>(j.col_scale[0]) | reinterpret_cast<uintptr_t>(j.col_scale[1])) % 16 == 0;
  P.counters = reinterpret_cast<uint32_t*>(counts);
  P.parts = reinterpret_cast<float*>(parts);
  P.err = err;
  using B = __nv_bfloat16;
  if (j.i8) {
    if (j.epi == kGlu)
      return j.row_max != nullptr ? tc::launch<kGlu, tc::kI8, float, true>(P, pairs, pdl, stream)
                                  : tc::launch<kGlu, tc::kI8, float>(P, pairs, pdl, stream);
    return j.dtype == DSCA_BF16 ? tc::launch<kStore, tc::kI8, B>(P, pairs, pdl, stream)
                                : tc::launch<kStore, tc::kI8, float>(P, pairs, pdl, stream);
  }
  if (f32) {
    if (j.epi == kGlu) return tc::launch<kGlu, tc::kF32, float>(P, pairs, pdl, stream);
    if (j.epi == kDGlu) return tc::launch<kDGlu, tc::kF32, float>(P, pairs, pdl, stream);
    return tc::launch<kStore, tc::kF32, float>(P, pairs, pdl, stream);
  }
  if (j.epi == kGlu) return tc::launch<kGlu, tc::kBf16, B>(P, pairs, pdl, stream);
  if (j.epi == kDGlu) return tc::launch<kDGlu, tc::kBf16, B>(P, pairs, pdl, stream);
  return tc::launch<kStore, tc::kBf16, B>(P, pairs, pdl, stream);
}

}  // namespace dense
}  // namespace dsca
