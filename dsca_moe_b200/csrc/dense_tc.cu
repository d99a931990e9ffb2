// The products of dense.cuh on the tensor cores: CTA pairs, tcgen05 cta_group::2, TMA-fed.
//
// A tile is 256 m x up to 256 n: each CTA of a pair loads its 128 rows of A and half of the tile's rows of
// B, so an SM streams 32 KB for every 64-wide slice of k in 16 bits (128-wide in 8), and the even CTA issues
// the MMAs (M256 N<=256) into both CTAs' tensor memory.  TMEM lane = m, the output's contiguous index, column
// = n: a token tile of 20 rows costs 32 columns, not 256.
//   warp 0      TMA producer (one thread), 128-byte swizzle, three stages of two 128-byte k boxes
//   warp 1      TMEM (512 columns: two accumulators); in the even CTA the MMA issuer
//   warps 2-9   epilogue: two warps to a lane quarter, alternate chunks of 32 columns
// Operands: a K-major one is loaded as boxes of 128 bytes of k by its rows; an MN-major one as boxes of 64
// rows of k by 64 values of m or n, which the MMA reads transposed, so that the gradients' products take
// weights and activations as they lie.
//
// Gated products (kGlu): a CTA's 128 rows of A are 64 gate rows and the up rows of the same channels, so the
// epilogue warps of lane quarters q and q + 2 hold the gate and up values of the same 32 channels.  For each
// chunk of 32 columns the gate warp forms the products of the first 16 and the up warp those of the last,
// after handing each other the other half through shared memory.  (Alternating boxes of 16 gate and 16 up
// rows would bring both into one warp, but eight small boxes instead of two cost more than the exchange:
// 4096 x 2048 x 5632 188 us against 152.)
// Saved for the backward pass in 16 bits: g and u as fp16 with one power of two for a channel's 32 tokens
// (11 bits of significand for every value within 2^29 of the largest), half of fp32's bytes, which the
// backward pass reads against the clock of its first product.
//
// 32-bit inputs (kF32): every value is split into three bf16 terms (8 + 8 + 8 bits, dense_split.cu) and the
// product is six MMA passes over k: hi.hi into one accumulator, hi.mid, mid.hi, hi.lo, mid.mid and lo.hi into
// another, which the epilogue adds.  What is left out is 2^-24 of the product's terms.
//
// Long k with few tiles: the k boxes are split over several pairs, each stores its fp32 tile to the workspace,
// and for every warp's part the last one to arrive adds the parts in the order of k: the result does not
// depend on who is last.
//
// Every wait is bounded (2 s); on a timeout the kernel records DSCA_ERR_WAIT_TIMEOUT, drains what it can
// observe, waits a grace period for copies into the pair, frees TMEM and returns.
#include "dense.cuh"

#include <algorithm>
#include <type_traits>

namespace dsca {
namespace dense {
namespace tc {

#ifndef KSUB
#define KSUB 2
#endif
constexpr int kSub = KSUB;                       // k boxes of a stage
constexpr int kStages = 6 / kSub;
constexpr int kBoxBytes = 128 * 128;             // an operand's part of one k box
constexpr int kStageBytes = 2 * kSub * kBoxBytes;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kStgBytes = 2 * 32 * 32 * 2;       // per epilogue warp: two 32 x 32 blocks of bf16
constexpr int kSmemBytes = kStages * kStageBytes + kEpiWarps * kStgBytes + 1024;
static_assert(kSmemBytes <= 227 * 1024, "shared memory of a CTA");

enum In { kBf16 = 0, kI8 = 1, kF32 = 2 };

struct Prob {
  int M, N, K;
  int nseg, kb;          // segments; k boxes of each
  int boxes;             // nseg * terms * kb
  int a_mn, b_mn;
  int tiles_m, tiles_n, tn;
  int splits, per;       // k splits and boxes of each (even)
  int first;             // the problem's first unit of work
  int a_plane, b_plane;  // kF32: rows between the planes of three terms
  int vec;               // out rows start on 16-byte boundaries
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
  uint8_t* save_e;  // fp16: the exponents, [2][ceil(N / 32)][ldo]
  void* out2;
  const float* row_scale;
  const float* col_scale[2];
  const void* bias;
  float* parts;
  uint32_t* counters;
  int32_t* err;
};

struct Ctl {
  uint64_t full[kStages], empty[kStages], tmem_full[2], tmem_empty[2], mma_done;
  uint32_t tmem_base;
  int abort_flag;
  int pair_ok[kEpiWarps], pair_old[kEpiWarps];
};

struct Tile {
  int p, m, n0, ntok, box0, box1, split;
  int64_t tile;  // within the problem
};

__device__ __forceinline__ Tile decode(const Params& P, int unit) {
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
  t.m = 8 * g + r % gm;
  t.n0 = (r / gm) * q.tn;
  t.ntok = min(q.tn, q.N - t.n0);
  t.box0 = t.split * q.per;
  t.box1 = min(q.boxes, t.box0 + q.per);
  return t;
}

// MMA N of a tile with ntok rows of B: each CTA holds half, whole 8-row groups (64 rows if MN-major)
__device__ __forceinline__ int mma_n(const Prob& q, int ntok) {
  return q.b_mn ? (ntok + 127) & ~127 : max(16, (ntok + 15) & ~15);
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

__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Where box b of a problem lies: slice k of a segment and, for 32-bit inputs, one of the six terms, which follow
// one another within a slice.  Divisions once a tile, then counted on.
template <int IN>
struct BoxAt {
  int seg, term, k;
  __device__ __forceinline__ BoxAt(const Prob& q, int b) {
    int s = b;
    term = 0;
    if constexpr (IN == kF32) {
      s = b / 6;
      term = b - 6 * s;
    }
    seg = s >= q.kb ? 1 : 0;
    k = s - seg * q.kb;
  }
  __device__ __forceinline__ void next(int kb) {
    if constexpr (IN == kF32) {
      if (++term < 6) return;
      term = 0;
    }
    if (++k == kb) {
      k = 0;
      ++seg;
    }
  }
};
// the planes (hi 0, mid 1, lo 2) that term t multiplies
__device__ __forceinline__ int plane_a(int t) { return t == 2 || t == 4 ? 1 : t == 5 ? 2 : 0; }
__device__ __forceinline__ int plane_b(int t) { return t == 1 || t == 4 ? 1 : t == 3 ? 2 : 0; }

// The two warps (64 threads) that exchange gate and up values.
__device__ __forceinline__ void pair_barrier(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// 32 tokens of one channel as fp16 times a power of two that brings the largest finite one to [2^14, 2^15); the
// exponent byte is the largest's, at least 14 so that the factor is a normal number.
__device__ __forceinline__ void save_f16(const Params& P, const Prob& q, int up, int ch, int n, int ntok, const float (&v)[32]) {
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const float a = fabsf(v[j]);
    if (j < ntok && a <= 3.4028234663852886e38f) m = fmaxf(m, a);
  }
  const uint32_t e = max(14u, __float_as_uint(m) >> 23);
  const float s = __uint_as_float((268u - e) << 23);  // 2^(141 - e)
  if (ch >= q.M) return;
  __half* at = reinterpret_cast<__half*>(up ? P.save_u : P.save_g) + (int64_t)n * q.ldo + ch;
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (j < ntok) at[j * q.ldo] = __float2half_rn(v[j] * s);
  P.save_e[((int64_t)up * ((q.N + 31) / 32) + n / 32) * q.ldo + ch] = (uint8_t)e;
}

// g and u of the chunk after the one in work (kDGlu, 16 bits): 32 tokens x 32 channels each, 16 bytes a load.
struct Ahead {
  uint4 v[8];
  uint32_t e[2];
  __device__ __forceinline__ void load(const Params& P, const Prob& q, const Tile& t, uint32_t rank, int q4, int lane, int c) {
    const int m0 = t.m * 256 + 128 * (int)rank + 32 * q4, ch = m0 + 8 * (lane & 3);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int tok = c + (i & 3) * 8 + (lane >> 2);
      const __half* p = reinterpret_cast<const __half*>(i < 4 ? P.save_g : P.save_u);
      v[i] = ch < q.M && tok < t.ntok ? __ldg(reinterpret_cast<const uint4*>(p + (int64_t)(t.n0 + tok) * q.ldo + ch))
                                      : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      e[i] = m0 + lane < q.M && c < t.ntok
                 ? P.save_e[((int64_t)i * ((q.N + 31) / 32) + (t.n0 + c) / 32) * q.ldo + m0 + lane] : 141u;
  }
  __device__ __forceinline__ void store(uint8_t* stg, int lane) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *reinterpret_cast<uint4*>(stg + (i >> 2) * 2048 + ((i & 3) * 8 + (lane >> 2)) * 64 + 16 * (lane & 3)) = v[i];
  }
  __device__ __forceinline__ float scale(int i) const {  // 2^(e - 141)
    const int x = (int)e[i] - 14;  // its biased exponent; 0 and 1 from e = 14, 15 on
    return x > 0 ? __uint_as_float((uint32_t)x << 23) : 5.877471754111438e-39f;
  }
};

template <int EPI, int IN, typename O>
__global__ void __launch_bounds__(kThreads, 1) dense_kernel(const __grid_constant__ Params P) {
  constexpr bool kGluE = EPI == kGlu;
  constexpr int KE = IN == kI8 ? 128 : 64;   // k elements of a box
  constexpr int KS = IN == kI8 ? 32 : 16;    // ... and of one MMA
  constexpr bool kFast = sizeof(O) == 2 && IN != kI8;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ Ctl ctl;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_a = smem_u32(smem), smem_b = smem_a + kSub * kBoxBytes;  // of stage 0
  const int warp = warp_id(), lane = lane_id();
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

  if (warp == 0) {
    // ---------------- TMA producer
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      int pending[kStages];
      for (int i = 0; i < kStages; ++i) pending[i] = -1;
      bool ok = true;
      for (int unit = unit0; ok && unit < P.total; unit += units) {
        const Tile t = decode(P, unit);
        const Prob& q = P.prob[t.p];
        const int half = mma_n(q, t.ntok) / 2;
        const int b_row = t.n0 + half * (int)rank;
        const uint32_t b_bytes = (uint32_t)(q.tn / 2) * 128u;  // a whole box lands; rows past the tile are not used
        const int kb = q.kb, a_mn = q.a_mn, b_atoms = q.b_mn ? q.tn / 128 : 0;
        const CUtensorMap *ma = P.a[t.p], *mb = P.b[t.p];
        BoxAt<IN> at(q, t.box0);
        for (int b = t.box0; b < t.box1; b += kSub) {
          if (!mbar_wait(smem_u32(&ctl.empty[s]), ph ^ 1u, abort_flag, P.err)) { ok = false; break; }
          const uint32_t fb0 = mapa_shared(smem_u32(&ctl.full[s]), 0);
          const int nb = min(kSub, t.box1 - b);
          if (rank == 0)
            mbar_arrive_expect_tx(smem_u32(&ctl.full[s]), 2u * (uint32_t)nb * ((uint32_t)kBoxBytes + b_bytes));
          for (int h = 0; h < nb; ++h, at.next(kb)) {
            const uint32_t da = smem_a + s * kStageBytes + h * kBoxBytes, db = smem_b + s * kStageBytes + h * kBoxBytes;
            const int pa = IN == kF32 ? plane_a(at.term) * q.a_plane : 0, pb = IN == kF32 ? plane_b(at.term) * q.b_plane : 0;
            const int kx = at.k * KE;
            if constexpr (kGluE) {
              const int r0 = t.m * 128 + 64 * (int)rank + pa;
              tma_load_2d_pair(da, ma, fb0, kx, r0);
              tma_load_2d_pair(da + 8192, ma + 1, fb0, kx, r0);
            } else if (a_mn) {
              const int r0 = t.m * 256 + 128 * (int)rank;
              tma_load_2d_pair(da, ma + at.seg, fb0, r0, kx + pa);
              tma_load_2d_pair(da + 8192, ma + at.seg, fb0, r0 + 64, kx + pa);
            } else {
              tma_load_2d_pair(da, ma + at.seg, fb0, kx, t.m * 256 + 128 * (int)rank + pa);
            }
            if (b_atoms) {
              tma_load_2d_pair(db, mb + at.seg, fb0, b_row, kx + pb);
              if (b_atoms > 1) tma_load_2d_pair(db + 8192, mb + at.seg, fb0, b_row + 64, kx + pb);
            } else {
              tma_load_2d_pair(db, mb + at.seg, fb0, kx, b_row + pb);
            }
          }
          pending[s] = (int)ph;
          if (++s == kStages) { s = 0; ph ^= 1u; }
        }
      }
      if (!ok && rank == 0)
        for (int i = 0; i < kStages; ++i)
          if (pending[i] >= 0) drain(smem_u32(&ctl.full[i]), (uint32_t)pending[i]);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (even CTA)
    if (lane == 0 && rank == 0) {
      int s = 0, it = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int unit = unit0; ok && unit < P.total; unit += units, ++it) {
        const Tile t = decode(P, unit);
        const Prob& q = P.prob[t.p];
        const int acc = it & 1;
        // D f32 (1) or s32 (2); A, B bf16 (1) or signed 8-bit (1); majors; N; M = 256
        const uint32_t idesc = ((IN == kI8 ? 2u : 1u) << 4) | (1u << 7) | (1u << 10) | ((uint32_t)q.a_mn << 15) |
                               ((uint32_t)q.b_mn << 16) | ((uint32_t)(mma_n(q, t.ntok) >> 3) << 17) | (16u << 24);
        if (!mbar_wait(smem_u32(&ctl.tmem_empty[acc]), (uint32_t)(((it >> 1) & 1) ^ 1), abort_flag, P.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(acc * 256);
        // descriptors but for the stage, and their steps of one MMA (in 16 bytes: 2 KB or 32 bytes)
        const uint64_t ad0 = q.a_mn ? sw128_mnmajor_desc(smem_a) : sw128_kmajor_desc(smem_a);
        const uint64_t bd0 = q.b_mn ? sw128_mnmajor_desc(smem_b) : sw128_kmajor_desc(smem_b);
        const uint64_t astep = q.a_mn ? 128u : 2u, bstep = q.b_mn ? 128u : 2u;
        const int kb = q.kb, last_steps = (q.K - (kb - 1) * KE + KS - 1) / KS;
        uint32_t used0 = 0u, used1 = 0u;
        BoxAt<IN> at(q, t.box0);
        for (int b = t.box0; b < t.box1; b += kSub) {
          if (!mbar_wait(smem_u32(&ctl.full[s]), ph, abort_flag, P.err)) { ok = false; break; }
          tc_fence_after();
          const int nb = min(kSub, t.box1 - b);
#pragma unroll
          for (int h = 0; h < kSub; ++h) {
            if (h < nb) {
              const uint64_t off = (uint64_t)((s * kStageBytes + h * kBoxBytes) >> 4);
              const uint64_t ad = ad0 + off, bd = bd0 + off;
              const int steps = at.k == kb - 1 ? last_steps : 4;
              const bool corr = IN == kF32 && at.term != 0;
              const uint32_t dd = corr ? d + 128u : d;
              uint32_t used = corr ? used1 : used0;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (i < steps) {
                  if constexpr (IN == kI8) umma_i8_pair(dd, ad + astep * i, bd + bstep * i, idesc, used);
                  else umma_f16_pair(dd, ad + astep * i, bd + bstep * i, idesc, used);
                  used = 1u;
                }
              if (corr) used1 = 1u;
              else used0 = 1u;
              at.next(kb);
            }
          }
          umma_commit_pair_both(smem_u32(&ctl.empty[s]));
          if (++s == kStages) { s = 0; ph ^= 1u; }
        }
        if (!ok) break;
        umma_commit_pair_both(smem_u32(&ctl.tmem_full[acc]));
      }
      if (!ok) {  // every MMA issued has completed before TMEM is freed
        umma_commit_pair(mapa_shared(smem_u32(&ctl.mma_done), 0));
        drain(smem_u32(&ctl.mma_done), 0);
      }
    }
  } else {
    // ---------------- epilogue
    const int q4 = warp & 3, ew = warp - 2, eh = ew >> 2;
    uint8_t* stg = smem + kStages * kStageBytes + ew * kStgBytes;
    __nv_bfloat16* stg16 = reinterpret_cast<__nv_bfloat16*>(stg);
    int it = 0, xb = 0;
    Ahead ahead;
    for (int unit = unit0; unit < P.total; unit += units, ++it) {
      const Tile t = decode(P, unit);
      const Prob& q = P.prob[t.p];
      const int acc = it & 1;
      if constexpr (EPI == kDGlu && IN == kBf16) ahead.load(P, q, t, rank, q4, lane, 32 * eh);
      int w_ok = 1;
      if (lane == 0) w_ok = mbar_wait(smem_u32(&ctl.tmem_full[acc]), (uint32_t)((it >> 1) & 1), abort_flag, P.err) ? 1 : 0;
      w_ok = __shfl_sync(0xffffffffu, w_ok, 0);
      if constexpr (kGluE) {
        // the two warps of an exchange go on or leave together
        if (lane == 0) ctl.pair_ok[ew] = w_ok;
        pair_barrier(1 + (ew & 1) + 2 * eh);
        w_ok = *reinterpret_cast<volatile int*>(&ctl.pair_ok[ew ^ 2]) & w_ok;
      }
      if (!w_ok) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * 256);
      const int ncol = mma_n(q, t.ntok);
      // a chunk of the accumulator: lane's m, 32 columns from c on
      auto chunk = [&](int c, uint32_t (&v)[32]) {
        tmem_ld32(taddr + c, v);
        if constexpr (IN == kF32) {
          uint32_t w[32];
          tmem_ld32(taddr + 128 + c, w);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(w[j]));
        } else {
          tmem_wait_ld();
        }
      };
      bool mine = true;
      float* part = nullptr;
      int64_t part_step = 0;
      if (q.splits > 1) {
        // this warp's part of the tile: [split][column][lane]
        part_step = (int64_t)2 * q.tn * 128;
        part = P.parts + q.part + t.tile * q.splits * part_step + (int64_t)rank * q.tn * 128 + q4 * 32 + lane;
        for (int c = 32 * eh; c < ncol; c += 64) {
          uint32_t v[32];
          chunk(c, v);
          float* at = part + t.split * part_step + (int64_t)c * 128;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j < t.ntok) at[(int64_t)j * 128] = __uint_as_float(v[j]);
        }
        __threadfence();
        __syncwarp();
        uint32_t old = 0;
        uint32_t* counter = P.counters + q.counter + (t.tile * 2 + rank) * kEpiWarps + ew;
        if constexpr (kGluE) {
          // one count for the two warps of an exchange, which finish a tile together
          pair_barrier(1 + (ew & 1) + 2 * eh);
          if (!(q4 >> 1) && lane == 0) {
            __threadfence();
            ctl.pair_old[ew] = (int)atomicAdd(counter, 1u);
          }
          pair_barrier(1 + (ew & 1) + 2 * eh);
          old = (uint32_t)*reinterpret_cast<volatile int*>(&ctl.pair_old[ew | 2]);  // the gate warps are 2, 3, 6, 7
        } else {
          if (lane == 0) old = atomicAdd(counter, 1u);
          old = __shfl_sync(0xffffffffu, old, 0);
        }
        mine = old == (uint32_t)q.splits - 1u;
        if (mine) __threadfence();
      }
      if (mine) {
        const int mrow = t.m * 256 + 128 * (int)rank + 32 * q4 + lane;  // this lane's m (not kGlu)
        const int gch = t.m * 128 + 64 * (int)rank + 32 * (q4 & 1) + lane;  // kGlu: its channel
        const int up = q4 >> 1;                                              // ... of gate (0) or up (1)
        float cs = 1.0f, bias = 0.0f;
        if constexpr (IN == kI8) {
          if constexpr (kGluE) cs = gch < q.M ? __ldg((up ? P.col_scale[1] : P.col_scale[0]) + gch) : 0.0f;
          else cs = mrow < q.M ? __ldg(P.col_scale[0] + mrow) : 0.0f;
        }
        if constexpr (EPI == kStore && IN == kI8) {
          if (P.bias != nullptr && mrow < q.M) {
            if constexpr (sizeof(O) == 2) bias = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(P.bias)[mrow]);
            else bias = reinterpret_cast<const float*>(P.bias)[mrow];
          }
        }
#pragma unroll 1
        for (int c = 32 * eh; c < ncol; c += 64) {
          if (c >= t.ntok) break;
          float gv[32], uv[32];
          if constexpr (EPI == kDGlu && IN == kBf16) {
            // the chunk's g and u go through shared memory to the lane of their channel; the next chunk's
            // are on their way meanwhile
            const float sg = ahead.scale(0), su = ahead.scale(1);
            ahead.store(stg, lane);
            __syncwarp();
            if (c + 64 < ncol) ahead.load(P, q, t, rank, q4, lane, c + 64);
            const __half* sh = reinterpret_cast<const __half*>(stg);
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              gv[j] = __half2float(sh[j * 32 + lane]) * sg;
              uv[j] = __half2float(sh[1024 + j * 32 + lane]) * su;
            }
            __syncwarp();
          } else if constexpr (EPI == kDGlu) {  // on their way before the accumulator is read
            const int64_t at = (int64_t)(t.n0 + c) * q.ldo + mrow;
            const float *pg = reinterpret_cast<const float*>(P.save_g), *pu = reinterpret_cast<const float*>(P.save_u);
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const bool in = mrow < q.M && c + j < t.ntok;
              gv[j] = in ? __ldg(pg + at + j * q.ldo) : 0.0f;
              uv[j] = in ? __ldg(pu + at + j * q.ldo) : 0.0f;
            }
          }
          float v[32];
          {
            uint32_t r[32];
            if (q.splits > 1) {
              // the parts in the order of k (8-bit: int32 sums)
#pragma unroll
              for (int j = 0; j < 32; ++j) r[j] = 0u;
              for (int s = 0; s < q.splits; ++s) {
                const float* at = part + s * part_step + (int64_t)c * 128;
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (c + j < t.ntok) {
                    const float x = __ldcg(at + (int64_t)j * 128);
                    if constexpr (IN == kI8) r[j] += __float_as_uint(x);
                    else r[j] = __float_as_uint(__uint_as_float(r[j]) + x);
                  }
              }
            } else {
              chunk(c, r);
            }
            if constexpr (IN == kI8) {
              const float rs = c + lane < t.ntok ? __ldg(P.row_scale + t.n0 + c + lane) : 0.0f;
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = (float)(int)r[j] * (cs * __shfl_sync(0xffffffffu, rs, j));
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
            }
          }
          if constexpr (kGluE) {
            if (P.save_g != nullptr) {
              if constexpr (IN == kBf16) save_f16(P, q, up, gch, t.n0 + c, t.ntok - c, v);
              else if (gch < q.M) {
                float* at = reinterpret_cast<float*>(up ? P.save_u : P.save_g) + (int64_t)(t.n0 + c) * q.ldo + gch;
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (c + j < t.ntok) at[j * q.ldo] = v[j];
              }
            }
            // the gate warp forms columns 0-15 of the chunk, the up warp 16-31; two buffers, so that one
            // barrier a chunk is enough
            float* mine_x = reinterpret_cast<float*>(stg) + xb * 512;
            float* other_x = reinterpret_cast<float*>(smem + kStages * kStageBytes + (ew ^ 2) * kStgBytes) + xb * 512;
            xb ^= 1;
#pragma unroll
            for (int j = 0; j < 16; ++j) mine_x[j * 32 + lane] = up ? v[j] : v[16 + j];
            pair_barrier(1 + (ew & 1) + 2 * eh);
            float o[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float got = other_x[j * 32 + lane];
              const float g = up ? got : v[j], u = up ? v[16 + j] : got;
              o[j] = gate<kFast>(g, P.act) * u;
            }
            const int tok0 = c + 16 * up;
            O* out = reinterpret_cast<O*>(q.out);
            if (sizeof(O) == 2 && q.vec && (gch & ~31) + 32 <= q.M) {
              if constexpr (sizeof(O) == 2) {
                // staged where the other warp's values lay, which this warp alone reads
                __nv_bfloat16* st = reinterpret_cast<__nv_bfloat16*>(other_x);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 16; ++j) st[j * 32 + lane] = __float2bfloat16_rn(o[j]);
                __syncwarp();
#pragma unroll
                for (int rr = 0; rr < 2; ++rr) {
                  const int tok = rr * 8 + (lane >> 2);
                  if (tok0 + tok < t.ntok)
                    *reinterpret_cast<uint4*>(out + (int64_t)(t.n0 + tok0 + tok) * q.ldo + (gch & ~31) + 8 * (lane & 3)) =
                        *reinterpret_cast<const uint4*>(st + tok * 32 + 8 * (lane & 3));
                }
              }
            } else if (gch < q.M) {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (tok0 + j < t.ntok) {
                  O* at = out + (int64_t)(t.n0 + tok0 + j) * q.ldo + gch;
                  if constexpr (sizeof(O) == 2) *at = __float2bfloat16_rn(o[j]);
                  else *at = o[j];
                }
            }
          } else {
            constexpr int NO = EPI == kDGlu ? 2 : 1;
            if constexpr (EPI == kDGlu) {
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                float a, da;
                gate_grad<kFast>(gv[j], P.act, &a, &da);
                const float dh = v[j];
                v[j] = dh * uv[j] * da;
                uv[j] = dh * a;
              }
            }
            if constexpr (EPI == kStore && IN == kI8) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] += bias;
            }
            O* outs[2] = {reinterpret_cast<O*>(q.out), reinterpret_cast<O*>(P.out2)};
            if (sizeof(O) == 2 && q.vec && t.m * 256 + 128 * (int)rank + 32 * q4 + 32 <= q.M) {
              if constexpr (sizeof(O) == 2) {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  stg16[j * 32 + lane] = __float2bfloat16_rn(v[j]);
                  if constexpr (NO == 2) stg16[1024 + j * 32 + lane] = __float2bfloat16_rn(uv[j]);
                }
                __syncwarp();
#pragma unroll
                for (int o = 0; o < NO; ++o)
#pragma unroll
                  for (int rr = 0; rr < 4; ++rr) {
                    const int tok = rr * 8 + (lane >> 2);
                    if (c + tok < t.ntok)
                      *reinterpret_cast<uint4*>(outs[o] + (int64_t)(t.n0 + c + tok) * q.ldo + (mrow & ~31) + 8 * (lane & 3)) =
                          *reinterpret_cast<const uint4*>(stg16 + o * 1024 + tok * 32 + 8 * (lane & 3));
                  }
                __syncwarp();
              }
            } else if (mrow < q.M) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (c + j < t.ntok) {
                  const int64_t at = (int64_t)(t.n0 + c + j) * q.ldo + mrow;
                  if constexpr (sizeof(O) == 2) outs[0][at] = __float2bfloat16_rn(v[j]);
                  else outs[0][at] = v[j];
                  if constexpr (NO == 2) {
                    if constexpr (sizeof(O) == 2) outs[1][at] = __float2bfloat16_rn(uv[j]);
                    else outs[1][at] = uv[j];
                  }
                }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&ctl.tmem_empty[acc]), 0));
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

template <int EPI, int IN, typename O>
int launch(const Params& P, int pairs, bool pdl, cudaStream_t stream) {
  static PerDeviceOnce once;
  auto kern = dense_kernel<EPI, IN, O>;
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
    q.M = s.M; q.N = s.N; q.K = s.K;
    q.nseg = j.epi == kGlu ? 1 : s.nseg;
    q.kb = ceil_div(s.K, ke);
    q.boxes = q.nseg * (f32 ? 6 : 1) * q.kb;
    q.a_mn = s.a[0].mn; q.b_mn = s.b[0].mn;
    q.tiles_m = ceil_div(s.M, j.epi == kGlu ? 128 : 256);
    // rows of n a tile: the waves of tiles by a tile's time, which is mostly the 256 rows of A (2048 x 5632, us a
    // stage of two boxes: 1.15 at 256 rows of n, 0.95 at 192, 0.86 at 128)
    q.tn = most;
    if (q.b_mn) {
      if (s.N <= 128) q.tn = 128;
    } else {
      double best = 0;
      const int unit = j.epi == kStore ? 16 : 32;  // g and u are saved by whole 32 tokens
      for (int nt = ceil_div(s.N, most), e = nt + 4; nt <= e; ++nt) {
        const int tn = std::max(unit, (ceil_div(s.N, nt) + unit - 1) / unit * unit);
        const int64_t tiles = (int64_t)q.tiles_m * ceil_div(s.N, tn);
        const double cost = (j.nprob == 1 ? (double)ceil_div(tiles, pairs) : (double)tiles / pairs) * (tn + 280);
        if (best == 0 || cost < best * 0.99) {
          best = cost;
          q.tn = tn;
        }
      }
    }
    q.tiles_n = ceil_div(s.N, q.tn);
    q.splits = 1;
    q.per = (q.boxes + 1) / 2 * 2;
    const int64_t tiles = (int64_t)q.tiles_m * q.tiles_n;
    if (j.nprob == 1 && tiles * 2 <= pairs) {
      // at least four stages (eight boxes) a split
      const int want = (int)std::min<int64_t>(pairs / tiles, q.boxes / 8);
      if (want > 1) {
        const int whole = f32 ? 6 : 2;  // all terms of a slice, whole stages
        q.per = ceil_div(ceil_div(q.boxes, want), whole) * whole;
        q.splits = ceil_div(q.boxes, q.per);
      }
    }
    if (q.splits > 1) {
      q.part = (int64_t)*floats;
      q.counter = (int)*counters;
      *floats += (size_t)tiles * q.splits * 2 * q.tn * 128;
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

size_t tc_workspace(const Job& j) {
  tc::Params P;
  size_t floats, counters;
  if (tc::plan(j, P, tc::resident_pairs(), &floats, &counters) < 0) return 0;
  return (counters * 4 + 255) / 256 * 256 + floats * 4;
}

// The counters lie at the start of ws (zeroed by the caller), the partial tiles behind them.
int launch_tc(const Job& j, void* ws, int32_t* err, bool pdl, cudaStream_t stream) {
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
    const int oes = j.dtype == DSCA_BF16 ? 2 : 4;
    q.vec = reinterpret_cast<uintptr_t>(s.out) % 16 == 0 && s.ldo * oes % 16 == 0 &&
            reinterpret_cast<uintptr_t>(j.out2) % 16 == 0;
    const int planes = f32 ? 3 : 1;
    q.a_plane = (int)s.a[0].plane;
    q.b_plane = (int)s.b[0].plane;
    for (int g = 0; g < 2; ++g) {
      const Operand &a = s.a[g], &b = s.b[g];
      const bool has_a = g == 0 || j.epi == kGlu || s.nseg > 1, has_b = g == 0 || (j.epi != kGlu && s.nseg > 1);
      // fp32: three planes of rows (an MN-major plane ends on a whole MMA step of zeros)
      auto rows = [&](const Operand& o, int r) { return f32 ? planes * o.plane : (int64_t)(o.mn ? s.K : r); };
      if (has_a)
        if (int rc = tc::make_map(&P.a[i][g], a.p, rows(a, s.M), a.mn ? s.M : s.K, a.ld, es,
                                  a.mn || j.epi == kGlu ? 64 : 128))
          return rc;
      if (has_b)
        if (int rc = tc::make_map(&P.b[i][g], b.p, rows(b, s.N), b.mn ? s.N : s.K, b.ld, es, b.mn ? 64 : q.tn / 2))
          return rc;
    }
  }
  P.act = j.act;
  P.save_g = j.save_g; P.save_u = j.save_u; P.save_e = j.save_e; P.out2 = j.out2;
  P.row_scale = j.row_scale; P.col_scale[0] = j.col_scale[0]; P.col_scale[1] = j.col_scale[1]; P.bias = j.bias;
  P.counters = reinterpret_cast<uint32_t*>(ws);
  P.parts = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(ws) + (counters * 4 + 255) / 256 * 256);
  P.err = err;
  using B = __nv_bfloat16;
  if (j.i8) {
    if (j.epi == kGlu) return tc::launch<kGlu, tc::kI8, float>(P, pairs, pdl, stream);
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

// Bytes of counters at the start of the workspace that have to be zero at the launch.
size_t tc_zero_bytes(const Job& j) {
  tc::Params P;
  size_t floats, counters;
  if (tc::plan(j, P, tc::resident_pairs(), &floats, &counters) < 0) return 0;
  return counters * 4;
}

}  // namespace dense
}  // namespace dsca
