// The whole MoE block for a few tokens (at most 32) in one kernel.
//
//   logits = round(x W_r^T)          p = softmax(logits)      S_t = the k largest p (lowest id first)
//   h_te   = w_te act(up_e x_t)      out_t = sum_{e in S_t} down_e h_te + sigmoid(round(x.g)) shared(x_t)
//
// Such a call's time is the reading of the chosen experts' weights (17 MB an expert of the Qwen block
// in bf16, 69 MB for its shared expert, against 4 KB a token), so everything here serves one
// uninterrupted stream of weight bytes:
//  - one persistent CTA per SM.  Two producer warps copy boxes of 16 weight rows x 64 to 384 bytes into
//    shared memory by TMA (plain bulk copies, one a row, cost 60 ns of issue each: 16 times as much
//    per byte); each of twelve compute warps has its own ring of boxes, its share of k, and its sums in
//    registers, so that one warp's wait for its tokens' values (L2) passes under the others' products.
//    The values for the next box are asked for before the present one is multiplied.  Two service
//    warps run the router at the start; then, in turn, they add the twelve parts of each unit (16
//    rows of a matrix), apply the activation and store (in the warp that is the last with its part this
//    stood in the way of its next box: one token 43 us instead of 35);
//  - the weights are cut 16 rows at a time (8 gate + 8 up rows, or 16 rows of any other matrix), fine
//    enough that 148 SMs get nearly equal shares, where a 128-row tensor-memory tile would leave
//    two fifths of them idle at one token.  16 rows x 8 tokens is the shape of mma.sync, which
//    has to run at one 16x8x16 product per 20 clocks to keep up with DRAM;
//  - the order is shared GEMM1, routed GEMM1, shared GEMM2, routed GEMM2: the shared expert needs no
//    routing, so its weights are on their way while the router runs, and by the time a CTA needs
//    the intermediates of another one they have mostly been published.
//  - the routing weight is multiplied into the intermediate, so GEMM2 adds every expert's part into
//    the same fp32 sums and a CTA owns its rows of the output.  Where that would leave a CTA few rows
//    (a narrow model, or more than eight tokens, whose boxes are 32 rows high), several CTAs share a
//    tile of rows, each with its share of every row's boxes, and the last one to finish adds their
//    sums in order.
//
// Measured, against the weights' bytes at the 6.5 TB/s of a copy: the Qwen block (d 2048, 60 experts of 1408, 4
// a token, a shared one of 5632) 1 token in bf16 31.3 us (4.4 TB/s, 68%), with fp8 weights 28 us (38%),
// 8 tokens in bf16 92-96 us (84%), 20 tokens 178 us, 32 tokens with fp8 weights 138 us (55%); a Switch block (d 768, 64
// experts of 2048) 16 tokens 35.5 us (39%); fp32 (d 712, 13 experts of 333) 5 tokens 27.7 us where the bytes
// take 5.3.  At one token some 13 us are not the stream's: launch (3), router (7, half of it under the
// shared expert's weights), the two GEMMs' border (3), the last rows (2).  (The pairs of times beside the rules below
// are those of the builds that the rules were chosen with; with fp8 weights those took 2 us less at one token and
// 6 us at 32, before the intermediate's copies and bounds described below.)
//
// A warp spends 150 to 400 instructions on a box, at one in eight clocks (three or four warps a scheduler,
// each waiting for its own last result); this, not the products, is what keeps it from DRAM speed.  Every form of the
// kernel takes the 128 registers a thread that 16 warps leave, and spills 28 to 114 bytes a thread beyond them
// (68 to 260 bytes read back).  So the boxes are as large as the shares allow; up to eight tokens, whose rows every
// unit multiplies in full, x stays in registers through GEMM1 and the sums through GEMM2; with more,
// an expert's few tokens are gathered for it, and units and tiles are 32 rows high where the rows are
// short enough, so that 32 rows share one gathering.
//
// Lane layout: lane (g, t) = (lane / 4, lane % 4) reads 16 bytes of weight rows g and g + 8 at offset
// 16 t of each 64-byte block, and the same positions of token g.  A dot product does not mind in
// which order its terms come, so these bytes go into the tensor core's operand registers as they
// are: the k index that the instruction thinks it sees is a permutation of the real one, the same
// for both operands.
//
// The intermediate is kept as two bf16 terms (16 significant bits; with fp32 weights in fp32, with fp8 weights
// as one f16 term, see below); everything is summed in fp32, the router in fp64 (bf16 products are exact in fp32, so
// the logits round correctly).
//
// fp8 weights go through f16: e4m3 converts to it exactly with one instruction a pair (to bf16 it
// takes four, which alone cost more than the weights' DRAM time).  A token row times a power of two
// that takes its largest value to [2^14, 2^15) is exact in f16 down to 2^-29 of that value.  The
// intermediate (one f16 term: it is off by 2^-11 at most where the output's bf16 is by 2^-9 and the weights'
// own rounding by 2^-4; with a second one, twice the loads and products of
// GEMM2, 32 tokens took 183 us instead of 153 and one took 31 instead of 27) needs a scale before it is known.  An
// e4m3 weight is 448 times its row's scale at most, so |h| <= B = max(s_gate s_up) (448 sum|x|)^2 (SwiGLU; max(s) 448
// sum|x| with ReLU), the maximum over the expert's channels, and 2^14 / B rounded down to a power of two cannot
// overflow.  The maxima are taken anew in every call, while the router runs: they go with whatever the scales hold
// then.  How far below the bound a row's values are depends on the weights (some 2^15 to 2^20 where all rows are
// alike, 2^40 and more where a few are much larger, or are all zeros and have the scale 1), so the intermediate is
// stored three times, each copy 2^20 times the one before (infinite where it overflows), and it is noted for each row
// whether its largest magnitude reaches 2^-9 in the first copy or in the second: GEMM2 reads the first copy in which
// it does, where every value has 11 significant bits or is off by 2^-16 of the row's largest, as long as that is at
// least 2^-58 of B (2^-63, and the exponents' rounding up takes some 2^4).  Mostly that is the first copy for all rows,
// as the values of an expert's first unit show already, and then nothing has to be looked up.
#include <type_traits>

#include "common.cuh"
#include "dsca_b200_block.h"

namespace dsca {
namespace few {

constexpr int kCompute = 12;              // compute warps 0 .. 11: they split every row along k
constexpr int kProducer = kCompute;       // first of the producer warps
constexpr int kProducers = 2;
constexpr int kService = kProducer + kProducers;  // first of the service warps
constexpr int kServices = 2;              // they run the router, then finish the units in turn
constexpr int kThreads = (kService + kServices) * 32;
constexpr int kMaxStages = 8;             // boxes of a compute warp's ring, at most
constexpr int kMaxBox = 384;              // bytes of a weight row in a box, at most
constexpr int kVals = 8;                  // 16-byte vectors of token values that a lane holds for a box
constexpr int kSmem = 227 * 1024;         // shared memory of a CTA
constexpr int kLgPitch = 64;              // logits of a token in the scratch: E + 1 <= 64
constexpr int kDotParts = 4;              // warps that share a logit's dot product
constexpr int kCopies = 3;                // of the intermediate, fp8 weights
constexpr int kCopyExp = 20;              // each is 2^20 times the one before

// words of the counter block
// kCtrBound + e: fp8 weights, 1 + the largest exponent (GLU: sum of the exponents) of the scales of expert e's channels,
// as they are stored (biased); e = E: the shared expert
// behind kCtrShared and kCtrRouted: fp8 weights, how many rows of that intermediate reach kReaches0 in their first unit
// (the first three are added to as pairs of words: nothing else lies in them)
enum { kCtrLogits = 0, kCtrShared = 2, kCtrRouted = 4, kCtrExit = 6, kCtrTiles = 8, kCtrBound = 128 };
static_assert(kCtrBound + DSCA_MAX_EXPERTS <= DSCA_FEW_ZERO_BYTES / 4, "counters are within the zeroed bytes");

struct Args {
  const void* x;
  const void* w_router;
  const void* w_gate;
  const uint8_t *w1, *w2, *ws1, *ws2;
  const float *w1s, *w2s, *ws1s, *ws2s;
  void* out;
  void* logits;
  int32_t* topk_ids;
  float* topk_w;
  int64_t* expert_index;
  double* lg;       // [T][64][4] parts of the logits, column E = shared gate
  uint8_t* x16;     // fp8 weights, more than eight tokens: [T][d] token rows in f16
  float* xmeta;     // and [T][2]: 1 / their scale, the largest power of two below sum|x|
  uint32_t* reach;  // fp8 weights: [T * k], then [T]: the sizes (h_reach) that values of a row of h / hs have
  uint8_t* h;       // [T * k][hp] intermediate: high terms, then the low terms; or fp32; or the f16 copies
  uint8_t* hs;      // [T][hsp] the shared expert's
  uint32_t* ctr;
  int32_t* err;
  int T, d, E, k, mode, norm_topk, glu;
  int n1p, ip, dp, s_ip;
  int inter, s_inter;     // channels of a routed expert / of the shared one
  int hp, hsp;            // row pitch of h / hs in values
  int upe, ups;           // units (16 or 32 weight rows of GEMM1) per routed expert / of the shared expert
  int k2, k2s;            // values of a row of w2 / ws2 that are read
  int b1, b2, b2s;        // values of a row in a box: GEMM1, routed and shared GEMM2
  int n1, n2, n2s;        // boxes of a row
  int n2_cta;             // boxes of a row of w2 for one of the CTAs that share a tile, rounded up
  int rt, tiles, splits;  // rows of a GEMM2 tile, tiles, CTAs that share one
  float* partial;         // their sums: [tiles * splits][tokens in eights][kSub2][32][4]
  int stage, stages;      // bytes of a stage, stages of a warp's ring
  uint64_t wait_ns;       // limit of every wait
};

struct Bf16 {
  using X = __nv_bfloat16;
  static constexpr int kSize = 1 << 1, kBlock = 32;  // bytes of a weight, weights in 64 bytes
};
struct F32 {
  using X = float;
  static constexpr int kSize = 4, kBlock = 16;
};
struct Fp8 {
  using X = __nv_bfloat16;
  static constexpr int kSize = 1, kBlock = 64;
};

// One box of a tensor map (weights of this GPU) into this CTA's shared memory.
__device__ __forceinline__ void box_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(policy)
      : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four e4m3 values -> two f16 pairs, exact
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)v));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(v >> 16)));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// 2^e
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// Exponent of the scale that takes a row whose largest magnitude has these bf16 bits to [2^14, 2^15),
// within what fp32 holds together with its inverse.
__device__ __forceinline__ int x_scale_exp(uint32_t max_bits) { return 141 - max(15, min(254, (int)(max_bits >> 7))); }
// Exponent of the scale of the intermediate's first copy (see the top): sum|x| < 2^(e + 1), bound: the expert's word
// at kCtrBound (a stored exponent x stands for less than 2^(x - 126), and 448 < 2^9).  At most 80, so that the
// last copy's inverse is a normal float.
__device__ __forceinline__ int h_scale_exp(int e, int bound, bool glu) {
  const int b = glu ? bound - 1 - 2 * 126 + 18 + 2 * (e + 1) : bound - 1 - 126 + 9 + e + 1;
  return max(-126, min(80, 14 - b));
}
// The sizes that a value of the first copy brings to its row (an infinity or a NaN brings both), and the copy to read
// of a row with these.
constexpr uint32_t kReaches0 = 1, kReaches1 = 2;
__device__ __forceinline__ uint32_t h_reach(float v) { return fabsf(v) < 0x1p-29f ? 0u : fabsf(v) < 0x1p-9f ? kReaches1 : kReaches0 | kReaches1; }
__device__ __forceinline__ int h_copy(uint32_t reach) { return reach & kReaches0 ? 0 : reach & kReaches1 ? 1 : 2; }
// the exponent of a non-negative float
__device__ __forceinline__ int exp_of(float v) { return (int)(__float_as_uint(v) >> 23) - 127; }
// eight bf16 values times s -> f16
__device__ __forceinline__ uint4 to_f16(uint4 u, float s) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = pack_f16x2(__uint_as_float(w[i] << 16) * s, __uint_as_float(w[i] & 0xffff0000u) * s);
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// the largest magnitude bits and the magnitudes' sum of eight bf16 values, joined to (m, l1)
__device__ __forceinline__ void magnitudes(uint4 u, uint32_t& m, float& l1) {
  const uint32_t w[4] = {u.x & 0x7fff7fffu, u.y & 0x7fff7fffu, u.z & 0x7fff7fffu, u.w & 0x7fff7fffu};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m = max(m, max(w[i] & 0xffffu, w[i] >> 16));
    l1 += __uint_as_float(w[i] << 16) + __uint_as_float(w[i] & 0xffff0000u);
  }
}

// whether the phase of this parity is complete, without waiting
__device__ __forceinline__ bool mbar_test_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint64_t ld_acquire(const uint32_t* p) {
  uint64_t v;
  asm volatile("ld.acquire.gpu.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
// The kernel's waits, every one bounded.  One that has run out records the error and raises the CTA's flag,
// after which every other wait of the CTA returns at its first look (false, unless what it waits for has come):
// each role then runs to its end on whatever it has, without another copy, and takes part in every barrier.
struct Waits {
  volatile int* abort;
  int32_t* err;
  uint64_t limit;  // nanoseconds
  __device__ __forceinline__ bool over(uint64_t t0) const {
    if (globaltimer_ns() - t0 <= limit) return false;
    record_error(err, kErrWaitTimeout);
    *abort = 1;
    return true;
  }
  // the phase of this parity of an mbarrier
  __device__ __forceinline__ bool bar(uint32_t b, uint32_t parity) const {
    if (mbar_test_wait(b, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t it = 1;; ++it) {
      if (*abort) return false;
      if (mbar_try_wait(b, parity)) return true;
      if ((it & 15u) == 0u && over(t0)) return false;
    }
  }
  // until *p has reached `target` (one thread; the counters only grow during a call); the word behind it at that
  // moment, 0 if the wait was given up.  As a signed distance: a workspace whose counter starts too low makes the
  // wait run out.
  __device__ __forceinline__ uint32_t counter(const uint32_t* p, uint32_t target) const {
    uint64_t v = ld_acquire(p);
    if ((int32_t)((uint32_t)v - target) >= 0) return (uint32_t)(v >> 32);
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t it = 1;; ++it) {
      v = ld_acquire(p);
      if ((int32_t)((uint32_t)v - target) >= 0) return (uint32_t)(v >> 32);
      if ((it & 15u) == 0u && (*abort || over(t0))) return 0u;
    }
  }
};
// n to *p, and `behind` to the word behind it
__device__ __forceinline__ void ctr_add(uint32_t* p, uint32_t n, uint32_t behind = 0u) {
  __threadfence();
  atomicAdd(reinterpret_cast<unsigned long long*>(p), (unsigned long long)behind << 32 | n);
}

// ---------------------------------------------------------------- shared memory
// What a kernel for up to 8 NT tokens does.  SUB: 16-row tiles of a GEMM1 unit.
template <typename W, int NT, int SUB>
struct Form {
  static constexpr bool kF32 = W::kSize == 4, kHalf = W::kSize == 1;
  // the tensor core's columns are the tokens of the call (else the tokens of the expert at hand)
  static constexpr bool kDirect = NT == 1 && !kF32;
  static constexpr int kSub2 = kDirect || kF32 ? 1 : 2;  // 16-row tiles of a GEMM2 tile
  static constexpr int kTerms = kHalf ? 1 : 2;           // of the intermediate (see the top)
  // tiles of eight tokens that a unit's sums are handed over in at a time
  static constexpr int kHand = SUB == 2 ? 1 : NT;
};

// Sums wait for their service warp in one of kParts buffers, one for each service warp: all compute warps
// take part in every handing over, so a warp that has seen number n knows the buffer's use before
// n + kParts to be complete (a parity wait cannot look two phases ahead).
constexpr int kParts = kServices;
template <typename W, int NT, int SUB>
struct Smem {
  using F = Form<W, NT, SUB>;
  union {
    float part[kParts][kCompute][F::kHand][SUB][32][4];
    float sums[F::kDirect ? 1 : kCompute][NT][F::kSub2][32][4];  // GEMM2, all tokens (not kDirect)
  };
  uint64_t full[kCompute][kMaxStages], empty[kCompute][kMaxStages];
  uint64_t part_full[kParts], part_empty[kParts];
  uint64_t routed;
  bool last;                                // this CTA's sums of a tile were the last to come
  float wt[8 * NT * DSCA_MAX_TOPK];         // routing weights by assignment
  float sg[8 * NT];                         // shared-expert gate
  float xinv[8 * NT];                       // fp8: 1 / scale of a token's row
  int xexp[8 * NT];                         // and the exponent of the sum of its magnitudes
  // fp8: which copy of a row of the intermediate is read: routed rows, then from kShared on tokens
  static constexpr int kShared = 8 * NT * DSCA_MAX_TOPK;
  uint8_t copy[F::kHalf ? kShared + 8 * NT : 1];
  float undo[F::kHalf && !F::kDirect ? kShared + 8 * NT : 1];  // and 1 / scale of its first copy
  uint32_t bound[F::kHalf ? DSCA_MAX_EXPERTS : 1];  // the words at kCtrBound
  uint32_t xmax[kCompute][8];               // fp8, up to eight tokens: a warp's share of a row
  float xsum[kCompute][8];
  uint32_t emask[DSCA_MAX_EXPERTS];         // tokens of an expert
  uint8_t act[DSCA_MAX_EXPERTS];            // experts with tokens ("active"), ascending
  // active expert i: its number, how many tokens it has (bits 8 ..), the compute warp that its first box
  // of GEMM2 goes to (bits 16 ..)
  uint32_t info[DSCA_MAX_EXPERTS];
  uint32_t mask[DSCA_MAX_EXPERTS];          // and which
  // Its n-th token, and that assignment: token * k + choice, the row of h (kDirect: that of token n).  Where there
  // is none, the first's: what is read for it is dropped.
  uint8_t tok[DSCA_MAX_EXPERTS][8 * NT];
  uint8_t asg[DSCA_MAX_EXPERTS][8 * NT];
  uint8_t slot[DSCA_MAX_EXPERTS][8 * NT];   // choice of (expert, token)
  int n_act;
  uint32_t handed;                          // routed units' handings over, all CTAs'
  uint32_t left[kCompute];                  // where a ring's producer ended: stage, its parity (bit 8), gone round (bit 9)
  int abort;
};

// ---------------------------------------------------------------- router
// a logit in the router's type, rounded by way of fp32 as a cast from fp64 is
template <typename X>
__device__ __forceinline__ float round_to(double v);
template <>
__device__ __forceinline__ float round_to<__nv_bfloat16>(double v) { return round_bf16((float)v); }
template <>
__device__ __forceinline__ float round_to<float>(double v) { return (float)v; }

// Part `part` of x . w over one warp in fp64, the same on every lane.  The code is short and the parts are
// small because a call runs it cold: instructions come from L2 at some 75 ns for eight of them, so 64
// products unrolled took 2.5 us where 16 take 0.7.
__device__ __forceinline__ void dot_add(double (&s)[4], uint4 a, uint4 b, const __nv_bfloat16*) {
  const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // products of two 8-bit significands are exact in fp32
    s[i] += (double)(__uint_as_float(av[i] << 16) * __uint_as_float(bv[i] << 16));
    s[i] += (double)(__uint_as_float(av[i] & 0xffff0000u) * __uint_as_float(bv[i] & 0xffff0000u));
  }
}
__device__ __forceinline__ void dot_add(double (&s)[4], uint4 a, uint4 b, const float*) {
  s[0] = fma((double)__uint_as_float(a.x), (double)__uint_as_float(b.x), s[0]);
  s[1] = fma((double)__uint_as_float(a.y), (double)__uint_as_float(b.y), s[1]);
  s[2] = fma((double)__uint_as_float(a.z), (double)__uint_as_float(b.z), s[2]);
  s[3] = fma((double)__uint_as_float(a.w), (double)__uint_as_float(b.w), s[3]);
}
template <typename X>
__device__ __forceinline__ double dot64(const X* x, const X* w, int d, int part, int parts, int lane) {
  constexpr int kVec = 16 / sizeof(X);
  const int step = 32 * parts * kVec;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 1
  for (int k = (part * 32 + lane) * kVec; k < d; k += 2 * step) {
    const bool more = k + step < d;
    const uint4 a0 = __ldg(reinterpret_cast<const uint4*>(x + k)), b0 = __ldg(reinterpret_cast<const uint4*>(w + k));
    const uint4 a1 = more ? __ldg(reinterpret_cast<const uint4*>(x + k + step)) : zero;
    const uint4 b1 = more ? __ldg(reinterpret_cast<const uint4*>(w + k + step)) : zero;
    dot_add(s, a0, b0, x);
    dot_add(s, a1, b1, x);
  }
  double r = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll 1
  for (int off = 16; off >= 1; off >>= 1) r += __shfl_xor_sync(0xffffffffu, r, off);
  return r;
}

__device__ __forceinline__ uint32_t ord_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float ord_val(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// Softmax and selection of one token by one warp (lane holds experts lane and lane + 32), with the
// arithmetic and the tie rule of dsca_router_topk.  Every CTA does it for itself; CTA 0 writes the
// results.  dry: nothing is read or written (the code only comes into the instruction cache, in the
// time that the logits of other CTAs take: see dot64).
template <typename X, typename S>
__device__ __forceinline__ void select_token(const Args& a, S& s, int t, int parts, bool dry, int lane) {
  const int E = a.E, e0 = lane, e1 = lane + 32;
  auto logit = [&](int e) {
    if (dry) return 0.0f;
    const double* q = a.lg + (size_t)(t * kLgPitch + e) * parts;
    if (parts == 1) return round_to<X>(__ldcg(q));
    const double2* p = reinterpret_cast<const double2*>(q);
    const double2 u = __ldcg(p), v = __ldcg(p + 1);
    return round_to<X>((u.x + u.y) + (v.x + v.y));
  };
  const float l0 = logit(e0), l1 = logit(e1);
  const bool v0 = e0 < E, v1 = e1 < E, first = blockIdx.x == 0 && !dry;
  if (a.x16 != nullptr && lane == 0 && !dry) {
    s.xinv[t] = __ldcg(a.xmeta + 2 * t);
    s.xexp[t] = exp_of(__ldcg(a.xmeta + 2 * t + 1));
  }
  if (a.w_gate != nullptr && (e0 == E || e1 == E) && !dry) s.sg[t] = 1.0f / (1.0f + expf(-(e0 == E ? l0 : l1)));
  if (first) {
    X* lo = reinterpret_cast<X*>(a.logits) + (size_t)t * E;
    if (v0) lo[e0] = X(l0);
    if (v1) lo[e1] = X(l1);
  }
  const uint32_t mk = __reduce_max_sync(0xffffffffu, max(v0 ? ord_key(l0) : 0u, v1 ? ord_key(l1) : 0u));
  const float m = ord_val(mk);
  const float x0 = v0 ? exp_neg(__fsub_rn(l0, m)) : 0.0f, x1 = v1 ? exp_neg(__fsub_rn(l1, m)) : 0.0f;
  float ps = __fadd_rn(x0, x1);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) ps = __fadd_rn(ps, __shfl_xor_sync(0xffffffffu, ps, off));
  float p0 = __fdiv_rn(x0, ps), p1 = __fdiv_rn(x1, ps);
  const bool top1 = a.mode == DSCA_ROUTE_SWITCH_TOP1;
  if (top1 && sizeof(X) == 2) {
    p0 = round_bf16(p0);
    p1 = round_bf16(p1);
  }
  float my_p = 0.0f, sum = 0.0f;
  int my_id = 0;
  bool taken0 = !v0, taken1 = !v1;
  for (int j = 0; j < a.k; ++j) {
    // probabilities are >= +0: their bits order like the values; 0 = no candidate
    const uint32_t k0 = taken0 ? 0u : __float_as_uint(p0) + 1u, k1 = taken1 ? 0u : __float_as_uint(p1) + 1u;
    const uint32_t best = __reduce_max_sync(0xffffffffu, max(k0, k1));
    const uint32_t cand = k0 == best ? (uint32_t)e0 : (k1 == best ? (uint32_t)e1 : 0xffffffffu);
    const int bi = (int)__reduce_min_sync(0xffffffffu, cand);
    const float bv = __uint_as_float(best - 1u);
    taken0 = taken0 || bi == e0;
    taken1 = taken1 || bi == e1;
    if (lane == j) {
      my_p = bv;
      my_id = bi;
    }
    sum = __fadd_rn(sum, bv);
  }
  if (lane < a.k && !dry) {
    float w = my_p;
    if (!top1) {
      if (a.norm_topk) w = __fdiv_rn(my_p, sum);
      if (sizeof(X) == 2) w = round_bf16(w);
    }
    s.wt[t * a.k + lane] = w;
    s.slot[my_id][t] = (uint8_t)lane;
    atomicOr(&s.emask[my_id], 1u << t);
    if (first) {
      a.topk_ids[(size_t)t * a.k + lane] = my_id;
      a.topk_w[(size_t)t * a.k + lane] = w;
      if (lane == 0 && a.expert_index != nullptr) a.expert_index[t] = my_id;
    }
  }
}

// ---------------------------------------------------------------- products of one stage
__device__ __forceinline__ uint4 ld_b(const uint8_t* p, bool live, bool coherent) {
  if (!live) return make_uint4(0u, 0u, 0u, 0u);
  const uint4* q = reinterpret_cast<const uint4*>(p);
  return coherent ? __ldcg(q) : *q;
}

// A lane's token values for a box of bf16 or e4m3 weights: vector (i, m, q) holds eight values of 64-byte
// block i, term m (0: x or the high term, 1: the low term), part q.
//   row: this lane's token row (token g) at the box's first k, lo: byte distance to its low terms,
//   live: values of that row from there on.
template <typename W, int kTerms>
struct Layout {
  static constexpr int kPer = W::kBlock < 32 ? 1 : W::kBlock / 32;  // vectors of a block and term
  static constexpr int kBlocks = kVals / (kPer * kTerms);           // blocks of a box, at most
  static __device__ __forceinline__ int at(int i, int m, int q) { return (i * kTerms + m) * kPer + q; }
};
// full: all nkb blocks of the box lie inside the row (the same on all lanes); a lane without a token is
// given some row whose values it may read.
template <typename W, int kTerms, bool kCoherent>
__device__ __forceinline__ void load_vals(uint4 (&v)[kVals], const uint8_t* row, size_t lo, bool full, int nkb, int live, int lane) {
  using L = Layout<W, kTerms>;
  const int t8 = (lane & 3) * 8 * L::kPer;
  live -= t8;
  const uint8_t* p = row + t8 * 2;
  const uint8_t* pl = p + lo;
  if (full) {
#pragma unroll
    for (int i = 0; i < L::kBlocks; ++i) {
      if (i >= nkb) break;
#pragma unroll
      for (int q = 0; q < L::kPer; ++q) {
        const int k = i * W::kBlock + q * 8;
        v[L::at(i, 0, q)] = ld_b(p + k * 2, true, kCoherent);
        if constexpr (kTerms == 2) v[L::at(i, 1, q)] = ld_b(pl + k * 2, true, kCoherent);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < L::kBlocks; ++i)
#pragma unroll
      for (int q = 0; q < L::kPer; ++q) {
        const int k = i * W::kBlock + q * 8;
        v[L::at(i, 0, q)] = ld_b(p + k * 2, k < live, kCoherent);
        if constexpr (kTerms == 2) v[L::at(i, 1, q)] = ld_b(pl + k * 2, k < live, kCoherent);
      }
  }
}
// acc += SUB x 16 weight rows x 8 tokens over the nkb 64-byte blocks of a box.  box: this lane's place in
// its row g of the first 16 in shared memory, up: bytes from there to row g + 8, sub: to the next 16
// rows.  Four chains of products (a tensor-core product waits some 30 clocks for the one whose sum
// it adds to), added at the end.
template <typename W, int kTerms, int SUB>
__device__ __forceinline__ void box_mma(float (&acc)[SUB][4], uint32_t box, int up, int sub, int nkb, const uint4 (&v)[kVals]) {
  using L = Layout<W, kTerms>;
  constexpr int kCh = 4 / SUB;  // chains of a 16-row tile
  float c[SUB][kCh][4];
#pragma unroll
  for (int r = 0; r < SUB; ++r)
#pragma unroll
    for (int q = 0; q < kCh; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[r][q][i] = 0.0f;
#pragma unroll
  for (int i = 0; i < L::kBlocks; ++i) {
    if (i >= nkb) break;
#pragma unroll
    for (int r = 0; r < SUB; ++r) {
      const uint4 a0 = lds128(box + r * sub + i * 64), a1 = lds128(box + r * sub + up + i * 64);
      if constexpr (W::kBlock == 32) {
#pragma unroll
        for (int m = 0; m < kTerms; ++m) {
          const uint4 b = v[L::at(i, m, 0)];
          const int q = (kTerms == 1 ? (i & 1) * 2 : m * 2);
          mma_bf16(c[r][q % kCh], a0.x, a1.x, a0.y, a1.y, b.x, b.y);
          mma_bf16(c[r][(q + 1) % kCh], a0.z, a1.z, a0.w, a1.w, b.z, b.w);
        }
      } else {
        const uint32_t w0[4] = {a0.x, a0.y, a0.z, a0.w}, w1[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t p0, p1, q0, q1;
          e4m3x4_to_f16(w0[j], p0, p1);
          e4m3x4_to_f16(w1[j], q0, q1);
#pragma unroll
          for (int m = 0; m < kTerms; ++m) {
            const uint4 b = v[L::at(i, m, j / 2)];
            mma_f16(c[r][(kTerms == 1 ? j : m * 2 + (j & 1)) % kCh], p0, q0, p1, q1, (j & 1) ? b.z : b.x, (j & 1) ? b.w : b.y);
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < SUB; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kCh == 4) acc[r][i] += (c[r][0][i] + c[r][1][i]) + (c[r][2][i] + c[r][3][i]);
      else acc[r][i] += c[r][0][i] + c[r][1][i];
    }
}

// The same for fp32 weights on the CUDA cores, two tokens at a time: lane (g, t) sums rows g and g + 8 over its k,
// then the four lanes of a row are added into the layout of the tensor-core accumulators.  row(n): token
// row n at the box's first k, n < tokens.  Few instructions count for more than few reads of the box: a warp
// has a handful of boxes, and with eight tokens' sums side by side it waited for the code.  d 712, 1 / 5 / 8 /
// 32 tokens: eight side by side 21.2 / 32 / 38 / 103 us, one at a time 17.2 / 27.8 / 38.2 / 94, two 17.9 /
// 27.3 / 33.2 / 79, two with code of its own for an odd last one 19.0 / 28.6 / 34.6 / 84.
template <bool kCoherent, typename Row>
__device__ __forceinline__ void box_fma(float (&acc)[4], uint32_t box, int up, int nkb, Row row, int tokens, int live, int lane) {
  constexpr int kMost = kMaxBox / 64;
  const int t = lane & 3;
  nkb = min(nkb, max(0, (live - t * 4 + 15) / 16));
#pragma unroll 1
  for (int n = 0; n < tokens; n += 2) {
    float4 v[2][kMost];
    float s[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // an odd last token twice: the column behind it is dropped
      const float4* x = reinterpret_cast<const float4*>(row(min(n + i, tokens - 1)) + t * 4);
#pragma unroll
      for (int kb = 0; kb < kMost; ++kb)
        if (kb < nkb) v[i][kb] = kCoherent ? __ldcg(x + kb * 4) : x[kb * 4];
      s[i][0] = s[i][1] = 0.0f;
    }
#pragma unroll
    for (int kb = 0; kb < kMost; ++kb) {
      if (kb >= nkb) break;
      const uint4 u[2] = {lds128(box + kb * 64), lds128(box + up + kb * 64)};
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          s[i][r] = fmaf(__uint_as_float(u[r].w), v[i][kb].w, fmaf(__uint_as_float(u[r].z), v[i][kb].z,
                    fmaf(__uint_as_float(u[r].y), v[i][kb].y, fmaf(__uint_as_float(u[r].x), v[i][kb].x, s[i][r]))));
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        s[i][r] += __shfl_xor_sync(0xffffffffu, s[i][r], 1);
        s[i][r] += __shfl_xor_sync(0xffffffffu, s[i][r], 2);
        if (t == n / 2) acc[2 * r + i] += s[i][r];
      }
  }
}

// ---------------------------------------------------------------- the kernel
__device__ __forceinline__ void group_sync(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }

__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 2, %0;" ::"n"(kCompute * 32) : "memory"); }

// Where the compute warps do not route: one of the routing warps announces their share of the bounds.
__device__ __forceinline__ void bounds_arrive() { asm volatile("bar.arrive 3, %0;" ::"n"((kCompute + 1) * 32) : "memory"); }
__device__ __forceinline__ void bounds_sync() { asm volatile("bar.sync 3, %0;" ::"n"((kCompute + 1) * 32) : "memory"); }

// fp8: this warp's share of the bounds of all experts (see kCtrBound), 256 rows of w1 at a time.  Scales that are not
// finite are left out: their channels' values are not finite whatever the scale.
__device__ __forceinline__ void find_bounds(const Args& a, int warp, int lane) {
  const int per = a.glu ? 128 : 256, ce = (a.inter + per - 1) / per, cs = (a.s_inter + per - 1) / per;
  auto exponent = [](float s) { return __float_as_uint(s) >> 23 & 255u; };
#pragma unroll 1
  for (int q = warp * gridDim.x + blockIdx.x; q < a.E * ce + cs; q += kCompute * gridDim.x) {
    const bool sh = q >= a.E * ce;
    const int e = sh ? a.E : q / ce, c = sh ? q - a.E * ce : q % ce, left = (sh ? a.s_inter : a.inter) - c * per;
    const float* sc = (sh ? a.ws1s : a.w1s + (size_t)e * a.n1p) + c * 256 + lane;
    uint32_t m = 0u;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __ldg(sc + 32 * i);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t x = exponent(v[i]), y = a.glu ? exponent(v[(i + 4) & 7]) : 0u;
      if ((!a.glu || i < 4) && lane + 32 * i < left && x != 255u && y != 255u) m = max(m, x + y + 1u);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) atomicMax(a.ctr + kCtrBound + e, m);
  }
}

__device__ __forceinline__ void add(float4& c, float4 o) {
  c.x += o.x; c.y += o.y; c.z += o.z; c.w += o.w;
}
// A lane's sums of a tile, the parts of its `splits` CTAs added in order.
__device__ __forceinline__ float4 tile_sum(const float* all, int splits, int pitch) {
  float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int v = 0; v < splits; ++v) add(r, __ldcg(reinterpret_cast<const float4*>(all + (size_t)v * pitch)));
  return r;
}
// A lane's sums of 16-row tile q and token tile nt of an output tile.
template <typename W>
__device__ __forceinline__ void store_out(const Args& a, float4 v, int tile, int nt, int q, int lane) {
  using X = typename W::X;
  const int r0 = tile * a.rt, rows = min(a.rt, a.d - r0);
  X* out = reinterpret_cast<X*>(a.out);
  const float c[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int tk = nt * 8 + 2 * (lane & 3) + (i & 1), rr = 16 * q + (lane >> 2) + (i >> 1) * 8;
    if (tk < a.T && rr < rows) out[(size_t)tk * a.d + r0 + rr] = X(c[i]);
  }
}

// Router: fp64 dot products spread over the grid, then softmax, selection and the expert lists in every
// CTA for itself.  Warp wi of the nw warps that take part (they share named barrier 1).
template <typename X, int SUB, int kTokens, bool kDirect, bool kHalf, typename S>
__device__ __forceinline__ void route(const Args& a, S& s, const Waits& waits, int wi, int nw, int lane) {
  const int G = gridDim.x, cta = blockIdx.x;
  // a logit's product in four parts while that leaves a warp one (one token of the Qwen block 32.7 us, whole
  // 34.6), else whole (32 tokens with fp8 weights 130 us, four parts 133)
  const int R = a.E + (a.w_gate != nullptr ? 1 : 0), parts = a.T * R * kDotParts <= nw * G ? kDotParts : 1;
  const int nd = a.T * R * parts;
#pragma unroll 1
  for (int q = cta + wi * G; q < nd; q += nw * G) {
    const int part = q % parts, t = q / parts / R, r = q / parts % R;
    const X* w = r < a.E ? reinterpret_cast<const X*>(a.w_router) + (size_t)r * a.d : reinterpret_cast<const X*>(a.w_gate);
    const double v = dot64(reinterpret_cast<const X*>(a.x) + (size_t)t * a.d, w, a.d, part, parts, lane);
    if (lane == 0) a.lg[(size_t)(t * kLgPitch + r) * parts + part] = v;
  }
  if (kHalf && cta == 0)
    for (int r = wi * 32 + lane; r < a.T * (a.k + 1); r += nw * 32) a.reach[r] = 0u;
  // fp8 weights, more than eight tokens: the t-th last CTA (the first have one dot product
  // more) writes token t's row in f16 (eight or less: the compute warps convert what they keep of it)
  const int counted = kHalf ? G : min(nd, G);  // CTAs that have a part in this
  for (int tc = G - 1 - cta; a.x16 != nullptr && wi == nw - 1 && tc < a.T; tc += G) {
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const X*>(a.x) + (size_t)tc * a.d);
    uint4* dst = reinterpret_cast<uint4*>(a.x16) + (size_t)tc * (a.d / 8);
    uint32_t m = 0u;
    float l1 = 0.0f;
#pragma unroll 4
    for (int c = lane; c < a.d / 8; c += 32) magnitudes(__ldg(src + c), m, l1);
    m = __reduce_max_sync(0xffffffffu, m);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    const int e = x_scale_exp(m);
#pragma unroll 4
    for (int c = lane; c < a.d / 8; c += 32) dst[c] = to_f16(__ldg(src + c), pow2(e));
    if (lane == 0) {
      a.xmeta[2 * tc] = pow2(-e);
      a.xmeta[2 * tc + 1] = l1;
    }
  }
  group_sync(nw * 32);
  if (kHalf && wi == 0 && nw == kServices) bounds_sync();
  if (wi == 0 && lane == 0 && cta < counted) ctr_add(a.ctr + kCtrLogits, 1u);
  __syncwarp();
  for (int t = wi - nw; t < a.T; t += nw) {
    if (t >= 0 && t < nw) {
      if (wi == 0 && lane == 0) waits.counter(a.ctr + kCtrLogits, (uint32_t)counted);
      __syncwarp();
      group_sync(nw * 32);
    }
    select_token<X>(a, s, max(t, 0), parts, t < 0, lane);
  }
  if (wi >= a.T) {  // no token for this warp: the same barrier
    group_sync(nw * 32);
  }
  group_sync(nw * 32);
  if constexpr (kHalf) {
    if (wi == nw - 1) {
      s.bound[lane] = __ldcg(a.ctr + kCtrBound + lane);
      s.bound[lane + 32] = __ldcg(a.ctr + kCtrBound + lane + 32);
    }
  }
  if (wi == 0) {
    const uint32_t m0 = s.emask[lane], m1 = s.emask[lane + 32];
    const uint32_t b0 = __ballot_sync(0xffffffffu, m0 != 0u), b1 = __ballot_sync(0xffffffffu, m1 != 0u);
    const uint32_t below = (1u << lane) - 1u;
    if (m0) s.act[__popc(b0 & below)] = (uint8_t)lane;
    if (m1) s.act[__popc(b0) + __popc(b1 & below)] = (uint8_t)(lane + 32);
    // handings over of an expert's unit: one, or one for each eight of its tokens
    const uint32_t h0 = m0 == 0u ? 0u : (SUB == 2 ? (__popc(m0) + 7u) / 8u : 1u);
    const uint32_t h1 = m1 == 0u ? 0u : (SUB == 2 ? (__popc(m1) + 7u) / 8u : 1u);
    const uint32_t handed = __reduce_add_sync(0xffffffffu, h0 + h1) * (uint32_t)a.upe;
    if (lane == 0) {
      s.n_act = __popc(b0) + __popc(b1);
      s.handed = handed;
    }
  }
  group_sync(nw * 32);
  if constexpr (kHalf && !kDirect)
    if (wi == 0 && lane < a.T && a.w_gate != nullptr)
      s.undo[S::kShared + lane] = pow2(-h_scale_exp(s.xexp[lane], (int)s.bound[a.E], a.glu));
  for (int i = wi; i < s.n_act; i += nw) {
    const int e = s.act[i];
    const uint32_t m = s.emask[e];
    if (lane == 0) {
      s.mask[i] = m;
      s.info[i] = (uint32_t)e | (uint32_t)__popc(m) << 8 | (uint32_t)(e * a.n2_cta % kCompute) << 16;
    }
    const uint32_t below = (1u << lane) - 1u;
    const bool on = (m >> lane) & 1u;
    const int t = on ? lane : __ffs(m) - 1;
    const int n = kDirect ? lane : (on ? __popc(m & below) : __popc(m) + __popc(~m & below));
    if (n < kTokens) {
      s.tok[i][n] = (uint8_t)t;
      s.asg[i][n] = (uint8_t)(t * a.k + s.slot[e][t]);
      if constexpr (kHalf && !kDirect)
        if (on) s.undo[s.asg[i][n]] = pow2(-h_scale_exp(s.xexp[t], (int)s.bound[e], a.glu));
    }
  }
  group_sync(nw * 32);
  if (wi == 0 && lane == 0) mbar_arrive(smem_u32(&s.routed));
}

template <typename W, int NT, int SUB>
__global__ void __launch_bounds__(kThreads, 1)
    moe_few_kernel(const Args a, const __grid_constant__ CUtensorMap m1, const __grid_constant__ CUtensorMap m2,
                   const __grid_constant__ CUtensorMap ms1, const __grid_constant__ CUtensorMap ms2) {
  using X = typename W::X;
  using F = Form<W, NT, SUB>;
  constexpr bool kF32 = F::kF32, kHalf = F::kHalf, kDirect = F::kDirect;
  constexpr int kSub2 = F::kSub2, kHand = F::kHand, kTerms = F::kTerms;
  static_assert(SUB == 1 || !kDirect, "units of 32 rows are for gathered tokens");
  extern __shared__ __align__(128) uint8_t smem_raw[];
  using S = Smem<W, NT, SUB>;
  S& s = *reinterpret_cast<S*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int G = gridDim.x, cta = blockIdx.x;
  const uint32_t ring = smem_u32(smem_raw) + (uint32_t)((sizeof(S) + 127) / 128 * 128);
  volatile int* abort_flag = &s.abort;
  const Waits waits{abort_flag, a.err, a.wait_ns};

  if (threadIdx.x < kCompute * kMaxStages) {
    mbar_init(smem_u32(&s.full[0][0] + threadIdx.x), 1);
    mbar_init(smem_u32(&s.empty[0][0] + threadIdx.x), 1);
  }
  if (threadIdx.x < kParts) {
    mbar_init(smem_u32(&s.part_full[threadIdx.x]), kCompute);
    mbar_init(smem_u32(&s.part_empty[threadIdx.x]), 1);
  }
  if (threadIdx.x >= 128 && threadIdx.x < 128 + DSCA_MAX_EXPERTS) s.emask[threadIdx.x - 128] = 0u;
  if constexpr (kHalf)
    for (int i = threadIdx.x; i < (int)sizeof(s.copy); i += kThreads) s.copy[i] = 0;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&s.routed), 1);
    s.abort = 0;
    s.n_act = 0;
  }
  fence_mbar_init();
  __syncthreads();

  // ---- this CTA's work.  GEMM1: units cta, cta + G, ... of the shared expert, then consecutive units of the
  // routed experts, mostly of one expert, so that its tokens' values stay in registers (32 tokens, fp8: 140 us
  // against 147 with units G apart); the CTAs with one more of these are the last, those with one more of the
  // former the first.  GEMM2: items cta, cta + G,
  // ... : tile item / splits of the output's rows, and of each of its rows the boxes j with j mod splits =
  // item mod splits, first the shared expert's row, then the active experts'.  In GEMM1 box j goes to
  // compute warp j mod 12; in GEMM2 they count on from expert to expert (all experts, active or not: a
  // token's sums do not depend on the other tokens of the call).
  const int nu_s = a.ups > cta ? (a.ups - cta + G - 1) / G : 0;
  const int items = a.tiles * a.splits;
  auto routed_units = [&](int n_act) {
    const int units = n_act * a.upe, more = cta - (G - units % G);
    return int2{cta * (units / G) + max(0, more), units / G + (more >= 0)};  // the first of them, and how many
  };
  // Waits for the lists of experts (a whole warp); how many experts have tokens.  None where a lane's wait was given
  // up: nothing of the lists is read then, as they may not be there.
  auto wait_routed = [&]() {
    const bool there = waits.bar(smem_u32(&s.routed), 0u);
    return __all_sync(0xffffffffu, there) ? s.n_act : 0;
  };
  // warp w's first box (of this item's) of an active expert
  auto first_box = [&](int w, uint32_t info) {
    const int b = w - (int)(info >> 16);
    return b < 0 ? b + kCompute : b;
  };
  // The router runs on the service warps while the compute warps begin with the shared expert; on all
  // of them where there is no shared expert to begin with, or where the tokens are more than two
  // warps would do in the time of the first boxes (two warps, all: one token 32.7 us, 35.6; eight 103.6, 97.1;
  // 32 with fp8 weights 167, 132).
  const bool all_route = a.ups == 0 || a.T > 4;
  const int route_warps = all_route ? kCompute + kServices : kServices;

  if (warp >= kProducer && warp < kService) {
    // ================================================================ producers: one lane a ring
    // The lanes stay together (a lane that waits alone holds up the others of its warp), so a ring gets
    // its next box when the rings of all six have room.
    constexpr int kLanes = kCompute / kProducers;
    // every weight is read once, and leaves room in L2 for the code, the intermediates and the rows that are read
    // again (Qwen block, 8 tokens in bf16 97.5 us, so 92.3; 32 with fp8 weights 136.5, 131)
    const uint64_t once = l2_policy_evict_first();
    const bool on = lane < kLanes;
    const int w = (warp - kProducer) * kLanes + (on ? lane : 0);
    const uint32_t base = ring + (uint32_t)(w * a.stages * a.stage);
    int st = 0, last = -1;  // next stage, stage before it
    uint32_t phase = 0u;    // parity of the next stage's copy
    // While two warps route, one box a ring in flight: the router's loads queue behind them in DRAM (one token in
    // bf16 31.5 us, full rings 32.5).  Where all warps do, the rings fill at once.
    bool shallow = !all_route, wrapped = false, stop = false;
    // A box for this lane's ring, if there is one: load(bar, dst) once its stage is free.  one (only before
    // the routing is known, a constant elsewhere): not before the last one has come.
    auto box = [&](auto one, bool there, int bytes, auto load) {
      if (stop) return;
      const uint32_t e = smem_u32(&s.empty[w][st]), f = smem_u32(&s.full[w][max(last, 0)]);
      const bool we = there && wrapped, wf = there && one && last >= 0;
      uint64_t since = 0u;
      for (uint32_t it = 0;; ++it) {
        const bool ok = (!we || mbar_try_wait(e, phase ^ 1u)) && (!wf || mbar_try_wait(f, st == 0 ? phase ^ 1u : phase));
        if (__all_sync(0xffffffffu, ok && *abort_flag == 0)) break;
        if (lane == 0 && (it & 63u) == 63u) {
          const uint64_t now = globaltimer_ns();
          if (since == 0u) since = now;
          waits.over(since);
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, *abort_flag != 0)) {
          stop = true;
          break;
        }
      }
      if (there && !stop) {
        const uint32_t bar = smem_u32(&s.full[w][st]);
        mbar_arrive_expect_tx(bar, (uint32_t)bytes);
        load(bar, base + (uint32_t)(st * a.stage));
        last = st;
        if (++st == a.stages) {
          st = 0;
          phase ^= 1u;
          wrapped = true;
        }
      }
      __syncwarp();
    };
    int n_act = 0, nu_r = 0, r = 0, ai = 0, first = 0;
    for (int ul = 0; ul < nu_s + nu_r || ul == nu_s; ++ul) {
      const bool sh = ul < nu_s;
      if (ul == nu_s) {
        n_act = wait_routed();
        shallow = false;
        const int2 ru = routed_units(n_act);
        r = ru.x;
        nu_r = ru.y;
        if (nu_r == 0) break;
      }
      if (!sh) {
        if (ul > nu_s) ++r;
        while (r >= first + a.upe) {
          first += a.upe;
          ++ai;
        }
      }
      const int u = sh ? cta + ul * G : r - first, e = sh ? 0 : s.act[ai];
      const CUtensorMap* m = sh ? &ms1 : &m1;
      for (int j0 = 0; j0 < a.n1; j0 += kCompute) {
        const int j = j0 + w;
        box(shallow, on && j < a.n1, 16 * SUB * a.b1 * W::kSize, [&](uint32_t bar, uint32_t dst) {
          if (a.glu) box_load_4d(dst, m, bar, j * a.b1, 8 * SUB * u % 128, 0, e * (a.n1p / 256) + 8 * SUB * u / 128, once);
          else tma_load_2d_hint(dst, m, bar, j * a.b1, e * a.n1p + 16 * SUB * u, once);
        });
      }
    }
    for (int item = cta; item < items; item += G) {
      const int tile = item / a.splits, split = item % a.splits, per = kCompute * a.splits;
      for (int j0 = 0; j0 < a.n2s; j0 += per) {
        const int j = j0 + w * a.splits + split;
        box(std::false_type{}, on && j < a.n2s, a.rt * a.b2s * W::kSize,
            [&](uint32_t bar, uint32_t dst) { tma_load_2d_hint(dst, &ms2, bar, j * a.b2s, tile * a.rt, once); });
      }
      for (int i = 0; i < n_act; ++i) {
        const uint32_t info = s.info[i];
        const int e = info & 255u, fb = first_box(w, info);
        for (int j0 = 0; j0 < a.n2; j0 += per) {
          const int j = j0 + fb * a.splits + split;
          box(std::false_type{}, on && j < a.n2, a.rt * a.b2 * W::kSize,
              [&](uint32_t bar, uint32_t dst) { tma_load_2d_hint(dst, &m2, bar, j * a.b2, e * a.dp + tile * a.rt, once); });
        }
      }
    }
    if (on) s.left[w] = (uint32_t)st | phase << 8 | (uint32_t)wrapped << 9;
  } else if (warp < kCompute) {
    // ================================================================ compute
    if (kHalf && all_route) find_bounds(a, warp, lane);
    if (all_route) route<X, SUB, 8 * NT, kDirect, kHalf>(a, s, waits, kServices + warp, route_warps, lane);
    const uint32_t base = ring + (uint32_t)(warp * a.stages * a.stage);
    int st = 0, given = 0;  // next stage, sums handed over
    uint32_t phase = 0u;    // parity of the next stage's copy
    // the next box (then = 0) or the one behind it
    auto stage_of = [&](int then) { return st + then < a.stages ? st + then : 0; };
    auto box = [&](int pitch, int then = 0) { return base + (uint32_t)(stage_of(then) * a.stage + g * pitch + t4 * 16); };
    auto arrived = [&](int then = 0) {
      waits.bar(smem_u32(&s.full[warp][stage_of(then)]), st + then < a.stages ? phase : phase ^ 1u);
    };
    auto release = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s.empty[warp][st]));
      if (++st == a.stages) {
        st = 0;
        phase ^= 1u;
      }
    };
    // until the sums handed over as number n have been read
    auto wait_read = [&](int n) { waits.bar(smem_u32(&s.part_empty[n % kParts]), (uint32_t)(n / kParts) & 1u); };
    // this warp's part of the next buffer, free to be written
    auto buffer = [&]() {
      if (given >= kParts) wait_read(given - kParts);
      return &s.part[given % kParts][warp][0][0][0][0];
    };
    auto hand_over = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s.part_full[given % kParts]));
      ++given;
    };
    const int pitch1 = a.b1 * W::kSize, blk1 = a.b1 / W::kBlock, blk2 = a.b2 / W::kBlock, blk2s = a.b2s / W::kBlock;
    // GEMM1: from weight row g of a 16-row tile to row g + 8, and to the next tile
    const int up1 = (a.glu ? 8 * SUB : 8) * pitch1, sub1 = (a.glu ? 8 : 16) * pitch1;

    // ---- GEMM1
    // With kDirect a warp whose boxes of a row are one or two multiplies the same values in every unit
    // and keeps them.
    const bool keep = kDirect && a.n1 <= 2 * kCompute;
    uint4 va[kVals], vb[kVals];  // token values of the present and the next box, in turn
    bool ready = false;          // whether the next box's are on their way
    bool flip = false;           // and whether they are in vb
    // row n of active expert i's tokens (i < 0: of all) from k on; one of them where there is no such token
    auto x_row = [&](int i, int n_tok, int n, int k) {
      if (i < 0) n = min(n, n_tok - 1);
      return reinterpret_cast<const uint8_t*>(kHalf && !kDirect ? a.x16 : a.x) +
             ((size_t)(i < 0 ? n : (int)s.tok[i][n]) * a.d + k) * sizeof(X);
    };
    auto load_x = [&](uint4 (&v)[kVals], int i, int n_tok, int n, int k) {
      if constexpr (kDirect) {
        i = -1;
        n_tok = a.T;
      }
      load_vals<W, 1, false>(v, x_row(i, n_tok, n + g, k), 0, k + a.b1 <= a.d, blk1, a.d - k, lane);
    };
    if constexpr (kDirect) {
      if (keep) {
        if (warp < a.n1) load_x(va, -1, a.T, 0, warp * a.b1);
        if (warp + kCompute < a.n1) load_x(vb, -1, a.T, 0, (warp + kCompute) * a.b1);
      }
    }
    // behind the loads of x, which take as long
    if constexpr (kHalf) {
      if (!all_route) {
        find_bounds(a, warp, lane);
        bounds_arrive();
      }
    }
    float xs = 1.0f;  // the scale of token g's row
    auto halve = [&](uint4 (&v)[kVals]) {
#pragma unroll
      for (int i = 0; i < kVals; ++i) v[i] = to_f16(v[i], xs);
    };
    if constexpr (kDirect && kHalf) {
      // largest magnitude and sum of the magnitudes of token g's row: this warp's boxes, then all warps'
      uint32_t m = 0u;
      float l1 = 0.0f;
      for (int j = warp; j < a.n1; j += kCompute) {
        auto join = [&](const uint4 (&v)[kVals]) {
#pragma unroll
          for (int i = 0; i < kVals; ++i)
            if (i / 2 < blk1) magnitudes(v[i], m, l1);
        };
        if (keep) {
          if (j == warp) join(va);
          else join(vb);
        } else {
          uint4 v[kVals];
          load_x(v, -1, a.T, 0, j * a.b1);
          join(v);
        }
      }
#pragma unroll
      for (int off = 1; off <= 2; off <<= 1) {
        m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
      }
      if (t4 == 0) {
        s.xmax[warp][g] = m;
        s.xsum[warp][g] = l1;
      }
      compute_sync();
      m = 0u;
      l1 = 0.0f;
#pragma unroll
      for (int w = 0; w < kCompute; ++w) {
        m = max(m, s.xmax[w][g]);
        l1 += s.xsum[w][g];
      }
      const int e = x_scale_exp(m);
      xs = pow2(e);
      if (t4 == 0) {  // the same in every warp, which reads its own in GEMM2
        s.xinv[g] = pow2(-e);
        s.xexp[g] = exp_of(l1);
      }
      __syncwarp();
      if (keep) {
        halve(va);
        halve(vb);
      }
    }
    int holds = -1;  // active expert whose values are in va and vb
    int n_act = 0;                 // active experts
    int nu_r = 0, ai = -1, r = 0;  // routed units of this CTA; active expert and number of the present one
    for (int ul = 0; ul < nu_s + nu_r || ul == nu_s; ++ul) {
      if (ul == nu_s) {
        n_act = wait_routed();
        const int2 ru = routed_units(n_act);
        r = ru.x;
        nu_r = ru.y;
        if (nu_r == 0) break;
        ai = r / a.upe;
        ready = false;
      } else if (ul > nu_s) {
        ++r;
        if (r == (ai + 1) * a.upe) ++ai;
      }
      const int n_tok = ai < 0 ? a.T : (int)(s.info[ai] >> 8 & 255u);
      // asks for the values of the next unit's first box of this warp, if that unit is known
      auto ahead = [&](uint4 (&w)[kVals]) {
        if (ul + 1 < (ai < 0 ? nu_s : nu_s + nu_r)) {
          const int i = ai >= 0 && r + 1 == (ai + 1) * a.upe ? ai + 1 : ai;
          load_x(w, i, i < 0 ? a.T : (int)(s.info[i] >> 8 & 255u), 0, warp * a.b1);
          ready = true;
        }
      };
      if constexpr (SUB == 2) {
        // one box a warp and unit; the expert's tokens eight at a time
        const bool stay = n_tok <= 8 && ai >= 0 && ul + 1 < nu_s + nu_r && r + 1 < (ai + 1) * a.upe;
        const bool has = warp < a.n1;
        auto group = [&](int n0, uint4 (&v)[kVals], uint4 (&w)[kVals]) {
          const bool last = n0 + 8 >= n_tok;
          float acc[SUB][4];
#pragma unroll
          for (int q = 0; q < SUB; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[q][i] = 0.0f;
          if (has) {
            if (!ready) load_x(v, ai, n_tok, n0, warp * a.b1);
            // the same values again, if the next unit is of the same expert
            ready = !last || stay;
            if (!last) load_x(w, ai, n_tok, n0 + 8, warp * a.b1);
            else if (!stay) ahead(w);
            if (n0 == 0) arrived();
            box_mma<W, 1, SUB>(acc, box(pitch1), up1, sub1, blk1, v);
            if (last) release();
          }
          float* p = buffer();
          if (has) {
#pragma unroll
            for (int q = 0; q < SUB; ++q)
              *reinterpret_cast<float4*>(p + (q * 32 + lane) * 4) = make_float4(acc[q][0], acc[q][1], acc[q][2], acc[q][3]);
          }
          hand_over();
          if (!last || !stay) flip = !flip;
        };
        // two boxes a warp and unit, values of the first in va and of the second in vb: either's next ones are
        // asked for as soon as it is multiplied
        auto pair = [&](int n0) {
          const bool last = n0 + 8 >= n_tok, two = warp + kCompute < a.n1;
          const int i2 = last && ai >= 0 && r + 1 == (ai + 1) * a.upe ? ai + 1 : ai, n2 = last ? 0 : n0 + 8;
          const bool more = !last || ul + 1 < (ai < 0 ? nu_s : nu_s + nu_r), same = last && stay;
          const int tok2 = !more || i2 < 0 ? a.T : (int)(s.info[i2] >> 8 & 255u);
          float acc[SUB][4];
#pragma unroll
          for (int q = 0; q < SUB; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[q][i] = 0.0f;
          if (!ready) {
            load_x(va, ai, n_tok, n0, warp * a.b1);
            if (two) load_x(vb, ai, n_tok, n0, (warp + kCompute) * a.b1);
          }
          if (n0 == 0) arrived();
          box_mma<W, 1, SUB>(acc, box(pitch1), up1, sub1, blk1, va);
          if (more && !same) load_x(va, i2, tok2, n2, warp * a.b1);
          if (two) {
            if (n0 == 0) arrived(1);
            box_mma<W, 1, SUB>(acc, box(pitch1, 1), up1, sub1, blk1, vb);
            if (more && !same) load_x(vb, i2, tok2, n2, (warp + kCompute) * a.b1);
          }
          ready = more;
          if (last) {
            release();
            if (two) release();
          }
          float* p = buffer();
#pragma unroll
          for (int q = 0; q < SUB; ++q)
            *reinterpret_cast<float4*>(p + (q * 32 + lane) * 4) = make_float4(acc[q][0], acc[q][1], acc[q][2], acc[q][3]);
          hand_over();
        };
        if (a.n1 > kCompute) {
          for (int n0 = 0; n0 < n_tok; n0 += 8) pair(n0);
        } else {
          for (int n0 = 0; n0 < n_tok; n0 += 8) {
            if (flip) group(n0, vb, va);
            else group(n0, va, vb);
          }
        }
      } else {
        float acc[NT][1][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][0][i] = 0.0f;
        // box j, whose token values are in v (or not yet asked for); the next box's go to w
        auto step = [&](int j, uint4 (&v)[kVals], uint4 (&w)[kVals]) {
          const int k = j * a.b1;
          if constexpr (kF32) {
            arrived();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (nt * 8 >= n_tok) break;
              auto row = [&](int n) { return reinterpret_cast<const float*>(x_row(ai, n_tok, nt * 8 + n, k)); };
              box_fma<false>(acc[nt][0], box(pitch1), up1, blk1, row, min(8, n_tok - nt * 8), a.d - k, lane);
            }
          } else {
            if (!ready) load_x(v, ai, n_tok, 0, k);
            ready = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (nt * 8 >= n_tok) break;
              uint4(&now)[kVals] = nt % 2 == 0 ? v : w;
              uint4(&then)[kVals] = nt % 2 == 0 ? w : v;
              if (nt * 8 + 8 < n_tok) {
                load_x(then, ai, n_tok, nt * 8 + 8, k);
              } else if (j + kCompute < a.n1) {
                load_x(then, ai, n_tok, 0, k + kCompute * a.b1);
                ready = true;
              } else {
                ahead(then);
              }
              if (nt == 0) arrived();
              if constexpr (kDirect && kHalf) halve(now);
              box_mma<W, 1, 1>(acc[nt], box(pitch1), up1, 0, blk1, now);
              flip = !flip;
            }
          }
          release();
        };
        // the boxes of an expert's unit, the same values again in the next one (16 tokens of a
        // block of 2560 in bf16 171 us; asked for anew 180)
        bool held = keep;
        if constexpr (!kDirect && !kF32) {
          held = ai >= 0 && n_tok <= 8 && a.n1 <= 2 * kCompute;
          if (held && ai != holds) {
            if (warp < a.n1) load_x(va, ai, n_tok, 0, warp * a.b1);
            if (warp + kCompute < a.n1) load_x(vb, ai, n_tok, 0, (warp + kCompute) * a.b1);
          }
          holds = held ? ai : -1;
          ready = ready && !held;
        }
        if (held) {
          if (warp < a.n1) {
            arrived();
            box_mma<W, 1, 1>(acc[0], box(pitch1), up1, 0, blk1, va);
            release();
          }
          if (warp + kCompute < a.n1) {
            arrived();
            box_mma<W, 1, 1>(acc[0], box(pitch1), up1, 0, blk1, vb);
            release();
          }
        } else {
          for (int j = warp; j < a.n1; j += kCompute) {
            if (flip) step(j, vb, va);
            else step(j, va, vb);
          }
        }
        float* p = buffer();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          if ((kDirect || nt * 8 < n_tok) && warp < a.n1)
            *reinterpret_cast<float4*>(p + (nt * 32 + lane) * 4) =
                make_float4(acc[nt][0][0], acc[nt][0][1], acc[nt][0][2], acc[nt][0][3]);
        hand_over();
      }
    }

    // ---- GEMM2: segment -1 of an item is the shared expert's row, segment i active expert i's.  With
    // kDirect a token without the expert reads another one's row and its column is dropped, and the sums
    // of all experts stay in registers.  Else the columns are the expert's own tokens, and a box's sums
    // join the warp's sums of all tokens in shared memory (a lane's values have places of their own).
    const size_t h_lo = (size_t)a.T * a.k * a.hp * 2, hs_lo = (size_t)a.T * a.hsp * 2;
    bool have_s = false, have_r = false;  // the intermediates, which come from every CTA's service warps
    bool mixed = false;                   // fp8: not all rows of them are read from their first copy
    auto h_at = [&](int i, int n, int k) {
      int row = i < 0 ? n : s.asg[i][n];
      if constexpr (kHalf)
        if (mixed) row += s.copy[(i < 0 ? S::kShared : 0) + row] * (i < 0 ? a.T : a.T * a.k);
      return (i < 0 ? a.hs : a.h) + ((size_t)row * (i < 0 ? a.hsp : a.hp) + k) * (kF32 ? 4 : 2);
    };
    // fp8: the copy to read of each row of the (complete) shared or routed intermediate, where not all are known to be the
    // first.  Every warp writes the same for itself.
    auto choose_copies = [&](bool sh) {
#pragma unroll 1
      for (int r = lane; r < (sh ? a.T : a.T * a.k); r += 32)
        s.copy[(sh ? S::kShared : 0) + r] = (uint8_t)h_copy(__ldcg(a.reach + (sh ? a.T * a.k : 0) + r));
      __syncwarp();
    };
    auto load_h = [&](uint4 (&v)[kVals], int i, int n, int k) {
      const int kend = i < 0 ? a.k2s : a.k2, bk = i < 0 ? a.b2s : a.b2;
      const uint8_t* row = h_at(i, i < 0 ? min(n + g, a.T - 1) : n + g, k);
      load_vals<W, kTerms, true>(v, row, i < 0 ? hs_lo : h_lo, k + bk <= kend, i < 0 ? blk2s : blk2, kend - k, lane);
    };
    for (int item = cta; item < items; item += G) {
      const int tile = item / a.splits, split = item % a.splits, per = kCompute * a.splits;
      // this warp's first box at or behind (segment i, box j)
      auto seek = [&](int& i, int& j, uint32_t& info) {
        while (i < n_act && j >= (i < 0 ? a.n2s : a.n2)) {
          ++i;
          if (i < n_act) {
            info = s.info[i];
            j = first_box(warp, info) * a.splits + split;
          }
        }
      };
      const int r0 = tile * a.rt, rows = min(a.rt, a.d - r0);
      float* p;
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (kDirect) {
        p = buffer();
      } else {
        // the sums lie over all the buffers
        p = &s.sums[warp][0][0][0][0];
        for (int n = max(0, given - kParts); n < given; ++n) wait_read(n);
#pragma unroll
        for (int q = 0; q < NT * kSub2; ++q)
          *reinterpret_cast<float4*>(p + (q * 32 + lane) * 4) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        __syncwarp();
      }
      ready = false;
      int i = -1, j = warp * a.splits + split, n0 = 0;  // the tokens eight at a time
      uint32_t info = 0u;
      seek(i, j, info);
      auto step = [&](uint4 (&v)[kVals], uint4 (&w)[kVals]) {
        const bool sh = i < 0;
        const int bk = sh ? a.b2s : a.b2, pitch = bk * W::kSize, blk = sh ? blk2s : blk2, k = j * bk;
        if (sh ? !have_s : !have_r) {
          uint32_t reached = 0u;
          if (lane == 0)
            reached = sh ? waits.counter(a.ctr + kCtrShared, (uint32_t)(a.ups * (SUB == 2 ? (a.T + 7) / 8 : 1)))
                         : waits.counter(a.ctr + kCtrRouted, s.handed);
          __syncwarp();
          if (sh) have_s = true; else have_r = true;
          if constexpr (kHalf) {
            if (__shfl_sync(0xffffffffu, reached, 0) != (uint32_t)(sh ? a.T : a.T * a.k)) {
              mixed = true;
              choose_copies(sh);
            }
          }
        }
        const int n_tok = sh ? a.T : (int)(info >> 8 & 255u);
        uint32_t next = info;
        const bool last = kF32 || n0 + 8 >= n_tok;
        int ni = i, nj = j, nn = n0 + 8;
        if (last) {
          nn = 0;
          nj += per;
          seek(ni, nj, next);
        }
        float sc[kSub2][2];  // fp8: every (expert, row) has its own scale
#pragma unroll
        for (int q = 0; q < kSub2; ++q) {
          sc[q][0] = sc[q][1] = 1.0f;
          if constexpr (kHalf) {
            const float* f = (sh ? a.ws2s : a.w2s + (size_t)(info & 255u) * a.dp) + r0;
            sc[q][0] = __ldg(f + min(16 * q + g, rows - 1));
            sc[q][1] = __ldg(f + min(16 * q + g + 8, rows - 1));
          }
        }
        float un[2] = {1.0f, 1.0f};  // fp8: 1 / scale of the rows of this lane's two columns
        if constexpr (kHalf) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int n = n0 + 2 * t4 + c, row = sh ? S::kShared + min(n, a.T - 1) : (int)s.asg[i][n];
            if constexpr (kDirect) un[c] = pow2(-h_scale_exp(s.xexp[n], (int)s.bound[sh ? a.E : (int)(info & 255u)], a.glu));
            else un[c] = s.undo[row];
            if (mixed) un[c] *= pow2(-kCopyExp * s.copy[row]);
          }
        }
        auto scaled = [&](float v, int c) { return kHalf ? v * un[c] : v; };
        auto join = [&](const float (&acc)[kSub2][4], int n0) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int n = n0 + 2 * t4 + c;
            if (n < n_tok) {
              const int tk = sh ? n : (int)s.tok[i][n];
              float* o = p + ((tk >> 3) * kSub2 * 32 + g * 4 + ((tk & 7) >> 1)) * 4 + (tk & 1);
#pragma unroll
              for (int q = 0; q < kSub2; ++q) {
                o[q * 128] = fmaf(scaled(acc[q][c], c), sc[q][0], o[q * 128]);
                o[q * 128 + 2] = fmaf(scaled(acc[q][2 + c], c), sc[q][1], o[q * 128 + 2]);
              }
            }
          }
        };
        if constexpr (kF32) {
          arrived();
          for (int n0 = 0; n0 < n_tok; n0 += 8) {
            float acc[1][4] = {{0.0f, 0.0f, 0.0f, 0.0f}};
            auto row = [&](int n) { return reinterpret_cast<const float*>(h_at(i, n0 + n, k)); };
            box_fma<true>(acc[0], box(pitch), 8 * pitch, blk, row, min(8, n_tok - n0), (sh ? a.k2s : a.k2) - k, lane);
            join(acc, n0);
          }
        } else {
          if (!ready) load_h(v, i, n0, k);
          ready = ni < n_act && (ni < 0 || have_r);
          if (ready) load_h(w, ni, nn, nj * (ni < 0 ? a.b2s : a.b2));
          if (n0 == 0) arrived();
          // a box's sums join by the same operations in both forms: a token's result does not depend on
          // how many others there are
          float acc[kSub2][4];
#pragma unroll
          for (int q = 0; q < kSub2; ++q)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[q][c] = 0.0f;
          box_mma<W, kTerms, kSub2>(acc, box(pitch), 8 * pitch, 16 * pitch, blk, v);
          if constexpr (kDirect) {
            const uint32_t m = (sh ? 0xffu : s.mask[i]) >> (2 * t4);
            if (m & 1u) {
              sum[0] = fmaf(scaled(acc[0][0], 0), sc[0][0], sum[0]);
              sum[2] = fmaf(scaled(acc[0][2], 0), sc[0][1], sum[2]);
            }
            if (m & 2u) {
              sum[1] = fmaf(scaled(acc[0][1], 1), sc[0][0], sum[1]);
              sum[3] = fmaf(scaled(acc[0][3], 1), sc[0][1], sum[3]);
            }
          } else {
            join(acc, n0);
          }
        }
        if (last) release();
        i = ni;
        j = nj;
        n0 = nn;
        info = next;
      };
      while (i < n_act) {
        step(va, vb);
        if (i >= n_act) break;
        step(vb, va);
      }
      if constexpr (kDirect) {
        *reinterpret_cast<float4*>(p + lane * 4) = make_float4(sum[0], sum[1], sum[2], sum[3]);
        hand_over();
      } else {
        // The twelve warps' sums, a 16 x 8 tile a warp; no other work of this CTA is left to overlap with (few
        // CTAs have a second item), and one finishing warp took 6 us longer over 32 tokens' eight tiles.
        constexpr int kTiles = NT * kSub2;
        float* all = a.partial + (size_t)tile * a.splits * kTiles * 128 + lane * 4;
        compute_sync();
        for (int q = warp; q < kTiles; q += kCompute) {
          float4 c = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int w = 0; w < kCompute; ++w) add(c, *reinterpret_cast<const float4*>(s.sums[w][q / kSub2][q % kSub2][lane]));
          if (a.splits == 1) store_out<W>(a, c, tile, q / kSub2, q % kSub2, lane);
          else *reinterpret_cast<float4*>(all + (split * kTiles + q) * 128) = c;
        }
        if (a.splits > 1) {
          __threadfence();
          compute_sync();
          if (threadIdx.x == 0) {
            s.last = atomicAdd(a.ctr + kCtrTiles + tile, 1u) == (uint32_t)a.splits - 1u;
            if (s.last) a.ctr[kCtrTiles + tile] = 0u;
            __threadfence();
          }
          compute_sync();
          if (s.last)
            for (int q = warp; q < kTiles; q += kCompute)
              store_out<W>(a, tile_sum(all + q * 128, a.splits, kTiles * 128), tile, q / kSub2, q % kSub2, lane);
        }
        compute_sync();
      }
    }
  } else {
    // ================================================================ service
    const int sw = warp - kService;
    route<X, SUB, 8 * NT, kDirect, kHalf>(a, s, waits, sw, route_warps, lane);
    const int2 ru = routed_units(wait_routed());
    const int nu = nu_s + ru.y;
    const size_t h_lo = (size_t)a.T * a.k * a.hp, hs_lo = (size_t)a.T * a.hsp;
    uint32_t owed[2] = {0u, 0u};  // handings over of the shared expert / the routed experts stored, not announced
    uint32_t reached = 0u;        // fp8: rows that reach kReaches0 in these, if they are of first units
    auto announce = [&](int which, uint32_t* ctr) {
      if (owed[which] == 0u) return;
      __syncwarp();
      if (lane == 0) ctr_add(ctr, owed[which], reached);
      owed[which] = reached = 0u;
    };
    // Every second handing over is this warp's.
    int seq = 0;
    auto mine = [&]() { return seq % kServices == sw; };
    auto wait_parts = [&]() { waits.bar(smem_u32(&s.part_full[seq % kParts]), (uint32_t)(seq / kParts) & 1u); };
    auto free_parts = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s.part_empty[seq % kParts]));
    };
    int ai = 0, first = 0;  // active expert of the present routed unit, and that expert's first one
    // fp8: the sizes that this warp has noted for the tokens from seen_n0 on of active expert seen_by (-1: shared)
    uint32_t seen = 0u;
    int seen_n0 = -1, seen_by = -1;
    for (int un = 0; un < nu; ++un) {
      const bool sh = un < nu_s;
      if (un == nu_s) announce(0, a.ctr + kCtrShared);
      const int r = ru.x + un - nu_s;
      if (!sh)
        while (r >= first + a.upe) {
          first += a.upe;
          ++ai;
        }
      const int u = sh ? cta + un * G : r - first, e = sh ? 0 : s.act[ai];
      const int n_tok = sh ? a.T : (int)(s.info[ai] >> 8 & 255u);
      for (int h0 = 0; h0 < (kHand < NT ? n_tok : 1); h0 += 8, ++seq) {
        if (!mine()) continue;
        // where these sums go is looked up before they are there
        float s0[SUB], s1[SUB];
#pragma unroll
        for (int q = 0; q < SUB; ++q) {
          s0[q] = s1[q] = 1.0f;
          if constexpr (kHalf) {
            const int ch = 8 * SUB * u + 8 * q + g;
            const int row0 = a.glu ? (ch >> 7) * 256 + (ch & 127) : 16 * SUB * u + 16 * q + g, row1 = a.glu ? row0 + 128 : row0 + 8;
            const float* sc = sh ? a.ws1s : a.w1s + (size_t)e * a.n1p;
            s0[q] = __ldg(sc + row0);
            s1[q] = __ldg(sc + row1);
          }
        }
        // activation, routing weight, and the intermediate to where GEMM2 reads it
        uint8_t* base = sh ? a.hs : a.h;
        const size_t lo = sh ? hs_lo : h_lo;
        const uint32_t mask = sh ? 0xffffffffu : s.mask[ai];
        bool waited = false;
        for (int nt = 0; nt < kHand; ++nt) {
          const int n0 = kHand < NT ? h0 : nt * 8;
          if (n0 >= (kDirect ? a.T : n_tok)) break;
          float wt[2];
          size_t at[2];
          bool on[2];
          int tok[2];
          uint32_t reach[2] = {0u, 0u};  // fp8: sizes of these columns' values
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int n = n0 + 2 * t4 + i;  // column: the n-th token of the expert, or token n
            on[i] = n < (kDirect ? a.T : n_tok);
            if constexpr (kDirect) on[i] = on[i] && ((mask >> n) & 1u);
            const int row = on[i] ? (sh ? n : (int)s.asg[ai][n]) : 0;
            tok[i] = on[i] ? (sh || kDirect ? n : (int)s.tok[ai][n]) : 0;
            wt[i] = sh ? s.sg[row] : s.wt[row];
            at[i] = (size_t)row * (sh ? a.hsp : a.hp);
          }
          if (!waited) wait_parts();
          waited = true;
          float c[SUB][4];
#pragma unroll
          for (int q = 0; q < SUB; ++q) c[q][0] = c[q][1] = c[q][2] = c[q][3] = 0.0f;
#pragma unroll
          for (int w = 0; w < kCompute; ++w) {
            if (w >= a.n1) break;
#pragma unroll
            for (int q = 0; q < SUB; ++q) {
              const float4 o = *reinterpret_cast<const float4*>(s.part[seq % kParts][w][nt][q][lane]);
              c[q][0] += o.x; c[q][1] += o.y; c[q][2] += o.z; c[q][3] += o.w;
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (!on[i]) continue;
            const float xi = kHalf ? s.xinv[tok[i]] : 1.0f;
            const float f = kHalf ? wt[i] * pow2(h_scale_exp(s.xexp[tok[i]], (int)s.bound[sh ? a.E : e], a.glu)) : wt[i];
            auto put = [&](int ch, float val) {
              if constexpr (kF32) {
                reinterpret_cast<float*>(base)[at[i] + ch] = val;
              } else if constexpr (kHalf) {
                __half* o = reinterpret_cast<__half*>(base) + at[i] + ch;
#pragma unroll
                for (int c = 0; c < kCopies; ++c) o[c * lo] = __float2half_rn(val * pow2(kCopyExp * c));
                reach[i] |= h_reach(val);
              } else {
                const __nv_bfloat16 hi = __float2bfloat16_rn(val);
                const float rest = val - __bfloat162float(hi);
                __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(base) + at[i] + ch;
                o[0] = hi;
                // an infinite or NaN value is the high term alone
                o[lo] = __float2bfloat16_rn(fabsf(val) <= 3.38e38f ? rest : 0.0f);
              }
            };
#pragma unroll
            for (int q = 0; q < SUB; ++q) {
              const float c0 = c[q][i] * xi * s0[q], c1 = c[q][2 + i] * xi * s1[q];
              if (a.glu) {
                // the factor joins one side first: the product alone may leave fp32 where the scaled one does not
                put(8 * SUB * u + 8 * q + g, c0 / (1.0f + expf(-c0)) * f * c1);
              } else {
                put(16 * SUB * u + 16 * q + g, f * fmaxf(c0, 0.0f));
                put(16 * SUB * u + 16 * q + g + 8, f * fmaxf(c1, 0.0f));
              }
            }
          }
          if constexpr (kHalf) {
            // the eight tokens' sizes side by side; what an expert's units before this one have brought is there already
            if (n0 != seen_n0 || (sh ? -1 : ai) != seen_by) seen = 0u;
            seen_n0 = n0;
            seen_by = sh ? -1 : ai;
            const uint32_t all = __reduce_or_sync(0xffffffffu, reach[0] << (4 * t4) | reach[1] << (4 * t4 + 2));
            const uint32_t fresh = all & ~seen;
            seen |= all;
            if (u == 0) reached += __popc(all & kReaches0 * 0x5555u);
            if (lane < 8 && (fresh >> (2 * lane) & 3u))
              atomicOr(a.reach + (sh ? a.T * a.k + n0 + lane : (int)s.asg[ai][n0 + lane]), fresh >> (2 * lane) & 3u);
          }
        }
        free_parts();
        ++owed[sh ? 0 : 1];
      }
    }
    announce(0, a.ctr + kCtrShared);
    announce(1, a.ctr + kCtrRouted);
    // ---- the output's rows, one 16 x 8 tile an item (else the compute warps store them)
    if constexpr (kDirect) {
      for (int item = cta; item < items; item += G, ++seq) {
        if (!mine()) continue;
        const int tile = item / a.splits;
        wait_parts();
        float4 c = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kCompute; ++w) add(c, *reinterpret_cast<const float4*>(s.part[seq % kParts][w][0][0][lane]));
        if (a.splits == 1) {
          store_out<W>(a, c, tile, 0, 0, lane);
          free_parts();
        } else {
          float* all = a.partial + (size_t)tile * a.splits * 128 + lane * 4;
          *reinterpret_cast<float4*>(all + item % a.splits * 128) = c;
          free_parts();
          __threadfence();
          __syncwarp();
          uint32_t before = 0u;
          if (lane == 0) before = atomicAdd(a.ctr + kCtrTiles + tile, 1u);
          before = __shfl_sync(0xffffffffu, before, 0);
          if (before == (uint32_t)a.splits - 1u) {
            __threadfence();
            store_out<W>(a, tile_sum(all, a.splits, 128), tile, 0, 0, lane);
            if (lane == 0) a.ctr[kCtrTiles + tile] = 0u;
          }
        }
      }
    }
  }

  __syncthreads();
  // After an abort copies may still be on their way into this CTA's shared memory.  They come whatever the caller's
  // limit is, so it does not count here.
  if (*abort_flag) {
    if (threadIdx.x < kCompute) {
      const uint32_t left = s.left[threadIdx.x];
      const int st = (int)(left & 255u);
      const uint32_t phase = left >> 8 & 1u;
      for (int q = 0; q < ((left >> 9) ? a.stages : st); ++q) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(smem_u32(&s.full[threadIdx.x][q]), q < st ? phase : phase ^ 1u) &&
               globaltimer_ns() - t0 < kWaitLimitNs) {
        }
      }
    }
    __syncthreads();
  }
  // ---- the last CTA to leave zeroes the counters for the next call
  if (warp == 0) {
    uint32_t before = 0u;
    if (lane == 0) {
      __threadfence();
      before = atomicAdd(a.ctr + kCtrExit, 1u);
    }
    if (__shfl_sync(0xffffffffu, before, 0) == (uint32_t)G - 1u) {
      if (kHalf) a.ctr[kCtrBound + lane] = a.ctr[kCtrBound + 32 + lane] = 0u;
      if (lane < kCtrTiles) a.ctr[lane] = 0u;
      __threadfence();
    }
  }
}

constexpr int kHBytes = 2 * kCopies;  // of a value of the intermediate, at most
constexpr int kMaxItems = 256;  // items whose sums the workspace holds, 32 rows x 32 tokens each
constexpr size_t kPartialBytes = (size_t)kMaxItems * 4 * 2 * 512;

inline int round_up(int v, int m) { return (v + m - 1) / m * m; }

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_fn() {
  static EncodeTiled fn = nullptr;
  if (fn == nullptr) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(ptr);
  }
  return fn;
}

// Boxes of `rows` rows x `box` values of a row-major matrix [n, width]; glu: half of them gate rows, half the
// matching up rows of its 256-row blocks.  Values behind the row's end are filled with zeros.
template <typename W>
int make_map(CUtensorMap* m, const void* base, uint64_t n, int width, int box, int rows, bool glu) {
  EncodeTiled enc = encode_fn();
  if (enc == nullptr) return DSCA_ERR_CUDA;
  const CUtensorMapDataType type = W::kSize == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : W::kSize == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const cuuint64_t row = (cuuint64_t)width * W::kSize;
  const cuuint64_t dims[4] = {(cuuint64_t)width, glu ? 128u : n, 2, n / 256}, strides[3] = {row, row * 128, row * 256};
  const cuuint32_t boxes[4] = {(cuuint32_t)box, (cuuint32_t)(glu ? rows / 2 : rows), 2, 1}, one[4] = {1, 1, 1, 1};
  return enc(m, type, glu ? 4 : 2, const_cast<void*>(base), dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? DSCA_OK
             : DSCA_ERR_CUDA;
}

// Bytes of a row of `bytes` in a box: `warps` warps take a row's boxes in turn (GEMM2, where they go round from
// expert to expert: as one), and a warp's time for one is about that of 256 bytes for its instructions
// plus that of the box itself.  At most `most`, and the blocks whose
// token values a lane holds; tensor maps take at most 256 values.
template <typename W, int kTerms>
int box_of(int bytes, int warps, int most) {
  if (W::kSize != 4) most = min(most, Layout<W, kTerms>::kBlocks * 64);
  int best = 64, cost = 1 << 30;
  for (int b = 64; b <= most && b <= 256 * W::kSize; b += 64) {
    const int n = (bytes + b - 1) / b, c = (n + warps - 1) / warps * (b + 256);
    if (c < cost) {
      best = b;
      cost = c;
    }
  }
  return best;
}

// Output rows of a tile and CTAs that share one (see the top): tiles of `high` rows at most, as many CTAs to
// each as there are.  Against tiles for one CTA each: 32 tokens of the Qwen block with fp8 weights (28 rows
// by 2 CTAs, not 14 by one) 132 us, 165; 16 tokens of a Switch block of 768 (32 rows by 6, not 6 by one)
// 37 us, 58; one token of it 15.4 us, 15.9.
inline void plan_tiles(int d, int sms, int high, int* rt, int* tiles, int* splits) {
  const int full = (d + high - 1) / high;
  *splits = max(1, sms / full);
  const int ctas = sms / *splits, nt = ((d + ctas - 1) / ctas + high - 1) / high;
  *rt = (d + ctas * nt - 1) / (ctas * nt);
  *tiles = (d + *rt - 1) / *rt;
}

template <typename W, int NT, int SUB>
int launch(Args a, const dsca_few_args* p, int sms, cudaStream_t stream) {
  using F = Form<W, NT, SUB>;
  static PerDeviceOnce once;
  if (once.run([] {
        return cudaFuncSetAttribute(moe_few_kernel<W, NT, SUB>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
      }) != cudaSuccess)
    return DSCA_ERR_CUDA;
  constexpr int kFixed = (int)((sizeof(Smem<W, NT, SUB>) + 127) / 128 * 128);
  const int unit = (a.glu ? 8 : 16) * SUB, shared = p->w_shared_gate != nullptr ? p->shared_inter : 0;
  a.upe = (p->inter + unit - 1) / unit;
  a.ups = (shared + unit - 1) / unit;
  // GEMM2 reads whole 16-byte vectors: the channels behind the last are zero in both operands
  a.k2 = a.upe * unit;
  a.k2s = a.ups * unit;
  plan_tiles(a.d, sms, 16 * F::kSub2, &a.rt, &a.tiles, &a.splits);
  if (a.splits > 1 && (kCtrTiles + a.tiles > kCtrBound || a.tiles * a.splits > kMaxItems)) return DSCA_ERR_CAPACITY;
  // a stage holds whole 16-row tiles: the rows behind a tile's last are read, and dropped
  const int rows = 16 * max(SUB, F::kSub2), most = min(kMaxBox, (kSmem - kFixed) / (2 * kCompute * rows) / 64 * 64);
  a.b1 = box_of<W, 1>(a.d * W::kSize, kCompute, most) / W::kSize;
  a.b2 = box_of<W, F::kTerms>(a.k2 * W::kSize, 1, most) / W::kSize;
  a.b2s = box_of<W, F::kTerms>(a.k2s * W::kSize, 1, most) / W::kSize;
  a.n1 = (a.d + a.b1 - 1) / a.b1;
  a.n2 = (a.k2 + a.b2 - 1) / a.b2;
  a.n2s = (a.k2s + a.b2s - 1) / a.b2s;
  a.n2_cta = (a.n2 + a.splits - 1) / a.splits;
  if (SUB == 2 && a.n1 > 2 * kCompute) return DSCA_ERR_CAPACITY;
  const int bytes = max(16 * SUB * a.b1, 16 * F::kSub2 * max(a.b2, a.n2s ? a.b2s : 0)) * W::kSize;
  a.stage = (bytes + 127) / 128 * 128;
  a.stages = min(kMaxStages, (kSmem - kFixed) / (kCompute * a.stage));
  CUtensorMap m1, m2, ms1, ms2;
  int rc;
  if ((rc = make_map<W>(&m1, a.w1, (uint64_t)a.E * a.n1p, a.d, a.b1, 16 * SUB, a.glu))) return rc;
  if ((rc = make_map<W>(&m2, a.w2, (uint64_t)a.E * a.dp, a.ip, a.b2, a.rt, false))) return rc;
  ms1 = m1;
  ms2 = m2;
  if (a.ups) {
    if ((rc = make_map<W>(&ms1, a.ws1, (uint64_t)p->shared_n1p, a.d, a.b1, 16 * SUB, a.glu))) return rc;
    if ((rc = make_map<W>(&ms2, a.ws2, (uint64_t)a.dp, a.s_ip, a.b2s, a.rt, false))) return rc;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)sms);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)(kFixed + kCompute * a.stages * a.stage);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, moe_few_kernel<W, NT, SUB>, (const Args)a, m1, m2, ms1, ms2) == cudaSuccess ? DSCA_OK
                                                                                                             : DSCA_ERR_CUDA;
}

template <typename W>
int launch_t(const Args& a, const dsca_few_args* p, int sms, cudaStream_t stream) {
  if (a.T <= 8) return launch<W, 1, 1>(a, p, sms, stream);
  if constexpr (W::kSize != 4) {
    // units of 32 rows: one or two boxes of at most 192 bytes a warp (against 16 rows: of the Qwen
    // block 20 tokens in bf16 187 us, 216, 32 with fp8 weights 132 us, 165; 16 of the Switch block of 768 36.5 us, 40.4)
    if (a.d * W::kSize <= 2 * 192 * kCompute) {
      if (a.T <= 16) return launch<W, 2, 2>(a, p, sms, stream);
      return launch<W, 4, 2>(a, p, sms, stream);
    }
  }
  if (a.T <= 16) return launch<W, 2, 1>(a, p, sms, stream);
  return launch<W, 4, 1>(a, p, sms, stream);
}

}  // namespace few

size_t few_workspace_bytes(int T, int d, int k, int inter, int shared_inter) {
  const size_t hp = few::round_up(inter, 64), hsp = few::round_up(shared_inter, 64);
  const size_t x16 = T > 8 ? (size_t)T * (d * 2 + 8) : 0;  // fp8 weights
  return DSCA_FEW_ZERO_BYTES + (size_t)T * few::kLgPitch * few::kDotParts * 8 + (size_t)T * (k * hp + hsp) * few::kHBytes +
         few::round_up(T * (k + 1) * 4, 256) + (x16 + 255) / 256 * 256 + few::kPartialBytes;
}

int launch_moe_few(const dsca_few_args* p, int num_sms, cudaStream_t stream) {
  few::Args a = {};
  a.x = p->x; a.w_router = p->w_router; a.w_gate = p->w_shared_gate;
  a.w1 = (const uint8_t*)p->w1; a.w2 = (const uint8_t*)p->w2;
  a.ws1 = (const uint8_t*)p->ws1; a.ws2 = (const uint8_t*)p->ws2;
  a.w1s = p->w1_scale; a.w2s = p->w2_scale; a.ws1s = p->ws1_scale; a.ws2s = p->ws2_scale;
  a.out = p->out; a.logits = p->logits; a.topk_ids = p->topk_ids; a.topk_w = p->topk_w;
  a.expert_index = p->expert_index; a.err = p->err;
  a.wait_ns = p->wait_limit_ns ? p->wait_limit_ns : kWaitLimitNs;
  a.T = p->T; a.d = p->d; a.E = p->E; a.mode = p->mode; a.norm_topk = p->norm_topk;
  a.k = p->mode == DSCA_ROUTE_SWITCH_TOP1 ? 1 : p->top_k;
  a.glu = p->act == DSCA_ACT_SWIGLU;
  a.n1p = p->n1p; a.ip = p->ip; a.dp = p->dp; a.s_ip = p->shared_ip;
  const int shared = p->w_shared_gate != nullptr ? p->shared_inter : 0;
  a.inter = p->inter;
  a.s_inter = shared;
  a.hp = few::round_up(p->inter, 64);
  a.hsp = few::round_up(shared, 64);
  uint8_t* w = (uint8_t*)p->workspace;
  a.ctr = (uint32_t*)w;
  a.lg = (double*)(w + DSCA_FEW_ZERO_BYTES);
  a.h = w + DSCA_FEW_ZERO_BYTES + (size_t)a.T * few::kLgPitch * few::kDotParts * 8;
  a.hs = a.h + (size_t)a.T * a.k * a.hp * few::kHBytes;
  a.partial = (float*)(w + few_workspace_bytes(a.T, a.d, a.k, p->inter, shared) - few::kPartialBytes);
  if (p->weights == DSCA_F8E4M3) {
    a.reach = (uint32_t*)(a.hs + (size_t)a.T * a.hsp * few::kHBytes);
    if (a.T > 8) {
      a.x16 = (uint8_t*)a.reach + few::round_up(a.T * (a.k + 1) * 4, 256);
      a.xmeta = (float*)(a.x16 + (size_t)a.T * a.d * 2);
    }
  }
  if (p->weights == DSCA_BF16) return few::launch_t<few::Bf16>(a, p, num_sms, stream);
  if (p->weights == DSCA_F32) return few::launch_t<few::F32>(a, p, num_sms, stream);
  return few::launch_t<few::Fp8>(a, p, num_sms, stream);
}

}  // namespace dsca
