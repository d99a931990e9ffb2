// The whole MoE block for a few tokens (at most 32) in one kernel.
//
//   logits = round(x W_r^T)          p = softmax(logits)      S_t = the k largest p (lowest id first)
//   h_te   = w_te act(up_e x_t)      out_t = sum_{e in S_t} down_e h_te + sigmoid(round(x.g)) shared(x_t)
//
// Such a call's time is the reading of the chosen experts' weights (17 MB an expert of the Qwen block
// in bf16, 69 MB for its shared expert, against 4 KB a token), so everything here serves one
// uninterrupted stream of weight bytes:
//  - one persistent CTA per SM.  A producer warp copies pieces of 16 weight rows x up to 2 KB into a
//    ring of shared-memory stages (asynchronous bulk copies, 16 a piece); eight compute warps split
//    each piece along k, keep their sums in registers and hand them over at the end of a unit (16
//    rows of a matrix); three service warps add the eight parts, apply the activation and store, and
//    run the router at the start.  No role waits for another one's latency: the stream stalls only
//    when the whole ring is full;
//  - the weights are cut 16 rows at a time (8 gate + 8 up rows, or 16 rows of any other matrix), fine
//    enough that 148 SMs get nearly equal shares, where a 128-row tensor-memory tile would leave
//    two fifths of them idle at one token.  16 rows x 8 tokens is the shape of mma.sync, which
//    has to run at one 16x8x16 product per 20 clocks to keep up with DRAM;
//  - the order is shared GEMM1, routed GEMM1, shared GEMM2, routed GEMM2: the shared expert needs no
//    routing, so its weights are on their way while the router runs, and by the time a CTA needs
//    the intermediates of another one they have mostly been published.
//  - the routing weight is multiplied into the intermediate, so GEMM2 adds every expert's part into
//    the same fp32 registers and a CTA owns its rows of the output: no atomics, no second pass.
//
// Lane layout: lane (g, t) = (lane / 4, lane % 4) reads 16 bytes of weight rows g and g + 8 at offset
// 16 t of each 64-byte block, and the same positions of token g.  A dot product does not mind in
// which order its terms come, so these bytes go into the tensor core's operand registers as they
// are: the k index that the instruction thinks it sees is a permutation of the real one, the same
// for both operands.
//
// The intermediate is kept as two bf16 terms (16 significant bits); everything is summed in fp32,
// the router in fp64 (bf16 products are exact in fp32, so the logits round correctly).
#include "common.cuh"
#include "dsca_b200_block.h"

namespace dsca {
namespace few {

constexpr int kWarps = 8;                 // compute warps (0 .. 7)
constexpr int kProducer = kWarps;         // the warp that issues the copies
constexpr int kService = kProducer + 1;   // first of the service warps
constexpr int kServices = 3;
constexpr int kThreads = (kService + kServices) * 32;
constexpr int kMaxStages = 16;
constexpr int kPiece = 2048;              // bytes of one weight row in a stage, at most
constexpr int kSmem = 227 * 1024;         // shared memory of a CTA
constexpr int kLgPitch = 64;              // logits scratch: E + 1 <= 64 per token

// words of the counter block
enum { kCtrLogits = 0, kCtrShared = 1, kCtrRouted = 2, kCtrExit = 3 };

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
  float* lg;        // [T][64] logits as fp32 (rounded to the router's type), column E = shared gate
  uint8_t* h;       // [T * k][hp] intermediate: bf16 high terms, then the low terms; or fp32
  uint8_t* hs;      // [T][hsp] the shared expert's
  uint32_t* ctr;
  int32_t* err;
  int T, d, E, k, mode, norm_topk, glu;
  int n1p, ip, dp, s_ip;
  int hp, hsp;            // row pitch of h / hs in values
  int upe, ups;           // units (16 weight rows of GEMM1) per routed expert / of the shared expert
  int k2, k2s;            // values of a row of w2 / ws2 that are read
  int p1, p2, p2s;        // values of a row that one piece of GEMM1 / routed / shared GEMM2 holds
  int rt, tiles;          // rows of a GEMM2 tile, tiles
  int pitch, stages;      // bytes of a stage row, stages of the ring
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

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four e4m3 values -> two bf16 pairs, exact
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  uint32_t a, b;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"((uint16_t)v));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"((uint16_t)(v >> 16)));
  const float2 fa = __half22float2(*reinterpret_cast<__half2*>(&a)), fb = __half22float2(*reinterpret_cast<__half2*>(&b));
  lo = pack_bf16x2(fa.x, fa.y);
  hi = pack_bf16x2(fb.x, fb.y);
}

__device__ __forceinline__ uint32_t ld_acquire(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// Bounded wait until *p reaches `target` (one thread; the counters only grow during a call).
__device__ __forceinline__ bool ctr_wait(const uint32_t* p, uint32_t target, volatile int* abort_flag, int32_t* err) {
  if (ld_acquire(p) >= target) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (ld_acquire(p) >= target) return true;
    if ((it & 63u) == 0u) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        record_error(err, kErrWaitTimeout);
        *abort_flag = 1;
        return false;
      }
    }
  }
}
__device__ __forceinline__ void ctr_add(uint32_t* p, uint32_t n) {
  __threadfence();
  atomicAdd(p, n);
}

// ---------------------------------------------------------------- shared memory
// Units whose parts may wait for a service warp: as many as leave the ring five or six full stages.
// At least kServices, so that a service warp that has seen one unit's parts knows every earlier use of
// the buffer it waits for next to be complete (a parity wait cannot look two phases ahead).
constexpr int parts_of(int nt) { return nt == 1 ? 4 : 3; }
static_assert(parts_of(1) >= kServices && parts_of(4) >= kServices, "parity waits");
template <int NT>
struct Smem {
  static constexpr int kParts = parts_of(NT);
  float part[kParts][kWarps][NT][32][4];    // the compute warps' sums of a unit
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t part_full[kParts], part_empty[kParts];
  uint64_t routed;
  float wt[8 * NT][DSCA_MAX_TOPK];          // routing weights
  float sg[8 * NT];                         // shared-expert gate
  uint32_t emask[DSCA_MAX_EXPERTS];         // tokens of an expert
  uint8_t act[DSCA_MAX_EXPERTS];            // experts with tokens, ascending
  uint8_t tok[DSCA_MAX_EXPERTS][8 * NT];    // n-th token of an expert
  uint8_t slot[DSCA_MAX_EXPERTS][8 * NT];   // choice j of (expert, token)
  int n_act;
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

// x . w over one warp in fp64, the same on every lane
__device__ __forceinline__ double dot64(const __nv_bfloat16* x, const __nv_bfloat16* w, int d, int lane) {
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  for (int c = lane * 8; c < d; c += 256) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(x + c)), b = __ldg(reinterpret_cast<const uint4*>(w + c));
    const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // products of two 8-bit significands are exact in fp32
      s[i] += (double)(__uint_as_float(av[i] << 16) * __uint_as_float(bv[i] << 16));
      s[i] += (double)(__uint_as_float(av[i] & 0xffff0000u) * __uint_as_float(bv[i] & 0xffff0000u));
    }
  }
  double r = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) r += __shfl_xor_sync(0xffffffffu, r, off);
  return r;
}
__device__ __forceinline__ double dot64(const float* x, const float* w, int d, int lane) {
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  for (int c = lane * 4; c < d; c += 128) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(x + c)), b = __ldg(reinterpret_cast<const float4*>(w + c));
    s[0] = fma((double)a.x, (double)b.x, s[0]);
    s[1] = fma((double)a.y, (double)b.y, s[1]);
    s[2] = fma((double)a.z, (double)b.z, s[2]);
    s[3] = fma((double)a.w, (double)b.w, s[3]);
  }
  double r = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
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
// arithmetic and the tie rule of dsca_router_topk.  Every CTA does it for itself; CTA 0 writes the results.
template <typename X, int NT>
__device__ __forceinline__ void select_token(const Args& a, Smem<NT>& s, int t, int lane) {
  const int E = a.E, e0 = lane, e1 = lane + 32;
  const float l0 = __ldcg(a.lg + t * kLgPitch + e0), l1 = __ldcg(a.lg + t * kLgPitch + e1);
  const bool v0 = e0 < E, v1 = e1 < E, first = blockIdx.x == 0;
  if (a.w_gate != nullptr && (e0 == E || e1 == E)) s.sg[t] = 1.0f / (1.0f + expf(-(e0 == E ? l0 : l1)));
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
  if (lane < a.k) {
    float w = my_p;
    if (!top1) {
      if (a.norm_topk) w = __fdiv_rn(my_p, sum);
      if (sizeof(X) == 2) w = round_bf16(w);
    }
    s.wt[t][lane] = w;
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
// B operand of GEMM1 / GEMM2: the tokens' rows.  p[nt] = this lane's row (token 8 nt + g) or null;
// lo = byte distance to the low terms (GEMM2).  kTerms 1: x; 2: the intermediate.
template <int NT>
struct Rows {
  const uint8_t* p[NT];
};

__device__ __forceinline__ uint4 ld_b(const uint8_t* p, bool live, bool coherent) {
  if (!live) return make_uint4(0u, 0u, 0u, 0u);
  const uint4* q = reinterpret_cast<const uint4*>(p);
  return coherent ? __ldcg(q) : *q;
}

// acc += 16 weight rows x (up to 8 NT tokens) over the 64-byte blocks [kb0, kb1) of a piece of bf16 or
// e4m3 weights.
//   stage: shared address of the stage, len: bytes of its rows, k0: k of its first value, klim: first k
//   without a token value, ntm: token tiles in use.  wait(): until the stage has arrived.
template <typename W, int NT, int kTerms, typename Wait>
__device__ __forceinline__ void piece_mma(float (&acc)[NT][4], uint32_t stage, int pitch, int len, int kb0, int kb1, int k0,
                                          int klim, const Rows<NT>& b, size_t lo, uint32_t ntm, int lane, Wait wait) {
  constexpr int kPer = W::kBlock / 32;             // 16-byte token vectors per lane and 64-byte block
  constexpr int kGroup = NT == 1 ? 4 : (NT == 2 ? 2 : 1);  // blocks whose token values are loaded together
  const int g = lane >> 2, t = lane & 3;
  bool waited = false;
  for (int kg = kb0; kg < kb1; kg += kGroup) {
    uint4 bv[kGroup][NT][kTerms][kPer];
#pragma unroll
    for (int i = 0; i < kGroup; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (!((ntm >> nt) & 1u)) continue;
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          const int k = k0 + (kg + i) * W::kBlock + t * 8 * kPer + q * 8;
          const bool live = kg + i < kb1 && k < klim && b.p[nt] != nullptr;
#pragma unroll
          for (int m = 0; m < kTerms; ++m)
            bv[i][nt][m][q] = ld_b(b.p[nt] + (size_t)k * 2 + (m ? lo : 0), live, kTerms == 2);
        }
      }
    if (!waited) {
      wait();
      waited = true;
    }
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      if (kg + i >= kb1) break;
      const int off = (kg + i) * 64 + t * 16;
      uint4 a0 = make_uint4(0u, 0u, 0u, 0u), a1 = a0;
      if (off < len) {  // behind the row's end the stage holds other rows' bytes
        a0 = lds128(stage + g * pitch + off);
        a1 = lds128(stage + (g + 8) * pitch + off);
      }
      if constexpr (W::kBlock == 32) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (!((ntm >> nt) & 1u)) continue;
#pragma unroll
          for (int m = 0; m < kTerms; ++m) {
            const uint4 v = bv[i][nt][m][0];
            mma_bf16(acc[nt], a0.x, a1.x, a0.y, a1.y, v.x, v.y);
            mma_bf16(acc[nt], a0.z, a1.z, a0.w, a1.w, v.z, v.w);
          }
        }
      } else {
        const uint32_t w0[4] = {a0.x, a0.y, a0.z, a0.w}, w1[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t p0, p1, q0, q1;
          e4m3x4_to_bf16(w0[j], p0, p1);
          e4m3x4_to_bf16(w1[j], q0, q1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (!((ntm >> nt) & 1u)) continue;
#pragma unroll
            for (int m = 0; m < kTerms; ++m) {
              const uint4 v = bv[i][nt][m][j / 2];
              mma_bf16(acc[nt], p0, q0, p1, q1, (j & 1) ? v.z : v.x, (j & 1) ? v.w : v.y);
            }
          }
        }
      }
    }
  }
  if (!waited) wait();
}

// The same for fp32 weights on the CUDA cores: lane (g, t) sums rows g and g + 8 over its k for all
// eight tokens of a tile; f32_fold() adds the four lanes of a row and leaves the layout of the
// tensor-core accumulators.  row(nt, n): token row (or null), the same on all lanes.
template <int NT, bool kCoherent, typename Row, typename Wait>
__device__ __forceinline__ void piece_fma(float (&acc)[NT][16], uint32_t stage, int pitch, int len, int kb0, int kb1, int k0,
                                          int klim, Row row, uint32_t ntm, int lane, Wait wait) {
  const int g = lane >> 2, t = lane & 3;
  wait();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (!((ntm >> nt) & 1u)) continue;
    const float* rp[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) rp[n] = row(nt, n);
#pragma unroll 2
    for (int kb = kb0; kb < kb1; ++kb) {
      const int off = kb * 64 + t * 16;
      const int k = k0 + kb * 16 + t * 4;
      if (off >= len || k >= klim) continue;
      const uint4 u0 = lds128(stage + g * pitch + off), u1 = lds128(stage + (g + 8) * pitch + off);
      const float a0[4] = {__uint_as_float(u0.x), __uint_as_float(u0.y), __uint_as_float(u0.z), __uint_as_float(u0.w)};
      const float a1[4] = {__uint_as_float(u1.x), __uint_as_float(u1.y), __uint_as_float(u1.z), __uint_as_float(u1.w)};
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        if (rp[n] == nullptr) continue;
        const float4* q = reinterpret_cast<const float4*>(rp[n] + k);
        const float4 v = kCoherent ? __ldcg(q) : *q;
        acc[nt][2 * n] = fmaf(a0[3], v.w, fmaf(a0[2], v.z, fmaf(a0[1], v.y, fmaf(a0[0], v.x, acc[nt][2 * n]))));
        acc[nt][2 * n + 1] = fmaf(a1[3], v.w, fmaf(a1[2], v.z, fmaf(a1[1], v.y, fmaf(a1[0], v.x, acc[nt][2 * n + 1]))));
      }
    }
  }
}
template <int NT>
__device__ __forceinline__ void f32_fold(const float (&a)[NT][16], float (&acc)[NT][4], int lane) {
  const int t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float v = a[nt][2 * n + r];
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        v += __shfl_xor_sync(0xffffffffu, v, 2);
        if (t == n / 2) acc[nt][2 * r + (n & 1)] = v;
      }
}

// ---------------------------------------------------------------- the kernel
__device__ __forceinline__ void group_sync(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }

// Router: fp64 dot products spread over the grid, then softmax, selection and the expert lists in every
// CTA for itself.  Warp wi of the nw warps that take part (they share named barrier 1).
template <typename X, int NT>
__device__ __forceinline__ void route(const Args& a, Smem<NT>& s, int wi, int nw, int lane) {
  const int G = gridDim.x, cta = blockIdx.x;
  const int R = a.E + (a.w_gate != nullptr ? 1 : 0), nd = a.T * R;
  for (int q = cta + wi * G; q < nd; q += nw * G) {
    const int t = q / R, r = q % R;
    const X* w = r < a.E ? reinterpret_cast<const X*>(a.w_router) + (size_t)r * a.d : reinterpret_cast<const X*>(a.w_gate);
    const double v = dot64(reinterpret_cast<const X*>(a.x) + (size_t)t * a.d, w, a.d, lane);
    if (lane == 0) a.lg[t * kLgPitch + r] = round_to<X>(v);
  }
  group_sync(nw * 32);
  if (wi == 0 && lane == 0) {
    if (cta < nd) ctr_add(a.ctr + kCtrLogits, 1u);
    ctr_wait(a.ctr + kCtrLogits, (uint32_t)min(nd, G), &s.abort, a.err);
  }
  group_sync(nw * 32);
  for (int t = wi; t < a.T; t += nw) select_token<X, NT>(a, s, t, lane);
  group_sync(nw * 32);
  if (wi == 0) {
    const uint32_t m0 = s.emask[lane], m1 = s.emask[lane + 32];
    const uint32_t b0 = __ballot_sync(0xffffffffu, m0 != 0u), b1 = __ballot_sync(0xffffffffu, m1 != 0u);
    const uint32_t below = (1u << lane) - 1u;
    if (m0) s.act[__popc(b0 & below)] = (uint8_t)lane;
    if (m1) s.act[__popc(b0) + __popc(b1 & below)] = (uint8_t)(lane + 32);
    if (lane == 0) s.n_act = __popc(b0) + __popc(b1);
  }
  for (int i = wi * 32 + lane; i < DSCA_MAX_EXPERTS * 8 * NT; i += nw * 32) {
    const int e = i / (8 * NT), t = i % (8 * NT);
    const uint32_t m = s.emask[e];
    if ((m >> t) & 1u) s.tok[e][__popc(m & ((1u << t) - 1u))] = (uint8_t)t;
  }
  group_sync(nw * 32);
  if (wi == 0 && lane == 0) mbar_arrive(smem_u32(&s.routed));
}

template <typename W, int NT>
__global__ void __launch_bounds__(kThreads, 1) moe_few_kernel(const Args a) {
  using X = typename W::X;
  constexpr bool kF32 = W::kSize == 4;
  constexpr int kParts = Smem<NT>::kParts;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<NT>& s = *reinterpret_cast<Smem<NT>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int G = gridDim.x, cta = blockIdx.x;
  const uint32_t ring = smem_u32(smem_raw) + (uint32_t)((sizeof(Smem<NT>) + 127) / 128 * 128);
  const uint32_t stage_bytes = 16u * (uint32_t)a.pitch;
  volatile int* abort_flag = &s.abort;

  if (threadIdx.x < (unsigned)a.stages) {
    mbar_init(smem_u32(&s.full[threadIdx.x]), 1);
    mbar_init(smem_u32(&s.empty[threadIdx.x]), kWarps);
  }
  if (threadIdx.x < kParts) {
    mbar_init(smem_u32(&s.part_full[threadIdx.x]), kWarps);
    mbar_init(smem_u32(&s.part_empty[threadIdx.x]), 1);
  }
  if (threadIdx.x >= 64 && threadIdx.x < 64 + DSCA_MAX_EXPERTS) s.emask[threadIdx.x - 64] = 0u;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&s.routed), 1);
    s.abort = 0;
    s.n_act = 0;
  }
  fence_mbar_init();
  __syncthreads();

  // ---- this CTA's work.  GEMM1: units cta, cta + G, ... of the shared expert, then of the routed
  // experts (the first of them on the CTA behind the last shared unit's).  GEMM2: tiles cta, cta + G,
  // ... of the output's rows; the pieces of the shared expert's row, then of the active experts'.
  const int nu_s = a.ups > cta ? (a.ups - cta + G - 1) / G : 0;
  const int r_first = (cta + G - a.ups % G) % G;
  auto routed_units = [&](int n_act) {
    const int units = n_act * a.upe;
    return units > r_first ? (units - r_first + G - 1) / G : 0;
  };
  auto wait_routed = [&]() { mbar_wait(smem_u32(&s.routed), 0u, abort_flag, a.err); };
  // The router runs on the service warps while the compute warps begin with the shared expert; on all
  // of them where there is no shared expert to begin with, or where the tokens are more than three
  // warps would do in the time of the first stages.
  const bool all_route = a.ups == 0 || a.T > 4;
  const int route_warps = all_route ? kWarps + kServices : kServices;

  if (warp == kProducer) {
    // ================================================================ producer
    int it = 0;
    auto piece = [&](const uint8_t* src, int rows, int len) {
      const int st = it % a.stages;
      if (it >= a.stages) mbar_wait(smem_u32(&s.empty[st]), (uint32_t)(it / a.stages - 1) & 1u, abort_flag, a.err);
      if (__any_sync(0xffffffffu, *abort_flag != 0)) return;
      const uint32_t bar = smem_u32(&s.full[st]);
      if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(rows * len));
      __syncwarp();
      if (lane < rows) bulk_load(ring + (uint32_t)st * stage_bytes + (uint32_t)(lane * a.pitch), src, (uint32_t)len, bar);
      ++it;
    };
    const int l = lane & 15;
    int nu_r = 0;
    for (int ul = 0; ul < nu_s + nu_r || ul == nu_s; ++ul) {
      const bool sh = ul < nu_s;
      if (ul == nu_s) {
        wait_routed();
        nu_r = routed_units(s.n_act);
        if (nu_r == 0) break;
      }
      const int r = sh ? cta + ul * G : r_first + (ul - nu_s) * G;
      const int u = sh ? r : r % a.upe, e = sh ? 0 : s.act[r / a.upe];
      const int ch = 8 * u + (l & 7);
      const int row = a.glu ? (ch >> 7) * 256 + (ch & 127) + (l >> 3) * 128 : 16 * u + l;
      const uint8_t* src = (sh ? a.ws1 : a.w1) + ((size_t)e * a.n1p + row) * a.d * W::kSize;
      for (int k = 0; k < a.d; k += a.p1) piece(src + (size_t)k * W::kSize, 16, min(a.p1, a.d - k) * W::kSize);
    }
    const int n_act = s.n_act;
    for (int tile = cta; tile < a.tiles; tile += G) {
      const int r0 = tile * a.rt, rows = min(a.rt, a.d - r0), row = r0 + min(l, rows - 1);
      for (int k = 0; k < a.k2s; k += a.p2s)
        piece(a.ws2 + ((size_t)row * a.s_ip + k) * W::kSize, rows, (min(a.p2s, a.k2s - k) * W::kSize + 15) & ~15);
      for (int i = 0; i < n_act; ++i) {
        const uint8_t* src = a.w2 + ((size_t)s.act[i] * a.dp + row) * a.ip * W::kSize;
        for (int k = 0; k < a.k2; k += a.p2)
          piece(src + (size_t)k * W::kSize, rows, (min(a.p2, a.k2 - k) * W::kSize + 15) & ~15);
      }
    }
    // after an abort copies may still be on their way into this CTA's shared memory
    if (*abort_flag) {
      for (int i = max(0, it - a.stages); i < it; ++i) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(smem_u32(&s.full[i % a.stages]), (uint32_t)(i / a.stages) & 1u) &&
               globaltimer_ns() - t0 < kWaitLimitNs) {
        }
      }
    }
  } else if (warp < kWarps) {
    // ================================================================ compute
    if (all_route) route<X, NT>(a, s, kServices + warp, route_warps, lane);
    int it = 0, un = 0;  // pieces read, units handed over
    uint32_t st = ring;
    int len = 0, kb0 = 0, kb1 = 0;
    auto begin = [&](int bytes) {
      len = bytes;
      st = ring + (uint32_t)(it % a.stages) * stage_bytes;
      const int nkb = (len + 63) >> 6;
      kb0 = nkb * warp / kWarps;
      kb1 = nkb * (warp + 1) / kWarps;
    };
    auto arrived = [&]() { mbar_wait(smem_u32(&s.full[it % a.stages]), (uint32_t)(it / a.stages) & 1u, abort_flag, a.err); };
    auto release = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s.empty[it % a.stages]));
      ++it;
    };
    auto hand_over = [&](const float (&acc)[NT][4]) {
      const int b = un % kParts;
      if (un >= kParts) mbar_wait(smem_u32(&s.part_empty[b]), (uint32_t)(un / kParts - 1) & 1u, abort_flag, a.err);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        *reinterpret_cast<float4*>(s.part[b][warp][nt][lane]) = make_float4(acc[nt][0], acc[nt][1], acc[nt][2], acc[nt][3]);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s.part_full[b]));
      ++un;
    };
    int nu_r = 0;
    for (int ul = 0; ul < nu_s + nu_r || ul == nu_s; ++ul) {
      const bool sh = ul < nu_s;
      if (ul == nu_s) {
        wait_routed();
        nu_r = routed_units(s.n_act);
        if (nu_r == 0) break;
      }
      const int r = sh ? 0 : r_first + (ul - nu_s) * G;
      const int e = sh ? 0 : s.act[r / a.upe];
      const int n_tok = sh ? a.T : __popc(s.emask[e]);
      const uint32_t ntm = (1u << ((n_tok + 7) / 8)) - 1u;
      float acc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][i] = 0.0f;
      auto token = [&](int n) { return sh ? n : (int)s.tok[e][n]; };
      if constexpr (kF32) {
        float big[NT][16];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 16; ++i) big[nt][i] = 0.0f;
        auto row = [&](int nt, int n) {
          return 8 * nt + n < n_tok ? reinterpret_cast<const float*>(a.x) + (size_t)token(8 * nt + n) * a.d : nullptr;
        };
        for (int k = 0; k < a.d; k += a.p1) {
          begin(min(a.p1, a.d - k) * W::kSize);
          piece_fma<NT, false>(big, st, a.pitch, len, kb0, kb1, k, a.d, row, ntm, lane, arrived);
          release();
        }
        f32_fold<NT>(big, acc, lane);
      } else {
        Rows<NT> b;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          b.p[nt] = 8 * nt + g < n_tok ? reinterpret_cast<const uint8_t*>(a.x) + (size_t)token(8 * nt + g) * a.d * 2 : nullptr;
        for (int k = 0; k < a.d; k += a.p1) {
          begin(min(a.p1, a.d - k) * W::kSize);
          piece_mma<W, NT, 1>(acc, st, a.pitch, len, kb0, kb1, k, a.d, b, 0, ntm, lane, arrived);
          release();
        }
      }
      hand_over(acc);
    }
    // ---- GEMM2
    const int n_act = s.n_act;
    const size_t h_lo = (size_t)a.T * a.k * a.hp * 2, hs_lo = (size_t)a.T * a.hsp * 2;
    bool have_s = false, have_r = false;
    for (int tile = cta; tile < a.tiles; tile += G) {
      const int r0 = tile * a.rt, rows = min(a.rt, a.d - r0);
      float acc[NT][4];
      float big[kF32 ? NT : 1][16];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][i] = 0.0f;
      if constexpr (kF32) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 16; ++i) big[nt][i] = 0.0f;
      }
      // segment -1: the shared expert; i: active expert i
      for (int i = a.k2s ? -1 : 0; i < n_act; ++i) {
        const bool sh = i < 0;
        if (sh ? !have_s : !have_r) {
          // the intermediates come from every CTA's service warps
          if (lane == 0) {
            if (sh) ctr_wait(a.ctr + kCtrShared, (uint32_t)a.ups, abort_flag, a.err);
            else ctr_wait(a.ctr + kCtrRouted, (uint32_t)(n_act * a.upe), abort_flag, a.err);
          }
          __syncwarp();
          if (sh) have_s = true; else have_r = true;
        }
        const int e = sh ? 0 : s.act[i], kend = sh ? a.k2s : a.k2, pk = sh ? a.p2s : a.p2;
        const uint32_t mask = sh ? (a.T >= 32 ? 0xffffffffu : (1u << a.T) - 1u) : s.emask[e];
        uint32_t ntm = 0u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) ntm |= ((mask >> (8 * nt)) & 0xffu) ? 1u << nt : 0u;
        auto at = [&](int tk) { return sh ? (size_t)tk * a.hsp : ((size_t)tk * a.k + s.slot[e][tk]) * a.hp; };
        const uint8_t* base = sh ? a.hs : a.h;
        if constexpr (kF32) {
          auto row = [&](int nt, int n) {
            return (mask >> (8 * nt + n)) & 1u ? reinterpret_cast<const float*>(base) + at(8 * nt + n) : nullptr;
          };
          for (int k = 0; k < kend; k += pk) {
            begin((min(pk, kend - k) * W::kSize + 15) & ~15);
            piece_fma<NT, true>(big, st, a.pitch, len, kb0, kb1, k, kend, row, ntm, lane, arrived);
            release();
          }
        } else {
          Rows<NT> b;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) b.p[nt] = (mask >> (8 * nt + g)) & 1u ? base + at(8 * nt + g) * 2 : nullptr;
          const size_t lo = sh ? hs_lo : h_lo;
          if constexpr (W::kSize == 1) {
            // every (expert, row) has its own scale: an expert's sums are scaled before they join
            float part[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int q = 0; q < 4; ++q) part[nt][q] = 0.0f;
            const float* sc = sh ? a.ws2s : a.w2s + (size_t)e * a.dp;
            const float s0 = sc[r0 + min(g, rows - 1)], s1 = sc[r0 + min(g + 8, rows - 1)];
            for (int k = 0; k < kend; k += pk) {
              begin((min(pk, kend - k) * W::kSize + 15) & ~15);
              piece_mma<W, NT, 2>(part, st, a.pitch, len, kb0, kb1, k, kend, b, lo, ntm, lane, arrived);
              release();
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              acc[nt][0] = fmaf(part[nt][0], s0, acc[nt][0]);
              acc[nt][1] = fmaf(part[nt][1], s0, acc[nt][1]);
              acc[nt][2] = fmaf(part[nt][2], s1, acc[nt][2]);
              acc[nt][3] = fmaf(part[nt][3], s1, acc[nt][3]);
            }
          } else {
            for (int k = 0; k < kend; k += pk) {
              begin((min(pk, kend - k) * W::kSize + 15) & ~15);
              piece_mma<W, NT, 2>(acc, st, a.pitch, len, kb0, kb1, k, kend, b, lo, ntm, lane, arrived);
              release();
            }
          }
        }
      }
      if constexpr (kF32) f32_fold<NT>(big, acc, lane);
      hand_over(acc);
    }
  } else {
    // ================================================================ service
    const int sw = warp - kService;
    route<X, NT>(a, s, sw, route_warps, lane);
    wait_routed();
    const int n_act = s.n_act, n1 = nu_s + routed_units(n_act);
    const int n2 = a.tiles > cta ? (a.tiles - cta + G - 1) / G : 0;
    const size_t h_lo = (size_t)a.T * a.k * a.hp, hs_lo = (size_t)a.T * a.hsp;
    uint32_t owed[2] = {0u, 0u};  // stored units of the shared expert / the routed experts not yet announced
    auto announce = [&](int which, uint32_t* ctr) {
      if (owed[which] == 0u) return;
      __syncwarp();
      if (lane == 0) ctr_add(ctr, owed[which]);
      owed[which] = 0u;
    };
    for (int un = sw; un < n1 + n2; un += kServices) {
      const int b = un % kParts;
      // ---- where this unit's sums go, looked up before they are there
      const bool g1 = un < n1, sh = un < nu_s;
      if (!sh) announce(0, a.ctr + kCtrShared);
      if (!g1) announce(1, a.ctr + kCtrRouted);
      const int r = sh ? cta + un * G : r_first + (un - nu_s) * G;
      const int u = sh ? r : r % a.upe, e = (g1 && !sh) ? s.act[r / a.upe] : 0;
      const int n_tok = (sh || !g1) ? a.T : __popc(s.emask[e]);
      float s0 = 1.0f, s1 = 1.0f;
      if constexpr (W::kSize == 1) {
        if (g1) {
          const int ch = 8 * u + g;
          const int r0 = a.glu ? (ch >> 7) * 256 + (ch & 127) : 16 * u + g, r1 = a.glu ? r0 + 128 : r0 + 8;
          const float* sc = sh ? a.ws1s : a.w1s + (size_t)e * a.n1p;
          s0 = __ldg(sc + r0);
          s1 = __ldg(sc + r1);
        }
      }
      mbar_wait(smem_u32(&s.part_full[b]), (uint32_t)(un / kParts) & 1u, abort_flag, a.err);
      float c[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (nt * 8 >= n_tok) break;
        float4 v = *reinterpret_cast<const float4*>(s.part[b][0][nt][lane]);
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
          const float4 o = *reinterpret_cast<const float4*>(s.part[b][w][nt][lane]);
          v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
        }
        c[nt][0] = v.x; c[nt][1] = v.y; c[nt][2] = v.z; c[nt][3] = v.w;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s.part_empty[b]));
      if (g1) {
        // activation, routing weight, and the intermediate to where GEMM2 reads it
        uint8_t* base = sh ? a.hs : a.h;
        const size_t lo = sh ? hs_lo : h_lo;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (nt * 8 >= n_tok) break;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int n = nt * 8 + 2 * t4 + i;
            if (n >= n_tok) continue;
            const int tk = sh ? n : s.tok[e][n], j = sh ? 0 : s.slot[e][tk];
            const float w = sh ? s.sg[tk] : s.wt[tk][j];
            const size_t at = sh ? (size_t)tk * a.hsp : ((size_t)tk * a.k + j) * a.hp;
            auto put = [&](int ch, float val) {
              if constexpr (kF32) {
                reinterpret_cast<float*>(base)[at + ch] = val;
              } else {
                const __nv_bfloat16 hi = __float2bfloat16_rn(val);
                const float rest = val - __bfloat162float(hi);
                __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(base) + at + ch;
                o[0] = hi;
                // an infinite or NaN value is the high term alone
                o[lo] = __float2bfloat16_rn(fabsf(val) <= 3.38e38f ? rest : 0.0f);
              }
            };
            const float c0 = c[nt][i] * s0, c1 = c[nt][2 + i] * s1;
            if (a.glu) {
              put(8 * u + g, w * (c0 / (1.0f + expf(-c0)) * c1));
            } else {
              put(16 * u + g, w * fmaxf(c0, 0.0f));
              put(16 * u + g + 8, w * fmaxf(c1, 0.0f));
            }
          }
        }
        ++owed[sh ? 0 : 1];
      } else {
        const int r0 = (cta + (un - n1) * G) * a.rt, rows = min(a.rt, a.d - r0);
        X* out = reinterpret_cast<X*>(a.out);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tk = nt * 8 + 2 * t4 + (i & 1), rr = g + (i >> 1) * 8;
            if (tk < a.T && rr < rows) out[(size_t)tk * a.d + r0 + rr] = X(c[nt][i]);
          }
      }
    }
    announce(0, a.ctr + kCtrShared);
    announce(1, a.ctr + kCtrRouted);
  }

  // ---- the last CTA to leave zeroes the counters for the next call
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    if (atomicAdd(a.ctr + kCtrExit, 1u) == (uint32_t)G - 1u) {
      a.ctr[kCtrLogits] = a.ctr[kCtrShared] = a.ctr[kCtrRouted] = a.ctr[kCtrExit] = 0u;
      __threadfence();
    }
  }
}

inline int round_up(int v, int m) { return (v + m - 1) / m * m; }

template <typename W, int NT>
int launch(Args a, int sms, cudaStream_t stream) {
  static PerDeviceOnce once;
  if (once.run([] {
        return cudaFuncSetAttribute(moe_few_kernel<W, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
      }) != cudaSuccess)
    return DSCA_ERR_CUDA;
  constexpr int kFixed = (int)((sizeof(Smem<NT>) + 127) / 128 * 128);
  // a row in even pieces of whole 64-byte blocks; stage rows lie 64 bytes apart modulo 128, so that the
  // eight lanes of a shared-memory access phase (two rows) meet different banks
  auto piece = [](int k) {
    const int n = (k * W::kSize + kPiece - 1) / kPiece;
    return n ? round_up((k + n - 1) / n, W::kBlock) : 0;
  };
  a.p1 = piece(a.d);
  a.p2 = piece(a.k2);
  a.p2s = piece(a.k2s);
  a.pitch = max(a.p1, max(a.p2, a.p2s)) * W::kSize;
  if (a.pitch % 128 == 0) a.pitch += 64;
  a.stages = min(kMaxStages, (kSmem - kFixed) / (16 * a.pitch));
  // output rows in tiles of at most 16, as even as they come over the SMs
  const int per = (a.d + sms - 1) / sms, nt = (per + 15) / 16;
  a.rt = (a.d + sms * nt - 1) / (sms * nt);
  a.tiles = (a.d + a.rt - 1) / a.rt;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)sms);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)(kFixed + a.stages * 16 * a.pitch);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, moe_few_kernel<W, NT>, (const Args)a) == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

template <typename W>
int launch_t(const Args& a, int sms, cudaStream_t stream) {
  if (a.T <= 8) return launch<W, 1>(a, sms, stream);
  if (a.T <= 16) return launch<W, 2>(a, sms, stream);
  return launch<W, 4>(a, sms, stream);
}

}  // namespace few

size_t few_workspace_bytes(int T, int k, int inter, int shared_inter) {
  const size_t hp = few::round_up(inter, 64), hsp = few::round_up(shared_inter, 64);
  return DSCA_FEW_COUNTER_BYTES + (size_t)T * few::kLgPitch * 4 + (size_t)T * k * hp * 4 + (size_t)T * hsp * 4;
}

int launch_moe_few(const dsca_few_args* p, int num_sms, cudaStream_t stream) {
  few::Args a = {};
  a.x = p->x; a.w_router = p->w_router; a.w_gate = p->w_shared_gate;
  a.w1 = (const uint8_t*)p->w1; a.w2 = (const uint8_t*)p->w2;
  a.ws1 = (const uint8_t*)p->ws1; a.ws2 = (const uint8_t*)p->ws2;
  a.w1s = p->w1_scale; a.w2s = p->w2_scale; a.ws1s = p->ws1_scale; a.ws2s = p->ws2_scale;
  a.out = p->out; a.logits = p->logits; a.topk_ids = p->topk_ids; a.topk_w = p->topk_w;
  a.expert_index = p->expert_index; a.err = p->err;
  a.T = p->T; a.d = p->d; a.E = p->E; a.mode = p->mode; a.norm_topk = p->norm_topk;
  a.k = p->mode == DSCA_ROUTE_SWITCH_TOP1 ? 1 : p->top_k;
  a.glu = p->act == DSCA_ACT_SWIGLU;
  a.n1p = p->n1p; a.ip = p->ip; a.dp = p->dp; a.s_ip = p->shared_ip;
  const int shared = p->w_shared_gate != nullptr ? p->shared_inter : 0, unit = a.glu ? 8 : 16;
  a.hp = few::round_up(p->inter, 64);
  a.hsp = few::round_up(shared, 64);
  a.upe = (p->inter + unit - 1) / unit;
  a.ups = (shared + unit - 1) / unit;
  // GEMM2 reads whole 16-byte vectors: the channels behind the last are zero in both operands
  a.k2 = a.upe * unit;
  a.k2s = a.ups * unit;
  uint8_t* w = (uint8_t*)p->workspace;
  a.ctr = (uint32_t*)w;
  a.lg = (float*)(w + DSCA_FEW_COUNTER_BYTES);
  a.h = w + DSCA_FEW_COUNTER_BYTES + (size_t)a.T * few::kLgPitch * 4;
  a.hs = a.h + (size_t)a.T * a.k * a.hp * 4;
  if (p->weights == DSCA_BF16) return few::launch_t<few::Bf16>(a, num_sms, stream);
  if (p->weights == DSCA_F32) return few::launch_t<few::F32>(a, num_sms, stream);
  return few::launch_t<few::Fp8>(a, num_sms, stream);
}

}  // namespace dsca
