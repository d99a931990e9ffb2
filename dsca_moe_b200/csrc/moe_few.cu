// The whole MoE block for a few tokens (at most 32) in one kernel.
//
//   logits = round(x W_r^T)          p = softmax(logits)      S_t = the k largest p (lowest id first)
//   h_te   = w_te act(up_e x_t)      out_t = sum_{e in S_t} down_e h_te + sigmoid(round(x.g)) shared(x_t)
//
// Such a call's time is the reading of the chosen experts' weights (17 MB an expert of the Qwen block
// in bf16, 69 MB for its shared expert, against 4 KB a token), so everything here serves one
// uninterrupted stream of weight bytes:
//  - one persistent CTA per SM; each of its 8 warps keeps its own ring of asynchronous bulk copies
//    (16 weight rows x up to 512 bytes a stage) and multiplies what has arrived, so no warp waits
//    for another one's data and a stage is refilled as soon as it is read;
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

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxStages = 8;
constexpr int kPiece = 512;               // bytes of one weight row in a stage, at most
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
  int kc1;                // values of a GEMM1 row that one warp reads
  int rt, tiles;          // rows of a GEMM2 tile, tiles
  int pitch, stages;      // bytes of a stage row, stages of a warp's ring
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
__device__ __forceinline__ void ctr_add(uint32_t* p) {
  __threadfence();
  atomicAdd(p, 1u);
}

// ---------------------------------------------------------------- shared memory
template <int NT>
struct Smem {
  float part[2][kWarps][NT][32][4];         // partial sums of a unit or tile, double buffered
  uint64_t bar[kWarps][kMaxStages];
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

// acc += 16 weight rows x (up to 8 NT tokens) over one stage of bf16 or e4m3 weights.
//   stage: shared address of the stage, len: bytes of its rows, k0: first k, klim: first k without a
//   token value, ntu: token tiles in use (bit nt of ntm).  wait(): until the stage has arrived.
template <typename W, int NT, int kTerms, typename Wait>
__device__ __forceinline__ void stage_mma(float (&acc)[NT][4], uint32_t stage, int pitch, int len, int k0, int klim,
                                          const Rows<NT>& b, size_t lo, uint32_t ntm, int lane, Wait wait) {
  constexpr int kPer = W::kBlock / 32;                  // 16-byte token vectors per lane and 64-byte block
  constexpr int kGroupRaw = 8 / (NT * kTerms * kPer);   // 64-byte blocks whose token values are loaded together
  constexpr int kGroup = kGroupRaw < 1 ? 1 : kGroupRaw;
  const int g = lane >> 2, t = lane & 3;
  const int nkb = (len + 63) >> 6;
  bool waited = false;
  for (int kb0 = 0; kb0 < nkb; kb0 += kGroup) {
    uint4 bv[kGroup][NT][kTerms][kPer];
#pragma unroll
    for (int i = 0; i < kGroup; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (!((ntm >> nt) & 1u)) continue;
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          const int k = k0 + (kb0 + i) * W::kBlock + t * 8 * kPer + q * 8;
          const bool live = kb0 + i < nkb && k < klim && b.p[nt] != nullptr;
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
      const int kb = kb0 + i;
      if (kb >= nkb) break;
      const int off = kb * 64 + t * 16;
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
__device__ __forceinline__ void stage_fma(float (&acc)[NT][16], uint32_t stage, int pitch, int len, int k0, int klim, Row row,
                                          uint32_t ntm, int lane, Wait wait) {
  const int g = lane >> 2, t = lane & 3;
  const int nkb = (len + 63) >> 6;
  wait();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (!((ntm >> nt) & 1u)) continue;
    const float* rp[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) rp[n] = row(nt, n);
#pragma unroll 2
    for (int kb = 0; kb < nkb; ++kb) {
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
template <typename W, int NT>
__global__ void __launch_bounds__(kThreads, 1) moe_few_kernel(const Args a) {
  using X = typename W::X;
  constexpr bool kF32 = W::kSize == 4;
  constexpr int kKC = kPiece / W::kSize;  // values of a full stage row
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<NT>& s = *reinterpret_cast<Smem<NT>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int G = gridDim.x, cta = blockIdx.x;
  const uint32_t ring = smem_u32(smem_raw) + (uint32_t)((sizeof(Smem<NT>) + 127) / 128 * 128) +
                        (uint32_t)(warp * a.stages * 16 * a.pitch);
  const uint32_t bars = smem_u32(&s.bar[warp][0]);
  volatile int* abort_flag = &s.abort;

  if (lane < a.stages) mbar_init(bars + 8 * lane, 1);
  fence_mbar_init();
  for (int i = threadIdx.x; i < DSCA_MAX_EXPERTS; i += kThreads) s.emask[i] = 0u;
  if (threadIdx.x == 0) {
    s.abort = 0;
    s.n_act = 0;
  }
  __syncthreads();

  // ---- this warp's list of stages.  GEMM1: units cta, cta + G, ... of the shared expert, then of
  // the routed experts (the first of them on the CTA behind the last shared unit's); of every unit
  // the warp has its own range of k.  GEMM2: tiles cta, cta + G, ...; the pieces of the shared row,
  // then of the active experts' rows, go round the warps.
  const int k1a = min(a.d, warp * a.kc1), k1b = min(a.d, k1a + a.kc1);
  const int ppu = (k1b - k1a + kKC - 1) / kKC;  // stages a unit (0: this warp has no share of d)
  const int nu_s = a.ups > cta ? (a.ups - cta + G - 1) / G : 0;
  const int r_first = (cta + G - a.ups % G) % G;
  const int n2s = (a.k2s + kKC - 1) / kKC, n2r = (a.k2 + kKC - 1) / kKC;
  int nu_r = 0, n2w = 0, n1 = nu_s * ppu, total = n1;  // until the routing is known

  auto issue = [&](int i) {
    const int st = i % a.stages;
    const uint32_t bar = bars + 8 * st, dst = ring + (uint32_t)(st * 16 + (lane & 15)) * a.pitch;
    const uint8_t* src;
    int rows = 16, len;
    if (i < n1) {
      const int ul = i / ppu, kb = k1a + (i % ppu) * kKC;
      const bool sh = ul < nu_s;
      const int r = sh ? cta + ul * G : r_first + (ul - nu_s) * G;
      const int u = sh ? r : r % a.upe, e = sh ? 0 : s.act[r / a.upe];
      const int l = lane & 15;
      const int ch = 8 * u + (l & 7);
      const int row = a.glu ? (ch >> 7) * 256 + (ch & 127) + (l >> 3) * 128 : 16 * u + l;
      len = min(kKC, k1b - kb) * W::kSize;
      src = (sh ? a.ws1 : a.w1) + (((size_t)e * a.n1p + row) * a.d + kb) * W::kSize;
    } else {
      const int j = i - n1, tile = cta + (j / n2w) * G, q = warp + kWarps * (j % n2w);
      const int r0 = tile * a.rt;
      rows = min(a.rt, a.d - r0);
      const bool sh = q < n2s;
      const int e = sh ? 0 : s.act[(q - n2s) / n2r], kb = (sh ? q : (q - n2s) % n2r) * kKC;
      const int row = r0 + min(lane & 15, rows - 1);
      len = (min(kKC, (sh ? a.k2s : a.k2) - kb) * W::kSize + 15) & ~15;
      src = sh ? a.ws2 + ((size_t)row * a.s_ip + kb) * W::kSize
               : a.w2 + (((size_t)e * a.dp + row) * a.ip + kb) * W::kSize;
    }
    if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(rows * len));
    __syncwarp();
    if (lane < rows) bulk_load(dst, src, (uint32_t)len, bar);
  };
  int issued = 0, done = 0;
  // every lane has read stage `done`: refill it with the stage that follows the last one issued
  // (none after an abort, so that the copies in flight can be waited for at the end)
  auto release = [&]() {
    const bool stop = __any_sync(0xffffffffu, *abort_flag != 0);
    ++done;
    if (issued < total && !stop) issue(issued++);
  };
  auto wait_stage = [&]() {
    mbar_wait(bars + 8 * (done % a.stages), (uint32_t)(done / a.stages) & 1u, abort_flag, a.err);
  };
  while (issued < min(a.stages, total)) issue(issued++);

  // ---- router: one warp a dot product, spread over the grid
  {
    const int R = a.E + (a.w_gate != nullptr ? 1 : 0), nd = a.T * R;
    for (int q = cta + warp * G; q < nd; q += kWarps * G) {
      const int t = q / R, r = q % R;
      const X* w = r < a.E ? reinterpret_cast<const X*>(a.w_router) + (size_t)r * a.d : reinterpret_cast<const X*>(a.w_gate);
      const double v = dot64(reinterpret_cast<const X*>(a.x) + (size_t)t * a.d, w, a.d, lane);
      if (lane == 0) a.lg[t * kLgPitch + r] = round_to<X>(v);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      if (cta < nd) ctr_add(a.ctr + kCtrLogits);
      ctr_wait(a.ctr + kCtrLogits, (uint32_t)min(nd, G), abort_flag, a.err);
    }
    __syncthreads();
  }
  for (int t = warp; t < a.T; t += kWarps) select_token<X, NT>(a, s, t, lane);
  __syncthreads();
  if (warp == 0) {
    const uint32_t m0 = s.emask[lane], m1 = s.emask[lane + 32];
    const uint32_t b0 = __ballot_sync(0xffffffffu, m0 != 0u), b1 = __ballot_sync(0xffffffffu, m1 != 0u);
    const uint32_t below = (1u << lane) - 1u;
    if (m0) s.act[__popc(b0 & below)] = (uint8_t)lane;
    if (m1) s.act[__popc(b0) + __popc(b1 & below)] = (uint8_t)(lane + 32);
    if (lane == 0) s.n_act = __popc(b0) + __popc(b1);
  }
  for (int i = threadIdx.x; i < DSCA_MAX_EXPERTS * 8 * NT; i += kThreads) {
    const int e = i / (8 * NT), t = i % (8 * NT);
    const uint32_t m = s.emask[e];
    if ((m >> t) & 1u) s.tok[e][__popc(m & ((1u << t) - 1u))] = (uint8_t)t;
  }
  __syncthreads();
  const int n_act = s.n_act;
  {
    const int units = n_act * a.upe;
    nu_r = units > r_first ? (units - r_first + G - 1) / G : 0;
    const int n2 = n2s + n_act * n2r;
    n2w = n2 > warp ? (n2 - warp + kWarps - 1) / kWarps : 0;
    const int tl = a.tiles > cta ? (a.tiles - cta + G - 1) / G : 0;
    n1 = (nu_s + nu_r) * ppu;
    total = n1 + tl * n2w;
  }
  while (issued < min(a.stages, total)) issue(issued++);

  // ---- GEMM1
  const size_t h_lo = (size_t)a.T * a.k * a.hp * 2, hs_lo = (size_t)a.T * a.hsp * 2;
  const int nw1 = (a.d + a.kc1 - 1) / a.kc1;  // warps with a share of d
  for (int ul = 0; ul < nu_s + nu_r; ++ul) {
    const bool sh = ul < nu_s;
    const int r = sh ? cta + ul * G : r_first + (ul - nu_s) * G;
    const int u = sh ? r : r % a.upe, e = sh ? 0 : s.act[r / a.upe];
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
      for (int p = 0; p < ppu; ++p) {
        const int kb = k1a + p * kKC, len = min(kKC, k1b - kb) * W::kSize;
        stage_fma<NT, false>(big, ring + (uint32_t)((done % a.stages) * 16) * a.pitch, a.pitch, len, kb, a.d, row, ntm, lane,
                             wait_stage);
        release();
      }
      f32_fold<NT>(big, acc, lane);
    } else {
      Rows<NT> b;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        b.p[nt] = 8 * nt + g < n_tok ? reinterpret_cast<const uint8_t*>(a.x) + (size_t)token(8 * nt + g) * a.d * 2 : nullptr;
      for (int p = 0; p < ppu; ++p) {
        const int kb = k1a + p * kKC, len = min(kKC, k1b - kb) * W::kSize;
        stage_mma<W, NT, 1>(acc, ring + (uint32_t)((done % a.stages) * 16) * a.pitch, a.pitch, len, kb, a.d, b, 0, ntm, lane,
                            wait_stage);
        release();
      }
    }
    float(*part)[NT][32][4] = s.part[ul & 1];
    if (ppu > 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        if ((ntm >> nt) & 1u) *reinterpret_cast<float4*>(part[warp][nt][lane]) = make_float4(acc[nt][0], acc[nt][1], acc[nt][2], acc[nt][3]);
    }
    // double buffered: this buffer is written again two units on, behind the next unit's barrier,
    // which the finishing warp reaches only after it has read it
    __syncthreads();
    if (warp == (ul & (kWarps - 1))) {
      for (int nt = 0; nt * 8 < n_tok; ++nt) {
        float4 v = *reinterpret_cast<const float4*>(part[0][nt][lane]);
        for (int w = 1; w < nw1; ++w) {
          const float4 o = *reinterpret_cast<const float4*>(part[w][nt][lane]);
          v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
        }
        float c[4] = {v.x, v.y, v.z, v.w};
        if constexpr (W::kSize == 1) {
          const int ch = 8 * u + g;
          const int r0 = a.glu ? (ch >> 7) * 256 + (ch & 127) : 16 * u + g, r1 = a.glu ? r0 + 128 : r0 + 8;
          const float* sc = sh ? a.ws1s : a.w1s + (size_t)e * a.n1p;
          const float s0 = sc[r0], s1 = sc[r1];
          c[0] *= s0; c[1] *= s0; c[2] *= s1; c[3] *= s1;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = nt * 8 + 2 * t4 + i;
          if (n >= n_tok) continue;
          const int tk = token(n), j = sh ? 0 : s.slot[e][tk];
          const float w = sh ? s.sg[tk] : s.wt[tk][j];
          const size_t at = sh ? (size_t)tk * a.hsp : ((size_t)tk * a.k + j) * a.hp;
          uint8_t* base = sh ? a.hs : a.h;
          auto put = [&](int ch, float val) {
            if constexpr (kF32) {
              reinterpret_cast<float*>(base)[at + ch] = val;
            } else {
              const __nv_bfloat16 hi = __float2bfloat16_rn(val);
              const float rest = val - __bfloat162float(hi);
              __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(base) + at + ch;
              o[0] = hi;
              // an infinite or NaN value is the high term alone
              o[(sh ? hs_lo : h_lo) / 2] = __float2bfloat16_rn(fabsf(val) <= 3.38e38f ? rest : 0.0f);
            }
          };
          if (a.glu) {
            put(8 * u + g, w * (c[i] / (1.0f + expf(-c[i])) * c[2 + i]));
          } else {
            put(16 * u + g, w * fmaxf(c[i], 0.0f));
            put(16 * u + g + 8, w * fmaxf(c[2 + i], 0.0f));
          }
        }
      }
      __syncwarp();
      if (lane == 0) ctr_add(a.ctr + (sh ? kCtrShared : kCtrRouted));
    }
  }

  // ---- GEMM2
  bool have_s = n2s == 0, have_r = false;
  for (int tile = cta, tn = 0; tile < a.tiles; tile += G, ++tn) {
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
    for (int jj = 0; jj < n2w; ++jj) {
      const int q = warp + kWarps * jj;
      const bool sh = q < n2s;
      if (sh ? !have_s : !have_r) {
        // the intermediates come from every CTA's finishing warps
        if (lane == 0) {
          if (sh) ctr_wait(a.ctr + kCtrShared, (uint32_t)a.ups, abort_flag, a.err);
          else ctr_wait(a.ctr + kCtrRouted, (uint32_t)(n_act * a.upe), abort_flag, a.err);
        }
        __syncwarp();
        if (sh) have_s = true; else have_r = true;
      }
      const int e = sh ? 0 : s.act[(q - n2s) / n2r], kb = (sh ? q : (q - n2s) % n2r) * kKC;
      const int kend = sh ? a.k2s : a.k2;
      const int len = (min(kKC, kend - kb) * W::kSize + 15) & ~15;
      const uint32_t mask = sh ? (a.T >= 32 ? 0xffffffffu : (1u << a.T) - 1u) : s.emask[e];
      uint32_t ntm = 0u;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) ntm |= ((mask >> (8 * nt)) & 0xffu) ? 1u << nt : 0u;
      const uint32_t st = ring + (uint32_t)((done % a.stages) * 16) * a.pitch;
      auto at = [&](int tk) { return sh ? (size_t)tk * a.hsp : ((size_t)tk * a.k + s.slot[e][tk]) * a.hp; };
      const uint8_t* base = sh ? a.hs : a.h;
      if constexpr (kF32) {
        auto row = [&](int nt, int n) {
          return (mask >> (8 * nt + n)) & 1u ? reinterpret_cast<const float*>(base) + at(8 * nt + n) : nullptr;
        };
        stage_fma<NT, true>(big, st, a.pitch, len, kb, kend, row, ntm, lane, wait_stage);
      } else {
        Rows<NT> b;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) b.p[nt] = (mask >> (8 * nt + g)) & 1u ? base + at(8 * nt + g) * 2 : nullptr;
        if constexpr (W::kSize == 1) {
          // every (expert, row) has its own scale: this stage's sums are scaled before they join
          float part[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[nt][i] = 0.0f;
          const float* sc = sh ? a.ws2s : a.w2s + (size_t)e * a.dp;
          const float s0 = sc[r0 + min(g, rows - 1)], s1 = sc[r0 + min(g + 8, rows - 1)];
          stage_mma<W, NT, 2>(part, st, a.pitch, len, kb, kend, b, sh ? hs_lo : h_lo, ntm, lane, wait_stage);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            acc[nt][0] = fmaf(part[nt][0], s0, acc[nt][0]);
            acc[nt][1] = fmaf(part[nt][1], s0, acc[nt][1]);
            acc[nt][2] = fmaf(part[nt][2], s1, acc[nt][2]);
            acc[nt][3] = fmaf(part[nt][3], s1, acc[nt][3]);
          }
        } else {
          stage_mma<W, NT, 2>(acc, st, a.pitch, len, kb, kend, b, sh ? hs_lo : h_lo, ntm, lane, wait_stage);
        }
      }
      release();
    }
    if constexpr (kF32) f32_fold<NT>(big, acc, lane);
    float(*part)[NT][32][4] = s.part[tn & 1];
    if (tn == 0) __syncthreads();  // the last units' finishing warps may still read the buffers
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      *reinterpret_cast<float4*>(part[warp][nt][lane]) = make_float4(acc[nt][0], acc[nt][1], acc[nt][2], acc[nt][3]);
    __syncthreads();
    if (warp < NT) {
      float4 v = *reinterpret_cast<const float4*>(part[0][warp][lane]);
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 o = *reinterpret_cast<const float4*>(part[w][warp][lane]);
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
      }
      const float c[4] = {v.x, v.y, v.z, v.w};
      X* out = reinterpret_cast<X*>(a.out);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tk = warp * 8 + 2 * t4 + (i & 1), r = g + (i >> 1) * 8;
        if (tk < a.T && r < rows) out[(size_t)tk * a.d + r0 + r] = X(c[i]);
      }
    }
  }

  // ---- after an abort stages may still be on their way into this CTA's shared memory
  if (*abort_flag) {
    for (int i = max(0, issued - a.stages); i < issued; ++i) {
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(bars + 8 * (i % a.stages), (uint32_t)(i / a.stages) & 1u) && globaltimer_ns() - t0 < kWaitLimitNs) {
      }
    }
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
  // a warp's share of a GEMM1 row, and the bytes of a stage row: rows 64 bytes apart modulo 128, so
  // that the eight lanes of a shared-memory access phase (two rows) meet different banks
  a.kc1 = round_up((a.d + kWarps - 1) / kWarps, W::kBlock);
  const int widest = max(a.kc1, max(a.k2, a.k2s)) * W::kSize;
  a.pitch = round_up(min(kPiece, widest), 64);
  if (a.pitch % 128 == 0) a.pitch += 64;
  a.stages = min(kMaxStages, (kSmem - kFixed) / (kWarps * 16 * a.pitch));
  // output rows in tiles of at most 16, as even as they come over the SMs
  const int per = (a.d + sms - 1) / sms, nt = (per + 15) / 16;
  a.rt = (a.d + sms * nt - 1) / (sms * nt);
  a.tiles = (a.d + a.rt - 1) / a.rt;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)sms);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)(kFixed + kWarps * a.stages * 16 * a.pitch);
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
