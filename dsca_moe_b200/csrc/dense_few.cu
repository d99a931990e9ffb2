// The products of dense.cuh for at most 16 tokens (fp32: 32): the weights' stream through the warps' registers.
//
// Such a call reads every weight once and has nothing else to wait for, so the weights go from memory straight into
// mma.sync fragments: a lane's 16 bytes of a weight row are eight bf16 (16 codes) in a row, and since a sum over k may
// take its terms in any order, the lane's four words serve as the fragments of two MMAs whose k slots are those
// very values; the tokens' words are taken from the same places.  No shared memory, no transposition.
//   tile      16 weight rows (m16); gated: 8 gate rows and the up rows of the same channels, so that a thread holds
//             both values of a channel
//   CTA       eight warps share the tile's k, batches of kU steps of 64 bytes a row, the next batch's weights on their
//             way while one is multiplied
//   cluster   where a product has fewer tiles than fill the GPU, up to eight CTAs share a tile's k and add their parts
//             over distributed shared memory, in the order of k
// A launch that follows another of the call (programmatic dependent) asks for its first weights before it waits for the
// tokens that the other one makes.
//
// fp32: both sides as three bf16 terms each, made in registers; the six products of terms down to 2^-16 of the largest
// (what is left out is below 2^-21 of it), since the CUDA cores took 8 tokens' loads of x for each weight (133 us, now 41).
//
// Bound by DRAM while it streams (92 MB a product and more: 5 to 6 TB/s), by launch, first and last loads and the joining of
// sums in small products: one token through a 2048 x 5632 block 18.4 us in bf16 (69 MB; 10.6 at the copy rate), 15.8 us with
// 8-bit weights (four launches); 16 tokens 23.4 us.  fp32 40 us for up to 8 tokens (138 MB; 28 with one product of terms, 33
// with three: the MMAs and the splitting), 16 tokens 53 us, 24 67 us, 32 82 us.
#include "dense.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

namespace dsca {
namespace dense {
namespace few {

constexpr int kWarps = 8;
constexpr int kU = 2;  // steps of a batch

struct Params {
  const void* w[2];
  int64_t ldw[2];
  const void* x;
  int64_t ldx;
  int T, M, K, tiles, act;
  int tail;  // codes behind the last whole 16 (K does not count them)
  int per;  // steps of one CTA of the cluster
  void* out;
  int64_t ldo;
  void* save_g;
  void* save_u;
  uint8_t* save_e;
  int groups;  // exponents of a saved row
  const float* row_scale;  // close: row_max
  int close;
  const float* col_scale[2];
  const void* bias;
  const uint8_t* ahead;  // the next product's weights: asked into L2 by this one's CTAs, `ahead_step` bytes each
  int64_t ahead_bytes;
  int ahead_step;
};

template <typename T>
struct Traits;
template <>
struct Traits<__nv_bfloat16> {
  using Acc = float;
  static constexpr int kVals = 8;  // of 16 bytes
};
template <>
struct Traits<int8_t> {
  using Acc = int;
  static constexpr int kVals = 16;
};
template <>
struct Traits<float> {
  using Acc = float;
  static constexpr int kVals = 4;
};

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row from element k on, zeros past K; `live` false: zeros.  kVec: rows on 16-byte boundaries that
// hold whole 16 bytes.  kOnce: read by this CTA alone.
template <typename T, bool kVec, bool kOnce>
__device__ __forceinline__ uint4 load16(const T* row, int k, int K, bool live) {
  constexpr int V = Traits<T>::kVals;
  if (!live || k >= K) return make_uint4(0u, 0u, 0u, 0u);
  if constexpr (kVec) {
    uint4 r;
    if constexpr (kOnce)
      asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(row + k));
    else
      asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(row + k));
    return r;
  } else {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (k + i < K) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(row[k + i]);
        else w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[k + i] << (16 * (i % 2));
      }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The products of the first n < 16 of 16 codes; what lies behind them is read and does not count.
__device__ __forceinline__ int tail_sum(const int8_t* x, const int8_t* w, int n) {
  const uint4 a = *reinterpret_cast<const uint4*>(x), b = *reinterpret_cast<const uint4*>(w);
  const uint32_t xs[4] = {a.x, a.y, a.z, a.w}, ws[4] = {b.x, b.y, b.z, b.w};
  int sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int keep = n - 4 * i;
    const uint32_t v = keep >= 4 ? xs[i] : keep > 0 ? xs[i] & ((1u << (8 * keep)) - 1u) : 0u;
    sum = __dp4a((int)v, (int)ws[i], sum);
  }
  return sum;
}

// Four fp32 values in a row as three bf16 terms, which hold them exactly: the upper 8 bits of significand cut off (never
// beyond the largest bf16), the next 8 rounded, what is left.  In each term's two words the values' own order.
struct Terms {
  uint32_t t[3][2];
  __device__ __forceinline__ explicit Terms(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t p = w[2 * i], q = w[2 * i + 1];
      const float rp = __uint_as_float(p) - __uint_as_float(p & 0xffff0000u), rq = __uint_as_float(q) - __uint_as_float(q & 0xffff0000u);
      const uint32_t m = pack_bf16x2(rp, rq);
      t[0][i] = __byte_perm(p, q, 0x7632);
      t[1][i] = m;
      t[2][i] = __byte_perm(__float_as_uint(rp - __uint_as_float(m << 16)), __float_as_uint(rq - __uint_as_float(m & 0xffff0000u)), 0x7632);
    }
  }
};

__device__ __forceinline__ float value(float v) { return v; }
__device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// NT groups of eight tokens.  (Two: four CTAs an SM, 16 tokens through a 2048 x 5632 bf16 block 23.3 us, 25.5 with the three
// that 70 registers a thread let in; three and four, fp32: two CTAs, 32 tokens 82 us, 103 without, for all that two values
// a thread are spilled; one group loses by any such bound.)
template <typename T, typename O, int EPI, int NT, bool kVecW, bool kVecX>
__global__ void __launch_bounds__(32 * kWarps, NT == 1 ? 0 : NT == 2 ? 4 : 2) few_kernel(const __grid_constant__ Params p) {
  using Acc = typename Traits<T>::Acc;
  constexpr int V = Traits<T>::kVals;
  constexpr int STEP = 4 * V;  // k of a step: 64 bytes of a row
  constexpr bool kGluE = EPI == kGlu;
  constexpr bool kF = std::is_same<T, float>::value;
  __shared__ Acc red[kWarps][16][8 * NT + 1];
  __shared__ Acc sum[16][8 * NT];
  const int warp = warp_id(), lane = lane_id(), g = lane >> 2, t4 = lane & 3;
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const int splits = (int)cluster.num_blocks(), split = (int)cluster.block_rank(), tile = blockIdx.x / splits;
  // this lane's two weight rows
  const int m0 = kGluE ? tile * 8 + g : tile * 16 + g, m1 = kGluE ? m0 : m0 + 8;
  const T* w0 = reinterpret_cast<const T*>(p.w[0]) + (int64_t)m0 * p.ldw[0];
  const T* w1 = reinterpret_cast<const T*>(kGluE ? p.w[1] : p.w[0]) + (int64_t)m1 * p.ldw[kGluE ? 1 : 0];
  const bool l0 = m0 < p.M, l1 = m1 < p.M;
  const int steps = (p.K + STEP - 1) / STEP;
  const int s_end = min(steps, (split + 1) * p.per);
  // the warps take steps in turn, so that together they read consecutive bytes of the rows
  int s = split * p.per + warp;
  pdl_launch_dependents();

  const T* x = reinterpret_cast<const T*>(p.x);
  uint4 a[kU], b[kU], u[kU][NT];
  auto fetch = [&](int s0, uint4 (&ra)[kU], uint4 (&rb)[kU]) {
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      const int at = s0 + i * kWarps, k = at * STEP + t4 * V;
      ra[i] = load16<T, kVecW, true>(w0, k, p.K, l0 && at < s_end);
      rb[i] = load16<T, kVecW, true>(w1, k, p.K, l1 && at < s_end);
    }
  };
  auto fetch_x = [&](int s0, uint4 (&ru)[kU][NT]) {
#pragma unroll
    for (int i = 0; i < kU; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int at = s0 + i * kWarps, tok = 8 * n + g;
        ru[i][n] = load16<T, kVecX, false>(x + (int64_t)tok * p.ldx, at * STEP + t4 * V, p.K, tok < p.T && at < s_end);
      }
  };
  fetch(s, a, b);
  pdl_wait();
  fetch_x(s, u);

  Acc acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = 0;
  for (; s < s_end; s += kU * kWarps) {
    uint4 na[kU], nb[kU], nu[kU][NT];
    fetch(s + kU * kWarps, na, nb);
    fetch_x(s + kU * kWarps, nu);
    if constexpr (kF) {
      // a batch's sums, the six products of terms down to 2^-16 of the largest; the smaller five apart, and both
      // added in fp32, since MMAs cut their sums off
      float big[NT][4], small[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) big[n][e] = small[n][e] = 0.0f;
#pragma unroll
      for (int i = 0; i < kU; ++i) {
        const Terms A(a[i]), B(b[i]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const Terms X(u[i][n]);
#pragma unroll
          for (int o = 2; o >= 0; --o)
#pragma unroll
            for (int w = 0; w <= o; ++w)
              mma(o == 0 ? big[n] : small[n], A.t[w][0], B.t[w][0], A.t[w][1], B.t[w][1], X.t[o - w][0], X.t[o - w][1]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] += big[n][e] + small[n][e];
    } else {
#pragma unroll
      for (int i = 0; i < kU; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma(acc[n], a[i].x, b[i].x, a[i].y, b[i].y, u[i][n].x, u[i][n].y);
          mma(acc[n], a[i].z, b[i].z, a[i].w, b[i].w, u[i][n].z, u[i][n].w);
        }
    }
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      a[i] = na[i];
      b[i] = nb[i];
#pragma unroll
      for (int n = 0; n < NT; ++n) u[i][n] = nu[i][n];
    }
  }

  // this CTA's weights have all been asked for: a share of the next product's, so that DRAM does not rest while the
  // sums are joined and the next launch starts
  if (p.ahead != nullptr && threadIdx.x == 0) {
    const int64_t from = (int64_t)blockIdx.x * p.ahead_step;
    const int64_t n = min((int64_t)p.ahead_step, p.ahead_bytes - from);
    if (n > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.ahead + from), "r"((uint32_t)n) : "memory");
  }

  // ---- the warps' parts, added in their order
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][g + 8 * (e >> 1)][8 * n + 2 * t4 + (e & 1)] = acc[n][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 8 * NT; i += 32 * kWarps) {
    const int r = i / (8 * NT), n = i % (8 * NT);
    Acc v = red[0][r][n];
#pragma unroll
    for (int k = 1; k < kWarps; ++k) v += red[k][r][n];
    sum[r][n] = v;
  }
  if (splits > 1) cluster.sync();
  else __syncthreads();

  // ---- the CTAs' parts in the order of k; each CTA finishes its share of the tokens
  constexpr int C = kGluE ? 8 : 16;  // output columns of a tile
  for (int i = threadIdx.x; i < C * 8 * NT; i += 32 * kWarps) {
    const int c = i % C, n = i / C;
    const int m = tile * C + c;
    if (n >= p.T || n % splits != split) continue;  // (whole groups of C threads)
    Acc va = 0, vb = 0;
    for (int k = 0; k < splits; ++k) {
      const Acc(*part)[8 * NT] = splits > 1 ? cluster.map_shared_rank(sum, k) : sum;
      va += part[c][n];
      if constexpr (kGluE) vb += part[c + 8][n];
    }
    const bool in = m < p.M;
    if constexpr (std::is_same<T, int8_t>::value) {
      if (p.tail != 0 && in) {
        const int8_t* xt = reinterpret_cast<const int8_t*>(p.x) + (int64_t)n * p.ldx + p.K;
        va += tail_sum(xt, reinterpret_cast<const int8_t*>(p.w[0]) + (int64_t)m * p.ldw[0] + p.K, p.tail);
        if constexpr (kGluE) vb += tail_sum(xt, reinterpret_cast<const int8_t*>(p.w[1]) + (int64_t)m * p.ldw[1] + p.K, p.tail);
      }
    }
    if constexpr (kGluE && std::is_same<T, int8_t>::value) {
      if (p.close) {
        if (in) {
          const int g[1] = {va}, u[1] = {vb};
          const float gs[1] = {p.col_scale[0][m]}, us[1] = {p.col_scale[1][m]};
          const Two xs[1] = {scale_two(p.row_scale[n])};
          float h[1];
          close_all(h, g, u, gs, us, xs, p.act);
          reinterpret_cast<float*>(p.out)[(int64_t)n * p.ldo + m] = h[0];
        }
        continue;
      }
    }
    float v = (float)va, u = (float)vb;
    if constexpr (std::is_same<T, int8_t>::value) {
      const float rs = p.row_scale[n];
      constexpr bool kBigI8 = !kGluE && sizeof(O) == 4;  // as in the other kernel
      v = in ? scaled<kBigI8>(va, p.col_scale[0][m], rs) : 0.0f;
      if constexpr (kGluE) u = in ? scaled<kBigI8>(vb, p.col_scale[1][m], rs) : 0.0f;
    }
    if constexpr (kGluE) {
      if (p.save_g != nullptr) {
        if constexpr (sizeof(O) == 2) {
          // the exponents of eight channels (the other kernels write four equal ones for 32)
          const unsigned mask = 0xffu << (lane & 24);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float own = h ? u : v;
            float big = in && fabsf(own) <= 3.4028234663852886e38f ? fabsf(own) : 0.0f;
#pragma unroll
            for (int o = 4; o > 0; o /= 2) big = fmaxf(big, __shfl_xor_sync(mask, big, o));
            const uint32_t e = f16_exp(big);
            if (in) reinterpret_cast<__half*>(h ? p.save_u : p.save_g)[(int64_t)n * p.ldo + m] = __float2half_rn(own * f16_factor(e));
            if (c == 0) p.save_e[((int64_t)h * p.T + n) * p.groups + tile] = (uint8_t)e;
          }
        } else if (in) {
          reinterpret_cast<float*>(p.save_g)[(int64_t)n * p.ldo + m] = v;
          reinterpret_cast<float*>(p.save_u)[(int64_t)n * p.ldo + m] = u;
        }
      }
      v = gate<!kF>(v, p.act) * u;
    } else if constexpr (std::is_same<T, int8_t>::value) {
      if (p.bias != nullptr && in) v += value(reinterpret_cast<const O*>(p.bias)[m]);
    }
    if (in) put(reinterpret_cast<O*>(p.out) + (int64_t)n * p.ldo + m, v);
  }
  if (splits > 1) cluster.sync();  // until every CTA has read this one's part
}

template <typename T, typename O, int EPI, int NT, bool kVecW, bool kVecX>
int launch(Params& p, bool pdl, cudaStream_t stream) {
  constexpr int STEP = 4 * Traits<T>::kVals;
  p.tiles = (p.M + (EPI == kGlu ? 8 : 16) - 1) / (EPI == kGlu ? 8 : 16);
  const int steps = std::max(1, (p.K + STEP - 1) / STEP), sms = current_device_sms();
  // CTAs to a tile: up to some three CTAs an SM, and a whole batch of steps for each warp
  int splits = 1;
  while (splits < 8 && p.tiles * splits * 2 <= 4 * sms && steps >= splits * 2 * kU * kWarps) splits *= 2;
  p.per = (steps + splits - 1) / splits;
  const int ctas = splits * p.tiles;
  p.ahead_step = (int)(((p.ahead_bytes + ctas - 1) / ctas + 127) / 128 * 128);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(splits * p.tiles));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, few_kernel<T, O, EPI, NT, kVecW, kVecX>, p) == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

template <typename T, typename O, int EPI, int NT>
int by_vec(Params& p, bool vw, bool vx, bool pdl, cudaStream_t stream) {
  if constexpr (std::is_same<T, int8_t>::value) return launch<T, O, EPI, NT, true, true>(p, pdl, stream);
  else {
    if (vw && vx) return launch<T, O, EPI, NT, true, true>(p, pdl, stream);
    // h lies on 16-byte boundaries whatever the weights do, but a row of it need not be whole 16 bytes wide
    return launch<T, O, EPI, NT, false, false>(p, pdl, stream);
  }
}

template <typename T, typename O, int EPI>
int by_tokens(Params& p, bool vw, bool vx, bool pdl, cudaStream_t stream) {
  if (p.T <= 8) return by_vec<T, O, EPI, 1>(p, vw, vx, pdl, stream);
  if constexpr (std::is_same<T, float>::value) {
    if (p.T > 24) return by_vec<T, O, EPI, 4>(p, vw, vx, pdl, stream);
    if (p.T > 16) return by_vec<T, O, EPI, 3>(p, vw, vx, pdl, stream);
  }
  return by_vec<T, O, EPI, 2>(p, vw, vx, pdl, stream);
}

}  // namespace few

bool few_fits(const Job& j, bool alone) {
  // Against the tensor-memory products, us (sets of weights larger than L2, 2048 wide).  Up to 8 tokens: bf16 block of 5632
  // 19 | 31, of 45056 99 | 106; 8-bit product of 5632 6 | 10, of 151936 59.5 | 59.  9 to 16 tokens: bf16 block of 5632
  // 23 | 31, of 22528 (185 MB of gate and up) 66 | 66, of 45056 121 | 107; 8-bit block of 22528 50 | 60; but 8-bit product of
  // 5632 (12 MB) 7.6 | 9.7, of 11264 11.9 | 11.5, of 45056 29 | 24, whose other form has no operands to lay out.  17 to 24
  // tokens: bf16 block of 5632 33 | 31, 8-bit 28 | 29, 8-bit product 10.8 | 9.8.  fp32,
  // whose other form splits the weights in memory first: block of 5632 1 token 40 | 122, 16 tokens 53 | 122,
  // 24 67 | 122, 32 82 | 122; of 11008 (4096 wide) 32 271 | 417; 712 x 1021 32 18 | 33
  const Problem& s = j.prob[0];
  if (j.nprob != 1 || s.nseg != 1 || j.epi == kDGlu || s.a[0].mn) return false;
  if (s.N <= 8 || (!j.i8 && j.dtype == DSCA_F32)) return s.N <= 32;
  const int64_t bytes = (int64_t)s.M * s.K * (j.i8 ? 1 : 2) * (j.epi == kGlu ? 2 : 1);
  return s.N <= 16 && bytes <= (alone ? 16ll << 20 : 128ll << 20);
}

int launch_few(const Job& j, const Job* next, bool pdl, cudaStream_t stream) {
  const Problem& s = j.prob[0];
  few::Params p = {};
  const int es = j.i8 ? 1 : j.dtype == DSCA_BF16 ? 2 : 4;
  auto whole = [&](const Operand& o) { return reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.ld * es % 16 == 0 && s.K * es % 16 == 0; };
  p.w[0] = s.a[0].p; p.ldw[0] = s.a[0].ld;
  p.w[1] = s.a[1].p; p.ldw[1] = s.a[1].ld;
  p.x = s.b[0].p; p.ldx = s.b[0].ld;
  const bool vw = whole(s.a[0]) && (j.epi != kGlu || whole(s.a[1])), vx = whole(s.b[0]);
  p.T = s.N; p.M = s.M;
  p.tail = j.i8 ? s.K % 16 : 0;
  p.K = s.K - p.tail;
  p.act = j.act;
  p.out = s.out; p.ldo = s.ldo;
  p.save_g = j.save_g; p.save_u = j.save_u; p.save_e = j.save_e; p.groups = exp_groups(s.M);
  p.close = j.row_max != nullptr;
  p.row_scale = p.close ? j.row_max : j.row_scale; p.col_scale[0] = j.col_scale[0]; p.col_scale[1] = j.col_scale[1]; p.bias = j.bias;
  if (next != nullptr) {
    const Operand& w = next->prob[0].a[0];
    const int64_t bytes = ((next->prob[0].M - 1) * w.ld + next->prob[0].K) * es & ~15ll;  // up to the last row's end
    // rows that (nearly) follow one another, and no more than a part of L2 keeps
    if (reinterpret_cast<uintptr_t>(w.p) % 16 == 0 && w.ld < next->prob[0].K + 16 && bytes <= (48 << 20)) {
      p.ahead = reinterpret_cast<const uint8_t*>(w.p);
      p.ahead_bytes = bytes;
    }
  }
  using B = __nv_bfloat16;
  if (j.i8) {
    if (j.epi == kGlu) return few::by_tokens<int8_t, float, kGlu>(p, true, true, pdl, stream);
    return j.dtype == DSCA_BF16 ? few::by_tokens<int8_t, B, kStore>(p, true, true, pdl, stream)
                                : few::by_tokens<int8_t, float, kStore>(p, true, true, pdl, stream);
  }
  if (j.dtype == DSCA_BF16)
    return j.epi == kGlu ? few::by_tokens<B, B, kGlu>(p, vw, vx, pdl, stream) : few::by_tokens<B, B, kStore>(p, vw, vx, pdl, stream);
  return j.epi == kGlu ? few::by_tokens<float, float, kGlu>(p, vw, vx, pdl, stream)
                       : few::by_tokens<float, float, kStore>(p, vw, vx, pdl, stream);
}

}  // namespace dense
}  // namespace dsca
