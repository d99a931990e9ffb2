// The products of dense.cuh on the CUDA cores: any sizes, strides and majors.
//
// A CTA makes a 64 x 64 tile of the output (64 of m, 64 of n) over K slices of 16 in shared memory, 4 x 4
// values a thread; a gated product holds a gate and an up accumulator.  fp32 sums run over k in order.
#include "dense.cuh"

#include <algorithm>
#include <type_traits>

namespace dsca {
namespace dense {
namespace simt {

constexpr int BM = 64, BN = 64, BK = 16;

__device__ __forceinline__ float ld(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float ld(const __nv_bfloat16* p, int64_t i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ int ld(const int8_t* p, int64_t i) { return p[i]; }
__device__ __forceinline__ void st(float* p, float v) { *p = v; }
__device__ __forceinline__ void st(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// BK x 64 slice of an operand at rows r0, columns k0 (zeros outside).
template <typename T, typename A>
__device__ __forceinline__ void load_slice(A (*s)[64 + 4], const Operand& o, int rows, int K, int r0, int k0) {
  const T* p = reinterpret_cast<const T*>(o.p);
  for (int i = threadIdx.x; i < 64 * BK; i += 256) {
    const int r = o.mn ? i % 64 : i / BK, k = o.mn ? i / 64 : i % BK;
    A v = 0;
    if (r0 + r < rows && k0 + k < K)
      v = ld(p, o.mn ? (int64_t)(k0 + k) * o.ld + r0 + r : (int64_t)(r0 + r) * o.ld + k0 + k);
    s[k][r] = v;
  }
}

template <typename T, typename O, int EPI>
__global__ void __launch_bounds__(256) simt_kernel(const __grid_constant__ Job j) {
  using A = typename std::conditional<std::is_same<T, int8_t>::value, int, float>::type;
  constexpr bool kFast = sizeof(O) == 2;
  constexpr int NA = EPI == kGlu ? 2 : 1;
  __shared__ A sa[NA][BK][BM + 4], sb[BK][BN + 4];
  const Problem& p = j.prob[blockIdx.z];
  const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  for (int64_t tile = blockIdx.x; tile < (int64_t)tiles_m * tiles_n; tile += gridDim.x) {
    const int m0 = (int)(tile % tiles_m) * BM, n0 = (int)(tile / tiles_m) * BN;
    A acc[NA][4][4] = {};
    for (int s = 0; s < p.nseg; ++s)
      for (int k0 = 0; k0 < p.K; k0 += BK) {
        __syncthreads();
#pragma unroll
        for (int a = 0; a < NA; ++a) load_slice<T, A>(sa[a], p.a[EPI == kGlu ? a : s], p.M, p.K, m0, k0);
        load_slice<T, A>(sb, p.b[s], p.N, p.K, n0, k0);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < BK; ++k) {
          A vb[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) vb[i] = sb[k][ty * 4 + i];
#pragma unroll
          for (int a = 0; a < NA; ++a)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const A va = sa[a][k][tx + 16 * m];
#pragma unroll
              for (int n = 0; n < 4; ++n) acc[a][n][m] += va * vb[n];
            }
        }
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + ty * 4 + i;
      if (n >= p.N) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = m0 + tx + 16 * q;
        if (m >= p.M) continue;
        const int64_t at = (int64_t)n * p.ldo + m;
        float v = (float)acc[0][i][q];
        if (j.i8) v *= j.row_scale[n] * j.col_scale[0][m];
        O* out = reinterpret_cast<O*>(p.out);
        if constexpr (EPI == kStore) {
          if (j.bias != nullptr) v += ld(reinterpret_cast<const O*>(j.bias), m);
          st(out + at, v);
        } else if constexpr (EPI == kGlu) {
          float u = (float)acc[1][i][q];
          if (j.i8) u *= j.row_scale[n] * j.col_scale[1][m];
          st(out + at, gate<kFast>(v, j.act) * u);
          if (j.save_g != nullptr) {
            st(reinterpret_cast<O*>(j.save_g) + at, v);
            st(reinterpret_cast<O*>(j.save_u) + at, u);
          }
        } else {
          float a, da;
          gate_grad<kFast>(ld(reinterpret_cast<const O*>(j.save_g), at), j.act, &a, &da);
          st(out + at, v * ld(reinterpret_cast<const O*>(j.save_u), at) * da);
          st(reinterpret_cast<O*>(j.out2) + at, v * a);
        }
      }
    }
  }
}

template <typename T, typename O, int EPI>
int run(const Job& j, cudaStream_t stream) {
  int64_t most = 0;
  for (int i = 0; i < j.nprob; ++i)
    most = std::max<int64_t>(most, (int64_t)((j.prob[i].M + BM - 1) / BM) * ((j.prob[i].N + BN - 1) / BN));
  if (most == 0) return DSCA_OK;
  simt_kernel<T, O, EPI><<<dim3((unsigned)std::min<int64_t>(most, 1 << 20), 1, j.nprob), 256, 0, stream>>>(j);
  return cudaGetLastError() == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

template <typename T, typename O>
int by_epi(const Job& j, cudaStream_t stream) {
  if (j.epi == kStore) return run<T, O, kStore>(j, stream);
  if (j.epi == kGlu) return run<T, O, kGlu>(j, stream);
  if constexpr (std::is_same<T, O>::value) return run<T, O, kDGlu>(j, stream);
  return DSCA_ERR_BAD_ARG;
}

}  // namespace simt

int launch_simt(const Job& j, cudaStream_t stream) {
  if (j.i8)
    return j.dtype == DSCA_BF16 ? simt::by_epi<int8_t, __nv_bfloat16>(j, stream) : simt::by_epi<int8_t, float>(j, stream);
  return j.dtype == DSCA_BF16 ? simt::by_epi<__nv_bfloat16, __nv_bfloat16>(j, stream)
                              : simt::by_epi<float, float>(j, stream);
}

}  // namespace dense
}  // namespace dsca
