// Matrices as the tensor-core products load them, several in one launch.
//
// bf16 rows that do not lie on 16-byte boundaries are copied to rows that do.  fp32 values are split into three
// bf16 terms, x = hi + mid + lo: each term is the nearest bf16 to what is left (8 bits of significand), so the
// three hold x to 2^-24 of its value.  A plane of rows follows a plane of rows; rows past the last up to the
// next multiple of 16 are zeros, since a product over rows takes 16 at a time.
#include "dense.cuh"

namespace dsca {
namespace dense {
namespace {

__device__ __forceinline__ void split3(float x, float* hi, float* mid, float* lo) {
  float h = round_bf16(x);
  if (isinf(h) && !isinf(x)) h = copysignf(3.3895313892515355e38f, x);  // the largest bf16
  const float r = isinf(h) || h != h ? 0.0f : x - h;  // exact
  const float m = round_bf16(r);
  *hi = h;
  *mid = m;
  *lo = r - m;  // exact; rounded when stored
}

__global__ void __launch_bounds__(256) relay_kernel(const __grid_constant__ RelayList L) {
  if (L.zero != nullptr)
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < L.zero_bytes / 4; i += (size_t)gridDim.x * 256)
      reinterpret_cast<uint32_t*>(L.zero)[i] = 0u;
  int e = 0;
  while (e + 1 < L.n && blockIdx.x >= L.item[e + 1].first) ++e;
  const Relay& m = L.item[e];
  const int64_t i = (int64_t)(blockIdx.x - m.first) * 256 + threadIdx.x;
  const int chunks = (int)(m.ldd / 8);
  const int64_t row = i / chunks;
  const int c = (int)(i - row * chunks) * 8;
  if (row >= m.rows_p) return;
  __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(m.dst) + row * m.ldd + c;
  const bool in = row < m.rows;
  if (m.dtype == DSCA_BF16) {
    const uint16_t* src = reinterpret_cast<const uint16_t*>(m.src) + row * m.lds + c;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t a = in && c + 2 * k < m.cols ? src[2 * k] : 0u, b = in && c + 2 * k + 1 < m.cols ? src[2 * k + 1] : 0u;
      w[k] = a | b << 16;
    }
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    return;
  }
  const float* src = reinterpret_cast<const float*>(m.src) + row * m.lds + c;
  float v[8];
  if (in && m.vec && c + 8 <= m.cols) {
    const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = in && c + k < m.cols ? src[k] : 0.0f;
  }
  float t[3][8];
#pragma unroll
  for (int k = 0; k < 8; ++k) split3(v[k], &t[0][k], &t[1][k], &t[2][k]);
#pragma unroll
  for (int p = 0; p < 3; ++p)
    *reinterpret_cast<uint4*>(dst + p * m.rows_p * m.ldd) =
        make_uint4(pack_bf16x2(t[p][0], t[p][1]), pack_bf16x2(t[p][2], t[p][3]), pack_bf16x2(t[p][4], t[p][5]),
                   pack_bf16x2(t[p][6], t[p][7]));
}

}  // namespace

int launch_relay(RelayList& L, cudaStream_t stream) {
  int64_t blocks = 0;
  for (int i = 0; i < L.n; ++i) {
    Relay& m = L.item[i];
    m.first = (uint32_t)blocks;
    m.vec = reinterpret_cast<uintptr_t>(m.src) % 16 == 0 && m.lds % 4 == 0;
    blocks += (m.rows_p * (m.ldd / 8) + 255) / 256;
  }
  if (blocks == 0) return DSCA_OK;
  if (blocks > 0x7fffffff) return DSCA_ERR_CAPACITY;
  relay_kernel<<<(unsigned)blocks, 256, 0, stream>>>(L);
  return cudaGetLastError() == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

}  // namespace dense
}  // namespace dsca
