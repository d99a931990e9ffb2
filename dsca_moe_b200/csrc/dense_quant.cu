// Rows in 8-bit integers: scale = max|x| / 127, code = the quotient 127 x / max|x| rounded to the
// nearest integer, ties to even, exactly.
//
// Why the exact quotient and not x / scale: the scale is rounded, so values half way between two
// codes (x = max|x| / 2 is 63.5) would fall to either side by the row.  A product with 127 / max|x| finds the code of
// all values but those close to a tie, which take the quotient: 127 x is exact in fp32 for a bf16 x and IEEE
// division rounds the exact quotient, which is never within 2^-9 of a tie without being one; for an fp32 x it is
// taken in 64 bits.
//
// Bound by DRAM from a few thousand rows on: a row is read once into registers (up to 8192 values;
// longer rows are read a second time from L2).
#include "dense.cuh"

#include <algorithm>

namespace dsca {
namespace dense {
namespace quant {

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ float value(const T* p, int64_t i) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(p[i]);
  else return p[i];
}

// The exact code of x in a row whose largest magnitude is amax (> 0).
template <typename T>
__device__ __noinline__ float exact_code(float x, float amax) {
  if (sizeof(T) == 2 && amax < 1e36f && amax > 1e-30f) return rintf(__fdiv_rn(__fmul_rn(127.0f, x), amax));
  return (float)rint(127.0 * (double)x / (double)amax);
}

// Four codes in a word.  inv is 127 / amax to 2^-23: a product with it is off by less than 2^-16, so only values
// that close to a tie need the exact quotient.  Adding 1.5 * 2^23 rounds to an integer, whose low byte is the code.
template <typename T>
__device__ __forceinline__ uint32_t codes4(const float* x, float amax, float inv) {
  constexpr float kRound = 12582912.0f;
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v = x[i] * inv;
    float r = v + kRound;
    if (fabsf(v - (r - kRound)) > 0.49996f) r = exact_code<T>(x[i], amax) + kRound;
    b[i] = __float_as_uint(r);
  }
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// TPR threads a row, CH chunks of eight values a thread in registers (CH = 0: longer rows).
template <typename T, int TPR, int CH, bool kVec>
__global__ void __launch_bounds__(256) quantize_kernel(const dsca_quantize_rows_args a) {
  __shared__ float red[8];
  constexpr int kRows = 256 / TPR;
  const int sub = threadIdx.x / TPR, tid = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * kRows + sub;
  const bool live = row < a.rows;
  pdl_launch_dependents();  // a product that follows asks for its first weights meanwhile
  pdl_wait();
  const T* x = reinterpret_cast<const T*>(a.x) + (live ? row : 0) * a.ld_x;
  float v[CH > 0 ? CH : 1][8];
  float m = 0.0f;
  auto load = [&](int c, float (&o)[8]) {
    if (kVec && c * 8 + 8 <= a.k) {
      if constexpr (sizeof(T) == 2) {
        const uint4 u = *reinterpret_cast<const uint4*>(x + c * 8);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[2 * i] = __uint_as_float(w[i] << 16);
          o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 f = *reinterpret_cast<const float4*>(x + c * 8 + 4 * i);
          o[4 * i] = f.x; o[4 * i + 1] = f.y; o[4 * i + 2] = f.z; o[4 * i + 3] = f.w;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = c * 8 + i < a.k ? value(x, c * 8 + i) : 0.0f;
    }
  };
  const int chunks = (int)((a.ld_q) / 8);  // those past k are zeros
  if (live) {
    if constexpr (CH > 0) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = i * TPR + tid;
        if (c < chunks) {
          load(c, v[i]);
#pragma unroll
          for (int e = 0; e < 8; ++e) m = max_nan(m, fabsf(v[i][e]));
        }
      }
    } else {
      for (int c = tid; c < chunks; c += TPR) {
        load(c, v[0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max_nan(m, fabsf(v[0][e]));
      }
    }
  }
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o /= 2) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if constexpr (TPR > 32) {
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = m;
    __syncthreads();
    m = red[sub * (TPR / 32)];
#pragma unroll
    for (int i = 1; i < TPR / 32; ++i) m = max_nan(m, red[sub * (TPR / 32) + i]);
  }
  if (!live) return;
  if (tid == 0) a.scale[row] = m == 0.0f ? 1.0f : __fdiv_rn(m, 127.0f);
  // codes mean nothing in a row that is not finite: zeros
  const bool usable = m > 0.0f && m < INFINITY;
  const bool ends = m < 1e-30f || m > 1e36f;  // 127 / m or 127 x leaves fp32's normal numbers
  const float inv = usable && !ends ? __fdiv_rn(127.0f, m) : 0.0f;
  auto store = [&](int c, float (&o)[8]) {
    uint2 w = make_uint2(0u, 0u);
    if (usable) {
      if (ends) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float r = exact_code<T>(o[e], m);
          const uint32_t byte = (uint32_t)((int)r & 255) << (8 * (e % 4));
          if (e < 4) w.x |= byte;
          else w.y |= byte;
        }
      } else {
        w = make_uint2(codes4<T>(o, m, inv), codes4<T>(o + 4, m, inv));
      }
    }
    *reinterpret_cast<uint2*>(a.q + row * a.ld_q + c * 8) = w;
  };
  if constexpr (CH > 0) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = i * TPR + tid;
      if (c < chunks) store(c, v[i]);
    }
  } else {
    for (int c = tid; c < chunks; c += TPR) {
      load(c, v[0]);
      store(c, v[0]);
    }
  }
}

template <typename T, int TPR, int CH>
int launch(const dsca_quantize_rows_args& a, bool pdl, cudaStream_t stream) {
  const unsigned grid = (unsigned)(((int64_t)a.rows * TPR + 255) / 256);
  const bool vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && (a.ld_x * (int64_t)sizeof(T)) % 16 == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  auto kern = vec ? quantize_kernel<T, TPR, CH, true> : quantize_kernel<T, TPR, CH, false>;
  return cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

template <typename T>
int run(const dsca_quantize_rows_args& a, bool pdl, cudaStream_t stream) {
  const int chunks = (int)(a.ld_q / 8);
  if (a.rows > 4 * current_device_sms()) {  // a warp a row while a warp holds it
    if (chunks <= 32) return launch<T, 32, 1>(a, pdl, stream);
    if (chunks <= 64) return launch<T, 32, 2>(a, pdl, stream);
    if (chunks <= 128) return launch<T, 64, 2>(a, pdl, stream);
    if (chunks <= 256) return launch<T, 128, 2>(a, pdl, stream);
  }
  if (chunks <= 256) return launch<T, 256, 1>(a, pdl, stream);
  if (chunks <= 512) return launch<T, 256, 2>(a, pdl, stream);
  if (chunks <= 768) return launch<T, 256, 3>(a, pdl, stream);
  if (chunks <= 1024) return launch<T, 256, 4>(a, pdl, stream);
  return launch<T, 256, 0>(a, pdl, stream);
}

}  // namespace quant

int launch_quantize_rows(const dsca_quantize_rows_args* a, bool pdl, cudaStream_t stream) {
  return a->dtype == DSCA_BF16 ? quant::run<__nv_bfloat16>(*a, pdl, stream) : quant::run<float>(*a, pdl, stream);
}

}  // namespace dense
}  // namespace dsca
