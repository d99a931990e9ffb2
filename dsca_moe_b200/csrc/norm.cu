// Root-mean-square norm in front of an MoE block, with the residual's addition and an optional
// 8-bit copy of the normed rows:
//
//   h = round(x + r);   y = w * h / sqrt(sum(h^2) / d + eps)
//
// h is rounded to the rows' type before it is squared, because that rounded row is the residual
// stream that the layers behind it add to.  The squares, their sum and y are fp32; y is rounded
// once, when it is stored.
//
// 8-bit rows: "e4m3" scales the unrounded y by s = max|y| / 448 (1 for a zero row), the row format
// of the fp8 expert weights; "split" writes the rounded y as two e4m3 terms with a power-of-two
// scale (fp8_split.cuh), the token operand of the fp8-weight GEMMs.
//
// One pass over the data: a row lives in the registers of its TPR threads (up to 64 values each)
// between the sum and the stores, so DRAM sees every input and output once.
#include "common.cuh"
#include "dsca_b200_block.h"
#include "fp8_split.cuh"

namespace dsca {
namespace norm {

struct Args {
  const void* x;
  const void* res;
  const void* w;
  void* y;
  void* h;
  uint8_t* q;
  float* scale;
  long long ld_x, ld_res, ld_y, ld_h;
  int rows, d, w_f32, quant;
  int vx, vres, vw;  // rows of x / residual / the weight start on 16-byte boundaries
  float eps;
};

// the larger of two values, NaN if one is (a row with a NaN gets a NaN scale)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float from_f(float v) { return v; }

// Eight consecutive values from a 16-byte aligned place.
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
// Eight consecutive values, one by one where they are not aligned (a warp's eight loads cover the
// same lines, so all but the first find them in L1).
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool aligned, float (&v)[8]) {
  if (aligned) {
    load8(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f<T>(p[j]);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                    pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = pack8(v);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// Sum / max over the TPR threads of a row, the same value on every thread; the order of the
// additions is fixed.  Every thread of the CTA calls it (rows past the end too).
template <int TPR, bool kMax>
__device__ __forceinline__ float row_reduce(float v, float* sm) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, off);
    v = kMax ? max_nan(v, o) : v + o;
  }
  if (TPR == 32) return v;
  const int warp = threadIdx.x >> 5, first = (threadIdx.x / TPR) * (TPR / 32);
  __syncthreads();  // sm may still be read for the row's previous reduction
  if ((threadIdx.x & 31) == 0) sm[warp] = v;
  __syncthreads();
  v = sm[first];
#pragma unroll
  for (int i = 1; i < TPR / 32; ++i) v = kMax ? max_nan(v, sm[first + i]) : v + sm[first + i];
  return v;
}

// VEC: d % 8 == 0 and every output row 16-byte aligned; thread i of a row holds chunks i, i + TPR, ...
// of eight values.  Otherwise the thread holds single values TPR apart, so that loads and stores
// stay coalesced at any width and alignment.
template <typename T, bool VEC, int VPT, int TPR, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_kernel(const Args a) {
  __shared__ float sm[THREADS / 32];
  const int tid = threadIdx.x % TPR;
  const long long row = (long long)blockIdx.x * (THREADS / TPR) + threadIdx.x / TPR;
  const bool live = row < a.rows;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld_x;
  const T* res = a.res ? reinterpret_cast<const T*>(a.res) + row * a.ld_res : nullptr;
  T* ho = a.h ? reinterpret_cast<T*>(a.h) + row * a.ld_h : nullptr;
  float v[VPT][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if constexpr (VEC) {
      const int c = (i * TPR + tid) * 8;
      if (live && c < a.d) {
        load8<T>(x + c, a.vx, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = (i * 8 + j) * TPR + tid;
        v[i][j] = live && c < a.d ? to_f<T>(x[c]) : 0.0f;
      }
    }
  }
  if (res != nullptr) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if constexpr (VEC) {
        const int c = (i * TPR + tid) * 8;
        if (live && c < a.d) {
          float r[8];
          load8<T>(res + c, a.vres, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = to_f<T>(from_f<T>(v[i][j] + r[j]));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = (i * 8 + j) * TPR + tid;
          if (live && c < a.d) v[i][j] = to_f<T>(from_f<T>(v[i][j] + to_f<T>(res[c])));
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
  ss = row_reduce<TPR, false>(ss, sm);
  // every thread of the row has read its inputs by now: the outputs may lie over them
  const float inv = __frsqrt_rn(__fdiv_rn(ss, (float)a.d) + a.eps);
  T* y = a.y ? reinterpret_cast<T*>(a.y) + row * a.ld_y : nullptr;
  float mx = 0.0f;
  uint32_t mbits = 0u;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if constexpr (VEC) {
      const int c = (i * TPR + tid) * 8;
      if (live && c < a.d) {
        if (ho != nullptr) store8(ho + c, v[i]);
        float w[8];
        if (a.w_f32) load8<float>(reinterpret_cast<const float*>(a.w) + c, a.vw, w);
        else load8<T>(reinterpret_cast<const T*>(a.w) + c, a.vw, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * inv * w[j];
        if (y != nullptr) store8(y + c, v[i]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = (i * 8 + j) * TPR + tid;
        if (live && c < a.d) {
          if (ho != nullptr) ho[c] = from_f<T>(v[i][j]);
          const float w = a.w_f32 ? reinterpret_cast<const float*>(a.w)[c] : to_f<T>(reinterpret_cast<const T*>(a.w)[c]);
          v[i][j] = v[i][j] * inv * w;
          if (y != nullptr) y[c] = from_f<T>(v[i][j]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mx = max_nan(mx, fabsf(v[i][j]));
      if constexpr (sizeof(T) == 2) mbits = max(mbits, (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v[i][j])) & 0x7fffu);
    }
  }
  if (a.quant == DSCA_NORM_Q_NONE) return;
  if (a.quant == DSCA_NORM_Q_E4M3) {
    mx = row_reduce<TPR, true>(mx, sm);
    const float s = (mx > 0.0f || mx != mx) ? __fdiv_rn(mx, 448.0f) : 1.0f;
    if (live && tid == 0) a.scale[row] = s;
    uint8_t* q = a.q + row * a.d;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if constexpr (VEC) {
        const int c = (i * TPR + tid) * 8;
        if (live && c < a.d) {
          uint32_t b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = f8s::e4m3x2_rn(__fdiv_rn(v[i][2 * j], s), __fdiv_rn(v[i][2 * j + 1], s));
          *reinterpret_cast<uint2*>(q + c) = make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = (i * 8 + j) * TPR + tid;
          if (live && c < a.d) q[c] = (uint8_t)f8s::e4m3x2_rn(__fdiv_rn(v[i][j], s), 0.0f);
        }
      }
    }
    return;
  }
  if constexpr (VEC && sizeof(T) == 2) {
    // bf16 bits without the sign order like integers, and are exact as fp32 integers
    mbits = (uint32_t)row_reduce<TPR, true>((float)mbits, sm);
    float s, is;
    f8s::row_scale(mbits, s, is);
    if (!live) return;
    if (tid == 0) a.scale[row] = is;
    const int kp = (a.d + 127) / 128 * 128;
    uint8_t* q = a.q + row * 2 * kp;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * TPR + tid) * 8;
      if (c < a.d) f8s::store_split(q, nullptr, kp, c / 8, pack8(v[i]), s);
    }
    for (int c = a.d + 8 * tid; c < kp; c += 8 * TPR) {
      *reinterpret_cast<uint2*>(q + c) = make_uint2(0u, 0u);
      *reinterpret_cast<uint2*>(q + kp + c) = make_uint2(0u, 0u);
    }
  }
}

template <typename T, bool VEC, int VPT, int TPR>
int launch(const Args& a, cudaStream_t stream) {
  constexpr int kThreads = TPR > 256 ? TPR : 256;
  constexpr int kRows = kThreads / TPR;
  const unsigned grid = (unsigned)(((long long)a.rows + kRows - 1) / kRows);
  rms_norm_kernel<T, VEC, VPT, TPR, kThreads><<<grid, kThreads, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

template <typename T, bool VEC>
int dispatch(const Args& a, cudaStream_t stream) {
  const int chunks = (a.d + 7) / 8;
  if (chunks <= 32) return launch<T, VEC, 1, 32>(a, stream);
  if (chunks <= 64) return launch<T, VEC, 2, 32>(a, stream);
  if (chunks <= 128) return launch<T, VEC, 4, 32>(a, stream);
  if (chunks <= 256) return launch<T, VEC, 8, 32>(a, stream);
  if (chunks <= 1024) return launch<T, VEC, 4, 256>(a, stream);
  if (chunks <= 2048) return launch<T, VEC, 8, 256>(a, stream);
  return launch<T, VEC, 8, 512>(a, stream);
}

}  // namespace norm

int launch_rms_norm(const dsca_rms_norm_args* p, cudaStream_t stream) {
  norm::Args a;
  a.x = p->x; a.res = p->residual; a.w = p->weight; a.y = p->y; a.h = p->residual_out;
  a.q = reinterpret_cast<uint8_t*>(p->q); a.scale = p->scale;
  a.ld_x = p->ld_x; a.ld_res = p->ld_residual; a.ld_y = p->ld_y; a.ld_h = p->ld_residual_out;
  a.rows = p->rows; a.d = p->d; a.w_f32 = p->weight_dtype == DSCA_F32; a.quant = p->quant; a.eps = p->eps;
  const int esz = p->dtype == DSCA_BF16 ? 2 : 4;
  auto ok = [&](const void* q, long long ld) {
    return q == nullptr || (reinterpret_cast<uintptr_t>(q) % 16 == 0 && (ld * esz) % 16 == 0);
  };
  a.vx = ok(a.x, a.ld_x);
  a.vres = ok(a.res, a.ld_res);
  a.vw = ok(a.w, 0);
  const bool vec = p->d % 8 == 0 && reinterpret_cast<uintptr_t>(p->q) % 8 == 0 && ok(a.y, a.ld_y) && ok(a.h, a.ld_h);
  if (p->quant == DSCA_NORM_Q_SPLIT && !vec) return DSCA_ERR_BAD_ARG;
  if (p->dtype == DSCA_BF16)
    return vec ? norm::dispatch<__nv_bfloat16, true>(a, stream) : norm::dispatch<__nv_bfloat16, false>(a, stream);
  return vec ? norm::dispatch<float, true>(a, stream) : norm::dispatch<float, false>(a, stream);
}

}  // namespace dsca
