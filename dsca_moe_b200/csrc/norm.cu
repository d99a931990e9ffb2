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
// scale (fp8_split.cuh), the layout of the token operand of the fp8-weight GEMMs.
//
// One pass over the data: a row lives in the registers of its TPR threads (up to 64 values each)
// between the sum and the stores, so DRAM sees every input and output once: it is bound by DRAM from a few
// thousand rows on (with residual 16384 x 2048 bf16 41.5 us, 99% of a copy's 6.5 TB/s; 20000 x 768 with split
// rows 26.5 us, 89%; 4096 x 2048 with e4m3 rows 14.5 us, 80%), below that by the launch and two trips to
// memory (1 x 2048 2.1 us).
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

// Eight consecutive values as they lie in memory: h of a bf16 row takes half the registers of its
// floats, and the loads of x, residual and weight are all on their way before the first is used.
template <typename T>
struct Chunk;
template <>
struct Chunk<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = u; }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    u = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
};
template <>
struct Chunk<float> {
  float4 a, b;
  __device__ __forceinline__ void zero() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    a = make_float4(v[0], v[1], v[2], v[3]);
    b = make_float4(v[4], v[5], v[6], v[7]);
  }
};

__device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float one(const float* p) { return *p; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }

// Thread tid's chunk i of a row.  kVec (d % 8 == 0): eight consecutive values, loaded one by one where
// the row is not aligned (a warp's eight loads cover the same lines, so all but the first find them
// in L1).  Otherwise single values TPR apart, so that loads and stores stay coalesced at any width.
template <bool kVec, int TPR>
__device__ __forceinline__ int column(int i, int j, int tid) {
  return kVec ? (i * TPR + tid) * 8 + j : (i * 8 + j) * TPR + tid;
}
// Reads chunks i0 .. i0 + N - 1 of a row: every load is issued before the first value is packed.
template <typename T, bool kVec, int TPR, int N>
__device__ __forceinline__ void read(Chunk<T> (&c)[N], const T* row, bool aligned, int i0, int tid, int d) {
  if (kVec && aligned) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = column<true, TPR>(i0 + i, 0, tid);
      if (k < d) c[i].load(row + k);
      else c[i].zero();
    }
    return;
  }
  T raw[N][8];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = column<kVec, TPR>(i0 + i, j, tid);
      raw[i][j] = k < d ? row[k] : T(0.0f);
    }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = one(&raw[i][j]);
    c[i].set(v);
  }
}
template <typename T, bool kVec, int TPR>
__device__ __forceinline__ void write(const Chunk<T>& c, T* row, int i, int tid, int d) {
  if constexpr (kVec) {
    const int k = column<true, TPR>(i, 0, tid);
    if (k < d) c.store(row + k);
  } else {
    float v[8];
    c.get(v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = column<false, TPR>(i, j, tid);
      if (k < d) put(row + k, v[j]);
    }
  }
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

template <typename T, bool kVec, int VPT, int TPR, int THREADS, int QUANT>
__global__ void __launch_bounds__(THREADS) rms_norm_kernel(const Args a) {
  __shared__ float sm[THREADS / 32];
  const int tid = threadIdx.x % TPR;
  const long long row = (long long)blockIdx.x * (THREADS / TPR) + threadIdx.x / TPR;
  const bool live = row < a.rows;
  const int d = live ? a.d : 0;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld_x;
  // residual and weight in registers too, unless the row alone fills them (fp32, eight chunks)
  constexpr bool kHold = VPT * sizeof(T) <= 16;
  constexpr int kN = kHold ? VPT : 1;
  const bool w_held = kHold && !a.w_f32;
  const T* res = a.res ? reinterpret_cast<const T*>(a.res) + row * a.ld_res : nullptr;
  const T* wt = reinterpret_cast<const T*>(a.w);
  Chunk<T> h[VPT], w[kN];
  read<T, kVec, TPR>(h, x, a.vx, 0, tid, d);
  auto add = [&](Chunk<T>& c, const Chunk<T>& r) {
    float v[8], u[8];
    c.get(v);
    r.get(u);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += u[j];
    c.set(v);  // rounded: this is the stream
  };
  if (res != nullptr) {
    Chunk<T> r[kN];
    if constexpr (kHold) {
      read<T, kVec, TPR>(r, res, a.vres, 0, tid, d);
      if (w_held) read<T, kVec, TPR>(w, wt, a.vw, 0, tid, a.d);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if constexpr (!kHold) read<T, kVec, TPR>(r, res, a.vres, i, tid, d);
      add(h[i], r[kHold ? i : 0]);
    }
  } else if (w_held) {
    if constexpr (kHold) read<T, kVec, TPR>(w, wt, a.vw, 0, tid, a.d);
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float v[8];
    h[i].get(v);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
  }
  ss = row_reduce<TPR, false>(ss, sm);
  // every thread of the row has read its inputs by now: the outputs may lie over them
  const float inv = __frsqrt_rn(__fdiv_rn(ss, (float)a.d) + a.eps);
  // chunk i of the unrounded y
  auto normed = [&](int i, float (&v)[8]) {
    float f[8];
    h[i].get(v);
    if (w_held) {
      w[kHold ? i : 0].get(f);
    } else if (!a.w_f32) {
      Chunk<T> c[1];
      read<T, kVec, TPR>(c, wt, a.vw, i, tid, a.d);
      c[0].get(f);
    } else {
      Chunk<float> c[1];
      read<float, kVec, TPR>(c, reinterpret_cast<const float*>(a.w), a.vw, i, tid, a.d);
      c[0].get(f);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * f[j] * inv;  // of bf16 values the first product is exact
  };
  T* ho = a.h ? reinterpret_cast<T*>(a.h) + row * a.ld_h : nullptr;
  T* yo = a.y ? reinterpret_cast<T*>(a.y) + row * a.ld_y : nullptr;
  float mx = 0.0f;
  uint32_t mbits = 0u;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (ho != nullptr) write<T, kVec, TPR>(h[i], ho, i, tid, d);
    float v[8];
    normed(i, v);
    Chunk<T> y;
    y.set(v);
    if (yo != nullptr) write<T, kVec, TPR>(y, yo, i, tid, d);
    if constexpr (QUANT == DSCA_NORM_Q_E4M3) {
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = max_nan(mx, fabsf(v[j]));
    }
    if constexpr (QUANT == DSCA_NORM_Q_SPLIT) {
      const uint32_t q = __vmaxu2(__vmaxu2(y.u.x & 0x7fff7fffu, y.u.y & 0x7fff7fffu), __vmaxu2(y.u.z & 0x7fff7fffu, y.u.w & 0x7fff7fffu));
      mbits = max(mbits, max(q & 0xffffu, q >> 16));
      h[i] = y;  // the rounded row, which the two terms stand for
    }
  }
  if constexpr (QUANT == DSCA_NORM_Q_E4M3) {
    mx = row_reduce<TPR, true>(mx, sm);
    float s = (mx > 0.0f || mx != mx) ? __fdiv_rn(mx, 448.0f) : 1.0f;
    if (s == 0.0f) s = __uint_as_float(1u);  // a row below 2^-141: not divided by zero
    if (live && tid == 0) a.scale[row] = s;
    // y / s rounded to fp32, from the rounded 1 / s and the remainder that it leaves (Markstein's correction; a
    // division an element took twice the kernel's time).  Rows so small or large that 1 / s or the remainder
    // leaves fp32's normal range do divide.
    const bool divide = !(s >= 1e-30f && s <= 1e30f);
    const float rs = divide ? 0.0f : __frcp_rn(s);
    uint8_t* q = a.q + row * a.d;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float v[8];
      normed(i, v);
      uint32_t b[4];
      if (divide) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fdiv_rn(v[j], s);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float t = v[j] * rs;
          v[j] = fmaf(fmaf(t, s, -v[j]), -rs, t);  // in this order a zero keeps its sign
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = f8s::e4m3x2_rn(v[2 * j], v[2 * j + 1]);
      if constexpr (kVec) {
        const int k = column<true, TPR>(i, 0, tid);
        if (k < d) *reinterpret_cast<uint2*>(q + k) = make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int k = column<false, TPR>(i, j, tid);
          if (k < d) q[k] = (uint8_t)(b[j / 2] >> (8 * (j & 1)));
        }
      }
    }
  }
  if constexpr (QUANT == DSCA_NORM_Q_SPLIT) {
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
      const int c = i * TPR + tid;
      if (c * 8 < a.d) f8s::store_split(q, nullptr, kp, c, h[i].u, s);
    }
    for (int c = a.d + 8 * tid; c < kp; c += 8 * TPR) {
      *reinterpret_cast<uint2*>(q + c) = make_uint2(0u, 0u);
      *reinterpret_cast<uint2*>(q + kp + c) = make_uint2(0u, 0u);
    }
  }
}

template <typename T, bool kVec, int VPT, int TPR, int QUANT>
int launch(const Args& a, cudaStream_t stream) {
  constexpr int kThreads = TPR > 256 ? TPR : 256;
  constexpr int kRows = kThreads / TPR;
  const unsigned grid = (unsigned)(((long long)a.rows + kRows - 1) / kRows);
  rms_norm_kernel<T, kVec, VPT, TPR, kThreads, QUANT><<<grid, kThreads, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

// Threads a row: with many rows as few as hold it in two or three chunks each (fp32: one), so that a
// row's reduction passes under the loads of the other rows on the SM; with few rows a whole CTA.
// 4096 x 2048 bf16: 128 threads with 2 chunks 10.4 us, 256 with 1 11.1 us, a warp with 8 12.9 us.
// Few threads against a whole CTA, bf16 with residual: 32 x 768 2.5 us, 2.1; 400 x 2048 3.0 us, 2.8; 600 x 768
// 2.9 us both; 1200 x 768 3.3 us, 3.9; 1200 x 2048 4.3 us, 4.7.
template <typename T, bool kVec, int QUANT>
int dispatch(const Args& a, cudaStream_t stream) {
  const int chunks = (a.d + 7) / 8;
  if (a.rows > 4 * current_device_sms() && chunks <= 256) {
    if (chunks <= 32) return launch<T, kVec, 1, 32, QUANT>(a, stream);
    if constexpr (sizeof(T) == 2) {
      if (chunks <= 64) return launch<T, kVec, 2, 32, QUANT>(a, stream);
      if (chunks <= 96) return launch<T, kVec, 3, 32, QUANT>(a, stream);
      if (chunks <= 128) return launch<T, kVec, 2, 64, QUANT>(a, stream);
      return launch<T, kVec, 2, 128, QUANT>(a, stream);
    } else {
      if (chunks <= 64) return launch<T, kVec, 1, 64, QUANT>(a, stream);
      if (chunks <= 128) return launch<T, kVec, 1, 128, QUANT>(a, stream);
    }
  }
  if (chunks <= 256) return launch<T, kVec, 1, 256, QUANT>(a, stream);
  if (chunks <= 512) return launch<T, kVec, 2, 256, QUANT>(a, stream);
  if (chunks <= 1024) return launch<T, kVec, 4, 256, QUANT>(a, stream);
  return launch<T, kVec, 8, 512, QUANT>(a, stream);
}

template <typename T>
int run(const Args& a, bool vec, cudaStream_t stream) {
  if (a.quant == DSCA_NORM_Q_E4M3)
    return vec ? dispatch<T, true, DSCA_NORM_Q_E4M3>(a, stream) : dispatch<T, false, DSCA_NORM_Q_E4M3>(a, stream);
  if constexpr (sizeof(T) == 2)
    if (a.quant == DSCA_NORM_Q_SPLIT) return vec ? dispatch<T, true, DSCA_NORM_Q_SPLIT>(a, stream) : DSCA_ERR_BAD_ARG;
  return vec ? dispatch<T, true, DSCA_NORM_Q_NONE>(a, stream) : dispatch<T, false, DSCA_NORM_Q_NONE>(a, stream);
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
  return p->dtype == DSCA_BF16 ? norm::run<__nv_bfloat16>(a, vec, stream) : norm::run<float>(a, vec, stream);
}

}  // namespace dsca
