// Rows in 8-bit integers: scale = max|x| / 127, code = the quotient 127 x / max|x| rounded to the
// nearest integer, ties to even, exactly.
//
// Why the exact quotient and not x / scale: the scale is rounded, so values half way between two
// codes (x = max|x| / 2 is 63.5) would fall to either side by the row.  A product with 127 / max|x| is off by 2^-23
// of itself.  bf16 quotients are a tie or 2^-16 of themselves away from one, so the product rounded to 19 bits lies on
// the right side of each tie and on the tie where the quotient does; fp32 values close to a tie compare 127 x with the
// border times max|x|, exactly.  (The comparison for bf16 too: its ties are so common that a third of the warps took
// it, 16384 x 5632 57 us, now 43.)
//
// A row is read once (up to 8192 values; longer rows are read a second time from L2).  16384 x 5632 bf16 43 us (6.4
// TB/s, a copy's rate), 4096 x 5632 fp32 20.5 us (5.6 TB/s), one row 2.5 us.
#include "dense.cuh"

#include <algorithm>

namespace dsca {
namespace dense {
namespace quant {

// The code of x in a row whose largest magnitude is amax, by division in 64 bits.
__device__ __forceinline__ float divided_code(float x, float amax) { return (float)rint(127.0 * (double)x / (double)amax); }

// The code next to r that x has, r being one of the two integers around 127 x / amax: the sign of 127 x - h amax at the
// border h half way towards the other one decides, both products exact in 64 bits.
__device__ __forceinline__ float settled(float r, float toward, float x, float amax) {
  const float s = copysignf(1.0f, toward), h = r + 0.5f * s;
  const double over = fma(-(double)h, (double)amax, 127.0 * (double)x) * (double)s;  // beyond the border (> 0) or on it
  const bool odd = (int)r & 1;
  return over > 0.0 || (over == 0.0 && odd) ? r + s : r;
}

// Eight codes.  inv is 127 / amax to 2^-24, a product with it off by less than 2^-23 of itself.  Adding 1.5 * 2^23 rounds to
// an integer, ties to even, whose low byte is the code.
//
// bf16: x = X 2^a and amax = M 2^b with X and M from 128 to 255 (the quotient 127 X 2^e / M with e = a - b <= 0), so a
// border (2 j + 1) / 2 that is not the quotient is at least 2^e / (2 M) away from it, 1 / (254 X) > 2^-16 of it.  The product
// rounded to 19 bits, off by 2^-19 more, lies on the same side; and borders below 128, with their 8 bits, are among
// the 19-bit numbers, the nearest to products 2^-23 off.  (p - (33 p - 32 p), each step rounded: 24 - 5 bits.)
//
// fp32: only values within 2^-16 of a tie need the exact comparison; where one of the eight does, all take it.
template <typename T>
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float amax, float inv) {
  constexpr float kRound = 12582912.0f;
  uint32_t b[8];
  const float2 inv2 = make_float2(inv, inv), up = make_float2(kRound, kRound), minus = make_float2(-1.0f, -1.0f);
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {  // two values an instruction
      const float2 p = __fmul2_rn(make_float2(x[i], x[i + 1]), inv2), c = __ffma2_rn(p, make_float2(32.0f, 32.0f), p);
      const float2 low = __ffma2_rn(p, minus, c), r = __fadd2_rn(__ffma2_rn(low, minus, c), up);
      b[i] = __float_as_uint(r.x);
      b[i + 1] = __float_as_uint(r.y);
    }
  } else {
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float2 v = make_float2(x[i], x[i + 1]), r = __ffma2_rn(v, inv2, up);
      const float2 c = __ffma2_rn(r, minus, up);  // minus the code
      const float2 d = __ffma2_rn(v, inv2, c);
      far = fmaxf(far, fmaxf(fabsf(d.x), fabsf(d.y)));
      b[i] = __float_as_uint(r.x);
      b[i + 1] = __float_as_uint(r.y);
    }
    if (far > 0.49996f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float r = __uint_as_float(b[i]) - kRound;
        b[i] = __float_as_uint(settled(r, x[i] * inv - r, x[i], amax) + kRound);
      }
    }
  }
  return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

// Eight consecutive values as they lie in memory.
template <typename T>
struct Raw {
  static constexpr int W = sizeof(T) * 2;  // words
  uint32_t w[W];
  template <bool kVec>
  __device__ __forceinline__ void load(const T* x, int c, int k) {
    if (kVec && c * 8 + 8 <= k) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(x + c * 8) + 4 * i);
        w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c * 8 + i < k) {
          if constexpr (sizeof(T) == 2) w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(x)[c * 8 + i] << (16 * (i % 2));
          else w[i] = __float_as_uint(x[c * 8 + i]);
        }
    }
  }
  // the larger of m and the eight magnitudes, as bit patterns: of 32-bit values (NaN's are above infinity's); for bf16 two
  // 16-bit ones side by side, NaN where there is one
  __device__ __forceinline__ uint32_t largest(uint32_t m) const {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (sizeof(T) == 2) {
        __nv_bfloat162 x, y;
        memcpy(&x, &m, 4);
        memcpy(&y, &w[i], 4);
        x = __hmax2_nan(x, __habs2(y));
        memcpy(&m, &x, 4);
      } else m = max(m, w[i] & 0x7fffffffu);
    }
    return m;
  }
  static __device__ __forceinline__ float as_float(uint32_t m) {
    if constexpr (sizeof(T) == 2) return __uint_as_float(max(m << 16, m & 0xffff0000u));
    else return __uint_as_float(m);
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 2) return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return __uint_as_float(w[i]);
  }
};

// TPR threads a row, CH chunks of eight values a thread in registers (CH = 0: longer rows, read twice).  A CTA goes
// through rows with the next one's values on their way while one is turned into codes: with a CTA a row and no
// such overlap, 16384 x 5632 bf16 took 107 us.  bf16 rows of more than 2048 values come through a ring of two
// rows in shared memory, by copies that hold no registers (54 us with the next row in registers, 47 with a ring of
// one; 16384 x 4096 33 | 37); shorter rows do not gain (4096 x 2048 7.0 | 6.5 us), nor does fp32 (22 us either way).
template <typename T, int TPR, int CH, bool kVec>
constexpr bool in_ring() { return kVec && TPR * CH > 256 && sizeof(T) == 2; }
constexpr int kDepth = 2;

template <typename T, int TPR, int CH, bool kVec>
__global__ void __launch_bounds__(256) quantize_kernel(const dsca_quantize_rows_args a, float* row_max) {
  __shared__ uint32_t red[2][8];
  extern __shared__ uint4 ring[];  // [kDepth][CH][256], each thread's own chunks
  constexpr int kRows = 256 / TPR, N = CH > 0 ? CH : 1;
  constexpr bool kRing = in_ring<T, TPR, CH, kVec>();
  const int sub = threadIdx.x / TPR, tid = threadIdx.x % TPR;
  const int chunks = (int)(a.ld_q / 8);  // those past k are zeros
  const T* base = reinterpret_cast<const T*>(a.x);
  pdl_launch_dependents();  // a product that follows asks for its first weights meanwhile
  pdl_wait();
  Raw<T> next[N];
  auto fetch = [&](int64_t row, int slot) {
    if constexpr (CH > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = i * TPR + tid;
        if (row < a.rows && c < chunks) {
          if constexpr (kRing) {
            const int n = min(max(a.k - c * 8, 0), 8);  // the rest of the 16 bytes are zeros
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(&ring[(slot * N + i) * 256 + threadIdx.x])),
                         "l"(base + row * a.ld_x + (n > 0 ? c * 8 : 0)), "r"(2 * n)
                         : "memory");
          } else {
            next[i].template load<kVec>(base + row * a.ld_x, c, a.k);
          }
        }
      }
    }
    if constexpr (kRing) asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + sub;
  int slot = 0;
  fetch(row, 0);
  if constexpr (kRing) fetch(row + step, 1);
  // whole CTAs go round together (the reduction's barrier)
  for (int64_t first = (int64_t)blockIdx.x * kRows, it = 0; first < a.rows; first += step, row += step, ++it) {
    const bool live = row < a.rows;
    const T* x = base + (live ? row : 0) * a.ld_x;
    Raw<T> v[N];
    uint32_t bits = 0u;
    if constexpr (CH > 0) {
      if constexpr (kRing) asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if constexpr (kRing) *reinterpret_cast<uint4*>(v[i].w) = ring[(slot * N + i) * 256 + threadIdx.x];
        else v[i] = next[i];
        if (live && i * TPR + tid < chunks) bits = v[i].largest(bits);
      }
      if constexpr (!kRing) fetch(row + step, 0);
    } else if (live) {
      for (int c = tid; c < chunks; c += TPR) {
        v[0].template load<kVec>(x, c, a.k);
        bits = v[0].largest(bits);
      }
    }
    // a row's largest magnitude, NaN if there is one
    bits = __reduce_max_sync(0xffffffffu, __float_as_uint(Raw<T>::as_float(bits)));
    if constexpr (TPR > 32) {
      uint32_t* r = red[it & 1];  // two, so that one barrier a row is enough
      if (threadIdx.x % 32 == 0) r[threadIdx.x / 32] = bits;
      __syncthreads();
      bits = r[sub * (TPR / 32)];
#pragma unroll
      for (int i = 1; i < TPR / 32; ++i) bits = max(bits, r[sub * (TPR / 32) + i]);
    }
    const float m = __uint_as_float(bits);
    if constexpr (kRing) {  // m is known, so this thread's chunks have left the slot
      fetch(row + kDepth * step, slot);
      slot ^= 1;
    }
    if (!live) continue;
    if (tid == 0) {
      a.scale[row] = m == 0.0f ? 1.0f : __fdiv_rn(m, 127.0f);
      if (row_max != nullptr) row_max[row] = m;
    }
    // codes mean nothing in a row that is not finite: zeros
    const bool usable = m > 0.0f && m < INFINITY;
    const bool ends = m < 1e-30f || m > 1e36f;  // 127 / m or 127 x leaves fp32's normal numbers
    const float inv = usable && !ends ? __fdiv_rn(127.0f, m) : 0.0f;
    auto store = [&](int c, const Raw<T>& raw) {
      uint2 w = make_uint2(0u, 0u);
      if (usable) {
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = raw.get(e);
        if (!ends) {
          w = codes8<T>(o, m, inv);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t byte = (uint32_t)((int)divided_code(o[e], m) & 255) << (8 * (e % 4));
            if (e < 4) w.x |= byte;
            else w.y |= byte;
          }
        }
      }
      *reinterpret_cast<uint2*>(a.q + row * a.ld_q + c * 8) = w;
    };
    if constexpr (CH > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = i * TPR + tid;
        if (c < chunks) store(c, v[i]);
      }
    } else {
      for (int c = tid; c < chunks; c += TPR) {
        v[0].template load<kVec>(x, c, a.k);
        store(c, v[0]);
      }
    }
  }
}

template <typename T, int TPR, int CH>
int launch(const dsca_quantize_rows_args& a, float* row_max, bool pdl, cudaStream_t stream) {
  // CTAs go round, two for each that an SM holds at a time or nearly so (long fp32 rows: 80 registers a thread, three)
  constexpr int kCtas = sizeof(T) == 4 && CH > 2 ? 6 : 8;
  const unsigned grid = (unsigned)std::min<int64_t>(((int64_t)a.rows * TPR + 255) / 256, (int64_t)kCtas * current_device_sms());
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
  if (vec && in_ring<T, TPR, CH, true>()) cfg.dynamicSmemBytes = (size_t)kDepth * CH * 256 * 16;  // 24 or 32 KB
  auto kern = vec ? quantize_kernel<T, TPR, CH, true> : quantize_kernel<T, TPR, CH, false>;
  return cudaLaunchKernelEx(&cfg, kern, a, row_max) == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

// Rows of 64-bit values: the quotient in 64 bits, divided where the product with 127 / max is next to a tie.  TPR threads a
// row, four values each at a time; the row is read a second time from L1 or L2.
template <int TPR>
__global__ void __launch_bounds__(256) quantize64_kernel(const double* __restrict__ x, int rows, int k, int64_t ld, int8_t* q,
                                                         int64_t ld_q, float* scale) {
  __shared__ unsigned long long red[2][8];
  constexpr int kRows = 256 / TPR;
  const int sub = threadIdx.x / TPR, tid = threadIdx.x % TPR;
  const int pieces = (int)(ld_q / 4);
  pdl_launch_dependents();
  pdl_wait();
  int it = 0;
  for (int64_t first = (int64_t)blockIdx.x * kRows; first < rows; first += (int64_t)gridDim.x * kRows, it ^= 1) {
    const int64_t row = first + sub;
    const bool live = row < rows;
    const double* r = x + (live ? row : 0) * ld;
    // rows lie on 32-byte boundaries and hold a multiple of 16 values, of which those past k are not written
    auto load = [&](int c, double (&v)[4]) {
      const double2 a = c * 4 < k ? *reinterpret_cast<const double2*>(r + c * 4) : make_double2(0.0, 0.0);
      const double2 b = c * 4 + 2 < k ? *reinterpret_cast<const double2*>(r + c * 4 + 2) : make_double2(0.0, 0.0);
      v[0] = a.x;
      v[1] = c * 4 + 1 < k ? a.y : 0.0;
      v[2] = b.x;
      v[3] = c * 4 + 3 < k ? b.y : 0.0;
    };
    unsigned long long bits = 0;  // of the largest magnitude, a NaN's being the largest
    if (live) {
#pragma unroll 4
      for (int c = tid; c < pieces; c += TPR) {
        double v[4];
        load(c, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) bits = max(bits, (unsigned long long)__double_as_longlong(fabs(v[e])));
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
    if constexpr (TPR > 32) {
      if (threadIdx.x % 32 == 0) red[it][threadIdx.x / 32] = bits;
      __syncthreads();  // one a row: the next one writes the other half
#pragma unroll
      for (int i = 0; i < TPR / 32; ++i) bits = max(bits, red[it][sub * (TPR / 32) + i]);
    }
    if (!live) continue;
    const double m = __longlong_as_double((long long)bits);
    const float s = (float)(m / 127.0);
    if (tid == 0) scale[row] = m == 0.0 ? 1.0f : s;
    const bool usable = m > 0.0 && s < INFINITY;  // codes of other rows mean nothing
    const double inv = usable ? 127.0 / m : 0.0;
#pragma unroll 4
    for (int c = tid; c < pieces; c += TPR) {
      char4 w = make_char4(0, 0, 0, 0);
      if (usable) {
        double v[4];
        int o[4];
        load(c, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const double p = v[e] * inv;
          o[e] = __double2int_rn(p);
          if (fabs(p - (double)o[e]) > 0.5 - 1e-9) o[e] = __double2int_rn(127.0 * v[e] / m);  // p is good to 1e-13
        }
        w = make_char4((signed char)o[0], (signed char)o[1], (signed char)o[2], (signed char)o[3]);
      }
      *reinterpret_cast<char4*>(q + row * ld_q + c * 4) = w;
    }
  }
}

template <int TPR>
int launch64(const double* x, int rows, int k, int64_t ld, int8_t* q, int64_t ld_q, float* scale, bool pdl, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(((int64_t)rows * TPR + 255) / 256, (int64_t)8 * current_device_sms()));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, quantize64_kernel<TPR>, x, rows, k, ld, q, ld_q, scale) == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

template <typename T>
int run(const dsca_quantize_rows_args& a, float* row_max, bool pdl, cudaStream_t stream) {
  const int chunks = (int)(a.ld_q / 8);
  if (a.rows > 4 * current_device_sms()) {  // a warp a row while a warp holds it
    if (chunks <= 32) return launch<T, 32, 1>(a, row_max, pdl, stream);
    if (chunks <= 64) return launch<T, 32, 2>(a, row_max, pdl, stream);
    if (chunks <= 128) return launch<T, 64, 2>(a, row_max, pdl, stream);
    if (chunks <= 256) return launch<T, 128, 2>(a, row_max, pdl, stream);
  }
  if (chunks <= 256) return launch<T, 256, 1>(a, row_max, pdl, stream);
  if (chunks <= 512) return launch<T, 256, 2>(a, row_max, pdl, stream);
  if (chunks <= 768) return launch<T, 256, 3>(a, row_max, pdl, stream);
  if (chunks <= 1024) return launch<T, 256, 4>(a, row_max, pdl, stream);
  return launch<T, 256, 0>(a, row_max, pdl, stream);
}

}  // namespace quant

int launch_quantize_rows(const dsca_quantize_rows_args* a, float* row_max, bool pdl, cudaStream_t stream) {
  return a->dtype == DSCA_BF16 ? quant::run<__nv_bfloat16>(*a, row_max, pdl, stream) : quant::run<float>(*a, row_max, pdl, stream);
}

int launch_quantize_rows64(const double* x, int rows, int k, int64_t ld, int8_t* q, int64_t ld_q, float* scale, bool pdl,
                           cudaStream_t stream) {
  // a warp a row where there are rows for all of them and the rows are short
  return k <= 1024 && rows > 4 * current_device_sms() ? quant::launch64<32>(x, rows, k, ld, q, ld_q, scale, pdl, stream)
                                                      : quant::launch64<256>(x, rows, k, ld, q, ld_q, scale, pdl, stream);
}

}  // namespace dense
}  // namespace dsca
