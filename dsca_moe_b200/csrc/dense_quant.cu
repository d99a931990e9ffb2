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
//
// The intermediate of an 8-bit block on fp32 tokens takes the codes of its 64-bit value, although it comes in fp32 (kH, settle_kernel).
#include "dense.cuh"

#include <algorithm>
#include <type_traits>

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
// the 19-bit numbers, the nearest to products 2^-23 off.  (Veltkamp's splitting: 33 p - (33 p - p), each step rounded, 24 - 5 bits.)
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

// Rows of h (below): the largest value under which all codes are formed again, and the error of 127 h / max relative to itself:
// the bounds of h and of the largest, the rounded 127 / max and its product.
constexpr float kTiny = 1e-25f;
constexpr float kOpen = 2.1f * kCloseH + 2.4e-7f;

// Eight codes of h, and whether one of them is open.
__device__ __forceinline__ uint2 codes8_h(const float (&x)[8], float inv, bool& open) {
  constexpr float kRound = 12582912.0f;
  uint32_t b[8];
  const float2 inv2 = make_float2(inv, inv), up = make_float2(kRound, kRound), minus = make_float2(-1.0f, -1.0f);
  const float own = inv * kOpen;
  float far = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 v = make_float2(x[i], x[i + 1]), r = __ffma2_rn(v, inv2, up);
    const float2 c = __ffma2_rn(r, minus, up);  // minus the code
    const float2 d = __ffma2_rn(v, inv2, c);
    far = fmaxf(far, fmaxf(fmaf(fabsf(v.x), own, fabsf(d.x)), fmaf(fabsf(v.y), own, fabsf(d.y))));
    b[i] = __float_as_uint(r.x);
    b[i + 1] = __float_as_uint(r.y);
  }
  open |= far > 0.499999f;
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

// ---- The intermediate of an 8-bit block, by the codes of its 64-bit value (kH)
//
// h = act(g) u was formed within kCloseH of itself, and so was the row's largest.  Where that leaves open on which side of a border
// 127 h / max|h| lies (one value in 30000), warps form the h of that channel, and of those that may be the row's largest, again
// from the codes: two exact sums of d products, scales and gate in 64 bits.  Other rows' scale is off by kCloseH.
//
// A gate that is 0 in fp32 instead of 1e-36 and products below fp32's normal numbers matter only in rows whose largest value is
// tiny (kTiny): there all values are formed again.

// h of a row and channel in 64 bits, by a whole warp.  Codes of x past d are zeros, those of the weights do not count.
__device__ __noinline__ double warp_h(const dsca_gated_ffn_int8_args& a, int64_t row, int c, double xs) {
  const int8_t *x = a.q + row * a.ld_q, *g = a.w_gate + (int64_t)c * a.ld_gate, *u = a.w_up + (int64_t)c * a.ld_up;
  int sg = 0, su = 0;
#pragma unroll 4
  for (int i = 16 * (int)(threadIdx.x % 32); i < a.d; i += 512) {
    const int4 p = *reinterpret_cast<const int4*>(x + i), q = __ldg(reinterpret_cast<const int4*>(g + i)),
               r = __ldg(reinterpret_cast<const int4*>(u + i));
    sg = __dp4a(p.x, q.x, __dp4a(p.y, q.y, __dp4a(p.z, q.z, __dp4a(p.w, q.w, sg))));
    su = __dp4a(p.x, r.x, __dp4a(p.y, r.y, __dp4a(p.z, r.z, __dp4a(p.w, r.w, su))));
  }
  sg = __reduce_add_sync(0xffffffffu, sg);
  su = __reduce_add_sync(0xffffffffu, su);
  return gate64((double)sg * xs * (double)a.gate_scale[c], a.act) * ((double)su * xs * (double)a.up_scale[c]);
}

// TPR threads a row, CH chunks of eight values a thread in registers (CH = 0: longer rows, read twice).  A CTA goes
// through rows with the next one's values on their way while one is turned into codes: with a CTA a row and no
// such overlap, 16384 x 5632 bf16 took 107 us.  bf16 rows of more than 2048 values come through a ring of two
// rows in shared memory, by copies that hold no registers (54 us with the next row in registers, 47 with a ring of
// one; 16384 x 4096 33 | 37); shorter rows do not gain (4096 x 2048 7.0 | 6.5 us), nor does fp32 (22 us either way).
template <typename T, int TPR, int CH, bool kVec>
constexpr bool in_ring() { return kVec && TPR * CH > 256 && sizeof(T) == 2; }
constexpr int kDepth = 2;

// What the scales take: max / 127; the largest magnitude itself; max / 127 with the sign set where a code of the row (or of one
// that shares its CTA) is open.
enum Form { kScale = 0, kMax = 1, kH = 2 };

template <typename T, int TPR, int CH, bool kVec, int FORM>
__global__ void __launch_bounds__(256) quantize_kernel(const dsca_quantize_rows_args a) {
  static_assert(FORM == kScale || sizeof(T) == 4, "fp32 tokens");
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
    if (FORM != kH && !live) continue;
    const float scale = FORM == kMax ? m : m == 0.0f ? 1.0f : __fdiv_rn(m, 127.0f);
    if (FORM != kH && tid == 0) a.scale[row] = scale;
    // codes mean nothing in a row that is not finite: zeros
    const bool usable = m > 0.0f && m < INFINITY;
    const bool ends = FORM == kH ? m < kTiny : m < 1e-30f || m > 1e36f;  // 127 / m or 127 x leaves fp32's normal numbers
    bool open = FORM == kH && live && usable && ends;  // a code of this thread's
    const float inv = usable && !ends ? __fdiv_rn(127.0f, m) : 0.0f;
    auto store = [&](int c, const Raw<T>& raw) {
      uint2 w = make_uint2(0u, 0u);
      if (usable) {
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = raw.get(e);
        if constexpr (FORM == kH) {
          if (!ends) w = codes8_h(o, inv, open);
        } else if (!ends) {
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
        if (live && c < chunks) store(c, v[i]);
      }
    } else if (live) {
      for (int c = tid; c < chunks; c += TPR) {
        v[0].template load<kVec>(x, c, a.k);
        store(c, v[0]);
      }
    }
    if constexpr (FORM == kH) {
      bool any;
      if constexpr (TPR > 32) any = __syncthreads_or(open) != 0;
      else any = __any_sync(0xffffffffu, open) != 0;
      if (live && tid == 0) a.scale[row] = any && usable ? -scale : scale;
    }
  }
}

template <typename T, int TPR, int CH, int FORM>
int launch(const dsca_quantize_rows_args& a, bool pdl, cudaStream_t stream) {
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
  // (rows of h are on 16-byte boundaries)
  auto kern = FORM == kH || vec ? quantize_kernel<T, TPR, CH, true, FORM> : quantize_kernel<T, TPR, CH, FORM == kH, FORM>;
  return cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

template <typename T, int FORM>
int run(const dsca_quantize_rows_args& a, bool pdl, cudaStream_t stream) {
  const int chunks = (int)(a.ld_q / 8);
  if (a.rows > 4 * current_device_sms()) {  // a warp a row while a warp holds it
    if (chunks <= 32) return launch<T, 32, 1, FORM>(a, pdl, stream);
    if (chunks <= 64) return launch<T, 32, 2, FORM>(a, pdl, stream);
    if (chunks <= 128) return launch<T, 64, 2, FORM>(a, pdl, stream);
    if (chunks <= 256) return launch<T, 128, 2, FORM>(a, pdl, stream);
  }
  if (chunks <= 256) return launch<T, 256, 1, FORM>(a, pdl, stream);
  if (chunks <= 512) return launch<T, 256, 2, FORM>(a, pdl, stream);
  if (chunks <= 768) return launch<T, 256, 3, FORM>(a, pdl, stream);
  if (chunks <= 1024) return launch<T, 256, 4, FORM>(a, pdl, stream);
  return launch<T, 256, 0, FORM>(a, pdl, stream);
}

// Rows with open codes (their scale's sign is set): their largest value and those codes from 64 bits, a CTA a row.  The first open
// value of each lane is formed before the largest is known and held, so that most rows wait for one such sum.  A launch of its
// own: in the one above it took that kernel's registers and with them its speed (4096 x 5632 77 us, the two of them 42: 19 and 23).
__global__ void __launch_bounds__(256) settle_kernel(const __grid_constant__ dsca_gated_ffn_int8_args a) {
  __shared__ double red[2][8];
  const int lane = threadIdx.x % 32, k = a.inter;
  pdl_launch_dependents();
  pdl_wait();
  int it = 0;
  auto settle = [&](int64_t row, float s) {  // s: max / 127, rounded
    const float m = 127.0f * s;
    const bool all = m < 1.001f * kTiny;
    const float inv = all ? 0.0f : __fdiv_rn(1.0f, s), least = all ? 0.0f : m * (1.0f - kOpen - 2.4e-7f);
    const float* h = a.h + row * a.ld_h;
    const double xs = (double)a.scale[row] / 127.0;
    // f(channel, its lane, whether it may be the largest, whether its code is open) for each such value of the warp in turn
    auto scan = [&](auto f) {
      for (int c0 = 0; c0 < k; c0 += 8192) {  // 32 values a thread at a time
        float4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = c0 + 1024 * i + 4 * (int)threadIdx.x;  // rows hold a multiple of four values
          v[i] = at < k ? *reinterpret_cast<const float4*>(h + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        uint32_t top = 0, open = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float h4[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = h4[e] * inv;
            if (c0 + 1024 * i + 4 * (int)threadIdx.x + e < k) {
              top |= (uint32_t)(fabsf(h4[e]) >= least) << (4 * i + e);
              open |= (uint32_t)(all || fabsf(p - rintf(p)) > 0.499999f - fabsf(p) * (kOpen + 2.4e-7f)) << (4 * i + e);
            }
          }
        }
        uint32_t marks = top | open;
        for (unsigned any; (any = __ballot_sync(0xffffffffu, marks != 0u)) != 0u;) {
          const int src = __ffs(any) - 1, e = __ffs(__shfl_sync(0xffffffffu, marks, src)) - 1;
          const int c = c0 + 1024 * (e / 4) + 4 * ((int)(threadIdx.x & ~31u) + src) + e % 4;
          f(c, src, (__shfl_sync(0xffffffffu, top, src) >> e & 1u) != 0u, (__shfl_sync(0xffffffffu, open, src) >> e & 1u) != 0u);
          if (lane == src) marks &= marks - 1u;
        }
      }
    };
    double m64 = 0.0, held = 0.0;
    int held_c = -1;
    bool more = false;
    scan([&](int c, int src, bool top, bool open) {
      const bool hold = open && lane == src && held_c < 0;
      const double w = top || __any_sync(0xffffffffu, hold) ? warp_h(a, row, c, xs) : 0.0;
      if (top) m64 = fmax(m64, fabs(w));
      if (hold) {
        held = w;
        held_c = c;
      } else if (open && lane == src) {
        more = true;
      }
    });
    if (lane == 0) red[it][threadIdx.x / 32] = m64;  // the same in all lanes
    __syncthreads();                                 // one a row: the next one writes the other half
#pragma unroll
    for (int i = 0; i < 8; ++i) m64 = fmax(m64, red[it][i]);
    it ^= 1;
    int8_t* q = a.hq + row * a.ld_hq;
    auto put = [&](int c, double w) { q[c] = (int8_t)(m64 > 0.0 ? (int)rint(127.0 * w / m64) : 0); };
    if (held_c >= 0) put(held_c, held);
    if (__any_sync(0xffffffffu, more))
      scan([&](int c, int src, bool, bool open) {
        if (!__any_sync(0xffffffffu, open && lane == src && c != held_c)) return;
        const double w = warp_h(a, row, c, xs);
        if (lane == src) put(c, w);
      });
    if (threadIdx.x == 0) a.h_scale[row] = m64 == 0.0 ? 1.0f : (float)(m64 / 127.0);
  };
  // 32 rows' signs at a time
  for (int64_t first = blockIdx.x; first < a.rows; first += 32ll * gridDim.x) {
    const int64_t mine = first + (int64_t)lane * gridDim.x;
    const float s = mine < a.rows ? *const_cast<const volatile float*>(a.h_scale + mine) : 0.0f;
    __syncthreads();  // every warp has read them before a row is settled
    for (unsigned rows = __ballot_sync(0xffffffffu, __float_as_int(s) < 0 && s == s); rows != 0u; rows &= rows - 1u) {
      const int i = __ffs(rows) - 1;
      settle(first + (int64_t)i * gridDim.x, fabsf(__shfl_sync(0xffffffffu, s, i)));
    }
  }
}

}  // namespace quant

int launch_quantize_rows(const dsca_quantize_rows_args* a, bool max_alone, bool pdl, cudaStream_t stream) {
  if (a->dtype == DSCA_BF16) return quant::run<__nv_bfloat16, quant::kScale>(*a, pdl, stream);
  return max_alone ? quant::run<float, quant::kMax>(*a, pdl, stream) : quant::run<float, quant::kScale>(*a, pdl, stream);
}

int launch_quantize_h(const dsca_gated_ffn_int8_args* a, bool pdl, cudaStream_t stream) {
  const dsca_quantize_rows_args rows = {a->h, a->rows, a->inter, DSCA_F32, a->ld_h, a->hq, a->ld_hq, a->h_scale};
  if (int rc = quant::run<float, quant::kH>(rows, pdl, stream)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(a->rows, (int64_t)32 * current_device_sms()));  // more than fit: rows differ
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, quant::settle_kernel, *a) == cudaSuccess ? DSCA_OK : DSCA_ERR_CUDA;
}

}  // namespace dense
}  // namespace dsca
