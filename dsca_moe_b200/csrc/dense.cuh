// Shared by the dense gated feed-forward block and the 8-bit integer products (dsca_b200_dense.h).
//
// Every product is written as out[n][m] = sum_k A[m][k] B[n][k], m the contiguous index of the
// output's rows: for a forward product A is the weight and B the tokens, for a weight's gradient both
// are activations and k the tokens.  An operand is K-major (element [r][k] at p[r * ld + k], a
// weight as a Linear layer holds it) or MN-major (p[k * ld + r], the same matrix read the other way), so
// no product transposes a matrix in memory.
#pragma once
#include "common.cuh"
#include "dsca_b200_dense.h"

namespace dsca {
namespace dense {

struct Operand {
  const void* p;
  int64_t ld;     // elements
  int mn;         // 0 K-major, 1 MN-major
  int64_t plane;  // fp32 products: rows from one plane of bf16 terms to the next
};

// Up to two segments whose sums are added: out = sum_s A_s B_s^T (dx = dg Wg + du Wu).
struct Problem {
  Operand a[2], b[2];
  int nseg, M, N, K;
  void* out;  // [N, M]
  int64_t ldo;
};

// kStore: out = the product (8-bit: times row_scale[n] col_scale[0][m], plus bias[m]).
// kGlu:   a[0] gate, a[1] up rows: out = act(g) * u; g and u as well where save_g is given.
// kDGlu:  the product is dh; with g and u read: out = dh u act'(g), out2 = dh act(g).
enum Epi { kStore = 0, kGlu = 1, kDGlu = 2 };
constexpr int kMaxProblems = 4;

struct Job {
  int epi, act, nprob;
  int i8;         // operands are 8-bit integers, the sum int32
  int dtype;      // of the operands (unless i8) and of out
  Problem prob[kMaxProblems];
  void* save_g;   // kGlu: written; kDGlu: read (same for u); rows of prob[0].ldo
  void* save_u;
  uint8_t* save_e;
  void* out2;     // kDGlu: du
  const float* row_scale;
  const float* row_max;  // kGlu of 8-bit operands, instead of row_scale: the rows' largest magnitudes; h within kCloseH
  const float* col_scale[2];
  const void* bias;
};

// ---------------------------------------------------------------- gates
// kFast (16-bit and 8-bit operands): the hardware's exponential and reciprocal without the steps that keep subnormal
// numbers, good to 2^-18 here (where they flush to zero, 1 + e^-x is 1 or its reciprocal below 2^-126); otherwise
// the full-precision ones.
template <bool kFast>
__device__ __forceinline__ float sigmoid(float x) {
  if constexpr (kFast) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
  } else {
    return 1.0f / (1.0f + expf(-x));
  }
}

// the gelu gate: 0.5 (1 + tanh z) = sigmoid(2 z), z = sqrt(2 / pi) (g + 0.044715 g^3)
template <bool kFast>
__device__ __forceinline__ float gelu_p(float g) {
  return sigmoid<kFast>(1.5957691216057308f * (g + 0.044715f * g * g * g));
}

template <bool kFast>
__device__ __forceinline__ float gate(float g, int act) {
  if (act == DSCA_GATE_SILU) return kFast ? g * sigmoid<true>(g) : g / (1.0f + expf(-g));
  if (act == DSCA_GATE_RELU) return g <= 0.0f ? 0.0f : g;  // NaN stays
  return g * gelu_p<kFast>(g);
}

// The gate in 64 bits.
__device__ __forceinline__ double gate64(double g, int act) {
  if (act == DSCA_GATE_RELU) return g <= 0.0 ? 0.0 : g;
  const double z = act == DSCA_GATE_SILU ? g : 2.0 * 0.7978845608028654 * (g + 0.044715 * g * g * g);
  const double e = exp(-fabs(z));  // sigmoid(z), which does not cancel on either side
  return g * ((z >= 0.0 ? 1.0 : e) / (1.0 + e));
}

// act(g) and act'(g)
template <bool kFast>
__device__ __forceinline__ void gate_grad(float g, int act, float* a, float* da) {
  if (act == DSCA_GATE_SILU) {
    const float s = sigmoid<kFast>(g);
    *a = g * s;
    *da = s + *a * (1.0f - s);
  } else if (act == DSCA_GATE_RELU) {
    *a = g <= 0.0f ? 0.0f : g;
    *da = g <= 0.0f ? 0.0f : (g != g ? g : 1.0f);
  } else {
    const float p = gelu_p<kFast>(g);
    *a = g * p;
    const float q = p * (1.0f - p);
    *da = p + (q > 0.0f ? 2.0f * g * q * 0.7978845608028654f * (1.0f + 0.134145f * g * g) : 0.0f);
    if (g != g) *da = g;
  }
}

// A sum of codes times its two scales.  The scales' own product may be subnormal where the result is a normal number, so the
// sum is multiplied first: by the channel's scale, which the sum keeps normal; kBig: by the smaller of the two, so that a channel's
// scale above 2^97 does not make the sum infinite where the token's brings it back (fp32 tokens: in the epilogue of the 4096-token
// bf16 block the choice costs 2 of 130 us).
template <bool kBig>
__device__ __forceinline__ void in_turn(float& a, float& b) {
  if constexpr (kBig) {
    const float x = a, y = b;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(x), "f"(y));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(x), "f"(y));
  }
}
template <bool kBig>
__device__ __forceinline__ float scaled(int sum, float cs, float rs) {
  in_turn<kBig>(cs, rs);
  return (float)sum * cs * rs;
}

// ---- h of 8-bit products of fp32 tokens: off by at most kCloseH of itself, whatever g is (its 64-bit value's codes are asked for,
// and those that this leaves open are formed again).  A gate far below zero multiplies g's relative error by |g|, so g is held
// in two floats up to the exponential's argument.
//
// In units of 2^-24: the exponential 4 and its correction 1, 1 + e 1, its reciprocal 2, their product 1, g s 2; u: the sum's
// conversion, two products and the scale's correction 4; h 1: 16.
constexpr float kCloseH = 1e-6f;

struct Two {
  float hi, lo;
};
// A token's scale max|x| / 127 as hi (1 + lo).
__device__ __forceinline__ Two scale_two(float row_max) {
  Two r;
  r.hi = __fdiv_rn(row_max, 127.0f);
  r.lo = r.hi > 0.0f ? __fdiv_rn(fmaf(-127.0f, r.hi, row_max), row_max) : 0.0f;
  return r;
}

template <int ACT>
__device__ __forceinline__ float close_h(int sum_g, int sum_u, float gs, float us, Two xs) {
  float u = scaled<true>(sum_u, us, xs.hi);
  u = fmaf(u, xs.lo, u);
  float b = xs.hi;
  in_turn<true>(gs, b);
  const float s = (float)sum_g, p = s * gs;
  float pl = fmaf(s, gs, -p);
  if (abs(sum_g) > 1 << 24) pl = fmaf((float)(sum_g - (int)s), gs, pl);
  Two g;
  g.hi = p * b;
  g.lo = fmaf(g.hi, xs.lo, fmaf(pl, b, fmaf(p, b, -g.hi)));
  if constexpr (ACT == DSCA_GATE_RELU) return (g.hi <= 0.0f ? 0.0f : g.hi + g.lo) * u;
  Two z = g;
  if constexpr (ACT == DSCA_GATE_GELU) {  // 2 sqrt(2 / pi) g (1 + 0.044715 g^2), each constant in two floats
    constexpr float kA = (float)0.044715, kAl = (float)(0.044715 - (double)kA);
    constexpr float kC = (float)1.5957691216057308, kCl = (float)(1.5957691216057308 - (double)kC);
    const float q = g.hi * g.hi, ql = fmaf(2.0f * g.hi, g.lo, fmaf(g.hi, g.hi, -q));
    const float t = q * kA, tl = fmaf(q, kAl, fmaf(ql, kA, fmaf(q, kA, -t)));
    const float w = 1.0f + t, wt = w - 1.0f, wl = (1.0f - (w - wt)) + (t - wt) + tl;
    const float y = g.hi * w, yl = fmaf(g.lo, w, fmaf(g.hi, wl, fmaf(g.hi, w, -y)));
    z.hi = y * kC;
    z.lo = fmaf(y, kCl, fmaf(yl, kC, fmaf(y, kC, -z.hi)));
  }
  // e = 2^(-|z| log2(e)); below 2^-150 nothing
  constexpr float kL = (float)1.4426950408889634, kLl = (float)(1.4426950408889634 - (double)kL);
  const float n = -fabsf(z.hi), nl = z.hi < 0.0f ? z.lo : -z.lo;
  const float t = n * kL, tl = fmaf(nl, kL, fmaf(n, kLl, fmaf(n, kL, -t)));
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  e = t < -150.0f ? 0.0f : fmaf(e, 0.6931472f * tl, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  const float sg = z.hi < 0.0f ? e * r : r;
  return fmaf(g.lo, sg, g.hi * sg) * u;
}

// N of them; which gate is decided once, so that their chains of instructions overlap.
template <int ACT, int N>
__device__ __forceinline__ void close_loop(float (&h)[N], const int (&g)[N], const int (&u)[N], const float (&gs)[N], const float (&us)[N],
                                           const Two (&xs)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) h[j] = close_h<ACT>(g[j], u[j], gs[j], us[j], xs[j]);
}
template <int N>
__device__ __forceinline__ void close_all(float (&h)[N], const int (&g)[N], const int (&u)[N], const float (&gs)[N], const float (&us)[N],
                                          const Two (&xs)[N], int act) {
  if (act == DSCA_GATE_SILU) close_loop<DSCA_GATE_SILU>(h, g, u, gs, us, xs);
  else if (act == DSCA_GATE_RELU) close_loop<DSCA_GATE_RELU>(h, g, u, gs, us, xs);
  else close_loop<DSCA_GATE_GELU>(h, g, u, gs, us, xs);
}

// ---- g and u of 16-bit products for the backward pass: fp16 times a power of two that brings the largest finite one
// of its group of a token's channels to [2^14, 2^15).  The exponent byte is the largest's, at least 14 so that the
// factor is a normal number; a row has one for every eight channels (groups of 32 write four equal ones).
__host__ __device__ __forceinline__ int exp_groups(int cols) { return (cols + 31) / 32 * 4; }
__device__ __forceinline__ uint32_t f16_exp(float largest) { return max(14u, __float_as_uint(largest) >> 23); }
__device__ __forceinline__ float f16_factor(uint32_t e) { return __uint_as_float((268u - e) << 23); }  // 2^(141 - e)
__device__ __forceinline__ float f16_back(uint32_t e) {                                               // 2^(e - 141)
  return e > 14u ? __uint_as_float((e - 14u) << 23) : 5.877471754111438e-39f;
}

// Products for few tokens (dense_few.cu); no workspace, any alignment.  alone: a single product, not one of a block's two.
bool few_fits(const Job& j, bool alone);
// next: the product behind it, whose weights it asks into L2.
int launch_few(const Job& j, const Job* next, bool pdl, cudaStream_t stream);

// A matrix to lay out anew (dense_split.cu).
struct Relay {
  const void* src;
  void* dst;
  int64_t rows, rows_p, cols, lds, ldd;  // ldd a multiple of 8
  int dtype, vec;
  uint32_t first;
};
constexpr int kMaxRelays = 8;
struct RelayList {
  Relay item[kMaxRelays];
  int n;
  void* zero;         // words to zero as well, or NULL
  size_t zero_bytes;
};
int launch_relay(RelayList& list, cudaStream_t stream);

// Tensor-core products (dense_tc.cu), with tc_workspace()'s bytes of partial tiles and of counters, which are zero
// at the launch.
int tc_workspace(const Job& j, size_t* parts, size_t* counters);
int launch_tc(const Job& j, void* parts, void* counters, int32_t* err, bool pdl, cudaStream_t stream);
// max_alone (fp32): the scales take the rows' largest magnitudes themselves.
int launch_quantize_rows(const dsca_quantize_rows_args* a, bool max_alone, bool pdl, cudaStream_t stream);
// The intermediate's rows of an 8-bit block as its 64-bit values' codes; `scale` holds the tokens' largest magnitudes.
int launch_quantize_h(const dsca_gated_ffn_int8_args* a, bool pdl, cudaStream_t stream);

}  // namespace dense
}  // namespace dsca
