// Entry points of dsca_b200_dense.h: argument checks, workspaces and the order of the launches.
#include "dense.cuh"

#include <algorithm>

namespace dsca {
namespace dense {
namespace {

bool at(const void* p, uintptr_t n) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % n == 0; }
bool at_or_null(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int64_t esize(int dtype) { return dtype == DSCA_BF16 ? 2 : 4; }
bool dim_ok(int64_t v) { return v >= 1 && v <= DSCA_DENSE_MAX_DIM; }
// a row stride below 2^37 elements: TMA's 2^40 bytes, and every offset of 2^24 rows inside 64 bits
bool ld_ok(int64_t ld, int64_t width) { return ld >= width && ld < (int64_t(1) << 37); }
bool type_ok(int dtype) { return dtype == DSCA_BF16 || dtype == DSCA_F32; }
bool act_ok(int act) { return act == DSCA_GATE_SILU || act == DSCA_GATE_GELU || act == DSCA_GATE_RELU; }

Problem problem(Operand a, Operand b, int M, int N, int K, void* out, int64_t ldo) {
  Problem p = {};
  p.a[0] = a;
  p.b[0] = b;
  p.nseg = 1;
  p.M = M; p.N = N; p.K = K;
  p.out = out;
  p.ldo = ldo;
  return p;
}

int check(const dsca_gated_ffn_args* a) {
  if (a == nullptr || a->rows < 0 || !dim_ok(a->d) || !dim_ok(a->inter) || !type_ok(a->dtype) || !act_ok(a->act))
    return DSCA_ERR_BAD_ARG;
  if (a->rows > DSCA_DENSE_MAX_ROWS) return DSCA_ERR_CAPACITY;
  if (a->rows == 0) return DSCA_OK;
  const int64_t e = esize(a->dtype);
  if (!at(a->x, e) || !at(a->w_gate, e) || !at(a->w_up, e) || !at(a->w_down, e) || !at(a->y, e) || !at(a->h, 16) ||
      !at_or_null(a->g, 16) || !at_or_null(a->u, 16) || (a->g == nullptr) != (a->u == nullptr) ||
      (a->g != nullptr && a->dtype == DSCA_BF16 && !at(a->gu_exp, 4)))
    return DSCA_ERR_BAD_ARG;
  if (!ld_ok(a->ld_x, a->d) || !ld_ok(a->ld_gate, a->d) || !ld_ok(a->ld_up, a->d) || !ld_ok(a->ld_down, a->inter) ||
      !ld_ok(a->ld_y, a->d) || !ld_ok(a->ld_h, a->inter) || a->ld_h * e % 16 != 0)
    return DSCA_ERR_BAD_ARG;
  return DSCA_OK;
}

int check(const dsca_gated_ffn_backward_args* a) {
  if (a == nullptr || a->rows < 0 || !dim_ok(a->d) || !dim_ok(a->inter) || !type_ok(a->dtype) || !act_ok(a->act))
    return DSCA_ERR_BAD_ARG;
  if (a->rows > DSCA_DENSE_MAX_ROWS) return DSCA_ERR_CAPACITY;
  const int64_t e = esize(a->dtype);
  if (!at_or_null(a->dx, e) || !at_or_null(a->d_gate, e) || !at_or_null(a->d_up, e) || !at_or_null(a->d_down, e))
    return DSCA_ERR_BAD_ARG;
  if (a->rows == 0) return DSCA_OK;
  if (!at(a->x, e) || !at(a->w_gate, e) || !at(a->w_up, e) || !at(a->w_down, e) || !at(a->dy, e) || !at(a->g, 16) ||
      !at(a->u, 16) || !at(a->h, 16) || !at(a->dg, 16) || !at(a->du, 16) ||
      (a->dtype == DSCA_BF16 && !at(a->gu_exp, 4)))
    return DSCA_ERR_BAD_ARG;
  if (!ld_ok(a->ld_x, a->d) || !ld_ok(a->ld_gate, a->d) || !ld_ok(a->ld_up, a->d) || !ld_ok(a->ld_down, a->inter) ||
      !ld_ok(a->ld_dy, a->d) || !ld_ok(a->ld_h, a->inter) || a->ld_h * e % 16 != 0)
    return DSCA_ERR_BAD_ARG;
  return DSCA_OK;
}

int check(const dsca_quantize_rows_args* a) {
  if (a == nullptr || a->rows < 0 || !dim_ok(a->k) || !type_ok(a->dtype)) return DSCA_ERR_BAD_ARG;
  if (a->rows > DSCA_DENSE_MAX_ROWS) return DSCA_ERR_CAPACITY;
  if (a->rows == 0) return DSCA_OK;
  if (!at(a->x, esize(a->dtype)) || !at(a->q, 16) || !at(a->scale, 4) || !ld_ok(a->ld_x, a->k) ||
      !ld_ok(a->ld_q, a->k) || a->ld_q % 16 != 0 || a->ld_q > 2 * DSCA_DENSE_MAX_DIM)
    return DSCA_ERR_BAD_ARG;
  return DSCA_OK;
}

int check(const dsca_int8_linear_args* a) {
  if (a == nullptr || a->rows < 0 || !dim_ok(a->k) || !dim_ok(a->n) || !type_ok(a->dtype)) return DSCA_ERR_BAD_ARG;
  // a sum of k products of two codes stays inside 32 bits
  if (a->rows > DSCA_DENSE_MAX_ROWS || a->k > 131072) return DSCA_ERR_CAPACITY;
  if (a->rows == 0) return DSCA_OK;
  const int64_t e = esize(a->dtype);
  if (!at_or_null(a->x, e) || !at(a->q, 16) || !at(a->scale, 4) || !at(a->w, 16) || !at(a->w_scale, 4) ||
      !at_or_null(a->bias, e) || !at(a->y, e))
    return DSCA_ERR_BAD_ARG;
  if ((a->x != nullptr && !ld_ok(a->ld_x, a->k)) || !ld_ok(a->ld_q, a->k) || a->ld_q % 16 != 0 ||
      a->ld_q > 2 * DSCA_DENSE_MAX_DIM || !ld_ok(a->ld_w, a->k) || a->ld_w % 16 != 0 || !ld_ok(a->ld_y, a->n))
    return DSCA_ERR_BAD_ARG;
  return DSCA_OK;
}

int check(const dsca_gated_ffn_int8_args* a) {
  if (a == nullptr || a->rows < 0 || !dim_ok(a->d) || !dim_ok(a->inter) || !type_ok(a->dtype) || !act_ok(a->act))
    return DSCA_ERR_BAD_ARG;
  if (a->rows > DSCA_DENSE_MAX_ROWS || a->d > 131072 || a->inter > 131072) return DSCA_ERR_CAPACITY;
  if (a->rows == 0) return DSCA_OK;
  const int64_t e = esize(a->dtype);
  if (!at(a->x, e) || !at(a->q, 16) || !at(a->scale, 4) || !at(a->w_gate, 16) || !at(a->w_up, 16) ||
      !at(a->w_down, 16) || !at(a->gate_scale, 4) || !at(a->up_scale, 4) || !at(a->down_scale, 4) || !at(a->h, 16) ||
      !at(a->hq, 16) || !at(a->h_scale, 4) || !at(a->y, e))
    return DSCA_ERR_BAD_ARG;
  auto codes = [](int64_t ld, int64_t w) { return ld_ok(ld, w) && ld % 16 == 0 && ld <= 2 * DSCA_DENSE_MAX_DIM; };
  if (!ld_ok(a->ld_x, a->d) || !codes(a->ld_q, a->d) || !codes(a->ld_gate, a->d) || !codes(a->ld_up, a->d) ||
      !codes(a->ld_down, a->inter) || !codes(a->ld_hq, a->inter) || !ld_ok(a->ld_h, a->inter) || a->ld_h % 4 != 0 ||
      !ld_ok(a->ld_y, a->d))
    return DSCA_ERR_BAD_ARG;
  return DSCA_OK;
}

// ---------------------------------------------------------------- calls as lists of launches
//
// Each entry point is written once, as a function that lays out its workspace and issues its launches; `dry`, it
// only adds up the workspace's bytes.
struct Call {
  bool dry;
  uint8_t* base;
  size_t bytes;
  cudaStream_t stream;
  int32_t* err;
  size_t used = 0;
  RelayList relays = {};

  void* take(size_t n) {
    const size_t at = used;
    used += (n + 255) / 256 * 256;
    return dry ? nullptr : base + at;
  }
  bool fits() const { return dry || used <= bytes; }
  // A matrix as an operand: as it lies where TMA can load it, otherwise laid out anew (by relay()).
  Operand operand(const void* p, int64_t rows, int64_t cols, int64_t ld, int dtype, int mn) {
    if (dtype == DSCA_BF16 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0) return {p, ld, mn, 0};
    const bool f32 = dtype == DSCA_F32;
    const int64_t ldd = (cols + 7) / 8 * 8, rows_p = f32 ? (rows + 15) / 16 * 16 : rows;
    void* dst = take((size_t)(rows_p * ldd) * (f32 ? 6 : 2));
    relays.item[relays.n++] = {p, dst, rows, rows_p, cols, ld, ldd, dtype, 0, 0};
    return {dst, ldd, mn, rows_p};
  }
  // The launch that lays out what operand() collected, and zeroes the counters that reserve() left to it; *none when
  // there was nothing to launch.
  int relay(bool* none) {
    *none = relays.n == 0;
    int rc = DSCA_OK;
    if (!dry) {
      if (relays.n != 0) rc = launch_relay(relays, stream);
      else if (relays.zero != nullptr && cudaMemsetAsync(relays.zero, 0, relays.zero_bytes, stream) != cudaSuccess) rc = DSCA_ERR_CUDA;
    }
    relays.n = 0;
    relays.zero = nullptr;
    return rc;
  }
  // The jobs' own workspaces; their counters are zeroed by the relay() that has to come next, before the products, so
  // that nothing lies between those that follow one another.
  struct Own {
    void *parts = nullptr, *counters = nullptr;
  };
  int reserve(const Job* const* jobs, Own* own, int n) {
    size_t parts[2], counters[2], zero = 0;
    for (int i = 0; i < n; ++i) {
      if (int rc = tc_workspace(*jobs[i], &parts[i], &counters[i])) return rc;
      zero += counters[i];
    }
    if (zero == 0) return fits() ? DSCA_OK : DSCA_ERR_CAPACITY;
    uint8_t* at = reinterpret_cast<uint8_t*>(take(zero));
    for (int i = 0; i < n; ++i) {
      if (parts[i] != 0) own[i].parts = take(parts[i]);
      if (!dry) own[i].counters = at;
      at += counters[i];
    }
    if (!fits()) return DSCA_ERR_CAPACITY;
    relays.zero = own[0].counters;
    relays.zero_bytes = zero;
    return DSCA_OK;
  }
  int product(const Job& j, const Own& o, bool pdl) {
    return dry ? DSCA_OK : launch_tc(j, o.parts, o.counters, err, pdl, stream);
  }
  int quantize(const void* x, int rows, int k, int dtype, int64_t ld_x, int8_t* q, int64_t ld_q, float* scale, bool max_alone,
               bool pdl) {
    dsca_quantize_rows_args a = {x, rows, k, dtype, ld_x, q, ld_q, scale};
    return dry ? DSCA_OK : launch_quantize_rows(&a, max_alone, pdl, stream);
  }
};

Operand as(Operand o, int mn) {
  o.mn = mn;
  return o;
}

#define TRY(call) \
  if (int rc_ = (call)) return rc_

int run(Call& c, const dsca_gated_ffn_args* a) {
  const int dt = a->dtype, T = a->rows, d = a->d, I = a->inter;
  Job j = {}, k = {};
  if (T <= 32) {
    j.epi = kGlu; j.act = a->act; j.nprob = 1; j.dtype = dt;
    j.prob[0] = problem({a->w_gate, a->ld_gate, 0, 0}, {a->x, a->ld_x, 0, 0}, I, T, d, a->h, a->ld_h);
    j.prob[0].a[1] = {a->w_up, a->ld_up, 0, 0};
    j.save_g = a->g; j.save_u = a->u; j.save_e = a->gu_exp;
    k.epi = kStore; k.nprob = 1; k.dtype = dt;
    k.prob[0] = problem({a->w_down, a->ld_down, 0, 0}, {a->h, a->ld_h, 0, 0}, d, T, I, a->y, a->ld_y);
    if (few_fits(j, false) && few_fits(k, false)) {
      if (c.dry) return DSCA_OK;
      TRY(launch_few(j, &k, false, c.stream));
      return launch_few(k, nullptr, true, c.stream);
    }
    j = {};
    k = {};
  }
  j.epi = kGlu; j.act = a->act; j.nprob = 1; j.dtype = dt;
  j.prob[0] = problem(c.operand(a->w_gate, I, d, a->ld_gate, dt, 0), c.operand(a->x, T, d, a->ld_x, dt, 0), I, T, d,
                      a->h, a->ld_h);
  j.prob[0].a[1] = c.operand(a->w_up, I, d, a->ld_up, dt, 0);
  j.save_g = a->g; j.save_u = a->u; j.save_e = a->gu_exp;
  k.epi = kStore; k.nprob = 1; k.dtype = dt;
  k.prob[0] = problem(c.operand(a->w_down, d, I, a->ld_down, dt, 0), {}, d, T, I, a->y, a->ld_y);
  const Job* jobs[] = {&j, &k};
  Call::Own own[2];
  bool none;
  TRY(c.reserve(jobs, own, 2));
  TRY(c.relay(&none));
  const Operand h = c.operand(a->h, T, I, a->ld_h, dt, 0);
  if (!c.fits()) return DSCA_ERR_CAPACITY;
  TRY(c.product(j, own[0], false));
  k.prob[0].b[0] = h;
  TRY(c.relay(&none));
  return c.product(k, own[1], none);
}

int run(Call& c, const dsca_gated_ffn_backward_args* a) {
  const int dt = a->dtype, T = a->rows, d = a->d, I = a->inter;
  const bool weights = a->d_gate != nullptr || a->d_up != nullptr;
  const bool inner = a->dx != nullptr || weights;
  Job j = {}, k = {};
  bool none;
  // the first product's operands and those of the second that are there already
  const Operand dy = c.operand(a->dy, T, d, a->ld_dy, dt, 0);
  if (inner) {
    j.epi = kDGlu; j.act = a->act; j.nprob = 1; j.dtype = dt;
    j.prob[0] = problem(c.operand(a->w_down, d, I, a->ld_down, dt, 1), dy, I, T, d, a->dg, a->ld_h);
    j.save_g = const_cast<void*>(a->g); j.save_u = const_cast<void*>(a->u); j.out2 = a->du;
    j.save_e = const_cast<uint8_t*>(a->gu_exp);
  }
  k.epi = kStore; k.dtype = dt;
  Operand wg = {}, wu = {}, x = {}, h = {};
  if (a->dx != nullptr) {
    wg = c.operand(a->w_gate, I, d, a->ld_gate, dt, 1);
    wu = c.operand(a->w_up, I, d, a->ld_up, dt, 1);
  }
  if (weights) x = c.operand(a->x, T, d, a->ld_x, dt, 1);
  if (a->d_down != nullptr) h = c.operand(a->h, T, I, a->ld_h, dt, 1);
  // ... and those that the first product makes
  auto second = [&](Operand dg, Operand du) {
    k.nprob = 0;
    if (a->dx != nullptr) {
      Problem& p = k.prob[k.nprob++];
      p = problem(wg, as(dg, 0), d, T, I, a->dx, d);
      p.nseg = 2;
      p.a[1] = wu;
      p.b[1] = as(du, 0);
    }
    if (a->d_gate != nullptr) k.prob[k.nprob++] = problem(x, as(dg, 1), d, I, T, a->d_gate, d);
    if (a->d_up != nullptr) k.prob[k.nprob++] = problem(x, as(du, 1), d, I, T, a->d_up, d);
    if (a->d_down != nullptr) k.prob[k.nprob++] = problem(h, as(dy, 1), I, d, T, a->d_down, I);
  };
  second({}, {});
  if (k.nprob == 0) return DSCA_OK;
  const Job* jobs[] = {&k, &j};
  Call::Own own[2];
  TRY(c.reserve(jobs, own, inner ? 2 : 1));
  TRY(c.relay(&none));
  Operand dg = {}, du = {};
  if (a->dx != nullptr || a->d_gate != nullptr) dg = c.operand(a->dg, T, I, a->ld_h, dt, 0);
  if (a->dx != nullptr || a->d_up != nullptr) du = c.operand(a->du, T, I, a->ld_h, dt, 0);
  if (!c.fits()) return DSCA_ERR_CAPACITY;
  if (inner) TRY(c.product(j, own[1], false));
  second(dg, du);
  TRY(c.relay(&none));
  return c.product(k, own[0], inner && none);
}

int run(Call& c, const dsca_int8_linear_args* a) {
  Job j = {};
  j.epi = kStore; j.nprob = 1; j.dtype = a->dtype; j.i8 = 1;
  j.prob[0] = problem({a->w, a->ld_w, 0, 0}, {a->q, a->ld_q, 0, 0}, a->n, a->rows, a->k, a->y, a->ld_y);
  j.row_scale = a->scale; j.col_scale[0] = a->w_scale; j.bias = a->bias;
  const Job* jobs[] = {&j};
  Call::Own own[1];
  const bool few = few_fits(j, true);
  bool none;
  if (!few) TRY(c.reserve(jobs, own, 1));
  TRY(c.relay(&none));
  if (a->x != nullptr) TRY(c.quantize(a->x, a->rows, a->k, a->dtype, a->ld_x, a->q, a->ld_q, a->scale, false, false));
  if (few) return c.dry ? DSCA_OK : launch_few(j, nullptr, a->x != nullptr, c.stream);
  return c.product(j, own[0], a->x != nullptr);
}

int run(Call& c, const dsca_gated_ffn_int8_args* a) {
  Job j = {}, k = {};
  j.epi = kGlu; j.act = a->act; j.nprob = 1; j.dtype = DSCA_F32; j.i8 = 1;
  j.prob[0] = problem({a->w_gate, a->ld_gate, 0, 0}, {a->q, a->ld_q, 0, 0}, a->inter, a->rows, a->d, a->h, a->ld_h);
  j.prob[0].a[1] = {a->w_up, a->ld_up, 0, 0};
  const bool wide = a->dtype == DSCA_F32;
  if (wide) j.row_max = a->scale;
  j.row_scale = a->scale; j.col_scale[0] = a->gate_scale; j.col_scale[1] = a->up_scale;
  k.epi = kStore; k.nprob = 1; k.dtype = a->dtype; k.i8 = 1;
  k.prob[0] = problem({a->w_down, a->ld_down, 0, 0}, {a->hq, a->ld_hq, 0, 0}, a->d, a->rows, a->inter, a->y, a->ld_y);
  k.row_scale = a->h_scale; k.col_scale[0] = a->down_scale;
  const Job* jobs[] = {&j, &k};
  Call::Own own[2];
  const bool few = few_fits(j, false) && few_fits(k, false);
  bool none;
  if (!few) TRY(c.reserve(jobs, own, 2));
  TRY(c.relay(&none));
  TRY(c.quantize(a->x, a->rows, a->d, a->dtype, a->ld_x, a->q, a->ld_q, a->scale, wide, false));
  if (few && !c.dry) TRY(launch_few(j, &k, true, c.stream));
  if (!few) TRY(c.product(j, own[0], true));
  // fp32 tokens: one code on the other side of its border moves a token's y by 1e-3 of its size, and an h in fp32 has such
  // codes in every call.  (bf16 tokens' y is rounded by as much.)
  if (!wide) TRY(c.quantize(a->h, a->rows, a->inter, DSCA_F32, a->ld_h, a->hq, a->ld_hq, a->h_scale, false, true));
  if (wide && !c.dry) TRY(launch_quantize_h(a, true, c.stream));
  if (few) return c.dry ? DSCA_OK : launch_few(k, nullptr, true, c.stream);
  return c.product(k, own[1], true);
}

#undef TRY

// The kernels are sm_100a code.
int device_ok() {
  static volatile int known[kMaxDevices];  // 1 yes, 2 no
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return DSCA_ERR_CUDA;
  const int k = dev < kMaxDevices ? __atomic_load_n(&known[dev], __ATOMIC_ACQUIRE) : 0;
  if (k == 1) return DSCA_OK;
  if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess) return DSCA_ERR_CUDA;
  if (dev < kMaxDevices) __atomic_store_n(&known[dev], major == 10 ? 1 : 2, __ATOMIC_RELEASE);
  return major == 10 ? DSCA_OK : DSCA_ERR_UNSUPPORTED;
}

template <typename Args>
int call(const Args* a, cudaStream_t stream) {
  if (int rc = device_ok()) return rc;
  if (a->workspace_bytes != 0 && !at(a->workspace, 256)) return DSCA_ERR_BAD_ARG;
  Call c = {false, reinterpret_cast<uint8_t*>(a->workspace), a->workspace_bytes, stream, a->err};
  return run(c, a);
}

template <typename Args>
size_t workspace(const Args* a) {
  if (check(a) != DSCA_OK || a->rows == 0) return 0;
  Call size = {true, nullptr, 0, nullptr, nullptr};
  return run(size, a) == DSCA_OK ? size.used : 0;
}

}  // namespace
}  // namespace dense
}  // namespace dsca

using namespace dsca;

extern "C" {

int dsca_gated_ffn(const dsca_gated_ffn_args* a, dsca_stream_t stream) {
  if (int rc = dense::check(a)) return rc;
  return a->rows == 0 ? DSCA_OK : dense::call(a, stream);
}

int dsca_gated_ffn_backward(const dsca_gated_ffn_backward_args* a, dsca_stream_t stream) {
  if (int rc = dense::check(a)) return rc;
  if (a->rows == 0) {  // empty sums
    const size_t bytes = (size_t)a->d * a->inter * (a->dtype == DSCA_BF16 ? 2 : 4);
    for (void* p : {a->d_gate, a->d_up, a->d_down})
      if (p != nullptr && cudaMemsetAsync(p, 0, bytes, stream) != cudaSuccess) return DSCA_ERR_CUDA;
    return DSCA_OK;
  }
  return dense::call(a, stream);
}

int dsca_quantize_rows(const dsca_quantize_rows_args* a, dsca_stream_t stream) {
  if (int rc = dense::check(a)) return rc;
  if (a->rows == 0) return DSCA_OK;
  if (int rc = dense::device_ok()) return rc;
  return dense::launch_quantize_rows(a, false, false, stream);
}

int dsca_int8_linear(const dsca_int8_linear_args* a, dsca_stream_t stream) {
  if (int rc = dense::check(a)) return rc;
  return a->rows == 0 ? DSCA_OK : dense::call(a, stream);
}

int dsca_gated_ffn_int8(const dsca_gated_ffn_int8_args* a, dsca_stream_t stream) {
  if (int rc = dense::check(a)) return rc;
  return a->rows == 0 ? DSCA_OK : dense::call(a, stream);
}

size_t dsca_gated_ffn_workspace(const dsca_gated_ffn_args* a) { return dense::workspace(a); }
size_t dsca_gated_ffn_backward_workspace(const dsca_gated_ffn_backward_args* a) { return dense::workspace(a); }
size_t dsca_int8_linear_workspace(const dsca_int8_linear_args* a) { return dense::workspace(a); }
size_t dsca_gated_ffn_int8_workspace(const dsca_gated_ffn_int8_args* a) { return dense::workspace(a); }

}  // extern "C"
