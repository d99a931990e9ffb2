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
// a row stride no larger than 2^40 elements keeps every offset of 2^24 rows inside 64 bits
bool ld_ok(int64_t ld, int64_t width) { return ld >= width && ld < (int64_t(1) << 40); }
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
      !at_or_null(a->g, 16) || !at_or_null(a->u, 16) || (a->g == nullptr) != (a->u == nullptr))
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
      !at(a->u, 16) || !at(a->h, 16) || !at(a->dg, 16) || !at(a->du, 16))
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

int run(const dsca_gated_ffn_args* a, cudaStream_t s) {
  Job j = {};
  j.epi = kGlu; j.act = a->act; j.nprob = 1; j.dtype = a->dtype;
  j.prob[0] = problem({a->w_gate, a->ld_gate, 0}, {a->x, a->ld_x, 0}, a->inter, a->rows, a->d, a->h, a->ld_h);
  j.prob[0].a[1] = {a->w_up, a->ld_up, 0};
  j.save_g = a->g; j.save_u = a->u;
  if (int rc = launch_simt(j, s)) return rc;
  Job k = {};
  k.epi = kStore; k.nprob = 1; k.dtype = a->dtype;
  k.prob[0] = problem({a->w_down, a->ld_down, 0}, {a->h, a->ld_h, 0}, a->d, a->rows, a->inter, a->y, a->ld_y);
  return launch_simt(k, s);
}

int run(const dsca_gated_ffn_backward_args* a, cudaStream_t s) {
  const int T = a->rows, d = a->d, I = a->inter;
  Job j = {};
  j.epi = kDGlu; j.act = a->act; j.nprob = 1; j.dtype = a->dtype;
  j.prob[0] = problem({a->w_down, a->ld_down, 1}, {a->dy, a->ld_dy, 0}, I, T, d, a->dg, a->ld_h);
  j.save_g = const_cast<void*>(a->g); j.save_u = const_cast<void*>(a->u); j.out2 = a->du;
  if (a->dx != nullptr || a->d_gate != nullptr || a->d_up != nullptr)
    if (int rc = launch_simt(j, s)) return rc;
  Job k = {};
  k.epi = kStore; k.dtype = a->dtype;
  if (a->dx != nullptr) {
    Problem p = problem({a->w_gate, a->ld_gate, 1}, {a->dg, a->ld_h, 0}, d, T, I, a->dx, d);
    p.nseg = 2;
    p.a[1] = {a->w_up, a->ld_up, 1};
    p.b[1] = {a->du, a->ld_h, 0};
    k.prob[k.nprob++] = p;
  }
  const Operand x = {a->x, a->ld_x, 1};
  if (a->d_gate != nullptr) k.prob[k.nprob++] = problem(x, {a->dg, a->ld_h, 1}, d, I, T, a->d_gate, d);
  if (a->d_up != nullptr) k.prob[k.nprob++] = problem(x, {a->du, a->ld_h, 1}, d, I, T, a->d_up, d);
  if (a->d_down != nullptr)
    k.prob[k.nprob++] = problem({a->h, a->ld_h, 1}, {a->dy, a->ld_dy, 1}, I, d, T, a->d_down, I);
  return k.nprob ? launch_simt(k, s) : DSCA_OK;
}

int quantize(const void* x, int rows, int k, int dtype, int64_t ld_x, int8_t* q, int64_t ld_q, float* scale,
             cudaStream_t s) {
  dsca_quantize_rows_args a = {x, rows, k, dtype, ld_x, q, ld_q, scale};
  return launch_quantize_rows(&a, s);
}

int run(const dsca_int8_linear_args* a, cudaStream_t s) {
  if (a->x != nullptr)
    if (int rc = quantize(a->x, a->rows, a->k, a->dtype, a->ld_x, a->q, a->ld_q, a->scale, s)) return rc;
  Job j = {};
  j.epi = kStore; j.nprob = 1; j.dtype = a->dtype; j.i8 = 1;
  j.prob[0] = problem({a->w, a->ld_w, 0}, {a->q, a->ld_q, 0}, a->n, a->rows, a->k, a->y, a->ld_y);
  j.row_scale = a->scale; j.col_scale[0] = a->w_scale; j.bias = a->bias;
  return launch_simt(j, s);
}

int run(const dsca_gated_ffn_int8_args* a, cudaStream_t s) {
  if (int rc = quantize(a->x, a->rows, a->d, a->dtype, a->ld_x, a->q, a->ld_q, a->scale, s)) return rc;
  Job j = {};
  j.epi = kGlu; j.act = a->act; j.nprob = 1; j.dtype = DSCA_F32; j.i8 = 1;
  j.prob[0] = problem({a->w_gate, a->ld_gate, 0}, {a->q, a->ld_q, 0}, a->inter, a->rows, a->d, a->h, a->ld_h);
  j.prob[0].a[1] = {a->w_up, a->ld_up, 0};
  j.row_scale = a->scale; j.col_scale[0] = a->gate_scale; j.col_scale[1] = a->up_scale;
  if (int rc = launch_simt(j, s)) return rc;
  if (int rc = quantize(a->h, a->rows, a->inter, DSCA_F32, a->ld_h, a->hq, a->ld_hq, a->h_scale, s)) return rc;
  Job k = {};
  k.epi = kStore; k.nprob = 1; k.dtype = a->dtype; k.i8 = 1;
  k.prob[0] = problem({a->w_down, a->ld_down, 0}, {a->hq, a->ld_hq, 0}, a->d, a->rows, a->inter, a->y, a->ld_y);
  k.row_scale = a->h_scale; k.col_scale[0] = a->down_scale;
  return launch_simt(k, s);
}

}  // namespace
}  // namespace dense
}  // namespace dsca

using namespace dsca;

extern "C" {

int dsca_gated_ffn(const dsca_gated_ffn_args* a, dsca_stream_t stream) {
  if (int rc = dense::check(a)) return rc;
  return a->rows == 0 ? DSCA_OK : dense::run(a, stream);
}

int dsca_gated_ffn_backward(const dsca_gated_ffn_backward_args* a, dsca_stream_t stream) {
  if (int rc = dense::check(a)) return rc;
  if (a->rows == 0) {  // empty sums
    const size_t bytes = (size_t)a->d * a->inter * (a->dtype == DSCA_BF16 ? 2 : 4);
    for (void* p : {a->d_gate, a->d_up, a->d_down})
      if (p != nullptr && cudaMemsetAsync(p, 0, bytes, stream) != cudaSuccess) return DSCA_ERR_CUDA;
    return DSCA_OK;
  }
  return dense::run(a, stream);
}

int dsca_quantize_rows(const dsca_quantize_rows_args* a, dsca_stream_t stream) {
  if (int rc = dense::check(a)) return rc;
  return a->rows == 0 ? DSCA_OK : dense::launch_quantize_rows(a, stream);
}

int dsca_int8_linear(const dsca_int8_linear_args* a, dsca_stream_t stream) {
  if (int rc = dense::check(a)) return rc;
  return a->rows == 0 ? DSCA_OK : dense::run(a, stream);
}

int dsca_gated_ffn_int8(const dsca_gated_ffn_int8_args* a, dsca_stream_t stream) {
  if (int rc = dense::check(a)) return rc;
  return a->rows == 0 ? DSCA_OK : dense::run(a, stream);
}

size_t dsca_gated_ffn_workspace(const dsca_gated_ffn_args* a) { return dense::check(a) ? 0 : 0; }
size_t dsca_gated_ffn_backward_workspace(const dsca_gated_ffn_backward_args* a) { return dense::check(a) ? 0 : 0; }
size_t dsca_int8_linear_workspace(const dsca_int8_linear_args* a) { return dense::check(a) ? 0 : 0; }
size_t dsca_gated_ffn_int8_workspace(const dsca_gated_ffn_int8_args* a) { return dense::check(a) ? 0 : 0; }

}  // extern "C"
