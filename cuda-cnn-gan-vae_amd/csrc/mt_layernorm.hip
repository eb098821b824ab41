// Layer normalisation: every row of N values is normalised by its own mean and variance, so a sample's result does not depend
// on the batch.
//   mean = sum(x) / N,  ivar = 1 / sqrt(sum((x - mean)^2) / N + epsilon),  xhat = (x - mean) * ivar,  y = f(gamma * xhat + beta)
// Backward, with g = delta * f'(gamma * xhat + beta) and u = g * gamma:
//   error = ivar * (u - sum(u) / N - xhat * sum(u * xhat) / N),  dgamma = sum over the rows of g * xhat,  dbeta = of g
#include "mt_packed.h"

namespace {

using mt::cdiv;
using mt::PackedView;

constexpr int THREADS = 256;

// ---- where a row's input comes from in the backward pass: the fp32 tensor, or the 8 bits the forward pass kept ------------
struct RowsF32 {
  const float *p;
  uint32_t N;
  __device__ __forceinline__ float at(size_t row, uint32_t i) const { return p[row * N + i]; }
};
struct RowsPacked {
  PackedView v;
  uint32_t N, per_sample;  // rows of one sample
  __device__ __forceinline__ float at(size_t row, uint32_t i) const {
    const size_t w = row / per_sample;
    const uint32_t e = (uint32_t)(row - w * per_sample) * N + i;
    return mt::unpack_value(v.pair[w * v.groups + e / mt::PACK_GROUP], v.q[w * v.pitch + e]);
  }
};

__device__ __forceinline__ float block_sum(float v, float *part) {
  v = mt::wave_sum(v);
  __syncthreads();  // part may still be read from the sum before
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
  __syncthreads();
  float s = 0.f;
  for (uint32_t k = 0; k < blockDim.x / 64; k++) s += part[k];
  return s;
}

__global__ __launch_bounds__(THREADS) void ln_forward_kernel(float *out, const float *in, const float *gamma, const float *beta, float *mean_out, float *ivar_out,
                                                             size_t rows, uint32_t N, float eps, int func) {
  __shared__ float part[THREADS / 64];
  for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float *x = in + row * N;
    float s = 0.f;
    for (uint32_t i = threadIdx.x; i < N; i += THREADS) s += x[i];
    const float mean = block_sum(s, part) / (float)N;
    s = 0.f;
    for (uint32_t i = threadIdx.x; i < N; i += THREADS) {
      const float d = x[i] - mean;
      s += d * d;
    }
    const float ivar = 1.f / sqrtf(block_sum(s, part) / (float)N + eps);
    for (uint32_t i = threadIdx.x; i < N; i += THREADS) out[row * N + i] = mt::apply_func_epilogue(func, gamma[i] * ((x[i] - mean) * ivar) + beta[i]);
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[row] = mean;
      if (ivar_out) ivar_out[row] = ivar;
    }
  }
}

// the gradient in front of the function
__device__ __forceinline__ float front(int func, float delta, float gamma, float xhat, const float *beta, uint32_t i) {
  return func == MT_F_NONE ? delta : delta * mt::apply_func(MT_F_DIFFERENTIAL + func, gamma * xhat + beta[i]);
}

// sums over the rows first: the error may be written over delta
template <class Rows>
__global__ __launch_bounds__(THREADS) void ln_parameters_kernel(float *dgamma, float *dbeta, const float *delta, const float *gamma, const float *beta, Rows x,
                                                                const float *mean, const float *ivar, size_t rows, uint32_t N, int func, bool accumulate) {
  const uint32_t i = blockIdx.x * 64u + threadIdx.x % 64u, slice = threadIdx.x / 64u;
  __shared__ float part[2][4][64];
  float sg = 0.f, sb = 0.f;
  if (i < N)
    for (size_t row = slice; row < rows; row += 4) {
      const float xhat = (x.at(row, i) - mean[row]) * ivar[row];
      const float g = front(func, delta[row * N + i], gamma[i], xhat, beta, i);
      sg += g * xhat;
      sb += g;
    }
  part[0][slice][threadIdx.x % 64] = sg;
  part[1][slice][threadIdx.x % 64] = sb;
  __syncthreads();
  if (slice == 0 && i < N) {
    const uint32_t c = threadIdx.x;
    sg = ((part[0][0][c] + part[0][1][c]) + part[0][2][c]) + part[0][3][c];
    sb = ((part[1][0][c] + part[1][1][c]) + part[1][2][c]) + part[1][3][c];
    if (dgamma) dgamma[i] = accumulate ? dgamma[i] + sg : sg;
    if (dbeta) dbeta[i] = accumulate ? dbeta[i] + sb : sb;
  }
}

template <class Rows>
__global__ __launch_bounds__(THREADS) void ln_error_kernel(float *error, const float *delta, const float *gamma, const float *beta, Rows x, const float *mean,
                                                           const float *ivar, size_t rows, uint32_t N, int func) {
  __shared__ float part[THREADS / 64];
  for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float m = mean[row], iv = ivar[row];
    float s1 = 0.f, s2 = 0.f;
    for (uint32_t i = threadIdx.x; i < N; i += THREADS) {
      const float xhat = (x.at(row, i) - m) * iv, u = front(func, delta[row * N + i], gamma[i], xhat, beta, i) * gamma[i];
      s1 += u;
      s2 += u * xhat;
    }
    s1 = block_sum(s1, part) / (float)N;
    s2 = block_sum(s2, part) / (float)N;
    for (uint32_t i = threadIdx.x; i < N; i += THREADS) {
      const float xhat = (x.at(row, i) - m) * iv, u = front(func, delta[row * N + i], gamma[i], xhat, beta, i) * gamma[i];
      error[row * N + i] = iv * ((u - s1) - xhat * s2);
    }
  }
}

// ---- sizes ---------------------------------------------------------------------------------------------------------
struct Geometry {
  size_t rows;
  uint32_t N, per_sample;   // values per row, rows per sample
  uint32_t kept_z, kept_y;  // sizes of a statistic: [W,kept_z,kept_y,1]
};

// gamma names the sizes that a row spans
int geometry(const char *name, const mt_tensor *in, const mt_tensor *gamma, Geometry *g) {
  g->kept_z = g->kept_y = 1;
  bool ok = gamma->w == 1 && gamma->x == in->x;
  if (ok && gamma->y == in->y && gamma->z == in->z) {
  } else if (ok && gamma->y == in->y && gamma->z == 1) {
    g->kept_z = in->z;
  } else if (ok && gamma->y == 1 && gamma->z == 1) {
    g->kept_z = in->z;
    g->kept_y = in->y;
  } else {
    return mt::fail(MT_E_SHAPE, "%s: gamma must be [1,Z,Y,X], [1,1,Y,X] or [1,1,1,X] of the input's sizes", name);
  }
  const uint64_t per = (uint64_t)g->kept_z * g->kept_y, zy = (uint64_t)gamma->z * gamma->y;
  uint64_t N, rows;
  if (__builtin_mul_overflow(zy, (uint64_t)gamma->x, &N) || N > 0x7fffffefull || per > 0x7fffffffull || __builtin_mul_overflow(per, (uint64_t)in->w, &rows) || rows >= (1ull << 40))
    return mt::fail(MT_E_UNAVAILABLE, "%s: rows of 2^31 values or more are not supported", name);
  g->rows = rows;
  g->N = (uint32_t)N;
  g->per_sample = (uint32_t)per;
  return MT_OK;
}
bool same_sizes(const mt_tensor *a, const mt_tensor *b) { return mt::same_zyx(a, b) && a->w == b->w; }
bool is_statistic(const mt_tensor *t, const mt_tensor *in, const Geometry &g) { return t->w == in->w && t->z == g.kept_z && t->y == g.kept_y && t->x == 1; }

template <class Rows>
int backward(const char *name, const mt_tensor *error, const mt_tensor *dgamma, const mt_tensor *dbeta, const mt_tensor *delta, const mt_tensor *gamma,
             const mt_tensor *beta, const Rows &x, const mt_tensor *mean, const mt_tensor *ivar, int func, int accumulate, const Geometry &g) {
  mt::ProfileScope prof(name);
  const float *pb = beta ? beta->p : nullptr;
  if (dgamma || dbeta) {
    ln_parameters_kernel<<<cdiv(g.N, 64), THREADS, 0, mt::stream()>>>(dgamma ? dgamma->p : nullptr, dbeta ? dbeta->p : nullptr, delta->p, gamma->p, pb, x, mean->p, ivar->p,
                                                                      g.rows, g.N, func, accumulate != 0);
    MT_LAUNCH_CHECK(name);
  }
  ln_error_kernel<<<(unsigned)(g.rows < 8192 ? g.rows : 8192), THREADS, 0, mt::stream()>>>(error->p, delta->p, gamma->p, pb, x, mean->p, ivar->p, g.rows, g.N, func);
  MT_LAUNCH_CHECK(name);
  return MT_OK;
}

// the checks that both forms share
int backward_checks(const char *name, const mt_tensor *error, const mt_tensor *dgamma, const mt_tensor *dbeta, const mt_tensor *delta, const mt_tensor *gamma,
                    const mt_tensor *beta, const mt_tensor *mean, const mt_tensor *ivar, int *func, Geometry *g) {
  if (!mt::valid_func(*func, true) || (*func != MT_F_NONE && (*func & MT_F_DIFFERENTIAL))) return mt::fail(MT_E_ARGUMENT, "%s: unknown function id %d", name, *func);
  if (*func == MT_F_LINEAR) *func = MT_F_NONE;  // derivative 1
  for (auto t : {error, delta, gamma, mean, ivar})
    if (mt::bad(t)) return mt::fail(MT_E_ARGUMENT, "%s: null tensor", name);
  int rc = geometry(name, delta, gamma, g);
  if (rc) return rc;
  if (!same_sizes(error, delta)) return mt::fail(MT_E_SHAPE, "%s: sizes do not match", name);
  if (!is_statistic(mean, delta, *g) || !is_statistic(ivar, delta, *g)) return mt::fail(MT_E_SHAPE, "%s: mean and ivar must hold one value per row", name);
  if (*func != MT_F_NONE && (mt::bad(beta) || !same_sizes(beta, gamma))) return mt::fail(MT_E_SHAPE, "%s: beta must have the sizes of gamma when a function is given", name);
  for (auto t : {dgamma, dbeta})
    if (t && (mt::bad(t) || !same_sizes(t, gamma))) return mt::fail(MT_E_SHAPE, "%s: gradients must have the sizes of gamma", name);
  if (error->p != delta->p && mt::overlap(error, delta)) return mt::fail(MT_E_ARGUMENT, "%s: the error shares a part of its memory with delta", name);
  for (auto out : {error, dgamma, dbeta})
    for (auto t : {gamma, *func != MT_F_NONE ? beta : nullptr, mean, ivar, out == error ? nullptr : delta, out == error ? nullptr : error, out == dbeta ? dgamma : nullptr})
      if (out && t && mt::overlap(out, t)) return mt::fail(MT_E_ARGUMENT, "%s: a result shares memory with another tensor", name);
  return MT_OK;
}

// nothing to normalise: the sums over no rows are zero
int backward_empty(const mt_tensor *dgamma, const mt_tensor *dbeta, int accumulate) {
  if (accumulate) return MT_OK;
  for (auto t : {dgamma, dbeta}) {
    const int rc = t ? mt_fill(t, 0.f) : MT_OK;
    if (rc) return rc;
  }
  return MT_OK;
}

}  // namespace

extern "C" {

int mt_layernorm_forward_func(const mt_tensor *out, const mt_tensor *in, const mt_tensor *gamma, const mt_tensor *beta, const mt_tensor *mean, const mt_tensor *ivar,
                              const mt_packed_tensor *packed_input, float epsilon, int func) {
  const char *name = "mt_layernorm_forward_func";
  if (!mt::valid_func(func, true) || (func != MT_F_NONE && (func & MT_F_DIFFERENTIAL))) return mt::fail(MT_E_ARGUMENT, "%s: unknown function id %d", name, func);
  for (auto t : {out, in, gamma, beta})
    if (mt::bad(t)) return mt::fail(MT_E_ARGUMENT, "%s: null tensor", name);
  for (auto t : {mean, ivar})
    if (t && mt::bad(t)) return mt::fail(MT_E_ARGUMENT, "%s: null tensor", name);
  Geometry g;
  int rc = geometry(name, in, gamma, &g);
  if (rc) return rc;
  if (!same_sizes(out, in) || !same_sizes(beta, gamma)) return mt::fail(MT_E_SHAPE, "%s: sizes do not match", name);
  for (auto t : {mean, ivar})
    if (t && !is_statistic(t, in, g)) return mt::fail(MT_E_SHAPE, "%s: mean and ivar must hold one value per row", name);
  if (out->p != in->p && mt::overlap(out, in)) return mt::fail(MT_E_ARGUMENT, "%s: the output shares a part of its memory with the input", name);
  for (auto r : {out, mean, ivar})
    for (auto t : {gamma, beta, r == out ? nullptr : in, r == out ? nullptr : out, r == ivar ? mean : nullptr})
      if (r && t && mt::overlap(r, t)) return mt::fail(MT_E_ARGUMENT, "%s: a result shares memory with another tensor", name);
  PackedView packed{};
  if (packed_input) {
    if (mt::bad(packed_input)) return mt::fail(MT_E_ARGUMENT, "%s: packed memory that is null or not 16-byte aligned", name);
    if (packed_input->w != in->w || packed_input->z != in->z || packed_input->y != in->y || packed_input->x != in->x)
      return mt::fail(MT_E_SHAPE, "%s: the packed tensor must have the input's sizes", name);
    if (!mt::packed_view(packed_input, &packed)) return mt::fail(MT_E_UNAVAILABLE, "%s: a sample of 2^31 elements or more is not supported", name);
    for (auto t : {out, in, gamma, beta, mean, ivar})
      if (t && mt::overlap(t, packed)) return mt::fail(MT_E_ARGUMENT, "%s: the packed tensor shares memory with another tensor", name);
  }
  if (g.N == 0 || g.rows == 0) return MT_OK;
  for (auto t : {out, mean, ivar}) mt::note_write(t);
  if (packed_input && (rc = mt_pack(packed_input, in))) return rc;
  mt::ProfileScope prof(name);
  ln_forward_kernel<<<(unsigned)(g.rows < 8192 ? g.rows : 8192), THREADS, 0, mt::stream()>>>(out->p, in->p, gamma->p, beta->p, mean ? mean->p : nullptr,
                                                                                             ivar ? ivar->p : nullptr, g.rows, g.N, epsilon, func);
  MT_LAUNCH_CHECK(name);
  return MT_OK;
}

int mt_layernorm_backward_func(const mt_tensor *error, const mt_tensor *dgamma, const mt_tensor *dbeta, const mt_tensor *delta, const mt_tensor *gamma,
                               const mt_tensor *beta, const mt_tensor *input, const mt_tensor *mean, const mt_tensor *ivar, int func, int accumulate) {
  const char *name = "mt_layernorm_backward_func";
  Geometry g;
  if (mt::bad(input)) return mt::fail(MT_E_ARGUMENT, "%s: null tensor", name);
  int rc = backward_checks(name, error, dgamma, dbeta, delta, gamma, beta, mean, ivar, &func, &g);
  if (rc) return rc;
  if (!same_sizes(input, delta)) return mt::fail(MT_E_SHAPE, "%s: sizes do not match", name);
  for (auto t : {error, dgamma, dbeta})
    if (t && mt::overlap(t, input)) return mt::fail(MT_E_ARGUMENT, "%s: a result shares memory with the input", name);
  if (g.N == 0 || g.rows == 0) return backward_empty(dgamma, dbeta, accumulate);
  for (auto t : {error, dgamma, dbeta}) mt::note_write(t);
  return backward(name, error, dgamma, dbeta, delta, gamma, beta, RowsF32{input->p, g.N}, mean, ivar, func, accumulate, g);
}

int mt_layernorm_backward_packed_func(const mt_tensor *error, const mt_tensor *dgamma, const mt_tensor *dbeta, const mt_tensor *delta, const mt_tensor *gamma,
                                      const mt_tensor *beta, const mt_packed_tensor *input, const mt_tensor *mean, const mt_tensor *ivar, int func,
                                      int accumulate) {
  const char *name = "mt_layernorm_backward_packed_func";
  Geometry g;
  if (mt::bad(input)) return mt::fail(MT_E_ARGUMENT, "%s: packed memory that is null or not 16-byte aligned", name);
  int rc = backward_checks(name, error, dgamma, dbeta, delta, gamma, beta, mean, ivar, &func, &g);
  if (rc) return rc;
  if (input->w != delta->w || input->z != delta->z || input->y != delta->y || input->x != delta->x) return mt::fail(MT_E_SHAPE, "%s: sizes do not match", name);
  PackedView v;
  if (!mt::packed_view(input, &v)) return mt::fail(MT_E_UNAVAILABLE, "%s: a sample of 2^31 elements or more is not supported", name);
  for (auto t : {error, dgamma, dbeta})
    if (t && mt::overlap(t, v)) return mt::fail(MT_E_ARGUMENT, "%s: a result shares memory with the input", name);
  if (g.N == 0 || g.rows == 0) return backward_empty(dgamma, dbeta, accumulate);
  for (auto t : {error, dgamma, dbeta}) mt::note_write(t);
  return backward(name, error, dgamma, dbeta, delta, gamma, beta, RowsPacked{v, g.N, g.per_sample}, mean, ivar, func, accumulate, g);
}

}  // extern "C"
