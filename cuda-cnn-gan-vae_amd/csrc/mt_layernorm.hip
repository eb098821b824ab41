// Layer normalisation: every row of N values is normalised by its own mean and variance, so a sample's result does not depend
// on the batch.
//   mean = sum(x) / N,  ivar = 1 / sqrt(sum((x - mean)^2) / N + epsilon),  xhat = (x - mean) * ivar,  y = f(gamma * xhat + beta)
// Backward, with g = delta * f'(gamma * xhat + beta) and u = g * gamma:
//   error = ivar * (u - sum(u) / N - xhat * sum(u * xhat) / N),  dgamma = sum over the rows of g * xhat,  dbeta = of g
//
// All of it is bound by memory: the forward pass has to read x and write y, the backward pass to read delta and x and write the
// error.  A row is therefore held in registers between its sums and its results wherever it fits (8 to 1024 threads per row, up
// to 32 values per thread); longer rows are cut into pieces that several blocks share, and their second look at x finds it in
// the caches.  Variances are sums of squared deviations from the mean (two passes over registers), never E[x^2] - E[x]^2.
#include <initializer_list>
#include <type_traits>

#include "mt_packed.h"

namespace {

using mt::cdiv;
using mt::PackedView;

constexpr int THREADS = 256;

// ---- sums over the threads of a row; every thread gets the same bits ----------------------------------------------------
// over the L threads of a row; `part` (L / 64 values, rows of whole blocks) is used once: no second barrier
template <int L>
__device__ __forceinline__ float row_sum(float v, float *part) {
  v = mt::over_lanes<mt::Sum, L < 64 ? L : 64>(v);
  if (L > 64) {
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int k = 1; k < L / 64; k++) v += part[k];
  }
  return v;
}

// ---- the functions of the function layer that the kernels hold: the values of f_sigmoid_fast and f_tangence_fast, with a reciprocal
// that is not a division (two thirds of the instructions; 32 rows of 147456 with sigmoid 12.8 -> 11.8 us) ---------------------------
// (`e` the exponential, `r` the reciprocal of 1 + e: the derivatives are (1 - f) * f = e * r * r and 1 - f * f = 4 * e * r * r, without the
// difference of two neighbouring numbers)
struct Exponential {
  float e, r;
};
__device__ __forceinline__ Exponential exponential(float v) {
  Exponential t;
  t.e = __expf(v);
  t.r = mt::reciprocal(1.f + t.e);
  return t;
}
__device__ __forceinline__ Exponential for_sigmoid(float v) {
  if (v > 30.f) v = 29.99999f;
  if (v < -30.f) v = -29.99999f;
  return exponential(-v);
}
__device__ __forceinline__ Exponential for_tangence(float v) {
  if (v > 30.f) v = 30.f;  // 1 from there on; an infinite exponential has no reciprocal here
  return exponential(2.f * v);
}
template <int N>
__device__ __forceinline__ void apply(int func, float *v) {
  if (func == MT_F_SIGMOID) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = for_sigmoid(v[i]).r;
  } else if (func == MT_F_TANGENCE) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = 1.f - 2.f * for_tangence(v[i]).r;
  } else {
    mt::apply_func_cheap_many<N>(func, v);
  }
}

// ---- one step of a thread: one value, or four neighbouring ones: from a 16-byte boundary, the same past the caches, for tensors that are
// too large for them and touched once (option "nontemporal": 128 MiB and more; 16384 x 4096 forward 102 -> 98 us, backward 148 -> 139; a
// flag at run time does not do: the compiler merges the two accesses into the ordinary one), or from any address, for rows of any
// length (1344 x 10319 backward 73 us with single values, 59 so) ---------------------------------------------------------------------
enum Access { ONE, FOUR, FOUR_PAST, FOUR_ANY };
constexpr int kept(int access) { return access == FOUR_PAST ? FOUR : access; }  // for what is read again
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));
template <int ACCESS>
__device__ __forceinline__ void load_step(float *t, const float *p, int at) {
  if (ACCESS == ONE) {
    t[0] = p[at];
  } else {
    floatx4 v;
    if (ACCESS == FOUR_ANY)
      v = *reinterpret_cast<const floatx4_any *>(p + at);
    else if (ACCESS == FOUR_PAST)
      v = __builtin_nontemporal_load(reinterpret_cast<const floatx4 *>(p + at));
    else
      v = *reinterpret_cast<const floatx4 *>(p + at);
    t[0] = v.x; t[1] = v.y; t[2] = v.z; t[3] = v.w;
  }
}
// `left`: values from p to the end
template <int ACCESS>
__device__ __forceinline__ void store_step(float *p, const float *t, uint32_t left) {
  if (ACCESS == ONE) {
    *p = t[0];
  } else {
    const floatx4 v = {t[0], t[1], t[2], t[3]};
    if (ACCESS == FOUR_PAST)
      __builtin_nontemporal_store(v, reinterpret_cast<floatx4 *>(p));
    else if (ACCESS == FOUR)
      *reinterpret_cast<floatx4 *>(p) = v;
    else if (left >= 4)
      *reinterpret_cast<floatx4_any *>(p) = v;
    else
#pragma unroll
      for (uint32_t e = 0; e < 3; e++)
        if (e < left) p[e] = t[e];
  }
}
// Where the step that starts at `first` of N values loads: steps that would pass the end load the last four (a piece of fewer than four
// reaches into the piece before), and are then moved into place
template <int ACCESS>
__device__ __forceinline__ int load_at(uint32_t first, uint32_t N) { return min((int)first, (int)N - (ACCESS == ONE ? 1 : 4)); }
template <int ACCESS>
__device__ __forceinline__ void settle(float *t, uint32_t first, uint32_t N) {
  if (ACCESS == FOUR_ANY) {
    const uint32_t by = first < N && first + 4 > N ? first + 4 - N : 0u;  // 0 to 3
    const float a = t[0], b = t[1], c = t[2], d = t[3];  // (selects between elements of an array would put it into memory)
    t[0] = by == 0 ? a : by == 1 ? b : by == 2 ? c : d;
    t[1] = by == 0 ? b : by == 1 ? c : by == 2 ? d : 0.f;
    t[2] = by == 0 ? c : by == 1 ? d : 0.f;
    t[3] = by == 0 ? d : 0.f;
  }
}

// ---- how the L threads of a row share its N values: E each, in vectors of four 4 * L apart, or singly L apart ----------------
template <int L, int E, int ACCESS>
struct Share {
  static constexpr int STEPS = ACCESS != ONE ? E / 4 : E, WIDTH = ACCESS != ONE ? 4 : 1;
  static __device__ __forceinline__ uint32_t first(int j) { return (j * L + threadIdx.x % L) * WIDTH; }
  static __device__ __forceinline__ bool inside(int j, int e, uint32_t N) { return first(j) + (ACCESS == FOUR_ANY ? e : 0) < N; }
  // values behind the end count as 0
  template <int HOW = kept(ACCESS)>
  static __device__ __forceinline__ void load(float (&v)[E], const float *p, uint32_t N) {
#pragma unroll
    for (int j = 0; j < STEPS; j++) load_step<HOW>(v + j * WIDTH, p, load_at<HOW>(first(j), N));
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
      settle<HOW>(v + j * WIDTH, first(j), N);
#pragma unroll
      for (int e = 0; e < WIDTH; e++) v[j * WIDTH + e] = first(j) < N ? v[j * WIDTH + e] : 0.f;
    }
  }
};

// ---- where a row's input comes from in the backward pass: the fp32 tensor, or the 8 bits the forward pass kept.  Loading and
// decoding are two steps, so that all loads of a row are under way before the first is waited for ------------------------------
struct RowsF32 {
  static constexpr int BYTES = 4;  // of a value, about
  bool in_fours() const { return true; }
  const float *p;
  uint32_t N;
  template <bool VEC>
  struct Raw {
    float t[VEC ? 4 : 1];
    __device__ __forceinline__ void values(float *x) const {
#pragma unroll
      for (int k = 0; k < (VEC ? 4 : 1); k++) x[k] = t[k];
    }
  };
  struct Row {
    const float *p;
    template <int ACCESS>
    __device__ __forceinline__ void load(Raw<ACCESS != ONE> &raw, int at) const { load_step<ACCESS>(raw.t, p, at); }
  };
  template <int ACCESS>
  static __device__ __forceinline__ int at(uint32_t first, uint32_t N) { return load_at<ACCESS>(first, N); }
  template <int ACCESS>
  static __device__ __forceinline__ void settle_values(float *x, uint32_t first, uint32_t N) { settle<ACCESS>(x, first, N); }
  __device__ __forceinline__ Row row(uint32_t r) const { return Row{p + (size_t)r * N}; }
};
struct RowsPacked {
  static constexpr int BYTES = 1;
  PackedView v;
  uint32_t N, per_sample;  // rows of one sample
  bool in_fours() const { return N % 4 == 0 || per_sample == 1; }  // do four neighbouring values lie in one group
  template <bool VEC>
  struct Raw {
    float2 pair;
    uint32_t q;
    __device__ __forceinline__ void values(float *x) const {
#pragma unroll
      for (int k = 0; k < (VEC ? 4 : 1); k++) x[k] = mt::unpack_value(pair, VEC ? (q >> (8 * k)) & 255u : q);
    }
  };
  struct Row {
    const uint8_t *q;
    const float2 *pair;
    uint32_t first;  // the row's first value within its sample
    template <int ACCESS>
    __device__ __forceinline__ void load(Raw<ACCESS != ONE> &raw, int at) const {
      const uint32_t e = first + at;
      raw.pair = pair[e / mt::PACK_GROUP];
      raw.q = ACCESS != ONE ? *reinterpret_cast<const uint32_t *>(q + e) : q[e];
    }
  };
  // (four bytes of one group, from a multiple of four: those behind a sample's end are its padding)
  template <int ACCESS>
  static __device__ __forceinline__ int at(uint32_t first, uint32_t N) { return ACCESS == ONE ? min(first, N - 1) : min(first, (N - 1) & ~3u); }
  template <int ACCESS>
  static __device__ __forceinline__ void settle_values(float *, uint32_t, uint32_t) {}
  __device__ __forceinline__ Row row(uint32_t r) const {
    const uint32_t w = per_sample == 1 ? r : r / per_sample;
    return Row{v.q + (size_t)w * v.pitch, v.pair + (size_t)w * v.groups, (r - w * per_sample) * N};
  }
};

// the 8 bits of one vector per lane, 32 lanes a group: a lane's first `left` values are the row's; lanes behind the end of the sample
// write its padding
__device__ __forceinline__ void pack_step(const PackedView &out, size_t sample, uint32_t e, int left, const float *t) {
  const bool valid = left > 0;
  float u[4];
#pragma unroll
  for (int k = 0; k < 4; k++) u[k] = k < left ? t[k] : t[0];
  float low = mt::min_nan(mt::min_nan(u[0], u[1]), mt::min_nan(u[2], u[3])), high = mt::max_nan(mt::max_nan(u[0], u[1]), mt::max_nan(u[2], u[3]));
  low = mt::over_lanes<mt::Lowest, 32>(valid ? low : __int_as_float(0x7f800000));
  high = mt::over_lanes<mt::Highest, 32>(valid ? high : __int_as_float(0xff800000));
  const mt::PackScale s = mt::pack_scale(low, high);
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4; k++) w = mt::pack_into(s, u[k], k, w);
  if (left < 4) w &= valid ? (1u << 8 * left) - 1u : 0u;
  if (valid || (e >= out.n && e < out.pitch)) *reinterpret_cast<uint32_t *>(out.q + sample * out.pitch + e) = w;
  if (valid && e % mt::PACK_GROUP == 0) out.pair[sample * out.groups + e / mt::PACK_GROUP] = make_float2(s.low, s.step);
}

// ---- forward -------------------------------------------------------------------------------------------------------
struct Forward {
  float *out;
  const float *in, *gamma, *beta;
  float *mean, *ivar;  // null: not wanted
  PackedView packed;
  uint32_t first_row, rows, N, per_sample;  // first_row: of this launch
  float eps;
  int func;
};

// gamma and beta of a thread's share of a row: in registers, or loaded where they are used (1024 threads with 32 values of x each
// have no registers for them: 1000 x 32768 61 us, 65 with them)
template <int L, int E, int ACCESS>
struct Parameters {
  using S = Share<L, E, ACCESS>;
  static constexpr bool HELD = E <= 16;
  float gamma[HELD ? E : 1], beta[HELD ? E : 1];
  __device__ __forceinline__ void load(const float *g, const float *b, uint32_t N) {
    if constexpr (HELD) {
      S::load(gamma, g, N);
      S::load(beta, b, N);
    }
  }
  __device__ __forceinline__ void step(const float *g, const float *b, int j, uint32_t N, float *tg, float *tb) const {
    if constexpr (HELD) {
#pragma unroll
      for (int e = 0; e < S::WIDTH; e++) {
        tg[e] = gamma[j * S::WIDTH + e];
        tb[e] = beta[j * S::WIDTH + e];
      }
    } else {
      const uint32_t first = S::first(j);
      load_step<ACCESS>(tg, g, load_at<ACCESS>(first, N));
      load_step<ACCESS>(tb, b, load_at<ACCESS>(first, N));
      settle<ACCESS>(tg, first, N);
      settle<ACCESS>(tb, first, N);
    }
  }
};

// gamma * xhat + beta and the function, from x in registers
template <int L, int E, int ACCESS>
__device__ __forceinline__ void normalise(int func, float *out, const float (&x)[E], float mean, float ivar, const Parameters<L, E, kept(ACCESS)> &held, const float *gamma,
                                          const float *beta, uint32_t N) {
  using S = Share<L, E, ACCESS>;
#pragma unroll
  for (int j = 0; j < S::STEPS; j++) {
    if (S::first(j) >= N) continue;
    float g[S::WIDTH], b[S::WIDTH], y[S::WIDTH];
    held.step(gamma, beta, j, N, g, b);
#pragma unroll
    for (int e = 0; e < S::WIDTH; e++) y[e] = g[e] * ((x[j * S::WIDTH + e] - mean) * ivar) + b[e];
    apply<S::WIDTH>(func, y);
    store_step<ACCESS>(out + S::first(j), y, N - S::first(j));
  }
}

// rows that fit the registers of L threads
template <int L, int E, int ACCESS, bool PACK>
__global__ __launch_bounds__(L < 256 ? 256 : L) void ln_forward_kernel(Forward a) {
  using S = Share<L, E, ACCESS>;
  constexpr uint32_t PER_BLOCK = L < 256 ? 256 / L : 1;
  __shared__ float part[2][L / 64 + 1];
  const uint32_t want = a.first_row + blockIdx.x * PER_BLOCK + threadIdx.x / L, row = min(want, a.rows - 1);
  const bool mine = want < a.rows;
  float x[E];
  Parameters<L, E, kept(ACCESS)> held;
  S::template load<ACCESS>(x, a.in + (size_t)row * a.N, a.N);
  // the parameters are under way with the row where a wavefront or less holds it (12000 x 1024 20.6 -> 19.8 us, 60000 x 128 11.7 -> 10.6); more
  // threads per row lose more from the registers (2000 x 16384 55.3 -> 63.8)
  constexpr bool EARLY = L <= 64;
  if constexpr (EARLY) {
    held.load(a.gamma, a.beta, a.N);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (PACK) {
    const uint32_t w = a.per_sample == 1 ? row : row / a.per_sample, e0 = (row - w * a.per_sample) * a.N;
#pragma unroll
    for (int j = 0; j < S::STEPS; j++)
      if (mine) pack_step(a.packed, w, e0 + S::first(j), (int)a.N - (int)S::first(j), x + j * S::WIDTH);
  }
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < E; k++) s += x[k];
  const float mean = row_sum<L>(s, part[0]) / (float)a.N;
  s = 0.f;
#pragma unroll
  for (int j = 0; j < S::STEPS; j++)
#pragma unroll
    for (int e = 0; e < S::WIDTH; e++) {
      const float d = S::inside(j, e, a.N) ? x[j * S::WIDTH + e] - mean : 0.f;
      s += d * d;
    }
  const float ivar = 1.f / sqrtf(row_sum<L>(s, part[1]) / (float)a.N + a.eps);
  if (!mine) return;
  if constexpr (!EARLY) held.load(a.gamma, a.beta, a.N);
  normalise<L, E, ACCESS>(a.func, a.out + (size_t)row * a.N, x, mean, ivar, held, a.gamma, a.beta, a.N);
  if (threadIdx.x % L == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.ivar) a.ivar[row] = ivar;
  }
}

// longer rows: pieces of PIECE values, one block each.  First the mean and the sum of squared deviations of every piece ...
constexpr uint32_t PIECE = 4096;  // 32 x 196608 14.3 us, 16.0 in pieces of 2048, 14.8 of 8192
template <int ACCESS, bool PACK>
__global__ __launch_bounds__(THREADS) void ln_pieces_kernel(Forward a, float2 *stats, uint32_t pieces) {
  using S = Share<THREADS, PIECE / THREADS, ACCESS>;
  __shared__ float part[2][THREADS / 64];
  const uint32_t local = blockIdx.x / pieces, row = a.first_row + local, piece = blockIdx.x - local * pieces, n = min(PIECE, a.N - piece * PIECE);
  float x[PIECE / THREADS];
  S::load(x, a.in + (size_t)row * a.N + (size_t)piece * PIECE, n);
  if (PACK) {
    const uint32_t w = a.per_sample == 1 ? row : row / a.per_sample, e0 = (row - w * a.per_sample) * a.N + piece * PIECE;
#pragma unroll
    for (int j = 0; j < S::STEPS; j++) pack_step(a.packed, w, e0 + S::first(j), (int)n - (int)S::first(j), x + j * S::WIDTH);
  }
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < (int)(PIECE / THREADS); k++) s += x[k];
  const float mean = row_sum<THREADS>(s, part[0]) / (float)n;
  s = 0.f;
#pragma unroll
  for (int j = 0; j < S::STEPS; j++)
#pragma unroll
    for (int e = 0; e < S::WIDTH; e++) {
      const float d = S::inside(j, e, n) ? x[j * S::WIDTH + e] - mean : 0.f;
      s += d * d;
    }
  s = row_sum<THREADS>(s, part[1]);
  if (threadIdx.x == 0) stats[blockIdx.x] = make_float2(mean, s);
}
// ... then every block joins the pieces of its row (each wavefront for itself: the sum of deviations of a piece moves by
// n * (its mean - the row's mean)^2) and normalises its own piece
template <int ACCESS>
__global__ __launch_bounds__(THREADS) void ln_apply_kernel(Forward a, const float2 *stats, uint32_t pieces) {
  using S = Share<THREADS, PIECE / THREADS, ACCESS>;
  const uint32_t local = blockIdx.x / pieces, row = a.first_row + local, piece = blockIdx.x - local * pieces, lane = threadIdx.x % 64, n = min(PIECE, a.N - piece * PIECE);
  const size_t at = (size_t)row * a.N + (size_t)piece * PIECE;
  float x[PIECE / THREADS];
  S::template load<ACCESS>(x, a.in + at, n);
  stats += (size_t)local * pieces;
  float s = 0.f;
  for (uint32_t p = lane; p < pieces; p += 64) s += stats[p].x * (float)min(PIECE, a.N - p * PIECE);
  const float mean = mt::over_lanes<mt::Sum, 64>(s) / (float)a.N;
  s = 0.f;
  for (uint32_t p = lane; p < pieces; p += 64) {
    const float2 t = stats[p];
    const float d = t.x - mean;
    s += t.y + d * d * (float)min(PIECE, a.N - p * PIECE);
  }
  const float ivar = 1.f / sqrtf(mt::over_lanes<mt::Sum, 64>(s) / (float)a.N + a.eps);
  const float *gamma = a.gamma + (size_t)piece * PIECE, *beta = a.beta + (size_t)piece * PIECE;
  Parameters<THREADS, PIECE / THREADS, kept(ACCESS)> held;
  held.load(gamma, beta, n);
  normalise<THREADS, PIECE / THREADS, ACCESS>(a.func, a.out + at, x, mean, ivar, held, gamma, beta, n);
  if (piece == 0 && threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.ivar) a.ivar[row] = ivar;
  }
}

// ---- backward ------------------------------------------------------------------------------------------------------
struct Backward {
  float *error;
  float *dgamma, *dbeta;  // null: not wanted
  const float *delta, *gamma, *beta, *mean, *ivar;
  uint32_t rows, N;
  int func;
  bool accumulate;
};

// delta * f'(gamma * xhat + beta) for N values, one look at the (uniform) function for all of them; the kernels are compiled with and
// without a function (a look per value and a load of beta at every step made 8192 x 2048 take 81 us with tangence, 34 without)
template <int N>
__device__ __forceinline__ void fronts(int func, float *g, const float *gamma, const float *xhat, const float *beta) {
  if (func == MT_F_RELU) {
#pragma unroll
    for (int i = 0; i < N; i++) g[i] *= gamma[i] * xhat[i] + beta[i] >= 0.f ? 1.f : 0.f;
  } else if (func == MT_F_LEAKY_RELU) {
#pragma unroll
    for (int i = 0; i < N; i++) g[i] *= gamma[i] * xhat[i] + beta[i] >= 0.f ? 1.f : 0.1f;
  } else if (func == MT_F_SIGMOID) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const Exponential t = for_sigmoid(gamma[i] * xhat[i] + beta[i]);
      g[i] *= t.e * t.r * t.r;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const Exponential t = for_tangence(gamma[i] * xhat[i] + beta[i]);
      g[i] *= 4.f * (t.e * t.r) * t.r;
    }
  }
}

// the sums of `parts` rows of partial sums [2][parts][N] (of g * xhat, of g), joined in a fixed order.  Many parts: 32 columns per
// block, whose 32 slices take every 32nd row with eight loads under way (4 slices of 64 columns took 7.4 us for 512 rows of 2000, waiting
// for one batch of loads after the other; 16 of 64 take 4.8, 32 of 32 another 0.6 to 0.9 less).  Few parts of long rows: a
// thread per column (16 slices took 14 us for 8 rows of 147456).
constexpr uint32_t JOIN_MANY = 32, JOIN_COLUMNS = 32;
template <int SLICES>
__global__ __launch_bounds__(SLICES == 1 ? THREADS : JOIN_COLUMNS * SLICES) void ln_join_kernel(float *dgamma, float *dbeta, const float *partial, uint32_t parts, uint32_t N,
                                                                                     bool accumulate) {
  constexpr uint32_t COLUMNS = SLICES == 1 ? THREADS : JOIN_COLUMNS;
  __shared__ float sums[SLICES][COLUMNS];
  const uint32_t i = blockIdx.x * COLUMNS + threadIdx.x % COLUMNS, slice = threadIdx.x / COLUMNS;
  float *out = blockIdx.y == 0 ? dgamma : dbeta;
  if (out == nullptr) return;
  const float *p = partial + (size_t)blockIdx.y * parts * N + min(i, N - 1);
  float s = 0.f;
  for (uint32_t k = slice; k < parts; k += 8 * SLICES) {
    float t[8];
#pragma unroll
    for (int u = 0; u < 8; u++) t[u] = k + u * SLICES < parts ? p[(size_t)(k + u * SLICES) * N] : 0.f;
    s += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
  }
  if (SLICES > 1) {
    sums[slice][threadIdx.x % COLUMNS] = s;
    __syncthreads();
    if (slice != 0) return;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < SLICES; k += 4)
      s += (sums[k][threadIdx.x] + sums[k + 1 < SLICES ? k + 1 : 0][threadIdx.x]) + (sums[k + 2 < SLICES ? k + 2 : 0][threadIdx.x] + sums[k + 3 < SLICES ? k + 3 : 0][threadIdx.x]);
  }
  if (i < N) out[i] = accumulate ? out[i] + s : s;
}

// Threads of its block: two wavefronts per SIMD, whose sums are joined in LDS, where the registers of a row's loads leave room (256 threads:
// 4000 x 4001 49 us against 45, from 8 bits 46 against 38, 6000 x 777 17.4 against 14.8); sixteen values per thread in fours from 16-byte
// boundaries have enough under way with one (12000 x 1000 32.1 us, 34.1 with 512 threads)
constexpr int backward_block(int L, int E, int access) { return L > 256 ? L : E == 16 && (access == FOUR || access == FOUR_PAST) ? 256 : 512; }

// rows that fit the registers of L threads; a block walks over the rows and keeps its share of dgamma and dbeta in registers
template <int L, int E, int ACCESS, bool FUNC, class Rows>
__global__ __launch_bounds__(backward_block(L, E, ACCESS)) void ln_backward_kernel(Backward a, Rows rows, float *partial) {
  constexpr bool VEC = ACCESS != ONE;
  using S = Share<L, E, ACCESS>;
  constexpr uint32_t BLOCK = backward_block(L, E, ACCESS), PER_BLOCK = BLOCK / L;
  constexpr int W = S::WIDTH;
  __shared__ float part[2][2][PER_BLOCK][L / 64 + 1];
  __shared__ float shared[PER_BLOCK > 1 ? 2 * BLOCK * E : 1];
  const uint32_t sub = threadIdx.x / L, lane = threadIdx.x % L;
  constexpr bool HELD = L < 1024;  // gamma and beta stay in registers; 1024 threads load them for every row
  float dg[E], db[E], gamma[E], beta[FUNC ? E : 1];
  const auto load_parameters = [&] {
    S::load(gamma, a.gamma, a.N);
    if constexpr (FUNC) S::load(beta, a.beta, a.N);
  };
  if constexpr (HELD) load_parameters();
#pragma unroll
  for (int k = 0; k < E; k++) dg[k] = db[k] = 0.f;
  uint32_t turn = 0;
  // the next row is loaded before the row in hand is summed and stored, where the registers allow (1024 threads have 128 each; single
  // values need an address each).  The error may be written over delta: a row is stored after its own loads, and by the threads that
  // loaded it
  constexpr bool EARLY = VEC && L < 1024;
  const uint32_t stride = gridDim.x * PER_BLOCK;
  typedef typename Rows::template Raw<VEC> Raw;
  Raw raw[S::STEPS], next[EARLY ? S::STEPS : 1];
  float x[E], g[E], gn[EARLY ? E : 1], mean, ivar;
  const auto load = [&](uint32_t row, Raw *r, float (&gr)[E], float *m, float *v) {
    *m = a.mean[row];
    *v = a.ivar[row];
    const auto in = rows.row(row);
    S::template load<ACCESS>(gr, a.delta + (size_t)row * a.N, a.N);
#pragma unroll
    for (int j = 0; j < S::STEPS; j++) in.template load<ACCESS>(r[j], Rows::template at<ACCESS>(S::first(j), a.N));
  };
  if constexpr (EARLY) load(min(blockIdx.x * PER_BLOCK + sub, a.rows - 1), raw, g, &mean, &ivar);
  for (uint32_t first = blockIdx.x * PER_BLOCK; first < a.rows; first += stride, turn ^= 1u) {
    const uint32_t row = min(first + sub, a.rows - 1);
    const bool mine = first + sub < a.rows;
    float mean_n, ivar_n;
    if constexpr (EARLY)
      load(min(first + stride + sub, a.rows - 1), next, gn, &mean_n, &ivar_n);
    else
      load(row, raw, g, &mean, &ivar);
    if constexpr (!HELD) load_parameters();
    __builtin_amdgcn_sched_barrier(0);  // all loads before the first use of one
#pragma unroll
    for (int j = 0; j < S::STEPS; j++) {
      raw[j].values(x + j * W);
      Rows::template settle_values<ACCESS>(x + j * W, S::first(j), a.N);
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < E; k++) x[k] = (x[k] - mean) * ivar;
    if constexpr (FUNC) fronts<E>(a.func, g, gamma, x, beta);
#pragma unroll
    for (int j = 0; j < S::STEPS; j++) {
#pragma unroll
      for (int e = 0; e < W; e++) {
        const int k = j * W + e;
        if (S::first(j) >= a.N) x[k] = g[k] = 0.f;
        if (mine) {
          dg[k] += g[k] * x[k];
          db[k] += g[k];
        }
        g[k] *= gamma[k];
        s1 += g[k];
        s2 += g[k] * x[k];
      }
    }
    // both sums with one barrier; the next row uses the other half of `part`
    s1 = mt::over_lanes<mt::Sum, L < 64 ? L : 64>(s1);
    s2 = mt::over_lanes<mt::Sum, L < 64 ? L : 64>(s2);
    if (L > 64) {
      if (threadIdx.x % 64 == 0) {
        part[turn][0][sub][lane / 64] = s1;
        part[turn][1][sub][lane / 64] = s2;
      }
      __syncthreads();
      s1 = part[turn][0][sub][0];
      s2 = part[turn][1][sub][0];
#pragma unroll
      for (int k = 1; k < L / 64; k++) {
        s1 += part[turn][0][sub][k];
        s2 += part[turn][1][sub][k];
      }
    }
    s1 /= (float)a.N;
    s2 /= (float)a.N;
    float *error = a.error + (size_t)row * a.N;
    if (mine) {
#pragma unroll
      for (int j = 0; j < S::STEPS; j++) {
        if (S::first(j) >= a.N) continue;
        float t[W];
#pragma unroll
        for (int e = 0; e < W; e++) t[e] = ivar * ((g[j * W + e] - s1) - x[j * W + e] * s2);
        store_step<ACCESS>(error + S::first(j), t, a.N - S::first(j));
      }
    }
    if constexpr (EARLY) {
#pragma unroll
      for (int j = 0; j < S::STEPS; j++) raw[j] = next[j];
#pragma unroll
      for (int k = 0; k < E; k++) g[k] = gn[k];
      mean = mean_n;
      ivar = ivar_n;
    }
  }
  float *pg = partial + (size_t)blockIdx.x * a.N, *pb = partial + ((size_t)gridDim.x + blockIdx.x) * a.N;
  if (PER_BLOCK == 1) {
#pragma unroll
    for (int j = 0; j < S::STEPS; j++)
      if (S::first(j) < a.N) {
        store_step<kept(ACCESS)>(pg + S::first(j), dg + j * W, a.N - S::first(j));
        store_step<kept(ACCESS)>(pb + S::first(j), db + j * W, a.N - S::first(j));
      }
    return;
  }
  // the block's rows of partial sums, joined in LDS: [of g * xhat, of g][row of the block][value]
#pragma unroll
  for (int j = 0; j < S::STEPS; j++)
#pragma unroll
    for (int e = 0; e < W; e++) {
      shared[sub * (L * E) + S::first(j) + e] = dg[j * W + e];
      shared[BLOCK * E + sub * (L * E) + S::first(j) + e] = db[j * W + e];
    }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < a.N; i += BLOCK) {
    float sg = 0.f, sb = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < PER_BLOCK; k++) {
      sg += shared[k * (L * E) + i];
      sb += shared[BLOCK * E + k * (L * E) + i];
    }
    pg[i] = sg;
    pb[i] = sb;
  }
}

// The error alone, one row per L threads, and beside it in the same launch (blocks from error_blocks on) dgamma and dbeta straight
// from delta and x: they need no sum over a row.  That reads both a second time, from the caches, where the kernel above writes and
// joins partial sums: 256 rows of 4096 10.7 -> 5.2 us, 33 of 1001 7.0 -> 4.9; 8192 of 2048 would lose (36 us against 50).
template <int L, int E, int ACCESS, bool FUNC, class Rows>
__global__ __launch_bounds__(L < 256 ? 256 : L) void ln_backward_few_kernel(Backward a, Rows rows, uint32_t first_row, uint32_t error_blocks) {
  constexpr bool VEC = ACCESS != ONE;
  using S = Share<L, E, ACCESS>;
  constexpr uint32_t PER_BLOCK = L < 256 ? 256 / L : 1, BLOCK = L < 256 ? 256 : L;
  constexpr int W = S::WIDTH;
  if (blockIdx.x >= error_blocks) {
    // BLOCK / 16 columns, sixteen rows at a time with four loads of each operand in flight
    constexpr uint32_t COLUMNS = BLOCK / 16;
    __shared__ float sums[2][16][COLUMNS];
    const uint32_t c = threadIdx.x % COLUMNS, slice = threadIdx.x / COLUMNS, column = (blockIdx.x - error_blocks) * COLUMNS + c, i = min(column, a.N - 1);
    float gamma[4], beta[4] = {}, sg = 0.f, sb = 0.f;
    gamma[0] = gamma[1] = gamma[2] = gamma[3] = a.gamma[i];
    if (FUNC) beta[0] = beta[1] = beta[2] = beta[3] = a.beta[i];
    for (uint32_t k = slice; k < a.rows; k += 64) {
      typename Rows::template Raw<false> raw[4];
      float x[4], g[4], mean[4], ivar[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const uint32_t row = min(k + 16 * u, a.rows - 1);
        g[u] = a.delta[(size_t)row * a.N + i];
        rows.row(row).template load<ONE>(raw[u], i);
        mean[u] = a.mean[row];
        ivar[u] = a.ivar[row];
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        raw[u].values(x + u);
        x[u] = (x[u] - mean[u]) * ivar[u];
      }
      if constexpr (FUNC) fronts<4>(a.func, g, gamma, x, beta);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        if (k + 16 * u < a.rows) {
          sg += g[u] * x[u];
          sb += g[u];
        }
      }
    }
    sums[0][slice][c] = sg;
    sums[1][slice][c] = sb;
    __syncthreads();
    if (slice > 1 || column >= a.N) return;
    float *out = slice == 0 ? a.dgamma : a.dbeta;
    if (out == nullptr) return;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; k += 4) s += (sums[slice][k][c] + sums[slice][k + 1][c]) + (sums[slice][k + 2][c] + sums[slice][k + 3][c]);
    out[column] = a.accumulate ? out[column] + s : s;
    return;
  }
  __shared__ float part[2][L / 64 + 1];
  const uint32_t want = first_row + blockIdx.x * PER_BLOCK + threadIdx.x / L, row = min(want, a.rows - 1);
  const float mean = a.mean[row], ivar = a.ivar[row];
  const auto in = rows.row(row);
  typename Rows::template Raw<VEC> raw[S::STEPS];
  float x[E], g[E], gamma[E], beta[FUNC ? E : 1];
  S::template load<ACCESS>(g, a.delta + (size_t)row * a.N, a.N);
#pragma unroll
  for (int j = 0; j < S::STEPS; j++) in.template load<ACCESS>(raw[j], Rows::template at<ACCESS>(S::first(j), a.N));
  S::load(gamma, a.gamma, a.N);
  if constexpr (FUNC) S::load(beta, a.beta, a.N);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < S::STEPS; j++) {
    raw[j].values(x + j * W);
    Rows::template settle_values<ACCESS>(x + j * W, S::first(j), a.N);
  }
  float s1 = 0.f, s2 = 0.f;
#pragma unroll
  for (int k = 0; k < E; k++) x[k] = (x[k] - mean) * ivar;
  if constexpr (FUNC) fronts<E>(a.func, g, gamma, x, beta);
#pragma unroll
  for (int j = 0; j < S::STEPS; j++) {
#pragma unroll
    for (int e = 0; e < W; e++) {
      const int k = j * W + e;
      g[k] *= gamma[k];
      s1 += S::first(j) < a.N ? g[k] : 0.f;
      s2 += S::first(j) < a.N ? g[k] * x[k] : 0.f;
    }
  }
  s1 = row_sum<L>(s1, part[0]) / (float)a.N;
  s2 = row_sum<L>(s2, part[1]) / (float)a.N;
  if (want >= a.rows) return;
#pragma unroll
  for (int j = 0; j < S::STEPS; j++) {
    if (S::first(j) >= a.N) continue;
    float t[W];
#pragma unroll
    for (int e = 0; e < W; e++) t[e] = ivar * ((g[j * W + e] - s1) - x[j * W + e] * s2);
    store_step<ACCESS>(a.error + (size_t)row * a.N + S::first(j), t, a.N - S::first(j));
  }
}

// longer rows: the two sums of every piece ...
template <int ACCESS, bool FUNC, class Rows>
__global__ __launch_bounds__(THREADS) void ln_backward_pieces_kernel(Backward a, Rows rows, float2 *sums, uint32_t pieces) {
  constexpr bool VEC = ACCESS != ONE;
  using S = Share<THREADS, PIECE / THREADS, ACCESS>;
  constexpr int W = S::WIDTH;
  __shared__ float part[2][THREADS / 64];
  const uint32_t row = blockIdx.x / pieces, piece = blockIdx.x - row * pieces, n = min(PIECE, a.N - piece * PIECE), at = piece * PIECE;
  const float mean = a.mean[row], ivar = a.ivar[row];
  const auto in = rows.row(row);
  typename Rows::template Raw<VEC> raw[S::STEPS];
  float x[PIECE / THREADS], g[PIECE / THREADS];
  S::load(g, a.delta + (size_t)row * a.N + at, n);
#pragma unroll
  for (int j = 0; j < S::STEPS; j++) in.template load<ACCESS>(raw[j], (int)at + Rows::template at<ACCESS>(S::first(j), n));
  float gamma[PIECE / THREADS], beta[FUNC ? PIECE / THREADS : 1];
  S::load(gamma, a.gamma + at, n);
  if constexpr (FUNC) S::load(beta, a.beta + at, n);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < S::STEPS; j++) {
    raw[j].values(x + j * W);
    Rows::template settle_values<ACCESS>(x + j * W, S::first(j), n);
  }
  float s1 = 0.f, s2 = 0.f;
#pragma unroll
  for (int k = 0; k < (int)(PIECE / THREADS); k++) x[k] = (x[k] - mean) * ivar;
  if constexpr (FUNC) fronts<PIECE / THREADS>(a.func, g, gamma, x, beta);
#pragma unroll
  for (int j = 0; j < S::STEPS; j++) {
#pragma unroll
    for (int e = 0; e < W; e++) {
      const float u = S::first(j) < n ? g[j * W + e] * gamma[j * W + e] : 0.f;
      s1 += u;
      s2 += S::first(j) < n ? u * x[j * W + e] : 0.f;
    }
  }
  s1 = row_sum<THREADS>(s1, part[0]);
  s2 = row_sum<THREADS>(s2, part[1]);
  if (threadIdx.x == 0) sums[blockIdx.x] = make_float2(s1, s2);
}
// ... then blocks of 64 * WIDTH columns whose four wavefronts take every fourth row of a group: the error, and their columns' share of
// dgamma and dbeta, added in LDS.  Where the columns alone make enough blocks there is one group, and no sums are left to join
// (32 rows of 196608 with tangence 24.8 us; 28.8 with four groups of rows that each wrote their sums for a third launch).
constexpr uint32_t GROUP_ROWS = 256;  // rows of a group, at most
template <int ACCESS, bool FUNC, class Rows>
__global__ __launch_bounds__(THREADS) void ln_backward_columns_kernel(Backward a, Rows rows, const float2 *sums, uint32_t pieces, uint32_t groups, uint32_t per_group,
                                                                     float *partial) {
  constexpr bool VEC = ACCESS != ONE;
  constexpr uint32_t W = VEC ? 4 : 1, SLICES = THREADS / 64, AT_ONCE = 4;
  __shared__ float4 terms[GROUP_ROWS];  // of each row: mean, ivar, sum(u) / N, sum(u * xhat) / N
  __shared__ float shares[2][SLICES][W][64];
  const uint32_t lane = threadIdx.x % 64, slice = threadIdx.x / 64;
  const uint32_t group = blockIdx.x % groups, column = (blockIdx.x / groups * 64 + lane) * W;
  const int at = load_at<ACCESS>(column, a.N), input_at = Rows::template at<ACCESS>(column, a.N);
  const uint32_t first = group * per_group, count = min(per_group, a.rows - first);
  // four rows at a time, the next four loaded before the first of them is stored (the error may be written over delta: each row of a
  // column is read and written by one thread)
  typename Rows::template Raw<VEC> raw[AT_ONCE], raw_n[AT_ONCE];
  float g[AT_ONCE][W], g_n[AT_ONCE][W];
  const auto load = [&](uint32_t k0, typename Rows::template Raw<VEC> *r, float (*d)[W]) {
#pragma unroll
    for (uint32_t u = 0; u < AT_ONCE; u++) {
      const uint32_t row = first + min(k0 + u * SLICES, count - 1);
      load_step<ACCESS>(d[u], a.delta + (size_t)row * a.N, at);
      rows.row(row).template load<ACCESS>(r[u], input_at);
    }
  };
  load(slice, raw, g);
  float gamma[W], beta[W], dg[W] = {}, db[W] = {};
  load_step<kept(ACCESS)>(gamma, a.gamma, at);
  settle<ACCESS>(gamma, column, a.N);
  if (FUNC) {
    load_step<kept(ACCESS)>(beta, a.beta, at);
    settle<ACCESS>(beta, column, a.N);
  }
  // eight lanes per row, eight loads each under way
  for (uint32_t k = threadIdx.x / 8; k < count; k += THREADS / 8) {
    const float2 *p = sums + (size_t)(first + k) * pieces;
    float s1 = 0.f, s2 = 0.f;
    for (uint32_t i = threadIdx.x % 8; i < pieces; i += 64) {
      float2 t[8];
#pragma unroll
      for (uint32_t u = 0; u < 8; u++) t[u] = p[min(i + 8 * u, pieces - 1)];
#pragma unroll
      for (uint32_t u = 0; u < 8; u++) {
        s1 += i + 8 * u < pieces ? t[u].x : 0.f;
        s2 += i + 8 * u < pieces ? t[u].y : 0.f;
      }
    }
    s1 = mt::over_lanes<mt::Sum, 8>(s1) / (float)a.N;
    s2 = mt::over_lanes<mt::Sum, 8>(s2) / (float)a.N;
    if (threadIdx.x % 8 == 0) terms[k] = make_float4(a.mean[first + k], a.ivar[first + k], s1, s2);
  }
  __syncthreads();
  for (uint32_t k0 = slice; k0 < count; k0 += AT_ONCE * SLICES) {
    if (k0 + AT_ONCE * SLICES < count) load(k0 + AT_ONCE * SLICES, raw_n, g_n);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t u = 0; u < AT_ONCE; u++) {
      const uint32_t k = k0 + u * SLICES;
      if (k >= count) break;
      const float4 c = terms[k];
      float x[W], t[W];
      raw[u].values(x);
      Rows::template settle_values<ACCESS>(x, column, a.N);
      settle<ACCESS>(g[u], column, a.N);
#pragma unroll
      for (uint32_t e = 0; e < W; e++) x[e] = (x[e] - c.x) * c.y;
      if constexpr (FUNC) fronts<W>(a.func, g[u], gamma, x, beta);
#pragma unroll
      for (uint32_t e = 0; e < W; e++) {
        dg[e] += g[u][e] * x[e];
        db[e] += g[u][e];
        t[e] = c.y * ((g[u][e] * gamma[e] - c.z) - x[e] * c.w);
      }
      if (column < a.N) store_step<ACCESS>(a.error + (size_t)(first + k) * a.N + column, t, a.N - column);
    }
#pragma unroll
    for (uint32_t u = 0; u < AT_ONCE; u++) {
      raw[u] = raw_n[u];
#pragma unroll
      for (uint32_t e = 0; e < W; e++) g[u][e] = g_n[u][e];
    }
  }
#pragma unroll
  for (uint32_t e = 0; e < W; e++) {
    shares[0][slice][e][lane] = dg[e];
    shares[1][slice][e][lane] = db[e];
  }
  __syncthreads();
  if (slice > 1 || column >= a.N) return;
  float *out = slice == 0 ? a.dgamma : a.dbeta;
  if (out == nullptr) return;
  if (groups > 1) out = partial + ((size_t)slice * groups + group) * a.N;
#pragma unroll
  for (uint32_t e = 0; e < W; e++) {
    float s = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < SLICES; k++) s += shares[slice][k][e][lane];
    if (ACCESS != FOUR_ANY || column + e < a.N) out[column + e] = a.accumulate && groups == 1 ? out[column + e] + s : s;
  }
}

// The derivative of what the forward pass computes for GeLU, v * s(v) with s(v) = 1 / (1 + exp(-2 u)) and u = sqrt(2 / pi) * (v + 0.044715 * v^3):
//   s + 2 * v * s * (1 - s) * u'
// with e = exp(-2 |u|), s * (1 - s) = e / (1 + e)^2: no difference of neighbouring numbers.  (Not MT_F_DIFFERENTIAL + MT_F_GELU: that is the
// function layer's formula, as the reference's layer trains with it, and up to three quarters away from the slope.)
__device__ __forceinline__ float gelu_slope(float v) {
  const float a = sqrtf(2.f / 3.141592654f), u = a * (v + 0.044715f * (v * v * v)), size = fabsf(u);
  const float e = expf(-2.f * size), r = mt::reciprocal(1.f + e), s = u < 0.f ? e * r : r;
  // (beyond 40 the product is below 1e-30, but an infinite cube would make it a NaN; a NaN stays one in s)
  return size < 40.f ? s + 2.f * v * (e * r * r) * (a * (1.f + 0.134145f * (v * v))) : s;
}

// error = delta * f'(gamma * xhat + beta) alone, for GeLU, whose exponential and polynomial the kernels above do not hold; the backward
// pass then starts from it
template <class Rows>
__global__ __launch_bounds__(THREADS) void ln_front_kernel(Backward a, Rows rows) {
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.mean[row], ivar = a.ivar[row];
    const auto in = rows.row(row);
    for (uint32_t i = blockIdx.y * THREADS + threadIdx.x; i < a.N; i += gridDim.y * THREADS) {
      typename Rows::template Raw<false> raw;
      float x;
      in.template load<ONE>(raw, i);
      raw.values(&x);
      const size_t e = (size_t)row * a.N + i;
      a.error[e] = a.delta[e] * gelu_slope(a.gamma[i] * ((x - mean) * ivar) + a.beta[i]);
    }
  }
}

mt::Workspace g_ln_ws;
int ln_workspace(size_t floats, float **p) { return mt::workspace_get(g_ln_ws, "layer-norm sums", floats, p); }

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

// ---- sizes ---------------------------------------------------------------------------------------------------------
struct Geometry {
  uint32_t rows, N, per_sample;  // rows, values per row, rows per sample
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
  if (__builtin_mul_overflow(zy, (uint64_t)gamma->x, &N) || N > 0x7fffffefull || per > 0x7fffffffull || __builtin_mul_overflow(per, (uint64_t)in->w, &rows) || rows > 0x7fffffffull)
    return mt::fail(MT_E_UNAVAILABLE, "%s: 2^31 rows, or rows of 2^31 values, are not supported", name);
  g->rows = (uint32_t)rows;
  g->N = (uint32_t)N;
  g->per_sample = (uint32_t)per;
  return MT_OK;
}
bool same_sizes(const mt_tensor *a, const mt_tensor *b) { return mt::same_zyx(a, b) && a->w == b->w; }
// does a result share no memory with the tensors; null: not there
bool apart(const mt_tensor *result, std::initializer_list<const mt_tensor *> tensors) {
  for (auto t : tensors)
    if (result && t && mt::overlap(result, t)) return false;
  return true;
}
bool is_statistic(const mt_tensor *t, const mt_tensor *in, const Geometry &g) { return t->w == in->w && t->z == g.kept_z && t->y == g.kept_y && t->x == 1; }

// rows of up to this many values are held in registers.  In the backward pass 1024 threads have room for 16 values each and their share
// of two sums, but not for a function's parameters too (2000 x 16384 with tangence 134 us against 114 in pieces).  In fours from any address
// they have it from fp32 input and pay for it with many rows (2000 x 16383 110 against 136, but 600 x 10319 34 against 27; from 8 bits
// 1344 x 10319 62 against 48)
constexpr uint32_t FORWARD_ROW = 32768, BACKWARD_ROW = 16384, BACKWARD_ROW_TIGHT = 8192;

// Tensors of long rows that the 256 MB of cache cannot hold are normalised so many bytes at a time, so that the second look at x finds
// them there (4000 x 40000 334 -> 285 us; 298 in parts of 48 MiB, and smaller tensors only pay for the launches)
constexpr uint64_t CACHE = 256ull << 20, FORWARD_AT_ONCE = 160ull << 20;
// blocks of one launch, at most: a grid has fewer than 2^32 threads
constexpr uint32_t MOST_BLOCKS = 1u << 21;

// calls f with how a kernel accesses the tensors
template <class F>
void with_access(int access, F &&f) {
  if (access == FOUR_PAST)
    f(std::integral_constant<int, FOUR_PAST>{});
  else if (access == FOUR)
    f(std::integral_constant<int, FOUR>{});
  else if (access == FOUR_ANY)
    f(std::integral_constant<int, FOUR_ANY>{});
  else
    f(std::integral_constant<int, ONE>{});
}
// Four values per access where rows are a multiple of four from 16-byte boundaries (`whole`), and from any address in rows of more than a
// wavefront (1344 x 10319 backward 73 -> 59 us, 2000 x 16383 152 -> 111, 4000 x 4001 forward with 8 bits 47 -> 34).  Shorter rows have
// more ends to take apart than accesses to save (30000 x 333 forward 14.2 us singly, 17.4 in fours)
constexpr uint32_t ANY_ROW = 1024;
int access_of(bool whole, uint32_t N, uint64_t bytes) { return whole ? mt::past_caches(bytes) ? FOUR_PAST : FOUR : N > ANY_ROW ? FOUR_ANY : ONE; }

template <int L, int E>
void forward_rows(Forward a, int access, bool pack) {
  constexpr uint32_t PER_BLOCK = L < 256 ? 256 / L : 1, BLOCK = L < 256 ? 256 : L;
  for (;;) {
    const uint32_t left = a.rows - a.first_row, grid = cdiv(left, PER_BLOCK) < MOST_BLOCKS ? cdiv(left, PER_BLOCK) : MOST_BLOCKS;
    const auto go = [&](auto acc) {
      constexpr int ACCESS = decltype(acc)::value;
      if constexpr (L >= 64 && ACCESS != ONE) {  // (a group of 128 by 32 lanes)
        if (pack) {
          ln_forward_kernel<L, E, ACCESS, true><<<grid, BLOCK, 0, mt::stream()>>>(a);
          return;
        }
      }
      if constexpr (ACCESS != FOUR_ANY || L * E > (int)ANY_ROW) ln_forward_kernel<L, E, ACCESS, false><<<grid, BLOCK, 0, mt::stream()>>>(a);
    };
    with_access(access, go);
    if (left <= grid * PER_BLOCK) return;
    a.first_row += grid * PER_BLOCK;
  }
}

// calls f with the threads per row and the values per thread that hold a row of N values
template <class F>
int with_share(uint32_t N, F &&f) {
  using std::integral_constant;
#define MT_LN_SHARE(L, E) \
  if (N <= L * E) return f(integral_constant<int, L>{}, integral_constant<int, E>{})
  MT_LN_SHARE(8, 4);
  MT_LN_SHARE(16, 8);
  MT_LN_SHARE(64, 4);
  MT_LN_SHARE(64, 8);
  MT_LN_SHARE(64, 16);
  MT_LN_SHARE(256, 8);
  MT_LN_SHARE(256, 16);
  MT_LN_SHARE(512, 16);
  MT_LN_SHARE(1024, 16);
#undef MT_LN_SHARE
  return f(integral_constant<int, 1024>{}, integral_constant<int, 32>{});
}

// calls f with that and whether a function stands behind the norm
template <class F>
void with_kind(int access, bool func, F &&f) {
  with_access(access, [&](auto acc) {
    if (func) f(acc, std::true_type{}); else f(acc, std::false_type{});
  });
}

template <class Rows>
int backward(const char *name, const mt_tensor *error, const mt_tensor *dgamma, const mt_tensor *dbeta, const mt_tensor *delta, const mt_tensor *gamma,
             const mt_tensor *beta, const Rows &x, bool x_aligned, const mt_tensor *mean, const mt_tensor *ivar, int func, int accumulate, const Geometry &g) {
  mt::ProfileScope prof(name);
  Backward a{};
  a.error = error->p; a.dgamma = dgamma ? dgamma->p : nullptr; a.dbeta = dbeta ? dbeta->p : nullptr;
  a.delta = delta->p; a.gamma = gamma->p; a.beta = beta ? beta->p : nullptr; a.mean = mean->p; a.ivar = ivar->p;
  a.rows = g.rows; a.N = g.N; a.func = func; a.accumulate = accumulate != 0;
  const Backward given = a;
  if (func == MT_F_GELU) {
    a.delta = a.error;
    a.func = MT_F_NONE;
  }
  // the first launch, once nothing can be refused any more: it writes over the error, which may be delta
  const auto front = [&] {
    if (func == MT_F_GELU) ln_front_kernel<<<dim3(g.rows < 4096 ? g.rows : 4096, g.N < 65536 ? 1 : 16), THREADS, 0, mt::stream()>>>(given, x);
  };
  const bool params = dgamma || dbeta;
  const bool whole = g.N % 4 == 0 && x_aligned && aligned16(a.error) && aligned16(a.delta) && aligned16(a.gamma) && (a.func == MT_F_NONE || aligned16(a.beta));
  // (half of what the pass moves stands for the size of a tensor that is read and written: 4096 x 6144 62.6 -> 58.2 us)
  const int access = x.in_fours() ? access_of(whole, g.N, mt::count(delta) * (8 + Rows::BYTES) / 2) : ONE;
  const bool vec = access != ONE;
  // few rows: the parameter gradients beside the error instead of partial sums and their join
  const bool few = g.rows <= 512;
  uint32_t parts = 0;
  float *partial = nullptr;
  const bool beside = !params || few;  // no sums over rows in the error's threads
  const bool held = a.func == MT_F_NONE && (whole || (access == FOUR_ANY && Rows::BYTES == 4 && g.rows >= 1024));
  if (g.N <= (beside || held ? BACKWARD_ROW : BACKWARD_ROW_TIGHT)) {
    int rc = with_share(g.N, [&](auto l, auto e) {
      constexpr int L = l, E = e;
      if constexpr (L * E <= (int)BACKWARD_ROW) {
        const uint32_t per_block = L < 256 ? 256 / L : 1, threads = L < 256 ? 256 : L;
        if (beside) {
          front();
          const uint32_t error_blocks = cdiv(g.rows, per_block), param_blocks = params ? cdiv(g.N, threads / 16) : 0;
          const auto go = [&](uint32_t first_row, uint32_t grid, uint32_t first_param_block) {
            with_kind(access, a.func != MT_F_NONE, [&](auto v, auto f) {
              constexpr int ACCESS = decltype(v)::value;
              if constexpr (ACCESS != FOUR_ANY || L * E > (int)ANY_ROW)
                ln_backward_few_kernel<L, E, ACCESS, decltype(f)::value, Rows><<<grid, threads, 0, mt::stream()>>>(a, x, first_row, first_param_block);
            });
          };
          if (params && a.error != a.delta) {
            go(0, error_blocks + param_blocks, error_blocks);
          } else {
            if (params) go(0, param_blocks, 0);  // written in place: the sums before the error
            for (uint32_t b = 0; b < error_blocks; b += MOST_BLOCKS) {
              const uint32_t grid = error_blocks - b < MOST_BLOCKS ? error_blocks - b : MOST_BLOCKS;
              go(b * per_block, grid, grid);
            }
          }
          return (int)MT_OK;
        }
        const int block = backward_block(L, E, access);
        parts = cdiv(g.rows, block / L);
        // one block per compute unit: its next row is on the way while it sums, and more blocks mean more partial sums (4096 x 6144: 60.0 us
        // with 256, 66.1 with 512, 74.7 with 1024; 1024 x 8192: 23.0, 30.6, 41.7)
        if (parts > 256) parts = 256;
        int rc = ln_workspace(2 * (size_t)parts * g.N, &partial);
        if (rc) return rc;
        front();
        with_kind(access, a.func != MT_F_NONE, [&](auto v, auto f) {
          constexpr int ACCESS = decltype(v)::value;
          constexpr bool FUNC = decltype(f)::value;
          constexpr bool fits = L * E <= (int)BACKWARD_ROW_TIGHT || (!FUNC && (ACCESS == FOUR || ACCESS == FOUR_PAST || (ACCESS == FOUR_ANY && Rows::BYTES == 4)));
          if constexpr (fits && (ACCESS != FOUR_ANY || L * E > (int)ANY_ROW)) ln_backward_kernel<L, E, ACCESS, FUNC, Rows><<<parts, block, 0, mt::stream()>>>(a, x, partial);
        });
      }
      return (int)MT_OK;
    });
    if (rc) return rc;
    MT_LAUNCH_CHECK(name);
  } else {
    const uint32_t pieces = cdiv(g.N, PIECE), strips = cdiv(g.N, 64 * (vec ? 4 : 1));
    // enough blocks to keep the memory busy, but groups of at least 16 rows: every group writes and joins 16 bytes per column where a
    // row moves 20
    const uint32_t blocks = vec ? 768 : 2048;  // that the compute units hold at once
    uint32_t groups = strips < blocks / 2 ? blocks / strips : 1;
    if (groups > cdiv(g.rows, 16)) groups = cdiv(g.rows, 16);
    uint32_t per_group = cdiv(g.rows, groups);
    if (per_group > GROUP_ROWS) per_group = GROUP_ROWS;
    groups = cdiv(g.rows, per_group);
    if ((uint64_t)g.rows * pieces >= (1u << 24) || (uint64_t)groups * strips >= (1u << 24)) return mt::fail(MT_E_UNAVAILABLE, "%s: too many elements for one launch", name);
    const size_t sums = 2 * (size_t)g.rows * pieces;
    float *ws = nullptr;
    int rc = ln_workspace(sums + (params && groups > 1 ? 2 * (size_t)groups * g.N : 0), &ws);
    if (rc) return rc;
    float2 *piece_sums = reinterpret_cast<float2 *>(ws);
    partial = ws + sums;
    parts = groups > 1 ? groups : 0;
    front();
    with_kind(access, a.func != MT_F_NONE, [&](auto v, auto f) {
      constexpr int ACCESS = decltype(v)::value;
      constexpr bool FUNC = decltype(f)::value;
      ln_backward_pieces_kernel<kept(ACCESS), FUNC><<<g.rows * pieces, THREADS, 0, mt::stream()>>>(a, x, piece_sums, pieces);
      ln_backward_columns_kernel<ACCESS, FUNC><<<groups * strips, THREADS, 0, mt::stream()>>>(a, x, piece_sums, pieces, groups, per_group, partial);
    });
    MT_LAUNCH_CHECK(name);
  }
  if (params && parts) {
    if (parts > 16)
      ln_join_kernel<JOIN_MANY><<<dim3(cdiv(g.N, JOIN_COLUMNS), 2), JOIN_COLUMNS * JOIN_MANY, 0, mt::stream()>>>(a.dgamma, a.dbeta, partial, parts, g.N, a.accumulate);
    else
      ln_join_kernel<1><<<dim3(cdiv(g.N, THREADS), 2), THREADS, 0, mt::stream()>>>(a.dgamma, a.dbeta, partial, parts, g.N, a.accumulate);
    MT_LAUNCH_CHECK(name);
  }
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
  const mt_tensor *read = *func != MT_F_NONE ? beta : nullptr;
  if (!apart(error, {gamma, read, mean, ivar}) || !apart(dgamma, {gamma, read, mean, ivar, delta, error}) || !apart(dbeta, {gamma, read, mean, ivar, delta, error, dgamma}))
    return mt::fail(MT_E_ARGUMENT, "%s: a result shares memory with another tensor", name);
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
  if (!apart(out, {gamma, beta}) || !apart(mean, {gamma, beta, in, out}) || !apart(ivar, {gamma, beta, in, out, mean}))
    return mt::fail(MT_E_ARGUMENT, "%s: a result shares memory with another tensor", name);
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
  Forward a{};
  a.out = out->p; a.in = in->p; a.gamma = gamma->p; a.beta = beta->p; a.mean = mean ? mean->p : nullptr; a.ivar = ivar ? ivar->p : nullptr;
  a.packed = packed; a.rows = g.rows; a.N = g.N; a.per_sample = g.per_sample; a.eps = epsilon;
  a.func = func == MT_F_GELU ? MT_F_NONE : func;  // GeLU (double arithmetic, a library function) runs over the output afterwards
  const bool whole = g.N % 4 == 0 && aligned16(a.out) && aligned16(a.in) && aligned16(a.gamma) && aligned16(a.beta);
  // the same pass can leave the 8 bits where a row starts at a group's first value and 32 lanes hold a group; it takes fours from any address
  // then (12000 x 1001 33 us in two passes, 29 in one; 33 x 1001 7.2 and 4.6)
  const bool pack = packed_input && g.N > 128 && (g.N % mt::PACK_GROUP == 0 || g.per_sample == 1);
  int access = access_of(whole, g.N, mt::count(in) * 4);
  if (pack && access == ONE) access = FOUR_ANY;
  if (packed_input && !pack && (rc = mt_pack(packed_input, in))) return rc;
  if (packed_input) mt::note_write(packed.q, mt::packed_bytes(packed));
  {
    mt::ProfileScope prof(name);
    if (g.N <= FORWARD_ROW) {
      rc = with_share(g.N, [&](auto l, auto e) {
        forward_rows<decltype(l)::value, decltype(e)::value>(a, access, pack);
        return (int)MT_OK;
      });
      MT_LAUNCH_CHECK(name);
    } else {
      const uint32_t pieces = cdiv(g.N, PIECE);
      const uint64_t row_bytes = (uint64_t)g.N * 4;
      const uint32_t at_once = g.rows * row_bytes <= CACHE ? g.rows : row_bytes >= FORWARD_AT_ONCE ? 1 : (uint32_t)(FORWARD_AT_ONCE / row_bytes);
      float *ws = nullptr;
      if ((rc = ln_workspace(2 * (size_t)at_once * pieces, &ws))) return rc;
      float2 *stats = reinterpret_cast<float2 *>(ws);
      for (; a.first_row < g.rows; a.first_row += at_once) {
        const unsigned grid = (g.rows - a.first_row < at_once ? g.rows - a.first_row : at_once) * pieces;
        with_access(access == FOUR_PAST ? FOUR : access, [&](auto acc) {
          constexpr int ACCESS = kept(decltype(acc)::value);
          if (pack)
            ln_pieces_kernel<ACCESS, true><<<grid, THREADS, 0, mt::stream()>>>(a, stats, pieces);
          else
            ln_pieces_kernel<ACCESS, false><<<grid, THREADS, 0, mt::stream()>>>(a, stats, pieces);
        });
        MT_LAUNCH_CHECK(name);
        with_access(access, [&](auto acc) { ln_apply_kernel<decltype(acc)::value><<<grid, THREADS, 0, mt::stream()>>>(a, stats, pieces); });
        MT_LAUNCH_CHECK(name);
      }
    }
  }
  return func == MT_F_GELU ? mt_apply_func(out, out, func) : MT_OK;
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
  return backward(name, error, dgamma, dbeta, delta, gamma, beta, RowsF32{input->p, g.N}, aligned16(input->p), mean, ivar, func, accumulate, g);
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
  return backward(name, error, dgamma, dbeta, delta, gamma, beta, RowsPacked{v, g.N, g.per_sample}, true, mean, ivar, func, accumulate, g);
}

}  // extern "C"
