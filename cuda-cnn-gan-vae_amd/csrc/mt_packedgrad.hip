// The linear layer's weight gradient from an input kept in 8 bits, on the 16-bit matrix cores with fp32 results.
//
//   dweight[o][i] = sum_b delta[b][o] * (low[b][g] + step[b][g] * q[b][i]),  g = the group of 128 columns that i is in
//                 = sum_b (delta * step)[b][o] * (q - zero)[b][i]  +  sum_b delta[b][o] * (low + zero * step)[b][g]
//
// zero = -low / step rounded to 0 ... 255: the count of steps that stands for 0, or for the value of the group's range that is nearest to it.
// So both sums are of the size of the values themselves, and a value of 0 adds nothing where low is 0 (what a ReLU leaves): a feature that
// is 0 in every sample has a gradient of exactly 0.  (The middle of the range, 128, left it the rounding of two large sums, 3e-7 beside
// gradients of 1; no centre at all costs activations of both signs four to nine times the error.  Relative error of all weights at 512
// samples, this / 128 / none / a plain fp32 product: of normal activations 1.1e-7, 1.8e-7, 1e-6, 3e-7; behind a ReLU 1.1e-7, 6e-7, 1.1e-7, 2e-7.  The counts in front of the subtraction cost
// 2 % of the largest products' time.)
// q - zero is a whole number between -255 and 255: exact in 16 bits.  delta * step, one fp32 product, is written as a sum of 16-bit numbers,
// whose products with q - zero the matrix cores add up in fp32, in one of two ways.
//   Three bf16 numbers: its upper 8 significant bits, the next 8, the last 8 (cutting instead of rounding makes every remainder
//   exact; products below 2^-110 lose the bits that no normal bf16 number holds).
//   Two fp16 numbers, rounded: the first (11 significant bits) off by at most 2^-11 of the product, the second by 2^-12 of what is left:
//   2^-23 of the product at most, twice the rounding of an fp32 product (root mean square over all mantissas 3.7e-8, of fp32 2.4e-8).  That is
//   a bit less than the three numbers hold, for two thirds of the matrix instructions; sums of thousands of such products carry fp32
//   roundings of that size anyway.  fp16 has little range: powers of two per row of dweight (of the largest delta) and per group (of the largest step)
//   bring all products below 2^15, and small ones are off by 2^-25 (fp16 keeps its subnormal numbers here, in the matrix instruction
//   too): nothing beside the rounding of the row's largest as long as that is not small itself.  The block checks that, and starts
//   again with three numbers where it is not so.  The powers need a look at all of delta before (a launch that reads it once and sums
//   the columns for dbias on the way), so this is for products that are worth it.
// Three (two) 16-bit matrix instructions multiply what one fp32 product would, at a third (half) of a rate where the library's bf16
// product reaches 1295 TFLOP/s; the fp32 matrix instructions reach 157 at most.  4096^3: 310 to 326 us in two numbers, 363 to 372 in three; a block
// that starts again takes both (651 us where all do).  The clock falls with the load: 603000 cycles per launch are 300 us at 2.0 GHz in
// launches apart, 356 in twenty without a pause; the matrix cores work in 43 % of the cycles, the vector units in 47 %.  The second sum is one fp32 multiply-add per element of
// delta on the way.
//
// A column tile is one group, so that a sample has one (low, step) in it.  A block is four wavefronts, each with its own 32 or
// 64 rows (output features) and all 128 columns: no other wavefront needs its rows, so delta goes from memory to registers in
// the lane layout of the matrix instruction and is scaled and cut there, never through LDS.  The columns, which all four
// need, are turned into 16-bit numbers once and shared through LDS, eight samples of one column per 16 bytes: that is what a lane
// reads.  The block takes 64 samples per step; the next step's columns are loaded before and written after the step's
// products, the next 16 samples of delta are loaded before the products of the 16 in hand.
#include "mt_packed.h"

namespace {

using mt::cdiv;
using mt::PackedView;
using mt::xcd_swizzle;

constexpr int THREADS = 256;    // of one group of four wavefronts
constexpr uint32_t KSTEP = 64;  // samples per step

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4_of_any __attribute__((ext_vector_type(4), may_alias));

// the next rows of an operand, at most `most` of the `left` that there are (none: left <= 0): what lies behind them reads as
// zero.  most * row_bytes <= 2^30: 16 rows of delta or dweight, 64 of the packed bytes, fewer than 2^24 features.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void *p, int left, int most, uint32_t row_bytes) {
  const uint32_t rows = __builtin_amdgcn_readfirstlane(max(0, min(left, most)));  // (a clamp is a vector instruction: back to a scalar)
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (int)(rows * row_bytes), 0x00020000);
}

__device__ __forceinline__ uint32_t upper_halves(float a, float b) {  // the bf16 numbers of a (low half) and b, cut off
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ uint32_t halves_of(float a, float b) {  // a (low half) and b rounded to fp16
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2{a, b}), halfx2));
}
// The power of two of a largest magnitude, between 2^-126 and 2^126; 0 for an infinity, whose row is lost anyway
__device__ __forceinline__ int exponent_of(float most) {
  const int e = (int)(__float_as_uint(most) >> 23) - 127;
  return e == 128 ? 0 : max(-126, min(e, 126));
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // e from -126 to 127
__device__ __forceinline__ float cut(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }

struct WgradArgs {
  const float *delta;
  PackedView in;
  float *dweight, *dbias;    // split == 1: the gradients; else [split][Out*In] and [split][Out] partial sums
  uint32_t Out, tiles_m, split, per_split;  // per_split: samples of one part, a multiple of KSTEP
  bool accumulate;
  // of a look at delta before (HALVES), over each part of the samples: [parts][Out + groups] largest magnitudes of delta and of the steps,
  // [parts][Out] sums of delta
  const float *ranges, *column_sums;
  uint32_t parts;
  bool accumulate_bias;
};

template <int TM>
struct WgradSums {
  floatx16 acc[TM][4];           // matrix-core sums: 32 rows x 32 columns each
  float offset[TM], bias[TM];    // the second sum and the sum of delta: row lane % 32, half of the samples each
  uint32_t seen[TM];             // the bits of all first fp16 numbers of a row
};

// the product over the samples k0 ... k1 (`steps` steps; those behind k1 add nothing).  The sum of delta is taken by all blocks though only those of the first group need it:
// one addition in ten, where a second copy of the loop made those blocks the last ones (and the kernel's code twice as long).
// HALVES: in two fp16 numbers; `row` and `step_scale` are the powers of two that bring delta * step below 2^15
template <int TM, bool HALVES, bool BIAS>
__device__ __forceinline__ void packed_wgrad_loop(const WgradArgs &a, uint32_t g, uint32_t m0, uint32_t k0, uint32_t k1, uint32_t steps, uintx4 (*cols)[KSTEP / 8][128],
                                                  float2 (*scale)[KSTEP], uint16_t (*zeros)[KSTEP], const float (&row)[TM], float step_scale, WgradSums<TM> &sums) {
  const uint32_t tid = threadIdx.x % THREADS, lane = tid & 63u, r = lane & 31u, half = lane >> 5;
  // this lane's rows r * TM ... of eight samples, AHEAD times 16 samples ahead of the products: 16 where two row tiles fill the
  // registers (two wavefronts per SIMD hide the rest), a whole step where there is room and often one wavefront
  constexpr int AHEAD = TM == 1 ? 4 : 1;
  float d[AHEAD][8][TM];
  uint32_t voff[8];
#pragma unroll
  for (int j = 0; j < 8; j++) voff[j] = ((half * 8u + j) * a.Out + m0 + r * TM) * 4u;

  auto load_delta = [&](uint32_t k, float (&d)[8][TM]) {
    const auto rsrc = rows_rsrc(a.delta + (size_t)k * a.Out, (int)k1 - (int)k, 16, a.Out * 4u);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if (TM == 2) {
        const uintx2 v = __builtin_amdgcn_raw_buffer_load_b64(rsrc, (int)voff[j], 0, 0);
        d[j][0] = __uint_as_float(v[0]);
        d[j][TM - 1] = __uint_as_float(v[1]);
      } else {
        d[j][0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc, (int)voff[j], 0, 0));
      }
    }
  };
  const uint32_t kg = tid / 32u, c4 = (tid & 31u) * 4u;  // this thread's eight samples and four columns of a step
  uint32_t q[8];
  uintx2 pair;
  auto load_cols = [&](uint32_t k) {
    const auto rsrc = rows_rsrc(a.in.q + (size_t)k * a.in.pitch, (int)k1 - (int)k, KSTEP, a.in.pitch);
#pragma unroll
    for (int j = 0; j < 8; j++) q[j] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, (int)((kg * 8u + j) * a.in.pitch + g * 128u + c4), 0, 0);
    // (samples behind the end have a step and a lowest value of zero, whatever follows in memory)
    pair = __builtin_amdgcn_raw_buffer_load_b64(rows_rsrc(a.in.pair + (size_t)k * a.in.groups, (int)k1 - (int)k, KSTEP, a.in.groups * 8u),
                                                (int)((tid % KSTEP) * a.in.groups * 8u + g * 8u), 0, 0);
  };
  auto store_cols = [&](uint32_t buf) {
    // lane l of every wavefront has the pair of sample l of the step; what it makes of it goes to the lanes that have the sample's bytes, within the
    // wavefront, whose accesses to LDS are in order (a constant group counts as 0: its step is 0)
    const float low = __uint_as_float(pair.x), step = __uint_as_float(pair.y);
    const float zero = fminf(fmaxf(rintf(-low * (step > 0.f ? mt::reciprocal(step) : 0.f)), 0.f), 255.f);
    zeros[tid / 64u][lane] = (uint16_t)zero;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (no instruction: the compiler must not take the load for one of other memory)
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const uintx4 z = *reinterpret_cast<const uintx4_of_any *>(&zeros[tid / 64u][kg * 8u]);
#pragma unroll
    for (int c = 0; c < 4; c++) {
      uintx4 w;
      if constexpr (HALVES) {
        // whole numbers under the exponent of 1024 are 1024 + q and 1024 + zero: their difference is exact
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t t = __builtin_amdgcn_perm(q[2 * j + 1], q[2 * j], 0x0c040c00u + 0x00010001u * c) | 0x64006400u;
          w[j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(halfx2, t) - __builtin_bit_cast(halfx2, z[j] | 0x64006400u));
        }
      } else {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = (float)((q[j] >> (8 * c)) & 255u) - (float)((z[j / 2] >> (16 * (j % 2))) & 0xffffu);
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = upper_halves(v[2 * j], v[2 * j + 1]);
      }
      cols[buf][kg][c4 + c] = w;
    }
    if (tid < KSTEP) scale[buf][tid] = make_float2(step * step_scale, __builtin_fmaf(zero, step, low));
  };

  load_cols(k0);
#pragma unroll
  for (int u = 0; u < AHEAD; u++) load_delta(k0 + 16u * u, d[u]);
  store_cols(0);
  __syncthreads();
  for (uint32_t s = 0; s < steps; s++) {
    const uint32_t buf = s & 1u, k = k0 + s * KSTEP;
    load_cols(k + KSTEP);
    float offset[TM] = {}, bias[TM] = {};  // of this step: sums of sums keep their error at the root of 32 and of the steps
#pragma unroll
    for (int kk = 0; kk < 4; kk++) {
      uintx4 col[4];
#pragma unroll
      for (int n = 0; n < 4; n++) col[n] = cols[buf][kk * 2 + half][n * 32 + r];
#pragma unroll
      for (int m = 0; m < TM; m++) {
        constexpr int CUTS = HALVES ? 2 : 3;
        uintx4 cuts[CUTS];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          float x[2], y[2], z[2];
          halfx2 h, l;
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float v = d[kk % AHEAD][2 * j + e][m];
            const float2 sc = scale[buf][kk * 16 + half * 8u + 2 * j + e];
            if constexpr (BIAS) bias[m] += v;
            offset[m] = __builtin_fmaf(v, sc.y, offset[m]);
            if constexpr (HALVES) {
              // (a fused product and sum of fp32 and fp16 numbers, rounded to fp16, is one instruction)
              x[e] = v * row[m];
              y[e] = sc.x;
            } else {
              x[e] = v * sc.x;
              y[e] = x[e] - cut(x[e]);
              z[e] = y[e] - cut(y[e]);
            }
          }
          if constexpr (HALVES) {
#pragma unroll
            for (int e = 0; e < 2; e++) h[e] = (_Float16)__builtin_fmaf(x[e], y[e], 0.f);
            uint32_t first = __builtin_bit_cast(uint32_t, h);
            asm volatile("" : "+v"(first));  // (the compiler would compute the second number again, into a low half)
            h = __builtin_bit_cast(halfx2, first);
            cuts[0][j] = first;
            sums.seen[m] |= first;
#pragma unroll
            for (int e = 0; e < 2; e++) l[e] = (_Float16)__builtin_fmaf(x[e], y[e], -(float)h[e]);
            cuts[1][j] = __builtin_bit_cast(uint32_t, l);
          } else {
            cuts[0][j] = upper_halves(x[0], x[1]);
            cuts[1][j] = upper_halves(y[0], y[1]);
            cuts[CUTS - 1][j] = upper_halves(z[0], z[1]);
          }
        }
        // (the compiler would leave these sums for the end of the step and keep four times the registers of delta for them)
        asm volatile("" : "+v"(offset[m]));
        if constexpr (BIAS) asm volatile("" : "+v"(bias[m]));
        if (m == TM - 1) load_delta(k + 16u * (kk + AHEAD), d[kk % AHEAD]);
#pragma unroll
        for (int p = 0; p < CUTS; p++)
#pragma unroll
          for (int n = 0; n < 4; n++) {
            if constexpr (HALVES)
              sums.acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, cuts[p]), __builtin_bit_cast(halfx8, col[n]), sums.acc[m][n], 0, 0, 0);
            else
              sums.acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, cuts[p]), __builtin_bit_cast(bf16x8, col[n]), sums.acc[m][n], 0, 0, 0);
          }
      }
      __builtin_amdgcn_sched_barrier(0);  // nothing of the next 16 samples moves up: the registers are full
    }
#pragma unroll
    for (int m = 0; m < TM; m++) {
      sums.offset[m] += offset[m];
      sums.bias[m] += bias[m];
    }
    store_cols(buf ^ 1u);
    __syncthreads();
  }
}

// Stores column tiles N0 ... N1 of a wavefront's sums
template <int TM, int N0, int N1, bool HALVES>
__device__ __forceinline__ void packed_wgrad_store(const WgradArgs &a, float *dw, uint32_t g, uint32_t m0, const float4 (*offsets)[8], const int4 (*powers)[8],
                                                   const WgradSums<TM> &sums) {
  const uint32_t lane = threadIdx.x & 63u, r = lane & 31u, half = lane >> 5;
  // accumulator i of tile (m, n): row 8 * (i / 4) + 4 * half + i % 4, column 32 * n + r.  Rows and columns that do not exist have
  // offsets behind the end of the buffer: their stores are dropped
  const uint32_t row_bytes = a.in.n * 4u;
  uint32_t voff[4];
#pragma unroll
  for (int n = N0; n < N1; n++) {
    const uint32_t c = g * 128u + n * 32u + r;
    voff[n] = c < a.in.n ? 4u * half * TM * row_bytes + c * 4u : 0x80000000u;
  }
#pragma unroll
  for (int i4 = 0; i4 < 4; i4++) {
    const uint32_t o0 = __builtin_amdgcn_readfirstlane(m0 + 8u * i4 * TM);
    const auto rsrc = rows_rsrc(dw + (size_t)o0 * a.in.n, (int)a.Out - (int)o0, 8 * TM, row_bytes);
#pragma unroll
    for (int m = 0; m < TM; m++) {
      const float4 c4 = offsets[m][i4 * 2 + half];
      const float c[4] = {c4.x, c4.y, c4.z, c4.w};
      const int4 p4 = HALVES ? powers[m][i4 * 2 + half] : int4{};
      const int power[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t row = (i * TM + m) * row_bytes;
        float v[4];
#pragma unroll
        for (int n = N0; n < N1; n++) v[n] = (HALVES ? __builtin_amdgcn_ldexpf(sums.acc[m][n][i4 * 4 + i], power[i]) : sums.acc[m][n][i4 * 4 + i]) + c[i];
        if (a.accumulate) {
#pragma unroll
          for (int n = N0; n < N1; n++) v[n] += __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc, (int)(voff[n] + row), 0, 0));
        }
#pragma unroll
        for (int n = N0; n < N1; n++) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[n]), rsrc, (int)(voff[n] + row), 0, 0);
      }
    }
  }
}

// KW groups of four wavefronts per block.  Two groups take half of the block's samples each, with their own columns in LDS, and add
// their sums at the end: where the tiles are few, the second wavefront per SIMD that fills the first one's waits comes from the
// same tile instead of from another part of the batch, whose sums would go through memory.
template <int TM, int KW, bool HALVES>
__global__ __launch_bounds__(THREADS * KW, 2 / KW) void packed_wgrad_kernel(WgradArgs a) {
  __shared__ uintx4 cols[KW][2][KSTEP / 8][128];  // [eight samples][column]
  __shared__ float2 scale[KW][2][KSTEP];          // (step, low + zero * step)
  __shared__ alignas(16) uint16_t zeros[KW][4][KSTEP];  // the samples' counts that stand for 0, of each wavefront
  __shared__ float4 offsets[4][TM][8];            // the second sum of every row of a wavefront
  __shared__ int4 powers[HALVES ? 4 : 1][TM][8];  // the power of two that its products lack
  __shared__ float halves[KW > 1 ? 2 : 1][4][TM][32];
  const uint32_t lane = threadIdx.x & 63u, r = lane & 31u, half = lane >> 5;
  const uint32_t kw = __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u % 4u);
  // neighbouring blocks of an XCD share their rows of delta (the larger operand) and walk over the groups
  uint32_t t = __builtin_amdgcn_readfirstlane(xcd_swizzle(blockIdx.x, gridDim.x));
  const uint32_t g = t % a.in.groups;
  t /= a.in.groups;
  const uint32_t m0 = (t % a.tiles_m) * (128u * TM) + wave * (32u * TM), part = t / a.tiles_m;
  const uint32_t k0 = part * a.per_split, k1 = min(a.in.w, k0 + a.per_split);
  const uint32_t steps = ((k1 - k0 + KSTEP - 1) / KSTEP + KW - 1) / KW;  // of each group
  const bool bias = a.dbias != nullptr && g == 0 && (!HALVES || part == 0);
  WgradSums<TM> sums;
  const auto clear = [&] {
#pragma unroll
    for (int m = 0; m < TM; m++) {
      sums.offset[m] = 0.f;
#pragma unroll
      for (int n = 0; n < 4; n++) sums.acc[m][n] = 0.f;
    }
  };
  clear();
#pragma unroll
  for (int m = 0; m < TM; m++) {
    sums.bias[m] = 0.f;
    sums.seen[m] = 0u;
  }
  const uint32_t first = min(k1, k0 + kw * steps * KSTEP), last = min(k1, first + steps * KSTEP);
  if constexpr (HALVES) {
    __shared__ uint32_t seen[KW][4][TM][32];
    float most[TM] = {}, most_step = 0.f;
    const uint32_t stride = a.Out + a.in.groups;
    uint32_t o[TM];
#pragma unroll
    for (int m = 0; m < TM; m++) o[m] = min(m0 + r * TM + m, a.Out - 1);
    for (uint32_t p0 = 0; p0 < a.parts; p0 += 8) {
#pragma unroll
      for (uint32_t u = 0; u < 8; u++) {
        const float *ranges = a.ranges + (size_t)min(p0 + u, a.parts - 1) * stride;
#pragma unroll
        for (int m = 0; m < TM; m++) most[m] = fmaxf(most[m], ranges[o[m]]);
        most_step = fmaxf(most_step, ranges[a.Out + g]);
      }
    }
    if (bias && kw == 0 && half == 0) {
      for (uint32_t p0 = 0; p0 < a.parts; p0 += 8) {
        float t[8][TM];
#pragma unroll
        for (uint32_t u = 0; u < 8; u++)
#pragma unroll
          for (int m = 0; m < TM; m++) t[u][m] = p0 + u < a.parts ? a.column_sums[(size_t)(p0 + u) * a.Out + o[m]] : 0.f;
#pragma unroll
        for (uint32_t u = 0; u < 8; u++)
#pragma unroll
          for (int m = 0; m < TM; m++) sums.bias[m] += t[u][m];
      }
    }
    const int step_power = min(127, 12 - exponent_of(most_step));
    float row[TM];
#pragma unroll
    for (int m = 0; m < TM; m++) {
      const int e = exponent_of(most[m]);
      row[m] = power_of_two(-e);
      if (kw == 0 && half == 0) reinterpret_cast<int *>(powers[wave][m])[r] = e - step_power;
    }
    packed_wgrad_loop<TM, true, false>(a, g, m0, first, last, steps, cols[kw], scale[kw], zeros[kw], row, power_of_two(step_power), sums);
    // Was every row's largest product near the product of the largest delta and the largest step?  A first number of 2 or more (the upper
    // exponent bit) says so: what a smaller one of its row lacks is at most 2^-26 of it.  If not (a sample of huge values that has no
    // delta, say), the block starts again with the three numbers that have fp32's range
#pragma unroll
    for (int m = 0; m < TM; m++) {
      sums.seen[m] |= __shfl_xor(sums.seen[m], 32, 64);
      seen[kw][wave][m][r] = sums.seen[m];
    }
    __syncthreads();
    bool good = true;
#pragma unroll
    for (int m = 0; m < TM; m++) {
      const bool large = ((seen[0][wave][m][r] | seen[KW - 1][wave][m][r]) & 0x40004000u) != 0u;
      good = good && (large || m0 + r * TM + m >= a.Out || most[m] == 0.f || most_step == 0.f);
    }
    if (!__syncthreads_and(good)) {
      clear();
#pragma unroll
      for (int m = 0; m < TM; m++) {
        row[m] = 1.f;
        if (kw == 0 && half == 0) reinterpret_cast<int *>(powers[wave][m])[r] = 0;
      }
      packed_wgrad_loop<TM, false, false>(a, g, m0, first, last, steps, cols[kw], scale[kw], zeros[kw], row, 1.f, sums);
    }
  } else {
    const float row[TM] = {};
    packed_wgrad_loop<TM, false, true>(a, g, m0, first, last, steps, cols[kw], scale[kw], zeros[kw], row, 1.f, sums);
  }

  float *dw = a.dweight, *db = a.dbias;
  if (a.split > 1) {
    dw += (size_t)part * a.Out * a.in.n;
    if (bias && !HALVES) db += (size_t)part * a.Out;
  }
  float c[TM], sum[TM];
#pragma unroll
  for (int m = 0; m < TM; m++) {
    c[m] = sums.offset[m] + __shfl_xor(sums.offset[m], 32, 64);
    sum[m] = sums.bias[m] + __shfl_xor(sums.bias[m], 32, 64);
    if (KW > 1 && kw == 1 && half == 0) {
      halves[0][wave][m][r] = c[m];
      halves[KW > 1 ? 1 : 0][wave][m][r] = sum[m];
    }
  }
  if (KW > 1) {
    // each group hands the other two of its four column tiles: 32 values per thread and row tile, through the columns' memory
    float *swap = reinterpret_cast<float *>(&cols[0][0][0][0]);
    const uint32_t tid = threadIdx.x % THREADS;
#pragma unroll
    for (int m = 0; m < TM; m++) {
      __syncthreads();  // the columns, or the values of the row tile before, are no longer read
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 16; i++) swap[(kw * 32u + n * 16u + i) * THREADS + tid] = kw == 0 ? sums.acc[m][n + 2][i] : sums.acc[m][n][i];
      __syncthreads();
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float other = swap[((kw ^ 1u) * 32u + n * 16u + i) * THREADS + tid];
          if (kw == 0)
            sums.acc[m][n][i] += other;
          else
            sums.acc[m][n + 2][i] = other + sums.acc[m][n + 2][i];
        }
    }
  }
  if (kw == 0 && half == 0) {
#pragma unroll
    for (int m = 0; m < TM; m++) {
      if (KW > 1) {
        c[m] += halves[0][wave][m][r];
        sum[m] += halves[KW > 1 ? 1 : 0][wave][m][r];
      }
      reinterpret_cast<float *>(offsets[wave][m])[r] = c[m];
      if (bias && m0 + r * TM + m < a.Out) {
        float *p = db + m0 + r * TM + m;
        *p = (HALVES ? a.accumulate_bias : a.accumulate) ? *p + sum[m] : sum[m];
      }
    }
  }
  __syncthreads();
  if constexpr (KW == 1) {
    packed_wgrad_store<TM, 0, 4, HALVES>(a, dw, g, m0, offsets[wave], powers[HALVES ? wave : 0], sums);
  } else if (kw == 0) {
    packed_wgrad_store<TM, 0, 2, HALVES>(a, dw, g, m0, offsets[wave], powers[HALVES ? wave : 0], sums);
  } else {
    packed_wgrad_store<TM, 2, 4, HALVES>(a, dw, g, m0, offsets[wave], powers[HALVES ? wave : 0], sums);
  }
}

// the largest magnitude (a NaN counts as none) of every column of delta, then of the steps of every group, over `per_part` samples, and
// the columns' sums
__global__ __launch_bounds__(THREADS) void packed_wgrad_ranges_kernel(float *ranges, float *sums, const float *delta, PackedView in, uint32_t Out, uint32_t per_part) {
  const uint32_t i = blockIdx.x * THREADS + threadIdx.x, k0 = blockIdx.y * per_part, count = min(per_part, in.w - k0);
  if (i >= Out + in.groups) return;
  const bool steps = i >= Out;
  const size_t stride = steps ? (size_t)in.groups * 2 : Out;
  const float *p = steps ? &in.pair[(size_t)k0 * in.groups + (i - Out)].y : delta + (size_t)k0 * Out + i;
  float most = 0.f, sum = 0.f;
  for (uint32_t k = 0; k < count; k += 16) {
    float t[16], s = 0.f;
#pragma unroll
    for (uint32_t u = 0; u < 16; u++) t[u] = p[(size_t)min(k + u, count - 1) * stride];
#pragma unroll
    for (uint32_t u = 0; u < 16; u++) {
      most = fmaxf(most, fabsf(t[u]));
      s += k + u < count ? t[u] : 0.f;
    }
    sum += s;
  }
  ranges[(size_t)blockIdx.y * (Out + in.groups) + i] = most;
  if (!steps) sums[(size_t)blockIdx.y * Out + i] = sum;
}

// the parts of a split sum, in a fixed order: first the weights' n values, then the bias's Out; SLICES threads per value, which take
// every SLICES-th part
template <int SLICES>
__global__ __launch_bounds__(THREADS) void packed_wgrad_join_kernel(float *dweight, float *dbias, const float *partial, const float *partial_bias, uint32_t split, size_t n,
                                                                   uint32_t Out, bool accumulate) {
  constexpr uint32_t VALUES = THREADS / SLICES;
  __shared__ float sums[SLICES][VALUES];
  const uint32_t c = threadIdx.x % VALUES, slice = threadIdx.x / VALUES;
  const size_t i = (size_t)blockIdx.x * VALUES + c;
  const bool weight = i < n, exists = weight || (dbias != nullptr && i - n < Out);
  const float *p = weight ? partial + i : partial_bias + (i - n);
  const size_t stride = weight ? n : Out;
  float s = 0.f;
  if (exists)
    for (uint32_t k = slice; k < split; k += 8 * SLICES) {
      float t[8];
#pragma unroll
      for (int u = 0; u < 8; u++) t[u] = k + u * SLICES < split ? p[(size_t)(k + u * SLICES) * stride] : 0.f;
      s += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
    }
  if (SLICES > 1) {
    sums[slice][c] = s;
    __syncthreads();
    if (slice != 0) return;
#pragma unroll
    for (int k = 1; k < SLICES; k++) s += sums[k][c];
  }
  if (!exists) return;
  float *out = weight ? dweight + i : dbias + (i - n);
  *out = accumulate ? *out + s : s;
}

// dbias alone, for a layer without input features
__global__ __launch_bounds__(THREADS) void bias_only_kernel(float *dbias, const float *delta, uint32_t w, uint32_t Out, bool accumulate) {
  const uint32_t o = blockIdx.x * THREADS + threadIdx.x;
  if (o >= Out) return;
  float s = 0.f;
  for (uint32_t b = 0; b < w; b++) s += delta[(size_t)b * Out + o];
  dbias[o] = accumulate ? dbias[o] + s : s;
}

mt::Workspace g_wgrad_ws;

// The variant: rows per block (256: each sample's columns are turned into 16-bit numbers for twice the products; 128: twice the blocks), one or
// two groups of wavefronts per block, parts of the batch.  The estimate of each variant's time in microseconds is its fixed part plus
// the steps that the busiest compute unit takes, at the measured time of a step with one or two blocks on it, plus writing and
// joining the parts' sums; two fp16 numbers instead of three bf16 ones take 0.82 of the steps' time and a look at delta before.  Measured
// against one another, in three numbers: 4096^3 372 us with 256 rows, 407 with 128; 2048^3 59 with 128 rows and two groups, 66 with one,
// 108 with 256 rows; 1777 samples, 1000 -> 1000 28.4 in four parts, 31.0 with two groups in two, 55 in one part; 512^3 11.4 in four parts, 18.4
// in one.  In two numbers against three: 4096^3 314 and 372, 1024 samples, 4096 -> 8192 171 and 196, 2048^3 55.9 and 58.6, 256 x 4096 x 4096
// 34.0 and 33.6, 512^3 18.7 and 15.7.
struct Plan {
  uint32_t rows, split;
  bool pair, half;
};
int g_linear_packed = 0;  // option "linear_packed": 0 choose, else variant 1 ... 5 and ten times the parts of the batch
constexpr uint32_t MOST_PARTS = 128;
Plan choose(uint32_t Out, uint32_t groups, uint32_t samples, size_t n) {
  const uint32_t steps = cdiv(samples, KSTEP);
  if (g_linear_packed != 0) {
    const int variant = g_linear_packed % 10;
    const bool wide = (variant == 3 || variant == 5) && Out % 2 == 0;
    const uint32_t parts = g_linear_packed / 10 ? g_linear_packed / 10 : 1;
    return Plan{wide ? 256u : 128u, n >= (1u << 29) ? 1 : parts < steps ? parts : steps, variant != 1 && !wide, variant >= 4};
  }
  const double look = 4.0 + (double)samples * Out * 4 / 5.6e6;  // what the launch before and its results cost
  Plan best{128, 1, false, false};
  double least = 1e30;
  for (int kind = 0; kind < 3; kind++) {
    const uint32_t rows = kind == 2 ? 256 : 128;
    const bool pair = kind == 1;
    if (rows == 256 && Out % 2 != 0) continue;  // rows are loaded in pairs there, which must not straddle the end
    const double fixed = kind == 0 ? 5.0 : kind == 1 ? 6.0 : 6.5, one = kind == 0 ? 1.75 : kind == 1 ? 3.0 : 2.8, two = kind == 0 ? 3.25 : kind == 1 ? 6.0 : 5.7;
    const size_t tiles = (size_t)cdiv(Out, rows) * groups;
    for (uint32_t split = 1; split <= MOST_PARTS && split <= steps; split += split < 4 ? 1 : split / 2) {
      if (split > 1 && n >= (1u << 29)) break;  // a join is one launch of fewer than 2^32 threads
      const size_t blocks = tiles * split;
      const size_t rest = blocks % 512;
      const double turn = blocks / 512 * two + (rest > 256 ? two : rest > 0 ? one : 0.0);
      const uint32_t each = cdiv(cdiv(steps, split), pair ? 2 : 1);
      const double rest_us = fixed + (split > 1 ? 4.0 + split * (double)n * 2e-6 : 0.0), loop_us = each * turn;
      const bool half = kind != 0 && 0.82 * loop_us + look < loop_us;  // (kind 0 is for few steps)
      const double us = rest_us + (half ? 0.82 * loop_us + look : loop_us);
      if (us < least) {
        least = us;
        best = Plan{rows, split, pair, half};
      }
    }
  }
  return best;
}

}  // namespace

namespace mt {
int set_linear_packed(int v) {
  const int variant = v % 10;
  if (v < 0 || (v != 0 && (variant < 1 || variant > 5)) || v / 10 > (int)MOST_PARTS)
    return fail(MT_E_ARGUMENT, "linear_packed must be 0 (choose) or a variant 1 to 5 plus ten times 0 to %u parts of the batch", MOST_PARTS);
  g_linear_packed = v;
  return MT_OK;
}
}  // namespace mt

extern "C" {

int mt_linear_backward_weights_sum_packed(const mt_tensor *dweight, const mt_tensor *dbias, const mt_packed_tensor *input, const mt_tensor *delta, int accumulate) {
  const char *name = "mt_linear_backward_weights_sum_packed";
  if (mt::bad(dweight) || (dbias && mt::bad(dbias)) || mt::bad(input) || mt::bad(delta))
    return mt::fail(MT_E_ARGUMENT, "%s: null tensor, or packed memory that is not 16-byte aligned", name);
  PackedView v;
  if (!mt::packed_view(input, &v)) return mt::fail(MT_E_UNAVAILABLE, "%s: a sample of 2^31 elements or more is not supported", name);
  const uint64_t out = (uint64_t)delta->z * delta->y * delta->x;  // the layer's output may be seen under any sizes of Out values
  if (dweight->w != 1 || dweight->z != 1 || dweight->x != v.n || dweight->y != out || delta->w != v.w)
    return mt::fail(MT_E_SHAPE, "%s: dweight must be [1,1,Out,In], the input [B,...] of In values, delta [B,...] of Out values", name);
  if (dbias && (dbias->w != 1 || dbias->z != 1 || dbias->x != 1 || dbias->y != out)) return mt::fail(MT_E_SHAPE, "%s: dbias must be [1,1,Out,1]", name);
  // the rows of a step are addressed with 32-bit offsets
  if (v.n >= (1u << 24) || out >= (1u << 24)) return mt::fail(MT_E_UNAVAILABLE, "%s: 2^24 features or more are not supported", name);
  if (v.w >= 0x7fff0000u) return mt::fail(MT_E_UNAVAILABLE, "%s: nearly 2^31 samples or more are not supported", name);
  const uint32_t Out = (uint32_t)out;
  if (Out == 0) return MT_OK;
  for (auto t : {dweight, dbias})
    if (t && (mt::overlap(t, delta) || mt::overlap(t, v))) return mt::fail(MT_E_ARGUMENT, "%s: a gradient shares memory with an input", name);
  if (dbias && mt::overlap(dbias, dweight)) return mt::fail(MT_E_ARGUMENT, "%s: dbias shares memory with dweight", name);
  if (v.w == 0) {  // an empty batch: the sums are zero
    if (accumulate) return MT_OK;
    int rc = mt_fill(dweight, 0.f);
    return rc || !dbias ? rc : mt_fill(dbias, 0.f);
  }
  mt::note_write(dweight);
  mt::note_write(dbias);
  mt::ProfileScope prof(name);
  if (v.n == 0) {
    if (dbias) bias_only_kernel<<<cdiv(Out, THREADS), THREADS, 0, mt::stream()>>>(dbias->p, delta->p, v.w, Out, accumulate != 0);
    MT_LAUNCH_CHECK(name);
    return MT_OK;
  }
  WgradArgs a{};
  a.delta = delta->p; a.in = v; a.Out = Out; a.accumulate = accumulate != 0;
  const size_t n = (size_t)Out * v.n;
  const Plan plan = choose(Out, v.groups, v.w, n);
  const bool wide = plan.rows == 256, pair = plan.pair;
  const uint32_t split = plan.split;
  a.tiles_m = cdiv(Out, plan.rows);
  const size_t tiles = (size_t)a.tiles_m * v.groups;
  a.per_split = cdiv(cdiv(v.w, split), KSTEP) * KSTEP;
  a.split = cdiv(v.w, a.per_split);
  const uint32_t columns = Out + v.groups, column_blocks = cdiv(columns, THREADS);
  uint32_t parts = 0, per_part = 0;
  if (plan.half) {
    // enough blocks for the whole chip, parts of at least 32 samples, few enough for every thread to read them all
    parts = cdiv(512, column_blocks);
    parts = parts > 32 ? 32 : parts;
    per_part = cdiv(v.w, parts) < 32 ? 32 : cdiv(v.w, parts);
    parts = cdiv(v.w, per_part);
  }
  const size_t sums = a.split > 1 ? a.split * (n + Out) : 0, ranges = (size_t)parts * columns, column_sums = (size_t)parts * Out;
  float *ws = nullptr;
  if (sums + ranges) {
    int rc = mt::workspace_get(g_wgrad_ws, "packed weight gradient", sums + ranges + column_sums, &ws);
    if (rc) return rc;
  }
  if (plan.half) {
    a.ranges = ws + sums;
    a.column_sums = a.ranges + ranges;
    a.parts = parts;
    a.accumulate_bias = a.accumulate;
  }
  if (a.split > 1) {
    a.dweight = ws;
    a.dbias = !dbias ? nullptr : plan.half ? dbias->p : ws + a.split * n;
    a.accumulate = false;
  } else {
    a.dweight = dweight->p;
    a.dbias = dbias ? dbias->p : nullptr;
  }
  const size_t grid = tiles * a.split;
  if (grid >= (1u << 23)) return mt::fail(MT_E_UNAVAILABLE, "%s: too many weights for one launch", name);  // a grid has fewer than 2^32 threads
  if (plan.half) packed_wgrad_ranges_kernel<<<dim3(column_blocks, parts), THREADS, 0, mt::stream()>>>(ws + sums, ws + sums + ranges, delta->p, v, Out, per_part);
  if (wide && plan.half)
    packed_wgrad_kernel<2, 1, true><<<(unsigned)grid, THREADS, 0, mt::stream()>>>(a);
  else if (wide)
    packed_wgrad_kernel<2, 1, false><<<(unsigned)grid, THREADS, 0, mt::stream()>>>(a);
  else if (pair && plan.half)
    packed_wgrad_kernel<1, 2, true><<<(unsigned)grid, 2 * THREADS, 0, mt::stream()>>>(a);
  else if (pair)
    packed_wgrad_kernel<1, 2, false><<<(unsigned)grid, 2 * THREADS, 0, mt::stream()>>>(a);
  else
    packed_wgrad_kernel<1, 1, false><<<(unsigned)grid, THREADS, 0, mt::stream()>>>(a);
  MT_LAUNCH_CHECK(name);
  if (a.split > 1) {
    float *db = dbias && !plan.half ? dbias->p : nullptr;
    if (a.split > 8)
      packed_wgrad_join_kernel<4><<<cdiv(n + Out, THREADS / 4), THREADS, 0, mt::stream()>>>(dweight->p, db, ws, ws + a.split * n, a.split, n, Out, accumulate != 0);
    else
      packed_wgrad_join_kernel<1><<<cdiv(n + Out, THREADS), THREADS, 0, mt::stream()>>>(dweight->p, db, ws, ws + a.split * n, a.split, n, Out, accumulate != 0);
    MT_LAUNCH_CHECK(name);
  }
  return MT_OK;
}

}  // extern "C"
