// Activations kept in 8 bits between the forward and the backward pass (mt_packed_tensor): the layout, and what the
// kernels that write and read it share.
//
// A sample's n = Z*Y*X values are cut into groups of 128 consecutive ones (the last may be shorter).  A group holds its
// lowest value and a step of 1/255 of its range as fp32, an element the number of steps (0..255) above the lowest value:
//     value = low + step * q,   |value - x| <= step / 2 (+ fp32 rounding of low, step and the sum)
// A range with its own offset suits activations: what a ReLU leaves has no negative half to waste a bit on, and a feature
// with a large mean keeps the resolution of its spread.  128 elements: 8 bytes of (low, step) are 6 % of the group,
// and one column tile of the weight-gradient product has one pair per sample.
//
// Memory: [w][pitch] bytes of q, pitch = n rounded up to 16 (so a sample's bytes start 16-byte aligned; the padding is zero),
// then [w][groups] pairs (low, step).
#pragma once

#include <float.h>

#include "mt_common.h"

namespace mt {

constexpr uint32_t PACK_GROUP = 128;

struct PackedView {
  uint8_t *q;
  float2 *pair;
  uint32_t w, n, groups, pitch;
};

// Elements of a sample and bytes of a packed tensor; false where a sample has (nearly) 2^31 elements or more.
inline bool packed_size(uint32_t w, uint32_t z, uint32_t y, uint32_t x, uint32_t *n, uint64_t *bytes) {
  uint64_t zy = (uint64_t)z * y, s;
  if (__builtin_mul_overflow(zy, (uint64_t)x, &s) || s > 0x7fffffefull) return false;
  *n = (uint32_t)s;
  const uint64_t pitch = (s + 15) / 16 * 16, groups = (s + PACK_GROUP - 1) / PACK_GROUP;
  *bytes = (uint64_t)w * (pitch + 8 * groups);  // below 2^32 * 2^31 * 17/16: no overflow
  return true;
}

inline bool packed_view(const mt_packed_tensor *t, PackedView *v) {
  uint64_t bytes;
  if (!packed_size(t->w, t->z, t->y, t->x, &v->n, &bytes)) return false;
  v->w = t->w;
  v->pitch = (v->n + 15) / 16 * 16;
  v->groups = cdiv(v->n, PACK_GROUP);
  v->q = static_cast<uint8_t *>(t->p);
  v->pair = reinterpret_cast<float2 *>(v->q + (size_t)v->w * v->pitch);
  return true;
}
inline uint64_t packed_bytes(const PackedView &v) { return (uint64_t)v.w * (v.pitch + 8ull * v.groups); }
// null where the sizes need memory, or not aligned as the layout needs it
inline bool bad(const mt_packed_tensor *t) {
  if (t == nullptr) return true;
  const bool empty = t->w == 0 || t->z == 0 || t->y == 0 || t->x == 0;
  return !empty && (t->p == nullptr || ((uintptr_t)t->p & 15u) != 0);
}

// do the two byte ranges share memory
inline bool overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
  const uintptr_t pa = (uintptr_t)a, pb = (uintptr_t)b;
  return na != 0 && nb != 0 && pa < pb + nb && pb < pa + na;
}
inline bool overlap(const mt_tensor *a, const mt_tensor *b) { return overlap(a->p, count(a) * 4, b->p, count(b) * 4); }
inline bool overlap(const mt_tensor *a, const PackedView &b) { return overlap(a->p, count(a) * 4, b.q, packed_bytes(b)); }

// ---- device side ---------------------------------------------------------------------------------------------------
// 1 / y for a normal y up to 2^125, correctly rounded: the hardware's reciprocal and one step of Newton's method give the rounded
// quotient for every mantissa (all 2^23 compared with the division at ten exponents), without the ten instructions of a division
__device__ __forceinline__ float reciprocal(float y) {
  const float r = __builtin_amdgcn_rcpf(y);
  return __builtin_fmaf(__builtin_fmaf(-y, r, 1.f), r, r);
}

// (low, step, 1/step) of a group from its lowest and highest value.  A range that is not a finite number (a NaN or an
// infinity in the group, or values 3.4e38 apart) makes every value of the group NaN: what was lost shows.  A step below the
// smallest normal number counts as none, so that its reciprocal exists.
struct PackScale {
  float low, step, inverse;
};
__device__ __forceinline__ PackScale pack_scale(float low, float high) {
  PackScale s;
  const float range = high - low;
  const bool finite = range <= FLT_MAX;
  s.step = finite ? range * (1.f / 255.f) : 0.f;
  if (s.step < FLT_MIN) s.step = 0.f;
  s.low = finite ? low : __int_as_float(0x7fc00000);
  s.inverse = s.step > 0.f ? reciprocal(s.step) : 0.f;
  return s;
}
// the count of steps put into byte k of w: the instruction rounds half to even and holds the result within 0..255
__device__ __forceinline__ uint32_t pack_into(const PackScale &s, float x, int k, uint32_t w) { return __builtin_amdgcn_cvt_pk_u8_f32((x - s.low) * s.inverse, k, w); }
__device__ __forceinline__ float unpack_value(float2 pair, uint32_t q) { return pair.x + pair.y * (float)q; }

// minimum and maximum that let a NaN through
__device__ __forceinline__ float min_nan(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// sums, minima and maxima over 8, 16, 32 or 64 neighbouring lanes without LDS; every lane gets the same bits
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
struct Sum {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct Lowest {
  static __device__ __forceinline__ float of(float a, float b) { return min_nan(a, b); }
};
struct Highest {
  static __device__ __forceinline__ float of(float a, float b) { return max_nan(a, b); }
};
template <class Op, int L>
__device__ __forceinline__ float over_lanes(float v) {
  v = Op::of(v, dpp<0xb1>(v));                  // neighbours
  v = Op::of(v, dpp<0x4e>(v));                  // pairs of a quad
  v = Op::of(v, dpp<0x141>(v));                 // quads of eight lanes
  if (L > 8) v = Op::of(v, dpp<0x140>(v));      // halves of sixteen
  if (L > 16) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = Op::of(__uint_as_float(p[0]), __uint_as_float(p[1]));
  }
  if (L > 32) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = Op::of(__uint_as_float(p[0]), __uint_as_float(p[1]));
  }
  return v;
}

}  // namespace mt
