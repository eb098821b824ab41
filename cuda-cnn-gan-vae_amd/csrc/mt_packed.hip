// Activations in 8 bits: mt_pack and mt_unpack.
#include <type_traits>

#include "mt_packed.h"

namespace {

using mt::PackedView;

constexpr int THREADS = 256;
constexpr int LANES = 32;  // lanes that share a group: four values each

// Both kernels move 5 bytes per value and compute little.  32 lanes take a group, four values each as one 128-bit access: from a 16-byte
// boundary, the same past the caches (option "nontemporal"), or from any address, where the last lane of a sample may have fewer.  One
// group per 32 lanes and many blocks: 256 x 64 x 32 x 32 packed and unpacked 35.2 us, 36.7 with two groups under way at a time, 39.9 with
// four (samples far shorter than a group would gain by two: 100000 x 30 12.4 us against 10.5).  Single values 32 apart took 20000 samples
// of 1001 30 us to unpack, this 25.6.
// Samples of whole groups are one long row of groups (`rows` false): no division by the groups of a sample is needed then.
enum Access { FOUR, FOUR_PAST, FOUR_ANY };
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));

struct PackJob {
  PackedView v;
  uint64_t total;  // groups of the whole tensor
  bool rows;
};
struct Place {
  size_t tensor, bytes;  // where the group starts in the fp32 tensor and among the bytes
  uint32_t count, room;  // its values, and its bytes with the sample's padding
};
template <class Index>
__device__ __forceinline__ Place place(const PackJob &job, uint64_t g) {
  if (!job.rows) return Place{(size_t)g * mt::PACK_GROUP, (size_t)g * mt::PACK_GROUP, mt::PACK_GROUP, mt::PACK_GROUP};
  const Index w = (Index)g / job.v.groups;
  const uint32_t first = (uint32_t)((Index)g - w * job.v.groups) * mt::PACK_GROUP;
  return Place{(size_t)w * job.v.n + first, (size_t)w * job.v.pitch + first, min(mt::PACK_GROUP, job.v.n - first), min(mt::PACK_GROUP, job.v.pitch - first)};
}

template <int ACCESS, class Index>
__global__ __launch_bounds__(THREADS) void pack_kernel(PackJob job, const float *in) {
  const uint32_t lane = threadIdx.x % LANES, e = lane * 4u;
  const uint64_t step = (uint64_t)gridDim.x * (THREADS / LANES);
  for (uint64_t g = (uint64_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES; g < job.total; g += step) {
    const Place at = place<Index>(job, g);
    const float *p = in + at.tensor;
    float v[4];
    if (ACCESS != FOUR_ANY || e + 4u <= at.count) {
      const float *q = p + (ACCESS == FOUR_ANY ? e : min(e, at.count - 4u));  // behind the end: values of the group again
      floatx4 t;
      if (ACCESS == FOUR_ANY)
        t = *reinterpret_cast<const floatx4_any *>(q);
      else if (ACCESS == FOUR_PAST)
        t = __builtin_nontemporal_load(reinterpret_cast<const floatx4 *>(q));
      else
        t = *reinterpret_cast<const floatx4 *>(q);
      v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++) v[k] = p[min(e + k, at.count - 1u)];
    }
    const float low = mt::over_lanes<mt::Lowest, LANES>(mt::min_nan(mt::min_nan(v[0], v[1]), mt::min_nan(v[2], v[3])));
    const float high = mt::over_lanes<mt::Highest, LANES>(mt::max_nan(mt::max_nan(v[0], v[1]), mt::max_nan(v[2], v[3])));
    const mt::PackScale s = mt::pack_scale(low, high);
    if (lane == 0) job.v.pair[g] = make_float2(s.low, s.step);
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) w = mt::pack_into(s, v[k], k, w);
    // bytes behind the sample's end are its padding
    if (ACCESS == FOUR_ANY && e < at.count && e + 4u > at.count) w &= (1u << 8 * (at.count - e)) - 1u;
    if (e < at.room) *reinterpret_cast<uint32_t *>(job.v.q + at.bytes + e) = e < at.count ? w : 0u;
  }
}

template <int ACCESS, class Index>
__global__ __launch_bounds__(THREADS) void unpack_kernel(float *out, PackJob job) {
  const uint32_t lane = threadIdx.x % LANES, e = lane * 4u;
  const uint64_t step = (uint64_t)gridDim.x * (THREADS / LANES);
  for (uint64_t g = (uint64_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES; g < job.total; g += step) {
    const Place at = place<Index>(job, g);
    const float2 pair = job.v.pair[g];
    const uint32_t q = *reinterpret_cast<const uint32_t *>(job.v.q + at.bytes + min(e, at.room - 4u));
    float t[4];
#pragma unroll
    for (int k = 0; k < 4; k++) t[k] = mt::unpack_value(pair, (q >> (8 * k)) & 255u);
    float *p = out + at.tensor + e;
    const floatx4 v = {t[0], t[1], t[2], t[3]};
    if (ACCESS == FOUR_ANY) {
      if (e + 4u <= at.count) {
        *reinterpret_cast<floatx4_any *>(p) = v;
      } else {
#pragma unroll
        for (uint32_t k = 0; k < 3; k++)
          if (e + k < at.count) p[k] = t[k];
      }
    } else if (e < at.count) {
      if (ACCESS == FOUR_PAST)
        __builtin_nontemporal_store(v, reinterpret_cast<floatx4 *>(p));
      else
        *reinterpret_cast<floatx4 *>(p) = v;
    }
  }
}

// calls f with the job, how a lane accesses its four values, and the width that a group's number needs
template <class F>
void with_job(const PackedView &v, const float *tensor, F &&f) {
  PackJob job{v, (uint64_t)v.w * v.groups, v.n % mt::PACK_GROUP != 0};
  const uint64_t blocks = (job.total + THREADS / LANES - 1) / (THREADS / LANES);
  const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
  const bool whole = v.n % 4 == 0 && ((uintptr_t)tensor & 15u) == 0, past = whole && mt::past_caches((size_t)v.w * v.n * 4);
  const auto with_index = [&](auto access) {
    if (job.rows && job.total > 0xffffffffull) f(job, grid, access, uint64_t{}); else f(job, grid, access, uint32_t{});
  };
  if (past)
    with_index(std::integral_constant<int, FOUR_PAST>{});
  else if (whole)
    with_index(std::integral_constant<int, FOUR>{});
  else
    with_index(std::integral_constant<int, FOUR_ANY>{});
}

}  // namespace

extern "C" {

int mt_packed_bytes(uint32_t w, uint32_t z, uint32_t y, uint32_t x, uint64_t *bytes) {
  uint32_t n;
  uint64_t b;
  if (bytes == nullptr) return mt::fail(MT_E_ARGUMENT, "mt_packed_bytes: null result pointer");
  if (!mt::packed_size(w, z, y, x, &n, &b)) return mt::fail(MT_E_UNAVAILABLE, "mt_packed_bytes: a sample of 2^31 elements or more is not supported");
  *bytes = b;
  return MT_OK;
}

int mt_pack(const mt_packed_tensor *out, const mt_tensor *in) {
  if (mt::bad(out) || mt::bad(in)) return mt::fail(MT_E_ARGUMENT, "mt_pack: null tensor, or packed memory that is not 16-byte aligned");
  if (out->w != in->w || out->z != in->z || out->y != in->y || out->x != in->x) return mt::fail(MT_E_SHAPE, "mt_pack: sizes do not match");
  PackedView v;
  if (!mt::packed_view(out, &v)) return mt::fail(MT_E_UNAVAILABLE, "mt_pack: a sample of 2^31 elements or more is not supported");
  if (v.w == 0 || v.n == 0) return MT_OK;
  if (mt::overlap(in, v)) return mt::fail(MT_E_ARGUMENT, "mt_pack: the packed tensor shares memory with the input");
  mt::note_write(v.q, mt::packed_bytes(v));
  mt::ProfileScope prof("mt_pack");
  with_job(v, in->p, [&](const PackJob &job, unsigned grid, auto access, auto index) {
    pack_kernel<decltype(access)::value, decltype(index)><<<grid, THREADS, 0, mt::stream()>>>(job, in->p);
  });
  MT_LAUNCH_CHECK("mt_pack");
  return MT_OK;
}

int mt_unpack(const mt_tensor *out, const mt_packed_tensor *in) {
  if (mt::bad(out) || mt::bad(in)) return mt::fail(MT_E_ARGUMENT, "mt_unpack: null tensor, or packed memory that is not 16-byte aligned");
  if (out->w != in->w || out->z != in->z || out->y != in->y || out->x != in->x) return mt::fail(MT_E_SHAPE, "mt_unpack: sizes do not match");
  PackedView v;
  if (!mt::packed_view(in, &v)) return mt::fail(MT_E_UNAVAILABLE, "mt_unpack: a sample of 2^31 elements or more is not supported");
  if (v.w == 0 || v.n == 0) return MT_OK;
  if (mt::overlap(out, v)) return mt::fail(MT_E_ARGUMENT, "mt_unpack: the packed tensor shares memory with the output");
  mt::note_write(out);
  mt::ProfileScope prof("mt_unpack");
  with_job(v, out->p, [&](const PackJob &job, unsigned grid, auto access, auto index) {
    unpack_kernel<decltype(access)::value, decltype(index)><<<grid, THREADS, 0, mt::stream()>>>(out->p, job);
  });
  MT_LAUNCH_CHECK("mt_unpack");
  return MT_OK;
}

}  // extern "C"
