// Activations in 8 bits: mt_pack and mt_unpack.
#include <type_traits>

#include "mt_packed.h"

namespace {

using mt::PackedView;

constexpr int THREADS = 256;
constexpr int LANES = 32;    // lanes that share a group: four values each
constexpr int AT_ONCE = 4;   // groups in flight per 32 lanes

// Both kernels move 5 bytes per value and compute little: what they need is enough loads in flight.  32 lanes take a group, four
// values each (one 128-bit access where the tensor allows, four values 32 apart otherwise), and work on four groups at once.
// Samples of whole groups are one long row of groups (`rows` false): no division by the groups of a sample is needed then.
typedef float floatx4 __attribute__((ext_vector_type(4)));

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
// value k of a lane within its group, and whether a lane's four are next to each other
template <bool VEC>
__device__ __forceinline__ uint32_t within(uint32_t lane, int k) { return VEC ? lane * 4u + k : lane + 32u * k; }

template <bool VEC, bool PAST, class Index>
__global__ __launch_bounds__(THREADS) void pack_kernel(PackJob job, const float *in) {
  const uint32_t lane = threadIdx.x % LANES;
  const uint64_t step = (uint64_t)gridDim.x * (THREADS / LANES);
  for (uint64_t g0 = (uint64_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES; g0 < job.total; g0 += AT_ONCE * step) {
    Place at[AT_ONCE];
    float v[AT_ONCE][4];
#pragma unroll
    for (int u = 0; u < AT_ONCE; u++) {
      const uint64_t g = g0 + u * step < job.total ? g0 + u * step : g0;
      at[u] = place<Index>(job, g);
      if (VEC) {
        const floatx4 *p = reinterpret_cast<const floatx4 *>(in + at[u].tensor + min(lane * 4u, at[u].count - 4u));  // behind the end: values of the group again
        const floatx4 t = PAST ? __builtin_nontemporal_load(p) : *p;
        v[u][0] = t.x; v[u][1] = t.y; v[u][2] = t.z; v[u][3] = t.w;
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++) v[u][k] = in[at[u].tensor + min(within<VEC>(lane, k), at[u].count - 1u)];
      }
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; u++) {
      if (g0 + u * step >= job.total) return;
      const float low = mt::over_lanes<mt::Lowest, LANES>(mt::min_nan(mt::min_nan(v[u][0], v[u][1]), mt::min_nan(v[u][2], v[u][3])));
      const float high = mt::over_lanes<mt::Highest, LANES>(mt::max_nan(mt::max_nan(v[u][0], v[u][1]), mt::max_nan(v[u][2], v[u][3])));
      const mt::PackScale s = mt::pack_scale(low, high);
      if (lane == 0) job.v.pair[g0 + u * step] = make_float2(s.low, s.step);
      uint8_t *p = job.v.q + at[u].bytes;
      if (VEC) {
        uint32_t w = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) w = mt::pack_into(s, v[u][k], k, w);
        if (lane * 4u < at[u].room) *reinterpret_cast<uint32_t *>(p + lane * 4u) = lane * 4u < at[u].count ? w : 0u;
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (within<VEC>(lane, k) < at[u].room) p[within<VEC>(lane, k)] = within<VEC>(lane, k) < at[u].count ? (uint8_t)mt::pack_into(s, v[u][k], 0, 0u) : (uint8_t)0;
      }
    }
  }
}

template <bool VEC, bool PAST, class Index>
__global__ __launch_bounds__(THREADS) void unpack_kernel(float *out, PackJob job) {
  const uint32_t lane = threadIdx.x % LANES;
  const uint64_t step = (uint64_t)gridDim.x * (THREADS / LANES);
  for (uint64_t g0 = (uint64_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES; g0 < job.total; g0 += AT_ONCE * step) {
    Place at[AT_ONCE];
    float2 pair[AT_ONCE];
    uint32_t q[AT_ONCE][4];
#pragma unroll
    for (int u = 0; u < AT_ONCE; u++) {
      const uint64_t g = g0 + u * step < job.total ? g0 + u * step : g0;
      at[u] = place<Index>(job, g);
      pair[u] = job.v.pair[g];
      const uint8_t *p = job.v.q + at[u].bytes;
      if (VEC) {
        q[u][0] = *reinterpret_cast<const uint32_t *>(p + min(lane * 4u, at[u].count - 4u));
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++) q[u][k] = p[min(within<VEC>(lane, k), at[u].count - 1u)];
      }
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; u++) {
      if (g0 + u * step >= job.total) return;
      float *p = out + at[u].tensor;
      if (VEC) {
        float t[4];
#pragma unroll
        for (int k = 0; k < 4; k++) t[k] = mt::unpack_value(pair[u], (q[u][0] >> (8 * k)) & 255u);
        if (lane * 4u < at[u].count) {
          const floatx4 v = {t[0], t[1], t[2], t[3]};
          if (PAST)
            __builtin_nontemporal_store(v, reinterpret_cast<floatx4 *>(p + lane * 4u));
          else
            *reinterpret_cast<floatx4 *>(p + lane * 4u) = v;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (within<VEC>(lane, k) < at[u].count) p[within<VEC>(lane, k)] = mt::unpack_value(pair[u], q[u][k]);
      }
    }
  }
}

// calls f with the job, how a lane accesses its four values (singly, as one access, as one access past the caches: option
// "nontemporal"), and the width that a group's number needs
template <class F>
void with_job(const PackedView &v, const float *tensor, F &&f) {
  PackJob job{v, (uint64_t)v.w * v.groups, v.n % mt::PACK_GROUP != 0};
  const uint64_t blocks = (job.total + THREADS / LANES * AT_ONCE - 1) / (THREADS / LANES * AT_ONCE);
  const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
  const bool vec = v.n % 4 == 0 && ((uintptr_t)tensor & 15u) == 0, past = vec && mt::past_caches((size_t)v.w * v.n * 4);
  const auto with_index = [&](auto vec_, auto past_) {
    if (job.rows && job.total > 0xffffffffull) f(job, grid, vec_, past_, uint64_t{}); else f(job, grid, vec_, past_, uint32_t{});
  };
  if (past)
    with_index(std::true_type{}, std::true_type{});
  else if (vec)
    with_index(std::true_type{}, std::false_type{});
  else
    with_index(std::false_type{}, std::false_type{});
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
  with_job(v, in->p, [&](const PackJob &job, unsigned grid, auto vec, auto past, auto index) {
    pack_kernel<decltype(vec)::value, decltype(past)::value, decltype(index)><<<grid, THREADS, 0, mt::stream()>>>(job, in->p);
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
  with_job(v, out->p, [&](const PackJob &job, unsigned grid, auto vec, auto past, auto index) {
    unpack_kernel<decltype(vec)::value, decltype(past)::value, decltype(index)><<<grid, THREADS, 0, mt::stream()>>>(out->p, job);
  });
  MT_LAUNCH_CHECK("mt_unpack");
  return MT_OK;
}

}  // extern "C"
