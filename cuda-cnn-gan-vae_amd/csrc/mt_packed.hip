// Activations in 8 bits: mt_pack and mt_unpack.
#include "mt_packed.h"

namespace {

using mt::cdiv;
using mt::PackedView;

constexpr int THREADS = 256;

inline unsigned blocks_for(size_t units, size_t per_block) {
  const size_t b = (units + per_block - 1) / per_block;
  return (unsigned)(b < 16384 ? b : 16384);
}

// 32 lanes per group, four elements 32 apart per lane
__global__ __launch_bounds__(THREADS) void pack_kernel(PackedView out, const float *in, size_t total) {
  const uint32_t lane = threadIdx.x & 31u;
  for (size_t g = (size_t)blockIdx.x * (THREADS / 32) + threadIdx.x / 32; g < total; g += (size_t)gridDim.x * (THREADS / 32)) {
    const size_t w = g / out.groups;
    const uint32_t first = (uint32_t)(g - w * out.groups) * mt::PACK_GROUP;
    const float *src = in + w * out.n;
    float v[4], low, high;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t i = first + lane + 32u * k;
      v[k] = src[i < out.n ? i : first];  // behind the end: a value of the group again
      low = k ? mt::min_nan(low, v[k]) : v[k];
      high = k ? mt::max_nan(high, v[k]) : v[k];
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      low = mt::min_nan(low, __shfl_xor(low, off, 64));
      high = mt::max_nan(high, __shfl_xor(high, off, 64));
    }
    const mt::PackScale s = mt::pack_scale(low, high);
    if (lane == 0) out.pair[g] = make_float2(s.low, s.step);
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t i = first + lane + 32u * k;
      if (i < out.pitch) out.q[w * out.pitch + i] = i < out.n ? (uint8_t)mt::pack_value(s, v[k]) : (uint8_t)0;
    }
  }
}

__global__ __launch_bounds__(THREADS) void unpack_kernel(float *out, PackedView in, size_t total) {
  for (size_t e = (size_t)blockIdx.x * THREADS + threadIdx.x; e < total; e += (size_t)gridDim.x * THREADS) {
    const size_t w = e / in.n;
    const uint32_t i = (uint32_t)(e - w * in.n);
    out[e] = mt::unpack_value(in.pair[w * in.groups + i / mt::PACK_GROUP], in.q[w * in.pitch + i]);
  }
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
  const size_t total = (size_t)v.w * v.groups;
  pack_kernel<<<blocks_for(total, THREADS / 32), THREADS, 0, mt::stream()>>>(v, in->p, total);
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
  const size_t total = (size_t)v.w * v.n;
  unpack_kernel<<<blocks_for(total, THREADS), THREADS, 0, mt::stream()>>>(out->p, v, total);
  MT_LAUNCH_CHECK("mt_unpack");
  return MT_OK;
}

}  // extern "C"
