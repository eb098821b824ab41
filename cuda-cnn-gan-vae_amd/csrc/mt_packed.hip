// Activations in 8 bits: mt_pack, mt_unpack and the linear layer's weight gradient from a packed input.
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

// dweight[o][i] (+)= sum_b delta[b][o] * value[b][i], dbias[o] (+)= sum_b delta[b][o]: one thread per weight
__global__ __launch_bounds__(THREADS) void linear_weights_kernel(float *dweight, float *dbias, const float *delta, PackedView in, uint32_t Out, bool accumulate) {
  const uint32_t i = blockIdx.x * 64u + threadIdx.x % 64u;
  for (uint32_t o = blockIdx.y * 4u + threadIdx.x / 64u; o < Out; o += gridDim.y * 4u) {
    float acc = 0.f, sum = 0.f;
    if (i < in.n || i == 0)
      for (uint32_t b = 0; b < in.w; b++) {
        const float d = delta[(size_t)b * Out + o];
        if (i < in.n) acc += d * mt::unpack_value(in.pair[(size_t)b * in.groups + i / mt::PACK_GROUP], in.q[(size_t)b * in.pitch + i]);
        sum += d;
      }
    if (i < in.n) {
      const size_t e = (size_t)o * in.n + i;
      dweight[e] = accumulate ? dweight[e] + acc : acc;
    }
    if (i == 0 && dbias) dbias[o] = accumulate ? dbias[o] + sum : sum;
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
  const unsigned gy = cdiv(Out, 4);
  linear_weights_kernel<<<dim3(cdiv(v.n ? v.n : 1, 64), gy < 4096 ? gy : 4096), THREADS, 0, mt::stream()>>>(dweight->p, dbias ? dbias->p : nullptr, delta->p, v, Out,
                                                                                                           accumulate != 0);
  MT_LAUNCH_CHECK(name);
  return MT_OK;
}

}  // extern "C"
