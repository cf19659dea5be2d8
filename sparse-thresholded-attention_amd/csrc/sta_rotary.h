// sta_rotary.h -- what the rotation and the normed rotation share: 16 bytes of a row in fp32 and back, and a token's
// angles.
#pragma once
#include "sta_cache.h"
#include "sta_device.h"

namespace sta {

template <int DT>
constexpr int ROT_V = DT == DT_F32 ? 4 : 8;       // elements in 16 bytes

template <int DT>
__device__ __forceinline__ void unpack16(const u32x4& w, float* o) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT == DT_F32) {
      o[e] = __uint_as_float(w[e]);
    } else if constexpr (DT == DT_BF16) {
      o[2 * e] = __uint_as_float(w[e] << 16);
      o[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    } else {
      o[2 * e] = f16_bits_to_f32(w[e] & 0xffffu);
      o[2 * e + 1] = f16_bits_to_f32(w[e] >> 16);
    }
  }
}

template <int DT>
__device__ __forceinline__ u32x4 pack16(const float* o) {
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT == DT_F32) w[e] = __float_as_uint(o[e]);
    else w[e] = pack2_dt<DT>(o[2 * e], o[2 * e + 1]);
  }
  return w;
}

__device__ __forceinline__ double position(const sta_rotary_args& a, int axis, int64_t t) {
  const int64_t i = axis * a.pos_axis_stride + t * a.pos_tok_stride;
  if (a.pos_type == STA_POS_I64) return (double)((const int64_t*)a.positions)[i];
  if (a.pos_type == STA_POS_F32) return (double)((const float*)a.positions)[i];
  return (double)((const int32_t*)a.positions)[i];
}

// (cos, sin) of frequency f at token t, times the scale; the sine's sign turned for the inverse
__device__ __forceinline__ float2 turn_of(const sta_rotary_args& a, int f, int64_t t) {
  int axis = 0, first = 0;
  while (axis + 1 < a.axes && f >= first + a.section[axis]) first += a.section[axis++];
  double turns = position(a, axis, t) * (double)a.pos_scale * (double)a.inv_freq[f];
  turns *= 0.15915494309189533577;
  turns -= rint(turns);
  float s, c;
  sincospif((float)(2.0 * turns), &s, &c);
  return make_float2(c * a.rope_scale, (a.inverse ? -s : s) * a.rope_scale);
}

}  // namespace sta
