// Device helpers of the row-wise kernels: vectors of four values at any alignment with a ragged end, sums over a wave.
#pragma once

#include "mg_common.h"

namespace mg {

template <int N>
struct int_c { static constexpr int value = N; };

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));

// Four values from p on, of which the first `left` exist
__device__ __forceinline__ f4 load4(const float* p, int left) {
  f4 r = io4<float>::fill(0.0f);
  if (left >= 4) {
    const f32x4u x = *reinterpret_cast<const f32x4u*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = x[j];
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < left) r.v[j] = p[j];
  }
  return r;
}
__device__ __forceinline__ f4 load4(const bf16_t* p, int left) {
  f4 r = io4<float>::fill(0.0f);
  if (left >= 4) {
    const u16x4u x = *reinterpret_cast<const u16x4u*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = bf16_to_f32(x[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < left) r.v[j] = bf16_to_f32(p[j]);
  }
  return r;
}
__device__ __forceinline__ void store4(float* p, const f4& v, int left) {
  if (left >= 4) {
    const f32x4u x = {v.v[0], v.v[1], v.v[2], v.v[3]};
    *reinterpret_cast<f32x4u*>(p) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < left) p[j] = v.v[j];
  }
}
__device__ __forceinline__ void store4(bf16_t* p, const f4& v, int left) {
  if (left >= 4) {
    u16x4u x;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = f32_to_bf16(v.v[j]);
    *reinterpret_cast<u16x4u*>(p) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < left) p[j] = f32_to_bf16(v.v[j]);
  }
}

// The sum over a wave's lanes, in every lane: within rows of 16 lanes by cross-lane operands, then
// from row to row, where the last lane has the whole
__device__ __forceinline__ float wave_sum(float x) {
  const auto add = [](float x, auto ctrl, auto rows) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  x = add(x, int_c<0xb1>{}, int_c<0xf>{});   // lane ^ 1
  x = add(x, int_c<0x4e>{}, int_c<0xf>{});   // lane ^ 2
  x = add(x, int_c<0x141>{}, int_c<0xf>{});  // mirrored in 8
  x = add(x, int_c<0x140>{}, int_c<0xf>{});  // mirrored in 16
  x = add(x, int_c<0x142>{}, int_c<0xa>{});  // row 0 into 1, 2 into 3
  x = add(x, int_c<0x143>{}, int_c<0xc>{});  // the lower half into the upper
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

}  // namespace mg
