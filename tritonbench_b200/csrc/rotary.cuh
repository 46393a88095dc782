// Rotary positions on registers, shared by the stand-alone kernel (rotary.cu) and the cache append (kv_append.cu).
//
//   y_a = x_a * cos - x_b * sin,    y_b = x_b * cos + x_a * sin
//
// for every pair (a, b) of a head: (i, i + rot/2) in the half layout, (2i, 2i + 1) in the interleaved one.  The table
// holds cos and sin in fp32 ([max_pos][rot]: rot/2 cosines, then rot/2 sines; angles computed in 64 bits when it is
// built, because an fp32 angle of position 100000 is off by 4e-3 rad).  Every product and sum is rounded on its own
// (no fused multiply-add), so the result has the same bits as the elementwise expression and the e4m3 codes made from
// it do not depend on which kernel computed them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200fp8 {

__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s) {
  const float ya = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  const float yb = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = ya;
  b = yb;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// 16 bytes of T <-> fp32
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& raw, float (&v)[16 / sizeof(T)]) {
  const T* h = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) v[i] = to_f32<T>(h[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&v)[16 / sizeof(T)]) {
  uint4 raw;
  T* h = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) h[i] = from_f32<T>(v[i]);
  return raw;
}

// A slot is the 2 * kN elements of a head that one thread owns, as two vectors a and b.  Half layout: a and b are the
// two halves of kN pairs.  Interleaved: 2 * kN neighbouring elements, kN pairs.  c and s: the kN cosines and sines.
template <int kN, bool kInterleaved>
__device__ __forceinline__ void rotate_slot(float (&a)[kN], float (&b)[kN], const float (&c)[kN], const float (&s)[kN]) {
  if constexpr (kInterleaved && kN > 1) {
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) rotate_pair(a[2 * i], a[2 * i + 1], c[i], s[i]);
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) rotate_pair(b[2 * i], b[2 * i + 1], c[kN / 2 + i], s[kN / 2 + i]);
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) rotate_pair(a[i], b[i], c[i], s[i]);
  }
}

// kN table entries from p (16-byte aligned when kN is a multiple of 4)
template <int kN>
__device__ __forceinline__ void load_table(const float* p, float (&v)[kN]) {
  if constexpr (kN % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kN / 4; ++i) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p) + i);
      v[4 * i] = f.x;
      v[4 * i + 1] = f.y;
      v[4 * i + 2] = f.z;
      v[4 * i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = __ldg(p + i);
  }
}

}  // namespace b200fp8
