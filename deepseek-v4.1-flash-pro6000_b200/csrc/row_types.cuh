// Logits rows of FP32, BF16 or FP16: conversion by 16-byte vectors and by elements, where a row's vectors lie, and the ids that
// one CTA of a team holds.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include "ds41_b200.h"

namespace ds41 {

template <class T> struct RowType;
template <> struct RowType<float> {
  static constexpr int kVec = 4;
  static constexpr float kMax = 3.402823466e+38f;
  static __device__ __forceinline__ float load(float v) { return v; }
  static __device__ __forceinline__ float store(float v) { return v; }
  // 0, or NaN once any value that went through was NaN or infinite
  using Finite = float;
  static __device__ __forceinline__ Finite check(const uint4 &q, Finite f) {
    return fmaf(__uint_as_float(q.x), 0.f, fmaf(__uint_as_float(q.y), 0.f, fmaf(__uint_as_float(q.z), 0.f, fmaf(__uint_as_float(q.w), 0.f, f))));
  }
  static __device__ __forceinline__ bool all_finite(Finite f) { return f == 0.f; }
  // -inf everywhere; q where `in` has a bit, -inf elsewhere; the largest of the vectors' values (NaN passed over)
  static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  static __device__ __forceinline__ uint4 only(const uint4 &q, unsigned in) {
    return make_uint4(in & 1u ? q.x : 0xff800000u, in & 2u ? q.y : 0xff800000u, in & 4u ? q.z : 0xff800000u, in & 8u ? q.w : 0xff800000u);
  }
  template <int kCount> static __device__ __forceinline__ float largest(const uint4 (&q)[kCount]) {
    float m[2] = {__uint_as_float(q[0].x), __uint_as_float(q[0].y)};
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
      m[0] = fmaxf(m[0], fmaxf(__uint_as_float(q[u].x), __uint_as_float(q[u].y)));
      m[1] = fmaxf(m[1], fmaxf(__uint_as_float(q[u].z), __uint_as_float(q[u].w)));
    }
    return fmaxf(m[0], m[1]);
  }
  static __device__ __forceinline__ void unpack(const uint4 &q, float (&x)[4]) {
    x[0] = __uint_as_float(q.x); x[1] = __uint_as_float(q.y); x[2] = __uint_as_float(q.z); x[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <> struct RowType<__nv_bfloat16> {
  static constexpr int kVec = 8;
  static constexpr float kMax = 3.38953139e+38f;   // 0x7f7f
  static __device__ __forceinline__ float load(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 store(float v) { return __float2bfloat16_rn(v); }
  using Finite = __nv_bfloat162;
  static __device__ __forceinline__ Finite check(const uint4 &q, Finite f) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      Finite v;
      *reinterpret_cast<uint32_t *>(&v) = w[k];
      f = __hfma2(v, __float2bfloat162_rn(0.f), f);
    }
    return f;
  }
  static __device__ __forceinline__ bool all_finite(Finite f) { return __low2float(f) == 0.f && __high2float(f) == 0.f; }
  static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  static __device__ __forceinline__ uint4 only(const uint4 &q, unsigned in) {
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t keep = ((in >> 2 * k) & 1u) * 0xffffu | ((in >> (2 * k + 1)) & 1u) * 0xffff0000u;
      w[k] = (w[k] & keep) | (0xff80ff80u & ~keep);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  template <int kCount> static __device__ __forceinline__ float largest(const uint4 (&q)[kCount]) {
    const Finite *v = reinterpret_cast<const Finite *>(q);
    Finite m[2] = {v[0], v[1]};
#pragma unroll
    for (int i = 2; i < 4 * kCount; ++i) m[i & 1] = __hmax2(m[i & 1], v[i]);
    m[0] = __hmax2(m[0], m[1]);
    return fmaxf(__low2float(m[0]), __high2float(m[0]));
  }
  static __device__ __forceinline__ void unpack(const uint4 &q, float (&x)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) { x[2 * k] = __uint_as_float(w[k] << 16); x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u); }
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(x[2 * k + 1]), "f"(x[2 * k]));
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct RowType<__half> {
  static constexpr int kVec = 8;
  static constexpr float kMax = 65504.f;
  static __device__ __forceinline__ float load(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half store(float v) { return __float2half_rn(v); }
  using Finite = __half2;
  static __device__ __forceinline__ Finite check(const uint4 &q, Finite f) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      Finite v;
      *reinterpret_cast<uint32_t *>(&v) = w[k];
      f = __hfma2(v, __float2half2_rn(0.f), f);
    }
    return f;
  }
  static __device__ __forceinline__ bool all_finite(Finite f) { return __low2float(f) == 0.f && __high2float(f) == 0.f; }
  static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
  static __device__ __forceinline__ uint4 only(const uint4 &q, unsigned in) {
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t keep = ((in >> 2 * k) & 1u) * 0xffffu | ((in >> (2 * k + 1)) & 1u) * 0xffff0000u;
      w[k] = (w[k] & keep) | (0xfc00fc00u & ~keep);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  template <int kCount> static __device__ __forceinline__ float largest(const uint4 (&q)[kCount]) {
    const Finite *v = reinterpret_cast<const Finite *>(q);
    Finite m[2] = {v[0], v[1]};
#pragma unroll
    for (int i = 2; i < 4 * kCount; ++i) m[i & 1] = __hmax2(m[i & 1], v[i]);
    m[0] = __hmax2(m[0], m[1]);
    return fmaxf(__low2float(m[0]), __high2float(m[0]));
  }
  static __device__ __forceinline__ void unpack(const uint4 &q, float (&x)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      __half2 h;
      *reinterpret_cast<uint32_t *>(&h) = w[k];
      const float2 f = __half22float2(h);
      x[2 * k] = f.x; x[2 * k + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(x[2 * k + 1]), "f"(x[2 * k]));
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

__device__ __forceinline__ bool finite_bits(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

inline size_t row_type_bytes(int dtype) { return dtype == DS41_B200_F32 ? 4 : 2; }

// Whether `out` (rows of `width` elements, out_stride apart) can be written while `in` is read: in place (the same rows), or no byte in
// common.  Views of the same buffer side by side (the same stride, columns apart) are apart.
inline bool rows_apart_or_same(const void *in, int64_t in_stride, const void *out, int64_t out_stride, int rows, int width, size_t bytes) {
  if (rows == 1) in_stride = out_stride = width;
  if (in == out && in_stride == out_stride) return true;
  const uintptr_t a = reinterpret_cast<uintptr_t>(in), b = reinterpret_cast<uintptr_t>(out);
  const uintptr_t a_end = a + (uintptr_t(rows - 1) * uintptr_t(in_stride) + uintptr_t(width)) * bytes;
  const uintptr_t b_end = b + (uintptr_t(rows - 1) * uintptr_t(out_stride) + uintptr_t(width)) * bytes;
  if (a_end <= b || b_end <= a) return true;
  if (in_stride != out_stride || in_stride == 0) return false;
  const uintptr_t apart = (a < b ? b - a : a - b) % (uintptr_t(in_stride) * bytes);
  return apart >= uintptr_t(width) * bytes && apart + uintptr_t(width) * bytes <= uintptr_t(in_stride) * bytes;
}

}  // namespace ds41
