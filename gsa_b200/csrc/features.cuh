// SPDX-License-Identifier: Apache-2.0
// Shared definitions of the point-feature operators: element types, 16-byte
// vectors of them, and the scene offsets of packed rows.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "common.cuh"
#include "point_features.h"

namespace gsa {

// Element types at the C boundary (include/point_features.h).
enum Element {
  kF32 = POINT_FEATURES_F32,
  kF16 = POINT_FEATURES_F16,
  kBF16 = POINT_FEATURES_BF16
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_huge_valf();

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(float x) { return x; }
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) {
  return __bfloat162float(x);
}

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) {
  return __float2bfloat16_rn(x);
}

// Two floats rounded to nearest into one 32-bit word, the first one low.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// A 16-byte vector: V elements as floats.
template <typename T>
struct Vec {
  static constexpr int V = 16 / sizeof(T);
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) unpack2(w[i], f + 2 * i);
    }
  }
  static __device__ __forceinline__ void unpack2(uint32_t w, float* f) {
    if constexpr (__is_same(T, __nv_bfloat16)) {
      f[0] = __uint_as_float(w << 16);
      f[1] = __uint_as_float(w & 0xffff0000u);
    } else {
      const float2 p = __half22float2(*reinterpret_cast<__half2*>(&w));
      f[0] = p.x;
      f[1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint4 u;
    if constexpr (sizeof(T) == 4) {
      u.x = __float_as_uint(f[0]);
      u.y = __float_as_uint(f[1]);
      u.z = __float_as_uint(f[2]);
      u.w = __float_as_uint(f[3]);
    } else {
      u.x = pack2<T>(f[0], f[1]);
      u.y = pack2<T>(f[2], f[3]);
      u.z = pack2<T>(f[4], f[5]);
      u.w = pack2<T>(f[6], f[7]);
    }
    return u;
  }
};

// Scene of a packed row: the i with seg[i] <= row < seg[i + 1] (scenes may
// be empty; row < seg[scenes]).
__device__ __forceinline__ int scene_of(const int* seg, int scenes, int row) {
  int lo = 0, hi = scenes;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(seg + mid) <= row) lo = mid; else hi = mid;
  }
  return lo;
}

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

constexpr long long kMaxInt = (1ll << 31) - 1;

// Rows that take 16-byte vectors.
inline bool vector_rows(const feature_rows& t, long long type) {
  const long long size = type == kF32 ? 4 : 2;
  return t.data && ((uintptr_t)t.data & 15) == 0 && t.row * size % 16 == 0 &&
         t.head * size % 16 == 0;
}
inline bool vector_address(const void* p) {
  return p && ((uintptr_t)p & 15) == 0;
}

// The sizes that all attention entries share.
inline bool attention_sizes(const attention_args* a) {
  return a && a->type >= kF32 && a->type <= kBF16 && a->n_q >= 0 &&
         a->n_k >= 0 && a->n_q < kMaxInt && a->n_k < kMaxInt &&
         a->scenes >= 1 && a->scenes < kMaxInt && a->heads >= 1 &&
         a->kv_heads >= 1 && a->heads < (1 << 20) &&
         a->heads % a->kv_heads == 0 && a->dim >= 8 && a->dim <= 128 &&
         a->dim % 8 == 0 && a->n_q * a->heads / 4 < kMaxInt &&
         a->n_k * a->kv_heads / 4 < kMaxInt;
}
inline bool attention_scale(double scale) {
  return scale >= 1. / (1 << 24) && scale <= (double)(1 << 24);
}

}  // namespace gsa
