// Loads and stores of V consecutive values of f32, f16 or bf16 as f32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace b200moe {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// V values kept as loaded; V = 1 any address, else pieces of at most 16 bytes
// at addresses aligned to the whole vector or to 16 bytes, whichever is less.
template <typename T, int V>
struct Vec {
  static constexpr int kBytes = V * int(sizeof(T));
  static constexpr int kPiece = kBytes < 16 ? kBytes : 16;
  static_assert(kBytes % kPiece == 0, "whole pieces");
  T v[V] __attribute__((aligned(kPiece)));
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) {
      v[0] = *p;
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / kPiece; ++i) {
        if constexpr (kPiece == 16)
          reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
        else if constexpr (kPiece == 8)
          reinterpret_cast<uint2*>(v)[i] = reinterpret_cast<const uint2*>(p)[i];
        else
          reinterpret_cast<uint32_t*>(v)[i] = reinterpret_cast<const uint32_t*>(p)[i];
      }
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 1) {
      *p = v[0];
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / kPiece; ++i) {
        if constexpr (kPiece == 16)
          reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
        else if constexpr (kPiece == 8)
          reinterpret_cast<uint2*>(p)[i] = reinterpret_cast<const uint2*>(v)[i];
        else
          reinterpret_cast<uint32_t*>(p)[i] = reinterpret_cast<const uint32_t*>(v)[i];
      }
    }
  }
  __device__ __forceinline__ float get(int i) const { return to_f32(v[i]); }
};

// Rounded once, to nearest even.
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[V]) {
  Vec<T, V> o;
#pragma unroll
  for (int i = 0; i < V; ++i) o.v[i] = from_f32<T>(x[i]);
  o.store(p);
}

// V columns of a row per thread: WIDE, consecutive ones from c (whole aligned
// vectors); else single ones, `step` apart, those below n. The second form serves
// rows of any width and alignment: neighbouring threads hold neighbouring columns,
// so a warp's access is one run of bytes, and V of them are in flight per thread.
template <bool WIDE, typename T, int V>
__device__ __forceinline__ void load_columns(Vec<T, V>& y, const T* row, int c, int step, int n) {
  if constexpr (WIDE) {
    y.load(row + c);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) y.v[i] = c + i * step < n ? row[c + i * step] : from_f32<T>(0.f);
  }
}
template <bool WIDE, typename T, int V>
__device__ __forceinline__ void store_columns(T* row, int c, int step, int n, const float (&x)[V]) {
  if constexpr (WIDE) {
    store_vec<T, V>(row + c, x);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i * step < n) row[c + i * step] = from_f32<T>(x[i]);
  }
}

}  // namespace b200moe
