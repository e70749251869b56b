// The limited SwiGLU of the row quantizers and its gradient.
#pragma once

#include <cuda_runtime.h>

namespace b200moe {

// Minimum / maximum that keep a NaN.
__device__ __forceinline__ float min_nan(float a, float b) {
  float o;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(o) : "f"(a), "f"(b));
  return o;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float o;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(o) : "f"(a), "f"(b));
  return o;
}

// The limited gate: min(gate, limit), and a finite value for -inf: from -89 down e^-g is infinite in f32 and the SwiGLU
// and its gradient are 0, where -inf itself would give NaN.
__device__ __forceinline__ float limited_gate(float gate, float limit) { return max_nan(min_nan(gate, limit), -128.f); }
__device__ __forceinline__ float limited_up(float up, float limit) { return max_nan(min_nan(up, limit), -limit); }

// Limited SwiGLU (the framework's): g = min(gate, limit), u = clamp(up, +-limit), g / (1 + e^-g) * u.
__device__ __forceinline__ float swiglu(float gate, float up, float limit) {
  const float g = limited_gate(gate, limit);
  return __fdiv_rn(g, 1.f + expf(-g)) * limited_up(up, limit);
}

}  // namespace b200moe
