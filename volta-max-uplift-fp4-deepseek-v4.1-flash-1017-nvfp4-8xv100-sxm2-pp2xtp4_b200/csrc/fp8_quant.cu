// Rows and weights to E4M3 with a scale per block of 128, the limited SwiGLU
// fused in front of the rows' quantizer, its gradient, and the transpose of
// packed weights (the gradient of a product's rows contracts over the weights'
// other axis).
//
// Row blocks are 1 x 128: sixteen lanes hold a block, eight columns each (one
// 16-byte load of 16-bit values), so the maximum is four shuffles and a block
// is read once.  Weight blocks are 128 x 128: a CTA holds one in registers.
// Bound: HBM (f32 or 16-bit columns in, one byte out).
#include <algorithm>

#include "fp8_device.cuh"
#include "internal.h"

namespace b200moe {
namespace {

constexpr int kQuantThreads = 256;

// Limited SwiGLU (the framework's): g = min(gate, limit), u = clamp(up, +-limit), g / (1 + e^-g) * u.
__device__ __forceinline__ float swiglu(float g, float u, float limit) {
  g = g > limit ? limit : g;
  u = u > limit ? limit : u;
  u = u < -limit ? -limit : u;
  return __fmul_rn(__fdiv_rn(g, __fadd_rn(1.f, expf(-g))), u);
}

// Eight values from p, those at or past `left` zero.
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* p, int64_t left, float (&v)[8]) {
  if constexpr (WIDE) {  // whole pieces of eight
    if (left > 0) {
      Vec<T, 8> x;
      x.load(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = x.get(i);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = !WIDE && i < left ? to_f32(p[i]) : 0.f;
}

template <typename T, bool SWIGLU, bool WIDE>
__global__ void __launch_bounds__(kQuantThreads) fp8_rows_kernel(const T* __restrict__ x, int64_t x_stride, int rows,
                                                                 int width, float limit, uint8_t* __restrict__ q,
                                                                 float* __restrict__ scale) {
  const int nb = (width + kFp8Block - 1) / kFp8Block, l = threadIdx.x & 15;
  const int64_t groups = int64_t(rows) * nb, step = int64_t(gridDim.x) * (kQuantThreads / 16);
  pdl_wait();
  pdl_trigger();
  // both halves of a warp take the same number of turns: the shuffles want every lane
  const int64_t turns = (groups + step - 1) / step;
  int64_t gi = int64_t(blockIdx.x) * (kQuantThreads / 16) + threadIdx.x / 16;
  for (int64_t t = 0; t < turns; ++t, gi += step) {
    const bool live = gi < groups;
    const int64_t row = live ? gi / nb : 0;
    const int b = live ? int(gi - row * nb) : 0;
    const int c = b * kFp8Block + l * 8;
    const int64_t left = live ? width - c : 0;
    const T* src = x + row * x_stride + c;
    float v[8];
    load8<T, WIDE>(src, left, v);
    if constexpr (SWIGLU) {
      float u[8];
      load8<T, WIDE>(src + width, left, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = swiglu(v[i], u[i], limit);
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
#pragma unroll
    for (int d = 8; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    const Fp8Scale s = fp8_scale(m);
    const uint32_t lo = e4m3x4(v[0] * s.inv, v[1] * s.inv, v[2] * s.inv, v[3] * s.inv);
    const uint32_t hi = e4m3x4(v[4] * s.inv, v[5] * s.inv, v[6] * s.inv, v[7] * s.inv);
    uint8_t* dst = q + row * width + c;
    if (WIDE) {
      if (left > 0) *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) dst[i] = uint8_t((i < 4 ? lo : hi) >> (8 * (i & 3)));
    }
    if (live && l == 0) scale[gi] = s.scale;
  }
}

// d gate = d u s (1 + g (1 - s)) where gate <= limit, d up = d g s where |up| <= limit, s = 1 / (1 + e^-g).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kQuantThreads) swiglu_grad_kernel(const T* __restrict__ h, int64_t h_stride,
                                                                    const T* __restrict__ grad, int64_t grad_stride,
                                                                    int rows, int width, float limit,
                                                                    T* __restrict__ grad_h) {
  const int per_row = (width + 7) / 8;
  const int64_t n = int64_t(rows) * per_row, step = int64_t(gridDim.x) * kQuantThreads;
  pdl_wait();
  pdl_trigger();
  for (int64_t i0 = int64_t(blockIdx.x) * kQuantThreads + threadIdx.x; i0 < n; i0 += step) {
    const int64_t row = i0 / per_row;
    const int c = int(i0 - row * per_row) * 8;
    const int left = width - c;
    float gate[8], up[8], d[8], dg[8], du[8];
    load8<T, WIDE>(h + row * h_stride + c, left, gate);
    load8<T, WIDE>(h + row * h_stride + width + c, left, up);
    load8<T, WIDE>(grad + row * grad_stride + c, left, d);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float g = gate[i] > limit ? limit : gate[i];
      const float u0 = up[i] > limit ? limit : up[i], u = u0 < -limit ? -limit : u0;
      const float s = __fdiv_rn(1.f, 1.f + expf(-g));
      dg[i] = gate[i] > limit ? 0.f : d[i] * u * (s * (1.f + g * (1.f - s)));
      du[i] = fabsf(up[i]) > limit ? 0.f : d[i] * (g * s);
    }
    T* dst = grad_h + row * 2 * width + c;
    if (WIDE) {
      store_vec<T, 8>(dst, dg);
      store_vec<T, 8>(dst + width, du);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) {
          dst[i] = from_f32<T>(dg[i]);
          dst[width + i] = from_f32<T>(du[i]);
        }
    }
  }
}

// A CTA per 128 x 128 block of one matrix [n][k]; its 64 values per thread stay in registers.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) fp8_weight_kernel(const T* __restrict__ w, int n, int k, uint8_t* __restrict__ q,
                                                         float* __restrict__ scale) {
  __shared__ uint32_t warp_max[8];
  const int kb = blockIdx.x, nb = blockIdx.y;
  const int64_t mat = blockIdx.z;
  const int c = kb * kFp8Block + (threadIdx.x & 15) * 8, r0 = nb * kFp8Block + threadIdx.x / 16;
  pdl_wait();
  pdl_trigger();
  float v[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = r0 + 16 * j;
    load8<T, WIDE>(w + (mat * n + r) * k + c, r < n ? k - c : 0, v[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[j][i]));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, warp_max[j]);
  const Fp8Scale s = fp8_scale(m);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = r0 + 16 * j;
    if (r >= n || c >= k) continue;
    uint32_t o[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      o[h] = e4m3x4(v[j][4 * h] * s.inv, v[j][4 * h + 1] * s.inv, v[j][4 * h + 2] * s.inv, v[j][4 * h + 3] * s.inv);
    uint8_t* dst = q + (mat * n + r) * k + c;
    if (WIDE) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
    } else {
      for (int i = 0; i < 8 && c + i < k; ++i) dst[i] = uint8_t(o[i >> 2] >> (8 * (i & 3)));
    }
  }
  if (threadIdx.x == 0) scale[(mat * gridDim.y + nb) * gridDim.x + kb] = s.scale;
}

// out [k][n] = in [n][k] bytes, a CTA per 128 x 128 tile through shared memory, and the tile's scale.
__global__ void __launch_bounds__(256) fp8_transpose_kernel(const uint8_t* __restrict__ in,
                                                            const float* __restrict__ scale, int n, int k,
                                                            uint8_t* __restrict__ out, float* __restrict__ out_scale) {
  __shared__ uint8_t tile[128][132];  // a column of four-byte words falls in 32 different banks
  const int c0 = blockIdx.x * 128, r0 = blockIdx.y * 128, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t mat = blockIdx.z;
  pdl_wait();
  pdl_trigger();
  const uint8_t* src = in + mat * n * k;
  uint8_t* dst = out + mat * n * k;
  for (int r = warp; r < 128 && r0 + r < n; r += 8) {
    const int c = c0 + lane * 4;
    const uint8_t* p = src + int64_t(r0 + r) * k + c;
    if (k % 4 == 0 && c < k) {
      *reinterpret_cast<uint32_t*>(&tile[r][lane * 4]) = *reinterpret_cast<const uint32_t*>(p);
    } else {
      for (int i = 0; i < 4; ++i)
        if (c + i < k) tile[r][lane * 4 + i] = p[i];
    }
  }
  __syncthreads();
  for (int c = warp; c < 128 && c0 + c < k; c += 8) {
    const int r = r0 + lane * 4;
    uint8_t* p = dst + int64_t(c0 + c) * n + r;
    if (n % 4 == 0 && r < n) {
      uint32_t v = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) v |= uint32_t(tile[lane * 4 + i][c]) << (8 * i);
      *reinterpret_cast<uint32_t*>(p) = v;
    } else {
      for (int i = 0; i < 4; ++i)
        if (r + i < n) p[i] = tile[lane * 4 + i][c];
    }
  }
  if (threadIdx.x == 0)
    out_scale[(mat * gridDim.x + blockIdx.x) * gridDim.y + blockIdx.y] =
        scale[(mat * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x];
}

int status(cudaError_t e) {
  if (e == cudaSuccess) return B200MOE_OK;
  cudaGetLastError();
  return B200MOE_ERR_CUDA;
}

bool wide(const void* p, int64_t stride_bytes, int n) {
  return reinterpret_cast<uintptr_t>(p) % n == 0 && stride_bytes % n == 0;
}

template <typename T, bool SWIGLU>
cudaError_t run_rows(cudaStream_t s, const void* x, int64_t x_stride, int rows, int width, float limit, uint8_t* q,
                     float* scale) {
  const bool w = width % 8 == 0 && wide(x, x_stride * int64_t(sizeof(T)), 16) &&
                 (!SWIGLU || (width * int64_t(sizeof(T))) % 16 == 0) && wide(q, 8, 8);
  const int64_t groups = int64_t(rows) * ((width + kFp8Block - 1) / kFp8Block);
  const int64_t blocks = std::min<int64_t>((groups + kQuantThreads / 16 - 1) / (kQuantThreads / 16), 148 * 16);
  auto kernel = w ? fp8_rows_kernel<T, SWIGLU, true> : fp8_rows_kernel<T, SWIGLU, false>;
  return launch_chain(kernel, dim3(unsigned(blocks)), dim3(kQuantThreads), 0, s, static_cast<const T*>(x), x_stride,
                      rows, width, limit, q, scale);
}

template <typename T>
cudaError_t run_swiglu_grad(cudaStream_t s, const void* h, int64_t h_stride, const void* grad, int64_t grad_stride,
                            int rows, int width, float limit, void* grad_h) {
  const int64_t b = sizeof(T);
  const bool w = width % 8 == 0 && wide(h, h_stride * b, 16) && wide(grad, grad_stride * b, 16) && wide(grad_h, 16, 16);
  const int64_t n = int64_t(rows) * ((width + 7) / 8);
  const int64_t blocks = std::min<int64_t>((n + kQuantThreads - 1) / kQuantThreads, 148 * 16);
  auto kernel = w ? swiglu_grad_kernel<T, true> : swiglu_grad_kernel<T, false>;
  return launch_chain(kernel, dim3(unsigned(blocks)), dim3(kQuantThreads), 0, s, static_cast<const T*>(h), h_stride,
                      static_cast<const T*>(grad), grad_stride, rows, width, limit, static_cast<T*>(grad_h));
}

template <typename T>
cudaError_t run_weight(cudaStream_t s, const void* w, int mats, int n, int k, uint8_t* q, float* scale) {
  const bool wd = k % 8 == 0 && wide(w, 16, 16) && wide(q, 8, 8);
  auto kernel = wd ? fp8_weight_kernel<T, true> : fp8_weight_kernel<T, false>;
  return launch_chain(kernel, dim3((k + 127) / 128, (n + 127) / 128, mats), dim3(256), 0, s,
                      static_cast<const T*>(w), n, k, q, scale);
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_fp8_quantize(void* stream, const void* x, int dtype, int64_t x_stride, int rows, int width,
                                    int swiglu, float limit, void* q, float* scale) {
  if (!x || !q || !scale || rows < 1 || width < 1 || width > (1 << 28) || x_stride < 0 || !(limit > 0.f))
    return B200MOE_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  auto run = dtype == B200MOE_F16    ? (swiglu ? run_rows<__half, true> : run_rows<__half, false>)
             : dtype == B200MOE_BF16 ? (swiglu ? run_rows<__nv_bfloat16, true> : run_rows<__nv_bfloat16, false>)
                                     : (swiglu ? run_rows<float, true> : run_rows<float, false>);
  return status(run(static_cast<cudaStream_t>(stream), x, x_stride, rows, width, limit, static_cast<uint8_t*>(q),
                    scale));
}

extern "C" int b200moe_swiglu_grad(void* stream, const void* h, int dtype, int64_t h_stride, const void* grad,
                                   int64_t grad_stride, int rows, int width, float limit, void* grad_h) {
  if (!h || !grad || !grad_h || rows < 1 || width < 1 || width > (1 << 28) || h_stride < 0 || grad_stride < 0 ||
      !(limit > 0.f))
    return B200MOE_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  auto run = dtype == B200MOE_F16    ? run_swiglu_grad<__half>
             : dtype == B200MOE_BF16 ? run_swiglu_grad<__nv_bfloat16>
                                     : run_swiglu_grad<float>;
  return status(run(static_cast<cudaStream_t>(stream), h, h_stride, grad, grad_stride, rows, width, limit, grad_h));
}

extern "C" int b200moe_fp8_quantize_weight(void* stream, const void* w, int dtype, int mats, int n, int k, void* q,
                                           float* scale) {
  if (!w || !q || !scale || mats < 1 || mats > 65535 || n < 1 || k < 1 || (n + 127) / 128 > 65535)
    return B200MOE_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  auto run = dtype == B200MOE_F16 ? run_weight<__half> : dtype == B200MOE_BF16 ? run_weight<__nv_bfloat16>
                                                                               : run_weight<float>;
  return status(run(static_cast<cudaStream_t>(stream), w, mats, n, k, static_cast<uint8_t*>(q), scale));
}

extern "C" int b200moe_fp8_transpose_weight(void* stream, const void* w, const float* scale, int mats, int n, int k,
                                            void* out, float* out_scale) {
  if (!w || !scale || !out || !out_scale || mats < 1 || mats > 65535 || n < 1 || k < 1 || (n + 127) / 128 > 65535)
    return B200MOE_ERR_INVALID_ARG;
  if ((k % 4 == 0 && reinterpret_cast<uintptr_t>(w) % 4) || (n % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 4))
    return B200MOE_ERR_ALIGN;
  return status(launch_chain(fp8_transpose_kernel, dim3((k + 127) / 128, (n + 127) / 128, mats), dim3(256), 0,
                             static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(w), scale, n, k,
                             static_cast<uint8_t*>(out), out_scale));
}
