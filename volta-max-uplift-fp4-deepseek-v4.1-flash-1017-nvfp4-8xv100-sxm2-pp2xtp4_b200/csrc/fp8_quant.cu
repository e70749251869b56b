// Rows and weights to E4M3 with a scale per block of 128, the limited SwiGLU
// fused in front of the rows' quantizer, its gradient, and the transpose of
// packed weights (the gradient of a product's rows contracts over the weights'
// other axis).
//
// Row blocks are 1 x 128: eight lanes hold a block, sixteen columns each (two
// 16-byte loads of 16-bit values), so the maximum is three shuffles and a block
// is read once.  Weight blocks are 128 x 128: a CTA holds one in registers.
// Bound: HBM (f32 or 16-bit columns in, one byte out) for rows as they are: 8192 x
// 4096 bf16 in 18 to 19 us; instruction issue for the SwiGLU: 39 per value with f32's
// own exponential and division, 74 % of the slots, 49152 x 1408 in 96 us (floor 53).
// Its gradient issues 47 per value and takes 115 us (floor 106). The hardware's
// power of two and reciprocal in their place took 66 and 102 us and moved single
// codes off the definition's; launch bounds of five or six CTAs per SM 96 and 106.
#include <algorithm>

#include "fp8_device.cuh"
#include "internal.h"

namespace b200moe {
namespace {

constexpr int kQuantThreads = 256;
constexpr int kQuantBlocks = kQuantThreads / 8;  // row blocks of a CTA's turn
// CTAs at most, for walks of several turns: SwiGLU of 49152 x 1408 takes 97 us with 16 per SM, 102 with 8 and 99
// without a cap, its gradient 113 us with 48 per SM, 128 without a cap and 116 with 16 (115 now, its steps fixed since)
constexpr int64_t kCtaCap = 148 * 16, kGradCap = 148 * 48, kAnyCap = 148 * 32;

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

// Position (row, block) of a walk over rows x blocks in steps of d_row rows and d_b blocks: one division at its start.
struct Walk {
  int64_t row;
  int b;
  __device__ __forceinline__ Walk(int64_t first, int blocks) {
    if (first <= INT32_MAX) {
      row = unsigned(first) / unsigned(blocks);
      b = int(unsigned(first) - unsigned(row) * unsigned(blocks));
    } else {
      row = first / blocks;
      b = int(first - row * blocks);
    }
  }
  __device__ __forceinline__ void next(int d_row, int d_b, int blocks) {
    row += d_row;
    b += d_b;
    if (b >= blocks) {
      b -= blocks;
      ++row;
    }
  }
};

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

// Rows of whole aligned vectors: eight lanes per block, sixteen columns each: what a block costs beside its values (its place, the maximum's
// shuffles, the division) is shared by sixteen values per lane. Several blocks are in flight before the first is
// worked on.
template <typename T, bool SWIGLU>
__host__ __device__ constexpr int blocks_in_flight() {
  return SWIGLU || sizeof(T) == 4 ? 1 : 2;
}

template <typename T, bool SWIGLU>
__global__ void __launch_bounds__(kQuantThreads) fp8_rows_kernel(const T* __restrict__ x, int64_t x_stride, int rows,
                                                                 int width, float limit, int d_row, int d_b,
                                                                 uint8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int U = blocks_in_flight<T, SWIGLU>();
  const int nb = (width + kFp8Block - 1) / kFp8Block, l = threadIdx.x & 7;
  const int64_t step = int64_t(gridDim.x) * kQuantBlocks;
  pdl_wait();
  pdl_trigger();
  // the warp's first block decides: its four take the same turns, as the shuffles want every lane
  const int64_t first = int64_t(blockIdx.x) * kQuantBlocks + threadIdx.x / 8;
  const int64_t groups = int64_t(rows) * nb;
  Walk at(first, nb);
  for (int64_t base = first & ~int64_t(3); base < groups; base += U * step) {
    float v[U][2][8], w[SWIGLU ? U : 1][2][8];
    int64_t row[U];
    int c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      row[u] = at.row;
      c[u] = at.b * kFp8Block + l * 16;
      at.next(d_row, d_b, nb);
      const int64_t left = row[u] < rows ? width - c[u] : 0;
      const T* src = x + row[u] * x_stride + c[u];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load8<T, true>(src + 8 * h, left - 8 * h, v[u][h]);
        if constexpr (SWIGLU) load8<T, true>(src + width + 8 * h, left - 8 * h, w[u][h]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float m = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (SWIGLU) v[u][h][i] = swiglu(v[u][h][i], w[u][h][i], limit);
          m = max_nan(m, fabsf(v[u][h][i]));
        }
#pragma unroll
      for (int d = 4; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
      // both quotients of fp8_scale in one division: even lanes 448 / amax, odd lanes amax / 448
      const float amax = max_nan(m, kAmaxFloor);
      const float ratio = __fdiv_rn(l & 1 ? amax : kE4m3Max, l & 1 ? kE4m3Max : amax);
      const float inv = __shfl_sync(0xffffffffu, ratio, 0, 8);
      if (row[u] >= rows) continue;
      uint8_t* dst = q + row[u] * width + c[u];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float(&y)[8] = v[u][h];
        const uint32_t lo = e4m3x4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        const uint32_t hi = e4m3x4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv);
        if (c[u] + 8 * h < width) *reinterpret_cast<uint2*>(dst + 8 * h) = make_uint2(lo, hi);
      }
      if (l == 1) scale[row[u] * nb + c[u] / kFp8Block] = ratio;
    }
  }
}

// Rows of any width and alignment: a warp per block, single columns 32 apart, so that a warp's access is one run of
// bytes; several blocks in flight.
template <typename T, bool SWIGLU>
__global__ void __launch_bounds__(kQuantThreads) fp8_rows_any_kernel(const T* __restrict__ x, int64_t x_stride, int rows,
                                                                     int width, float limit, int d_row, int d_b,
                                                                     uint8_t* __restrict__ q,
                                                                     float* __restrict__ scale) {
  constexpr int U = SWIGLU ? 2 : 4;
  const int nb = (width + kFp8Block - 1) / kFp8Block, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  Walk at(int64_t(blockIdx.x) * (kQuantThreads / 32) + threadIdx.x / 32, nb);
  while (at.row < rows) {
    Vec<T, 4> v[U], w[SWIGLU ? U : 1];
    int64_t row[U];
    int c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      row[u] = at.row;
      c[u] = at.b * kFp8Block + lane;
      at.next(d_row, d_b, nb);
      const int n = row[u] < rows ? width : 0;
      const T* src = x + row[u] * x_stride;
      load_columns<false>(v[u], src, c[u], 32, n);
      if constexpr (SWIGLU) load_columns<false>(w[u], src + width, c[u], 32, n);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (row[u] >= rows) break;  // the same for the whole warp
      float y[4], m = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = v[u].get(i);
        if constexpr (SWIGLU) y[i] = swiglu(y[i], w[u].get(i), limit);
        m = max_nan(m, fabsf(y[i]));
      }
      const uint32_t amax_bits = __reduce_max_sync(0xffffffffu, abs_bits(m));  // a NaN is above every value
      const float amax = max_nan(__uint_as_float(amax_bits), kAmaxFloor);
      const float ratio = __fdiv_rn(lane & 1 ? amax : kE4m3Max, lane & 1 ? kE4m3Max : amax);
      const float inv = __shfl_sync(0xffffffffu, ratio, 0);
      const uint32_t o = e4m3x4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
      uint8_t* dst = q + row[u] * width;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c[u] + 32 * i < width) dst[c[u] + 32 * i] = uint8_t(o >> (8 * i));
      if (lane == 1) scale[row[u] * nb + c[u] / kFp8Block] = ratio;
    }
  }
}

// d gate = d u (s (1 + g (1 - s))) where gate <= limit, d up = d (g s) where |up| <= limit, s = 1 / (1 + e^-g), one f32
// operation at a time: the bits do not depend on which products the compiler fuses.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kQuantThreads) swiglu_grad_kernel(const T* __restrict__ h, int64_t h_stride,
                                                                    const T* __restrict__ grad, int64_t grad_stride,
                                                                    int rows, int width, float limit, int d_row,
                                                                    int d_b, T* __restrict__ grad_h) {
  // WIDE: a thread's eight consecutive columns; else a warp's 256, eight single ones per thread, 32 apart
  const int per_row = WIDE ? (width + 7) / 8 : (width + 255) / 256, step = WIDE ? 0 : 32;
  const int64_t first = int64_t(blockIdx.x) * kQuantThreads + threadIdx.x;
  pdl_wait();
  pdl_trigger();
  for (Walk at(WIDE ? first : first / 32, per_row); at.row < rows; at.next(d_row, d_b, per_row)) {
    const int c = WIDE ? at.b * 8 : at.b * 256 + (threadIdx.x & 31);
    if (c >= width) continue;
    Vec<T, 8> gate, up, d;
    load_columns<WIDE>(gate, h + at.row * h_stride, c, step, width);
    load_columns<WIDE>(up, h + at.row * h_stride + width, c, step, width);
    load_columns<WIDE>(d, grad + at.row * grad_stride, c, step, width);
    float dg[8], du[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float g0 = gate.get(i), u0 = up.get(i), di = d.get(i);
      const float g = limited_gate(g0, limit), u = limited_up(u0, limit);
      const float s = __frcp_rn(1.f + expf(-g));
      const float slope = __fmul_rn(s, __fadd_rn(1.f, __fmul_rn(g, __fsub_rn(1.f, s))));
      dg[i] = g0 > limit ? 0.f : __fmul_rn(__fmul_rn(di, u), slope);
      du[i] = fabsf(u0) > limit ? 0.f : __fmul_rn(di, __fmul_rn(g, s));
    }
    T* dst = grad_h + at.row * 2 * width;
    store_columns<WIDE>(dst, c, step, width, dg);
    store_columns<WIDE>(dst + width, c, step, width, du);
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
  const int nb = (width + kFp8Block - 1) / kFp8Block;
  const int per_cta = w ? kQuantBlocks : kQuantThreads / 32;
  const int64_t turn = per_cta * (w ? blocks_in_flight<T, SWIGLU>() : SWIGLU ? 2 : 4);
  const int64_t blocks = std::min<int64_t>((int64_t(rows) * nb + turn - 1) / turn, w ? kCtaCap : kAnyCap);
  const int64_t step = blocks * per_cta;
  auto kernel = w ? fp8_rows_kernel<T, SWIGLU> : fp8_rows_any_kernel<T, SWIGLU>;
  return launch_chain(kernel, dim3(unsigned(blocks)), dim3(kQuantThreads), 0, s, static_cast<const T*>(x), x_stride,
                      rows, width, limit, int(step / nb), int(step % nb), q, scale);
}

template <typename T>
cudaError_t run_swiglu_grad(cudaStream_t s, const void* h, int64_t h_stride, const void* grad, int64_t grad_stride,
                            int rows, int width, float limit, void* grad_h) {
  const int64_t b = sizeof(T);
  const bool w = width % 8 == 0 && wide(h, h_stride * b, 16) && wide(grad, grad_stride * b, 16) && wide(grad_h, 16, 16);
  const int per_row = w ? (width + 7) / 8 : (width + 255) / 256, units = w ? kQuantThreads : kQuantThreads / 32;
  const int64_t blocks = std::min<int64_t>((int64_t(rows) * per_row + units - 1) / units, kGradCap);
  const int64_t step = blocks * units;
  auto kernel = w ? swiglu_grad_kernel<T, true> : swiglu_grad_kernel<T, false>;
  return launch_chain(kernel, dim3(unsigned(blocks)), dim3(kQuantThreads), 0, s, static_cast<const T*>(h), h_stride,
                      static_cast<const T*>(grad), grad_stride, rows, width, limit, int(step / per_row),
                      int(step % per_row), static_cast<T*>(grad_h));
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
