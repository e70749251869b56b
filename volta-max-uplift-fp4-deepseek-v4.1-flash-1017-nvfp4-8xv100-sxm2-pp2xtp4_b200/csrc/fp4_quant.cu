// Rows and weights to 4-bit floating point (fp4_rows.cuh), the limited SwiGLU
// fused in front of the rows' quantizer, and the values that records stand for.
//
// A thread holds 16 columns.  NVFP4 needs the row's maximum before its first
// code: a CTA or, of many rows, a warp holds a row in registers, so that it is read
// once; longer rows than a CTA holds are read twice.  MXFP4's blocks stand
// alone and take two threads each, whatever their row.
// Bound: HBM for rows as they are: 16384 x 4096 bf16 MXFP4 30 us (5.8 TB/s), NVFP4 40 (the
// barrier and the quotients), values back 34; instruction issue for the SwiGLU, whose
// exponential and division are f32's own: 49152 x 1408 bf16 MXFP4 87 us, NVFP4 109.
#include <algorithm>

#include "fp4_rows.cuh"
#include "internal.h"

namespace b200moe {
namespace {

constexpr int kMaxRowThreads = 512;

// 16 columns of a row as loaded (SWIGLU: and of the row's second half), and their values.
template <typename T, bool SWIGLU, bool WIDE>
struct Piece {
  Vec<T, 16> a, b;
  __device__ __forceinline__ void load(const T* row, int c, int width) {
    if constexpr (WIDE) {
      a.load(row + c);
      if constexpr (SWIGLU) b.load(row + width + c);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        a.v[i] = row[c + i];
        if constexpr (SWIGLU) b.v[i] = row[width + c + i];
      }
    }
  }
  __device__ __forceinline__ void values(float limit, float (&v)[16]) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      v[i] = a.get(i);
      if constexpr (SWIGLU) v[i] = swiglu(v[i], b.get(i), limit);
    }
  }
};

// A warp per row, its columns in registers as N pieces of 16 a lane: no barrier, for as many rows as keep the GPU's warps
// busy.
template <typename T, bool SWIGLU, bool WIDE, int N>
__global__ void __launch_bounds__(256, N <= 3 ? 3 : 2)
    nvfp4_warp_rows_kernel(const T* __restrict__ x, int64_t x_stride, int rows, int width, float limit,
                           uint8_t* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int64_t row = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  pdl_wait();
  pdl_trigger();
  if (row >= rows) return;
  const int pieces = width / 16;
  float v[N][16], mag[N];
  uint32_t m = 0;
  Piece<T, SWIGLU, WIDE> raw[N];
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (lane + 32 * n < pieces) raw[n].load(x + row * x_stride, (lane + 32 * n) * 16, width);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (lane + 32 * n >= pieces) continue;
    raw[n].values(limit, v[n]);
    mag[n] = magnitude16(v[n]);
    m = max(m, abs_bits(mag[n]));
  }
  const float factor = nvfp4_factor(__reduce_max_sync(0xffffffffu, m));
  uint8_t* rec = out + row * fp4_stride(kNv, width);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int p = lane + 32 * n;
    if (p >= pieces) continue;
    float unit;
    const uint32_t s = nvfp4_scale(mag[n], factor, unit);
    *reinterpret_cast<uint2*>(rec + p * 8) = nvfp4_codes(v[n], unit);
    rec[width / 2 + p] = uint8_t(s);
  }
  if (lane == 0) finish_record(rec, kNv, width, factor);
}

// A CTA walks rows. Where its threads hold all of a row (once), the next row is on its way while this one is worked on.
template <typename T, bool SWIGLU, bool WIDE>
__global__ void __launch_bounds__(kMaxRowThreads, sizeof(T) == 2 ? 2 : 1)
    nvfp4_rows_kernel(const T* __restrict__ x, int64_t x_stride, int rows, int width, float limit,
                      uint8_t* __restrict__ out) {
  __shared__ uint32_t warp_max[2][kMaxRowThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = threadIdx.x, threads = blockDim.x;
  const int pieces = width / 16;
  const bool once = pieces <= threads, in = tid < pieces;
  pdl_wait();
  pdl_trigger();
  constexpr bool kAhead = !SWIGLU;  // what the SwiGLU wants is warps
  Piece<T, SWIGLU, WIDE> next;
  if (kAhead && once && in && blockIdx.x < rows) next.load(x + blockIdx.x * x_stride, tid * 16, width);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const T* src = x + row * x_stride;
    float v[16], top = 0.f;
    uint32_t m = 0;
    if (once) {
      if (in) {
        if (!kAhead) next.load(src, tid * 16, width);
        next.values(limit, v);
        top = magnitude16(v);
        if (kAhead && row + gridDim.x < rows) next.load(src + gridDim.x * x_stride, tid * 16, width);
      }
      m = abs_bits(top);
    } else {
      for (int p = tid; p < pieces; p += threads) {
        next.load(src, p * 16, width);
        next.values(limit, v);
        m = max(m, abs_bits(magnitude16(v)));
      }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) warp_max[turn][warp] = m;  // the places are those of the row before last, which every thread has read
    __syncthreads();
    for (int i = 0; i < threads / 32; ++i) m = max(m, warp_max[turn][i]);
    const float factor = nvfp4_factor(m);
    uint8_t* rec = out + row * fp4_stride(kNv, width);
    for (int p = tid; p < pieces; p += threads) {
      if (!once) {
        next.load(src, p * 16, width);
        next.values(limit, v);
        top = magnitude16(v);
      }
      float unit;
      const uint32_t s = nvfp4_scale(top, factor, unit);
      *reinterpret_cast<uint2*>(rec + p * 8) = nvfp4_codes(v, unit);
      rec[width / 2 + p] = uint8_t(s);
    }
    if (tid == 0) finish_record(rec, kNv, width, factor);
  }
}

// Two neighbouring threads per block of 32 columns of any row.
template <typename T, bool SWIGLU, bool WIDE>
__global__ void __launch_bounds__(256) mxfp4_rows_kernel(const T* __restrict__ x, int64_t x_stride, int rows, int width,
                                                         float limit, uint8_t* __restrict__ out) {
  const int pieces = width / 16, stride = fp4_stride(kMx, width);
  const int64_t total = int64_t(rows) * pieces, step = int64_t(gridDim.x) * blockDim.x;
  pdl_wait();
  pdl_trigger();
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; __any_sync(0xffffffffu, i < total); i += step) {
    const bool in = i < total;  // the same for both threads of a block: pieces is even
    const int64_t row = in ? (i <= INT32_MAX ? int64_t(uint32_t(i) / uint32_t(pieces)) : i / pieces) : 0;
    const int p = in ? int(i - row * pieces) : 0;
    float v[16], inv;
    if (in) {
      Piece<T, SWIGLU, WIDE> piece;
      piece.load(x + row * x_stride, p * 16, width);
      piece.values(limit, v);
    }
    float m = in ? magnitude16(v) : 0.f;
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
    if (!in) continue;
    const uint32_t s = mxfp4_scale(m, inv);
    uint8_t* rec = out + row * stride;
    *reinterpret_cast<uint2*>(rec + p * 8) = mxfp4_codes(v, inv);
    if (!(p & 1)) rec[width / 2 + p / 2] = uint8_t(s);
    if (p == pieces - 1) finish_record(rec, kMx, width, 1.f);
  }
}

// ------------------------------------------------------------------ weights
// Sixteen values from p: by vectors where every address allows it.
template <typename T>
__device__ __forceinline__ void load16(const T* p, int vec, float (&v)[16]) {
  Vec<T, 16> x;
  if (vec) {
    x.load(p);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x.v[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = x.get(i);
}

// Largest magnitude of each matrix, as bits, into its factor's place (zero before).  n: its pieces of 16.
template <typename T>
__global__ void __launch_bounds__(256) fp4_weight_max_kernel(const T* __restrict__ w, int64_t n, int vec,
                                                             uint32_t* __restrict__ top) {
  const T* src = w + int64_t(blockIdx.y) * n * 16;
  uint32_t m = 0;
  pdl_wait();
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    float v[16];
    load16(src + i * 16, vec, v);
    m = max(m, abs_bits(magnitude16(v)));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0 && m) atomicMax(top + blockIdx.y, m);  // a maximum: any order gives the same
  pdl_trigger();
}
__global__ void fp4_weight_factor_kernel(uint32_t* top, int mats) {
  pdl_wait();
  for (int i = threadIdx.x; i < mats; i += blockDim.x) top[i] = __float_as_uint(nvfp4_factor(top[i]));
  pdl_trigger();
}

// A thread per 16 columns of any matrix; codes and scales in arrays of their own.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) fp4_weight_kernel(const T* __restrict__ w, int64_t per_mat, int64_t total, int vec,
                                                         const float* __restrict__ factor, uint8_t* __restrict__ codes,
                                                         uint8_t* __restrict__ scale) {
  pdl_wait();
  pdl_trigger();
  const int64_t step = int64_t(gridDim.x) * 256;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; __any_sync(0xffffffffu, i < total); i += step) {
    const bool in = i < total;
    float v[16], m = 0.f;
    if (in) {
      load16(w + i * 16, vec, v);
      m = magnitude16(v);
    }
    if constexpr (FMT == kMx) {
      float inv;
      m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
      if (!in) continue;
      const uint32_t s = mxfp4_scale(m, inv);
      reinterpret_cast<uint2*>(codes)[i] = mxfp4_codes(v, inv);
      if (!(i & 1)) scale[i / 2] = uint8_t(s);
    } else {
      if (!in) continue;
      float unit;
      scale[i] = uint8_t(nvfp4_scale(m, factor[i / per_mat], unit));
      reinterpret_cast<uint2*>(codes)[i] = nvfp4_codes(v, unit);
    }
  }
}

// ---------------------------------------------------------------- read back
// A value has six bits: times a power of two, as a quantized row's factor is, the product is exact in f32. Times a factor of
// 24 bits, as a pack's, f32 would round it first, for one in 2^14 (f16) or 2^17 (bf16) to a border of the 16-bit type that it
// is not on: so towards zero, with the last bit set where something was cut off, which the type rounds as it would the
// product itself. 16 x 4096 x 4096 to bf16 160 us, with a pack's factors 200 (with a test of each product for a border 178,
// f16 252, and rows pay for it: 16384 x 4096 39 us instead of 35).
__device__ __forceinline__ float product_odd(float value, float factor) {
  const uint32_t cut = __float_as_uint(__fmul_rz(value, factor));
  return __uint_as_float(cut | uint32_t(__fmul_rd(value, factor) < __fmul_ru(value, factor)));
}
// Pieces of 8 columns, neighbouring threads' side by side, four of a thread's in flight: value * scale (exact) * factor,
// rounded once.  d_row, d_piece: the grid's step over rows of width / 8 pieces.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) fp4_values_kernel(const uint8_t* __restrict__ codes, int64_t ld_codes,
                                                         const uint8_t* __restrict__ scale, int64_t ld_scale,
                                                         const uint8_t* __restrict__ factor, int64_t ld_factor,
                                                         int64_t rows, int width, int64_t d_row, int d_piece,
                                                         T* __restrict__ out) {
  constexpr int U = 4;
  const int pieces = width / 8;
  const int64_t first = int64_t(blockIdx.x) * 256 + threadIdx.x;
  int64_t row = first / pieces;
  int p = int(first - row * pieces);
  pdl_wait();
  pdl_trigger();
  while (row < rows) {
    uint32_t w[U], sb[U];
    float f[U];
    int64_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      at[u] = -1;
      if (row < rows) {
        at[u] = row * pieces + p;
        w[u] = __ldg(reinterpret_cast<const uint32_t*>(codes + row * ld_codes) + p);
        sb[u] = __ldg(scale + row * ld_scale + p / (FMT == kMx ? 4 : 2));
        f[u] = factor ? __ldg(reinterpret_cast<const float*>(factor + row * ld_factor)) : 1.f;
      }
      row += d_row;
      p += d_piece;
      if (p >= pieces) {
        p -= pieces;
        ++row;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at[u] < 0) break;
      const float m = FMT == kMx ? e8m0_f32(sb[u]) : e4m3_f32(sb[u]);
      const uint32_t h[4] = {e2m1x2_byte<0>(w[u]), e2m1x2_byte<1>(w[u]), e2m1x2_byte<2>(w[u]), e2m1x2_byte<3>(w[u])};
      float v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&h[k]));
        v[2 * k] = q.x * m;
        v[2 * k + 1] = q.y * m;
      }
      if (sizeof(T) == 4 || FMT == kMx || !(__float_as_uint(f[u]) & 0x7fffffu)) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= f[u];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = product_odd(v[k], f[u]);
      }
      store_vec<T, 8>(out + at[u] * 8, v);
    }
  }
}

int status(cudaError_t e) {
  if (e == cudaSuccess) return B200MOE_OK;
  cudaGetLastError();
  return B200MOE_ERR_CUDA;
}

bool on(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

unsigned grid_of(int64_t threads) { return unsigned(std::min<int64_t>((threads + 255) / 256, int64_t(sm_count()) * 32)); }

template <typename T, bool SWIGLU>
cudaError_t run_rows(cudaStream_t s, int fmt, const void* x, int64_t x_stride, int rows, int width, float limit,
                     uint8_t* out) {
  const bool wide = on(x, 16) && x_stride * int64_t(sizeof(T)) % 16 == 0;
  const T* src = static_cast<const T*>(x);
  if (fmt == kMx) {
    auto kernel = wide ? mxfp4_rows_kernel<T, SWIGLU, true> : mxfp4_rows_kernel<T, SWIGLU, false>;
    return launch_chain(kernel, dim3(grid_of(int64_t(rows) * (width / 16))), dim3(256), 0, s, src, x_stride, rows, width,
                        limit, out);
  }
  // a warp per row where all of a row's pieces fit its lanes' registers and every SM gets eight rows, or a row fits one
  // piece per lane: SwiGLU of 49152 x 1408 takes 109 us so and 132 with a CTA per row
  const int pieces = width / 16, per_lane = (pieces + 31) / 32;
  if (per_lane == 1 || (per_lane <= 4 && rows >= 8 * sm_count())) {
    auto go = [&](auto kernel) {
      const dim3 grid(unsigned((int64_t(rows) + 7) / 8));
      return launch_chain(kernel, grid, dim3(256), 0, s, src, x_stride, rows, width, limit, out);
    };
    if (per_lane == 1)
      return wide ? go(nvfp4_warp_rows_kernel<T, SWIGLU, true, 1>) : go(nvfp4_warp_rows_kernel<T, SWIGLU, false, 1>);
    if (per_lane == 2)
      return wide ? go(nvfp4_warp_rows_kernel<T, SWIGLU, true, 2>) : go(nvfp4_warp_rows_kernel<T, SWIGLU, false, 2>);
    if (per_lane == 3)
      return wide ? go(nvfp4_warp_rows_kernel<T, SWIGLU, true, 3>) : go(nvfp4_warp_rows_kernel<T, SWIGLU, false, 3>);
    return wide ? go(nvfp4_warp_rows_kernel<T, SWIGLU, true, 4>) : go(nvfp4_warp_rows_kernel<T, SWIGLU, false, 4>);
  }
  const int threads = std::min(kMaxRowThreads, (pieces + 31) / 32 * 32);
  auto kernel = wide ? nvfp4_rows_kernel<T, SWIGLU, true> : nvfp4_rows_kernel<T, SWIGLU, false>;
  static Residents residents[2];  // by kernel
  const int64_t grid = std::min<int64_t>(rows, residents[wide].ctas(kernel, threads));
  return launch_chain(kernel, dim3(unsigned(grid)), dim3(threads), 0, s, src, x_stride, rows, width, limit, out);
}

template <typename T>
cudaError_t run_weight(cudaStream_t s, int fmt, const void* w, int mats, int64_t n, uint8_t* codes, uint8_t* scale,
                       float* factor) {
  const T* src = static_cast<const T*>(w);
  const int64_t total = mats * (n / 16);
  const int vec = on(w, 16);
  if (fmt == kMx)
    return launch_chain(fp4_weight_kernel<T, kMx>, dim3(grid_of(total)), dim3(256), 0, s, src, n / 16, total, vec,
                        static_cast<const float*>(nullptr), codes, scale);
  cudaError_t e = cudaMemsetAsync(factor, 0, mats * sizeof(float), s);
  uint32_t* top = reinterpret_cast<uint32_t*>(factor);
  const unsigned per = unsigned(std::min<int64_t>((n + 4095) / 4096, std::max(1, sm_count() * 16 / mats)));
  if (e == cudaSuccess)
    e = launch_chain(fp4_weight_max_kernel<T>, dim3(per, mats), dim3(256), 0, s, src, n / 16, vec, top);
  if (e == cudaSuccess) e = launch_chain(fp4_weight_factor_kernel, dim3(1), dim3(256), 0, s, top, mats);
  if (e == cudaSuccess)
    e = launch_chain(fp4_weight_kernel<T, kNv>, dim3(grid_of(total)), dim3(256), 0, s, src, n / 16, total, vec,
                     static_cast<const float*>(factor), codes, scale);
  return e;
}

template <typename T>
cudaError_t run_values(cudaStream_t s, int fmt, const uint8_t* codes, int64_t ld_codes, const uint8_t* scale,
                       int64_t ld_scale, const uint8_t* factor, int64_t ld_factor, int64_t rows, int width, void* out) {
  auto kernel = fmt == kMx ? fp4_values_kernel<T, kMx> : fp4_values_kernel<T, kNv>;
  const int pieces = width / 8;
  const unsigned grid = grid_of((rows * pieces + 3) / 4);
  const int64_t step = int64_t(grid) * 256;
  return launch_chain(kernel, dim3(grid), dim3(256), 0, s, codes, ld_codes, scale, ld_scale, factor, ld_factor, rows, width,
                      step / pieces, int(step % pieces), static_cast<T*>(out));
}

bool bad_format(int fmt) { return fmt != kNv && fmt != kMx; }

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_fp4_record_bytes(int format, int k) {
  return bad_format(format) || k < 32 || k % 32 || k > (1 << 28) ? 0 : fp4_stride(format, k);
}

extern "C" int b200moe_fp4_quantize(void* stream, const void* x, int dtype, int64_t x_stride, int rows, int k, int format,
                                    int swiglu, float limit, void* records) {
  if (!x || !records || rows < 1 || !b200moe_fp4_record_bytes(format, k) || x_stride < 0 || !(limit > 0.f))
    return B200MOE_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  if (!on(records, 16)) return B200MOE_ERR_ALIGN;
  auto run = dtype == B200MOE_F16    ? (swiglu ? run_rows<__half, true> : run_rows<__half, false>)
             : dtype == B200MOE_BF16 ? (swiglu ? run_rows<__nv_bfloat16, true> : run_rows<__nv_bfloat16, false>)
                                     : (swiglu ? run_rows<float, true> : run_rows<float, false>);
  return status(run(static_cast<cudaStream_t>(stream), format, x, x_stride, rows, k, limit, static_cast<uint8_t*>(records)));
}

extern "C" int b200moe_fp4_quantize_weight(void* stream, const void* w, int dtype, int mats, int n, int k, int format,
                                           void* codes, void* scale, float* factor) {
  if (!w || !codes || !scale || mats < 1 || mats > 65535 || n < 1 || !b200moe_fp4_record_bytes(format, k) ||
      (format == kNv && !factor))
    return B200MOE_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  if (!on(codes, 16)) return B200MOE_ERR_ALIGN;
  auto run = dtype == B200MOE_F16 ? run_weight<__half> : dtype == B200MOE_BF16 ? run_weight<__nv_bfloat16>
                                                                               : run_weight<float>;
  return status(run(static_cast<cudaStream_t>(stream), format, w, mats, int64_t(n) * k, static_cast<uint8_t*>(codes),
                    static_cast<uint8_t*>(scale), factor));
}

extern "C" int b200moe_fp4_values(void* stream, const void* codes, int64_t ld_codes, const void* scale, int64_t ld_scale,
                                  const void* factor, int64_t ld_factor, int64_t rows, int k, int format, void* out,
                                  int dtype) {
  if (!codes || !scale || !out || rows < 1 || !b200moe_fp4_record_bytes(format, k) || ld_codes < 0 || ld_scale < 0 ||
      ld_factor < 0)
    return B200MOE_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  if (!on(codes, 4) || ld_codes % 4 || !on(factor, 4) || ld_factor % 4 || !on(out, 16)) return B200MOE_ERR_ALIGN;
  auto run = dtype == B200MOE_F16 ? run_values<__half> : dtype == B200MOE_BF16 ? run_values<__nv_bfloat16>
                                                                               : run_values<float>;
  return status(run(static_cast<cudaStream_t>(stream), format, static_cast<const uint8_t*>(codes), ld_codes,
                    static_cast<const uint8_t*>(scale), ld_scale, static_cast<const uint8_t*>(factor), ld_factor, rows, k,
                    out));
}
