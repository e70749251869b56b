// Root-mean-square norm of rows after the residual's addition, with the rows
// quantized for the product that follows or as they are, and its gradient:
//
//   s = round(x + r)    rstd = 1 / sqrt(mean(s^2) + eps)    y = (s rstd) w
//   ds = rstd (g - u mean(g u)) + (the sum's own gradient),  g = w dy, u = s rstd
//   dw = sum over rows of dy u
//
// s is rounded to the residual's type once, as it is stored, and the norm is that
// of the stored sum, so the gradient that reads it again is the same function's.
// Sums run in f32.  Where a row's squares pass f32's range the row is scaled by
// 2^-100 first (both are uniform branches that ordinary rows do not take).
//
// Forward: CTAs walk rows (a warp per row up to 512 columns), 16 columns a thread,
// the row kept in registers between its sum and its outputs, so every byte moves
// once, and the next row on its way meanwhile.
// The quantizers take y in f32: 128 columns' maximum for E4M3, the row's for
// NVFP4 (a second sum over the CTA), 32 columns' for MXFP4.
// Backward: a CTA walks rows (rows apart by the grid), holds its columns' part of
// dw in registers, and loads the next row before it works on this one; the parts
// are joined by a second launch in a fixed order, so equal inputs give equal bits.
// Bound: HBM. 16384 x 4096 bf16 with a residual: rows 83 us (6.4 TB/s), E4M3 76, MXFP4 69
// (6.4), NVFP4 91 (4.9: two sums over the CTA, and the codes' quotients), gradient 98
// (5.5). What held it back was instructions: 41 per value forward and 56 backward by
// single conversions and sums read one by one, 109 (NVFP4) and 187 us. The gradient
// with its weights and the sum's gradient a row ahead in registers too: 115, spilled.
// Wider rows hold two or four pieces per thread, and one CTA per SM leaves few warps
// for the memory's latency (5120 columns: 176 registers, 8 % of the warps): the same 67
// million values take, in rows / E4M3 / NVFP4 / MXFP4 / gradient, 137 / 160 / 191 / 99 / 198 us
// at 5120 columns, 111 / 125 / 153 / 125 / 160 at 7168, 104 / 115 / 145 / 114 / 149 at 8192, 109 /
// 130 / 146 / 126 / 198 to 208 at 12288 and 96 / 111 / 126 / 107 / 166 to 174 at 16384.
#include <algorithm>

#include "fp4_rows.cuh"
#include "internal.h"

namespace b200moe {
namespace {

constexpr int kMaxThreads = 256;
constexpr int kMaxWidth = kMaxThreads * 16 * 4;
enum Out { kRows = 0, kFp8 = 1, kNvOut = 2, kMxOut = 3 };

// A thread's columns: WIDE (a width of whole eights), consecutive ones; else single ones 32 apart, so that a warp's access
// is one run of bytes.  The order of a row's sums goes by its width alone: whether WIDE columns move as vectors (vec, where
// every address allows it) changes no bit.

// Eight values by pairs: 16-bit types take one instruction per two of them into the type, one per value out of it.
__device__ __forceinline__ void unpack8(const Vec<float, 8>& x, float* v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = x.v[i];
}
__device__ __forceinline__ void unpack8(const Vec<__nv_bfloat16, 8>& x, float* v) {
  const uint32_t(&u)[4] = reinterpret_cast<const uint32_t(&)[4]>(x.v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(u[i] << 16);
    v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack8(const Vec<__half, 8>& x, float* v) {
  const __half2(&h)[4] = reinterpret_cast<const __half2(&)[4]>(x.v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void pack8(Vec<float, 8>& x, const float* v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x.v[i] = v[i];
}
__device__ __forceinline__ void pack8(Vec<__nv_bfloat16, 8>& x, const float* v) {
  __nv_bfloat162(&h)[4] = reinterpret_cast<__nv_bfloat162(&)[4]>(x.v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void pack8(Vec<__half, 8>& x, const float* v) {
  __half2(&h)[4] = reinterpret_cast<__half2(&)[4]>(x.v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
}

// The thread's 8 PARTS values of a row of T from the warp's first column; zeros past the width.
template <typename T, bool WIDE, int PARTS>
__device__ __forceinline__ void load_raw(const T* row, int base, int lane, int width, int vec, Vec<T, 8> (&v)[PARTS]) {
#pragma unroll
  for (int h = 0; h < PARTS; ++h) {
    if constexpr (WIDE) {
      const int c = base + lane * 8 * PARTS + 8 * h;
      if (c < width && vec) {
        v[h].load(row + c);
      } else if (c < width) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[h].v[i] = row[c + i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[h].v[i] = from_f32<T>(0.f);
      }
    } else {
      load_columns<false>(v[h], row, base + lane + 256 * h, 32, width);
    }
  }
}
template <typename T, bool WIDE, int N>
__device__ __forceinline__ void load_row(const T* row, int base, int lane, int width, int vec, float (&v)[N]) {
  Vec<T, 8> r[N / 8];
  load_raw<T, WIDE>(row, base, lane, width, vec, r);
#pragma unroll
  for (int h = 0; h < N / 8; ++h) unpack8(r[h], v + 8 * h);
}
template <typename T, bool WIDE, int PARTS>
__device__ __forceinline__ void store_raw(T* row, int base, int lane, int width, int vec, const Vec<T, 8> (&v)[PARTS]) {
#pragma unroll
  for (int h = 0; h < PARTS; ++h) {
    const int c = WIDE ? base + lane * 8 * PARTS + 8 * h : base + lane + 256 * h;
    if (WIDE && vec) {
      if (c < width) v[h].store(row + c);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = WIDE ? c + i : c + 32 * i;
        if (at < width) row[at] = v[h].v[i];
      }
    }
  }
}
template <typename T, bool WIDE, int N>
__device__ __forceinline__ void store_row(T* row, int base, int lane, int width, int vec, const float (&v)[N]) {
  Vec<T, 8> r[N / 8];
#pragma unroll
  for (int h = 0; h < N / 8; ++h) pack8(r[h], v + 8 * h);
  store_raw<T, WIDE>(row, base, lane, width, vec, r);
}
// A row of the weight: T, or float where f32 is set.
template <typename T, bool WIDE, int N>
__device__ __forceinline__ void load_weight(const void* p, int f32, int base, int lane, int width, int vec, float (&v)[N]) {
  if (sizeof(T) == 4 || f32)
    load_row<float, WIDE>(static_cast<const float*>(p), base, lane, width, vec, v);
  else
    load_row<T, WIDE>(static_cast<const T*>(p), base, lane, width, vec, v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// The sums over the row's threads, the same bits in each; red: a place of its own for each warp, zeros in those that the CTA
// does not have, that no sum before used since the last barrier.
__device__ __forceinline__ float row_sum(float v, int per_warp, float (&red)[kMaxThreads / 32]) {
  v = warp_sum(v);
  if (per_warp) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  static_assert(kMaxThreads == 256, "eight warps");
  const float4 a = reinterpret_cast<const float4*>(red)[0], b = reinterpret_cast<const float4*>(red)[1];
  return ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
}

constexpr float kFar = 0x1p-100f;  // what a row is scaled by where its squares pass f32

struct NormArgs {
  const void* x;
  int64_t x_stride;
  const void* residual;  // null: none
  int64_t r_stride;
  const void* weight;
  int w_f32;
  float eps;
  int rows, width, per_warp;
  int vec;  // every address on 16 bytes
  void* sum;         // [rows][width], with a residual
  void* y;           // [rows][width] of x's type, or null
  uint8_t* q;        // E4M3 [rows][width], or records
  float* scale;      // E4M3: [rows][ceil(width / 128)]
};

// CTAs per SM that the registers have to leave room for. f32 rows hold twice the registers of 16-bit ones ahead: 8192 x
// 4096 take 105 us with two CTAs and 118 with three, E4M3 81 and 97, 8192 x 2001 E4M3 36 and 67; NVFP4 100 and 97.
// E4M3 of 16-bit rows with an f32 residual, one column at a time, 16384 x 3999: 166 and 251 (rows 150 and 139; with a
// 16-bit residual E4M3 of 16384 x 2001 90 and 87). Two pieces per thread take one: with two, 16-bit rows of 5120
// to 8192 columns take less (rows 83, NVFP4 91 to 99, MXFP4 77 to 83 us; the gradient 152 at 5120 and the same above), f32
// rows more (7168: 217 and 243, gradient 258 and 278).
template <typename T, typename TR, int OUT, bool WIDE, int C>
__host__ __device__ constexpr int norm_ctas() {
  if (C > 1) return 1;
  if (sizeof(T) == 4 && OUT != kNvOut) return 2;
  if (sizeof(TR) == 4 && OUT == kFp8 && !WIDE) return 2;
  return sizeof(TR) == 2 && OUT == kMxOut ? 4 : 3;
}

// T: x's type, TR: the residual's and the sum's.
template <typename T, typename TR, int OUT, bool WIDE, int C>
__global__ void __launch_bounds__(kMaxThreads, norm_ctas<T, TR, OUT, WIDE, C>()) norm_kernel(const NormArgs a) {
  __shared__ __align__(16) float red[3][2][kMaxThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < 3 * 2 * kMaxThreads / 32) (&red[0][0][0])[threadIdx.x] = 0.f;
  if (!a.per_warp) __syncthreads();
  const int warps = a.per_warp ? 1 : blockDim.x / 32, first = a.per_warp ? 0 : warp;
  const int64_t slot = a.per_warp ? int64_t(blockIdx.x) * (blockDim.x / 32) + warp : blockIdx.x;
  const int64_t slots = a.per_warp ? int64_t(gridDim.x) * (blockDim.x / 32) : gridDim.x;
  Vec<T, 8> x[C][2];
  Vec<TR, 8> r[C][2];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int base = (c * warps + first) * 512;
      load_raw<T, WIDE>(static_cast<const T*>(a.x) + row * a.x_stride, base, lane, a.width, a.vec, x[c]);
      if (a.residual)
        load_raw<TR, WIDE>(static_cast<const TR*>(a.residual) + row * a.r_stride, base, lane, a.width, a.vec, r[c]);
    }
  };
  pdl_wait();
  pdl_trigger();
  if (slot < a.rows) fetch(slot);
  int turn = 0;  // the sums' places are those of the row before last, which every thread has read
  for (int64_t row = slot; row < a.rows; row += slots, turn ^= 1) {
    float v[C][16];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int base = (c * warps + first) * 512;
#pragma unroll
      for (int h = 0; h < 2; ++h) unpack8(x[c][h], v[c] + 8 * h);
      if (a.residual) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float add[8];
          unpack8(r[c][h], add);
#pragma unroll
          for (int i = 0; i < 8; ++i) add[i] += v[c][8 * h + i];
          pack8(r[c][h], add);  // the one rounding, as stored
          unpack8(r[c][h], v[c] + 8 * h);
        }
        store_raw<TR, WIDE>(static_cast<TR*>(a.sum) + row * a.width, base, lane, a.width, a.vec, r[c]);
      }
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) part = fmaf(v[c][i], v[c][i], part);
      ss += part;
    }
    if (row + slots < a.rows) fetch(row + slots);
    ss = row_sum(ss, a.per_warp, red[0][turn]);
    float eps = a.eps;
    if (!(ss < INFINITY)) {  // too large for f32, or not finite
      eps = ss = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          v[c][i] *= kFar;
          ss = fmaf(v[c][i], v[c][i], ss);
        }
      ss = row_sum(ss, a.per_warp, red[1][turn]);
    }
    const float rstd = __frsqrt_rn(__fdiv_rn(ss, float(a.width)) + eps);
    uint32_t top = 0;
    float mag[C];  // of each piece
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int base = (c * warps + first) * 512;
      float w[16];
      load_weight<T, WIDE>(a.weight, a.w_f32, base, lane, a.width, a.vec, w);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[c][i] = v[c][i] * rstd * w[i];
      if (a.y) store_row<T, WIDE>(static_cast<T*>(a.y) + row * a.width, base, lane, a.width, a.vec, v[c]);
      if constexpr (OUT == kNvOut) {
        mag[c] = magnitude16(v[c]);
        if (base + lane * 16 < a.width) top = max(top, abs_bits(mag[c]));
      }
    }
    if constexpr (OUT == kFp8) {
      const int nb = (a.width + kFp8Block - 1) / kFp8Block;
      uint8_t* q = a.q + row * a.width;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int base = (c * warps + first) * 512;
        if constexpr (WIDE) {  // eight lanes hold a block
          float m = magnitude16(v[c]);
#pragma unroll
          for (int d = 4; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
          const Fp8Scale s = fp8_scale(abs_bits(m));
          const int col = base + lane * 16;
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[j] = e4m3x4(v[c][4 * j] * s.inv, v[c][4 * j + 1] * s.inv, v[c][4 * j + 2] * s.inv, v[c][4 * j + 3] * s.inv);
          if (col < a.width) *reinterpret_cast<uint2*>(q + col) = make_uint2(o[0], o[1]);
          if (col + 8 < a.width) *reinterpret_cast<uint2*>(q + col + 8) = make_uint2(o[2], o[3]);
          if ((lane & 7) == 0 && col < a.width) a.scale[row * nb + col / kFp8Block] = s.scale;
        } else {  // a warp's four columns of each lane are a block
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = max(m, abs_bits(v[c][4 * b + i]));
            const Fp8Scale s = fp8_scale(__reduce_max_sync(0xffffffffu, m));
            const uint32_t o = e4m3x4(v[c][4 * b] * s.inv, v[c][4 * b + 1] * s.inv, v[c][4 * b + 2] * s.inv,
                                      v[c][4 * b + 3] * s.inv);
            const int col = base + 128 * b + lane;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (col + 32 * i < a.width) q[col + 32 * i] = uint8_t(o >> (8 * i));
            if (lane == 0 && col < a.width) a.scale[row * nb + col / kFp8Block] = s.scale;
          }
        }
      }
    }
    if constexpr (OUT == kNvOut) {
      top = __reduce_max_sync(0xffffffffu, top);
      if (!a.per_warp) {
        uint32_t* tops = reinterpret_cast<uint32_t*>(red[2][turn]);
        if (lane == 0) tops[warp] = top;
        __syncthreads();
        const uint4 t0 = reinterpret_cast<const uint4*>(tops)[0], t1 = reinterpret_cast<const uint4*>(tops)[1];
        top = max(max(max(t0.x, t0.y), max(t0.z, t0.w)), max(max(t1.x, t1.y), max(t1.z, t1.w)));
      }
      const float factor = nvfp4_factor(top);
      uint8_t* rec = a.q + row * fp4_stride(kNv, a.width);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int col = (c * warps + first) * 512 + lane * 16;
        if (col >= a.width) continue;
        float unit;
        const uint32_t s = nvfp4_scale(mag[c], factor, unit);
        *reinterpret_cast<uint2*>(rec + col / 2) = nvfp4_codes(v[c], unit);
        rec[a.width / 2 + col / 16] = uint8_t(s);
      }
      if (first == 0 && lane == 0) finish_record(rec, kNv, a.width, factor);
    }
    if constexpr (OUT == kMxOut) {
      uint8_t* rec = a.q + row * fp4_stride(kMx, a.width);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int col = (c * warps + first) * 512 + lane * 16;
        float m = magnitude16(v[c]), inv;
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
        if (col >= a.width) continue;
        const uint32_t s = mxfp4_scale(m, inv);
        *reinterpret_cast<uint2*>(rec + col / 2) = mxfp4_codes(v[c], inv);
        if (!(lane & 1)) rec[a.width / 2 + col / 32] = uint8_t(s);
      }
      if (first == 0 && lane == 0) finish_record(rec, kMx, a.width, 1.f);
    }
  }
}

// ----------------------------------------------------------------- gradient
struct GradArgs {
  const void* s;  // the stored sum (or x)
  int64_t s_stride;
  const void* dy;  // T
  int64_t dy_stride;
  const void* ds;  // the sum's own gradient, of the sum's type, or null
  int64_t ds_stride;
  const void* weight;
  int w_f32;
  float eps;
  int rows, width, per_warp;
  int vec;  // every address on 16 bytes
  void* grad_x;    // T, or null
  void* grad_sum;  // the sum's type, or null
  float* parts;    // [slots][width], or null
};

// T: x's and grad_y's type, TS: the sum's.
template <typename T, typename TS, bool WIDE, int C>
__global__ void __launch_bounds__(kMaxThreads, C == 1 ? 2 : 1) norm_grad_kernel(const GradArgs a) {
  __shared__ __align__(16) float2 red[2][kMaxThreads / 32];
  __shared__ __align__(16) float far[2][kMaxThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int warps = a.per_warp ? 1 : blockDim.x / 32, first = a.per_warp ? 0 : warp;
  const int64_t slot = a.per_warp ? int64_t(blockIdx.x) * (blockDim.x / 32) + warp : blockIdx.x;
  const int64_t slots = a.per_warp ? int64_t(gridDim.x) * (blockDim.x / 32) : gridDim.x;
  if (threadIdx.x < 2 * kMaxThreads / 32) {
    (&red[0][0])[threadIdx.x] = make_float2(0.f, 0.f);
    (&far[0][0])[threadIdx.x] = 0.f;
  }
  if (!a.per_warp) __syncthreads();
  // 16-bit rows stay as loaded, so that two of them fit in the registers; f32 rows are fetched when their turn comes
  constexpr bool kAhead = C == 1 && sizeof(TS) == 2;
  float dw[C][16];
  Vec<TS, 8> rs[C][2];
  Vec<T, 8> ry[C][2];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int base = (c * warps + first) * 512;
      load_raw<TS, WIDE>(static_cast<const TS*>(a.s) + row * a.s_stride, base, lane, a.width, a.vec, rs[c]);
      load_raw<T, WIDE>(static_cast<const T*>(a.dy) + row * a.dy_stride, base, lane, a.width, a.vec, ry[c]);
    }
  };
  pdl_wait();
  pdl_trigger();
  if (kAhead && slot < a.rows) fetch(slot);
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) dw[c][i] = 0.f;
  const float inv_width = __fdiv_rn(1.f, float(a.width));
  int turn = 0;
  for (int64_t row = slot; row < a.rows; row += slots, turn ^= 1) {  // the same turns for every thread of a row
    if (!kAhead) fetch(row);
    float u[C][16];  // s
    Vec<TS, 8> cd[C][2];
    Vec<T, 8> cy[C][2];
    if (a.ds) {
#pragma unroll
      for (int c = 0; c < C; ++c)  // wanted behind the sums
        load_raw<TS, WIDE>(static_cast<const TS*>(a.ds) + row * a.ds_stride, (c * warps + first) * 512, lane, a.width, a.vec,
                           cd[c]);
    }
    float ss = 0.f, dot = 0.f;
    auto weights = [&](int c, float(&w)[16]) {  // from L1 where they are used: registers hold rows on their way
      load_weight<T, WIDE>(a.weight, a.w_f32, (c * warps + first) * 512, lane, a.width, a.vec, w);
    };
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float w[16], dy[16], part = 0.f, part_dot = 0.f;
      weights(c, w);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        unpack8(rs[c][h], u[c] + 8 * h);
        unpack8(ry[c][h], dy + 8 * h);
        cy[c][h] = ry[c][h];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        part = fmaf(u[c][i], u[c][i], part);
        part_dot = fmaf(dy[i] * w[i], u[c][i], part_dot);
      }
      ss += part;
      dot += part_dot;
    }
    if (kAhead && row + slots < a.rows) fetch(row + slots);
    // both sums at once; the places are those of the row before last, which every thread has read
    ss = warp_sum(ss);
    dot = warp_sum(dot);
    if (!a.per_warp) {
      if (lane == 0) red[turn][warp] = make_float2(ss, dot);
      __syncthreads();
      static_assert(kMaxThreads == 256, "eight warps");
      const float4* r = reinterpret_cast<const float4*>(red[turn]);
      const float4 r0 = r[0], r1 = r[1], r2 = r[2], r3 = r[3];
      ss = ((r0.x + r0.z) + (r1.x + r1.z)) + ((r2.x + r2.z) + (r3.x + r3.z));
      dot = ((r0.y + r0.w) + (r1.y + r1.w)) + ((r2.y + r2.w) + (r3.y + r3.w));
    }
    float k = 1.f, rstd = __frsqrt_rn(__fmul_rn(ss, inv_width) + a.eps);
    float mean = dot * rstd * inv_width;  // of g u
    if (!(ss < INFINITY) || !(fabsf(dot) < INFINITY)) {
      float s2 = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) s2 = fmaf(u[c][i] * kFar, u[c][i] * kFar, s2);
      if (!a.per_warp) __syncthreads();  // the places' last readers
      s2 = row_sum(s2, a.per_warp, far[0]);
      if (!(ss < INFINITY)) {
        k = kFar;
        rstd = __frsqrt_rn(__fmul_rn(s2, inv_width));
      }
      dot = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float w[16], dy[16];
        weights(c, w);
#pragma unroll
        for (int h = 0; h < 2; ++h) unpack8(cy[c][h], dy + 8 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) dot = fmaf(dy[i] * w[i], u[c][i] * k * rstd, dot);
      }
      mean = row_sum(dot, a.per_warp, far[1]) * inv_width;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) u[c][i] *= k;
    }
    const float scale = rstd * k;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int base = (c * warps + first) * 512;
      float d[16], dy[16], w[16];
      weights(c, w);
#pragma unroll
      for (int h = 0; h < 2; ++h) unpack8(cy[c][h], dy + 8 * h);
      if (a.ds) {
#pragma unroll
        for (int h = 0; h < 2; ++h) unpack8(cd[c][h], d + 8 * h);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) d[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float n = u[c][i] * rstd;
        dw[c][i] = fmaf(dy[i], n, dw[c][i]);
        d[i] = fmaf(scale, fmaf(-n, mean, dy[i] * w[i]), d[i]);
      }
      if (a.grad_sum) store_row<TS, WIDE>(static_cast<TS*>(a.grad_sum) + row * a.width, base, lane, a.width, a.vec, d);
      if (a.grad_x) store_row<T, WIDE>(static_cast<T*>(a.grad_x) + row * a.width, base, lane, a.width, a.vec, d);
    }
  }
  if (a.parts) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      store_row<float, WIDE>(a.parts + slot * a.width, (c * warps + first) * 512, lane, a.width, a.vec, dw[c]);
  }
}

// dw[column] = sum over the slots in a fixed order: 32 columns per CTA, 32 runs of slots, joined by a tree.
template <typename TW>
__global__ void __launch_bounds__(1024) norm_parts_kernel(const float* __restrict__ parts, int64_t slots, int width,
                                                          TW* __restrict__ out) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  pdl_wait();
  pdl_trigger();
  float v = 0.f;
  if (col < width)
    for (int64_t p = run; p < slots; p += 32) v += parts[p * width + col];
  sums[run][lane] = v;
  __syncthreads();
  if (run == 0 && col < width) {
    float t[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) t[i] = sums[i][lane];
#pragma unroll
    for (int d = 16; d; d >>= 1)
#pragma unroll
      for (int i = 0; i < d; ++i) t[i] += t[i + d];
    out[col] = from_f32<TW>(t[0]);
  }
}

int status(cudaError_t e) {
  if (e == cudaSuccess) return B200MOE_OK;
  cudaGetLastError();
  return B200MOE_ERR_CUDA;
}

bool whole(const void* p, int64_t stride, int size) {  // null, or rows on 16 bytes
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0;
}

// How a row's threads are laid out: a warp per row (8 rows per CTA), or a CTA per row with C pieces of 16 per thread.
struct Shape {
  int per_warp, threads, pieces;
};
Shape shape_of(int width) {
  if (width <= 512) return {1, 256, 1};
  const int c = width <= kMaxThreads * 16 ? 1 : width <= kMaxThreads * 32 ? 2 : 4;
  return {0, (width + 512 * c - 1) / (512 * c) * 32, c};
}

template <typename T, typename TR, int OUT>
cudaError_t run_norm(cudaStream_t s, const NormArgs& a, const Shape& sh) {
  static Residents residents[6];  // by kernel
  auto go = [&](auto kernel, int which) {
    const int64_t most = a.per_warp ? (int64_t(a.rows) + 7) / 8 : a.rows;
    const int64_t grid = std::min(most, residents[which].ctas(kernel, sh.threads));
    return launch_chain(kernel, dim3(unsigned(grid)), dim3(sh.threads), 0, s, a);
  };
  if constexpr (OUT == kRows || OUT == kFp8) {  // 4-bit rows have whole blocks of 32 columns
    if (a.width % 8)
      return sh.pieces == 1   ? go(norm_kernel<T, TR, OUT, false, 1>, 0)
             : sh.pieces == 2 ? go(norm_kernel<T, TR, OUT, false, 2>, 1)
                              : go(norm_kernel<T, TR, OUT, false, 4>, 2);
  }
  return sh.pieces == 1   ? go(norm_kernel<T, TR, OUT, true, 1>, 3)
         : sh.pieces == 2 ? go(norm_kernel<T, TR, OUT, true, 2>, 4)
                          : go(norm_kernel<T, TR, OUT, true, 4>, 5);
}

template <typename T, typename TR>
cudaError_t run_out(cudaStream_t s, const NormArgs& a, const Shape& sh, int out) {
  return out == kRows    ? run_norm<T, TR, kRows>(s, a, sh)
         : out == kFp8   ? run_norm<T, TR, kFp8>(s, a, sh)
         : out == kNvOut ? run_norm<T, TR, kNvOut>(s, a, sh)
                         : run_norm<T, TR, kMxOut>(s, a, sh);
}

// CTAs of a gradient's walk, at most one per row: their number fixes the order of the weight's gradient and its
// workspace, so it goes by sizes alone and not by what runs at once.
int64_t grad_grid(int rows, const Shape& sh) {
  const int64_t per_sm = std::max(1, 512 / sh.threads);
  const int64_t rows_per_cta = sh.per_warp ? sh.threads / 32 : 1;
  return std::min<int64_t>((rows + rows_per_cta - 1) / rows_per_cta, per_sm * sm_count());
}

template <typename T, typename TS>
cudaError_t run_grad(cudaStream_t s, const GradArgs& a, const Shape& sh) {
  auto go = [&](auto kernel) {
    return launch_chain(kernel, dim3(unsigned(grad_grid(a.rows, sh))), dim3(sh.threads), 0, s, a);
  };
  if (a.width % 8 == 0)
    return sh.pieces == 1   ? go(norm_grad_kernel<T, TS, true, 1>)
           : sh.pieces == 2 ? go(norm_grad_kernel<T, TS, true, 2>)
                            : go(norm_grad_kernel<T, TS, true, 4>);
  return sh.pieces == 1   ? go(norm_grad_kernel<T, TS, false, 1>)
         : sh.pieces == 2 ? go(norm_grad_kernel<T, TS, false, 2>)
                          : go(norm_grad_kernel<T, TS, false, 4>);
}

template <typename TW>
cudaError_t join(cudaStream_t s, const float* parts, int64_t slots, int width, void* out) {
  return launch_chain(norm_parts_kernel<TW>, dim3((width + 31) / 32), dim3(1024), 0, s, parts, slots, width,
                      static_cast<TW*>(out));
}

bool bad_sizes(int rows, int width, float eps) {
  return rows < 1 || width < 1 || width > kMaxWidth || !(eps >= 1e-20f) || !(eps < INFINITY);
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_rms_norm(void* stream, const void* x, int dtype, int64_t x_stride, const void* residual,
                                int residual_f32, int64_t residual_stride, const void* weight, int weight_f32, float eps,
                                int rows, int width, void* sum, void* y, int out, void* q, float* scale) {
  if (!x || !weight || bad_sizes(rows, width, eps) || x_stride < 0 || residual_stride < 0 || (residual && !sum) ||
      out < kRows || out > kMxOut || (out == kRows ? !y : !q) || (out == kFp8 && !scale) ||
      (out >= kNvOut && width % 32))
    return B200MOE_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  const int b = dtype == B200MOE_F32 ? 4 : 2, rb = residual_f32 ? 4 : b, wb = weight_f32 ? 4 : b;
  const Shape sh = shape_of(width);
  if (!whole(q, 0, 1)) return B200MOE_ERR_ALIGN;
  const int vec = whole(x, x_stride, b) && whole(residual, residual_stride, rb) && whole(weight, 0, wb) &&
                  whole(sum, width, rb) && whole(y, width, b);
  const NormArgs a{x,   x_stride, residual, residual_stride, weight, weight_f32, eps, rows, width, sh.per_warp,
                   vec, sum,      y,        static_cast<uint8_t*>(q), scale};
  const bool far = residual_f32 && residual;  // a residual of another type than 16-bit rows
  auto run = dtype == B200MOE_F16    ? (far ? run_out<__half, float> : run_out<__half, __half>)
             : dtype == B200MOE_BF16 ? (far ? run_out<__nv_bfloat16, float> : run_out<__nv_bfloat16, __nv_bfloat16>)
                                     : run_out<float, float>;
  return status(run(static_cast<cudaStream_t>(stream), a, sh, out));
}

extern "C" size_t b200moe_rms_norm_grad_workspace_bytes(int rows, int width) {
  if (bad_sizes(rows, width, 1.f)) return 0;
  const Shape sh = shape_of(width);
  return size_t(grad_grid(rows, sh)) * (sh.per_warp ? sh.threads / 32 : 1) * width * sizeof(float);
}

extern "C" int b200moe_rms_norm_grad(void* stream, const void* s, int s_f32, int64_t s_stride, const void* grad_y,
                                     int dtype, int64_t grad_y_stride, const void* grad_s, int64_t grad_s_stride,
                                     const void* weight, int weight_f32, float eps, int rows, int width, void* grad_x,
                                     void* grad_sum, void* grad_weight, void* workspace, size_t workspace_bytes) {
  if (!s || !grad_y || !weight || bad_sizes(rows, width, eps) || s_stride < 0 || grad_y_stride < 0 || grad_s_stride < 0)
    return B200MOE_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  const Shape sh = shape_of(width);
  const int64_t slots = grad_grid(rows, sh) * (sh.per_warp ? sh.threads / 32 : 1);
  if (grad_weight && (!workspace || workspace_bytes < size_t(slots) * width * sizeof(float)))
    return B200MOE_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return B200MOE_ERR_ALIGN;
  const int b = dtype == B200MOE_F32 ? 4 : 2, sb = s_f32 ? 4 : b, wb = weight_f32 ? 4 : b;
  const int vec = whole(s, s_stride, sb) && whole(grad_y, grad_y_stride, b) && whole(grad_s, grad_s_stride, sb) &&
                  whole(weight, 0, wb) && whole(grad_x, width, b) && whole(grad_sum, width, sb);
  float* parts = grad_weight ? static_cast<float*>(workspace) : nullptr;
  const GradArgs a{s, s_stride, grad_y, grad_y_stride, grad_s, grad_s_stride, weight, weight_f32, eps, rows, width,
                   sh.per_warp, vec, grad_x, grad_sum, parts};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = dtype == B200MOE_F16    ? (s_f32 ? run_grad<__half, float> : run_grad<__half, __half>)
             : dtype == B200MOE_BF16 ? (s_f32 ? run_grad<__nv_bfloat16, float> : run_grad<__nv_bfloat16, __nv_bfloat16>)
                                     : run_grad<float, float>;
  cudaError_t e = run(st, a, sh);
  if (e == cudaSuccess && grad_weight)
    e = weight_f32 || dtype == B200MOE_F32 ? join<float>(st, parts, slots, width, grad_weight)
        : dtype == B200MOE_F16             ? join<__half>(st, parts, slots, width, grad_weight)
                                           : join<__nv_bfloat16>(st, parts, slots, width, grad_weight);
  return status(e);
}
