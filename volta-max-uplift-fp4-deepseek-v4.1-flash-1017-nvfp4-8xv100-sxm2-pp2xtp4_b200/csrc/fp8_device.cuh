// Device pieces shared by the FP8 (E4M3) kernels: the quantizer's arithmetic
// and the table of an expert-sorted product's tiles.
//
// A value block of 128 columns stands for q * scale with
//   amax = max(max |x|, 1e-30), scale = amax / 448, q = e4m3(x * (448 / amax)),
// every step one IEEE f32 operation and the last a rounding to nearest even:
// 448 is E4M3's largest value, the floor keeps both factors finite and a block
// of zeros zero.  A NaN or an infinity makes its whole block NaN, so that the
// product's rows show it.
#pragma once

#include "common.cuh"
#include "vec.cuh"

namespace b200moe {

constexpr int kFp8Block = 128;
constexpr float kE4m3Max = 448.f;
constexpr float kAmaxFloor = 1e-30f;

// |v| as an integer that orders like the value; NaN above infinity, so a NaN survives the maximum.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Fp8Scale {
  float scale, inv;
};
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t amax_bits) {
  const uint32_t floor_bits = 0x0da24260u;  // 1e-30f
  const float amax = __uint_as_float(max(amax_bits, floor_bits));
  return {__fdiv_rn(amax, kE4m3Max), __fdiv_rn(kE4m3Max, amax)};
}

// Two values to E4M3, v0 in the low byte.  An infinity never gets here: its block's inv is 0.
__device__ __forceinline__ uint32_t e4m3x2(float v0, float v1) {
  uint16_t o;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(o) : "f"(v1), "f"(v0));
  return o;
}
__device__ __forceinline__ uint32_t e4m3x4(float v0, float v1, float v2, float v3) {
  return e4m3x2(v0, v1) | (e4m3x2(v2, v3) << 16);
}

// Tiles of a product whose rows are sorted by expert: expert e has
// ceil(count / rows_per_tile) * per_row_tile tiles, from start[e] on.  Called by
// every thread of the CTA; off and start are shared int [E + 1].  Offsets that
// fall or pass n_rows are cut to what lies inside, and reported.
__device__ __forceinline__ void build_tile_table(const int32_t* __restrict__ offsets, int E, int n_rows,
                                                 int rows_per_tile, int per_row_tile, int* off, int* start,
                                                 uint32_t* err) {
  if (!offsets) {  // one matrix, all rows
    if (threadIdx.x == 0) {
      off[0] = start[0] = 0;
      off[1] = n_rows;
      start[1] = (n_rows + rows_per_tile - 1) / rows_per_tile * per_row_tile;
    }
    __syncthreads();
    return;
  }
  for (int e = threadIdx.x; e <= E; e += blockDim.x) off[e] = offsets[e];
  __syncthreads();
  if (threadIdx.x < 32) {
    int carry = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + threadIdx.x;
      int tiles = 0;
      if (e < E) {
        const int lo = off[e], hi = off[e + 1];
        if (lo < 0 || hi < lo || hi > n_rows)
          set_error(err, kErrBounds);
        else
          tiles = (hi - lo + rows_per_tile - 1) / rows_per_tile * per_row_tile;
      }
      int incl = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, d);
        incl += int(threadIdx.x) >= d ? v : 0;
      }
      if (e < E) start[e] = carry + incl - tiles;
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (threadIdx.x == 0) start[E] = carry;
  }
  __syncthreads();
}

// The expert whose tiles hold item (start[e] <= item < start[e + 1]).
__device__ __forceinline__ int tile_expert(const int* start, int E, int item) {
  int lo = 0, hi = E;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= item)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Rows of out [S][N] without an expert, before the first expert's and past the last one's, are zeros.
template <typename TO>
__device__ __forceinline__ void zero_rows(TO* out, int64_t N, int first, int last, int S, int tid, int threads) {
  const int before = min(max(first, 0), S);
  for (int64_t r = blockIdx.x; r < before; r += gridDim.x)
    for (int64_t c = tid; c < N; c += threads) out[r * N + c] = from_f32<TO>(0.f);
  for (int64_t r = max(last, before) + int64_t(blockIdx.x); r < S; r += gridDim.x)
    for (int64_t c = tid; c < N; c += threads) out[r * N + c] = from_f32<TO>(0.f);
}

}  // namespace b200moe
