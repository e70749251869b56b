// Launchers of the products of 4-bit floating point rows and weights.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace b200moe {

// out [S][N] = rows of a [S][K] . w [E][N][K]^T with their scales and factors; with offsets [E + 1] (device) rows
// offsets[e] .. offsets[e + 1] use w[e] and rows before offsets[0] and from offsets[E] on become zeros, without them E
// is 1.  a: records (fp4_rows.cuh) `stride` bytes apart; w: codes [E][N][K / 2] on 16 bytes, scales [E][N][K / 16 or 32],
// NVFP4 factors [E].  K is a multiple of 32.
struct Fp4Product {
  const uint8_t* a;
  const uint8_t* w;
  const uint8_t* w_scale;
  const float* w_factor;
  const int32_t* offsets;
  void* out;
  int format;
  int S, N, K, E;
};

// tcgen05 kernel (fp4_matmul.cu): rows the MMA's M, tiles of 128 rows x 128 columns
int launch_fp4_tiles(cudaStream_t s, const Fp4Product& p, int out_dtype);
// tcgen05 kernel of pairs of CTAs (fp4_pair.cu): tiles of 256 rows x 256 columns
int launch_fp4_pairs(cudaStream_t s, const Fp4Product& p, int out_dtype);
// the same with the weights as the MMA's M, for few rows per matrix: tiles of 16, 32 or 64 rows x 128 columns
int launch_fp4_stream(cudaStream_t s, const Fp4Product& p, int rows_per_tile, int out_dtype);
// kernel for one matrix and few rows, NVFP4 eight at most, MXFP4 three (fp4_skinny.cu): records, or rows x of f16 or bf16
// (stride ldx) that it quantizes itself
int launch_fp4_skinny(cudaStream_t s, const Fp4Product& p, const void* x, int x_dtype, int64_t ldx, int out_dtype);
// whether its rows fit in shared memory and its CTAs run in one wave
bool fp4_skinny_fits(const Fp4Product& p);
// whether it quantizes rows itself: as many values as its threads hold at once, 16 each. One row of 4096 columns takes 6.3 us
// so, 7.1 by a launch of its own; two, with turns, 7.9 and 7.5
constexpr int kFp4SkinnyThreads = 256;
inline bool fp4_skinny_quantizes(int S, int K) { return int64_t(S) * K <= 16 * kFp4SkinnyThreads; }

}  // namespace b200moe
