// Launchers of the E4M3 products with a scale per block of 128.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace b200moe {

// out [S][N] = rows of a [S][K] . w [E][N][K]^T; with offsets [E + 1] (device)
// rows offsets[e] .. offsets[e + 1] use w[e] and rows before offsets[0] and from
// offsets[E] on become zeros, without them E is 1.  K is a multiple of 16, a and w start on 16 bytes.
struct Fp8Product {
  const void* a;
  const float* a_scale;  // [S][ceil(K / 128)]
  int64_t a_scale_stride;
  const void* w;
  const float* w_scale;  // [E][ceil(N / 128)][ceil(K / 128)]
  const int32_t* offsets;
  void* out;
  int S, N, K, E;
};

// tcgen05 kernel (fp8_gemm.cu): tiles of 128 rows
int launch_fp8_gemm(cudaStream_t s, const Fp8Product& p, int out_dtype);
// tcgen05 kernel for few rows per matrix, the weights as the MMA's M (fp8_stream.cu): tiles of 16 or 32 rows
int launch_fp8_stream(cudaStream_t s, const Fp8Product& p, int rows_per_tile, int out_dtype);
// whether a tile's row scales fit in its shared memory
bool fp8_stream_fits(int K, int rows_per_tile);
// kernel for one matrix and at most eight rows (fp8_skinny.cu)
int launch_fp8_skinny(cudaStream_t s, const Fp8Product& p, int out_dtype);
// the same on rows of f16 or bf16 (x [S][K], row stride ldx), quantized in the kernel
int launch_fp8_skinny_x(cudaStream_t s, const Fp8Product& p, const void* x, int x_dtype, int64_t ldx, int out_dtype);
// whether its rows fit in shared memory and its CTAs run in one wave
bool fp8_skinny_fits(const Fp8Product& p);

}  // namespace b200moe
