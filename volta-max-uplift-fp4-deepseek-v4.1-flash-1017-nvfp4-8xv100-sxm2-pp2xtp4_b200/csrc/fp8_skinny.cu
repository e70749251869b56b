// E4M3 products of at most eight rows with one matrix and a scale per block of
// 128: the weights go straight from global memory into the registers of the
// warps that multiply them. One launch does it all: rows of f16 or bf16 are
// quantized by every CTA for itself (eight rows are little next to the weights).
//
// A warp owns 16 weight rows and every KS-th K block; per block each lane loads
// four 16-byte pieces (rows g and g + 8, columns 16 q .. of each half; g = lane
// / 4, q = lane % 4).  E4M3 values are f16 values, so a word of four becomes the
// operands of an mma.m16n8k16 in f16 by two conversions.  Both operands take the
// columns in the same order, so no value moves between lanes.  The block's
// product leaves the tensor core's accumulator after 128 columns and joins the
// f32 sums times both scales.  The KS warps of a row tile add their sums in
// shared memory in a fixed order.
//
// Bound: latency. All of a small matrix is in flight at once (16.8 MB for 4096 x
// 4096: 8 KB per warp, two CTAs per SM): 6.4 us at one row, 8.0 at eight, where the
// copies and MMAs of the streaming kernel (fp8_stream.cu) take 9.4. It is taken as
// long as all CTAs, of 16 or 32 weight rows, run at once (4736 x 4096: 6.7 us, 9.5
// streamed): CTAs that walk on to a second tile take 9.9 us for 4752 x 4096, streamed 9.5.
#include <algorithm>
#include <atomic>

#include "fp8_device.cuh"
#include "fp8_ops.h"
#include "internal.h"

namespace b200moe {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTokens = 8;
constexpr int kDeep = 4;  // K blocks of a warp in flight
constexpr int kSkinnySmem = 200 * 1024;

__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {  // weights: read once
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

struct SkinnyArgs {
  const uint8_t* a;  // [S][K] E4M3, or the rows to quantize (f16 / bf16, stride ldx)
  int64_t ldx;
  const float* a_scale;
  int64_t lda_s;
  const uint8_t* w;
  const float* w_scale;
  void* out;
  int S, N, K, KB, NB;
};

// The token rows as f16 in shared memory, zeros past S and past K: rows of KB * 256 bytes, 16 bytes apart in the banks
// so that a fragment load's rows do not meet.
__host__ __device__ constexpr int row_pitch(int KB) { return KB * 2 * kFp8Block + 16; }

// Four E4M3 values -> two f16x2 (exact).
__device__ __forceinline__ uint2 e4m3x4_to_f16(uint32_t v) {
  return make_uint2(e4m3x2_to_f16x2(v & 0xffffu), e4m3x2_to_f16x2(v >> 16));
}
__device__ __forceinline__ void store_tokens16(uint8_t* dst, uint4 v) {
  const uint2 a = e4m3x4_to_f16(v.x), b = e4m3x4_to_f16(v.y), c = e4m3x4_to_f16(v.z), d = e4m3x4_to_f16(v.w);
  reinterpret_cast<uint4*>(dst)[0] = make_uint4(a.x, a.y, b.x, b.y);
  reinterpret_cast<uint4*>(dst)[1] = make_uint4(c.x, c.y, d.x, d.y);
}

template <typename TX>
__device__ __forceinline__ void stage_tokens(const SkinnyArgs& A, uint8_t* xs, float* ss) {
  const int pitch = row_pitch(A.KB), pieces = A.KB * 8, live = A.S * pieces;
  for (int i = live + threadIdx.x; i < kTokens * pieces; i += kThreads) {  // rows past S
    const int r = i / pieces, col = (i - r * pieces) * 16;
    store_tokens16(xs + r * pitch + col * 2, make_uint4(0, 0, 0, 0));
    if (col % kFp8Block == 0) ss[r * A.KB + col / kFp8Block] = 0.f;
  }
  // eight lanes hold a block, 16 columns each; whole warps take the same turns
  for (int i0 = threadIdx.x & ~31; i0 < live; i0 += kThreads) {
    const int i = i0 + (threadIdx.x & 31);
    const int r = i < live ? i / pieces : 0, col = i < live ? (i - r * pieces) * 16 : A.K;
    if constexpr (sizeof(TX) == 1) {
      if (i >= live) continue;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (col < A.K) v = __ldg(reinterpret_cast<const uint4*>(A.a + int64_t(r) * A.K + col));
      store_tokens16(xs + r * pitch + col * 2, v);
      if (col % kFp8Block == 0) ss[r * A.KB + col / kFp8Block] = __ldg(A.a_scale + r * A.lda_s + col / kFp8Block);
    } else {
      float v[16];
      uint32_t m = 0;
      Vec<TX, 16> x;
      const bool in = col < A.K;
      if (in) x.load(reinterpret_cast<const TX*>(A.a) + r * A.ldx + col);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        v[j] = in ? x.get(j) : 0.f;
        m = max(m, abs_bits(v[j]));
      }
#pragma unroll
      for (int d = 4; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
      const Fp8Scale s = fp8_scale(m);
      if (i < live) {
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[j] = e4m3x4(v[4 * j] * s.inv, v[4 * j + 1] * s.inv, v[4 * j + 2] * s.inv, v[4 * j + 3] * s.inv);
        store_tokens16(xs + r * pitch + col * 2, make_uint4(o[0], o[1], o[2], o[3]));
        if (col % kFp8Block == 0) ss[r * A.KB + col / kFp8Block] = s.scale;
      }
    }
  }
}

template <typename TX, typename TO, int KS>
__global__ void __launch_bounds__(kThreads, 2) fp8_skinny_kernel(const SkinnyArgs A) {
  constexpr int RT = kWarps / KS;  // 16-row tiles of w per CTA
  __shared__ float red[kWarps][4][32];
  extern __shared__ __align__(16) uint8_t skinny_smem[];
  uint8_t* xs = skinny_smem;                                                     // [8][row_pitch]
  float* ss = reinterpret_cast<float*>(skinny_smem + kTokens * row_pitch(A.KB));  // [8][KB]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int ksub = warp % KS, rsub = warp / KS;
  const int n0 = (blockIdx.x * RT + rsub) * 16;
  const int per_warp = (A.KB + KS - 1) / KS, n_steps = (per_warp + kDeep - 1) / kDeep;
  pdl_wait();

  uint4 w[kDeep][4];
  float fb[kDeep];  // the blocks' weight scales, in flight with them
  auto fetch = [&](int step, int j) {
    const int kb = (step * kDeep + j) * KS + ksub;
    fb[j] = __ldg(A.w_scale + int64_t(min(n0 / kFp8Block, A.NB - 1)) * A.KB + min(kb, A.KB - 1));
    const uint8_t* p = A.w + int64_t(n0 + g) * A.K + kb * kFp8Block + q * 16;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bool in = n0 + g + 8 * h < A.N && kb * kFp8Block + c * 64 + q * 16 < A.K;
        w[j][h * 2 + c] = in ? ld_stream(p + int64_t(8 * h) * A.K + c * 64) : make_uint4(0, 0, 0, 0);
      }
  };

#pragma unroll
  for (int j = 0; j < kDeep; ++j) fetch(0, j);
  stage_tokens<TX>(A, xs, ss);
  __syncthreads();
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int step = 0; step < n_steps; ++step) {
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const int kb = (step * kDeep + j) * KS + ksub;
      if (kb < A.KB) {  // the same for the whole warp
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t lo[4] = {w[j][c].x, w[j][c].y, w[j][c].z, w[j][c].w};
          const uint32_t hi[4] = {w[j][2 + c].x, w[j][2 + c].y, w[j][2 + c].z, w[j][2 + c].w};
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // eight columns of this lane: two MMAs of 16 columns
            const uint2 l0 = e4m3x4_to_f16(lo[2 * h]), l1 = e4m3x4_to_f16(lo[2 * h + 1]);
            const uint2 h0 = e4m3x4_to_f16(hi[2 * h]), h1 = e4m3x4_to_f16(hi[2 * h + 1]);
            const uint4 x = *reinterpret_cast<const uint4*>(
                xs + g * row_pitch(A.KB) + (kb * kFp8Block + c * 64 + q * 16 + h * 8) * 2);
            mma_16816(d, {l0.x, h0.x, l0.y, h0.y}, x.x, x.y);
            mma_16816(d, {l1.x, h1.x, l1.y, h1.y}, x.z, x.w);
          }
        }
        const float* sp = ss + 2 * q * A.KB + kb;
        const float s0 = sp[0] * fb[j], s1 = sp[A.KB] * fb[j];
        acc[0] = fmaf(d[0], s0, acc[0]);
        acc[1] = fmaf(d[1], s1, acc[1]);
        acc[2] = fmaf(d[2], s0, acc[2]);
        acc[3] = fmaf(d[3], s1, acc[3]);
      }
      if (step + 1 < n_steps) fetch(step + 1, j);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[warp][i][lane] = acc[i];
  __syncthreads();
  for (int o = ksub * 32 + lane; o < 16 * kTokens; o += KS * 32) {
    const int t = o >> 4, r = o & 15, col = n0 + r;
    const int slot = (r >> 3) * 2 + (t & 1), src = (r & 7) * 4 + (t >> 1);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) sum += red[rsub * KS + k][slot][src];
    if (t < A.S && col < A.N) static_cast<TO*>(A.out)[int64_t(t) * A.N + col] = from_f32<TO>(sum);
  }
  pdl_trigger();
}

// Eight warps along K where each still has four K blocks, else two row tiles of four warps: one row of 4096 x 4096
// takes 6.4 us with eight and 8.3 with four, of 4096 x 2176 4.2 and 5.0, of 2816 x 2048 3.9 and 3.5.
bool deep(int KB) { return KB > 4 * kDeep; }
int skinny_grid(int N, int KB) {
  const int rows = 16 * (deep(KB) ? 1 : 2);
  return (N + rows - 1) / rows;
}

size_t skinny_smem_bytes(int KB) { return size_t(kTokens) * (row_pitch(KB) + KB * sizeof(float)); }
int skinny_ctas(int KB) { return sm_count() * (skinny_smem_bytes(KB) <= 100 * 1024 ? 2 : 1); }  // that run at once

template <typename TX, typename TO, int KS>
int launch_one(cudaStream_t s, const SkinnyArgs& a) {
  auto kernel = fp8_skinny_kernel<TX, TO, KS>;
  static std::atomic<uint64_t> attr_set{0};  // devices whose attribute is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -1;
  if (!(attr_set.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSkinnySmem) != cudaSuccess)
      return -1;
    attr_set.fetch_or(uint64_t(1) << dev);
  }
  return launch_chain(kernel, dim3(skinny_grid(a.N, a.KB)), dim3(kThreads), skinny_smem_bytes(a.KB), s, a) == cudaSuccess
             ? 0
             : -1;
}

template <typename TX>
int launch_out(cudaStream_t s, const SkinnyArgs& a, int out_dtype) {
  const bool d = deep(a.KB);
  if (out_dtype == B200MOE_F16) return d ? launch_one<TX, __half, 8>(s, a) : launch_one<TX, __half, 4>(s, a);
  if (out_dtype == B200MOE_BF16)
    return d ? launch_one<TX, __nv_bfloat16, 8>(s, a) : launch_one<TX, __nv_bfloat16, 4>(s, a);
  return d ? launch_one<TX, float, 8>(s, a) : launch_one<TX, float, 4>(s, a);
}

SkinnyArgs args_of(const Fp8Product& p) {
  SkinnyArgs a{};
  a.a = static_cast<const uint8_t*>(p.a);
  a.a_scale = p.a_scale;
  a.lda_s = p.a_scale_stride;
  a.w = static_cast<const uint8_t*>(p.w);
  a.w_scale = p.w_scale;
  a.out = p.out;
  a.S = p.S;
  a.N = p.N;
  a.K = p.K;
  a.KB = (p.K + kFp8Block - 1) / kFp8Block;
  a.NB = (p.N + kFp8Block - 1) / kFp8Block;
  return a;
}

}  // namespace

bool fp8_skinny_fits(const Fp8Product& p) {
  const int KB = (p.K + kFp8Block - 1) / kFp8Block;
  return p.E == 1 && !p.offsets && p.S <= kTokens && skinny_smem_bytes(KB) <= size_t(kSkinnySmem) &&
         skinny_grid(p.N, KB) <= skinny_ctas(KB);
}

int launch_fp8_skinny(cudaStream_t s, const Fp8Product& p, int out_dtype) {
  return launch_out<uint8_t>(s, args_of(p), out_dtype);
}

int launch_fp8_skinny_x(cudaStream_t s, const Fp8Product& p, const void* x, int x_dtype, int64_t ldx, int out_dtype) {
  SkinnyArgs a = args_of(p);
  a.a = static_cast<const uint8_t*>(x);
  a.ldx = ldx;
  return x_dtype == B200MOE_F16 ? launch_out<__half>(s, a, out_dtype) : launch_out<__nv_bfloat16>(s, a, out_dtype);
}

}  // namespace b200moe
