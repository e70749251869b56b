// E4M3 products of few rows with a scale per block of 128: the weights are read
// once, straight from global memory into the registers of the warps that
// multiply them.
//
// A warp owns 16 weight rows and every KS-th K block; per block each lane loads
// four 16-byte pieces (rows g and g + 8, columns 16 q .. of each half; g = lane
// / 4, q = lane % 4).  Both operands of mma.m16n8k32 take the columns in the
// same order, so a piece's four words are the K groups of two MMAs with no
// shuffle, and tokens are loaded by the same pattern (token g).  The block's
// product leaves the tensor core's accumulator after 128 columns and joins the
// f32 sums times both scales.  The KS warps of a row tile add their sums in
// shared memory in a fixed order.
//
// Bound: the weight bytes.  A warp refills the registers of a K block as soon as
// its MMAs have read them, with the next item's block, so 8 KB per warp stay in
// flight across items and no barrier is waited for by a load.
#include <algorithm>
#include <atomic>

#include "fp8_device.cuh"
#include "fp8_ops.h"
#include "internal.h"

namespace b200moe {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxExperts = 1024;
constexpr int kDeep = 4;  // K blocks of a warp in flight

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {  // weights: read once
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
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
  const int32_t* offsets;
  void* out;
  int S, N, K, E, KB, NB;
  uint32_t* err;
};

// One K block of the tokens as MMA operands: words of columns 128 kb + 64 c + 16 q.
template <typename TX>
struct Tokens {  // quantized here: four lanes hold a token's block
  float scale;
  uint32_t b[2][4];
  __device__ __forceinline__ void load(const SkinnyArgs& A, int row, int end, int kb, int q) {
    float v[2][16];
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int col = kb * kFp8Block + c * 64 + q * 16;
      Vec<TX, 16> x;
      const bool in = row < end && col < A.K;
      if (in) x.load(reinterpret_cast<const TX*>(A.a) + row * A.ldx + col);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        v[c][i] = in ? x.get(i) : 0.f;
        m = max(m, abs_bits(v[c][i]));
      }
    }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const Fp8Scale s = fp8_scale(m);
    scale = s.scale;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        b[c][j] = e4m3x4(v[c][4 * j] * s.inv, v[c][4 * j + 1] * s.inv, v[c][4 * j + 2] * s.inv, v[c][4 * j + 3] * s.inv);
  }
  // scales of tokens 2 q and 2 q + 1, held by the lanes of those tokens
  __device__ __forceinline__ void scales(const SkinnyArgs&, int, int, int, int q, float& s0, float& s1) const {
    s0 = __shfl_sync(0xffffffffu, scale, 8 * q);
    s1 = __shfl_sync(0xffffffffu, scale, 8 * q + 4);
  }
};
template <>
struct Tokens<uint8_t> {
  uint32_t b[2][4];
  __device__ __forceinline__ void load(const SkinnyArgs& A, int row, int end, int kb, int q) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int col = kb * kFp8Block + c * 64 + q * 16;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row < end && col < A.K) v = __ldg(reinterpret_cast<const uint4*>(A.a + int64_t(row) * A.K + col));
      b[c][0] = v.x;
      b[c][1] = v.y;
      b[c][2] = v.z;
      b[c][3] = v.w;
    }
  }
  __device__ __forceinline__ void scales(const SkinnyArgs& A, int row0, int end, int kb, int q, float& s0,
                                         float& s1) const {
    const int r = row0 + 2 * q;
    s0 = r < end ? __ldg(A.a_scale + r * A.lda_s + kb) : 0.f;
    s1 = r + 1 < end ? __ldg(A.a_scale + (r + 1) * A.lda_s + kb) : 0.f;
  }
};

template <typename TX, typename TO, int NT, int KS>
__global__ void __launch_bounds__(kThreads, NT <= 2 ? 2 : 1) fp8_skinny_kernel(const SkinnyArgs A) {
  constexpr int RT = kWarps / KS;  // 16-row tiles of w per item
  constexpr int TOK = 8 * NT;
  __shared__ int off[kMaxExperts + 1], start[kMaxExperts + 1];
  __shared__ float red[2][kWarps][NT * 4][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int ksub = warp % KS, rsub = warp / KS;
  const int n_wt = (A.N + 16 * RT - 1) / (16 * RT);
  pdl_wait();
  build_tile_table(A.offsets, A.E, A.S, TOK, n_wt, off, start, A.err);
  const int n_items = start[A.E];
  const int per_warp = (A.KB + KS - 1) / KS, n_steps = (per_warp + kDeep - 1) / kDeep;

  struct Item {
    int e, row0, end, n0;
  };
  auto item_of = [&](int item) {
    Item t;
    t.e = tile_expert(start, A.E, item);
    const int local = item - start[t.e], m_tiles = (start[t.e + 1] - start[t.e]) / n_wt;
    t.row0 = off[t.e] + local % m_tiles * TOK;  // an expert's row tiles are neighbours: they share its weights
    t.end = off[t.e + 1];
    t.n0 = (local / m_tiles * RT + rsub) * 16;
    return t;
  };
  uint4 w[kDeep][4];
  auto fetch = [&](const Item& t, int step, int j) {
    const int kb = (step * kDeep + j) * KS + ksub;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = t.n0 + g + 8 * h, col = kb * kFp8Block + c * 64 + q * 16;
        w[j][h * 2 + c] = row < A.N && col < A.K ? ld_stream(A.w + (int64_t(t.e) * A.N + row) * A.K + col)
                                                 : make_uint4(0, 0, 0, 0);
      }
  };

  int item = blockIdx.x;
  Item cur{};
  if (item < n_items) {
    cur = item_of(item);
#pragma unroll
    for (int j = 0; j < kDeep; ++j) fetch(cur, 0, j);
  }
  int flip = 0;
  for (; item < n_items; item += gridDim.x, flip ^= 1) {
    const int next_item = item + gridDim.x;
    Item nxt{};
    if (next_item < n_items) nxt = item_of(next_item);
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
    const float* sb = A.w_scale + (int64_t(cur.e) * A.NB + min(cur.n0 / kFp8Block, A.NB - 1)) * A.KB;
    for (int step = 0; step < n_steps; ++step) {
      const bool last = step + 1 == n_steps;
#pragma unroll
      for (int j = 0; j < kDeep; ++j) {
        const int kb = (step * kDeep + j) * KS + ksub;
        if (kb < A.KB) {  // the same for the whole warp
          const float fb = __ldg(sb + kb);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            Tokens<TX> x;
            x.load(A, cur.row0 + 8 * n + g, cur.end, kb, q);
            float s0, s1;
            x.scales(A, cur.row0 + 8 * n, cur.end, kb, q, s0, s1);
            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint4 lo = w[j][c], hi = w[j][2 + c];
              mma_e4m3(d, lo.x, hi.x, lo.y, hi.y, x.b[c][0], x.b[c][1]);
              mma_e4m3(d, lo.z, hi.z, lo.w, hi.w, x.b[c][2], x.b[c][3]);
            }
            s0 *= fb;
            s1 *= fb;
            acc[n][0] = fmaf(d[0], s0, acc[n][0]);
            acc[n][1] = fmaf(d[1], s1, acc[n][1]);
            acc[n][2] = fmaf(d[2], s0, acc[n][2]);
            acc[n][3] = fmaf(d[3], s1, acc[n][3]);
          }
        }
        if (!last)
          fetch(cur, step + 1, j);
        else if (next_item < n_items)
          fetch(nxt, 0, j);
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[flip][warp][n * 4 + i][lane] = acc[n][i];
    __syncthreads();  // the other buffer's readers have passed the last item's barrier
    for (int o = ksub * 32 + lane; o < 16 * TOK; o += KS * 32) {
      const int t = o >> 4, r = o & 15, token = cur.row0 + t, col = cur.n0 + r;
      const int slot = (t >> 3) * 4 + (r >> 3) * 2 + (t & 1), src = (r & 7) * 4 + ((t & 7) >> 1);
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) sum += red[flip][rsub * KS + s][slot][src];
      if (token < cur.end && col < A.N) static_cast<TO*>(A.out)[int64_t(token) * A.N + col] = from_f32<TO>(sum);
    }
    cur = nxt;
  }
  if (A.offsets) zero_rows(static_cast<TO*>(A.out), A.N, off[A.E], A.S, threadIdx.x, kThreads);
  pdl_trigger();
}

template <typename TX, typename TO, int NT, int KS>
int launch_one(cudaStream_t s, const SkinnyArgs& a, int64_t m_tiles) {
  const int n_wt = (a.N + 16 * (kWarps / KS) - 1) / (16 * (kWarps / KS));
  const int64_t ctas = int64_t(sm_count()) * (NT <= 2 ? 2 : 1);
  return launch_chain(fp8_skinny_kernel<TX, TO, NT, KS>, dim3(unsigned(std::min(ctas, m_tiles * n_wt))),
                      dim3(kThreads), 0, s, a) == cudaSuccess
             ? 0
             : -1;
}

// Eight warps along K where each still has four K blocks, else two row tiles of four warps.
template <typename TX, typename TO, int NT>
int launch_ks(cudaStream_t s, const SkinnyArgs& a, int64_t m_tiles) {
  return a.KB > 4 * kDeep ? launch_one<TX, TO, NT, 8>(s, a, m_tiles) : launch_one<TX, TO, NT, 4>(s, a, m_tiles);
}

template <typename TX, int NT>
int launch_out(cudaStream_t s, const SkinnyArgs& a, int64_t m_tiles, int out_dtype) {
  if (out_dtype == B200MOE_F16) return launch_ks<TX, __half, NT>(s, a, m_tiles);
  if (out_dtype == B200MOE_BF16) return launch_ks<TX, __nv_bfloat16, NT>(s, a, m_tiles);
  return launch_ks<TX, float, NT>(s, a, m_tiles);
}

SkinnyArgs args_of(const Fp8Product& p) {
  SkinnyArgs a{};
  a.a = static_cast<const uint8_t*>(p.a);
  a.a_scale = p.a_scale;
  a.lda_s = p.a_scale_stride;
  a.w = static_cast<const uint8_t*>(p.w);
  a.w_scale = p.w_scale;
  a.offsets = p.offsets;
  a.out = p.out;
  a.S = p.S;
  a.N = p.N;
  a.K = p.K;
  a.E = p.E;
  a.KB = (p.K + kFp8Block - 1) / kFp8Block;
  a.NB = (p.N + kFp8Block - 1) / kFp8Block;
  a.err = op_error_word();
  return a;
}

}  // namespace

int launch_fp8_skinny(cudaStream_t s, const Fp8Product& p, int rows_per_tile, int out_dtype) {
  const SkinnyArgs a = args_of(p);
  // upper bound of the row tiles: a tile per rows_per_tile rows and one more for every expert with rows
  const int64_t m_tiles = p.offsets ? int64_t(p.S) / rows_per_tile + std::min(p.E, p.S)
                                    : (p.S + rows_per_tile - 1) / rows_per_tile;
  if (rows_per_tile == 8) return launch_out<uint8_t, 1>(s, a, m_tiles, out_dtype);
  if (rows_per_tile == 16) return launch_out<uint8_t, 2>(s, a, m_tiles, out_dtype);
  return launch_out<uint8_t, 4>(s, a, m_tiles, out_dtype);
}

int launch_fp8_skinny_x(cudaStream_t s, const Fp8Product& p, const void* x, int x_dtype, int64_t ldx, int out_dtype) {
  SkinnyArgs a = args_of(p);
  a.a = static_cast<const uint8_t*>(x);
  a.ldx = ldx;
  if (x_dtype == B200MOE_F16) return launch_out<__half, 1>(s, a, 1, out_dtype);
  return launch_out<__nv_bfloat16, 1>(s, a, 1, out_dtype);
}

}  // namespace b200moe
