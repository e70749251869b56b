// 4-bit products of at most eight rows with one matrix: the weights go straight from
// global memory into the registers of the warps that multiply them. One launch does
// it all: up to 4096 values of f16 or bf16 rows (one row of 4096 columns, eight of
// 512) are quantized by every CTA for itself.
//
// A warp owns 16 weight rows and every KS-th block of 256 columns.  NVFP4: each lane
// loads four 16-byte pieces per block (32 columns each: rows g and g + 8, pieces q and q + 4; g =
// lane / 4, q = lane % 4) and their scales.  Operands are f16, which holds a value times
// its block's scale exactly (six bits, 2^-10 to 2688), by one conversion and one product
// per two values; both operands take the columns in the same order, so no value moves
// between lanes.  MXFP4's scales pass f16's range, so its operands are the codes' values
// and a scale block's product leaves the accumulator for f32 sums times both scales:
// there the four lanes of a row load four bytes each of one block, since an MMA's 16
// columns have to share their scales.  The KS warps of a row tile add their f32 sums in
// shared memory in a fixed order.
//
// Bound: latency, and above a few rows the rows' way into every CTA's shared memory: all
// of a small matrix is in flight at once. 4096 x 4096: NVFP4 5.4 us at one row, 6.7 at
// four, 8.5 at eight, where the streaming kernel takes 8.7 to 8.8; MXFP4 7.6, 8.2 at two,
// 8.7 at three, 9.3 at four (8.6), so three rows at most. 2816 x 2048: 3.8 and 4.6 at one
// row (5.5).  Taken as long as all CTAs, of 16 or 32 weight rows, run at once: to N 4736
// at K above 2048 (5.5 us, one row NVFP4). Past it tiles of 128 weight rows give 38 CTAs
// and more: 8.8 us at N 4864, 9.4 at 8192, 9.8 at 11008, where the bytes take 1.7, 2.9
// and 3.9. Longer K runs block after block, two in flight: one row x 4096 x 7168 8.2 us
// (2.6), x 14336 14.3 (5.1), eight rows 12.2 and, streamed, 20.3.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "fp4_ops.h"
#include "fp4_rows.cuh"
#include "internal.h"

namespace b200moe {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
static_assert(kThreads == kFp4SkinnyThreads, "16 values of the rows that it quantizes per thread");
constexpr int kTokens = 8;
constexpr int kBlockK = 256;
constexpr int kDeep = 2;  // blocks of a warp in flight
constexpr int kSmemMost = 200 * 1024;
// Bytes of 32 columns of a row in shared memory, f16 (NVFP4: and 16 more, so that a fragment load's lanes do not meet), and
// of a row: 64 above a multiple of 128, so that neighbouring rows do not meet either.
__host__ __device__ constexpr int piece_bytes(int fmt) { return fmt == kMx ? 64 : 80; }
__host__ __device__ constexpr int row_pitch(int fmt, int K) { return (K / 32 * piece_bytes(fmt) + 63) / 128 * 128 + 64; }

struct SkinnyArgs {
  const uint8_t* a;  // records, or the rows to quantize (stride ldx elements)
  int64_t ldx;
  const uint8_t* w;
  const uint8_t* w_scale;
  const float* w_factor;
  void* out;
  int S, N, K;
};

__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {  // weights: read once
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
// 16 columns of a row, as codes, times scale to shared memory as f16.  The codes' values come from their bits: with
// cvt.rn.f16x2.e2m1x2 of bytes that the same thread had just converted (CUDA 12.9), rows came out as zeros, while rows whose
// codes were loaded came out right; why was not found.
__device__ __forceinline__ void put_tokens(uint8_t* dst, uint2 codes, float scale) {
  const __half2 s = __float2half2_rn(scale);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t w = h ? codes.y : codes.x;
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // exponent and mantissa bits in f16's place are the value times 2^-14
      const uint32_t b = w >> (8 * i);
      const uint32_t bits = (b & 7u) << 9 | (b & 8u) << 12 | (b & 0x70u) << 21 | (b & 0x80u) << 24;
      o[i] = hmul2(hmul2(bits, 0x74007400u), *reinterpret_cast<const uint32_t*>(&s));
    }
    reinterpret_cast<uint4*>(dst)[h] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// The rows' values in shared memory and their factors (MXFP4: their blocks' scales, [block][8 rows]); TX of one byte:
// records.
template <typename TX, int FMT>
__device__ __forceinline__ void stage_tokens(const SkinnyArgs& A, uint8_t* xs, float* factor, uint32_t* top, float* scales) {
  const int pieces = A.K / 16, total = A.S * pieces, pitch = row_pitch(FMT, A.K);
  auto place = [&](int r, int p) { return xs + r * pitch + p / 2 * piece_bytes(FMT) + (p & 1) * 32; };
  if constexpr (FMT == kMx) {
    for (int i = threadIdx.x; i < pieces / 2 * kTokens; i += kThreads)
      if (i % kTokens >= A.S) scales[i] = 0.f;  // rows that are not there
  }
  if constexpr (sizeof(TX) == 1) {
    const int stride = fp4_stride(FMT, A.K);
    for (int i = threadIdx.x; i < total; i += kThreads) {
      const int r = i / pieces, p = i - r * pieces;
      const uint8_t* rec = A.a + int64_t(r) * stride;
      const uint2 codes = __ldg(reinterpret_cast<const uint2*>(rec) + p);
      if constexpr (FMT == kMx) {
        put_tokens(place(r, p), codes, 1.f);
        if (!(p & 1)) scales[p / 2 * kTokens + r] = e8m0_f32(__ldg(rec + A.K / 2 + p / 2));
      } else {
        put_tokens(place(r, p), codes, e4m3_f32(__ldg(rec + A.K / 2 + p)));
      }
    }
    if (FMT == kNv && threadIdx.x < A.S)
      factor[threadIdx.x] = *reinterpret_cast<const float*>(A.a + int64_t(threadIdx.x) * stride + fp4_factor_at(A.K));
  } else {
    // a piece per thread; pieces is even, so both halves of an MXFP4 block are in one warp
    const int i = threadIdx.x, r = i / pieces, p = i - r * pieces;
    const bool in = i < total;
    float v[16], m = 0.f;
    if (in) {
      Vec<TX, 16> raw;
      raw.load(reinterpret_cast<const TX*>(A.a) + r * A.ldx + p * 16);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = raw.get(j);
      m = magnitude16(v);
    }
    if constexpr (FMT == kMx) {
      m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
      if (in) {
        float inv;
        const uint32_t s = mxfp4_scale(m, inv);
        put_tokens(place(r, p), mxfp4_codes(v, inv), 1.f);
        if (!(p & 1)) scales[p / 2 * kTokens + r] = e8m0_f32(s);
      }
    } else {
      if (threadIdx.x < kTokens) top[threadIdx.x] = 0;
      __syncthreads();
      uint32_t t = in ? abs_bits(m) : 0u;
      if (pieces % 32 == 0) t = __reduce_max_sync(0xffffffffu, t);  // the warp's columns are of one row
      if (in && (pieces % 32 || threadIdx.x % 32 == 0)) atomicMax(top + r, t);  // in any order, a maximum is the same
      __syncthreads();
      if (threadIdx.x < A.S) factor[threadIdx.x] = nvfp4_factor(top[threadIdx.x]);
      if (in) {
        float unit;
        const uint32_t s = nvfp4_scale(m, nvfp4_factor(top[r]), unit);
        put_tokens(place(r, p), nvfp4_codes(v, unit), e4m3_f32(s));
      }
    }
  }
}

// The KS warps' sums of a row tile, joined in a fixed order, times both factors.
template <typename TO, int KS>
__device__ __forceinline__ void join(const SkinnyArgs& A, float (&red)[kWarps][4][32], const float (&acc)[4], int n0,
                                     const float* factor, float fw) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ksub = warp % KS, rsub = warp / KS;
#pragma unroll
  for (int i = 0; i < 4; ++i) red[warp][i][lane] = acc[i];
  __syncthreads();
  for (int o = ksub * 32 + lane; o < 16 * kTokens; o += KS * 32) {
    const int t = o >> 4, r = o & 15, col = n0 + r;
    const int slot = (r >> 3) * 2 + (t & 1), src = (r & 7) * 4 + (t >> 1);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) sum += red[rsub * KS + k][slot][src];
    if (t < A.S && col < A.N) {
      const Fp4Factors f = factor ? fp4_factors(factor[t], fw) : Fp4Factors{1.f, 1.f};
      static_cast<TO*>(A.out)[int64_t(t) * A.N + col] = from_f32<TO>(sum * f.first * f.second);
    }
  }
}

template <typename TX, typename TO, int KS>
__global__ void __launch_bounds__(kThreads, 2) nvfp4_skinny_kernel(const SkinnyArgs A) {
  constexpr int RT = kWarps / KS;  // 16-row tiles of w per CTA
  __shared__ float red[kWarps][4][32];
  __shared__ float factor[kTokens];
  __shared__ uint32_t top[kTokens];
  extern __shared__ __align__(16) uint8_t xs[];  // [S][row_pitch]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int ksub = warp % KS, rsub = warp / KS;
  const int n0 = (blockIdx.x * RT + rsub) * 16, KB = (A.K + kBlockK - 1) / kBlockK;
  const int per_warp = (KB + KS - 1) / KS, n_steps = (per_warp + kDeep - 1) / kDeep;
  const int half_k = A.K / 2, scales = A.K / 16;
  pdl_wait();

  uint4 w[kDeep][4];
  uint32_t ws[kDeep][4];  // the pieces' scale bytes
  auto fetch = [&](int step, int j) {
    const int kb = (step * kDeep + j) * KS + ksub;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = n0 + g + 8 * h, piece = kb * 8 + c * 4 + q;
        const bool in = row < A.N && piece * 32 < A.K;
        w[j][h * 2 + c] = in ? ld_stream(A.w + int64_t(row) * half_k + piece * 16) : make_uint4(0, 0, 0, 0);
        ws[j][h * 2 + c] =
            in ? uint32_t(__ldg(reinterpret_cast<const uint16_t*>(A.w_scale + int64_t(row) * scales + 2 * piece))) : 0u;
      }
  };

#pragma unroll
  for (int j = 0; j < kDeep; ++j) fetch(0, j);
  stage_tokens<TX, kNv>(A, xs, factor, top, nullptr);
  __syncthreads();
  const uint8_t* mine = xs + g * row_pitch(kNv, A.K);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int step = 0; step < n_steps; ++step) {
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const int kb = (step * kDeep + j) * KS + ksub;
      if (kb < KB) {  // the same for the whole warp
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int piece = kb * 8 + c * 4 + q;
          const uint32_t lo[4] = {w[j][c].x, w[j][c].y, w[j][c].z, w[j][c].w};
          const uint32_t hi[4] = {w[j][2 + c].x, w[j][2 + c].y, w[j][2 + c].z, w[j][2 + c].w};
          const uint32_t ml = e4m3x2_to_f16x2(ws[j][c]), mh = e4m3x2_to_f16x2(ws[j][2 + c]);  // of both halves
          const bool in = g < A.S && piece * 32 < A.K;
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // eight columns of this lane: two MMAs of 16 columns
            const uint8_t* from = mine + piece * piece_bytes(kNv) + i * 16;
            const uint4 x = in ? *reinterpret_cast<const uint4*>(from) : make_uint4(0, 0, 0, 0);
            uint32_t a[4], b[4];
            e2m1x8_scaled(lo[i], i < 2 ? lo_half2(ml) : hi_half2(ml), a);
            e2m1x8_scaled(hi[i], i < 2 ? lo_half2(mh) : hi_half2(mh), b);
            mma_16816(acc, {a[0], b[0], a[1], b[1]}, x.x, x.y);
            mma_16816(acc, {a[2], b[2], a[3], b[3]}, x.z, x.w);
          }
        }
      }
      if (step + 1 < n_steps) fetch(step + 1, j);
    }
  }
  join<TO, KS>(A, red, acc, n0, factor, *A.w_factor);
  pdl_trigger();
}

template <typename TX, typename TO, int KS>
__global__ void __launch_bounds__(kThreads, 2) mxfp4_skinny_kernel(const SkinnyArgs A) {
  constexpr int RT = kWarps / KS;  // 16-row tiles of w per CTA
  __shared__ float red[kWarps][4][32];
  extern __shared__ __align__(16) uint8_t xs[];  // [S][row_pitch], then the scales [K / 32][8]
  float* ss = reinterpret_cast<float*>(xs + A.S * row_pitch(kMx, A.K));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int ksub = warp % KS, rsub = warp / KS;
  const int n0 = (blockIdx.x * RT + rsub) * 16, KB = (A.K + kBlockK - 1) / kBlockK;
  const int per_warp = (KB + KS - 1) / KS, n_steps = (per_warp + kDeep - 1) / kDeep;
  const int half_k = A.K / 2, scales = A.K / 32;
  const bool by_eight = scales % 8 == 0 && reinterpret_cast<uintptr_t>(A.w_scale) % 8 == 0;
  pdl_wait();

  uint32_t w[kDeep][2][8];  // rows g and g + 8: four bytes of each scale block
  uint2 ws[kDeep][2];       // the eight blocks' scale bytes
  auto fetch = [&](int step, int j) {
    const int kb = (step * kDeep + j) * KS + ksub;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = n0 + g + 8 * h;
      const uint8_t* p = A.w + int64_t(row) * half_k + kb * (kBlockK / 2) + q * 4;
      const uint8_t* s = A.w_scale + int64_t(row) * scales + kb * 8;
#pragma unroll
      for (int b = 0; b < 8; ++b)
        w[j][h][b] = row < A.N && (kb * 8 + b) * 32 < A.K ? __ldg(reinterpret_cast<const uint32_t*>(p + b * 16)) : 0u;
      ws[j][h] = make_uint2(0, 0);
      if (by_eight) {
        if (row < A.N && kb < KB) ws[j][h] = __ldg(reinterpret_cast<const uint2*>(s));
      } else {
        uint32_t t[2] = {0, 0};
#pragma unroll
        for (int b = 0; b < 8; ++b)
          if (row < A.N && kb * 8 + b < scales) t[b / 4] |= uint32_t(__ldg(s + b)) << (8 * (b % 4));
        ws[j][h] = make_uint2(t[0], t[1]);
      }
    }
  };

#pragma unroll
  for (int j = 0; j < kDeep; ++j) fetch(0, j);
  stage_tokens<TX, kMx>(A, xs, nullptr, nullptr, ss);
  __syncthreads();
  const uint8_t* mine = xs + g * row_pitch(kMx, A.K) + q * 16;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int step = 0; step < n_steps; ++step) {
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const int kb = (step * kDeep + j) * KS + ksub;
      auto blocks = [&](auto careful) {
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          const int block = kb * 8 + b;
          if (block >= scales) break;  // the same for the whole warp
          const uint32_t lo = w[j][0][b], hi = w[j][1][b];
          const uint4 x = g < A.S ? *reinterpret_cast<const uint4*>(mine + block * piece_bytes(kMx)) : make_uint4(0, 0, 0, 0);
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma_16816(d, {e2m1x2_byte<0>(lo), e2m1x2_byte<0>(hi), e2m1x2_byte<1>(lo), e2m1x2_byte<1>(hi)}, x.x, x.y);
          mma_16816(d, {e2m1x2_byte<2>(lo), e2m1x2_byte<2>(hi), e2m1x2_byte<3>(lo), e2m1x2_byte<3>(hi)}, x.z, x.w);
          const float sl = e8m0_f32((b < 4 ? ws[j][0].x : ws[j][0].y) >> (8 * (b % 4)) & 255u);
          const float sh = e8m0_f32((b < 4 ? ws[j][1].x : ws[j][1].y) >> (8 * (b % 4)) & 255u);
          const float2 sa = *reinterpret_cast<const float2*>(ss + block * kTokens + 2 * q);
          auto add = [&](float& to, float sum, float sw, float sx) {
            if constexpr (careful)
              to = fmaf(sum * min_nan(sw, sx), max_nan(sw, sx), to);
            else
              to = fmaf(sum * sw, sx, to);
          };
          add(acc[0], d[0], sl, sa.x);
          add(acc[1], d[1], sl, sa.y);
          add(acc[2], d[2], sh, sa.x);
          add(acc[3], d[3], sh, sa.y);
        }
      };
      // A block's sum (a multiple of 1/4 up to 1152) times the weights' scale alone is exact below 1 and passes f32 from
      // 2^118 up, where the row's scale would bring it back: weights with a byte from 192 (2^65) up take the smaller scale
      // first (for all weights that costs 5 %: 4096 x 4096, one row, 7.9 us instead of 7.5).
      if (kb < KB) {  // the same for the whole warp
        const uint32_t s0 = ws[j][0].x, s1 = ws[j][0].y, s2 = ws[j][1].x, s3 = ws[j][1].y;
        const uint32_t high = (s0 & s0 << 1) | (s1 & s1 << 1) | (s2 & s2 << 1) | (s3 & s3 << 1);
        if (__any_sync(0xffffffffu, high & 0x80808080u))
          blocks(std::true_type{});
        else
          blocks(std::false_type{});
      }
      if (step + 1 < n_steps) fetch(step + 1, j);
    }
  }
  join<TO, KS>(A, red, acc, n0, nullptr, 1.f);
  pdl_trigger();
}

// Eight warps along K where each has two blocks, else two row tiles of four warps.
bool deep(int K) { return K > 4 * kDeep * kBlockK; }
int skinny_grid(int N, int K) {
  const int rows = 16 * (deep(K) ? 1 : 2);
  return (N + rows - 1) / rows;
}
size_t skinny_smem(int fmt, int S, int K) {
  return size_t(S) * row_pitch(fmt, K) + (fmt == kMx ? size_t(K) / 32 * kTokens * sizeof(float) : 0);
}

template <typename TX, typename TO, int FMT, int KS>
int launch_one(cudaStream_t s, const SkinnyArgs& a) {
  auto kernel = FMT == kMx ? mxfp4_skinny_kernel<TX, TO, KS> : nvfp4_skinny_kernel<TX, TO, KS>;
  static std::atomic<uint64_t> attr_set{0};  // devices whose attribute is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -1;
  if (!(attr_set.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost) != cudaSuccess) return -1;
    attr_set.fetch_or(uint64_t(1) << dev);
  }
  return launch_chain(kernel, dim3(skinny_grid(a.N, a.K)), dim3(kThreads), skinny_smem(FMT, a.S, a.K), s, a) == cudaSuccess
             ? 0
             : -1;
}

template <typename TX, int FMT>
int launch_out(cudaStream_t s, const SkinnyArgs& a, int out_dtype) {
  const bool d = deep(a.K);
  if (out_dtype == B200MOE_F16) return d ? launch_one<TX, __half, FMT, 8>(s, a) : launch_one<TX, __half, FMT, 4>(s, a);
  if (out_dtype == B200MOE_BF16)
    return d ? launch_one<TX, __nv_bfloat16, FMT, 8>(s, a) : launch_one<TX, __nv_bfloat16, FMT, 4>(s, a);
  return d ? launch_one<TX, float, FMT, 8>(s, a) : launch_one<TX, float, FMT, 4>(s, a);
}

template <typename TX>
int launch_format(cudaStream_t s, const SkinnyArgs& a, int format, int out_dtype) {
  return format == kMx ? launch_out<TX, kMx>(s, a, out_dtype) : launch_out<TX, kNv>(s, a, out_dtype);
}

}  // namespace

bool fp4_skinny_fits(const Fp4Product& p) {
  const int most = p.format == kMx ? 3 : kTokens;
  if (p.E != 1 || p.offsets || p.S > most || reinterpret_cast<uintptr_t>(p.w_scale) % 2) return false;
  const size_t smem = skinny_smem(p.format, p.S, p.K);
  return smem <= kSmemMost && skinny_grid(p.N, p.K) <= sm_count() * (smem <= 100 * 1024 ? 2 : 1);
}

int launch_fp4_skinny(cudaStream_t s, const Fp4Product& p, const void* x, int x_dtype, int64_t ldx, int out_dtype) {
  const SkinnyArgs a{x ? static_cast<const uint8_t*>(x) : p.a, ldx, p.w, p.w_scale, p.w_factor, p.out, p.S, p.N, p.K};
  if (!x) return launch_format<uint8_t>(s, a, p.format, out_dtype);
  return x_dtype == B200MOE_F16 ? launch_format<__half>(s, a, p.format, out_dtype)
                                : launch_format<__nv_bfloat16>(s, a, p.format, out_dtype);
}

}  // namespace b200moe
