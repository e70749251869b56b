// E4M3 matrix products with a scale per block of 128 on the 5th-generation
// tensor cores: out[m][n] = sum_b sa[m][b] sb[n / 128][b] sum_{k in block b} a[m][k] w[n][k],
// dense, or with the rows sorted by expert and each expert's own weights.
//
// The scales change with every 128 columns of K, so the tensor core's own
// accumulation may run over one block only.  A persistent CTA per SM walks tiles
// of 128 rows x BN columns; per K block
//   warp 0 (producer): two TMA boxes (128 rows of a, BN rows of w; 128 columns,
//     128-byte swizzle) into a ring of stages;
//   warp 1 (MMA): one thread issues 4 x tcgen05.mma.kind::f8f6f4 (M 128, N BN,
//     K 32) into one of the TMEM buffers of BN columns and commits;
//   warps 2-9 (sums): read the block's product (a thread holds one row and half
//     the columns, so both scales are one factor per thread and block) and add
//     factor * product to f32 sums in registers, two columns per instruction,
//     while the tensor core fills the next buffer.
// At BN = 256 the block's MMAs take 512 clocks and its sums about 300 of each
// scheduler's issue slots, so the tensor pipe stays the bound.  The finished
// tile goes through shared memory so that rows are stored in 64-byte pieces.
// Rows of a tile that belong to the next expert are computed and not stored.
// Every wait is bounded; after an abort the roles drain in-flight copies and
// MMAs before TMEM is freed.
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "fp8_device.cuh"
#include "fp8_ops.h"
#include "internal.h"

namespace b200moe {
namespace {

constexpr int kBM = 128;
constexpr int kSumWarps = 8;
constexpr int kThreads = (2 + kSumWarps) * 32;
constexpr int kMaxExperts = 1024;
constexpr int kABytes = kBM * kFp8Block;
constexpr int kOutBytes = 32 * 64;  // per sum warp: 32 rows in pieces of 64 bytes

template <int BN>
struct Cfg {
  static constexpr int kWBytes = BN * kFp8Block;
  static constexpr int kStages = BN == 256 ? 4 : 6;
  static constexpr int kBufs = 512 / BN > 4 ? 4 : 512 / BN;  // TMEM buffers
  static constexpr int kCols = BN / 2;                        // columns per sum thread
  static constexpr size_t kSmem = 1024 + size_t(kStages) * (kABytes + kWBytes) + kSumWarps * kOutBytes + 256;
  static constexpr uint32_t kIdesc = (1u << 4) | (uint32_t(BN >> 3) << 17) | (uint32_t(kBM >> 4) << 24);
  static_assert(kSmem + 8 * (kMaxExperts + 1) + 64 <= 227 * 1024, "shared memory, with the tile table");
};

__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
  // K-major, 128-byte swizzle: rows of 128 bytes, 8-row atoms 1024 bytes apart
  return uint64_t((addr >> 4) & 0x3FFF) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}

__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p; }" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// 16 columns of this thread's TMEM lane; the values are there after tmem_wait on the same array.
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
// The registers pass through the wait, so no use of them can move above it.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// acc += s * p for two columns at once (each an f32 fma)
__device__ __forceinline__ void fma2(uint64_t& acc, uint32_t p0, uint32_t p1, uint64_t s2) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "r"(p0), "r"(p1));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(p), "l"(s2));
}

struct GemmArgs {
  const float* a_scale;  // [S][KB], row stride lda_s
  int64_t lda_s;
  const float* w_scale;  // [E][NB][KB]
  const int32_t* offsets;  // [E + 1], null: one matrix, all S rows
  void* out;             // [S][N]
  int S, N, K, E, KB, NB;
  uint32_t* err;
};

template <int BN, typename TO>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_gemm_kernel(const GemmArgs a, const __grid_constant__ CUtensorMap map_a,
                    const __grid_constant__ CUtensorMap map_w) {
  using C = Cfg<BN>;
  constexpr int ST = C::kStages, NBUF = C::kBufs, COLS = C::kCols;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int off[kMaxExperts + 1], start[kMaxExperts + 1];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_flag;
  const uint32_t base_u32 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base = smem_raw + (base_u32 - smem_u32(smem_raw));
  uint8_t* at = base;                       // [ST][16 KB]
  uint8_t* wt = at + ST * kABytes;          // [ST][BN x 128]
  uint8_t* stage_out = wt + ST * C::kWBytes;  // [8][2 KB]
  uint64_t* full = reinterpret_cast<uint64_t*>(stage_out + kSumWarps * kOutBytes);
  uint64_t* empty = full + ST;
  uint64_t* acc_full = empty + ST;
  uint64_t* acc_empty = acc_full + NBUF;
  volatile int* abort_ptr = &abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < NBUF; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kSumWarps);
    }
    fence_barrier_init();
    abort_flag = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_sh)),
                 "r"(uint32_t(NBUF * BN)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_base_sh;
  pdl_wait();
  const int n_nt = (a.N + BN - 1) / BN;
  build_tile_table(a.offsets, a.E, a.S, kBM, n_nt, off, start, a.err);
  const int n_items = start[a.E];

  if (warp == 0) {
    if (lane == 0) {
      uint32_t g = 0, issued = 0, par = 0;
      for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        const int e = tile_expert(start, a.E, item), local = item - start[e];
        const int row = off[e] + local / n_nt * kBM, wrow = e * a.N + local % n_nt * BN;
        for (int kb = 0; kb < a.KB; ++kb, ++g) {
          const int s = g % ST;
          const uint32_t ph = (g / ST) & 1u;
          if (*abort_ptr || !mbar_wait(&empty[s], ph ^ 1u, a.err)) {
            *abort_ptr = 1;
            break;
          }
          mbar_arrive_expect_tx(&full[s], uint32_t(kABytes + C::kWBytes));
          tma_2d(at + s * kABytes, &map_a, kb * kFp8Block, row, &full[s]);
          tma_2d(wt + s * C::kWBytes, &map_w, kb * kFp8Block, wrow, &full[s]);
          issued |= 1u << s;
          par = (par & ~(1u << s)) | (ph << s);
        }
        if (*abort_ptr) break;
      }
      // no copy may be in flight when the CTA exits
      for (int s = 0; s < ST; ++s)
        if (issued & (1u << s)) mbar_wait(&full[s], (par >> s) & 1u, a.err);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t g = 0;
      bool ok = true, committed = false;
      int last_b = 0;
      uint32_t last_ph = 0;
      for (int item = blockIdx.x; ok && item < n_items; item += gridDim.x) {
        for (int kb = 0; kb < a.KB; ++kb, ++g) {
          const int s = g % ST, b = g % NBUF;
          const uint32_t ph = (g / ST) & 1u, bph = (g / NBUF) & 1u;
          if (*abort_ptr || !mbar_wait(&acc_empty[b], bph ^ 1u, a.err) || !mbar_wait(&full[s], ph, a.err)) {
            *abort_ptr = 1;
            ok = false;
            break;
          }
          fence_after();
          const uint64_t da = desc_sw128(smem_u32(at + s * kABytes)), dw = desc_sw128(smem_u32(wt + s * C::kWBytes));
#pragma unroll
          for (int k = 0; k < 4; ++k)  // 32 columns = 32 bytes of the swizzled row each
            mma_f8(tmem + b * BN, da + 2 * k, dw + 2 * k, C::kIdesc, k != 0);
          commit(&empty[s]);
          commit(&acc_full[b]);
          committed = true;
          last_b = b;
          last_ph = bph;
        }
      }
      if (committed) mbar_wait(&acc_full[last_b], last_ph, a.err);
    }
  } else {
    // a warp may read the TMEM lanes 32 (warp % 4) ..; the two warps of a quarter split the columns
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    uint8_t* mine = stage_out + (warp - 2) * kOutBytes;
    uint32_t g = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < n_items; item += gridDim.x) {
      const int e = tile_expert(start, a.E, item), local = item - start[e];
      const int row0 = off[e] + local / n_nt * kBM + quarter * 32, end = off[e + 1];
      const int col0 = local % n_nt * BN + half * COLS;
      const int nb = min(col0 / kFp8Block, a.NB - 1);
      const float* sa = a.a_scale + int64_t(min(row0 + lane, a.S - 1)) * a.lda_s;
      const float* sb = a.w_scale + (int64_t(e) * a.NB + nb) * a.KB;
      uint64_t acc[COLS / 2];
#pragma unroll
      for (int i = 0; i < COLS / 2; ++i) acc[i] = 0;
      float sa_next = __ldg(sa), sb_next = __ldg(sb);
      for (int kb = 0; kb < a.KB; ++kb, ++g) {
        const float f = sa_next * sb_next;
        if (kb + 1 < a.KB) {
          sa_next = __ldg(sa + kb + 1);
          sb_next = __ldg(sb + kb + 1);
        }
        uint64_t f2;
        asm("mov.b64 %0, {%1, %1};" : "=l"(f2) : "r"(__float_as_uint(f)));
        const int b = g % NBUF;
        ok = !*abort_ptr && mbar_wait(&acc_full[b], (g / NBUF) & 1u, a.err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
        const uint32_t addr = tmem + (uint32_t(quarter * 32) << 16) + b * BN + half * COLS;
        uint32_t p[2][16];
        tmem_ld16(addr, p[0]);
#pragma unroll
        for (int c = 0; c < COLS / 16; ++c) {
          tmem_wait(p[c & 1]);
          if (c + 1 < COLS / 16) tmem_ld16(addr + (c + 1) * 16, p[(c + 1) & 1]);
#pragma unroll
          for (int i = 0; i < 8; ++i) fma2(acc[c * 8 + i], p[c & 1][2 * i], p[c & 1][2 * i + 1], f2);
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[b]);
      }
      if (!ok) {
        *abort_ptr = 1;
        break;
      }
      // through shared memory in pieces of 64 bytes per row, 16-byte chunks swizzled by pairs of rows
      constexpr int PW = 64 / int(sizeof(TO));  // columns per piece
      constexpr int CW = 16 / int(sizeof(TO));  // columns per chunk
      TO* out = static_cast<TO*>(a.out);
      const bool vec = (int64_t(a.N) * sizeof(TO)) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
#pragma unroll
      for (int pc = 0; pc < COLS / PW; ++pc) {
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          float v[CW];
#pragma unroll
          for (int i = 0; i < CW / 2; ++i) {
            const uint64_t u = acc[(pc * PW + ch * CW) / 2 + i];
            v[2 * i] = __uint_as_float(uint32_t(u));
            v[2 * i + 1] = __uint_as_float(uint32_t(u >> 32));
          }
          store_vec<TO, CW>(reinterpret_cast<TO*>(mine + lane * 64 + ((ch ^ ((lane >> 1) & 3)) << 4)), v);
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = j * 8 + (lane >> 2), ch = lane & 3;
          const TO* src = reinterpret_cast<const TO*>(mine + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4));
          const int col = col0 + pc * PW + ch * CW;
          if (row0 + r < end) {
            TO* dst = out + int64_t(row0 + r) * a.N + col;
            if (vec && col + CW <= a.N) {
              *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
            } else {
              for (int i = 0; i < CW; ++i)
                if (col + i < a.N) dst[i] = src[i];
            }
          }
        }
        __syncwarp();
      }
    }
    if (a.offsets) zero_rows(static_cast<TO*>(a.out), a.N, off[a.E], a.S, threadIdx.x - 64, kSumWarps * 32);
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(uint32_t(NBUF * BN)));
  }
  pdl_trigger();
}

template <int BN, typename TO>
int launch_one(cudaStream_t s, const GemmArgs& a, const CUtensorMap& ma, const CUtensorMap& mw, int grid) {
  static std::atomic<uint64_t> attr_set{0};  // devices whose attribute is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -1;
  if (!(attr_set.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(fp8_gemm_kernel<BN, TO>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             int(Cfg<BN>::kSmem)) != cudaSuccess)
      return -1;
    attr_set.fetch_or(uint64_t(1) << dev);
  }
  return launch_chain(fp8_gemm_kernel<BN, TO>, dim3(grid), dim3(kThreads), Cfg<BN>::kSmem, s, a, ma, mw) == cudaSuccess
             ? 0
             : -1;
}

}  // namespace

int launch_fp8_gemm(cudaStream_t s, const Fp8Product& p, int out_dtype) {
  GemmArgs a{};
  a.a_scale = p.a_scale;
  a.lda_s = p.a_scale_stride;
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
  const int sms = sm_count();
  // upper bound of the row tiles: a tile per 128 rows and one more for every expert with rows
  const int64_t m_tiles = p.offsets ? int64_t(p.S) / kBM + std::min(p.E, p.S) : (p.S + kBM - 1) / kBM;
  const int64_t wide_tiles = m_tiles * ((p.N + 255) / 256);
  const bool wide = wide_tiles >= sms;
  const int bn = wide ? 256 : 128;
  CUtensorMap ma, mw;
  if (make_u8_tile_map(&ma, p.a, p.S, p.K, kFp8Block, kBM) ||
      make_u8_tile_map(&mw, p.w, int64_t(p.E) * p.N, p.K, kFp8Block, bn))
    return -1;
  const int grid = int(std::min<int64_t>(sms, m_tiles * ((p.N + bn - 1) / bn)));
  auto run = [&](auto one) { return one(s, a, ma, mw, grid); };
  if (out_dtype == B200MOE_F16) return run(wide ? launch_one<256, __half> : launch_one<128, __half>);
  if (out_dtype == B200MOE_BF16) return run(wide ? launch_one<256, __nv_bfloat16> : launch_one<128, __nv_bfloat16>);
  return run(wide ? launch_one<256, float> : launch_one<128, float>);
}

}  // namespace b200moe

using namespace b200moe;

namespace {

int product_status(const Fp8Product& p, int out_dtype) {
  if (!p.w || !p.w_scale || !p.out || p.S < 1 || p.N < 1 || p.K < 16 || p.K % 16 || p.E < 1 || p.E > kMaxExperts ||
      (!p.offsets && p.E != 1) || int64_t(p.E) * p.N > INT32_MAX - 256 || p.K > (1 << 24))
    return B200MOE_ERR_INVALID_ARG;
  if (out_dtype < 0 || out_dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  if (reinterpret_cast<uintptr_t>(p.w) % 16) return B200MOE_ERR_ALIGN;
  return B200MOE_OK;
}

int launch_status(int rc) {
  if (rc == 0) return B200MOE_OK;
  cudaGetLastError();
  return B200MOE_ERR_CUDA;
}

}  // namespace

extern "C" int b200moe_fp8_matmul(void* stream, const void* a, const float* a_scale, int64_t a_scale_stride,
                                  const void* w, const float* w_scale, const int32_t* offsets, int S, int N, int K,
                                  int E, void* out, int out_dtype) {
  const Fp8Product p{a, a_scale, a_scale_stride, w, w_scale, offsets, out, S, N, K, E};
  const int st = product_status(p, out_dtype);
  if (st) return st;
  if (!a || !a_scale || a_scale_stride < 0) return B200MOE_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(a) % 16) return B200MOE_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (S <= 8 * int64_t(E)) return launch_status(launch_fp8_skinny(s, p, 8, out_dtype));
  if (S <= 16 * int64_t(E)) return launch_status(launch_fp8_skinny(s, p, 16, out_dtype));
  return launch_status(launch_fp8_gemm(s, p, out_dtype));
}

extern "C" int b200moe_fp8_linear(void* stream, const void* x, int x_dtype, int64_t ldx, const void* w,
                                  const float* w_scale, int S, int N, int K, void* out, int out_dtype) {
  const Fp8Product p{nullptr, nullptr, 0, w, w_scale, nullptr, out, S, N, K, 1};
  const int st = product_status(p, out_dtype);
  if (st) return st;
  if (!x || ldx < 0 || S > 8) return B200MOE_ERR_INVALID_ARG;
  if (x_dtype != B200MOE_F16 && x_dtype != B200MOE_BF16) return B200MOE_ERR_DTYPE;
  if (reinterpret_cast<uintptr_t>(x) % 16 || ldx % 8) return B200MOE_ERR_ALIGN;
  return launch_status(
      launch_fp8_skinny_x(static_cast<cudaStream_t>(stream), p, x, x_dtype, ldx, out_dtype));
}
