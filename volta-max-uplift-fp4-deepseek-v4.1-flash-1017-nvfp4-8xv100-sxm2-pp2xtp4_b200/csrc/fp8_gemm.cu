// E4M3 matrix products with a scale per block of 128 on the 5th-generation
// tensor cores: out[m][n] = sum_b sa[m][b] sb[n / 128][b] sum_{k in block b} a[m][k] w[n][k],
// dense, or with the rows sorted by expert and each expert's own weights.
//
// The scales change with every 128 columns of K, so the tensor core's own
// accumulation may run over one block only.  A persistent CTA per SM walks tiles
// of 128 rows x BN columns; per K block
//   warp 0 (producer): two TMA boxes (128 rows of a, BN rows of w; 128 columns,
//     128-byte swizzle) into a ring of stages;
//   warp 1 (MMA; at BN = 128 also warp 2, a block each in turn): one lane issues 4 x tcgen05.mma.kind::f8f6f4 (M 128, N BN,
//     K 32) into one of the TMEM buffers of BN columns and commits; the whole
//     warp runs the loop, so that its operands stay in uniform registers (issued
//     by a lone lane of a diverged warp the four MMAs take 345 clocks);
//   warps 4-11 (sums): read the block's product (a thread holds one row and half
//     the columns, so both scales are one factor per thread and block) and add
//     factor * product to f32 sums in registers while the tensor core fills the
//     next buffer.
// The finished tile leaves through shared memory by TMA stores of 32 rows x 64
// bytes.  Rows of a tile that belong to the next expert are computed and not
// stored.  Every wait is bounded; after an abort the roles drain in-flight copies
// and MMAs before TMEM is freed.
//
// Bound: at BN = 256 a block's MMAs take 516 clocks by themselves, beside copies,
// TMEM reads and sums too (each measured apart), and the kernel takes about 780 a
// block: the sums 470 (256 fused multiply-adds and 256 columns of TMEM reads per
// scheduler), and with two buffers their waits, the issue and the commit's arrival
// (290 together) and the MMA warp's turns among the sums' instructions are not
// hidden. 8192 x 4096 x 4096: 126 us, 2.18 PFLOP/s, the tensor pipe 59 % busy.
// Measured and not kept: sums by packed f32x2 (157 us: half the rate of the scalar
// ones), by sixteen warps (151 us), from 16 columns at a time (167 us), blocks in
// halves of 128 columns with barriers of their own (138 us), the factors computed by
// two more warps (134 us), BN = 128 with four buffers (163 us), L2 prefetch of the
// next blocks (138 us).
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "fp8_device.cuh"
#include "fp8_ops.h"
#include "fp8_tc.cuh"
#include "internal.h"

namespace b200moe {
namespace {

constexpr int kBM = 128;
constexpr int kSumWarps = 8;
constexpr int kSumWarp0 = 4;  // warps 0-3: producer, MMA, the rest without work (a register share is a group of four)
constexpr int kThreads = (kSumWarp0 + kSumWarps) * 32;
// registers per thread: the launch's 384 x 168 split as 128 x 40 + 256 x 232
constexpr int kFewRegs = 40, kSumRegs = 232;
constexpr int kMaxExperts = 1024;
constexpr int kABytes = kBM * kFp8Block;
constexpr int kOutBytes = 32 * 64;  // per sum warp: 32 rows in pieces of 64 bytes
constexpr int kAhead = 4;           // K blocks whose scales are loaded ahead of their sums

template <int BN>
struct Cfg {
  static constexpr int kWBytes = BN * kFp8Block;
  static constexpr int kStages = BN == 256 ? 4 : 6;
  static constexpr int kBufs = 512 / BN > 4 ? 4 : 512 / BN;  // TMEM buffers
  // at BN = 128 a block's issue takes as long as its MMAs: 333 x 2816 x 2048 in 7.3 us with two warps, 8.5 with one; at
  // 256 the sums are the longer part either way
  static constexpr int kMmaWarps = BN == 128 ? 2 : 1;
  static constexpr int kCols = BN / 2;                        // columns per sum thread
  static constexpr size_t kSmem = 1024 + size_t(kStages) * (kABytes + kWBytes) + kSumWarps * kOutBytes + 256;
  static constexpr uint32_t kIdesc = (1u << 4) | (uint32_t(BN >> 3) << 17) | (uint32_t(kBM >> 4) << 24);
  static_assert(kSmem + 8 * (kMaxExperts + 1) + 64 <= 227 * 1024, "shared memory, with the tile table");
};

struct GemmArgs {
  const float* a_scale;  // [S][KB], row stride lda_s
  int64_t lda_s;
  const float* w_scale;  // [E][NB][KB]
  const int32_t* offsets;  // [E + 1], null: one matrix, all S rows
  void* out;             // [S][N]
  int copy_out;          // its rows lie on 16 bytes
  int S, N, E, KB, NB;
  uint32_t* err;
};

template <int BN, typename TO>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_gemm_kernel(const GemmArgs a, const __grid_constant__ CUtensorMap map_a,
                    const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_out) {
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

  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
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

  if (warp < kSumWarp0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
    // whole warps run these loops (values stay uniform); one elected lane issues
    if (warp == 0) {
      int st = 0;
      uint32_t ph = 0, issued = 0, par = 0;
      bool ok = true;
      for (int item = blockIdx.x; ok && item < n_items; item += gridDim.x) {
        const int e = tile_expert(start, a.E, item), local = item - start[e];
        const int row = off[e] + local / n_nt * kBM, wrow = e * a.N + local % n_nt * BN;
        for (int kb = 0; kb < a.KB; ++kb) {
          ok = !__any_sync(0xffffffffu, *abort_ptr) && poll_warp(&empty[st], ph ^ 1u, a.err);
          if (!ok) break;
          if (elect_one()) {
            mbar_arrive_expect_tx(&full[st], uint32_t(kABytes + C::kWBytes));
            tma_2d(at + st * kABytes, &map_a, kb * kFp8Block, row, &full[st]);
            tma_2d(wt + st * C::kWBytes, &map_w, kb * kFp8Block, wrow, &full[st]);
          }
          issued |= 1u << st;
          par = (par & ~(1u << st)) | (ph << st);
          if (++st == ST) st = 0, ph ^= 1u;
        }
      }
      if (!ok) *abort_ptr = 1;
      // no copy may be in flight when the CTA exits
      for (int s = 0; s < ST; ++s)
        if (issued & (1u << s)) poll_warp(&full[s], (par >> s) & 1u, a.err);
    }
    if (warp >= 1 && warp <= C::kMmaWarps) {
      // the warps take the K blocks in turn, whatever their tiles: a block's issue by one then runs beside another's
      // waits. Stages and buffers are multiples of them, so that each stays with one warp: were a stage shared, one warp
      // could wait for its second filling before the first has landed, and a parity wait would take the phase before
      // for it.
      constexpr int MW = C::kMmaWarps;
      static_assert(ST % MW == 0 && NBUF % MW == 0, "stages and buffers by MMA warp");
      const int tiles = int(blockIdx.x) < n_items ? (n_items - 1 - int(blockIdx.x)) / int(gridDim.x) + 1 : 0;
      const int64_t total = int64_t(tiles) * a.KB;
      int st = warp - 1, b = st, last = 0;
      uint32_t ph = 0, bph = 0, last_ph = 0;
      bool ok = true, committed = false;
      const uint64_t da0 = desc_sw128(smem_u32(at)), dw0 = desc_sw128(smem_u32(wt));
      for (int64_t g = st; g < total; g += MW) {
        ok = poll_warp(&full[st], ph, a.err) && poll_warp(&acc_empty[b], bph ^ 1u, a.err);
        if (!ok) break;
        fence_after();
        const uint64_t da = da0 + st * (kABytes >> 4), dw = dw0 + st * (C::kWBytes >> 4);
        if (elect_one()) {
          mma_block(tmem + b * BN, da, dw, C::kIdesc);
          commit(&empty[st]);
          commit(&acc_full[b]);
        }
        __syncwarp();
        committed = true;
        last = b;
        last_ph = bph;
        if ((st += MW) >= ST) st -= ST, ph ^= 1u;
        if ((b += MW) >= NBUF) b -= NBUF, bph ^= 1u;
      }
      if (!ok) *abort_ptr = 1;
      if (committed) poll_warp(&acc_full[last], last_ph, a.err);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
    // a warp may read the TMEM lanes 32 (warp % 4) ..; the two warps of a quarter split the columns
    const int quarter = warp & 3, half = (warp - kSumWarp0) >> 2;
    uint8_t* mine = stage_out + (warp - kSumWarp0) * kOutBytes;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16) + half * COLS;
    int b = 0;
    uint32_t bph = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < n_items; item += gridDim.x) {
      const int e = tile_expert(start, a.E, item), local = item - start[e];
      const int row0 = off[e] + local / n_nt * kBM + quarter * 32, end = off[e + 1];
      const int col0 = local % n_nt * BN + half * COLS;
      const int nb = min(col0 / kFp8Block, a.NB - 1);
      const float* sa = a.a_scale + int64_t(min(row0 + lane, a.S - 1)) * a.lda_s;
      const float* sb = a.w_scale + (int64_t(e) * a.NB + nb) * a.KB;
      float acc[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) acc[i] = 0.f;
      float fa[kAhead], fb[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        fa[j] = __ldg(sa + min(j, a.KB - 1));
        fb[j] = __ldg(sb + min(j, a.KB - 1));
      }
      for (int kb0 = 0; ok && kb0 < a.KB; kb0 += kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const int kb = kb0 + j;
          if (kb >= a.KB) break;
          const float f = fa[j] * fb[j];
          const int ahead = min(kb + kAhead, a.KB - 1);
          fa[j] = __ldg(sa + ahead);
          fb[j] = __ldg(sb + ahead);
          ok = poll_warp(&acc_full[b], bph, a.err);
          if (!ok) break;
          fence_after();
          const uint32_t addr = lanes + b * BN;
          uint32_t p[32];
#pragma unroll
          for (int c = 0; c < COLS / 32; ++c) {
            tmem_ld32(addr + c * 32, p);
            tmem_wait(p);
            if (c + 1 == COLS / 32) {  // all of the block's columns are in registers: the buffer is free
              fence_before();  // every lane's reads come before the MMA that overwrites them, across the barrier
              __syncwarp();
              if (lane == 0) mbar_arrive(&acc_empty[b]);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c * 32 + i] = fmaf(__uint_as_float(p[i]), f, acc[c * 32 + i]);
          }
          if (++b == NBUF) b = 0, bph ^= 1u;
        }
      }
      if (!ok) {
        *abort_ptr = 1;
        break;
      }
      // through shared memory in pieces of 64 bytes per row, 16-byte chunks swizzled by pairs of rows
      constexpr int PW = 64 / int(sizeof(TO));  // columns per piece
      constexpr int CW = 16 / int(sizeof(TO));  // columns per chunk
      TO* dst = static_cast<TO*>(a.out) + int64_t(row0 + (lane >> 2)) * a.N + col0 + (lane & 3) * CW;
      // whole rows of one expert leave by a copy of their own (the warp's 32 rows, 64 bytes each, swizzled as the map
      // says); a tile that ends inside, or rows off 16 bytes, by the threads
      const bool copies = a.copy_out && row0 + 32 <= end;
#pragma unroll
      for (int pc = 0; pc < COLS / PW; ++pc) {
        if (lane == 0) tma_stores_read();  // the piece before has left
        __syncwarp();
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          float v[CW];
#pragma unroll
          for (int i = 0; i < CW; ++i) v[i] = acc[pc * PW + ch * CW + i];
          store_vec<TO, CW>(reinterpret_cast<TO*>(mine + lane * 64 + ((ch ^ ((lane >> 1) & 3)) << 4)), v);
        }
        const int col = col0 + pc * PW;
        if (copies) {
          fence_async();
          __syncwarp();
          if (lane == 0 && col < a.N) tma_store_2d(&map_out, col * int(sizeof(TO)), row0, mine);
        } else {
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = j * 8 + (lane >> 2), c = col + (lane & 3) * CW;
            const TO* src = reinterpret_cast<const TO*>(mine + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
            TO* d = dst + j * 8 * int64_t(a.N) + pc * PW;
            if (row0 + r >= end) continue;
            if (a.copy_out && c + CW <= a.N) {
              *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(src);
            } else {
              for (int i = 0; i < CW; ++i)
                if (c + i < a.N) d[i] = src[i];
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) tma_stores_done();
    if (a.offsets) zero_rows(static_cast<TO*>(a.out), a.N, off[0], off[a.E], a.S, threadIdx.x - kSumWarp0 * 32, kSumWarps * 32);
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
int launch_one(cudaStream_t s, const GemmArgs& a, const CUtensorMap& ma, const CUtensorMap& mw, const CUtensorMap& mo,
               int grid) {
  static std::atomic<uint64_t> attr_set{0};  // devices whose attribute is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -1;
  if (!(attr_set.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(fp8_gemm_kernel<BN, TO>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             int(Cfg<BN>::kSmem)) != cudaSuccess)
      return -1;
    attr_set.fetch_or(uint64_t(1) << dev);
  }
  return launch_chain(fp8_gemm_kernel<BN, TO>, dim3(grid), dim3(kThreads), Cfg<BN>::kSmem, s, a, ma, mw, mo) ==
                 cudaSuccess
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
  const int64_t out_bytes = int64_t(p.N) * (out_dtype == B200MOE_F32 ? 4 : 2);
  a.copy_out = out_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  CUtensorMap ma, mw, mo{};
  if (make_u8_tile_map(&ma, p.a, p.S, p.K, kFp8Block, kBM) ||
      make_u8_tile_map(&mw, p.w, int64_t(p.E) * p.N, p.K, kFp8Block, bn))
    return -1;
  if (a.copy_out && make_u8_store_map(&mo, p.out, p.S, out_bytes, 32)) return -1;
  const int grid = int(std::min<int64_t>(sms, m_tiles * ((p.N + bn - 1) / bn)));
  auto run = [&](auto one) { return one(s, a, ma, mw, mo, grid); };
  if (out_dtype == B200MOE_F16) return run(wide ? launch_one<256, __half> : launch_one<128, __half>);
  if (out_dtype == B200MOE_BF16) return run(wide ? launch_one<256, __nv_bfloat16> : launch_one<128, __nv_bfloat16>);
  return run(wide ? launch_one<256, float> : launch_one<128, float>);
}

}  // namespace b200moe

using namespace b200moe;

namespace {

int product_status(const Fp8Product& p, int out_dtype) {
  if (!p.w || !p.w_scale || !p.out || p.S < 1 || p.S > INT32_MAX - 256 || p.N < 1 || p.K < 16 || p.K % 16 || p.E < 1 || p.E > kMaxExperts ||
      (!p.offsets && p.E != 1) || int64_t(p.E) * p.N > INT32_MAX - 256 || p.K > (1 << 24))
    return B200MOE_ERR_INVALID_ARG;
  if (out_dtype < 0 || out_dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  if (reinterpret_cast<uintptr_t>(p.w) % 16) return B200MOE_ERR_ALIGN;
  return B200MOE_OK;
}

// The kernel by rows per matrix, as measured on B200 (us; kernels of 8, 16, 32 and 128 rows per tile, weights from HBM):
//   one matrix 4096 x 4096: 6.4 / 9.4 / 10.7 / 12.2 at 1 row, 8.0 / 9.5 / 10.8 / 12.0 at 8, - / 9.7 / 11.2 / 11.9 at 32,
//   - / 9.9 / 11.2 / 12.0 at 64, - / 15.9 / 11.3 / 12.2 at 96, - / 22.4 / 18.4 / 12.4 at 192: a tile of fewer rows gives
//   more CTAs, so the smallest whose tiles still run in one wave. So for the first too: 9472 x 2048 5.9 / 7.1 / 7.6 / -
//   in one wave; 9504 x 2048 8.9 / 7.1 / 7.6 / - with CTAs that walk on to a second tile, 14336 x 4096 19.1 / 13.0 /
//   13.7 / 21.5. The one wrong choice seen in one wave: 4096 x 6144, 13.7 / 12.6.
//   64 matrices 2816 x 2048, kernels of 32 and 128: 63 / 69 at 8 rows each, 65 / 71 at 24, 66 / 71 at 32, 111 / 72 at 48,
//   where experts above 32 rows read their weights twice; with rows as a Poisson draw 64 / 71 at 24 on average, 68 / 71
//   at 28, 87 / 71 at 32. 64 matrices 4096 x 4096: 163 / 169 at 8, 167 / 172 at 24, 252 / 178 at 32 drawn. 384 matrices
//   4096 x 4096: 900 / 1010 at 2, 1000 / 1020 at 8, 1070 / 1010 at 16, 1100 / 1015 at 24: there 24 is past the crossing.
//   S counts rows without an expert too, and no spread is known here: 288 rows over 48 matrices 2816 x 2048 with 2,016
//   rows dropped take 60 us and would take 56; 2,000 of 8,000 rows on one of 384 experts 1090 with either.
// Returns 8, 16, 32 or 128.
int choose(const Fp8Product& p) {
  if (!p.offsets) {
    const int64_t n_tiles = (p.N + 127) / 128;
    if (fp8_skinny_fits(p)) return 8;
    for (int t = 16; t <= 32; t *= 2)
      if ((p.S + t - 1) / t * n_tiles <= sm_count() && fp8_stream_fits(p.K, t)) return t;
    // more columns than one wave holds, bound by their bytes as long as one tile has all rows
    return p.S <= 32 && fp8_stream_fits(p.K, 32) ? 32 : 128;
  }
  return p.S <= 24 * int64_t(p.E) && fp8_stream_fits(p.K, 32) ? 32 : 128;
}

int launch_status(int rc) {
  if (rc == 0) return B200MOE_OK;
  cudaGetLastError();
  return B200MOE_ERR_CUDA;
}

}  // namespace

static int run_product(cudaStream_t s, const Fp8Product& p, int out_dtype) {
  const int kind = choose(p);
  return launch_status(kind == 8     ? launch_fp8_skinny(s, p, out_dtype)
                       : kind == 128 ? launch_fp8_gemm(s, p, out_dtype)
                                     : launch_fp8_stream(s, p, kind, out_dtype));
}

extern "C" int b200moe_fp8_matmul(void* stream, const void* a, const float* a_scale, int64_t a_scale_stride,
                                  const void* w, const float* w_scale, const int32_t* offsets, int S, int N, int K,
                                  int E, void* out, int out_dtype) {
  const Fp8Product p{a, a_scale, a_scale_stride, w, w_scale, offsets, out, S, N, K, E};
  const int st = product_status(p, out_dtype);
  if (st) return st;
  if (!a || !a_scale || a_scale_stride < 0) return B200MOE_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(a) % 16) return B200MOE_ERR_ALIGN;
  return run_product(static_cast<cudaStream_t>(stream), p, out_dtype);
}

extern "C" size_t b200moe_fp8_linear_workspace_bytes(int S, int N, int K) {
  const Fp8Product p{nullptr, nullptr, 0, nullptr, nullptr, nullptr, nullptr, S, N, K, 1};
  if (S < 1 || N < 1 || K < 1 || choose(p) == 8) return 0;
  const size_t q = (size_t(S) * K + 15) / 16 * 16;
  return q + size_t(S) * ((K + kFp8Block - 1) / kFp8Block) * sizeof(float);
}

extern "C" int b200moe_fp8_linear(void* stream, const void* x, int x_dtype, int64_t ldx, const void* w,
                                  const float* w_scale, int S, int N, int K, void* out, int out_dtype, void* workspace,
                                  size_t workspace_bytes) {
  Fp8Product p{nullptr, nullptr, 0, w, w_scale, nullptr, out, S, N, K, 1};
  const int st = product_status(p, out_dtype);
  if (st) return st;
  if (!x || ldx < 0) return B200MOE_ERR_INVALID_ARG;
  if (x_dtype < 0 || x_dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t ld_bytes = ldx * (x_dtype == B200MOE_F32 ? 4 : 2);
  if (choose(p) == 8 && x_dtype != B200MOE_F32 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld_bytes % 16 == 0)
    return launch_status(launch_fp8_skinny_x(s, p, x, x_dtype, ldx, out_dtype));
  const size_t q_bytes = (size_t(S) * K + 15) / 16 * 16, kb = (K + kFp8Block - 1) / kFp8Block;
  if (!workspace || workspace_bytes < q_bytes + size_t(S) * kb * sizeof(float)) return B200MOE_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return B200MOE_ERR_ALIGN;
  float* scale = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + q_bytes);
  const int qs = b200moe_fp8_quantize(stream, x, x_dtype, ldx, S, K, 0, 1.f, workspace, scale);
  if (qs) return qs;
  p.a = workspace;
  p.a_scale = scale;
  p.a_scale_stride = int64_t(kb);
  return run_product(s, p, out_dtype);
}
