// E4M3 products of few rows per matrix with a scale per block of 128, bound by
// the weight bytes: the weights are the tensor core's M (128 rows of w), the
// tokens its N (NTOK = 16 or 32 rows of a), so a weight byte goes from
// global memory to the tensor core through one TMA copy and no register.
//
// A persistent CTA per SM walks items = (expert, NTOK of its rows) x (128 weight
// rows), a contiguous range of them, so that it streams an expert's weights in
// order. Per K block of 128
//   warp 0 (producer): TMA boxes of 128 weight rows and NTOK token rows into a
//     ring of eight stages, 144 or 160 KB in flight;
//   warps 1 and 6 (MMA), a block each in turn: 4 x tcgen05.mma.kind::f8f6f4 (M 128,
//     N NTOK, K 32) into one of eight TMEM buffers;
//   warps 2-5 (sums): a thread holds one weight row; product times the weight
//     block's scale and each token's (in shared memory, four per load) joins the
//     f32 sums of its NTOK columns.
// 192 experts of 4096 x 4096 for 256 rows: 456 us, 7.06 TB/s (it reads only; a plain
// copy reaches 6.55). Streaming the weights through registers
// into mma.sync instead reached 4.9 TB/s at best. One matrix of 4096 x 4096 for 64
// rows has 32 x 4 items, so 20 SMs idle and each of the others walks K alone: 9.8 us,
// 0.18 per K block, the rest launch, first bytes and stores; one MMA warp took 1.5
// more. Up to 16 rows it has 32 items only and takes 9.6 us: K is not split.
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "fp8_device.cuh"
#include "fp8_ops.h"
#include "fp8_tc.cuh"
#include "internal.h"

namespace b200moe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kRows = 128;  // weight rows per item
constexpr int kThreads = 224;  // producer, four warps of sums, two of MMAs
constexpr int kWBytes = kRows * kFp8Block;
constexpr int kScaleBytes = 16 * 1024;  // the token tile's scales
constexpr int kBufs = 8;
constexpr int kAhead = 4;  // K blocks whose weight scales are loaded ahead

template <int NTOK>
struct Cfg {
  static constexpr int kStage = kWBytes + NTOK * kFp8Block;
  // even, as the TMEM buffers: a stage then stays with one of the two MMA warps. Were it shared, one warp could wait
  // for its second filling before the first has landed, and a parity wait would take the phase before for it. Eight
  // measure better than ten: 461 and 482 us for 190 experts of 4096 x 4096.
  static constexpr int kStages = 8;
  static_assert(kStages % 2 == 0 && kBufs % 2 == 0, "stages and buffers by MMA warp");
  static constexpr size_t kSmem = 1024 + size_t(kStages) * kStage + kScaleBytes + 512;
  static constexpr uint32_t kIdesc = (1u << 4) | (uint32_t(NTOK >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
  static_assert(kSmem + 8 * (kMaxExperts + 1) + 64 <= 227 * 1024, "shared memory, with the tile table");
  static_assert(kBufs * NTOK <= 512, "TMEM");
};

struct StreamArgs {
  const float* a_scale;
  int64_t lda_s;
  const float* w_scale;
  const int32_t* offsets;
  void* out;
  int S, N, E, KB, NB;
  uint32_t* err;
};

template <int NTOK, typename TO>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_stream_kernel(const StreamArgs a, const __grid_constant__ CUtensorMap map_a,
                      const __grid_constant__ CUtensorMap map_w) {
  using C = Cfg<NTOK>;
  constexpr int ST = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int off[kMaxExperts + 1], start[kMaxExperts + 1];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_flag;
  const uint32_t base_u32 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* stages = smem_raw + (base_u32 - smem_u32(smem_raw));          // [ST][weights 16 KB, tokens NTOK x 128]
  float* ss = reinterpret_cast<float*>(stages + ST * C::kStage);        // [KB][NTOK]
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(ss) + kScaleBytes);
  uint64_t* empty = full + ST;
  uint64_t* acc_full = empty + ST;
  uint64_t* acc_empty = acc_full + kBufs;
  volatile int* abort_ptr = &abort_flag;

  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kBufs; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4);
    }
    fence_barrier_init();
    abort_flag = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_sh)),
                 "r"(uint32_t(kBufs * NTOK)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_base_sh;
  pdl_wait();
  const int n_wt = (a.N + kRows - 1) / kRows;
  build_tile_table(a.offsets, a.E, a.S, NTOK, n_wt, off, start, a.err);
  const int n_items = start[a.E];
  const int first = int(int64_t(n_items) * blockIdx.x / gridDim.x);
  const int stop = int(int64_t(n_items) * (blockIdx.x + 1) / gridDim.x);

  if (warp == 0) {
    int st = 0;
    uint32_t ph = 0, issued = 0, par = 0;
    bool ok = true;
    for (int item = first; ok && item < stop; ++item) {
      const int e = tile_expert(start, a.E, item), local = item - start[e];
      const int row = off[e] + local / n_wt * NTOK, wrow = e * a.N + local % n_wt * kRows;
      for (int kb = 0; kb < a.KB; ++kb) {
        ok = !__any_sync(0xffffffffu, *abort_ptr) && poll_warp(&empty[st], ph ^ 1u, a.err);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* dst = stages + st * C::kStage;
          mbar_arrive_expect_tx(&full[st], uint32_t(C::kStage));
          tma_2d(dst, &map_w, kb * kFp8Block, wrow, &full[st]);
          tma_2d(dst + kWBytes, &map_a, kb * kFp8Block, row, &full[st]);
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
  } else if (warp == 1 || warp == 6) {
    // two warps take the K blocks in turn, whatever their items: one block's four MMAs and two commits take 250 clocks
    // to issue, where its bytes arrive in 180
    const int64_t total = int64_t(stop - first) * a.KB;
    int st = warp == 6, b = st, last = 0;
    uint32_t ph = 0, bph = 0, last_ph = 0;
    bool ok = true, committed = false;
    const uint64_t d0 = desc_sw128(smem_u32(stages));
    for (int64_t g = st; ok && g < total; g += 2) {
      ok = poll_warp(&full[st], ph, a.err) && poll_warp(&acc_empty[b], bph ^ 1u, a.err);
      if (!ok) break;
      fence_after();
      const uint64_t d = d0 + st * (C::kStage >> 4);
      if (elect_one()) {
        mma_block(tmem + b * NTOK, d, d + (kWBytes >> 4), C::kIdesc);
        commit(&empty[st]);
        commit(&acc_full[b]);
      }
      __syncwarp();
      committed = true;
      last = b;
      last_ph = bph;
      if ((st += 2) >= ST) st -= ST, ph ^= 1u;
      if ((b += 2) >= kBufs) b -= kBufs, bph ^= 1u;
    }
    if (!ok) *abort_ptr = 1;
    if (committed) poll_warp(&acc_full[last], last_ph, a.err);
  } else {
    const int quarter = warp & 3, tid = threadIdx.x - 64;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
    TO* out = static_cast<TO*>(a.out);
    int b = 0, staged = -1;
    uint32_t bph = 0;
    bool ok = true;
    // after a wait that ran out the items still pass, without waits and stores: the four warps meet at the same barriers
    for (int item = first; item < stop; ++item) {
      const int e = tile_expert(start, a.E, item), local = item - start[e];
      const int row0 = off[e] + local / n_wt * NTOK, end = off[e + 1], n0 = local % n_wt * kRows;
      if (row0 != staged) {  // a new token tile: its scales, by K block
        named_bar(1, 128);
        for (int i = tid; i < NTOK * a.KB; i += 128) {
          const int kb = i / NTOK, j = i - kb * NTOK;
          ss[i] = row0 + j < end ? __ldg(a.a_scale + (row0 + j) * a.lda_s + kb) : 0.f;
        }
        named_bar(1, 128);
        staged = row0;
      }
      const float* sb = a.w_scale + (int64_t(e) * a.NB + n0 / kFp8Block) * a.KB;
      float acc[NTOK], fb[kAhead];
#pragma unroll
      for (int i = 0; i < NTOK; ++i) acc[i] = 0.f;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) fb[j] = __ldg(sb + min(j, a.KB - 1));
      for (int kb0 = 0; ok && kb0 < a.KB; kb0 += kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const int kb = kb0 + j;
          if (kb >= a.KB) break;
          const float f = fb[j];
          fb[j] = __ldg(sb + min(kb + kAhead, a.KB - 1));
          ok = poll_warp(&acc_full[b], bph, a.err);
          if (!ok) break;
          fence_after();
          const float4* s4 = reinterpret_cast<const float4*>(ss + kb * NTOK);
#pragma unroll
          for (int c = 0; c < NTOK / 16; ++c) {
            uint32_t p[16];
            tmem_ld16(lanes + b * NTOK + c * 16, p);
            tmem_wait(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 s = s4[c * 4 + i];
              float* o = acc + c * 16 + i * 4;
              o[0] = fmaf(__uint_as_float(p[4 * i]), f * s.x, o[0]);
              o[1] = fmaf(__uint_as_float(p[4 * i + 1]), f * s.y, o[1]);
              o[2] = fmaf(__uint_as_float(p[4 * i + 2]), f * s.z, o[2]);
              o[3] = fmaf(__uint_as_float(p[4 * i + 3]), f * s.w, o[3]);
            }
          }
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[b]);
          if (++b == kBufs) b = 0, bph ^= 1u;
        }
      }
      if (!ok) *abort_ptr = 1;
      const int col = n0 + quarter * 32 + lane;
      if (ok && col < a.N) {
#pragma unroll
        for (int i = 0; i < NTOK; ++i)
          if (row0 + i < end) out[int64_t(row0 + i) * a.N + col] = from_f32<TO>(acc[i]);
      }
    }
    if (a.offsets) zero_rows(out, a.N, off[0], off[a.E], a.S, tid, 128);
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(uint32_t(kBufs * NTOK)));
  }
  pdl_trigger();
}

template <int NTOK, typename TO>
int launch_one(cudaStream_t s, const StreamArgs& a, const CUtensorMap& ma, const CUtensorMap& mw, int grid) {
  static std::atomic<uint64_t> attr_set{0};  // devices whose attribute is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -1;
  if (!(attr_set.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(fp8_stream_kernel<NTOK, TO>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             int(Cfg<NTOK>::kSmem)) != cudaSuccess)
      return -1;
    attr_set.fetch_or(uint64_t(1) << dev);
  }
  return launch_chain(fp8_stream_kernel<NTOK, TO>, dim3(grid), dim3(kThreads), Cfg<NTOK>::kSmem, s, a, ma, mw) ==
                 cudaSuccess
             ? 0
             : -1;
}

template <int NTOK>
int launch_tok(cudaStream_t s, const Fp8Product& p, int out_dtype) {
  StreamArgs a{};
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
  CUtensorMap ma, mw;
  if (make_u8_tile_map(&ma, p.a, p.S, p.K, kFp8Block, NTOK) ||
      make_u8_tile_map(&mw, p.w, int64_t(p.E) * p.N, p.K, kFp8Block, kRows))
    return -1;
  // upper bound of the token tiles: one per NTOK rows and one more for every expert with rows
  const int64_t tiles = p.offsets ? int64_t(p.S) / NTOK + std::min(p.E, p.S) : (p.S + NTOK - 1) / NTOK;
  const int grid = int(std::min<int64_t>(sm_count(), tiles * ((p.N + kRows - 1) / kRows)));
  if (out_dtype == B200MOE_F16) return launch_one<NTOK, __half>(s, a, ma, mw, grid);
  if (out_dtype == B200MOE_BF16) return launch_one<NTOK, __nv_bfloat16>(s, a, ma, mw, grid);
  return launch_one<NTOK, float>(s, a, ma, mw, grid);
}

}  // namespace

bool fp8_stream_fits(int K, int rows_per_tile) {
  return (K + kFp8Block - 1) / kFp8Block * rows_per_tile * int(sizeof(float)) <= kScaleBytes;
}

int launch_fp8_stream(cudaStream_t s, const Fp8Product& p, int rows_per_tile, int out_dtype) {
  return rows_per_tile <= 16 ? launch_tok<16>(s, p, out_dtype) : launch_tok<32>(s, p, out_dtype);
}

}  // namespace b200moe
