// Large products of 4-bit floating point rows and weights: as fp4_matmul.cu, with two
// CTAs of a cluster on one tile of 256 rows x 256 columns (tcgen05 cta_group::2).
//
// Each CTA brings 128 rows of a and 128 of w per stage, and the tensor cores of both
// read the other's half of w: 32 KB of codes per SM for the work that takes one CTA
// with a tile of 128 x 256 48 KB (whose TMA traffic alone, 16.8 TB/s from L2, takes 48
// us for 8192 x 4096 x 4096).  Accumulator, scales of the rows and epilogue are each
// CTA's own; the scales of all 256 columns are in both.  The even CTA's warp 1 issues
// for both; codes and scales of both count on its barriers, and its commits arrive at
// both CTAs' barriers.
//   warp 0 (producer), 1 (MMA, even CTA), 4-7 (epilogue), 2, 3, 8
//   and 9 (scales), 10 (their chunks).
// Two accumulators of 256 columns and the scales exceed TMEM's 512 columns: the
// accumulators share 64 columns, which the epilogue empties first.
//
// Bound: 8192 x 4096 x 4096 NVFP4 59 us, MXFP4 51 (4.7 and 5.3 PFLOP/s; 8192^3 5.1 and
// 6.1): the tensor pipe is busy 54 and 61 % of the time at the 1.65 GHz that the power
// cap leaves. Without MMAs the copies and scales take 48 us, without the scales 59 and
// without their copies to TMEM too 54: the copies' latency over a ring of 128 or 160 KB.
#include <algorithm>
#include <atomic>

#include "fp4_tiles.cuh"

namespace b200moe {
namespace {

constexpr int kThreads = 352;
constexpr int kTile = 256;  // rows and columns of a pair's tile
constexpr int kHalf = 128;  // of them that a CTA brings
constexpr int kStage = 2 * kFp4ABytes;
constexpr int kChunks = 2;
constexpr int kSfBytes = 3 * kSfBlock;
constexpr int kSfBufs = kScaleWarps;
constexpr int kOutBytes = 32 * 64;  // per epilogue warp
constexpr int kSharedCols = 64;     // of both accumulators
constexpr int kAcc1 = kTile - kSharedCols;
constexpr int kSf0 = 2 * kTile - kSharedCols;
constexpr int kSfCols = 12;  // TMEM columns of 64 columns of K
static_assert(kSf0 + 4 * kSfCols <= 512, "TMEM columns");
static_assert(4 * kOutBytes >= 4 * (kFp4MaxExperts + 1), "the offsets, while the tile table is made");

// NVFP4's chunks hold four stages (64 bytes of a row) beside four stages of codes, MXFP4's (32 bytes) beside five:
// 8192 x 4096 x 4096 takes NVFP4 59 us, 61 with the other's, and MXFP4 51, 53 to 64 with the other's.
template <int FMT>
struct Cfg {
  static constexpr int kStages = FMT == kMx ? 5 : 4;
  static constexpr int kChunkRow = FMT == kMx ? 32 : 64;  // bytes of a row's scales per chunk
  static constexpr int kChunk = (kHalf + kTile) * kChunkRow;
  static constexpr size_t kSmem = 1024 + kStages * kStage + kChunks * kChunk + kSfBufs * kSfBytes + 4 * kOutBytes +
                                  8 * (2 * kStages + 2 * kChunks + 2 * kSfBufs + 4);
  static_assert(kSmem + 4 * (kFp4MaxExperts + 2) + 64 <= 227 * 1024, "shared memory, with the tile table");
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// A shared address of this CTA as the even CTA's.
__device__ __forceinline__ uint32_t even_cta(const void* p) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// What these arrivals announce lies in the arriving CTA's own shared memory and TMEM, which its own SM reads for the pair's
// instruction, and is ordered before them by fence.proxy.async and tcgen05.fence: no release over the cluster, which takes
// 75 us for 8192 x 4096 x 4096 where the default one takes 59.
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// poll_warp for barriers that the other CTA arrives at.
__device__ __forceinline__ bool poll_cluster(uint64_t* bar, uint32_t parity, uint32_t* err) {
  const uint32_t addr = smem_u32(bar);
  uint64_t t0 = 0;
  for (uint32_t it = 1;; ++it) {
    uint32_t done;
    asm volatile(
        "{ .reg .pred p; mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, done)) return true;
    if ((it & 1023u) == 0) {
      const uint64_t t = __shfl_sync(0xffffffffu, global_timer_ns(), 0);
      if (t0 == 0) {
        t0 = t;
      } else if (t - t0 > kWaitLimitNs) {
        set_error(err, kErrTimeout);
        return false;
      }
    }
  }
}
// Into this CTA's shared memory, counted on a barrier of the pair.
__device__ __forceinline__ void tma_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// At the same place in both CTAs, when the MMAs and copies issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(smem_u32(bar)),
      "h"(uint16_t(3))
      : "memory");
}

template <int FMT, typename TO>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    fp4_pair_kernel(const TileArgs a, const __grid_constant__ TileMaps maps) {
  using C = Cfg<FMT>;
  constexpr int kStages = C::kStages, kChunkRow = C::kChunkRow, kChunk = C::kChunk;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int start[kFp4MaxExperts + 2];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_flag;
  const uint32_t base_u32 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* stages = smem_raw + (base_u32 - smem_u32(smem_raw));  // [kStages][a 16 KB, w 16 KB]
  uint8_t* chunks = stages + kStages * kStage;                  // [2][128 rows of a, 256 of w]
  uint8_t* sf = chunks + kChunks * kChunk;                      // [4][a 2 KB, w 4 KB]
  uint8_t* stage_out = sf + kSfBufs * kSfBytes;                 // [4][2 KB]
  uint64_t* full = reinterpret_cast<uint64_t*>(stage_out + 4 * kOutBytes);
  uint64_t* empty = full + kStages;
  uint64_t* chunk_full = empty + kStages;
  uint64_t* chunk_empty = chunk_full + kChunks;
  uint64_t* sf_full = chunk_empty + kChunks;
  uint64_t* sf_empty = sf_full + kSfBufs;
  uint64_t* acc_full = sf_empty + kSfBufs;  // [2]
  uint64_t* acc_empty = acc_full + 2;       // [2]
  volatile int* abort_ptr = &abort_flag;

  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = int(cluster_rank());
  const bool w_chunks = a.w_align == 16;  // else the weights' scales come by loads
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int c = 0; c < kChunks; ++c) {
      mbar_init(&chunk_full[c], 1);
      mbar_init(&chunk_empty[c], kScaleWarps);
    }
    for (int b = 0; b < kSfBufs; ++b) {
      mbar_init(&sf_full[b], 2);  // a warp of each CTA
      mbar_init(&sf_empty[b], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);  // four warps of both CTAs
    }
    fence_barrier_init();
    abort_flag = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_sh)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  if (threadIdx.x == 0) prefetch_maps(maps, w_chunks, a.copy_out);
  fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers stand before either arrives at the other's
  fence_after();
  const uint32_t tmem = tmem_base_sh;
  pdl_wait();
  const int n_ct = (a.N + kTile - 1) / kTile;
  // the offsets stand in the output's staging until the table is made, and are read from global memory after
  build_tile_table(a.offsets, a.E, a.S, kTile, n_ct, reinterpret_cast<int*>(stage_out), start, a.err);
  auto off = [&](int e) { return a.offsets ? __ldg(a.offsets + e) : e ? a.S : 0; };
  const Tiles tiles{int(blockIdx.x / 2), start[a.E], int(gridDim.x / 2)};
  const int n_kt = (a.K + kFp4StageK - 1) / kFp4StageK, n_k64 = (a.K + 63) / 64;

  if (warp == 0) {
    int st = 0;
    uint32_t ph = 0, issued = 0, par = 0;
    bool ok = true;
    for (int item = tiles.first(); ok && item < tiles.stop(); item = tiles.next(item)) {
      const int e = tile_expert(start, a.E, item), local = item - start[e];
      const int ra = off(e) + local / n_ct * kTile + rank * kHalf, rw = e * a.N + local % n_ct * kTile;
      for (int kt = 0; kt < n_kt; ++kt) {
        ok = !__any_sync(0xffffffffu, *abort_ptr) && poll_cluster(&empty[st], ph ^ 1u, a.err);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* dst = stages + st * kStage;
          if (rank == 0) mbar_arrive_expect_tx(&full[st], uint32_t(2 * kStage));  // the other CTA's too
          const uint32_t bar = even_cta(&full[st]);
          tma_2d_pair(dst, &maps.a, kt * kFp4RowBytes, ra, bar);
          tma_2d_pair(dst + kFp4ABytes, &maps.w, kt * kFp4RowBytes, rw + rank * kHalf, bar);
        }
        issued |= 1u << st;
        par = (par & ~(1u << st)) | (ph << st);
        if (++st == kStages) st = 0, ph ^= 1u;
      }
    }
    if (!ok) *abort_ptr = 1;
    // no copy may be in flight when the pair exits: the even CTA's barriers count both CTAs' codes
    for (int s = 0; rank == 0 && s < kStages; ++s)
      if (issued & (1u << s)) poll_cluster(&full[s], (par >> s) & 1u, a.err);
  } else if (warp == 1) {
    int st = 0, sb = 0, tile = 0, last = 0;
    uint32_t ph = 0, sph = 0, last_ph = 0;
    bool ok = true, committed = false;
    const uint64_t d0 = desc_sw128(smem_u32(stages)), s0 = desc_sf(smem_u32(sf));
    for (int item = rank == 0 ? tiles.first() : tiles.stop(); ok && item < tiles.stop(); item = tiles.next(item), ++tile) {
      const int b = tile & 1;
      if (tile >= 1) {  // the tile before has left the shared columns, and with that the one before it its own
        ok = poll_cluster(&acc_empty[b ^ 1], ((tile - 1) >> 1) & 1, a.err);
        if (!ok) break;
        fence_after();
      }
      const uint32_t d = tmem + b * kAcc1;
      for (int kt = 0; kt < n_kt; ++kt) {
        ok = poll_cluster(&full[st], ph, a.err) && poll_cluster(&sf_full[sb], sph, a.err);
        if (!ok) break;
        fence_after();
        const uint64_t da = d0 + st * (kStage >> 4), ds = s0 + sb * (kSfBytes >> 4);
        const int steps = min(4, n_k64 - 4 * kt);
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j >= steps) break;
            const uint32_t sfa = tmem + kSf0 + j * kSfCols, sfb = sfa + 4;
#pragma unroll
            for (int n = 0; n < 3; ++n) sf_copy<2>(sfa + 4 * n, ds + n * (kSfBlock >> 4) + j * 32);
            mma_fp4<2, FMT>(d, da + 2 * j, da + (kFp4ABytes >> 4) + 2 * j, sfa, sfb, uint32_t(kt | j),
                            fp4_idesc<kTile, kTile, FMT>());
          }
          commit_pair(&empty[st]);
          commit_pair(&sf_empty[sb]);
          if (kt == n_kt - 1) commit_pair(&acc_full[b]);
        }
        __syncwarp();
        if (++st == kStages) st = 0, ph ^= 1u;
        if (++sb == kSfBufs) sb = 0, sph ^= 1u;
      }
      if (!ok && elect_one()) commit_pair(&acc_full[b]);  // a partial tile too, so that its MMAs can be waited for
      __syncwarp();
      committed = true;
      last = b;
      last_ph = (tile >> 1) & 1;
    }
    if (!ok) *abort_ptr = 1;
    if (committed) poll_cluster(&acc_full[last], last_ph, a.err);
  } else if (warp >= 4 && warp < 8) {
    const int quarter = warp & 3;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
    int tile = 0;
    bool ok = true;
    for (int item = tiles.first(); ok && item < tiles.stop(); item = tiles.next(item), ++tile) {
      const int e = tile_expert(start, a.E, item), local = item - start[e], end = off(e + 1);
      const int row0 = off(e) + local / n_ct * kTile + rank * kHalf + quarter * 32, col0 = local % n_ct * kTile;
      const Fp4Factors f = fp4_factors(row_factor(a, row0 + lane), a.w_factor ? __ldg(a.w_factor + e) : 1.f);
      const int b = tile & 1;
      ok = poll_cluster(&acc_full[b], (tile >> 1) & 1, a.err);
      if (!ok) break;
      fence_after();
      const uint32_t bar = even_cta(&acc_empty[b]);
      // the shared columns first: the last two pieces of accumulator 0, the first two of accumulator 1
      constexpr int kTileOut = 32 * kTile * int(sizeof(TO));  // of a warp
      static_assert(4 * kTileOut <= kStages * kStage, "the last tile's room");
      const bool last = tiles.next(item) >= tiles.stop();
      uint8_t* mine = last ? stages + quarter * kTileOut : stage_out + quarter * kOutBytes;
      store_tile<kTile, TO>(a, &maps.out, lanes + b * kAcc1, mine, row0, end, col0, f, b ? 0 : kAcc1 / 32,
                            kSharedCols / 32, last, [&] { arrive_at(bar); });
    }
    if (!ok) *abort_ptr = 1;
    if (lane == 0) tma_stores_done();
    if (a.offsets)
      zero_rows(static_cast<TO*>(a.out), a.N, off(0), start[a.E + 1], a.S, threadIdx.x - 128, 128);
  } else {
    const ScaleWay way{chunks, kChunk, kChunks, chunk_full, chunk_empty, sf, sf_empty, kTile};
    auto w_row = [&](int item) {
      const int e = tile_expert(start, a.E, item);
      return e * a.N + (item - start[e]) % n_ct * kTile;
    };
    if (warp == 10) {
      auto load = [&](int slot, int item, int x, uint64_t* bar) {
        const int e = tile_expert(start, a.E, item), local = item - start[e];
        uint8_t* dst = chunks + slot * kChunk;
        tma_2d(dst, &maps.sa, x, off(e) + local / n_ct * kTile + rank * kHalf, bar);
        if (w_chunks) tma_2d(dst + kHalf * kChunkRow, &maps.sw, x, e * a.N + local % n_ct * kTile, bar);
      };
      chunk_warp<FMT, kChunkRow>(a, tiles, way, uint32_t((kHalf + (w_chunks ? kTile : 0)) * kChunkRow), load, abort_ptr);
    } else {
      scale_warp_by<FMT, kChunkRow, 3, false>(warp < 4 ? warp - 2 : warp - 6, a, tiles, way, w_row,
                                   [&](int b) { arrive_at(even_cta(&sf_full[b])); }, abort_ptr);
    }
  }
  fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA's memory goes while the other may use it
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
  pdl_trigger();
}

// Pairs that run at once: an SM without a partner in its group of SMs stays idle.
template <typename K>
int resident_pairs(K kernel, size_t smem) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (sm_count() / 2));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {2, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = sm_count() / 2;
  }
  return std::min(n, sm_count() / 2);
}

template <int FMT, typename TO>
int launch_one(cudaStream_t s, const TileArgs& a, const TileMaps& m, int64_t tiles) {
  static std::atomic<uint64_t> attr_set{0};  // devices whose attribute is set
  static std::atomic<int> pairs{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -1;
  auto kernel = fp4_pair_kernel<FMT, TO>;
  if (!(attr_set.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Cfg<FMT>::kSmem)) != cudaSuccess)
      return -1;
    attr_set.fetch_or(uint64_t(1) << dev);
  }
  if (!pairs.load()) pairs.store(resident_pairs(kernel, Cfg<FMT>::kSmem));
  const int grid = 2 * int(std::min<int64_t>(pairs.load(), tiles));
  return launch_chain(kernel, dim3(grid), dim3(kThreads), Cfg<FMT>::kSmem, s, a, m) == cudaSuccess ? 0 : -1;
}

}  // namespace

int launch_fp4_pairs(cudaStream_t s, const Fp4Product& p, int out_dtype) {
  TileArgs a{};
  TileMaps m{};
  const int chunk_row = p.format == kMx ? Cfg<kMx>::kChunkRow : Cfg<kNv>::kChunkRow;
  if (make_tile_args(p, out_dtype, kHalf, kHalf, kHalf, kTile, chunk_row, true, a, m)) return -1;
  // upper bound of the row tiles: one per 256 rows and one more for every expert with rows
  const int64_t row_tiles = p.offsets ? int64_t(p.S) / kTile + std::min(p.E, p.S) : (p.S + kTile - 1) / kTile;
  const int64_t tiles = row_tiles * ((p.N + kTile - 1) / kTile);
  auto run = [&](auto f16, auto bf16, auto f32) {
    return (out_dtype == B200MOE_F16 ? f16 : out_dtype == B200MOE_BF16 ? bf16 : f32)(s, a, m, tiles);
  };
  return p.format == kMx ? run(launch_one<kMx, __half>, launch_one<kMx, __nv_bfloat16>, launch_one<kMx, float>)
                         : run(launch_one<kNv, __half>, launch_one<kNv, __nv_bfloat16>, launch_one<kNv, float>);
}

}  // namespace b200moe
