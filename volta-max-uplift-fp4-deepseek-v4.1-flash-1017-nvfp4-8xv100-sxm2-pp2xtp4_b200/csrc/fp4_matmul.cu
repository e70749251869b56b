// Products of 4-bit floating point rows and weights on the 5th-generation tensor
// cores: tcgen05.mma.kind::mxf4nvf4 takes E2M1 operands as they are and their
// block scales (E4M3 per 16 for NVFP4, E8M0 per 32 for MXFP4) from TMEM, so one
// accumulation in TMEM runs over all of K and the epilogue has the rows' and the
// matrices' factors left to apply.
//
// A persistent CTA per SM walks tiles; per 256 columns of K (a stage: 128 bytes of
// codes per row, 128-byte swizzle)
//   warp 0 (producer): two TMA boxes of codes, 128 rows of the MMA's M and BN of
//     its N, into a ring of stages;
//   warp 10 brings the scales in chunks (fp4_tiles.cuh), and warps 2, 3, 8 and 9 put
//     a stage's each in turn in the order that tcgen05.cp wants;
//   warp 1 (MMA): per 64 columns tcgen05.cp of the block scales into one of four
//     places in TMEM and one MMA (M 128, N BN, K 64). Copies and MMAs of one
//     thread run in order, so a place is safe to write again four MMAs later;
//   warps 4-7 (epilogue): a thread holds one TMEM lane; the sums leave, times
//     both factors, while the next tile's MMAs run in the other accumulator.
// With rows as the MMA's M (BN = 128) it serves products of too few tiles for the
// pairs of CTAs of fp4_pair.cu.  SWAP: the weights are the MMA's M and BN = 16, 32
// or 64 rows of a its N, for few rows per matrix: then the kernel streams weights,
// and a thread of the epilogue holds one output column: 182 experts of 4096 x 4096
// for 256 rows in 255 us (6.7 TB/s; it reads only, a plain copy reaches 6.5).
#include <algorithm>
#include <atomic>

#include "fp4_tiles.cuh"

namespace b200moe {
namespace {

constexpr int kThreads = 352;
constexpr int kOutBytes = 32 * 64;  // per epilogue warp: 32 rows in pieces of 64 bytes
constexpr int kSfBufs = kScaleWarps;
constexpr int kChunkRow = 64;       // bytes of a row's scales per chunk

template <int BN>
struct Cfg {
  static constexpr int kStage = kFp4ABytes + BN * kFp4RowBytes;
  static constexpr int kStages = BN >= 128 ? 5 : BN >= 64 ? 6 : 8;
  static constexpr int kChunk = (kFp4M + BN) * kChunkRow;
  static constexpr int kChunks = BN >= 128 ? 2 : 3;
  static constexpr int kSfBytes = 2 * kSfBlock;
  static constexpr int kSf0 = 2 * BN;  // TMEM columns: two accumulators, four places for scales of 4 + 4 columns
  static constexpr int kTmem = kSf0 + 32 <= 64 ? 64 : kSf0 + 32 <= 128 ? 128 : kSf0 + 32 <= 256 ? 256 : 512;
  static constexpr size_t kSmem = 1024 + size_t(kStages) * kStage + kChunks * kChunk + kSfBufs * kSfBytes + 4 * kOutBytes +
                                  8 * (2 * kStages + 2 * kChunks + 2 * kSfBufs + 4);
  static_assert(4 * kOutBytes >= 4 * (kFp4MaxExperts + 1), "the offsets, while the tile table is made");
  static_assert(kSmem + 4 * (kFp4MaxExperts + 2) + 64 <= 227 * 1024, "shared memory, with the tile table");
};

template <int BN, bool SWAP, int FMT, typename TO>
__global__ void __launch_bounds__(kThreads, 1) fp4_kernel(const TileArgs a, const __grid_constant__ TileMaps maps) {
  using C = Cfg<BN>;
  constexpr int ST = C::kStages, CH = C::kChunks;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int start[kFp4MaxExperts + 2];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_flag;
  const uint32_t base_u32 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* stages = smem_raw + (base_u32 - smem_u32(smem_raw));  // [ST][M 16 KB, N BN x 128]
  uint8_t* chunks = stages + ST * C::kStage;                    // [CH][M 8 KB, N BN x 64]
  uint8_t* sf = chunks + CH * C::kChunk;                        // [4][M 2 KB, N 2 KB]
  uint8_t* stage_out = sf + kSfBufs * C::kSfBytes;              // [4][2 KB]
  uint64_t* full = reinterpret_cast<uint64_t*>(stage_out + 4 * kOutBytes);
  uint64_t* empty = full + ST;
  uint64_t* chunk_full = empty + ST;
  uint64_t* chunk_empty = chunk_full + CH;
  uint64_t* sf_full = chunk_empty + CH;
  uint64_t* sf_empty = sf_full + kSfBufs;
  uint64_t* acc_full = sf_empty + kSfBufs;  // [2]
  uint64_t* acc_empty = acc_full + 2;       // [2]
  volatile int* abort_ptr = &abort_flag;

  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const bool w_chunks = a.w_align == 16;  // else the weights' scales come by loads
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int c = 0; c < CH; ++c) {
      mbar_init(&chunk_full[c], 1);
      mbar_init(&chunk_empty[c], kScaleWarps);
    }
    for (int b = 0; b < kSfBufs; ++b) {
      mbar_init(&sf_full[b], 1);
      mbar_init(&sf_empty[b], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4);
    }
    fence_barrier_init();
    abort_flag = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_sh)),
                 "r"(uint32_t(C::kTmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 0) prefetch_maps(maps, w_chunks, a.copy_out);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_base_sh;
  pdl_wait();
  const int row_tile = SWAP ? BN : kFp4M, col_tile = SWAP ? kFp4M : BN;
  const int n_ct = (a.N + col_tile - 1) / col_tile;
  // the offsets stand in the output's staging until the table is made, and are read from global memory after
  build_tile_table(a.offsets, a.E, a.S, row_tile, n_ct, reinterpret_cast<int*>(stage_out), start, a.err);
  auto off = [&](int e) { return a.offsets ? __ldg(a.offsets + e) : e ? a.S : 0; };
  const int n_items = start[a.E];
  Tiles tiles{int(blockIdx.x), n_items, int(gridDim.x)};
  if (SWAP)
    tiles = {int(int64_t(n_items) * blockIdx.x / gridDim.x), int(int64_t(n_items) * (blockIdx.x + 1) / gridDim.x), 1};
  const int n_kt = (a.K + kFp4StageK - 1) / kFp4StageK, n_k64 = (a.K + 63) / 64;

  if (warp == 0) {
    int st = 0;
    uint32_t ph = 0, issued = 0, par = 0;
    bool ok = true;
    for (int item = tiles.first(); ok && item < tiles.stop(); item = tiles.next(item)) {
      const int e = tile_expert(start, a.E, item), local = item - start[e];
      const int ra = off(e) + local / n_ct * row_tile, rw = e * a.N + local % n_ct * col_tile;
      for (int kt = 0; kt < n_kt; ++kt) {
        ok = !__any_sync(0xffffffffu, *abort_ptr) && poll_warp(&empty[st], ph ^ 1u, a.err);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* dst = stages + st * C::kStage;
          mbar_arrive_expect_tx(&full[st], uint32_t(C::kStage));
          tma_2d(dst, SWAP ? &maps.w : &maps.a, kt * kFp4RowBytes, SWAP ? rw : ra, &full[st]);
          tma_2d(dst + kFp4ABytes, SWAP ? &maps.a : &maps.w, kt * kFp4RowBytes, SWAP ? ra : rw, &full[st]);
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
  } else if (warp == 1) {
    int st = 0, sb = 0, tile = 0, last = 0;
    uint32_t ph = 0, sph = 0, last_ph = 0;
    bool ok = true, committed = false;
    const uint64_t d0 = desc_sw128(smem_u32(stages)), s0 = desc_sf(smem_u32(sf));
    for (int item = tiles.first(); ok && item < tiles.stop(); item = tiles.next(item), ++tile) {
      const int b = tile & 1;
      if (tile >= 2) {
        ok = poll_warp(&acc_empty[b], ((tile >> 1) & 1) ^ 1, a.err);
        if (!ok) break;
        fence_after();
      }
      const uint32_t d = tmem + b * BN;
      for (int kt = 0; kt < n_kt; ++kt) {
        ok = poll_warp(&full[st], ph, a.err) && poll_warp(&sf_full[sb], sph, a.err);
        if (!ok) break;
        fence_after();
        const uint64_t da = d0 + st * (C::kStage >> 4), ds = s0 + sb * (C::kSfBytes >> 4);
        const int steps = min(4, n_k64 - 4 * kt);
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j >= steps) break;
            const uint32_t sfa = tmem + C::kSf0 + j * 8, sfb = sfa + 4;
            sf_copy<1>(sfa, ds + j * 32);
            sf_copy<1>(sfb, ds + (kSfBlock >> 4) + j * 32);
            mma_fp4<1, FMT>(d, da + 2 * j, da + (kFp4ABytes >> 4) + 2 * j, sfa, sfb, uint32_t(kt | j),
                            fp4_idesc<kFp4M, BN, FMT>());
          }
          commit(&empty[st]);
          commit(&sf_empty[sb]);
          if (kt == n_kt - 1) commit(&acc_full[b]);
        }
        __syncwarp();
        if (++st == ST) st = 0, ph ^= 1u;
        if (++sb == kSfBufs) sb = 0, sph ^= 1u;
      }
      if (!ok && elect_one()) commit(&acc_full[b]);  // a partial tile too, so that its MMAs can be waited for
      __syncwarp();
      committed = true;
      last = b;
      last_ph = (tile >> 1) & 1;
    }
    if (!ok) *abort_ptr = 1;
    if (committed) poll_warp(&acc_full[last], last_ph, a.err);
  } else if (warp >= 4 && warp < 8) {
    const int quarter = warp & 3;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
    TO* out = static_cast<TO*>(a.out);
    int tile = 0;
    bool ok = true;
    for (int item = tiles.first(); ok && item < tiles.stop(); item = tiles.next(item), ++tile) {
      const int e = tile_expert(start, a.E, item), local = item - start[e], end = off(e + 1);
      const int row0 = off(e) + local / n_ct * row_tile, col0 = local % n_ct * col_tile;
      const float fw = a.w_factor ? __ldg(a.w_factor + e) : 1.f;
      const int b = tile & 1;
      const uint32_t acc = lanes + b * BN;
      if constexpr (SWAP) {
        const Fp4Factors f0 = fp4_factors(lane < BN ? row_factor(a, row0 + lane) : 1.f, fw);
        const Fp4Factors f1 = BN > 32 ? fp4_factors(row_factor(a, row0 + 32 + lane), fw) : Fp4Factors{1.f, 1.f};
        const bool two = __any_sync(0xffffffffu, f0.second != 1.f || f1.second != 1.f);  // hardly ever
        const float last0 = two ? f0.second : f0.first, last1 = two ? f1.second : f1.first;
        ok = poll_warp(&acc_full[b], (tile >> 1) & 1, a.err);
        if (!ok) break;
        fence_after();
        uint32_t p[BN / 16][16];
#pragma unroll
        for (int c = 0; c < BN / 16; ++c) tmem_ld16(acc + c * 16, p[c]);
#pragma unroll
        for (int c = 0; c < BN / 16; ++c) tmem_wait(p[c]);
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[b]);
        const int col = col0 + quarter * 32 + lane;
        if (two) {
#pragma unroll
          for (int i = 0; i < BN; ++i)
            p[i / 16][i % 16] = __float_as_uint(__uint_as_float(p[i / 16][i % 16]) *
                                                __shfl_sync(0xffffffffu, i < 32 ? f0.first : f1.first, i & 31));
        }
#pragma unroll
        for (int i = 0; i < BN; ++i) {
          const float f = __shfl_sync(0xffffffffu, i < 32 ? last0 : last1, i & 31);
          if (row0 + i < end && col < a.N)
            out[int64_t(row0 + i) * a.N + col] = from_f32<TO>(__uint_as_float(p[i / 16][i % 16]) * f);
        }
      } else {
        constexpr int kTileOut = 32 * BN * int(sizeof(TO));  // of a warp
        static_assert(4 * kTileOut <= ST * C::kStage, "the last tile's room");
        const Fp4Factors f = fp4_factors(row_factor(a, row0 + quarter * 32 + lane), fw);
        ok = poll_warp(&acc_full[b], (tile >> 1) & 1, a.err);
        if (!ok) break;
        fence_after();
        const bool last = tiles.next(item) >= tiles.stop();
        store_tile<BN, TO>(a, &maps.out, acc, last ? stages + quarter * kTileOut : stage_out + quarter * kOutBytes,
                           row0 + quarter * 32, end, col0, f, 0, BN / 32, last, [&] { mbar_arrive(&acc_empty[b]); });
      }
    }
    if (!ok) *abort_ptr = 1;
    if (!SWAP && lane == 0) tma_stores_done();
    if (a.offsets) zero_rows(out, a.N, off(0), start[a.E + 1], a.S, threadIdx.x - 128, 128);
  } else {
    const ScaleWay way{chunks, C::kChunk, CH, chunk_full, chunk_empty, sf, sf_empty, BN};
    auto w_row = [&](int item) {
      const int e = tile_expert(start, a.E, item);
      return e * a.N + (item - start[e]) % n_ct * col_tile;
    };
    if (warp == 10) {
      auto load = [&](int slot, int item, int x, uint64_t* bar) {
        const int e = tile_expert(start, a.E, item), local = item - start[e];
        uint8_t *m = chunks + slot * C::kChunk, *n = m + kFp4M * kChunkRow;
        tma_2d(SWAP ? n : m, &maps.sa, x, off(e) + local / n_ct * row_tile, bar);
        if (w_chunks) tma_2d(SWAP ? m : n, &maps.sw, x, e * a.N + local % n_ct * col_tile, bar);
      };
      const uint32_t tx = uint32_t((row_tile + (w_chunks ? col_tile : 0)) * kChunkRow);
      chunk_warp<FMT, kChunkRow>(a, tiles, way, tx, load, abort_ptr);
    } else {
      scale_warp_by<FMT, kChunkRow, 2, SWAP>(warp < 4 ? warp - 2 : warp - 6, a, tiles, way, w_row,
                                  [&](int b) { mbar_arrive(&sf_full[b]); }, abort_ptr);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(uint32_t(C::kTmem)));
  }
  pdl_trigger();
}

template <int BN, bool SWAP, int FMT, typename TO>
int launch_one(cudaStream_t s, const TileArgs& a, const TileMaps& m, int grid) {
  static std::atomic<uint64_t> attr_set{0};  // devices whose attribute is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -1;
  auto kernel = fp4_kernel<BN, SWAP, FMT, TO>;
  if (!(attr_set.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Cfg<BN>::kSmem)) != cudaSuccess)
      return -1;
    attr_set.fetch_or(uint64_t(1) << dev);
  }
  return launch_chain(kernel, dim3(grid), dim3(kThreads), Cfg<BN>::kSmem, s, a, m) == cudaSuccess ? 0 : -1;
}

template <int BN, bool SWAP>
int launch_tiles(cudaStream_t s, const Fp4Product& p, int out_dtype) {
  const int row_tile = SWAP ? BN : kFp4M, col_tile = SWAP ? kFp4M : BN;
  TileArgs a{};
  TileMaps m{};
  if (make_tile_args(p, out_dtype, row_tile, col_tile, row_tile, col_tile, kChunkRow, !SWAP, a, m)) return -1;
  // upper bound of the row tiles: one per row_tile rows and one more for every expert with rows
  const int64_t row_tiles = p.offsets ? int64_t(p.S) / row_tile + std::min(p.E, p.S) : (p.S + row_tile - 1) / row_tile;
  const int grid = int(std::min<int64_t>(sm_count(), row_tiles * ((p.N + col_tile - 1) / col_tile)));
  auto run = [&](auto f16, auto bf16, auto f32) {
    return (out_dtype == B200MOE_F16 ? f16 : out_dtype == B200MOE_BF16 ? bf16 : f32)(s, a, m, grid);
  };
  return p.format == kMx ? run(launch_one<BN, SWAP, kMx, __half>, launch_one<BN, SWAP, kMx, __nv_bfloat16>,
                               launch_one<BN, SWAP, kMx, float>)
                         : run(launch_one<BN, SWAP, kNv, __half>, launch_one<BN, SWAP, kNv, __nv_bfloat16>,
                               launch_one<BN, SWAP, kNv, float>);
}

}  // namespace

int make_tile_args(const Fp4Product& p, int out_dtype, int a_box, int w_box, int sa_box, int sw_box, int cr, bool copy_out,
                  TileArgs& a, TileMaps& m) {
  const int stride = fp4_stride(p.format, p.K), scales = p.K / fp4_block(p.format);
  a.a_factor = p.format == kNv ? p.a + fp4_factor_at(p.K) : nullptr;
  a.a_stride = stride;
  a.w_scale = p.w_scale;
  a.w_stride = scales;
  a.w_align = 16;
  while (scales % a.w_align || reinterpret_cast<uintptr_t>(p.w_scale) % a.w_align) a.w_align /= 2;
  a.w_factor = p.format == kNv ? p.w_factor : nullptr;
  a.offsets = p.offsets;
  a.out = p.out;
  a.S = p.S;
  a.N = p.N;
  a.E = p.E;
  a.K = p.K;
  a.err = op_error_word();
  const int64_t out_bytes = int64_t(p.N) * (out_dtype == B200MOE_F32 ? 4 : 2);
  a.copy_out = copy_out && out_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  // a row's scales up to whole 16 bytes: inside its record, and for weights what lies on 16 bytes has no rest
  const int scale_row = (scales + 15) / 16 * 16;
  if (make_u8_tile_map(&m.a, p.a, p.S, p.K / 2, kFp4RowBytes, a_box, stride) ||
      make_u8_tile_map(&m.w, p.w, int64_t(p.E) * p.N, p.K / 2, kFp4RowBytes, w_box) ||
      make_u8_tile_map(&m.sa, p.a + p.K / 2, p.S, scale_row, cr, sa_box, stride) ||
      (a.w_align == 16 && make_u8_tile_map(&m.sw, p.w_scale, int64_t(p.E) * p.N, scales, cr, sw_box)) ||
      (a.copy_out && make_u8_store_map(&m.out, p.out, p.S, out_bytes, 32)))
    return -1;
  return 0;
}

int launch_fp4_tiles(cudaStream_t s, const Fp4Product& p, int out_dtype) { return launch_tiles<128, false>(s, p, out_dtype); }

int launch_fp4_stream(cudaStream_t s, const Fp4Product& p, int rows_per_tile, int out_dtype) {
  return rows_per_tile <= 16   ? launch_tiles<16, true>(s, p, out_dtype)
         : rows_per_tile <= 32 ? launch_tiles<32, true>(s, p, out_dtype)
                               : launch_tiles<64, true>(s, p, out_dtype);
}

}  // namespace b200moe

using namespace b200moe;

namespace {

int product_status(const Fp4Product& p, int out_dtype) {
  if (!p.w || !p.w_scale || !p.out || p.S < 1 || p.S > INT32_MAX - 256 || p.N < 1 || p.E < 1 || p.E > kFp4MaxExperts ||
      !b200moe_fp4_record_bytes(p.format, p.K) || (p.format == kNv && !p.w_factor) || (!p.offsets && p.E != 1) ||
      int64_t(p.E) * p.N > INT32_MAX - 256 || p.K > (1 << 24))
    return B200MOE_ERR_INVALID_ARG;
  if (out_dtype < 0 || out_dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  if (reinterpret_cast<uintptr_t>(p.w) % 16) return B200MOE_ERR_ALIGN;
  return B200MOE_OK;
}

// The kernel by rows per matrix: that of a few rows where it fits (fp4_skinny.cu), else as measured on B200 (us, NVFP4;
// kernels of 16, 32 and 64 rows as the MMA's N, of 128 as
// its M, and of 256 as that of two CTAs; weights from HBM):
//   one matrix 4096 x 4096: 8.7 / 9.2 / 10.0 / 10.5 / 12.7 at 1 row, 9.0 / 9.7 / 10.9 / 10.0 / 12.3 at 64, 13.8 / 9.8 /
//   10.9 / 10.1 / 12.4 at 96, 18.7 / 14.9 / 11.0 / 10.1 / 12.7 at 192, - / 24.7 / 16.7 / 10.3 / 12.8 at 512, - / - / 21.9 /
//   16.0 / 12.9 at 768: a tile of fewer rows or columns gives more CTAs, so the smallest whose tiles run in one wave, and
//   pairs where no kernel's do. 2816 x 2048: - / - / 11.5 / 7.1 / 8.7 at 768 (132 tiles of 128), 14.4 / 9.7 / 8.8 at 1024
//   (176). The 64-row kernel never leads there.
//   64 matrices 2816 x 2048: 46.6 / 40.7 / 40.6 / 46.7 / 54.0 at 16 rows each, 66.6 / 55.6 / 41.9 / 45.9 / 55.4 at 32,
//   102 / 58.7 / 45.7 / 48.1 / 55.7 at 48, - / 70.7 / 62.8 / 46.2 / 56.2 at 64, - / 108 / 72.8 / 47.1 / 57.1 at 96, 131 /
//   78.2 / 60.6 (the last three) at 192 (the last kernel by 6 us more in every other run): an expert above a tile's rows
//   reads its weights twice, and rows are drawn about their mean. 384 matrices 4096 x 4096: 555 / 554 / 616 at 8, 1070 /
//   601 / 643 / 737 / 839 at 24, 1875 / 1112 / 671 / 848 / 962 at 48, - / - / 1633 / 1225 / 885 at 128: there 20 is before
//   the crossing (7 % at 24).
//   S counts rows without an expert too, and no spread is known here.
// Returns 8 (fp4_skinny.cu), 16, 32, 64, 128 or 256.
int choose(const Fp4Product& p) {
  if (!p.offsets) {
    if (fp4_skinny_fits(p)) return 8;
    for (int t = 16; t <= 128; t *= 2)
      if (t != 64 && (p.S + t - 1) / t * int64_t((p.N + 127) / 128) <= sm_count()) return t;
    return p.S <= 32 ? 32 : p.S <= 128 ? 128 : 256;
  }
  const int64_t e = p.E;
  return p.S <= 20 * e ? 32 : p.S <= 52 * e ? 64 : p.S <= 112 * e ? 128 : 256;
}

int launch_status(int rc) {
  if (rc == 0) return B200MOE_OK;
  cudaGetLastError();
  return B200MOE_ERR_CUDA;
}

int run_product(cudaStream_t s, const Fp4Product& p, int out_dtype) {
  const int kind = choose(p);
  return launch_status(kind == 8     ? launch_fp4_skinny(s, p, nullptr, 0, 0, out_dtype)
                       : kind == 256 ? launch_fp4_pairs(s, p, out_dtype)
                       : kind == 128 ? launch_fp4_tiles(s, p, out_dtype)
                                     : launch_fp4_stream(s, p, kind, out_dtype));
}

}  // namespace

extern "C" int b200moe_fp4_matmul(void* stream, const void* a, const void* w, const void* w_scale, const float* w_factor,
                                  const int32_t* offsets, int S, int N, int K, int E, int format, void* out, int out_dtype) {
  const Fp4Product p{static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(w), static_cast<const uint8_t*>(w_scale),
                     w_factor, offsets, out, format, S, N, K, E};
  const int st = product_status(p, out_dtype);
  if (st) return st;
  if (!a) return B200MOE_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(a) % 16) return B200MOE_ERR_ALIGN;
  return run_product(static_cast<cudaStream_t>(stream), p, out_dtype);
}

extern "C" size_t b200moe_fp4_linear_workspace_bytes(int S, int N, int K, int format) {
  Fp4Product p{};
  p.format = format;
  p.S = S;
  p.N = N;
  p.K = K;
  p.E = 1;
  if (S < 1 || N < 1 || K < 32 || (choose(p) == 8 && fp4_skinny_quantizes(S, K))) return 0;
  return size_t(S) * b200moe_fp4_record_bytes(format, K);
}

extern "C" int b200moe_fp4_linear(void* stream, const void* x, int x_dtype, int64_t ldx, const void* w,
                                  const void* w_scale, const float* w_factor, int S, int N, int K, int format, void* out,
                                  int out_dtype, void* workspace, size_t workspace_bytes) {
  Fp4Product p{nullptr,  static_cast<const uint8_t*>(w), static_cast<const uint8_t*>(w_scale), w_factor, nullptr, out, format,
               S, N, K, 1};
  const int st = product_status(p, out_dtype);
  if (st) return st;
  if (!x || ldx < 0) return B200MOE_ERR_INVALID_ARG;
  if (x_dtype < 0 || x_dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = x_dtype != B200MOE_F32 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0;
  if (wide && choose(p) == 8 && fp4_skinny_quantizes(S, K))
    return launch_status(launch_fp4_skinny(s, p, x, x_dtype, ldx, out_dtype));
  if (!workspace || workspace_bytes < size_t(S) * b200moe_fp4_record_bytes(format, K)) return B200MOE_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return B200MOE_ERR_ALIGN;
  const int qs = b200moe_fp4_quantize(stream, x, x_dtype, ldx, S, K, format, 0, 1.f, workspace);
  if (qs) return qs;
  p.a = static_cast<const uint8_t*>(workspace);
  return run_product(s, p, out_dtype);
}
