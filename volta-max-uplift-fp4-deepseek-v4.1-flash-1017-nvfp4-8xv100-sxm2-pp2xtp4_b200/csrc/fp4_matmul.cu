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
//   warps 2, 3 and (BN = 256) 8 (scales): 128 rows each. A lane loads the scales
//     of rows lane, lane + 32, .. from global memory several stages ahead and
//     stores them in the order tcgen05.cp wants, a 512-byte block per 64 columns
//     of K (row r's four bytes at (r % 32) * 16 + (r / 32) * 4): four vector
//     stores without bank conflicts;
//   warp 1 (MMA): per 64 columns tcgen05.cp of the block scales into one of four
//     places in TMEM and one MMA (M 128, N BN, K 64). Copies and MMAs of one
//     thread run in order, so a place is safe to write again four MMAs later;
//   warps 4-7 (epilogue): a thread holds one TMEM lane; the sums leave, times
//     both factors, while the next tile's MMAs run.
// At BN = 256 two accumulators and the scales exceed TMEM's 512 columns: the
// accumulators share 64 columns, which the epilogue empties first.
//
// SWAP: the weights are the MMA's M and BN rows of a its N, for few rows per
// matrix: then the kernel streams weights, and a thread of the epilogue holds one
// output column.
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "fp4_ops.h"
#include "fp4_rows.cuh"
#include "fp8_tc.cuh"
#include "internal.h"

namespace b200moe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kBM = 128;
constexpr int kStageK = 256;             // columns of K per stage
constexpr int kRowBytes = kStageK / 2;   // codes of a row in a stage
constexpr int kABytes = kBM * kRowBytes;
constexpr int kSfBlock = 4 * 512;        // 128 rows' scales of a stage
constexpr int kSfBufs = 2;
constexpr int kSfAhead = 4;              // stages whose scales are loaded ahead
constexpr int kOutBytes = 32 * 64;       // per epilogue warp: 32 rows in pieces of 64 bytes

template <int BN>
struct Cfg {
  static constexpr int kNBlocks = BN > 128 ? 2 : 1;  // 128-row blocks of N
  static constexpr int kThreads = BN > 128 ? 288 : 256;
  static constexpr int kStage = kABytes + BN * kRowBytes;
  static constexpr int kStages = BN >= 256 ? 4 : BN >= 128 ? 6 : 8;
  static constexpr int kSfBytes = (1 + kNBlocks) * kSfBlock;
  static constexpr int kSfCols = 4 * (1 + kNBlocks);  // TMEM columns of 64 columns of K
  static constexpr int kShared = BN == 256 ? 64 : 0;  // columns that the two accumulators share
  static constexpr int kAcc1 = BN - kShared;
  static constexpr int kSf0 = 2 * BN - kShared;
  static constexpr int kTmem = kSf0 + 4 * kSfCols <= 64    ? 64
                               : kSf0 + 4 * kSfCols <= 128 ? 128
                               : kSf0 + 4 * kSfCols <= 256 ? 256
                                                           : 512;
  static_assert(kSf0 + 4 * kSfCols <= 512, "TMEM columns");
  static constexpr size_t kSmem =
      1024 + size_t(kStages) * kStage + kSfBufs * kSfBytes + 4 * kOutBytes + 8 * (2 * kStages + 2 * kSfBufs + 4);
  static_assert(kSmem + 8 * (kMaxExperts + 1) + 64 <= 227 * 1024, "shared memory, with the tile table");
};

// E2M1 operands, K-major, M 128, N BN; scales E4M3 per 16 or (bit 23) E8M0 per 32
template <int BN, int FMT>
constexpr uint32_t idesc() {
  return (1u << 7) | (1u << 10) | (uint32_t(BN >> 3) << 17) | (uint32_t(FMT) << 23) | (uint32_t(kBM >> 4) << 24);
}

// a 512-byte scale block: K-major, no swizzle, 8-row core matrices of 16-byte rows, 128 bytes apart
__device__ __forceinline__ uint64_t desc_sf(uint32_t addr) {
  return uint64_t((addr >> 4) & 0x3FFF) | (uint64_t(1) << 16) | (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
}
__device__ __forceinline__ void sf_copy(uint32_t col, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(col), "l"(desc));
}
template <int FMT>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t sfa, uint32_t sfb, uint32_t accumulate,
                                    uint32_t id) {
  if constexpr (FMT == kMx)
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p; }" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(sfa), "r"(sfb));
  else
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p; }" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(sfa), "r"(sfb));
}

struct Args {
  const uint8_t* a_scale;   // row 0's
  const uint8_t* a_factor;  // row 0's, null for MXFP4
  int64_t a_stride;         // bytes between records
  const uint8_t* w_scale;
  int64_t w_stride;         // bytes between a weight row's scales
  int w_align;              // of the weight rows' scales, bytes up to 16
  const float* w_factor;    // [E], null for MXFP4
  const int32_t* offsets;   // [E + 1], null: one matrix, all S rows
  void* out;                // [S][N]
  int copy_out;             // its rows lie on 16 bytes
  int S, N, E, K;
  uint32_t* err;
};

// The scale bytes of one row for a stage (NVFP4 16, MXFP4 8), zeros behind the row's last: a scale that is no number
// would spoil the zero codes that it stands beside.
template <int FMT>
__device__ __forceinline__ uint4 load_scales(const uint8_t* p, int align, int valid) {
  constexpr int kFull = FMT == kMx ? 8 : 16;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (valid >= kFull && align >= kFull) {
    if constexpr (FMT == kMx) {
      const uint2 h = __ldg(reinterpret_cast<const uint2*>(p));
      v.x = h.x;
      v.y = h.y;
    } else {
      v = __ldg(reinterpret_cast<const uint4*>(p));
    }
    return v;
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < kFull / 4; ++j) {
    if (align >= 4 && valid >= 4 * j + 4) {
      w[j] = __ldg(reinterpret_cast<const uint32_t*>(p) + j);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * j + i < valid) w[j] |= uint32_t(__ldg(p + 4 * j + i)) << (8 * i);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A warp's block of 128 rows: walks the tiles' stages, loads ahead and stores each stage's scales in the copies' order.
template <int FMT, typename Tiles, typename RowOf>
__device__ __forceinline__ void scale_warp(const Args& a, const Tiles& tiles, const RowOf& row_of, const uint8_t* base,
                                           int64_t stride, int align, int rows, int last, uint8_t* dst, int buf_bytes,
                                           uint64_t* full, uint64_t* empty, volatile int* abort_ptr) {
  const int lane = threadIdx.x & 31;
  const int n_kt = (a.K + kStageK - 1) / kStageK, bytes = a.K / fp4_block(FMT);
  constexpr int kFull = FMT == kMx ? 8 : 16;
  int sb = 0;
  uint32_t ph = 0;
  bool ok = true;
  for (int item = tiles.first(); ok && item < tiles.stop(); item = tiles.next(item)) {
    const int row0 = row_of(item);
    const uint8_t* p[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) p[m] = base + int64_t(min(row0 + lane + 32 * m, last)) * stride;
    uint4 v[kSfAhead][4];
    auto fetch = [&](int kt, uint4(&d)[4]) {
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (kt < n_kt && 32 * m < rows) d[m] = load_scales<FMT>(p[m] + kt * kFull, align, bytes - kt * kFull);
    };
#pragma unroll
    for (int d = 0; d < kSfAhead; ++d) {
#pragma unroll
      for (int m = 0; m < 4; ++m) v[d][m] = make_uint4(0, 0, 0, 0);
      fetch(d, v[d]);
    }
    for (int kt0 = 0; ok && kt0 < n_kt; kt0 += kSfAhead) {
#pragma unroll
      for (int d = 0; d < kSfAhead; ++d) {
        const int kt = kt0 + d;
        if (kt >= n_kt) break;
        ok = !__any_sync(0xffffffffu, *abort_ptr) && poll_warp(&empty[sb], ph ^ 1u, a.err);
        if (!ok) break;
        uint4* to = reinterpret_cast<uint4*>(dst + sb * buf_bytes) + lane;
        const uint4(&s)[4] = v[d];
        if constexpr (FMT == kMx) {  // two bytes per 64 columns
          to[0] = make_uint4(s[0].x & 0xffffu, s[1].x & 0xffffu, s[2].x & 0xffffu, s[3].x & 0xffffu);
          to[32] = make_uint4(s[0].x >> 16, s[1].x >> 16, s[2].x >> 16, s[3].x >> 16);
          to[64] = make_uint4(s[0].y & 0xffffu, s[1].y & 0xffffu, s[2].y & 0xffffu, s[3].y & 0xffffu);
          to[96] = make_uint4(s[0].y >> 16, s[1].y >> 16, s[2].y >> 16, s[3].y >> 16);
        } else {
          to[0] = make_uint4(s[0].x, s[1].x, s[2].x, s[3].x);
          to[32] = make_uint4(s[0].y, s[1].y, s[2].y, s[3].y);
          to[64] = make_uint4(s[0].z, s[1].z, s[2].z, s[3].z);
          to[96] = make_uint4(s[0].w, s[1].w, s[2].w, s[3].w);
        }
        fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[sb]);
        if (++sb == kSfBufs) sb = 0, ph ^= 1u;
        fetch(kt + kSfAhead, v[d]);
      }
    }
  }
  if (!ok) *abort_ptr = 1;
}

// The CTA's tiles. Rows as M: tiles apart by the grid, so that CTAs that run at once share rows and columns in L2; the
// weights as M: a contiguous range, so that it streams an expert's weights in order.
struct Tiles {
  int begin, end, step;
  __device__ __forceinline__ int first() const { return begin; }
  __device__ __forceinline__ int stop() const { return end; }
  __device__ __forceinline__ int next(int i) const { return i + step; }
};

template <int BN, bool SWAP, int FMT, typename TO>
__global__ void __launch_bounds__(Cfg<BN>::kThreads, 1)
    fp4_kernel(const Args a, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
               const __grid_constant__ CUtensorMap map_out) {
  using C = Cfg<BN>;
  constexpr int ST = C::kStages;
  constexpr int kScaleWarps = 1 + C::kNBlocks;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int off[kMaxExperts + 1], start[kMaxExperts + 1];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_flag;
  const uint32_t base_u32 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* stages = smem_raw + (base_u32 - smem_u32(smem_raw));  // [ST][M 16 KB, N BN x 128]
  uint8_t* sf = stages + ST * C::kStage;                        // [2][M 2 KB, N 2 or 4 KB]
  uint8_t* stage_out = sf + kSfBufs * C::kSfBytes;              // [4][2 KB]
  uint64_t* full = reinterpret_cast<uint64_t*>(stage_out + 4 * kOutBytes);
  uint64_t* empty = full + ST;
  uint64_t* sf_full = empty + ST;
  uint64_t* sf_empty = sf_full + kSfBufs;
  uint64_t* acc_full = sf_empty + kSfBufs;  // [2]
  uint64_t* acc_empty = acc_full + 2;       // [2]
  volatile int* abort_ptr = &abort_flag;

  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kSfBufs; ++b) {
      mbar_init(&sf_full[b], kScaleWarps);
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
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_base_sh;
  pdl_wait();
  const int row_tile = SWAP ? BN : kBM, col_tile = SWAP ? kBM : BN;
  const int n_ct = (a.N + col_tile - 1) / col_tile;
  build_tile_table(a.offsets, a.E, a.S, row_tile, n_ct, off, start, a.err);
  const int n_items = start[a.E];
  Tiles tiles{int(blockIdx.x), n_items, int(gridDim.x)};
  if (SWAP)
    tiles = {int(int64_t(n_items) * blockIdx.x / gridDim.x), int(int64_t(n_items) * (blockIdx.x + 1) / gridDim.x), 1};
  auto a_row = [&](int item) {
    const int e = tile_expert(start, a.E, item);
    return off[e] + (item - start[e]) / n_ct * row_tile;
  };
  auto w_row = [&](int item) {
    const int e = tile_expert(start, a.E, item);
    return e * a.N + (item - start[e]) % n_ct * col_tile;
  };
  const int n_kt = (a.K + kStageK - 1) / kStageK, n_k64 = (a.K + 63) / 64;

  if (warp == 0) {
    int st = 0;
    uint32_t ph = 0, issued = 0, par = 0;
    bool ok = true;
    for (int item = tiles.first(); ok && item < tiles.stop(); item = tiles.next(item)) {
      const int ra = a_row(item), rw = w_row(item);
      for (int kt = 0; kt < n_kt; ++kt) {
        ok = !__any_sync(0xffffffffu, *abort_ptr) && poll_warp(&empty[st], ph ^ 1u, a.err);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* dst = stages + st * C::kStage;
          mbar_arrive_expect_tx(&full[st], uint32_t(C::kStage));
          tma_2d(dst, SWAP ? &map_w : &map_a, kt * kRowBytes, SWAP ? rw : ra, &full[st]);
          tma_2d(dst + kABytes, SWAP ? &map_a : &map_w, kt * kRowBytes, SWAP ? ra : rw, &full[st]);
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
      // the columns this tile writes: those of the tile two before it, which the epilogue has left when it comes to the
      // one before, and where the accumulators overlap the shared columns of the one before
      if (C::kShared ? tile >= 1 : tile >= 2) {
        const int o = C::kShared ? tile - 1 : tile - 2;
        ok = poll_warp(&acc_empty[o & 1], (o >> 1) & 1, a.err);
        if (!ok) break;
        fence_after();
      }
      const uint32_t d = tmem + b * C::kAcc1;
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
            const uint32_t sfa = tmem + C::kSf0 + j * C::kSfCols, sfb = sfa + 4;
            sf_copy(sfa, ds + j * 32);
#pragma unroll
            for (int n = 0; n < C::kNBlocks; ++n) sf_copy(sfb + 4 * n, ds + (1 + n) * (kSfBlock >> 4) + j * 32);
            mma<FMT>(d, da + 2 * j, da + (kABytes >> 4) + 2 * j, sfa, sfb, uint32_t(kt | j), idesc<BN, FMT>());
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
    uint8_t* mine = stage_out + quarter * kOutBytes;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
    TO* out = static_cast<TO*>(a.out);
    int tile = 0;
    bool ok = true;
    for (int item = tiles.first(); ok && item < tiles.stop(); item = tiles.next(item), ++tile) {
      const int e = tile_expert(start, a.E, item), local = item - start[e], end = off[e + 1];
      const int row0 = off[e] + local / n_ct * row_tile, col0 = local % n_ct * col_tile;
      const float fw = a.w_factor ? __ldg(a.w_factor + e) : 1.f;
      const int b = tile & 1;
      const uint32_t acc = lanes + b * C::kAcc1;
      auto factor = [&](int row) {
        return a.a_factor ? __ldg(reinterpret_cast<const float*>(a.a_factor + int64_t(min(row, a.S - 1)) * a.a_stride)) : 1.f;
      };
      if constexpr (SWAP) {
        const float fa = lane < BN ? factor(row0 + lane) : 1.f, fa2 = BN > 32 ? factor(row0 + 32 + lane) : 1.f;
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
#pragma unroll
        for (int i = 0; i < BN; ++i) {
          const float f = __shfl_sync(0xffffffffu, i < 32 ? fa : fa2, i & 31);
          if (row0 + i < end && col < a.N)
            out[int64_t(row0 + i) * a.N + col] = from_f32<TO>(__uint_as_float(p[i / 16][i % 16]) * f * fw);
        }
      } else {
        const int row = row0 + quarter * 32 + lane;
        const float fa = factor(row);
        ok = poll_warp(&acc_full[b], (tile >> 1) & 1, a.err);
        if (!ok) break;
        fence_after();
        constexpr int PW = 64 / int(sizeof(TO)), CW = 16 / int(sizeof(TO));  // columns per piece, per 16-byte chunk
        // whole rows of one expert leave by a copy of the warp's 32 rows; a tile that ends inside, or rows off 16 bytes,
        // by the threads
        const bool copies = a.copy_out && row0 + quarter * 32 + 32 <= end;
#pragma unroll 1
        for (int i = 0; i < BN / 32; ++i) {
          // the shared columns first: the last two pieces of accumulator 0, the first two of accumulator 1
          const int c = C::kShared && b == 0 ? (i + BN / 32 - 2) % (BN / 32) : i;
          uint32_t p[32];
          tmem_ld32(acc + c * 32, p);
          tmem_wait(p);
          if (i == (C::kShared ? 1 : BN / 32 - 1)) {
            fence_before();  // every lane's reads come before the MMA that overwrites them, across the barrier
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
          }
#pragma unroll
          for (int pc = 0; pc < 32 / PW; ++pc) {
            if (lane == 0) tma_stores_read();  // the piece before has left
            __syncwarp();
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) {
              float v[CW];
#pragma unroll
              for (int k = 0; k < CW; ++k) v[k] = __uint_as_float(p[pc * PW + ch * CW + k]) * fa * fw;
              store_vec<TO, CW>(reinterpret_cast<TO*>(mine + lane * 64 + ((ch ^ ((lane >> 1) & 3)) << 4)), v);
            }
            const int col = col0 + c * 32 + pc * PW;
            if (copies) {
              fence_async();
              __syncwarp();
              if (lane == 0 && col < a.N)
                tma_store_2d(&map_out, col * int(sizeof(TO)), row0 + quarter * 32, mine);
            } else {
              __syncwarp();
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int r = j * 8 + (lane >> 2), at = col + (lane & 3) * CW;
                const TO* src = reinterpret_cast<const TO*>(mine + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
                if (row0 + quarter * 32 + r >= end) continue;
                TO* to = out + int64_t(row0 + quarter * 32 + r) * a.N + at;
                if (a.copy_out && at + CW <= a.N) {
                  *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(src);
                } else {
                  for (int k = 0; k < CW; ++k)
                    if (at + k < a.N) to[k] = src[k];
                }
              }
              __syncwarp();
            }
          }
        }
      }
    }
    if (!ok) *abort_ptr = 1;
    if (!SWAP && lane == 0) tma_stores_done();
    if (a.offsets) zero_rows(out, a.N, off[0], off[a.E], a.S, threadIdx.x - 128, 128);
  } else {
    // warp 2: the scales of the MMA's M; 3 and 8: of its N
    const int block = warp == 2 ? 0 : warp == 3 ? 1 : 2;
    const bool of_a = (block == 0) != SWAP;
    const int add = block == 2 ? 128 : 0;
    auto row_of = [&](int item) { return (of_a ? a_row(item) : w_row(item)) + add; };
    scale_warp<FMT>(a, tiles, row_of, of_a ? a.a_scale : a.w_scale, of_a ? a.a_stride : a.w_stride, of_a ? 16 : a.w_align,
                    block ? min(BN, 128) : kBM, of_a ? a.S - 1 : a.E * a.N - 1, sf + block * kSfBlock, C::kSfBytes, sf_full,
                    sf_empty, abort_ptr);
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
int launch_one(cudaStream_t s, const Args& a, const CUtensorMap& ma, const CUtensorMap& mw, const CUtensorMap& mo, int grid) {
  static std::atomic<uint64_t> attr_set{0};  // devices whose attribute is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -1;
  auto kernel = fp4_kernel<BN, SWAP, FMT, TO>;
  if (!(attr_set.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Cfg<BN>::kSmem)) != cudaSuccess)
      return -1;
    attr_set.fetch_or(uint64_t(1) << dev);
  }
  return launch_chain(kernel, dim3(grid), dim3(Cfg<BN>::kThreads), Cfg<BN>::kSmem, s, a, ma, mw, mo) == cudaSuccess ? 0 : -1;
}

template <int BN, bool SWAP>
int launch_tiles(cudaStream_t s, const Fp4Product& p, int out_dtype) {
  Args a{};
  const int stride = fp4_stride(p.format, p.K);
  a.a_scale = p.a + p.K / 2;
  a.a_factor = p.format == kNv ? p.a + fp4_factor_at(p.K) : nullptr;
  a.a_stride = stride;
  a.w_scale = p.w_scale;
  a.w_stride = p.K / fp4_block(p.format);
  a.w_align = 16;
  while (a.w_stride % a.w_align || reinterpret_cast<uintptr_t>(p.w_scale) % a.w_align) a.w_align /= 2;
  a.w_factor = p.format == kNv ? p.w_factor : nullptr;
  a.offsets = p.offsets;
  a.out = p.out;
  a.S = p.S;
  a.N = p.N;
  a.E = p.E;
  a.K = p.K;
  a.err = op_error_word();
  const int row_tile = SWAP ? BN : kBM, col_tile = SWAP ? kBM : BN;
  const int64_t out_bytes = int64_t(p.N) * (out_dtype == B200MOE_F32 ? 4 : 2);
  a.copy_out = !SWAP && out_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  CUtensorMap ma, mw, mo{};
  if (make_u8_tile_map(&ma, p.a, p.S, p.K / 2, kRowBytes, row_tile, stride) ||
      make_u8_tile_map(&mw, p.w, int64_t(p.E) * p.N, p.K / 2, kRowBytes, col_tile))
    return -1;
  if (a.copy_out && make_u8_store_map(&mo, p.out, p.S, out_bytes, 32)) return -1;
  // upper bound of the row tiles: one per row_tile rows and one more for every expert with rows
  const int64_t row_tiles = p.offsets ? int64_t(p.S) / row_tile + std::min(p.E, p.S) : (p.S + row_tile - 1) / row_tile;
  const int grid = int(std::min<int64_t>(sm_count(), row_tiles * ((p.N + col_tile - 1) / col_tile)));
  auto run = [&](auto f16, auto bf16, auto f32) {
    return (out_dtype == B200MOE_F16 ? f16 : out_dtype == B200MOE_BF16 ? bf16 : f32)(s, a, ma, mw, mo, grid);
  };
  return p.format == kMx ? run(launch_one<BN, SWAP, kMx, __half>, launch_one<BN, SWAP, kMx, __nv_bfloat16>,
                               launch_one<BN, SWAP, kMx, float>)
                         : run(launch_one<BN, SWAP, kNv, __half>, launch_one<BN, SWAP, kNv, __nv_bfloat16>,
                               launch_one<BN, SWAP, kNv, float>);
}

}  // namespace

int launch_fp4_tiles(cudaStream_t s, const Fp4Product& p, int out_dtype) {
  const int64_t row_tiles = p.offsets ? int64_t(p.S) / kBM + std::min(p.E, p.S) : (p.S + kBM - 1) / kBM;
  return row_tiles * ((p.N + 255) / 256) >= sm_count() ? launch_tiles<256, false>(s, p, out_dtype)
                                                       : launch_tiles<128, false>(s, p, out_dtype);
}

int launch_fp4_stream(cudaStream_t s, const Fp4Product& p, int rows_per_tile, int out_dtype) {
  return rows_per_tile <= 16   ? launch_tiles<16, true>(s, p, out_dtype)
         : rows_per_tile <= 32 ? launch_tiles<32, true>(s, p, out_dtype)
                               : launch_tiles<64, true>(s, p, out_dtype);
}

}  // namespace b200moe

using namespace b200moe;

namespace {

int product_status(const Fp4Product& p, int out_dtype) {
  if (!p.w || !p.w_scale || !p.out || p.S < 1 || p.S > INT32_MAX - 256 || p.N < 1 || p.E < 1 || p.E > kMaxExperts ||
      !b200moe_fp4_record_bytes(p.format, p.K) || (p.format == kNv && !p.w_factor) || (!p.offsets && p.E != 1) ||
      int64_t(p.E) * p.N > INT32_MAX - 256 || p.K > (1 << 24))
    return B200MOE_ERR_INVALID_ARG;
  if (out_dtype < 0 || out_dtype > B200MOE_F32) return B200MOE_ERR_DTYPE;
  if (reinterpret_cast<uintptr_t>(p.w) % 16) return B200MOE_ERR_ALIGN;
  return B200MOE_OK;
}

// The kernel by rows per matrix: 16, 32 or 64 rows as the MMA's N, 128 as its M.
int choose(const Fp4Product& p) {
  if (!p.offsets) {
    for (int t = 16; t <= 64; t *= 2)
      if ((p.S + t - 1) / t * int64_t((p.N + 127) / 128) <= sm_count()) return t;
    return p.S <= 64 ? 64 : 128;
  }
  return p.S <= 24 * int64_t(p.E) ? 32 : 128;
}

int launch_status(int rc) {
  if (rc == 0) return B200MOE_OK;
  cudaGetLastError();
  return B200MOE_ERR_CUDA;
}

int run_product(cudaStream_t s, const Fp4Product& p, int out_dtype) {
  const int kind = choose(p);
  return launch_status(kind == 128 ? launch_fp4_tiles(s, p, out_dtype) : launch_fp4_stream(s, p, kind, out_dtype));
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
  if (S < 1 || N < 1) return 0;
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
  if (!workspace || workspace_bytes < size_t(S) * b200moe_fp4_record_bytes(format, K)) return B200MOE_ERR_INVALID_ARG;
  const int qs = b200moe_fp4_quantize(stream, x, x_dtype, ldx, S, K, format, 0, 1.f, workspace);
  if (qs) return qs;
  p.a = static_cast<const uint8_t*>(workspace);
  return run_product(static_cast<cudaStream_t>(stream), p, out_dtype);
}
