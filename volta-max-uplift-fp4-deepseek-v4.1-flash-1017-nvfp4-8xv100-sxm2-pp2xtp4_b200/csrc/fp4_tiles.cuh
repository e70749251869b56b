// What the tcgen05 kernels of 4-bit products share: arguments, block-scaled MMAs
// and the way of the scales from global memory to the tensor core.
//
// tcgen05.mma reads block scales from TMEM, where tcgen05.cp puts them from 512-byte
// blocks of shared memory: 128 rows' bytes for 64 columns of K, row r's four at
// (r % 32) * 16 + (r / 32) * 4 (MXFP4: two bytes, two zeros).  In global memory a
// row's scales stand one after another.  TMA brings them as they are, 32 or 64 bytes of
// 128 rows at a time (a chunk: two or four stages of NVFP4, twice that of MXFP4), and four warps, a
// stage each in turn, put them in order: a lane reads 16 bytes of rows lane,
// lane + 32, .. and writes 16 bytes per block, without bank conflicts either way (the
// chunk is swizzled by TMA).  Loads by the lanes themselves, 16 bytes of a row each,
// took 91 us for 8192 x 4096 x 4096 where everything else takes 57: each touches 32
// lines, and behind the codes' TMA traffic their answers come late.  They are left for
// weights whose rows of scales do not lie on 16 bytes, which TMA cannot take.
#pragma once

#include <cuda.h>

#include "fp4_ops.h"
#include "fp4_rows.cuh"
#include "fp8_tc.cuh"
#include "internal.h"

namespace b200moe {

constexpr int kFp4MaxExperts = 1024;
constexpr int kFp4M = 128;                       // rows of the MMA's M per CTA
constexpr int kFp4StageK = 256;                  // columns of K per stage
constexpr int kFp4RowBytes = kFp4StageK / 2;     // codes of a row in a stage
constexpr int kFp4ABytes = kFp4M * kFp4RowBytes;
constexpr int kSfBlock = 4 * 512;                // 128 rows' scales of a stage, in the copies' order

struct TileArgs {
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

// E2M1 operands, K-major, M, N; scales E4M3 per 16 or (bit 23) E8M0 per 32
template <int M, int N, int FMT>
constexpr uint32_t fp4_idesc() {
  return (1u << 7) | (1u << 10) | (uint32_t(N >> 3) << 17) | (uint32_t(FMT) << 23) | (uint32_t(M >> 4) << 24);
}

// a 512-byte scale block: K-major, no swizzle, 8-row core matrices of 16-byte rows, 128 bytes apart
__device__ __forceinline__ uint64_t desc_sf(uint32_t addr) {
  return uint64_t((addr >> 4) & 0x3FFF) | (uint64_t(1) << 16) | (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
}
// CTAS: of the pair that the instruction works for, 1 or 2
template <int CTAS>
__device__ __forceinline__ void sf_copy(uint32_t col, uint64_t desc) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(col), "l"(desc));
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(col), "l"(desc));
}
template <int CTAS, int FMT>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate, uint32_t id) {
#define B200MOE_MMA(GROUP, BLOCK)                                                                                         \
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"                                                                  \
               "tcgen05.mma.cta_group::" GROUP ".kind::mxf4nvf4.block_scale." BLOCK " [%0], %1, %2, %3, [%5], [%6], p; }" \
               ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(sfa), "r"(sfb))
  if constexpr (CTAS == 2 && FMT == kMx)
    B200MOE_MMA("2", "block32");
  else if constexpr (CTAS == 2)
    B200MOE_MMA("2", "block16");
  else if constexpr (FMT == kMx)
    B200MOE_MMA("1", "block32");
  else
    B200MOE_MMA("1", "block16");
#undef B200MOE_MMA
}

// Sixteen scale bytes of a row of `bytes`, from byte `at`, by loads of W bytes, or W 1, at any address, from the aligned
// words that hold one of them (8192 x 2048 x 1376 by single bytes: 42 us, 1408 by eights 21); what stands behind the row's
// end is the caller's to clear.
template <int W>
__device__ __forceinline__ uint4 load_unit(const uint8_t* row, int at, int bytes) {
  uint32_t w[4] = {0, 0, 0, 0};
  if constexpr (W == 8) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (at + 8 * j < bytes) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(row + at) + j);
        w[2 * j] = v.x;
        w[2 * j + 1] = v.y;
      }
  } else if constexpr (W == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at + 4 * j < bytes) w[j] = __ldg(reinterpret_cast<const uint32_t*>(row + at) + j);
  } else {
    const uintptr_t p = reinterpret_cast<uintptr_t>(row + at);
    const int before = int(p & 3);
    const uint32_t* q = reinterpret_cast<const uint32_t*>(p - before);
    uint32_t u[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) u[j] = at + 4 * j - before < bytes && (j < 4 || before) ? __ldg(q + j) : 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(u[j], u[j + 1], 8 * before);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The first `valid` of four bytes.
__device__ __forceinline__ uint32_t first_bytes(uint32_t w, int valid) {
  return valid >= 4 ? w : valid <= 0 ? 0u : w & ((1u << (8 * valid)) - 1u);
}

// A unit's stage s of rows lane, lane + 32, lane + 64 and lane + 96, a 16-byte piece for each 64 columns.
template <int FMT>
__device__ __forceinline__ void put_scales(uint4* to, const uint4 (&v)[4], int s) {
  if constexpr (FMT == kMx) {  // two bytes per 64 columns
    const uint32_t x[4] = {s ? v[0].z : v[0].x, s ? v[1].z : v[1].x, s ? v[2].z : v[2].x, s ? v[3].z : v[3].x};
    const uint32_t y[4] = {s ? v[0].w : v[0].y, s ? v[1].w : v[1].y, s ? v[2].w : v[2].y, s ? v[3].w : v[3].y};
    to[0] = make_uint4(x[0] & 0xffffu, x[1] & 0xffffu, x[2] & 0xffffu, x[3] & 0xffffu);
    to[32] = make_uint4(x[0] >> 16, x[1] >> 16, x[2] >> 16, x[3] >> 16);
    to[64] = make_uint4(y[0] & 0xffffu, y[1] & 0xffffu, y[2] & 0xffffu, y[3] & 0xffffu);
    to[96] = make_uint4(y[0] >> 16, y[1] >> 16, y[2] >> 16, y[3] >> 16);
  } else {
    to[0] = make_uint4(v[0].x, v[1].x, v[2].x, v[3].x);
    to[32] = make_uint4(v[0].y, v[1].y, v[2].y, v[3].y);
    to[64] = make_uint4(v[0].z, v[1].z, v[2].z, v[3].z);
    to[96] = make_uint4(v[0].w, v[1].w, v[2].w, v[3].w);
  }
}

// The CTA's tiles. Rows as M: tiles apart by the grid, so that CTAs that run at once share rows and columns in L2; the
// weights as M: a contiguous range, so that it streams an expert's weights in order.
struct Tiles {
  int begin, end, step;
  __device__ __forceinline__ int first() const { return begin; }
  __device__ __forceinline__ int stop() const { return end; }
  __device__ __forceinline__ int next(int i) const { return i + step; }
};

// Where a CTA's scales come from and go.
struct ScaleWay {
  uint8_t* chunks;  // [n_chunks][128 rows of the MMA's M, then of its N, x CR bytes]
  int chunk_bytes, n_chunks;
  uint64_t *chunk_full, *chunk_empty;  // [n_chunks], the second counts the four warps
  uint8_t* bufs;                       // [4][BLOCKS][2 KB]
  uint64_t* empty;                     // [4], the buffers'
  int rows;                            // of N, in blocks of at most 128
};

constexpr int kScaleWarps = 4;  // and buffers: warp w puts every fourth stage into buffer w
// With one warp for all stages one row x 4096 x 4096 took 8.4 us.

// Warp w's walk over the tiles' stages.  CR: bytes of a row in a chunk, 32 or 64; BLOCKS: 128 rows of the MMA's M, then
// of its N; SWAP: the weights are M.  W 16: all scales from the chunks; else the weights' by loads of W bytes (row
// w_row(item) of a tile, four stages ahead).
// arrive(w) tells the MMA warp that buffer w holds a stage.
template <int FMT, int W, int CR, int BLOCKS, bool SWAP, typename RowOf, typename Arrive>
__device__ __forceinline__ void scale_warp(int w, const TileArgs& a, const Tiles& tiles, const ScaleWay& way,
                                           const RowOf& w_row, const Arrive& arrive, volatile int* abort_ptr) {
  constexpr int kUnitStages = FMT == kMx ? 2 : 1, kChunkStages = CR / 16 * kUnitStages;
  const int lane = threadIdx.x & 31;
  const int n_kt = (a.K + kFp4StageK - 1) / kFp4StageK, per_tile = (n_kt + kChunkStages - 1) / kChunkStages;
  const int bytes = a.K / fp4_block(FMT), last = a.E * a.N - 1;
  auto rows_of = [&](int block) { return block == 0 ? kFp4M : min(way.rows - (block - 1) * 128, 128); };
  auto loaded = [](int block) { return W != 16 && (block == 0) == SWAP; };
  uint4 ahead[W == 16 ? 1 : BLOCKS][4];
  int item = tiles.first(), kt = w, tile = 0;
  auto settle = [&] {  // kt may have passed its tile
    while (kt >= n_kt && item < tiles.stop()) {
      kt -= n_kt;
      item = tiles.next(item);
      ++tile;
    }
  };
  auto fetch = [&] {
    if (W == 16 || item >= tiles.stop()) return;
    const int row0 = w_row(item) + lane;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
      if (loaded(b)) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int row = row0 + (SWAP ? 0 : (b - 1) * 128) + min(32 * m, rows_of(b) - 1);
          ahead[W == 16 ? 0 : b][m] =
              load_unit<W == 16 ? 1 : W>(a.w_scale + int64_t(min(row, last)) * a.w_stride, kt / kUnitStages * 16, bytes);
        }
      }
  };
  int open = -1, slot = way.n_chunks - 1;  // the chunk in hand, of all tiles'
  uint32_t cph = 1, ph = 0;
  bool ok = true;
  auto leave = [&] {
    __syncwarp();
    if (lane == 0) mbar_arrive(&way.chunk_empty[slot]);
  };
  auto open_next = [&] {
    if (open >= 0) leave();
    ++open;
    if (++slot == way.n_chunks) slot = 0, cph ^= 1u;
    ok = poll_warp(&way.chunk_full[slot], cph, a.err);
  };
  settle();
  fetch();
  while (ok && item < tiles.stop()) {
    const int need = tile * per_tile + kt / kChunkStages;
    while (ok && open < need) open_next();
    if (!ok) break;
    const int unit = kt / kUnitStages, valid = bytes - unit * 16, piece = unit % (CR / 16);
    const uint8_t* c = way.chunks + slot * way.chunk_bytes;
    uint4 v[BLOCKS][4];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int r = lane + 32 * m, at = CR == 64 ? piece ^ ((r >> 1) & 3) : piece ^ ((r >> 2) & 1);  // TMA's swizzle
        if (loaded(b))
          v[b][m] = ahead[W == 16 ? 0 : b][m];
        else
          v[b][m] = r < rows_of(b) ? *reinterpret_cast<const uint4*>(c + (b * 128 + r) * CR + at * 16)
                                   : make_uint4(0, 0, 0, 0);
        if (valid < 16) {  // behind the row's last scale: one that is no number would spoil the zero codes beside it
          v[b][m].x = first_bytes(v[b][m].x, valid);
          v[b][m].y = first_bytes(v[b][m].y, valid - 4);
          v[b][m].z = first_bytes(v[b][m].z, valid - 8);
          v[b][m].w = first_bytes(v[b][m].w, valid - 12);
        }
      }
    ok = !__any_sync(0xffffffffu, *abort_ptr) && poll_warp(&way.empty[w], ph ^ 1u, a.err);
    if (!ok) break;
    ph ^= 1u;
    uint8_t* dst = way.bufs + w * BLOCKS * kSfBlock;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
      put_scales<FMT>(reinterpret_cast<uint4*>(dst + b * kSfBlock) + lane, v[b], FMT == kMx ? kt & 1 : 0);
    fence_async();
    __syncwarp();
    if (lane == 0) arrive(w);
    kt += kScaleWarps;
    settle();
    fetch();
  }
  const int total = (tiles.stop() - tiles.first() + tiles.step - 1) / tiles.step * per_tile;
  while (ok && open < total - 1) open_next();  // the chunks that other warps end with
  if (open >= 0) leave();
  if (!ok) *abort_ptr = 1;
}

// The warp that brings the chunks: on its own, so that the scales, which pass through two more hands, run ahead of the
// codes. load(slot, item, x, barrier) issues a chunk's copies of `tx` bytes.
template <int FMT, int CR, typename Load>
__device__ __forceinline__ void chunk_warp(const TileArgs& a, const Tiles& tiles, const ScaleWay& way, uint32_t tx,
                                           const Load& load, volatile int* abort_ptr) {
  constexpr int kChunkStages = CR / 16 * (FMT == kMx ? 2 : 1);
  const int n_kt = (a.K + kFp4StageK - 1) / kFp4StageK, per_tile = (n_kt + kChunkStages - 1) / kChunkStages;
  int slot = 0;
  uint32_t ph = 0, issued = 0, par = 0;
  bool ok = true;
  for (int item = tiles.first(); ok && item < tiles.stop(); item = tiles.next(item))
    for (int c = 0; c < per_tile; ++c) {
      ok = !__any_sync(0xffffffffu, *abort_ptr) && poll_warp(&way.chunk_empty[slot], ph ^ 1u, a.err);
      if (!ok) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(&way.chunk_full[slot], tx);
        load(slot, item, c * CR, &way.chunk_full[slot]);
      }
      issued |= 1u << slot;
      par = (par & ~(1u << slot)) | (ph << slot);
      if (++slot == way.n_chunks) slot = 0, ph ^= 1u;
    }
  if (!ok) *abort_ptr = 1;
  for (int c = 0; c < way.n_chunks; ++c)  // no copy may be in flight when the CTA exits
    if (issued & (1u << c)) poll_warp(&way.chunk_full[c], (par >> c) & 1u, a.err);
}

// The same with the width of the loads by the weights' alignment: 16 through the chunks.
template <int FMT, int CR, int BLOCKS, bool SWAP, typename RowOf, typename Arrive>
__device__ __forceinline__ void scale_warp_by(int w, const TileArgs& a, const Tiles& tiles, const ScaleWay& way,
                                              const RowOf& w_row, const Arrive& arrive, volatile int* abort_ptr) {
  if (a.w_align == 16)
    scale_warp<FMT, 16, CR, BLOCKS, SWAP>(w, a, tiles, way, w_row, arrive, abort_ptr);
  else if (a.w_align == 8)
    scale_warp<FMT, 8, CR, BLOCKS, SWAP>(w, a, tiles, way, w_row, arrive, abort_ptr);
  else if (a.w_align == 4)
    scale_warp<FMT, 4, CR, BLOCKS, SWAP>(w, a, tiles, way, w_row, arrive, abort_ptr);
  else
    scale_warp<FMT, 1, CR, BLOCKS, SWAP>(w, a, tiles, way, w_row, arrive, abort_ptr);
}

// A warp's 32 rows of a finished tile, BN columns of its TMEM lanes from `acc`, times both factors, through 2 KB of shared
// memory in pieces of 64 bytes per row, 16-byte chunks swizzled by pairs of rows.  Pieces of 32 columns are read from
// `first` on, around the end; after `release` of them `free()` tells the MMA warp.  row0: the warp's first; end: of the
// expert's rows.  roomy: the CTA's last tile, whose pieces find room of their own at `mine` and none waits for the one
// before to leave (the ring of stages, which is done with).
template <int BN, typename TO, typename Free>
__device__ __forceinline__ void store_tile(const TileArgs& a, const CUtensorMap* map_out, uint32_t acc, uint8_t* mine,
                                           int row0, int end, int col0, Fp4Factors f, int first, int release, bool roomy,
                                           const Free& free) {
  constexpr int PW = 64 / int(sizeof(TO)), CW = 16 / int(sizeof(TO));  // columns per piece, per 16-byte chunk
  const int lane = threadIdx.x & 31;
  TO* out = static_cast<TO*>(a.out);
  // whole rows of one expert leave by a copy of the warp's 32 rows; a tile that ends inside, or rows off 16 bytes, by the
  // threads
  const bool copies = a.copy_out && row0 + 32 <= end;
#pragma unroll 1
  for (int i = 0; i < BN / 32; ++i) {
    const int c = first + i < BN / 32 ? first + i : first + i - BN / 32;
    uint32_t p[32];
    tmem_ld32(acc + c * 32, p);
    tmem_wait(p);
    if (i == release - 1) {
      fence_before();  // every lane's reads come before the MMA that overwrites them, across the barrier
      __syncwarp();
      if (lane == 0) free();
    }
#pragma unroll
    for (int pc = 0; pc < 32 / PW; ++pc) {
      if (roomy) {
        if (i || pc) mine += 32 * 64;
      } else {
        if (lane == 0) tma_stores_read();  // the piece before has left
        __syncwarp();
      }
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        float v[CW];
#pragma unroll
        for (int k = 0; k < CW; ++k) v[k] = __uint_as_float(p[pc * PW + ch * CW + k]) * f.first * f.second;
        store_vec<TO, CW>(reinterpret_cast<TO*>(mine + lane * 64 + ((ch ^ ((lane >> 1) & 3)) << 4)), v);
      }
      const int col = col0 + c * 32 + pc * PW;
      if (copies) {
        fence_async();
        __syncwarp();
        if (lane == 0 && col < a.N) tma_store_2d(map_out, col * int(sizeof(TO)), row0, mine);
      } else {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = j * 8 + (lane >> 2), at = col + (lane & 3) * CW;
          const TO* src = reinterpret_cast<const TO*>(mine + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
          if (row0 + r >= end) continue;
          TO* to = out + int64_t(row0 + r) * a.N + at;
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

// A record's factor (1 without one).
__device__ __forceinline__ float row_factor(const TileArgs& a, int row) {
  return a.a_factor ? __ldg(reinterpret_cast<const float*>(a.a_factor + int64_t(min(row, a.S - 1)) * a.a_stride)) : 1.f;
}

// Tensor maps of a product (host): codes and scales of rows and weights, and the stores of 32 rows x 64 bytes.
struct TileMaps {
  CUtensorMap a, w, sa, sw, out;
};
// The descriptors in use, which the launch carries, on their way before the work that it waits for is done.
__device__ __forceinline__ void prefetch_maps(const TileMaps& m, bool w_chunks, bool copy_out) {
  auto one = [](const CUtensorMap& p) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&p)) : "memory");
  };
  one(m.a);
  one(m.w);
  one(m.sa);
  if (w_chunks) one(m.sw);
  if (copy_out) one(m.out);
}
int make_tile_args(const Fp4Product& p, int out_dtype, int a_box, int w_box, int sa_box, int sw_box, int cr, bool copy_out,
                  TileArgs& a, TileMaps& m);

}  // namespace b200moe
