// Token rows sorted by expert and back, with their gradients.
//
// row_of_route[t * k + s] = p: route s of token t is row p of the expert order
// (a stable sort of the routes by expert id; expert e owns rows offsets[e] ..
// offsets[e + 1]).  A route without an expert (id outside [0, E)) sorts last
// and holds ~p: its row p is kept as zeros and takes no part in any sum.  The
// map is a bijection of routes and rows, so every kernel below goes by token:
// a token's columns are read once and each of its k rows is touched once, with
// no inverse map, no atomics and sums in slot order (equal inputs give equal
// bits).
//
//   permute          rows[p] = x[t]                              reads T H, writes T k H
//   its gradient     gx[t] = sum_s g[p_s]                        reads T k H, writes T H
//   unpermute        out[t] = sum_s w[t, s] rows[p_s]            reads T k H, writes T H
//   its gradients    grows[p_s] = w[t, s] g[t], gw[t, s] = <g[t], rows[p_s]>
//                                                                reads T H + T k H, writes T k H
//
// All four are bound by HBM.  Products and sums are in f32, rounded once where
// a value is stored in fewer bits.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "internal.h"
#include "vec.cuh"

namespace b200moe {
namespace {

constexpr int kRunRoutes = 2048;  // routes that one CTA ranks: 64 per warp
constexpr int kSortMaxExperts = 1024;
constexpr int kUnpermuteCtas = 12;  // per SM: several waves even out the rows' latencies
constexpr int kGradCtas = 12;
// single columns per thread where rows are not whole aligned vectors: 4,001 x 2001 bf16, k 8, takes 37 us (gradients
// 102) with four, 42 (118) with two and 44 (111) with eight
constexpr int kColumns = 4;
constexpr int kSortMaxRoutes = 1 << 26;

// ------------------------------------------------------------------ sort
__device__ __forceinline__ int sort_key(const int32_t* ids, int i, int E) {
  const int id = ids[i];
  return unsigned(id) < unsigned(E) ? id : E;
}

// Lanes of the warp that hold this lane's key: one vote per key bit.
__device__ __forceinline__ uint32_t same_key_lanes(int key, int bits) {
  uint32_t m = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const uint32_t v = __ballot_sync(0xffffffffu, (key >> b) & 1);
    m &= (key >> b) & 1 ? v : ~v;
  }
  return m;
}

__global__ void __launch_bounds__(1024) sort_count_kernel(const int32_t* __restrict__ ids, int n, int E,
                                                          int32_t* __restrict__ counts) {
  __shared__ int hist[kSortMaxExperts + 1];
  pdl_wait();
  pdl_trigger();
  for (int e = threadIdx.x; e <= E; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  const int end = min(n, (int(blockIdx.x) + 1) * kRunRoutes);
  for (int i = blockIdx.x * kRunRoutes + threadIdx.x; i < end; i += blockDim.x) atomicAdd(&hist[sort_key(ids, i, E)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += blockDim.x) counts[int64_t(blockIdx.x) * (E + 1) + e] = hist[e];
}

// The rows of one run's routes (the thread's two: first, first + 32 of its warp's 64): ranks within a warp by votes,
// across the CTA's warps and the earlier runs by their counts. Also the offsets, by the CTA asked to.
__device__ __forceinline__ void sort_run(const int32_t* __restrict__ ids, int n, int E, int bits, int run, int runs,
                                         const int32_t* __restrict__ counts, int* smem, bool write_offsets,
                                         int32_t* __restrict__ offsets, int (&at)[2], int (&row)[2]) {
  const int nk = E + 1, warps = blockDim.x >> 5;
  int* base = smem;              // [nk] first row of each key, then of this run's share of it
  int* before = base + nk;       // [nk] rows of the key in earlier runs
  int* wsum = before + nk;       // [32]
  uint16_t* whist = reinterpret_cast<uint16_t*>(wsum + 32);  // [warps][nk]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < (warps * nk + 1) / 2; i += blockDim.x) reinterpret_cast<uint32_t*>(whist)[i] = 0;
  __syncthreads();

  const int first = run * kRunRoutes + warp * 64 + lane;
  int key[2], rank[2];
  uint16_t* mine = whist + warp * nk;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = at[j] = first + 32 * j;
    key[j] = i < n ? sort_key(ids, i, E) : nk;
    const uint32_t peers = same_key_lanes(key[j], bits);
    const int below = __popc(peers & ((1u << lane) - 1u));
    rank[j] = below + (i < n ? mine[key[j]] : 0);
    __syncwarp();
    if (i < n && below == 0) mine[key[j]] = uint16_t(mine[key[j]] + __popc(peers));
    __syncwarp();
  }
  __syncthreads();
  // exclusive prefix over the warps; the key's total over all runs
  for (int e = threadIdx.x; e < nk; e += blockDim.x) {
    int sum = 0;
    for (int w = 0; w < warps; ++w) {
      const int c = whist[w * nk + e];
      whist[w * nk + e] = uint16_t(sum);
      sum += c;
    }
    int earlier = 0;
    if (runs > 1) {
      sum = 0;
#pragma unroll 8
      for (int r = 0; r < runs; ++r) {
        const int c = counts[int64_t(r) * nk + e];
        sum += c;
        earlier += r < run ? c : 0;
      }
    }
    base[e] = sum;
    before[e] = earlier;
  }
  __syncthreads();
  // exclusive scan of the totals over the keys
  const int per = (nk + blockDim.x - 1) / blockDim.x;
  const int lo = min(nk, int(threadIdx.x) * per), hi = min(nk, lo + per);
  int own = 0;
  for (int e = lo; e < hi; ++e) own += base[e];
  int incl = own;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, d);
    incl += lane >= d ? v : 0;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  int sum = incl - own;
  for (int w = 0; w < warp; ++w) sum += wsum[w];
  for (int e = lo; e < hi; ++e) {
    const int c = base[e];
    if (write_offsets) offsets[e] = sum;
    base[e] = sum + before[e];
    sum += c;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (at[j] >= n) continue;
    const int r = base[key[j]] + whist[warp * nk + key[j]] + rank[j];
    row[j] = key[j] == E ? ~r : r;
  }
}

__global__ void __launch_bounds__(1024) sort_rows_kernel(const int32_t* __restrict__ ids, int n, int E, int bits,
                                                         const int32_t* __restrict__ counts,
                                                         int32_t* __restrict__ row_of_route,
                                                         int32_t* __restrict__ offsets) {
  extern __shared__ __align__(16) int sort_smem[];
  pdl_wait();
  pdl_trigger();
  int at[2], row[2];
  sort_run(ids, n, E, bits, blockIdx.x, gridDim.x, counts, sort_smem, blockIdx.x == 0, offsets, at, row);
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (at[j] < n) row_of_route[at[j]] = row[j];
}

size_t sort_smem_bytes(int E, int warps) {
  return size_t(2 * (E + 1) + 32) * sizeof(int) + (size_t(warps) * (E + 1) + 1) / 2 * 4;
}

// --------------------------------------------------------------- row copies
struct CopyArgs {
  const uint8_t* x;  // [T], x_stride bytes apart
  int64_t x_stride;
  int pieces;  // of sizeof(V) bytes per row
  const float* scale;
  int64_t scale_stride;
  int n_scale;
  int T, k;
  uint8_t* rows;
  float* row_scale;
  uint32_t* err;
};

// One token: its row in pieces of V, each stored to the token's k rows (rt: its part of row_of_route).
template <typename V>
__device__ __forceinline__ void copy_token(const CopyArgs& a, int t, const int32_t* rt) {
  const int64_t row_bytes = int64_t(a.pieces) * sizeof(V);
  const int S = a.T * a.k;
  const V* src = reinterpret_cast<const V*>(a.x + t * a.x_stride);
  constexpr int U = sizeof(V) == 16 ? 2 : 8;  // pieces in flight
  for (int c0 = threadIdx.x; c0 < a.pieces; c0 += U * blockDim.x) {
    V v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * blockDim.x;
      if (c < a.pieces) v[u] = src[c];
    }
    for (int s = 0; s < a.k; ++s) {
      const int r = rt[s], p = r < 0 ? ~r : r;
      if (p >= S) {
        set_error(a.err, kErrBounds);
        continue;
      }
      V* dst = reinterpret_cast<V*>(a.rows + p * row_bytes);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * blockDim.x;
        if (c < a.pieces) dst[c] = r < 0 ? V{} : v[u];
      }
    }
  }
  if (a.n_scale)
    for (int i = threadIdx.x; i < a.k * a.n_scale; i += blockDim.x) {
      const int s = i / a.n_scale, j = i - s * a.n_scale, r = rt[s], p = r < 0 ? ~r : r;
      if (p < S) a.row_scale[int64_t(p) * a.n_scale + j] = r < 0 ? 0.f : a.scale[t * a.scale_stride + j];
    }
}

template <typename V>
__global__ void __launch_bounds__(256) permute_rows_kernel(const CopyArgs a, const int32_t* __restrict__ row_of_route) {
  pdl_wait();
  pdl_trigger();
  for (int t = blockIdx.x; t < a.T; t += gridDim.x) copy_token<V>(a, t, row_of_route + int64_t(t) * a.k);
}

// Calls of one run: every CTA sorts all routes itself, CTA 0 writes the tables, and each copies its tokens' rows. One
// launch where the sort and the copies took two.
template <typename V>
__global__ void __launch_bounds__(1024) sort_permute_kernel(const int32_t* __restrict__ ids, int E, int bits,
                                                            const CopyArgs a, int32_t* __restrict__ row_of_route,
                                                            int32_t* __restrict__ offsets) {
  extern __shared__ __align__(16) int sort_smem[];
  __shared__ int32_t rows_sm[kRunRoutes];
  const int n = a.T * a.k;
  pdl_wait();
  pdl_trigger();
  int at[2], row[2];
  sort_run(ids, n, E, bits, 0, 1, nullptr, sort_smem, blockIdx.x == 0, offsets, at, row);
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (at[j] < n) {
      rows_sm[at[j]] = row[j];
      if (blockIdx.x == 0) row_of_route[at[j]] = row[j];
    }
  __syncthreads();
  for (int t = blockIdx.x; t < a.T; t += gridDim.x) copy_token<V>(a, t, rows_sm + t * a.k);
}

// ------------------------------------------------------- weighted return
// A thread owns V columns (of `load_columns`) of its CTA's tokens; eight slots' rows are in flight
// before the first is added, and the next token's routes are loaded (a lane per
// slot) while they are.
template <typename TI, typename TO, int V, bool WIDE>
__global__ void __launch_bounds__(256) unpermute_kernel(const TI* __restrict__ rows, const int32_t* __restrict__ row_of_route,
                                                        const float* __restrict__ weights, int T, int k, int H,
                                                        TO* __restrict__ out, uint32_t* err) {
  constexpr int U = 8;
  const int S = T * k, slot = threadIdx.x & (U - 1);
  const int step = blockDim.x;
  const int c = blockIdx.y * step * V + (WIDE ? threadIdx.x * V : threadIdx.x);
  pdl_wait();
  pdl_trigger();
  auto routes = [&](int t, int s0, int& r, float& w) {
    const bool in = t < T && s0 + slot < k;
    r = in ? row_of_route[int64_t(t) * k + s0 + slot] : -1;
    w = in && weights ? weights[int64_t(t) * k + s0 + slot] : 1.f;
    if (r >= S) {
      set_error(err, kErrBounds);
      r = -1;
    }
  };
  int r_next;
  float w_next;
  routes(blockIdx.x, 0, r_next, w_next);
  for (int t = blockIdx.x; t < T; t += gridDim.x) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int s0 = 0; s0 < k; s0 += U) {
      int r[U];
      float w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        r[u] = __shfl_sync(0xffffffffu, r_next, u);
        w[u] = __shfl_sync(0xffffffffu, w_next, u);
      }
      Vec<TI, V> y[U];
      if (c < H) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (r[u] >= 0) load_columns<WIDE>(y[u], rows + int64_t(r[u]) * H, c, step, H);
      }
      const bool more = s0 + U < k;
      routes(more ? t : t + gridDim.x, more ? s0 + U : 0, r_next, w_next);
      if (c < H) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (r[u] < 0) continue;
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = fmaf(w[u], y[u].get(i), acc[i]);
        }
      }
    }
    if (c < H) store_columns<WIDE>(out + int64_t(t) * H, c, step, H, acc);
  }
}

// The sums over a warp of eight values per lane, in 9 shuffles: each exchange
// halves what a lane still holds. Lane 4 j holds the sum of value j (bits 2-4 of
// the lane choose the value).
__device__ __forceinline__ float warp_sum8(const float (&v)[8], int lane) {
  float a[4], b[2];
  const bool h16 = lane & 16, h8 = lane & 8, h4 = lane & 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float send = h16 ? v[i] : v[i + 4], keep = h16 ? v[i + 4] : v[i];
    a[i] = keep + __shfl_xor_sync(0xffffffffu, send, 16);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float send = h8 ? a[i] : a[i + 2], keep = h8 ? a[i + 2] : a[i];
    b[i] = keep + __shfl_xor_sync(0xffffffffu, send, 8);
  }
  float c = (h4 ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, h4 ? b[0] : b[1], 4);
  c += __shfl_xor_sync(0xffffffffu, c, 2);
  c += __shfl_xor_sync(0xffffffffu, c, 1);
  return c;
}

// A CTA per token: g[t] is read once for up to eight slots; each slot's row is
// read for the dot product and its gradient row written in the same pass.
// CTAs per SM, for 4096 tokens of 8 x 4096: 16-bit rows and gradients take 98 us with three, 114 with two (although
// the 80 registers of three spill 72 to 80 bytes); f32 gradients of 16-bit rows 132 with three (160 bytes), 105 with two.
template <typename TG, typename TI, int V, bool WIDE>
__global__ void __launch_bounds__(256, WIDE && sizeof(TG) == 2 ? 3 : 2) unpermute_grad_kernel(const TG* __restrict__ grad, int64_t grad_stride,
                                                             const TI* __restrict__ rows,
                                                             const int32_t* __restrict__ row_of_route,
                                                             const float* __restrict__ weights, int T, int k, int H,
                                                             TI* __restrict__ grad_rows,
                                                             float* __restrict__ grad_weights, uint32_t* err) {
  constexpr int U = 8;
  __shared__ float part[2][U][8];
  const int S = T * k, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int slot = threadIdx.x & (U - 1);
  pdl_wait();
  pdl_trigger();
  auto routes = [&](int t, int s0, int& r, float& w) {
    const bool in = t < T && s0 + slot < k;
    r = in ? row_of_route[int64_t(t) * k + s0 + slot] : S;  // S: no row at all
    w = in && weights ? weights[int64_t(t) * k + s0 + slot] : 1.f;
    if (in && (r >= S || ~r >= S)) {
      set_error(err, kErrBounds);
      r = S;
    }
  };
  int r_next, flip = 0;
  float w_next;
  routes(blockIdx.x, 0, r_next, w_next);
  for (int t = blockIdx.x; t < T; t += gridDim.x) {
    for (int s0 = 0; s0 < k; s0 += U, flip ^= 1) {
      int r[U];
      float w[U], dot[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        r[u] = __shfl_sync(0xffffffffu, r_next, u);
        w[u] = __shfl_sync(0xffffffffu, w_next, u);
        if (r[u] < 0) w[u] = 0.f;
        dot[u] = 0.f;
      }
      const bool more = s0 + U < k;
      routes(more ? t : t + gridDim.x, more ? s0 + U : 0, r_next, w_next);
      const int step = blockDim.x;
      for (int c = WIDE ? threadIdx.x * V : threadIdx.x; c < H; c += step * V) {
        Vec<TG, V> g;
        Vec<TI, V> y[U];
        load_columns<WIDE>(g, grad + t * grad_stride, c, step, H);
        if (grad_weights) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (r[u] >= 0 && r[u] < S) load_columns<WIDE>(y[u], rows + int64_t(r[u]) * H, c, step, H);
        }
        float gv[V];
#pragma unroll
        for (int i = 0; i < V; ++i) gv[i] = g.get(i);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (r[u] >= S) continue;
          if (grad_weights && r[u] >= 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) dot[u] = fmaf(gv[i], y[u].get(i), dot[u]);
          }
          if (grad_rows) {
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = r[u] >= 0 ? w[u] * gv[i] : 0.f;  // zeros also where g is not finite
            store_columns<WIDE>(grad_rows + int64_t(r[u] >= 0 ? r[u] : ~r[u]) * H, c, step, H, o);
          }
        }
      }
      if (grad_weights) {
        const float sum = warp_sum8(dot, lane);
        if ((lane & 3) == 0) part[flip][lane >> 2][warp] = sum;
        __syncthreads();  // the other buffer's readers have passed the last barrier
        if (threadIdx.x < U && s0 + threadIdx.x < k) {
          float total = 0.f;
          for (int j = 0; j < warps; ++j) total += part[flip][threadIdx.x][j];
          grad_weights[int64_t(t) * k + s0 + threadIdx.x] = total;
        }
      }
    }
  }
}

bool aligned(const void* p, int64_t stride_bytes, int n) {
  return reinterpret_cast<uintptr_t>(p) % n == 0 && stride_bytes % n == 0;
}

template <typename TI, typename TO>
cudaError_t run_unpermute(cudaStream_t s, const void* rows, const int32_t* row_of_route, const float* weights, int T,
                          int k, int H, void* out, uint32_t* err) {
  constexpr int VB = 16 / sizeof(TI);
  const bool wide = H % VB == 0 && aligned(rows, 16, 16) && aligned(out, 16, 16);
  const int V = wide ? VB : kColumns;
  const int cols = (H + V - 1) / V;
  const int threads = std::min(256, (cols + 31) / 32 * 32);
  const int slices = (cols + threads - 1) / threads;
  const dim3 grid(std::min(T, std::max(1, sm_count() * kUnpermuteCtas / slices)), slices);
  auto kernel = wide ? unpermute_kernel<TI, TO, VB, true> : unpermute_kernel<TI, TO, kColumns, false>;
  return launch_chain(kernel, grid, dim3(threads), 0, s, static_cast<const TI*>(rows), row_of_route, weights, T, k, H,
                      static_cast<TO*>(out), err);
}

template <typename TG, typename TI>
cudaError_t run_unpermute_grad(cudaStream_t s, const void* grad, int64_t grad_stride, const void* rows,
                               const int32_t* row_of_route, const float* weights, int T, int k, int H,
                               void* grad_rows, float* grad_weights, uint32_t* err) {
  constexpr int VB = 16 / sizeof(TI);
  const bool wide = H % VB == 0 && aligned(rows, 16, 16) && aligned(grad, grad_stride * int64_t(sizeof(TG)), 16) &&
                    aligned(grad_rows, 16, 16);
  const int V = wide ? VB : kColumns;
  const int threads = std::min(256, ((H + V - 1) / V + 31) / 32 * 32);
  auto kernel = wide ? unpermute_grad_kernel<TG, TI, VB, true> : unpermute_grad_kernel<TG, TI, kColumns, false>;
  return launch_chain(kernel, dim3(std::min(T, sm_count() * kGradCtas)), dim3(threads), 0, s, static_cast<const TG*>(grad),
                      grad_stride, static_cast<const TI*>(rows), row_of_route, weights, T, k, H,
                      static_cast<TI*>(grad_rows), grad_weights, err);
}

bool sizes_ok(int T, int k) { return T >= 1 && k >= 1 && k <= 1024 && int64_t(T) * k <= kSortMaxRoutes; }

int status(cudaError_t e) {
  if (e == cudaSuccess) return B200MOE_OK;
  cudaGetLastError();
  return B200MOE_ERR_CUDA;
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" size_t b200moe_sort_workspace_bytes(int routes, int num_experts) {
  if (routes <= kRunRoutes || num_experts < 1) return 0;
  return size_t((routes + kRunRoutes - 1) / kRunRoutes) * (num_experts + 1) * sizeof(int32_t);
}

static int sort_warps(int routes) { return routes > kRunRoutes ? 32 : std::max(8, (routes + 63) / 64); }
static int key_bits(int E) {  // keys 0 .. E, and E + 1 past the last route
  int bits = 1;
  while ((E + 1) >> bits) ++bits;
  return bits;
}

// Lets a sort kernel use the shared memory of kSortMaxExperts.
template <typename K>
static cudaError_t sort_smem_limit(K kernel, std::atomic<uint64_t>& set) {
  int dev = 0;
  const cudaError_t g = cudaGetDevice(&dev);
  if (g != cudaSuccess || dev >= 64) return g != cudaSuccess ? g : cudaErrorInvalidDevice;
  if (set.load() >> dev & 1) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             int(sort_smem_bytes(kSortMaxExperts, 32)));
  if (e == cudaSuccess) set.fetch_or(uint64_t(1) << dev);
  return e;
}

template <typename V>
static cudaError_t run_sort_permute(cudaStream_t s, const int32_t* ids, int E, const CopyArgs& a, int32_t* row_of_route,
                                    int32_t* offsets) {
  static std::atomic<uint64_t> set{0};
  const cudaError_t e = sort_smem_limit(sort_permute_kernel<V>, set);
  if (e != cudaSuccess) return e;
  const int warps = sort_warps(a.T * a.k);
  return launch_chain(sort_permute_kernel<V>, dim3(std::min(a.T, sm_count())), dim3(warps * 32),
                      sort_smem_bytes(E, warps), s, ids, E, key_bits(E), a, row_of_route, offsets);
}

extern "C" int b200moe_sort_routes(void* stream, const int32_t* ids, int routes, int num_experts,
                                   int32_t* row_of_route, int32_t* offsets, void* workspace, size_t workspace_bytes) {
  if (!ids || !row_of_route || !offsets || routes < 1 || routes > kSortMaxRoutes || num_experts < 1 ||
      num_experts > kSortMaxExperts)
    return B200MOE_ERR_INVALID_ARG;
  const int runs = (routes + kRunRoutes - 1) / kRunRoutes;
  if (runs > 1 && (!workspace || workspace_bytes < b200moe_sort_workspace_bytes(routes, num_experts)))
    return B200MOE_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  static std::atomic<uint64_t> set{0};
  cudaError_t e = sort_smem_limit(sort_rows_kernel, set);
  if (e != cudaSuccess) return status(e);
  int32_t* counts = static_cast<int32_t*>(workspace);
  if (runs > 1) {
    e = launch_chain(sort_count_kernel, dim3(runs), dim3(1024), 0, s, ids, routes, num_experts, counts);
    if (e != cudaSuccess) return status(e);
  }
  const int warps = sort_warps(routes);
  return status(launch_chain(sort_rows_kernel, dim3(runs), dim3(warps * 32), sort_smem_bytes(num_experts, warps), s,
                             ids, routes, num_experts, key_bits(num_experts), static_cast<const int32_t*>(counts),
                             row_of_route, offsets));
}

extern "C" int b200moe_permute(void* stream, const int32_t* ids, int num_experts, const void* x, int64_t x_stride,
                               int64_t row_bytes, const float* scale, int64_t scale_stride, int n_scale, int T, int k,
                               int32_t* row_of_route, int32_t* offsets, void* rows, float* row_scale, void* workspace,
                               size_t workspace_bytes) {
  if (!ids || !x || !row_of_route || !offsets || !rows || !sizes_ok(T, k) || row_bytes < 1 || row_bytes > (1 << 30) ||
      x_stride < 0 || n_scale < 0 || (n_scale && (!scale || !row_scale)) || num_experts < 1 ||
      num_experts > kSortMaxExperts)
    return B200MOE_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto fits = [&](int n) { return row_bytes % n == 0 && aligned(x, x_stride, n) && aligned(rows, row_bytes, n); };
  const int piece = fits(16) ? 16 : fits(4) ? 4 : fits(2) ? 2 : 1;
  const CopyArgs a{static_cast<const uint8_t*>(x), x_stride, int(row_bytes / piece), scale, scale_stride, n_scale, T, k,
                   static_cast<uint8_t*>(rows), row_scale, op_error_word()};
  if (T * k <= kRunRoutes) {
    auto run = piece == 16  ? run_sort_permute<uint4>
               : piece == 4 ? run_sort_permute<uint32_t>
               : piece == 2 ? run_sort_permute<uint16_t>
                            : run_sort_permute<uint8_t>;
    return status(run(s, ids, num_experts, a, row_of_route, offsets));
  }
  const int st = b200moe_sort_routes(stream, ids, T * k, num_experts, row_of_route, offsets, workspace, workspace_bytes);
  if (st) return st;
  const int threads = std::min(256, (a.pieces + 31) / 32 * 32);
  auto kernel = piece == 16  ? permute_rows_kernel<uint4>
                : piece == 4 ? permute_rows_kernel<uint32_t>
                : piece == 2 ? permute_rows_kernel<uint16_t>
                             : permute_rows_kernel<uint8_t>;
  return status(launch_chain(kernel, dim3(std::min(T, 148 * 32)), dim3(threads), 0, s, a,
                             static_cast<const int32_t*>(row_of_route)));
}

extern "C" int b200moe_unpermute(void* stream, const void* rows, int dtype, const int32_t* row_of_route,
                                 const float* weights, int T, int k, int H, void* out, int out_dtype) {
  if (!rows || !row_of_route || !out || !sizes_ok(T, k) || H < 1 || H > (1 << 28)) return B200MOE_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > B200MOE_F32 || (out_dtype != dtype && out_dtype != B200MOE_F32)) return B200MOE_ERR_DTYPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint32_t* err = op_error_word();
  const bool f32 = out_dtype == B200MOE_F32;
  auto run = dtype == B200MOE_F16    ? (f32 ? run_unpermute<__half, float> : run_unpermute<__half, __half>)
             : dtype == B200MOE_BF16 ? (f32 ? run_unpermute<__nv_bfloat16, float>
                                            : run_unpermute<__nv_bfloat16, __nv_bfloat16>)
                                     : run_unpermute<float, float>;
  return status(run(s, rows, row_of_route, weights, T, k, H, out, err));
}

extern "C" int b200moe_unpermute_grad(void* stream, const void* grad, int grad_dtype, int64_t grad_stride,
                                      const void* rows, int dtype, const int32_t* row_of_route, const float* weights,
                                      int T, int k, int H, void* grad_rows, float* grad_weights) {
  if (!grad || !row_of_route || !sizes_ok(T, k) || H < 1 || H > (1 << 28) || grad_stride < 0 || (!grad_rows && !grad_weights) ||
      (grad_weights && !rows))
    return B200MOE_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > B200MOE_F32 || (grad_dtype != dtype && grad_dtype != B200MOE_F32)) return B200MOE_ERR_DTYPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint32_t* err = op_error_word();
  const bool f32 = grad_dtype == B200MOE_F32;
  auto run = dtype == B200MOE_F16    ? (f32 ? run_unpermute_grad<float, __half> : run_unpermute_grad<__half, __half>)
             : dtype == B200MOE_BF16 ? (f32 ? run_unpermute_grad<float, __nv_bfloat16>
                                            : run_unpermute_grad<__nv_bfloat16, __nv_bfloat16>)
                                     : run_unpermute_grad<float, float>;
  return status(run(s, grad, grad_stride, rows, row_of_route, weights, T, k, H, grad_rows, grad_weights, err));
}
