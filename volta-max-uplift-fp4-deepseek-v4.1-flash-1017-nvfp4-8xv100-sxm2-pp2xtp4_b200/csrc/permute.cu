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
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "vec.cuh"

namespace b200moe {
namespace {

constexpr int kRunRoutes = 2048;  // routes that one CTA ranks: 64 per warp
constexpr int kSortMaxExperts = 1024;
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

// One CTA ranks the routes of one run: ranks within a warp by votes, across
// its warps and the earlier runs by their counts.
__global__ void __launch_bounds__(1024) sort_rows_kernel(const int32_t* __restrict__ ids, int n, int E, int bits,
                                                         const int32_t* __restrict__ counts,
                                                         int32_t* __restrict__ row_of_route,
                                                         int32_t* __restrict__ offsets) {
  extern __shared__ __align__(16) int sort_smem[];
  const int nk = E + 1, warps = blockDim.x >> 5, runs = gridDim.x;
  int* base = sort_smem;         // [nk] first row of each key, then of this run's share of it
  int* before = base + nk;       // [nk] rows of the key in earlier runs
  int* wsum = before + nk;       // [32]
  uint16_t* whist = reinterpret_cast<uint16_t*>(wsum + 32);  // [warps][nk]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_trigger();
  for (int i = threadIdx.x; i < (warps * nk + 1) / 2; i += blockDim.x) reinterpret_cast<uint32_t*>(whist)[i] = 0;
  __syncthreads();

  const int first = blockIdx.x * kRunRoutes + warp * 64 + lane;
  int key[2], rank[2];
  uint16_t* mine = whist + warp * nk;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = first + 32 * j;
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
        earlier += r < int(blockIdx.x) ? c : 0;
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
  int at = incl - own;
  for (int w = 0; w < warp; ++w) at += wsum[w];
  for (int e = lo; e < hi; ++e) {
    const int c = base[e];
    if (blockIdx.x == 0) offsets[e] = at;
    base[e] = at + before[e];
    at += c;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = first + 32 * j;
    if (i >= n) continue;
    const int row = base[key[j]] + whist[warp * nk + key[j]] + rank[j];
    row_of_route[i] = key[j] == E ? ~row : row;
  }
}

size_t sort_smem_bytes(int E, int warps) {
  return size_t(2 * (E + 1) + 32) * sizeof(int) + (size_t(warps) * (E + 1) + 1) / 2 * 4;
}

// --------------------------------------------------------------- row copies
// A CTA per token: its row in pieces of V, each stored to the token's k rows.
template <typename V>
__global__ void __launch_bounds__(256) permute_rows_kernel(const uint8_t* __restrict__ x, int64_t x_stride, int pieces,
                                                           const float* __restrict__ scale, int64_t scale_stride,
                                                           int n_scale, const int32_t* __restrict__ row_of_route,
                                                           int T, int k, uint8_t* __restrict__ rows,
                                                           float* __restrict__ row_scale, uint32_t* err) {
  const int64_t row_bytes = int64_t(pieces) * sizeof(V);
  const int S = T * k;
  pdl_wait();
  pdl_trigger();
  for (int t = blockIdx.x; t < T; t += gridDim.x) {
    const V* src = reinterpret_cast<const V*>(x + t * x_stride);
    const int32_t* rt = row_of_route + int64_t(t) * k;
    constexpr int U = 2;
    for (int c0 = threadIdx.x; c0 < pieces; c0 += U * blockDim.x) {
      V v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * blockDim.x;
        if (c < pieces) v[u] = src[c];
      }
      for (int s = 0; s < k; ++s) {
        const int r = rt[s], p = r < 0 ? ~r : r;
        if (p >= S) {
          set_error(err, kErrBounds);
          continue;
        }
        V* dst = reinterpret_cast<V*>(rows + p * row_bytes);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c0 + u * blockDim.x;
          if (c < pieces) dst[c] = r < 0 ? V{} : v[u];
        }
      }
    }
    if (n_scale)
      for (int i = threadIdx.x; i < k * n_scale; i += blockDim.x) {
        const int s = i / n_scale, j = i - s * n_scale, r = rt[s], p = r < 0 ? ~r : r;
        if (p < S) row_scale[int64_t(p) * n_scale + j] = r < 0 ? 0.f : scale[t * scale_stride + j];
      }
  }
}

// ------------------------------------------------------- weighted return
// A thread owns V columns of one token; eight slots' rows are in flight before
// the first is added.
template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(256) unpermute_kernel(const TI* __restrict__ rows, const int32_t* __restrict__ row_of_route,
                                                        const float* __restrict__ weights, int T, int k, int H,
                                                        TO* __restrict__ out, uint32_t* err) {
  const int S = T * k;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  pdl_wait();
  pdl_trigger();
  if (c >= H) return;
  for (int t = blockIdx.x; t < T; t += gridDim.x) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    const int32_t* rt = row_of_route + int64_t(t) * k;
    const float* wt = weights ? weights + int64_t(t) * k : nullptr;
    constexpr int U = 8;
    for (int s0 = 0; s0 < k; s0 += U) {
      Vec<TI, V> y[U];
      int r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        r[u] = s0 + u < k ? rt[s0 + u] : -1;
        if (r[u] >= S) {
          set_error(err, kErrBounds);
          r[u] = -1;
        }
        if (r[u] >= 0) y[u].load(rows + int64_t(r[u]) * H + c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r[u] < 0) continue;
        const float w = wt ? wt[s0 + u] : 1.f;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(w, y[u].get(i), acc[i]);
      }
    }
    store_vec<TO, V>(out + int64_t(t) * H + c, acc);
  }
}

// A CTA per token: g[t] is read once for up to eight slots; each slot's row is
// read for the dot product and its gradient row written in the same pass.
template <typename TG, typename TI, int V>
__global__ void __launch_bounds__(256) unpermute_grad_kernel(const TG* __restrict__ grad, int64_t grad_stride,
                                                             const TI* __restrict__ rows,
                                                             const int32_t* __restrict__ row_of_route,
                                                             const float* __restrict__ weights, int T, int k, int H,
                                                             TI* __restrict__ grad_rows,
                                                             float* __restrict__ grad_weights, uint32_t* err) {
  constexpr int U = 8;
  __shared__ float part[U][8];
  const int S = T * k, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  pdl_wait();
  pdl_trigger();
  for (int t = blockIdx.x; t < T; t += gridDim.x) {
    const int32_t* rt = row_of_route + int64_t(t) * k;
    for (int s0 = 0; s0 < k; s0 += U) {
      int r[U];
      float w[U], dot[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        r[u] = s0 + u < k ? rt[s0 + u] : S;  // S: no row at all
        if (s0 + u < k && (r[u] >= S || ~r[u] >= S)) {
          set_error(err, kErrBounds);
          r[u] = S;
        }
        w[u] = s0 + u < k && weights ? weights[int64_t(t) * k + s0 + u] : 1.f;
        dot[u] = 0.f;
      }
      for (int c = threadIdx.x * V; c < H; c += blockDim.x * V) {
        Vec<TG, V> g;
        Vec<TI, V> y[U];
        g.load(grad + t * grad_stride + c);
        if (grad_weights) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (r[u] >= 0 && r[u] < S) y[u].load(rows + int64_t(r[u]) * H + c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (r[u] >= S) continue;
          const bool held = r[u] >= 0;
          float o[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float gi = g.get(i);
            if (held && grad_weights) dot[u] = fmaf(gi, y[u].get(i), dot[u]);
            o[i] = held ? w[u] * gi : 0.f;
          }
          if (grad_rows) store_vec<TI, V>(grad_rows + int64_t(held ? r[u] : ~r[u]) * H + c, o);
        }
      }
      if (grad_weights) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int d = 16; d; d >>= 1) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], d);
          if (lane == 0) part[u][warp] = dot[u];
        }
        __syncthreads();
        if (threadIdx.x < U && s0 + threadIdx.x < k) {
          float sum = 0.f;
          for (int j = 0; j < warps; ++j) sum += part[threadIdx.x][j];
          grad_weights[int64_t(t) * k + s0 + threadIdx.x] = sum;
        }
        __syncthreads();
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
  const int V = wide ? VB : 1;
  const int cols = (H + V - 1) / V;
  const int threads = std::min(256, (cols + 31) / 32 * 32);
  const dim3 grid(std::min(T, 65535), (cols + threads - 1) / threads);
  auto kernel = wide ? unpermute_kernel<TI, TO, VB> : unpermute_kernel<TI, TO, 1>;
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
  const int V = wide ? VB : 1;
  const int threads = std::min(256, ((H + V - 1) / V + 31) / 32 * 32);
  auto kernel = wide ? unpermute_grad_kernel<TG, TI, VB> : unpermute_grad_kernel<TG, TI, 1>;
  return launch_chain(kernel, dim3(std::min(T, 148 * 32)), dim3(threads), 0, s, static_cast<const TG*>(grad),
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

extern "C" int b200moe_sort_routes(void* stream, const int32_t* ids, int routes, int num_experts,
                                   int32_t* row_of_route, int32_t* offsets, void* workspace, size_t workspace_bytes) {
  if (!ids || !row_of_route || !offsets || routes < 1 || routes > kSortMaxRoutes || num_experts < 1 ||
      num_experts > kSortMaxExperts)
    return B200MOE_ERR_INVALID_ARG;
  const int runs = (routes + kRunRoutes - 1) / kRunRoutes;
  if (runs > 1 && (!workspace || workspace_bytes < b200moe_sort_workspace_bytes(routes, num_experts)))
    return B200MOE_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int warps = runs > 1 ? 32 : std::max(8, (routes + 63) / 64);
  const size_t smem = sort_smem_bytes(num_experts, warps);
  if (smem > 48 * 1024) {
    static std::atomic<uint64_t> attr_set{0};  // devices whose attribute is set
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return B200MOE_ERR_CUDA;
    if (!(attr_set.load() >> dev & 1)) {
      const cudaError_t e = cudaFuncSetAttribute(sort_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 int(sort_smem_bytes(kSortMaxExperts, 32)));
      if (e != cudaSuccess) return status(e);
      attr_set.fetch_or(uint64_t(1) << dev);
    }
  }
  int32_t* counts = static_cast<int32_t*>(workspace);
  if (runs > 1) {
    const cudaError_t e =
        launch_chain(sort_count_kernel, dim3(runs), dim3(1024), 0, s, ids, routes, num_experts, counts);
    if (e != cudaSuccess) return status(e);
  }
  int bits = 1;
  while ((num_experts + 1) >> bits) ++bits;  // keys 0 .. E, and E + 1 past the last route
  return status(launch_chain(sort_rows_kernel, dim3(runs), dim3(warps * 32), smem, s, ids, routes, num_experts, bits,
                             static_cast<const int32_t*>(counts), row_of_route, offsets));
}

extern "C" int b200moe_permute_rows(void* stream, const void* x, int64_t x_stride, int64_t row_bytes,
                                    const float* scale, int64_t scale_stride, int n_scale,
                                    const int32_t* row_of_route, int T, int k, void* rows, float* row_scale) {
  if (!x || !row_of_route || !rows || !sizes_ok(T, k) || row_bytes < 1 || row_bytes > (1 << 30) || x_stride < 0 ||
      n_scale < 0 || (n_scale && (!scale || !row_scale)))
    return B200MOE_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto fits = [&](int n) { return row_bytes % n == 0 && aligned(x, x_stride, n) && aligned(rows, row_bytes, n); };
  const int piece = fits(16) ? 16 : fits(4) ? 4 : fits(2) ? 2 : 1;
  const int pieces = int(row_bytes / piece);
  const int threads = std::min(256, (pieces + 31) / 32 * 32);
  auto kernel = piece == 16  ? permute_rows_kernel<uint4>
                : piece == 4 ? permute_rows_kernel<uint32_t>
                : piece == 2 ? permute_rows_kernel<uint16_t>
                             : permute_rows_kernel<uint8_t>;
  return status(launch_chain(kernel, dim3(std::min(T, 148 * 32)), dim3(threads), 0, s,
                             static_cast<const uint8_t*>(x), x_stride, pieces, scale, scale_stride, n_scale,
                             row_of_route, T, k, static_cast<uint8_t*>(rows), row_scale, op_error_word()));
}

extern "C" int b200moe_unpermute(void* stream, const void* rows, int dtype, const int32_t* row_of_route,
                                 const float* weights, int T, int k, int H, void* out, int out_dtype) {
  if (!rows || !row_of_route || !out || !sizes_ok(T, k) || H < 1) return B200MOE_ERR_INVALID_ARG;
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
  if (!grad || !row_of_route || !sizes_ok(T, k) || H < 1 || grad_stride < 0 || (!grad_rows && !grad_weights) ||
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
