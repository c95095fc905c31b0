// Rows between token order and expert order: a stable counting sort of the (token, choice) pairs by
// expert, the copy of every token's row to its experts, the weighted sum back, and their gradients.
//
//   slots[t,j]  = position of pair (t,j) among the pairs sorted by expert (ties: pair order), -1 when
//                 its expert is not one of 0..E-1
//   dispatch    out[slots[t,j]] = x[t]                   gradient: combine with unit weights
//   combine     out[t] = sum_j w[t,j] * rows[slots[t,j]]
//   its gradients: grad_rows[slots[t,j]] = w[t,j] * g[t],  grad_w[t,j] = <g[t], rows[slots[t,j]]>
//
// All row kernels run in token order: a token's row is read (or written) once and its k expert rows
// once, whole rows at a time, so nothing is scattered at less than a row and no atomics are used:
// HBM-bound.  Rows of the sorted array behind the last kept pair are written as zeros.
#include <stdio.h>
#include <type_traits>
#include "common.cuh"
#include "dtypes.cuh"

namespace gnn {
namespace {

constexpr int kMaxExperts = 1024;  // a counter per expert and warp in shared memory
constexpr int kMaxChoices = 32;
constexpr int kSortWarps = 8;
constexpr int kMinChunk = 2048;    // pairs per CTA of the sort

// Pairs per CTA: one CTA up to kMinChunk pairs, never more CTAs than 148 (every CTA reads all
// CTAs' counts).
int64_t sort_chunk(int64_t pairs) {
  int64_t c = (pairs + 147) / 148;
  if (c < kMinChunk) c = kMinChunk;
  return (c + 255) / 256 * 256;
}

__device__ __forceinline__ int expert_of(const void* ids, int wide, int64_t i, int64_t n, int E) {
  if (i >= n) return E;
  const int64_t v = wide ? static_cast<const int64_t*>(ids)[i] : static_cast<const int*>(ids)[i];
  return v >= 0 && v < E ? (int)v : E;  // E: belongs to no expert
}

// A warp's contiguous share of a chunk is walked 32 pairs at a time; lanes with the same expert find
// each other by a match, so ranks follow pair order without any atomic.
__device__ __forceinline__ void count_share(const void* ids, int wide, int64_t lo, int64_t hi, int64_t n, int E, int* counts) {
  const int lane = threadIdx.x & 31;
  for (int64_t i = lo; i < hi; i += 32) {
    const int e = expert_of(ids, wide, i + lane, n, E);
    const unsigned same = __match_any_sync(kFull, e);
    if (e < E && lane == __ffs(same) - 1) counts[e] += __popc(same);
    __syncwarp();
  }
}

// Counts of every chunk but none of the places: hist[chunk][E].
__global__ void __launch_bounds__(kSortWarps * 32) expert_count_kernel(const void* ids, int wide, int64_t n, int E, int64_t chunk,
                                                                       int* hist) {
  extern __shared__ int s_counts[];  // [warps][E]
  const int warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kSortWarps * E; i += blockDim.x) s_counts[i] = 0;
  __syncthreads();
  const int64_t share = chunk / kSortWarps, lo = blockIdx.x * chunk + warp * share;
  count_share(ids, wide, lo, min(lo + share, n), n, E, s_counts + warp * E);
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) sum += s_counts[w * E + e];
    hist[(size_t)blockIdx.x * E + e] = sum;
  }
}

// Places: first[e] = pairs of lower experts + pairs of e in earlier chunks, then the warps' shares in
// order.  hist == nullptr: a single chunk, whose own counts are all there is.
__global__ void __launch_bounds__(kSortWarps * 32) expert_place_kernel(const void* ids, int wide, int64_t n, int E, int64_t chunk,
                                                                       const int* hist, int* offsets, int* slots) {
  extern __shared__ int s_counts[];  // [warps][E], then first[E]
  __shared__ int s_warp[kSortWarps];
  int* const first = s_counts + kSortWarps * E;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * E; i += blockDim.x) s_counts[i] = 0;
  __syncthreads();
  const int64_t share = chunk / kSortWarps, lo = blockIdx.x * chunk + warp * share, hi = min(lo + share, n);
  count_share(ids, wide, lo, hi, n, E, s_counts + warp * E);
  __syncthreads();

  // totals and earlier chunks per expert, and the scan over experts, 256 experts at a time
  int carry = 0;
  for (int e0 = 0; e0 < E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    int total = 0, earlier = 0;
    if (e < E) {
      if (hist) {
        for (int c = 0; c < (int)gridDim.x; ++c) {
          const int v = __ldg(hist + (size_t)c * E + e);
          total += v;
          if (c < (int)blockIdx.x) earlier += v;
        }
      } else {
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) total += s_counts[w * E + e];
      }
    }
    int scan = total;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int up = __shfl_up_sync(kFull, scan, s);
      if (lane >= s) scan += up;
    }
    if (lane == 31) s_warp[warp] = scan;
    __syncthreads();
    int before = carry, all = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      if (w < warp) before += s_warp[w];
      all += s_warp[w];
    }
    carry += all;
    if (e < E) {
      const int start = before + scan - total;
      first[e] = start + earlier;
      if (blockIdx.x == 0) offsets[e] = start;
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) offsets[E] = carry;
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    int at = first[e];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = s_counts[w * E + e];
      s_counts[w * E + e] = at;
      at += c;
    }
  }
  __syncthreads();
  int* const next = s_counts + warp * E;
  for (int64_t i = lo; i < hi; i += 32) {
    const int e = expert_of(ids, wide, i + lane, n, E);
    const unsigned same = __match_any_sync(kFull, e);
    const int rank = __popc(same & ((1u << lane) - 1));
    int at = -1;
    if (e < E) at = next[e] + rank;
    __syncwarp();
    if (e < E && rank == 0) next[e] += __popc(same);
    __syncwarp();
    if (i + lane < n) slots[i + lane] = at;
  }
}

struct RowParams {
  const void* x;       // token rows: dispatch's input, combine's output gradient
  const void* rows;    // rows in expert order
  const void* weights; // [T,k] or nullptr (unit weights)
  const int* slots;    // [T,k]
  const int* kept;     // device: rows in use
  int w_f32;
  int64_t tokens;
  int k, width;
  void* out;           // rows the kernel writes
  void* grad_w;
};

// Zeros for the rows of the sorted array that no pair fills, spread over the grid.
template <class P>
__device__ __forceinline__ void zero_unused(P* out, int64_t used, int64_t rows, int nvec) {
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  P z;
  memset(&z, 0, sizeof z);
  for (int64_t r = used + (int64_t)blockIdx.x * warps + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * warps)
    for (int v = lane; v < nvec; v += 32) store_pack(out + r * nvec + v, z);
}

// A slot as an index that is inside the sorted array, or -1.
__device__ __forceinline__ int64_t slot_at(const int* slots, int64_t i, int64_t rows) {
  const int64_t s = __ldg(slots + i);
  return s >= 0 && s < rows ? s : -1;
}

// One warp moves one 32-lane segment of one token's row to its k places.
template <class P>
__global__ void __launch_bounds__(256) expert_dispatch_kernel(const RowParams p, int nvec, int segs) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = p.tokens * p.k;
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  P* const out = static_cast<P*>(p.out);
  if (unit < p.tokens * segs) {
    const int64_t t = unit / segs;
    const int v = (int)(unit - t * segs) * 32 + lane;
    if (v < nvec) {
      const P a = load_pack(static_cast<const P*>(p.x) + t * nvec + v);
      for (int j = 0; j < p.k; ++j) {
        const int64_t s = slot_at(p.slots, t * p.k + j, rows);
        if (s >= 0) store_pack(out + s * nvec + v, a);
      }
    }
  }
  zero_unused(out, min((int64_t)max(__ldg(p.kept), 0), rows), rows, nvec);
}

__device__ __forceinline__ float pair_weight(const RowParams& p, int64_t i, float) {
  return p.weights ? static_cast<const float*>(p.weights)[i] : 1.f;
}
template <class T>
__device__ __forceinline__ float pair_weight(const RowParams& p, int64_t i, T) {
  if (!p.weights) return 1.f;
  return p.w_f32 ? static_cast<const float*>(p.weights)[i] : to_f32(static_cast<const T*>(p.weights)[i]);
}

constexpr int kBatch = 8;  // expert rows of a token requested together

// One warp sums one 32-lane segment of one token's expert rows, in fp32 and in the order of the
// choices.
template <class T, int VEC>
__global__ void __launch_bounds__(256) expert_combine_kernel(const RowParams p, int nvec, int segs) {
  using P = Pack<T, VEC>;
  const int lane = threadIdx.x & 31;
  const int64_t rows = p.tokens * p.k;
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (unit >= p.tokens * segs) return;
  const int64_t t = unit / segs;
  const int v = (int)(unit - t * segs) * 32 + lane;
  if (v >= nvec) return;
  const P* const in = static_cast<const P*>(p.rows);
  float sum[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
  for (int j0 = 0; j0 < p.k; j0 += kBatch) {
    P a[kBatch];
    float w[kBatch];
    bool ok[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int64_t s = j0 + j < p.k ? slot_at(p.slots, t * p.k + j0 + j, rows) : -1;
      ok[j] = s >= 0;
      if (ok[j]) {
        a[j] = load_pack(in + s * nvec + v);
        w[j] = pair_weight(p, t * p.k + j0 + j, T{});
      }
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (ok[j]) {
        float f[VEC];
        a[j].widen(f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = fmaf(w[j], f[i], sum[i]);
      }
  }
  P o;
  o.round(sum);
  store_pack(static_cast<P*>(p.out) + t * nvec + v, o);
}

// `share` warps of a CTA work on one token: gradient rows and the k dot products.
template <class T, int VEC>
__global__ void __launch_bounds__(256) expert_combine_bwd_kernel(const RowParams p, int nvec, int share) {
  using P = Pack<T, VEC>;
  __shared__ float s_dot[8][kBatch];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = warp % share;
  const int64_t rows = p.tokens * p.k;
  const int64_t t = (int64_t)blockIdx.x * (8 / share) + warp / share;
  const bool live = t < p.tokens;
  const P* const in = static_cast<const P*>(p.rows);
  const P* const g = static_cast<const P*>(p.x) + (live ? t : 0) * nvec;
  P* const out = static_cast<P*>(p.out);
  for (int j0 = 0; j0 < p.k; j0 += kBatch) {
    int64_t s[kBatch];
    float w[kBatch], dot[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const bool is = live && j0 + j < p.k;
      s[j] = is ? slot_at(p.slots, t * p.k + j0 + j, rows) : -1;
      w[j] = is ? pair_weight(p, t * p.k + j0 + j, T{}) : 0.f;
      dot[j] = 0.f;
    }
    for (int v = part * 32 + lane; v < nvec; v += share * 32) {
      P a[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (s[j] >= 0) a[j] = load_pack(in + s[j] * nvec + v);
      float f[VEC];
      load_pack(g + v).widen(f);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (s[j] >= 0) {
          float r[VEC];
          a[j].widen(r);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            dot[j] = fmaf(f[i], r[i], dot[j]);
            r[i] = w[j] * f[i];
          }
          P o;
          o.round(r);
          store_pack(out + s[j] * nvec + v, o);
        }
    }
    warp_multi_sum<kBatch>(dot, lane);  // lane 4 j holds the sum of choice j
    if (share > 1) {
      if ((lane & 3) == 0) s_dot[warp][lane >> 2] = dot[0];
      __syncthreads();
      if (part == 0 && (lane & 3) == 0)
        for (int q = 1; q < share; ++q) dot[0] += s_dot[warp + q][lane >> 2];
      __syncthreads();
    }
    const int j = j0 + (lane >> 2);
    if (live && part == 0 && (lane & 3) == 0 && j < p.k && p.grad_w) {
      if (p.w_f32) static_cast<float*>(p.grad_w)[t * p.k + j] = dot[0];
      else static_cast<T*>(p.grad_w)[t * p.k + j] = from_f32<T>(dot[0]);
    }
  }
  zero_unused(out, min((int64_t)max(__ldg(p.kept), 0), rows), rows, nvec);
}

int fail(int code, const char* what, const char* why) {
  char msg[256];
  snprintf(msg, sizeof msg, "%s: %s", what, why);
  set_last_error(msg);
  return code;
}

int check_rows(const char* what, int dtype, int weight_dtype, int64_t tokens, int k, int64_t width) {
  if (dtype_bytes(dtype) == 0 || (weight_dtype != dtype && weight_dtype != GNN_F32))
    return fail(GNN_ERR_UNSUPPORTED, what, "rows are fp32, bf16 or fp16, weights of the same type or fp32");
  if (tokens < 0 || k < 1 || width < 1) return fail(GNN_ERR_INVALID_ARG, what, "bad size");
  if (k > kMaxChoices) return fail(GNN_ERR_LIMIT, what, "more than 32 choices a token");
  if (tokens * k >= (1LL << 31) || width >= (1LL << 31)) return fail(GNN_ERR_LIMIT, what, "size exceeds int32");
  return GNN_OK;
}

// Calls f with the type and the elements per access.
template <class F>
void dispatch_rows(int dtype, int vec, F&& f) {
  auto with = [&](auto tag) {
    constexpr int kFullVec = 16 / (int)sizeof(tag);
    if (vec == kFullVec) f(tag, std::integral_constant<int, kFullVec>{});
    else if (vec == 2) f(tag, std::integral_constant<int, 2>{});
    else f(tag, std::integral_constant<int, 1>{});
  };
  if (dtype == GNN_F32) with(float{});
  else if (dtype == GNN_BF16) with(__nv_bfloat16{});
  else with(__half{});
}

bool grid_for(int64_t units, int per_cta, unsigned* grid) {
  const int64_t g = (units + per_cta - 1) / per_cta;
  *grid = (unsigned)g;
  return g <= INT32_MAX;
}

}  // namespace
}  // namespace gnn

using namespace gnn;

extern "C" int gnn_expert_sort_workspace_bytes(int64_t pairs, int n_experts, size_t* bytes) {
  if (!bytes || pairs < 0 || n_experts < 1)
    return fail(GNN_ERR_INVALID_ARG, "gnn_expert_sort_workspace_bytes", "bad argument");
  const int64_t chunk = sort_chunk(pairs), chunks = (pairs + chunk - 1) / chunk;
  *bytes = chunks > 1 ? (size_t)chunks * n_experts * sizeof(int) + 16 : 0;
  return GNN_OK;
}

extern "C" int gnn_expert_sort(const void* ids, int ids_are_64_bit, int64_t pairs, int n_experts, int* offsets, int* slots,
                               void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  const char* const what = "gnn_expert_sort";
  if (pairs < 0 || n_experts < 1) return fail(GNN_ERR_INVALID_ARG, what, "bad size");
  if (n_experts > kMaxExperts) return fail(GNN_ERR_LIMIT, what, "more than 1024 experts");
  if (pairs >= (1LL << 31)) return fail(GNN_ERR_LIMIT, what, "2^31 pairs or more");
  if (!offsets || (pairs && (!ids || !slots))) return fail(GNN_ERR_INVALID_ARG, what, "null pointer");
  if (pairs == 0) {
    cudaMemsetAsync(offsets, 0, (size_t)(n_experts + 1) * sizeof(int), stream);
    return check_launch(what);
  }
  size_t need = 0;
  gnn_expert_sort_workspace_bytes(pairs, n_experts, &need);
  if (need && (!workspace || workspace_bytes < need)) return fail(GNN_ERR_WORKSPACE, what, "workspace too small");
  const int64_t chunk = sort_chunk(pairs);
  const int chunks = (int)((pairs + chunk - 1) / chunk);
  int* const hist = chunks > 1 ? (int*)(((uintptr_t)workspace + 15) & ~(uintptr_t)15) : nullptr;
  const size_t counts = (size_t)kSortWarps * n_experts * sizeof(int);
  if (hist) expert_count_kernel<<<chunks, kSortWarps * 32, counts, stream>>>(ids, ids_are_64_bit, pairs, n_experts, chunk, hist);
  expert_place_kernel<<<chunks, kSortWarps * 32, counts + n_experts * sizeof(int), stream>>>(
      ids, ids_are_64_bit, pairs, n_experts, chunk, hist, offsets, slots);
  return check_launch(what);
}

extern "C" int gnn_expert_dispatch(const void* x, const int* slots, const int* kept, int dtype, int64_t tokens, int k,
                                   int64_t width, void* out, cudaStream_t stream) {
  const char* const what = "gnn_expert_dispatch";
  if (int rc = check_rows(what, dtype, dtype, tokens, k, width)) return rc;
  if (tokens == 0) return GNN_OK;
  if (!x || !slots || !kept || !out) return fail(GNN_ERR_INVALID_ARG, what, "null pointer");
  const int vec = row_vec(width, dtype_bytes(dtype), (uintptr_t)x | (uintptr_t)out);
  RowParams p{x, nullptr, nullptr, slots, kept, 0, tokens, k, (int)width, out, nullptr};
  const int nvec = (int)(width / vec), segs = (nvec + 31) / 32;
  unsigned grid;
  if (!grid_for(tokens * segs, 8, &grid)) return fail(GNN_ERR_LIMIT, what, "too many rows");
  switch (vec * dtype_bytes(dtype)) {  // a copy: only the size of the access matters
    case 16: expert_dispatch_kernel<Pack<float, 4>><<<grid, 256, 0, stream>>>(p, nvec, segs); break;
    case 8: expert_dispatch_kernel<Pack<float, 2>><<<grid, 256, 0, stream>>>(p, nvec, segs); break;
    case 4: expert_dispatch_kernel<Pack<float, 1>><<<grid, 256, 0, stream>>>(p, nvec, segs); break;
    default: expert_dispatch_kernel<Pack<__half, 1>><<<grid, 256, 0, stream>>>(p, nvec, segs); break;
  }
  return check_launch(what);
}

extern "C" int gnn_expert_combine(const void* rows, const void* weights, const int* slots, int dtype, int weight_dtype,
                                  int64_t tokens, int k, int64_t width, void* out, cudaStream_t stream) {
  const char* const what = "gnn_expert_combine";
  if (int rc = check_rows(what, dtype, weight_dtype, tokens, k, width)) return rc;
  if (tokens == 0) return GNN_OK;
  if (!rows || !slots || !out) return fail(GNN_ERR_INVALID_ARG, what, "null pointer");
  const int vec = row_vec(width, dtype_bytes(dtype), (uintptr_t)rows | (uintptr_t)out);
  RowParams p{nullptr, rows, weights, slots, nullptr, weight_dtype == GNN_F32, tokens, k, (int)width, out, nullptr};
  const int nvec = (int)(width / vec), segs = (nvec + 31) / 32;
  unsigned grid;
  if (!grid_for(tokens * segs, 8, &grid)) return fail(GNN_ERR_LIMIT, what, "too many rows");
  dispatch_rows(dtype, vec, [&](auto tag, auto v) {
    expert_combine_kernel<decltype(tag), decltype(v)::value><<<grid, 256, 0, stream>>>(p, nvec, segs);
  });
  return check_launch(what);
}

extern "C" int gnn_expert_combine_bwd(const void* grad_out, const void* rows, const void* weights, const int* slots,
                                      const int* kept, int dtype, int weight_dtype, int64_t tokens, int k, int64_t width,
                                      void* grad_rows, void* grad_weights, cudaStream_t stream) {
  const char* const what = "gnn_expert_combine_bwd";
  if (int rc = check_rows(what, dtype, weight_dtype, tokens, k, width)) return rc;
  if (tokens == 0) return GNN_OK;
  if (!grad_out || !rows || !weights || !slots || !kept || !grad_rows) return fail(GNN_ERR_INVALID_ARG, what, "null pointer");
  const int vec = row_vec(width, dtype_bytes(dtype), (uintptr_t)grad_out | (uintptr_t)rows | (uintptr_t)grad_rows);
  RowParams p{grad_out, rows, weights, slots, kept, weight_dtype == GNN_F32, tokens, k, (int)width, grad_rows, grad_weights};
  const int nvec = (int)(width / vec), segs = (nvec + 31) / 32;
  // several warps a token while there are too few tokens to fill the GPU with a warp each
  int share = 1;
  while (share < 8 && share < segs && tokens * share < 148 * 32) share *= 2;
  unsigned grid;
  if (!grid_for(tokens, 8 / share, &grid)) return fail(GNN_ERR_LIMIT, what, "too many rows");
  dispatch_rows(dtype, vec, [&](auto tag, auto v) {
    expert_combine_bwd_kernel<decltype(tag), decltype(v)::value><<<grid, 256, 0, stream>>>(p, nvec, share);
  });
  return check_launch(what);
}
