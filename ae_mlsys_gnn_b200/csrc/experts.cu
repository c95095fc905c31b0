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
//
// Measured on a B200, 16411 tokens, 8 of 128 experts, width 2048 bf16, 1/8 of the tokens padding:
// dispatch 95 us (6.2 TB/s, 0.95 of the copy bandwidth), combine 103 us (5.1), its gradient 170 us (6.2),
// sort 19 us in two launches.  The combine's loads without branches between them were what counted:
// with a condition around each load the compiler moved the loads to their uses (303 us).
#include <stdio.h>
#include <type_traits>
#include "common.cuh"
#include "dtypes.cuh"

namespace gnn {
namespace {

constexpr int kMaxExperts = 1024;  // a counter per expert and warp in shared memory
constexpr int kMaxChoices = 32;
constexpr int kSortWarps = 8;
constexpr int kMinChunk = 1024;    // pairs per CTA of the sort
constexpr int kAhead = 4;          // groups of 32 ids a warp has under way

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

// A warp's contiguous share of a chunk is walked 32 pairs at a time, kAhead groups of ids requested
// together; lanes with the same expert find each other by a match, so ranks follow pair order without
// any atomic.  f(first pair of the group, this lane's expert).
template <class F>
__device__ __forceinline__ void walk_share(const void* ids, int wide, int64_t lo, int64_t hi, int64_t n, int E, F&& f) {
  const int lane = threadIdx.x & 31;
  for (int64_t i = lo; i < hi; i += 32 * kAhead) {
    int e[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) e[a] = i + 32 * a < hi ? expert_of(ids, wide, i + 32 * a + lane, n, E) : E;
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
      if (i + 32 * a < hi) f(i + 32 * a, e[a]);
  }
}
__device__ __forceinline__ void count_share(const void* ids, int wide, int64_t lo, int64_t hi, int64_t n, int E, int* counts) {
  const int lane = threadIdx.x & 31;
  walk_share(ids, wide, lo, hi, n, E, [&](int64_t, int e) {
    const unsigned same = __match_any_sync(kFull, e);
    if (e < E && lane == __ffs(same) - 1) counts[e] += __popc(same);
    __syncwarp();
  });
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
  extern __shared__ int s_counts[];  // [warps][E], then total[E] and earlier[E], later first[E]
  __shared__ int s_warp[kSortWarps];
  int* const s_total = s_counts + kSortWarps * E;
  int* const s_earlier = s_total + E;
  int* const first = s_total;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < (kSortWarps + 2) * E; i += blockDim.x) s_counts[i] = 0;
  __syncthreads();
  const int64_t share = chunk / kSortWarps, lo = blockIdx.x * chunk + warp * share, hi = min(lo + share, n);
  if (hist) {
    // every warp takes each eighth chunk, lanes along the experts; integer sums, so their order is free
    for (int e = lane; e < E; e += 32) {
      int total = 0, earlier = 0;
#pragma unroll 8
      for (int c = warp; c < (int)gridDim.x; c += kSortWarps) {
        const int v = __ldg(hist + (size_t)c * E + e);
        total += v;
        if (c < (int)blockIdx.x) earlier += v;
      }
      atomicAdd(s_total + e, total);
      atomicAdd(s_earlier + e, earlier);
    }
  }
  count_share(ids, wide, lo, hi, n, E, s_counts + warp * E);
  __syncthreads();

  // totals and earlier chunks per expert, and the scan over experts, 256 experts at a time
  int carry = 0;
  for (int e0 = 0; e0 < E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    int total = 0, earlier = 0;
    if (e < E) {
      if (hist) {
        total = s_total[e];
        earlier = s_earlier[e];
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
  walk_share(ids, wide, lo, hi, n, E, [&](int64_t i, int e) {
    const unsigned same = __match_any_sync(kFull, e);
    const int rank = __popc(same & ((1u << lane) - 1));
    int at = -1;
    if (e < E) at = next[e] + rank;
    __syncwarp();
    if (e < E && rank == 0) next[e] += __popc(same);
    __syncwarp();
    if (i + lane < n) slots[i + lane] = at;
  });
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

// One warp moves one segment of one token's row to its k places; narrow accesses move several pieces a
// lane.
template <class P>
constexpr int kCopies = sizeof(P) >= 8 ? 1 : 4;
template <class P>
__global__ void __launch_bounds__(256) expert_dispatch_kernel(const RowParams p, int nvec, int segs) {
  constexpr int U = kCopies<P>;
  const int lane = threadIdx.x & 31;
  const int64_t rows = p.tokens * p.k;
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  P* const out = static_cast<P*>(p.out);
  if (unit < p.tokens * segs) {
    const int64_t t = unit / segs;
    const int v = (int)(unit - t * segs) * (32 * U) + lane;
    // the slots of the token, one per lane (at most 32 choices)
    const int mine = lane < p.k ? (int)slot_at(p.slots, t * p.k + lane, rows) : -1;
    P a[U];
#pragma unroll
    for (int u = 0; u < U; ++u) a[u] = load_pack(static_cast<const P*>(p.x) + t * nvec + min(v + 32 * u, nvec - 1));
    for (int j = 0; j < p.k; ++j) {
      const int s = __shfl_sync(kFull, mine, j);
      if (s >= 0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (v + 32 * u < nvec) store_pack(out + (int64_t)s * nvec + v + 32 * u, a[u]);
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

// Expert rows of a token requested together (KB: the smallest of 2, 4, 8 that is not below k, or 8) and
// pieces of each that a lane requests with them, so that about 128 bytes a lane are under way
// whatever k and the access size are.
template <class P, int KB>
constexpr int kPieces = 8 / KB * (sizeof(P) >= 16 ? 1 : sizeof(P) >= 8 ? 2 : 4);

// `p` where `keep`, else zeros: what a row that must not count is replaced by, NaNs included.
template <class P>
__device__ __forceinline__ P keep_if(bool keep, P p) {
  if constexpr (sizeof(P) % 4 == 0) {
    uint32_t* const w = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
    for (int i = 0; i < (int)sizeof(P) / 4; ++i) w[i] = keep ? w[i] : 0u;
  } else {
    uint16_t* const w = reinterpret_cast<uint16_t*>(&p);
    *w = keep ? *w : (uint16_t)0;
  }
  return p;
}

// One warp sums one segment of one token's expert rows, in fp32 and in the order of the choices.  The
// slots and weights of the token lie one per lane; there are no branches between the loads (a pair
// that goes nowhere reads row 0 and counts as zeros).
template <class T, int VEC, int KB>
__global__ void __launch_bounds__(256) expert_combine_kernel(const RowParams p, int nvec, int segs) {
  using P = Pack<T, VEC>;
  constexpr int U = kPieces<P, KB>;
  const int lane = threadIdx.x & 31;
  const int64_t rows = p.tokens * p.k;
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (unit >= p.tokens * segs) return;
  const int64_t t = unit / segs;
  const int v0 = (int)(unit - t * segs) * (32 * U) + lane;
  const int my_slot = lane < p.k ? (int)slot_at(p.slots, t * p.k + lane, rows) : -1;
  const float my_w = lane < p.k ? pair_weight(p, t * p.k + lane, T{}) : 0.f;
  const P* const in = static_cast<const P*>(p.rows);
  float sum[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[u][i] = 0.f;
  for (int j0 = 0; j0 < p.k; j0 += KB) {
    P a[KB][U];
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      const P* const row = in + (int64_t)max(__shfl_sync(kFull, my_slot, (j0 + j) & 31), 0) * nvec;
#pragma unroll
      for (int u = 0; u < U; ++u) a[j][u] = load_pack(row + min(v0 + 32 * u, nvec - 1));
    }
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      const int s = __shfl_sync(kFull, my_slot, (j0 + j) & 31);
      const bool keep = s >= 0 && j0 + j < p.k;
      const float w = keep ? __shfl_sync(kFull, my_w, (j0 + j) & 31) : 0.f;  // keep is the warp's
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[VEC];
        keep_if(keep, a[j][u]).widen(f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[u][i] = fmaf(w, f[i], sum[u][i]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (v0 + 32 * u < nvec) {
      P o;
      o.round(sum[u]);
      store_pack(static_cast<P*>(p.out) + t * nvec + v0 + 32 * u, o);
    }
}

// `share` warps of a CTA work on one token: gradient rows and the k dot products.
template <class T, int VEC, int KB>
__global__ void __launch_bounds__(256) expert_combine_bwd_kernel(const RowParams p, int nvec, int share) {
  using P = Pack<T, VEC>;
  constexpr int U = kPieces<P, KB>;
  __shared__ float s_dot[8][KB];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = warp % share;
  const int64_t rows = p.tokens * p.k;
  const int64_t t = (int64_t)blockIdx.x * (8 / share) + warp / share;
  const bool live = t < p.tokens;
  const int my_slot = live && lane < p.k ? (int)slot_at(p.slots, t * p.k + lane, rows) : -1;
  const float my_w = live && lane < p.k ? pair_weight(p, t * p.k + lane, T{}) : 0.f;
  const P* const in = static_cast<const P*>(p.rows);
  const P* const g = static_cast<const P*>(p.x) + (live ? t : 0) * nvec;
  P* const out = static_cast<P*>(p.out);
  for (int j0 = 0; j0 < p.k; j0 += KB) {
    int s[KB];
    float w[KB], dot[KB];
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      const int at = __shfl_sync(kFull, my_slot, (j0 + j) & 31);
      s[j] = j0 + j < p.k ? at : -1;
      w[j] = __shfl_sync(kFull, my_w, (j0 + j) & 31);
      dot[j] = 0.f;
    }
    for (int v0 = part * (32 * U) + lane; v0 < nvec; v0 += share * (32 * U)) {
      P a[KB][U], b[U];
#pragma unroll
      for (int u = 0; u < U; ++u) b[u] = load_pack(g + min(v0 + 32 * u, nvec - 1));
#pragma unroll
      for (int j = 0; j < KB; ++j)
#pragma unroll
        for (int u = 0; u < U; ++u) a[j][u] = load_pack(in + (int64_t)max(s[j], 0) * nvec + min(v0 + 32 * u, nvec - 1));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[VEC];
        b[u].widen(f);
        const bool in_row = v0 + 32 * u < nvec;
#pragma unroll
        for (int j = 0; j < KB; ++j) {
          float r[VEC];
          keep_if(s[j] >= 0 && in_row, a[j][u]).widen(r);
          P o;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            dot[j] = fmaf(f[i], r[i], dot[j]);
            r[i] = w[j] * f[i];
          }
          o.round(r);
          if (s[j] >= 0 && in_row) store_pack(out + (int64_t)s[j] * nvec + v0 + 32 * u, o);
        }
      }
    }
    constexpr int kLanes = 32 / KB;  // lane kLanes * j holds the sum of choice j
    warp_multi_sum<KB>(dot, lane);
    if (share > 1) {
      if (lane % kLanes == 0) s_dot[warp][lane / kLanes] = dot[0];
      __syncthreads();
      if (part == 0 && lane % kLanes == 0)
        for (int q = 1; q < share; ++q) dot[0] += s_dot[warp + q][lane / kLanes];
      __syncthreads();
    }
    const int j = j0 + lane / kLanes;
    // a pair that goes nowhere has the gradient 0 even where grad_out is not finite
    const float d = __shfl_sync(kFull, my_slot, j & 31) >= 0 ? dot[0] : 0.f;
    if (live && part == 0 && lane % kLanes == 0 && j < p.k && p.grad_w) {
      if (p.w_f32) static_cast<float*>(p.grad_w)[t * p.k + j] = d;
      else static_cast<T*>(p.grad_w)[t * p.k + j] = from_f32<T>(d);
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

// Calls f with the type, the elements per access and the rows requested together.
template <class F>
void dispatch_rows(int dtype, int vec, int k, F&& f) {
  auto with_batch = [&](auto tag, auto v) {
    if (k <= 2) f(tag, v, std::integral_constant<int, 2>{});
    else if (k <= 4) f(tag, v, std::integral_constant<int, 4>{});
    else f(tag, v, std::integral_constant<int, 8>{});
  };
  auto with = [&](auto tag) {
    constexpr int kFullVec = 16 / (int)sizeof(tag);
    if (vec == kFullVec) with_batch(tag, std::integral_constant<int, kFullVec>{});
    else if (vec == 2) with_batch(tag, std::integral_constant<int, 2>{});
    else with_batch(tag, std::integral_constant<int, 1>{});
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
  expert_place_kernel<<<chunks, kSortWarps * 32, counts + 2 * n_experts * sizeof(int), stream>>>(
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
  const int nvec = (int)(width / vec), seg = 32 * (vec * dtype_bytes(dtype) >= 8 ? 1 : 4), segs = (nvec + seg - 1) / seg;
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
  const int nvec = (int)(width / vec);
  bool fits = true;
  dispatch_rows(dtype, vec, k, [&](auto tag, auto v, auto kb) {
    using T = decltype(tag);
    constexpr int V = decltype(v)::value, KB = decltype(kb)::value, kSeg = 32 * kPieces<Pack<T, V>, KB>;
    const int segs = (nvec + kSeg - 1) / kSeg;
    unsigned grid;
    fits = grid_for(tokens * segs, 8, &grid);
    if (fits) expert_combine_kernel<T, V, KB><<<grid, 256, 0, stream>>>(p, nvec, segs);
  });
  if (!fits) return fail(GNN_ERR_LIMIT, what, "too many rows");
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
  const int nvec = (int)(width / vec);
  bool fits = true;
  dispatch_rows(dtype, vec, k, [&](auto tag, auto v, auto kb) {
    using T = decltype(tag);
    constexpr int V = decltype(v)::value, KB = decltype(kb)::value, kSeg = 32 * kPieces<Pack<T, V>, KB>;
    const int segs = (nvec + kSeg - 1) / kSeg;
    // several warps a token while there are too few tokens to fill the GPU with a warp each
    int share = 1;
    while (share < 8 && share < segs && tokens * share < 148 * 32) share *= 2;
    unsigned grid;
    fits = grid_for(tokens, 8 / share, &grid);
    if (fits) expert_combine_bwd_kernel<T, V, KB><<<grid, 256, 0, stream>>>(p, nvec, share);
  });
  if (!fits) return fail(GNN_ERR_LIMIT, what, "too many rows");
  return check_launch(what);
}
