// Row layout shared by the root-mean-square norm kernels.
//
// A row of d elements belongs to a group of G threads (4, 8, 16 or 32 lanes of one warp, or any
// number of whole warps); thread t of the group owns the vectors t, t + G, t + 2G, ... (NV of them,
// VEC elements each), holds them in registers from the load to the store, and the row is
// therefore read once.  EPT = NV * VEC elements per thread.
#pragma once
#include "common.cuh"
#include "dtypes.cuh"

namespace gnn {

constexpr int kNormMaxWidth = 32768;  // 1024 threads of 32 elements

struct NormGeom {
  int vec, ept;        // elements per access, elements per thread
  int group;           // threads per row
  int threads, rows;   // threads and rows of a CTA
};

// Sum (or maximum of non-negative floats, as integers) over a group.  `slots` holds 32 words of
// shared memory per use in a row; only groups of several warps touch it, and then the whole CTA calls.
__device__ __forceinline__ float group_sum(float v, int G, float* slots) {
  if (G <= 32) {
    for (int s = G >> 1; s > 0; s >>= 1) v += __shfl_xor_sync(kFull, v, s);
    return v;
  }
  v = warp_sum(v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = threadIdx.x / G * (G >> 5);  // a CTA may hold several groups of whole warps
  if (lane == 0) slots[warp] = v;
  __syncthreads();
  return warp_sum(lane < (G >> 5) ? slots[first + lane] : 0.f);
}
// |x| >= 0, so the bit patterns order like the values, and a NaN orders above infinity: it is kept.
__device__ __forceinline__ int group_max_bits(int v, int G, int* slots) {
  v = __reduce_max_sync(kFull, v);
  if (G == 32) return v;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) slots[warp] = v;
  __syncthreads();
  return __reduce_max_sync(kFull, lane < (G >> 5) ? slots[lane] : 0);
}

// Weight vector in either type; w_f32 is uniform over the grid.
template <class T, int VEC>
__device__ __forceinline__ void load_weight(const void* w, int w_f32, int64_t col, float (&o)[VEC]) {
  if (w_f32) {
    const float* p = static_cast<const float*>(w) + col;
    if constexpr (VEC % 4 == 0) {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(p + i));
        o[i] = f.x; o[i + 1] = f.y; o[i + 2] = f.z; o[i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = __ldg(p + i);
    }
  } else {
    reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(w) + col)->widen(o);
  }
}

// Elements per thread.  Many threads with few elements each keep more loads in flight, but the wide
// rows of the forward pass run better as two CTAs of 512 threads an SM than as one of 1024 (8192 x
// 8192 bf16: 106 against 166 us); rows of narrow accesses (16384 x 4098: 166 against 217 us) and the
// gradient (8192 x 8192: 189 against 273 us), whose registers do not last for 16 elements, stay at 8 until 1024
// threads hold the row.  `mid`: the kernel has a form with 16.
inline int norm_ept(int64_t d, bool mid) {
  if (mid) return d <= 4096 ? 8 : d <= 8192 ? 16 : 32;
  return d <= 8192 ? 8 : 32;
}

// Threads per row and rows per CTA: `ept` elements a thread, at least `min_group` threads a row.
inline NormGeom norm_geom(int64_t d, int vec, int ept, int min_group) {
  NormGeom g;
  g.vec = vec;
  g.ept = ept;
  int need = (int)((d + ept - 1) / ept), group = min_group;
  while (group < need && group < 32) group *= 2;
  g.group = need > 32 ? (need + 31) / 32 * 32 : group;
  group = g.group;
  g.threads = group > 32 ? group : 128;
  g.rows = g.threads / group;
  return g;
}

// Calls f with compile-time (T, VEC, EPT) for a type code and a geometry.
template <bool MID, class T, class F>
void dispatch_vec_ept(int vec, int ept, F&& f) {
  constexpr int kFullVec = 16 / (int)sizeof(T);
  auto with_ept = [&](auto v) {
    constexpr int V = decltype(v)::value;
    if constexpr (MID && V == kFullVec)
      if (ept == 16) return f(T{}, v, std::integral_constant<int, 16 / V>{});
    if (ept == 8) return f(T{}, v, std::integral_constant<int, 8 / V>{});
    return f(T{}, v, std::integral_constant<int, 32 / V>{});
  };
  if (vec == kFullVec) return with_ept(std::integral_constant<int, kFullVec>{});
  if (vec == 2) return with_ept(std::integral_constant<int, 2>{});
  return with_ept(std::integral_constant<int, 1>{});
}
template <bool MID, class F>
void dispatch_norm(int dtype, int vec, int ept, F&& f) {
  if (dtype == GNN_F32) return dispatch_vec_ept<MID, float>(vec, ept, f);
  if (dtype == GNN_BF16) return dispatch_vec_ept<MID, __nv_bfloat16>(vec, ept, f);
  return dispatch_vec_ept<MID, __half>(vec, ept, f);
}

// Argument checks common to the three entry points; what = entry point's name for the message.
int norm_check(const char* what, int dtype, int weight_dtype, int64_t n, int64_t d);

}  // namespace gnn
