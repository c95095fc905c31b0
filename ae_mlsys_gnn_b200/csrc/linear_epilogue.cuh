// Device side of the linear layers' epilogue (LinearEpilogue).
#pragma once
#include "activation.cuh"
#include "dtypes.cuh"
#include "linear_tc.cuh"

namespace gnn {

// Eight consecutive values of type T at p (16-byte aligned), widened.
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&o)[8]) {
  constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < 8; i += V) {
    const Pack<T, V> a = load_pack(reinterpret_cast<const Pack<T, V>*>(p + i));
#pragma unroll
    for (int j = 0; j < V; ++j) o[i + j] = to_f32(a.v[j]);
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&o)[8]) {
  constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < 8; i += V) {
    Pack<T, V> a;
    a.round_from(o + i);
    store_pack(reinterpret_cast<Pack<T, V>*>(p + i), a);
  }
}

// The epilogue of one element, for outputs whose rows are not whole 16-byte units.
template <class T>
__device__ __forceinline__ void finish_one(const LinearEpilogue& ep, int64_t row, int col, int N, float v) {
  const int64_t at = row * N + col;
  if (ep.col_scale) v *= __ldg(ep.row_scale + row) * __ldg(ep.col_scale + col);
  if (ep.bias) v += to_f32(static_cast<const T*>(ep.bias)[col]);
  if (ep.z) static_cast<T*>(ep.z)[at] = from_f32<T>(v);
  v = act_value<sizeof(T) == 4>(v, ep.act, ep.slope);
  if (ep.residual) v += to_f32(static_cast<const T*>(ep.residual)[at]);
  static_cast<T*>(ep.out)[at] = from_f32<T>(v);
}

}  // namespace gnn
