// Element types of the feed-forward operators: vectors of VEC elements of float, bfloat16 or
// half, widened to fp32 on the way in and rounded once (to nearest even) on the way out.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <type_traits>
#include "../../include/gnn_b200.h"

namespace gnn {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// VEC elements of T moved with one access of VEC * sizeof(T) bytes (at most 16).
template <class T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
  static_assert(VEC * sizeof(T) <= 16, "one access moves at most 16 bytes");
  T v[VEC];
  __device__ __forceinline__ void widen(float (&o)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = to_f32(v[i]);
  }
  // Pairs are rounded by one instruction each.
  __device__ __forceinline__ void round(const float (&o)[VEC]) { round_from(o); }
  __device__ __forceinline__ void round_from(const float* o) {
    if constexpr (VEC % 2 == 0 && std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) reinterpret_cast<__nv_bfloat162*>(v)[i / 2] = __floats2bfloat162_rn(o[i], o[i + 1]);
    } else if constexpr (VEC % 2 == 0 && std::is_same_v<T, __half>) {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) reinterpret_cast<__half2*>(v)[i / 2] = __floats2half2_rn(o[i], o[i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = from_f32<T>(o[i]);
    }
  }
};

// One access of the whole pack, cached as usual.
template <class P>
__device__ __forceinline__ P load_pack(const P* p) {
  P o;
  if constexpr (sizeof(P) == 16) *reinterpret_cast<uint4*>(&o) = *reinterpret_cast<const uint4*>(p);
  else if constexpr (sizeof(P) == 8) *reinterpret_cast<uint2*>(&o) = *reinterpret_cast<const uint2*>(p);
  else if constexpr (sizeof(P) == 4) *reinterpret_cast<uint32_t*>(&o) = *reinterpret_cast<const uint32_t*>(p);
  else o = *p;
  return o;
}
template <class P>
__device__ __forceinline__ void store_pack(P* p, const P& o) {
  if constexpr (sizeof(P) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&o);
  else if constexpr (sizeof(P) == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(&o);
  else if constexpr (sizeof(P) == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(&o);
  else *p = o;
}

// Bytes of one element of a GNN_F32 / GNN_BF16 / GNN_F16 array, 0 for another code.
inline int dtype_bytes(int dtype) { return dtype == GNN_F32 ? 4 : dtype == GNN_BF16 || dtype == GNN_F16 ? 2 : 0; }

// Elements per access for rows of d elements: 16 bytes where every row starts on a 16-byte
// boundary, else pairs, else single elements.  The base pointers must allow it too.
inline int row_vec(int64_t d, int elt, uintptr_t all_pointers) {
  if ((d * elt) % 16 == 0 && all_pointers % 16 == 0) return 16 / elt;
  if (d % 2 == 0 && all_pointers % (2 * elt) == 0) return 2;
  return 1;
}

}  // namespace gnn
