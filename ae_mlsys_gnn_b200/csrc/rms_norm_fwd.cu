// Root-mean-square norm with the residual's addition, output in the input's type or in 8 bits.
//
//   h = x + residual        y = h * rsqrt(mean(h^2) + eps) * weight
//   fp8: scale = max(amax |y| / 448, 2^-126) per row or per 128 columns, q = e4m3(y / scale)
//
// Bound by HBM: x and residual are read once, y (or q) and h written once; the row stays in
// registers between the sum of squares and the scaling.  y comes from the unrounded fp32 h; the
// only roundings are those of the stored h, y and q.  One group of threads a row and many CTAs:
// walking rows with the next one's loads ahead, as the gradient does, measured slower here (16381 x
// 2048 bf16: 64 against 47 us).
//
// Measured on a B200 (bytes of the arrays over event time): 16381 x 2048 bf16 with residual 47 us,
// 5.7 TB/s = 0.87 of the copy bandwidth; 232965 x 256 fp32 78 us, 6.1 TB/s; 232965 x 602 fp32, whose rows
// allow 8-byte accesses only, 230 us, 4.9 TB/s; e4m3 output, 16384 x 4096, 103 us, 4.6 TB/s, where the
// conversions show (SM busy 0.78).  Rows of odd 16-bit widths move 2 bytes an access: 16384 x 4097
// bf16 206 us.
#include <cuda_fp8.h>
#include <stdio.h>
#include <type_traits>
#include "rms_norm.cuh"

namespace gnn {
namespace {

struct FwdParams {
  const void* x;
  const void* residual;  // nullptr: none
  const void* weight;
  int w_f32;
  int64_t n;
  int d, group;
  float eps;
  void* y;
  void* h;       // nullptr: not wanted
  float* rstd;   // nullptr: not wanted
  uint8_t* q;    // 8-bit form
  float* scale;
  int block;     // columns per scale (0: one scale a row)
  int n_blocks;
};

template <class T, int VEC, int NV, bool FP8, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 512 && sizeof(T) * VEC * NV <= 16 ? 4 : 1) rms_norm_kernel(const FwdParams p) {
  __shared__ float s_sum[32];
  __shared__ int s_max[32];
  extern __shared__ int s_block_max[];  // [rows of this CTA][n_blocks], FP8 with block scales
  const int G = p.group;
  const int local = threadIdx.x / G;
  const int t = threadIdx.x - local * G;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / G) + local;
  const bool live = row < p.n;
  using P = Pack<T, VEC>;
  const int nvec = p.d / VEC;

  if (FP8 && p.block) {
    for (int i = threadIdx.x; i < (int)(blockDim.x / G) * p.n_blocks; i += blockDim.x) s_block_max[i] = 0;
    __syncthreads();
  }

  P a[NV], r[NV];
  const P* xr = reinterpret_cast<const P*>(static_cast<const T*>(p.x) + (live ? row : 0) * p.d);
  const P* rr = reinterpret_cast<const P*>(static_cast<const T*>(p.residual) + (live ? row : 0) * p.d);
  // no condition around the loads (the compiler would move them to their uses): what lies behind the row
  // is its last piece again and is not used
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    a[i] = load_pack(xr + min(t + G * i, nvec - 1));
    if (p.residual) r[i] = load_pack(rr + min(t + G * i, nvec - 1));
  }

  float v[NV][VEC];
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (live && t + G * i < nvec) {
      a[i].widen(v[i]);
      if (p.residual) {
        float f[VEC];
        r[i].widen(f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] += f[j];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) sq = fmaf(v[i][j], v[i][j], sq);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
    }
  }
  const float rstd = rsqrtf(group_sum(sq, G, s_sum) / (float)p.d + p.eps);
  if (live && t == 0 && p.rstd) p.rstd[row] = rstd;

  if (p.h && live) {
    P* hr = reinterpret_cast<P*>(static_cast<T*>(p.h) + row * p.d);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + G * i < nvec) {
        P o;
        o.round(v[i]);
        store_pack(hr + t + G * i, o);
      }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (live && t + G * i < nvec) {
      float w[VEC];
      load_weight<T, VEC>(p.weight, p.w_f32, (int64_t)(t + G * i) * VEC, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = v[i][j] * rstd * w[j];
    }

  if constexpr (!FP8) {
    if (!live) return;
    P* yr = reinterpret_cast<P*>(static_cast<T*>(p.y) + row * p.d);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + G * i < nvec) {
        P o;
        o.round(v[i]);
        store_pack(yr + t + G * i, o);
      }
  } else {
    // G >= 32 here, so a warp's lanes are one row's neighbours
    int m[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      m[i] = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) m[i] = max(m[i], __float_as_int(fabsf(v[i][j])));
    }
    auto scale_of = [](int bits) {
      const float s = __int_as_float(bits) / 448.f;
      return s < 1.17549435e-38f ? 1.17549435e-38f : s;  // a row of zeros; a NaN stays one
    };
    float row_scale = 0.f;
    int* const bm = s_block_max + local * p.n_blocks;
    if (p.block) {
      // 32 lanes cover 32 * VEC consecutive columns from a multiple of that, i.e. two blocks of
      // 128 for 8 elements a lane and at most one for fewer
      const unsigned half = VEC == 8 ? (threadIdx.x & 16 ? 0xffff0000u : 0xffffu) : kFull;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int g = __reduce_max_sync(half, m[i]);
        const int col = (t + G * i) * VEC;
        if ((threadIdx.x & (VEC == 8 ? 15 : 31)) == 0 && col < p.d && live) atomicMax(bm + col / 128, g);
      }
      __syncthreads();
      if (live)
        for (int b = t; b < p.n_blocks; b += G) p.scale[row * p.n_blocks + b] = scale_of(bm[b]);
    } else {
      int all = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) all = max(all, m[i]);
      row_scale = scale_of(group_max_bits(all, G, s_max));
      if (live && t == 0) p.scale[row] = row_scale;
    }
    if (!live) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (t + G * i) * VEC;
      if (col < p.d) {
        const float inv = 1.f / (p.block ? scale_of(bm[col / 128]) : row_scale);
        Pack<uint8_t, VEC> o;
        if constexpr (VEC % 2 == 0) {  // pairs are rounded by one instruction each
#pragma unroll
          for (int j = 0; j < VEC; j += 2)
            reinterpret_cast<__nv_fp8x2_storage_t*>(o.v)[j / 2] =
                __nv_cvt_float2_to_fp8x2(make_float2(v[i][j] * inv, v[i][j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
        } else {
          o.v[0] = __nv_cvt_float_to_fp8(v[i][0] * inv, __NV_SATFINITE, __NV_E4M3);
        }
        store_pack(reinterpret_cast<Pack<uint8_t, VEC>*>(p.q + row * p.d + col), o);
      }
    }
  }
}

template <bool FP8>
int launch_fwd(FwdParams p, int dtype, int vec, cudaStream_t stream, const char* what) {
  const NormGeom g = norm_geom(p.d, vec, norm_ept(p.d, vec * dtype_bytes(dtype) == 16), FP8 ? 32 : 4);
  p.group = g.group;
  const int64_t grid = (p.n + g.rows - 1) / g.rows;
  if (grid > INT32_MAX) {
    set_last_error("gnn_rms_norm: too many rows");
    return GNN_ERR_LIMIT;
  }
  const size_t smem = FP8 && p.block ? (size_t)g.rows * p.n_blocks * sizeof(int) : 0;
  dispatch_norm<true>(dtype, vec, g.ept, [&](auto tag, auto v, auto nv) {
    using T = decltype(tag);
    constexpr int V = decltype(v)::value, NV = decltype(nv)::value;
    // with whole 16-byte accesses 8 or 16 elements a thread never need more than 512 threads
    constexpr bool kNarrowOnly = V * sizeof(T) == 16 && V * NV < 32;
    if (kNarrowOnly || g.threads <= 512) rms_norm_kernel<T, V, NV, FP8, 512><<<(unsigned)grid, g.threads, smem, stream>>>(p);
    else if constexpr (!kNarrowOnly) rms_norm_kernel<T, V, NV, FP8, 1024><<<(unsigned)grid, g.threads, smem, stream>>>(p);
  });
  return check_launch(what);
}

}  // namespace

int norm_check(const char* what, int dtype, int weight_dtype, int64_t n, int64_t d) {
  char msg[200];
  if (dtype_bytes(dtype) == 0 || (weight_dtype != dtype && weight_dtype != GNN_F32)) {
    snprintf(msg, sizeof msg, "%s: the rows are fp32, bf16 or fp16, the weight of the same type or fp32", what);
    set_last_error(msg);
    return GNN_ERR_UNSUPPORTED;
  }
  if (n < 0 || d < 1) {
    snprintf(msg, sizeof msg, "%s: bad size", what);
    set_last_error(msg);
    return GNN_ERR_INVALID_ARG;
  }
  if (d > kNormMaxWidth) {
    snprintf(msg, sizeof msg, "%s: rows of more than %d elements are not supported", what, kNormMaxWidth);
    set_last_error(msg);
    return GNN_ERR_LIMIT;
  }
  return GNN_OK;
}

}  // namespace gnn

using namespace gnn;

extern "C" int gnn_rms_norm_fwd(const void* x, const void* residual, const void* weight, int dtype, int weight_dtype,
                                int64_t n, int64_t d, float eps, void* y, void* h, float* rstd, cudaStream_t stream) {
  if (int rc = norm_check("gnn_rms_norm_fwd", dtype, weight_dtype, n, d)) return rc;
  if (n == 0) return GNN_OK;
  if (!x || !weight || !y) {
    set_last_error("gnn_rms_norm_fwd: null pointer");
    return GNN_ERR_INVALID_ARG;
  }
  const int elt = dtype_bytes(dtype);
  const int vec = row_vec(d, elt, (uintptr_t)x | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)y | (uintptr_t)h);
  FwdParams p{x, residual, weight, weight_dtype == GNN_F32 && dtype != GNN_F32, n, (int)d, 0, eps, y, h, rstd,
              nullptr, nullptr, 0, 0};
  return launch_fwd<false>(p, dtype, vec, stream, "gnn_rms_norm_fwd");
}

extern "C" int gnn_rms_norm_fp8(const void* x, const void* residual, const void* weight, int dtype, int weight_dtype,
                                int64_t n, int64_t d, float eps, int block, void* q, float* scale, void* h,
                                cudaStream_t stream) {
  if (int rc = norm_check("gnn_rms_norm_fp8", dtype, weight_dtype, n, d)) return rc;
  if (block != 0 && block != 128) {
    set_last_error("gnn_rms_norm_fp8: block must be 0 (one scale a row) or 128 columns");
    return GNN_ERR_UNSUPPORTED;
  }
  if (n == 0) return GNN_OK;
  if (!x || !weight || !q || !scale) {
    set_last_error("gnn_rms_norm_fp8: null pointer");
    return GNN_ERR_INVALID_ARG;
  }
  const int elt = dtype_bytes(dtype);
  int vec = row_vec(d, elt, (uintptr_t)x | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)h);
  while (vec > 1 && (uintptr_t)q % vec) vec = vec > 2 ? 2 : 1;
  const int n_blocks = block ? (int)((d + block - 1) / block) : 1;
  FwdParams p{x, residual, weight, weight_dtype == GNN_F32 && dtype != GNN_F32, n, (int)d, 0, eps, nullptr, h, nullptr,
              (uint8_t*)q, scale, block, n_blocks};
  return launch_fwd<true>(p, dtype, vec, stream, "gnn_rms_norm_fp8");
}
