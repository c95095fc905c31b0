// Gradients of the root-mean-square norm.
//
//   u = grad_y * weight, xhat = h * rstd
//   grad_x = rstd * (u - xhat * mean(u * xhat)) + grad_h,   grad_w = sum_rows grad_y * xhat
//
// One pass: grad_y, h and grad_h are read once and grad_x written once (HBM-bound).  A CTA walks
// many rows, with the next row's loads in flight while the current one is reduced, and its threads
// keep the weight gradient of their own columns in fp32 registers; the CTAs' sums go to a
// workspace and a second kernel adds them in a fixed order, so the result is reproducible.
//
// Measured on a B200: 16381 x 2048 bf16 with residual 73 us, 3.7 TB/s = 0.56 of the copy bandwidth
// (about 30 instructions an element and a reduction per row at three CTAs an SM bound it, DRAM is
// a third busy); 232965 x 256 fp32 120 us, 6.0 TB/s; 232965 x 602 fp32 376 us, 4.5 TB/s.
#include <algorithm>
#include <type_traits>
#include "rms_norm.cuh"

namespace gnn {
namespace {

constexpr int kBwdCtas = 148 * 4;  // partial sums of the weight gradient

struct BwdParams {
  const void* gy;
  const void* gh;  // nullptr: none
  const void* h;
  const void* weight;
  const float* rstd;
  int w_f32;
  int64_t n;
  int d, group;
  void* gx;
  float* partial;  // [gridDim.x][d], nullptr: no weight gradient
};

// The vectors of grad_y, h and grad_h that a thread holds of one row, as they lie in memory.
template <class T, int VEC, int NV>
struct RowParts {
  Pack<T, VEC> gy[NV], h[NV], gh[NV];
  float rstd;
};

// CTAs of MAXT threads that an SM holds: what the registers of a kernel without spills allow (8
// elements a thread: 85 for 16-bit rows, 112 for fp32).  16381 x 2048 bf16: 72.7 us at three CTAs of 256,
// 87 us at two, 84 us at four whose 64 registers spill.
template <class T, int EPT, int MAXT>
constexpr int kResident = MAXT == 256 ? (sizeof(T) == 2 ? 3 : 2) : MAXT == 512 && sizeof(T) * EPT <= 16 ? 2 : 1;

template <class T, int VEC, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, kResident<T, VEC * NV, MAXT>) rms_norm_bwd_kernel(const BwdParams p) {
  __shared__ float s_sum[2][32];
  extern __shared__ float s_gw[];  // [d], groups within one warp only
  using P = Pack<T, VEC>;
  // Narrow shares are requested one row ahead and keep their weights in registers; for wide ones
  // (32 elements a thread) the registers do not suffice, and more bytes are in flight anyway.
  constexpr bool kAhead = NV * VEC <= 8, kKeepWeight = kAhead;
  const int G = p.group;
  const int local = threadIdx.x / G, t = threadIdx.x - local * G;
  const int rows = blockDim.x / G;
  const int nvec = p.d / VEC;
  const T* const gy = static_cast<const T*>(p.gy);
  const T* const gh = static_cast<const T*>(p.gh);
  const T* const h = static_cast<const T*>(p.h);

  float gw[NV][VEC], wk[kKeepWeight ? NV : 1][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) gw[i][j] = 0.f;
    if constexpr (kKeepWeight)
      if (t + G * i < nvec) load_weight<T, VEC>(p.weight, p.w_f32, (int64_t)(t + G * i) * VEC, wk[i]);
  }

  const int64_t step = (int64_t)gridDim.x * rows;
  int64_t row = (int64_t)blockIdx.x * rows + local;  // of the parts requested next
  int64_t at = row * p.d + (int64_t)t * VEC;
  const int64_t stride = step * p.d;
  auto request = [&](RowParts<T, VEC, NV>& q) {
    if (row >= p.n) return;
    q.rstd = p.rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      // behind the row: with several pieces a thread the last one again, without a condition around the
      // loads (16384 x 4098 bf16: 472 against 628 us); a single piece saves the registers (16384 x 4096:
      // 161 against 234 us)
      if (NV == 1 && t >= nvec) break;
      const int k = NV == 1 ? 0 : min(G * i, nvec - 1 - t);
      q.gy[i] = load_pack(reinterpret_cast<const P*>(gy + at) + k);
      q.h[i] = load_pack(reinterpret_cast<const P*>(h + at) + k);
      if (gh) q.gh[i] = load_pack(reinterpret_cast<const P*>(gh + at) + k);
    }
  };

  // With s = rstd * grad_y * weight the products of a row are
  //   dot = sum(s * h) = sum(u * xhat),  grad_w += (rstd * grad_y) * h,
  //   grad_x = s - (rstd^2 * dot / d) * h + grad_h
  // and s stays in registers between the two halves (wide shares form it again).
  RowParts<T, VEC, NV> cur, next;
  if constexpr (kAhead) request(next);
  int turn = 0;
  const float inv_d = 1.f / (float)p.d;
  // every thread of the CTA makes the same number of turns: the sums below are collective
  for (int64_t first = (int64_t)blockIdx.x * rows; first < p.n; first += step, turn ^= 1) {
    const bool live = row < p.n;
    T* const gx = static_cast<T*>(p.gx) + at;
    if constexpr (kAhead) {
      cur = next;
      row += step;
      at += stride;
      request(next);
    } else {
      request(cur);
      row += step;
      at += stride;
    }
    float s[kAhead ? NV : 1][VEC];
    auto scaled = [&](int i, float (&g)[VEC], float (&out)[VEC]) {  // g = rstd * grad_y, out = s
      cur.gy[i].widen(g);
      float w[VEC];
      if constexpr (!kKeepWeight) load_weight<T, VEC>(p.weight, p.w_f32, (int64_t)(t + G * i) * VEC, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        g[j] *= cur.rstd;
        out[j] = g[j] * (kKeepWeight ? wk[kKeepWeight ? i : 0][j] : w[j]);
      }
    };
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (live && t + G * i < nvec) {
        float g[VEC], u[VEC], x[VEC];
        scaled(i, g, u);
        cur.h[i].widen(x);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          gw[i][j] = fmaf(g[j], x[j], gw[i][j]);
          dot = fmaf(u[j], x[j], dot);
          if constexpr (kAhead) s[i][j] = u[j];
        }
      }
    const float c = -cur.rstd * (cur.rstd * (group_sum(dot, G, s_sum[turn]) * inv_d));
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (t + G * i < nvec) {
          float g[VEC], u[VEC], x[VEC];
          if constexpr (!kAhead) scaled(i, g, u);
          cur.h[i].widen(x);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float v = kAhead ? s[kAhead ? i : 0][j] : u[j];
            if (gh) v += to_f32(cur.gh[i].v[j]);
            u[j] = fmaf(c, x[j], v);
          }
          P o;
          o.round(u);
          store_pack(reinterpret_cast<P*>(gx) + G * i, o);
        }
    }
  }

  if (!p.partial) return;
  float* const out = p.partial + (size_t)blockIdx.x * p.d;
  if (rows == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + G * i < nvec)
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[(t + G * i) * VEC + j] = gw[i][j];
  } else {
    // the CTA's groups add their sums one after the other: a fixed order
    for (int g = 0; g < rows; ++g) {
      if (local == g) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (t + G * i < nvec)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              float* const at = s_gw + (t + G * i) * VEC + j;
              *at = g == 0 ? gw[i][j] : *at + gw[i][j];
            }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < p.d; i += blockDim.x) out[i] = s_gw[i];
  }
}

// grad_w[col] = sum of the CTAs' partial sums, 32 columns and 32 row strands a CTA.
template <class W>
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* __restrict__ partial, int parts, int d, W* out) {
  __shared__ float s[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (col < d)
    for (int r = threadIdx.y; r < parts; r += 32) v += partial[(size_t)r * d + col];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = warp_sum(s[threadIdx.x][threadIdx.y]);
  const int c = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < d) out[c] = from_f32<W>(v);
}

NormGeom pick_bwd(int64_t d, int vec) {
  NormGeom g = norm_geom(d, vec, norm_ept(d, false), 4);
  if (g.group <= 128) {  // several rows side by side
    g.rows = 256 / g.group;
    g.threads = g.rows * g.group;
  }
  return g;
}

}  // namespace
}  // namespace gnn

using namespace gnn;

extern "C" int gnn_rms_norm_bwd_workspace_bytes(int64_t n, int64_t d, size_t* bytes) {
  if (!bytes || n < 0 || d < 1) {
    set_last_error("gnn_rms_norm_bwd_workspace_bytes: bad argument");
    return GNN_ERR_INVALID_ARG;
  }
  *bytes = (size_t)(n < kBwdCtas ? n : kBwdCtas) * d * sizeof(float) + 16;
  return GNN_OK;
}

extern "C" int gnn_rms_norm_bwd(const void* grad_y, const void* grad_h, const void* h, const void* weight,
                                const float* rstd, int dtype, int weight_dtype, int64_t n, int64_t d, void* grad_x,
                                void* grad_w, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (int rc = norm_check("gnn_rms_norm_bwd", dtype, weight_dtype, n, d)) return rc;
  const int elt = dtype_bytes(dtype);
  if (n == 0) {
    if (grad_w) cudaMemsetAsync(grad_w, 0, (size_t)d * dtype_bytes(weight_dtype), stream);
    return check_launch("gnn_rms_norm_bwd");
  }
  if (!grad_y || !h || !weight || !rstd || !grad_x) {
    set_last_error("gnn_rms_norm_bwd: null pointer");
    return GNN_ERR_INVALID_ARG;
  }
  size_t need = 0;
  gnn_rms_norm_bwd_workspace_bytes(n, d, &need);
  if (grad_w && (!workspace || workspace_bytes < need)) {
    set_last_error("gnn_rms_norm_bwd: workspace too small");
    return GNN_ERR_WORKSPACE;
  }
  const int vec = row_vec(d, elt, (uintptr_t)grad_y | (uintptr_t)grad_h | (uintptr_t)h | (uintptr_t)weight | (uintptr_t)grad_x);
  const NormGeom g = pick_bwd(d, vec);
  float* const partial = grad_w ? (float*)(((uintptr_t)workspace + 15) & ~(uintptr_t)15) : nullptr;
  BwdParams p{grad_y, grad_h, h, weight, rstd, weight_dtype == GNN_F32 && dtype != GNN_F32, n, (int)d, g.group, grad_x, partial};
  const size_t smem = g.rows > 1 ? (size_t)d * sizeof(float) : 0;
  int grid = 0;
  dispatch_norm<false>(dtype, vec, g.ept, [&](auto tag, auto v, auto nv) {
    using T = decltype(tag);
    constexpr int V = decltype(v)::value, NV = decltype(nv)::value;
    auto go = [&](auto kernel, int threads) {  // threads: resident on an SM
      const int64_t want = (n + g.rows - 1) / g.rows, most = 148 * std::max(1, std::min(4, threads / g.threads));
      grid = (int)std::min(want, most);
      kernel<<<grid, g.threads, smem, stream>>>(p);
    };
    if constexpr (V * NV == 8)  // 32 elements a thread begin beyond 256 threads
      if (g.threads <= 256) return go(rms_norm_bwd_kernel<T, V, NV, 256>, 256 * kResident<T, V * NV, 256>);
    if (g.threads <= 512) go(rms_norm_bwd_kernel<T, V, NV, 512>, 512 * kResident<T, V * NV, 512>);
    else go(rms_norm_bwd_kernel<T, V, NV, 1024>, 1024);
  });
  if (grad_w) {
    const dim3 block(32, 32);
    const unsigned cols = (unsigned)((d + 31) / 32);
    if (weight_dtype == GNN_F32) weight_grad_kernel<<<cols, block, 0, stream>>>(partial, grid, (int)d, (float*)grad_w);
    else if (weight_dtype == GNN_BF16) weight_grad_kernel<<<cols, block, 0, stream>>>(partial, grid, (int)d, (__nv_bfloat16*)grad_w);
    else weight_grad_kernel<<<cols, block, 0, stream>>>(partial, grid, (int)d, (__half*)grad_w);
  }
  return check_launch("gnn_rms_norm_bwd");
}
