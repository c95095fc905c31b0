// Entry points of the linear layer with bias, activation and residual, and the elementwise half of
// its gradient.
//
//   forward        z = x W^T + b,  y = act(z) + residual
//   elementwise    gz = grad_y * act'(z),  grad_b = sum_rows gz
//   products       grad_x = gz W,  grad_W = gz^T x
//
// 16-bit and 8-bit products run on linear_tc.cu, or for few rows on linear_few.cu and
// linear_narrow.cu; fp32 ones on the error-compensated 3xTF32 kernel with the same epilogue.  The
// tensor cores truncate when they add, so the fp32 kernel moves its sums to registers after every
// kChain32 blocks of 32.  Relative error (2-norm, random operands) and time of 232965 x 604 -> 256 by
// blocks in a chain: 2: 5.6e-7, 554 us; 3: 7.8e-7, 505 us; 4: 1.0e-6, 470 us.
//
// The elementwise pass, measured on a B200: 8192 x 8192 bf16 relu 75 us (5.4 TB/s), gelu 118 us (its
// arithmetic shows); 232965 x 256 fp32 elu 114 us (6.3 TB/s).
#include <stdio.h>
#include <type_traits>
#include "activation.cuh"
#include "common.cuh"
#include "dtypes.cuh"
#include "gemm_persistent.cuh"
#include "linear_tc.cuh"

namespace gnn {
namespace {

constexpr int kChain32 = 3, kChain32Long = 2;  // Long: the weights' gradient, whose reduction is the rows
constexpr int kGroupCols = 8;  // columns a thread owns in the elementwise gradient

int fail(int code, const char* what, const char* why) {
  char msg[256];
  snprintf(msg, sizeof msg, "%s: %s", what, why);
  set_last_error(msg);
  return code;
}

struct ActBwdParams {
  const void* gy;
  const void* z;    // nullptr: no activation
  void* gz;         // nullptr: not wanted
  float* partial;   // [gridDim.y][N] column sums, nullptr: not wanted
  int64_t M, rows_per_cta;
  int N, ldz, groups;  // ldz: elements from one row of gz to the next; groups: threads across columns (2^k <= 256)
  int act;
  float slope;
  int vec_ok;
};

// A CTA walks `rows_per_cta` rows of groups * 8 columns; a thread keeps its columns' sums in
// registers.  HBM-bound: grad_y and z read, gz written once.
template <class T>
__global__ void __launch_bounds__(256, 4) act_bwd_kernel(const ActBwdParams p) {
  __shared__ float s_sum[256][kGroupCols + 1];
  constexpr int V = 16 / (int)sizeof(T);
  const int g = threadIdx.x & (p.groups - 1), strand = threadIdx.x / p.groups, strands = blockDim.x / p.groups;
  const int col = (blockIdx.x * p.groups + g) * kGroupCols;
  float sum[kGroupCols];
#pragma unroll
  for (int j = 0; j < kGroupCols; ++j) sum[j] = 0.f;
  const int64_t lo = blockIdx.y * p.rows_per_cta, hi = min(lo + p.rows_per_cta, p.M);
  const T* const gy = static_cast<const T*>(p.gy);
  const T* const z = static_cast<const T*>(p.z);
  T* const gz = static_cast<T*>(p.gz);
  if (p.vec_ok && col < p.N) {
    // the loads of kRows rows are issued together, without branches between them (the compiler would
    // neither move a load across the stores, which could alias, nor out of a condition it shares with
    // its use); rows behind the last are read again and not counted
    constexpr int kRows = sizeof(T) == 2 ? 2 : 1, Q = kGroupCols / V;  // twice as many spill at 64 registers
    for (int64_t row0 = lo + strand; row0 < hi; row0 += strands * kRows) {
      Pack<T, V> q[kRows][Q], r[kRows][Q];
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const int64_t at = min(row0 + (int64_t)k * strands, hi - 1) * p.N + col;
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          q[k][i] = load_pack(reinterpret_cast<const Pack<T, V>*>(gy + at) + i);
          if (z) r[k][i] = load_pack(reinterpret_cast<const Pack<T, V>*>(z + at) + i);
        }
      }
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const int64_t row = row0 + (int64_t)k * strands;
        if (row < hi) {
          float v[kGroupCols], a[kGroupCols];
#pragma unroll
          for (int j = 0; j < kGroupCols; ++j) {
            v[j] = to_f32(q[k][j / V].v[j % V]);
            if (z) a[j] = to_f32(r[k][j / V].v[j % V]);
          }
          if (z) apply_act_slope<sizeof(T) == 4>(v, a, p.act, p.slope);
#pragma unroll
          for (int j = 0; j < kGroupCols; ++j) sum[j] += v[j];
          if (gz) {
#pragma unroll
            for (int i = 0; i < Q; ++i) {
              Pack<T, V> o;
              o.round_from(v + i * V);
              store_pack(reinterpret_cast<Pack<T, V>*>(gz + row * p.ldz + col) + i, o);
            }
          }
        }
      }
    }
  } else if (!p.vec_ok && col < p.ldz) {
#pragma unroll 1
    for (int64_t row = lo + strand; row < hi; row += strands) {
      const int64_t at = row * p.N + col;
      float v[kGroupCols], a[kGroupCols];
#pragma unroll
      for (int j = 0; j < kGroupCols; ++j) {
        const bool ok = col + j < p.N;
        v[j] = ok ? to_f32(gy[at + j]) : 0.f;
        a[j] = ok && z ? to_f32(z[at + j]) : 0.f;
      }
      if (z) apply_act_slope<sizeof(T) == 4>(v, a, p.act, p.slope);
#pragma unroll
      for (int j = 0; j < kGroupCols; ++j) {
        sum[j] += v[j];
        if (gz && col + j < p.ldz) gz[row * p.ldz + col + j] = from_f32<T>(v[j]);  // the columns behind N are zeros
      }
    }
  }
  if (!p.partial) return;
#pragma unroll
  for (int j = 0; j < kGroupCols; ++j) s_sum[threadIdx.x][j] = sum[j];
  __syncthreads();
  for (int i = threadIdx.x; i < p.groups * kGroupCols; i += blockDim.x) {
    const int c = blockIdx.x * p.groups * kGroupCols + i;
    if (c < p.N) {
      float s = 0.f;
      for (int r = 0; r < strands; ++r) s += s_sum[r * p.groups + i / kGroupCols][i % kGroupCols];
      p.partial[(size_t)blockIdx.y * p.N + c] = s;
    }
  }
}

// out[col] = sum of the CTAs' column sums, in a fixed order.
template <class W>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ partial, int parts, int n, W* out) {
  __shared__ float s[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (col < n)
    for (int r = threadIdx.y; r < parts; r += 32) v += partial[(size_t)r * n + col];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = warp_sum(s[threadIdx.x][threadIdx.y]);
  const int c = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < n) out[c] = from_f32<W>(v);
}

struct ActBwdGrid {
  int groups, col_ctas, row_ctas;
  int64_t rows_per_cta;
};
ActBwdGrid act_bwd_grid(int64_t M, int64_t ldz) {
  ActBwdGrid g;
  const int64_t need = (ldz + kGroupCols - 1) / kGroupCols;
  g.groups = 1;
  while (g.groups < 256 && g.groups < need) g.groups *= 2;  // up to 4 KB of a 16-bit row in one piece
  g.col_ctas = (int)((need + g.groups - 1) / g.groups);
  const int strands = 256 / g.groups;
  int64_t rows = (148 * 4) / g.col_ctas;  // four CTAs an SM at 64 registers a thread: one wave
  const int64_t most = (M + 2 * strands - 1) / (2 * strands);
  if (rows > most) rows = most;
  if (rows < 1) rows = 1;
  g.rows_per_cta = (M + rows - 1) / rows;
  g.row_ctas = (int)((M + g.rows_per_cta - 1) / g.rows_per_cta);
  return g;
}

// Rows of `cols` elements E copied to rows `ld` elements apart (a multiple of 16 bytes), zeros behind
// them.  One 16-byte unit of the copy per thread: its elements are read one by one, which neighbouring
// threads find in L1, and written at once.
template <class E>
__global__ void __launch_bounds__(256) pad_rows_kernel(const E* __restrict__ src, int64_t units, int cols, int units_per_row,
                                                       uint4* __restrict__ dst) {
  constexpr int V = 16 / (int)sizeof(E);
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= units) return;
  const int64_t row = i / units_per_row;
  const int c0 = (int)(i - row * units_per_row) * V;
  const E* const at = src + row * cols + c0;
  union { E e[V]; uint4 q; } o;
#pragma unroll
  for (int j = 0; j < V; ++j) o.e[j] = c0 + j < cols ? at[j] : E(0);
  dst[i] = o.q;
}

// fp32 products with few output tiles: ranges of the reduction axis, at least eight blocks of 32 each, so
// that the SMs are occupied (106 x 6592 -> 47 is a single tile: 147 us without).
int f32_splits(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = ((M + 127) / 128) * ((N + 127) / 128), kb = (K + 31) / 32;
  int64_t s = 148 / tiles;
  if (s > kb / 8) s = kb / 8;
  return s < 2 ? 1 : (int)s;
}
size_t f32_product_bytes(int64_t M, int64_t N, int64_t K) {  // of the weights' halves, then the planes
  size_t bytes = 0;
  gnn_gemm_tf32x3_workspace_bytes(M, N, K, &bytes);
  bytes = (bytes + 255) / 256 * 256;
  const int s = f32_splits(M, N, K);
  return bytes + (s > 1 ? (size_t)s * M * N * sizeof(float) + 256 : 0);
}
int f32_product(const float* a, const float* b, int b_is_n_by_k, float* c, int64_t M, int64_t N, int64_t K,
                const GemmFinish& fin, void* workspace, size_t workspace_bytes, int* status, cudaStream_t stream, const char* what) {
  if (!workspace || workspace_bytes < f32_product_bytes(M, N, K)) return fail(GNN_ERR_WORKSPACE, what, "workspace too small");
  const int splits = f32_splits(M, N, K);
  size_t halves = 0;
  gnn_gemm_tf32x3_workspace_bytes(M, N, K, &halves);
  float* const planes = (float*)(((uintptr_t)workspace + (halves + 255) / 256 * 256 + 255) & ~(uintptr_t)255);
  const int rc = tf32x3_product(a, b, b_is_n_by_k, c, M, N, K, workspace, halves, status, stream, nullptr, &fin, kChain32, what,
                                splits, planes);
  if (rc != GNN_OK || splits == 1) return rc;
  const LinearEpilogue ep{nullptr, nullptr, fin.bias, fin.z, fin.act, fin.slope, fin.residual, c, GNN_F32};
  launch_split_epilogue(planes, splits, M, N, ep, stream);
  return check_launch(what);
}

int check_sizes(const char* what, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 1 || K < 1) return fail(GNN_ERR_INVALID_ARG, what, "bad size");
  if (M >= (1LL << 31) || N >= (1LL << 31) || K >= (1LL << 31)) return fail(GNN_ERR_LIMIT, what, "size exceeds int32");
  return GNN_OK;
}

bool is_float(int t) { return dtype_bytes(t) != 0; }

}  // namespace
}  // namespace gnn

using namespace gnn;

extern "C" int gnn_linear_fwd_workspace_bytes(int64_t M, int64_t N, int64_t K, int in_type, size_t* bytes) {
  if (!bytes || M < 0 || N < 1 || K < 1 || in_type < GNN_F32 || in_type > GNN_E4M3)
    return fail(GNN_ERR_INVALID_ARG, "gnn_linear_fwd_workspace_bytes", "bad argument");
  *bytes = 0;
  if (linear_few_wanted(M, N, K, in_type) || linear_narrow_wanted(M, K, in_type)) return GNN_OK;
  *bytes = in_type == GNN_F32 ? f32_product_bytes(M, N, K) : linear_tc_workspace(M, N, K, in_type);
  return GNN_OK;
}

extern "C" int gnn_linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, int in_type, const float* x_scale,
                              const float* w_scale, const void* bias, int act, float slope, const void* residual, void* y,
                              void* z, int out_type, int64_t M, int64_t N, int64_t K, void* workspace,
                              size_t workspace_bytes, int* status, cudaStream_t stream) {
  const char* const what = "gnn_linear_fwd";
  if (int rc = check_sizes(what, M, N, K)) return rc;
  if (in_type < GNN_F32 || in_type > GNN_E4M3 || !is_float(out_type) || (in_type != GNN_E4M3 && in_type != out_type))
    return fail(GNN_ERR_UNSUPPORTED, what, "operands are fp32, bf16, fp16 (and so is the output) or e4m3");
  if (act < GNN_ACT_NONE || act > GNN_ACT_SILU) return fail(GNN_ERR_INVALID_ARG, what, "unknown activation");
  if ((in_type == GNN_E4M3) != (x_scale != nullptr) || (in_type == GNN_E4M3) != (w_scale != nullptr))
    return fail(GNN_ERR_INVALID_ARG, what, "e4m3 operands, and only they, come with their scales");
  if (M == 0) return GNN_OK;
  if (!x || !w || !y || !status) return fail(GNN_ERR_INVALID_ARG, what, "null pointer");
  if (ldx < K || ldw < K) return fail(GNN_ERR_INVALID_ARG, what, "a row is shorter than K");
  if (in_type == GNN_F32) {
    if (ldx != K || ldw != K) return fail(GNN_ERR_UNSUPPORTED, what, "fp32 rows must be K elements apart");
    if (linear_few_wanted(M, N, K, in_type) && K % 4 == 0 && (((uintptr_t)x | (uintptr_t)w) & 15) == 0) {
      const LinearEpilogue ep{nullptr, nullptr, bias, z, act, slope, residual, y, out_type};
      return launch_linear_few({x, K, false}, {w, K, false}, in_type, M, N, K, ep, stream, what);
    }
    const GemmFinish fin{static_cast<const float*>(bias), static_cast<float*>(z), act, slope,
                         static_cast<const float*>(residual)};
    if (K % 4 || (uintptr_t)x % 16) return fail(GNN_ERR_UNSUPPORTED, what, "fp32 rows must start on 16-byte boundaries");
    return f32_product(static_cast<const float*>(x), static_cast<const float*>(w), 1, static_cast<float*>(y), M, N, K, fin,
                       workspace, workspace_bytes, status, stream, what);
  }
  const TcOperand a{x, ldx, false}, b{w, ldw, false};
  const int elt = in_type == GNN_E4M3 ? 1 : 2;
  if (!tma_operand_ok(a, elt) || !tma_operand_ok(b, elt))
    return fail(GNN_ERR_UNSUPPORTED, what, "rows must start on 16-byte boundaries");
  const LinearEpilogue ep{x_scale, w_scale, bias, z, act, slope, residual, y, out_type};
  if (linear_few_wanted(M, N, K, in_type)) return launch_linear_few(a, b, in_type, M, N, K, ep, stream, what);
  if (linear_narrow_wanted(M, K, in_type)) return launch_linear_narrow(a, b, in_type, M, N, K, ep, status, stream, what);
  return launch_linear_tc(a, b, in_type, M, N, K, ep, workspace, workspace_bytes, status, stream, what);
}

extern "C" int gnn_linear_act_bwd_workspace_bytes(int64_t M, int64_t N, int64_t ldz, size_t* bytes) {
  if (!bytes || M < 0 || N < 1 || ldz < N)
    return fail(GNN_ERR_INVALID_ARG, "gnn_linear_act_bwd_workspace_bytes", "bad argument");
  *bytes = (size_t)(M ? act_bwd_grid(M, ldz).row_ctas : 1) * N * sizeof(float) + 16;
  return GNN_OK;
}

extern "C" int gnn_linear_act_bwd(const void* grad_y, const void* z, int act, float slope, int dtype, int64_t M, int64_t N,
                                  void* gz, int64_t ldz, void* grad_b, void* workspace, size_t workspace_bytes,
                                  cudaStream_t stream) {
  const char* const what = "gnn_linear_act_bwd";
  if (int rc = check_sizes(what, M, N, 1)) return rc;
  if (!is_float(dtype)) return fail(GNN_ERR_UNSUPPORTED, what, "rows are fp32, bf16 or fp16");
  if (act < GNN_ACT_NONE || act > GNN_ACT_SILU) return fail(GNN_ERR_INVALID_ARG, what, "unknown activation");
  if (ldz < N || ldz >= (1LL << 31)) return fail(GNN_ERR_INVALID_ARG, what, "bad row length of gz");
  if (M == 0) {
    if (grad_b) cudaMemsetAsync(grad_b, 0, (size_t)N * dtype_bytes(dtype), stream);
    return check_launch(what);
  }
  if (!grad_y || (act && !z) || (!gz && !grad_b)) return fail(GNN_ERR_INVALID_ARG, what, "null pointer");
  size_t need = 0;
  gnn_linear_act_bwd_workspace_bytes(M, N, ldz, &need);
  if (grad_b && (!workspace || workspace_bytes < need)) return fail(GNN_ERR_WORKSPACE, what, "workspace too small");
  const ActBwdGrid g = act_bwd_grid(M, ldz);
  float* const partial = grad_b ? (float*)(((uintptr_t)workspace + 15) & ~(uintptr_t)15) : nullptr;
  const uintptr_t all = (uintptr_t)grad_y | (act ? (uintptr_t)z : 0) | (uintptr_t)gz;
  ActBwdParams p{grad_y, act ? z : nullptr, gz, partial, M, g.rows_per_cta, (int)N, (int)ldz, g.groups, act, slope,
                 N % 8 == 0 && ldz == N && all % 16 == 0};
  const dim3 grid((unsigned)g.col_ctas, (unsigned)g.row_ctas);
  if (g.row_ctas > 65535) return fail(GNN_ERR_LIMIT, what, "too many rows");
  if (dtype == GNN_F32) act_bwd_kernel<float><<<grid, 256, 0, stream>>>(p);
  else if (dtype == GNN_BF16) act_bwd_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(p);
  else act_bwd_kernel<__half><<<grid, 256, 0, stream>>>(p);
  if (grad_b) {
    const unsigned cols = (unsigned)((N + 31) / 32);
    const dim3 block(32, 32);
    if (dtype == GNN_F32) column_sum_kernel<<<cols, block, 0, stream>>>(partial, g.row_ctas, (int)N, (float*)grad_b);
    else if (dtype == GNN_BF16) column_sum_kernel<<<cols, block, 0, stream>>>(partial, g.row_ctas, (int)N, (__nv_bfloat16*)grad_b);
    else column_sum_kernel<<<cols, block, 0, stream>>>(partial, g.row_ctas, (int)N, (__half*)grad_b);
  }
  return check_launch(what);
}

extern "C" int gnn_linear_dgrad_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, size_t* bytes) {
  if (!bytes || M < 0 || N < 1 || K < 1 || !is_float(dtype))
    return fail(GNN_ERR_INVALID_ARG, "gnn_linear_dgrad_workspace_bytes", "bad argument");
  *bytes = dtype == GNN_F32 ? f32_product_bytes(M, K, N) : linear_tc_workspace(M, K, N, dtype);
  return GNN_OK;
}

extern "C" int gnn_linear_dgrad(const void* gz, int64_t ldg, const void* w, int64_t ldw, int dtype, void* grad_x, int64_t M,
                                int64_t N, int64_t K, void* workspace, size_t workspace_bytes, int* status,
                                cudaStream_t stream) {
  const char* const what = "gnn_linear_dgrad";
  if (int rc = check_sizes(what, M, N, K)) return rc;
  if (!is_float(dtype)) return fail(GNN_ERR_UNSUPPORTED, what, "operands are fp32, bf16 or fp16");
  if (M == 0) return GNN_OK;
  if (!gz || !w || !grad_x || !status) return fail(GNN_ERR_INVALID_ARG, what, "null pointer");
  if (ldg < N || ldw < K) return fail(GNN_ERR_INVALID_ARG, what, "a row is shorter than its columns");
  if (dtype == GNN_F32) {
    if (ldg != N || ldw != K) return fail(GNN_ERR_UNSUPPORTED, what, "fp32 rows must lie one after the other");
    if (N % 4 || (uintptr_t)gz % 16) return fail(GNN_ERR_UNSUPPORTED, what, "fp32 rows must start on 16-byte boundaries");
    return f32_product(static_cast<const float*>(gz), static_cast<const float*>(w), 0, static_cast<float*>(grad_x), M, K, N,
                       GemmFinish{}, workspace, workspace_bytes, status, stream, what);
  }
  const TcOperand a{gz, ldg, false}, b{w, ldw, true};
  if (!tma_operand_ok(a, 2) || !tma_operand_ok(b, 2))
    return fail(GNN_ERR_UNSUPPORTED, what, "rows must start on 16-byte boundaries");
  const LinearEpilogue ep{nullptr, nullptr, nullptr, nullptr, GNN_ACT_NONE, 0.f, nullptr, grad_x, dtype};
  return launch_linear_tc(a, b, dtype, M, K, N, ep, workspace, workspace_bytes, status, stream, what);
}

extern "C" int gnn_linear_wgrad_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, size_t* bytes) {
  if (!bytes || M < 0 || N < 1 || K < 1 || !is_float(dtype))
    return fail(GNN_ERR_INVALID_ARG, "gnn_linear_wgrad_workspace_bytes", "bad argument");
  if (dtype == GNN_F32) return gnn_gemm_tf32x3_tn_workspace_bytes(M, N, K, bytes);
  *bytes = linear_tc_workspace(N, K, M, dtype);
  return GNN_OK;
}

extern "C" int gnn_linear_wgrad(const void* gz, int64_t ldg, const void* x, int64_t ldx, int dtype, void* grad_w, int64_t M,
                                int64_t N, int64_t K, void* workspace, size_t workspace_bytes, int* status,
                                cudaStream_t stream) {
  const char* const what = "gnn_linear_wgrad";
  if (int rc = check_sizes(what, M, N, K)) return rc;
  if (!is_float(dtype)) return fail(GNN_ERR_UNSUPPORTED, what, "operands are fp32, bf16 or fp16");
  if (!grad_w || !status || (M && (!gz || !x))) return fail(GNN_ERR_INVALID_ARG, what, "null pointer");
  if (M == 0) {
    cudaMemsetAsync(grad_w, 0, (size_t)N * K * dtype_bytes(dtype), stream);
    return check_launch(what);
  }
  if (ldg < N || ldx < K) return fail(GNN_ERR_INVALID_ARG, what, "a row is shorter than its columns");
  if (dtype == GNN_F32) {
    if (ldg != N || ldx != K) return fail(GNN_ERR_UNSUPPORTED, what, "fp32 rows must lie one after the other");
    return tf32x3_product_tn(static_cast<const float*>(gz), static_cast<const float*>(x), static_cast<float*>(grad_w), M, N,
                             K, workspace, workspace_bytes, status, stream, kChain32Long);
  }
  const TcOperand a{gz, ldg, true}, b{x, ldx, true};
  if (!tma_operand_ok(a, 2) || !tma_operand_ok(b, 2))
    return fail(GNN_ERR_UNSUPPORTED, what, "rows must start on 16-byte boundaries");
  const LinearEpilogue ep{nullptr, nullptr, nullptr, nullptr, GNN_ACT_NONE, 0.f, nullptr, grad_w, dtype};
  return launch_linear_tc(a, b, dtype, N, K, M, ep, workspace, workspace_bytes, status, stream, what);
}

// The three steps of a gradient in one call: small layers are bound by the host.
extern "C" int gnn_linear_bwd_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, int own_gz, size_t* bytes) {
  if (!bytes || M < 0 || N < 1 || K < 1 || !is_float(dtype))
    return fail(GNN_ERR_INVALID_ARG, "gnn_linear_bwd_workspace_bytes", "bad argument");
  const int64_t per = 16 / dtype_bytes(dtype), ldz = (N + per - 1) / per * per;
  size_t act = 0, dx = 0, dw = 0;
  gnn_linear_act_bwd_workspace_bytes(M, N, ldz, &act);
  gnn_linear_dgrad_workspace_bytes(M, N, K, dtype, &dx);
  gnn_linear_wgrad_workspace_bytes(M, N, K, dtype, &dw);
  const size_t most = act > dx ? (act > dw ? act : dw) : (dx > dw ? dx : dw);
  *bytes = most + 256 + (own_gz ? ((size_t)M * ldz * dtype_bytes(dtype) + 511) / 256 * 256 : 0);
  return GNN_OK;
}

extern "C" int gnn_linear_bwd(const void* grad_y, const void* z, int act, float slope, const void* x, int64_t ldx,
                              const void* w, int64_t ldw, int dtype, int own_gz, void* grad_x, void* grad_w, void* grad_b,
                              int64_t M, int64_t N, int64_t K, void* workspace, size_t workspace_bytes, int* status,
                              cudaStream_t stream) {
  const char* const what = "gnn_linear_bwd";
  if (int rc = check_sizes(what, M, N, K)) return rc;
  if (!is_float(dtype)) return fail(GNN_ERR_UNSUPPORTED, what, "operands are fp32, bf16 or fp16");
  if (act && !own_gz && (grad_x || grad_w)) return fail(GNN_ERR_INVALID_ARG, what, "an activation needs own_gz");
  size_t need = 0;
  gnn_linear_bwd_workspace_bytes(M, N, K, dtype, own_gz, &need);
  if (!workspace || workspace_bytes < need) return fail(GNN_ERR_WORKSPACE, what, "workspace too small");
  const int64_t per = 16 / dtype_bytes(dtype);
  uintptr_t at = ((uintptr_t)workspace + 255) & ~(uintptr_t)255;
  const void* gz = grad_y;
  int64_t ldg = N;
  void* own = nullptr;
  if (own_gz) {
    gz = own = (void*)at;
    ldg = (N + per - 1) / per * per;
    at = (at + (size_t)M * ldg * dtype_bytes(dtype) + 255) & ~(uintptr_t)255;
  }
  // the steps follow each other on the stream, so they share what is left
  void* const rest = (void*)at;
  const size_t left = (uintptr_t)workspace + workspace_bytes - at;
  if (own || grad_b)
    if (int rc = gnn_linear_act_bwd(grad_y, z, act, slope, dtype, M, N, own, ldg, grad_b, rest, left, stream)) return rc;
  if (grad_x)
    if (int rc = gnn_linear_dgrad(gz, ldg, w, ldw, dtype, grad_x, M, N, K, rest, left, status, stream)) return rc;
  if (grad_w)
    if (int rc = gnn_linear_wgrad(gz, ldg, x, ldx, dtype, grad_w, M, N, K, rest, left, status, stream)) return rc;
  return GNN_OK;
}

extern "C" int gnn_pad_rows(const void* src, int element_bytes, int64_t rows, int64_t cols, void* dst, int64_t ld,
                            cudaStream_t stream) {
  const char* const what = "gnn_pad_rows";
  if (int rc = check_sizes(what, rows, cols, 1)) return rc;
  if (element_bytes != 1 && element_bytes != 2 && element_bytes != 4)
    return fail(GNN_ERR_UNSUPPORTED, what, "elements of 1, 2 or 4 bytes");
  if (ld < cols || ld >= (1LL << 31) || ld * element_bytes % 16)
    return fail(GNN_ERR_INVALID_ARG, what, "ld must hold the columns in whole 16-byte units");
  if (rows == 0) return GNN_OK;
  if (!src || !dst || (uintptr_t)dst % 16 || (uintptr_t)src % element_bytes)
    return fail(GNN_ERR_INVALID_ARG, what, "null or misaligned pointer");
  const int64_t per_row = ld * element_bytes / 16, units = rows * per_row, grid = (units + 255) / 256;
  if (grid > INT32_MAX) return fail(GNN_ERR_LIMIT, what, "too many elements");
  if (element_bytes == 4)
    pad_rows_kernel<<<(unsigned)grid, 256, 0, stream>>>((const uint32_t*)src, units, (int)cols, (int)per_row, (uint4*)dst);
  else if (element_bytes == 2)
    pad_rows_kernel<<<(unsigned)grid, 256, 0, stream>>>((const uint16_t*)src, units, (int)cols, (int)per_row, (uint4*)dst);
  else
    pad_rows_kernel<<<(unsigned)grid, 256, 0, stream>>>((const uint8_t*)src, units, (int)cols, (int)per_row, (uint4*)dst);
  return check_launch(what);
}
