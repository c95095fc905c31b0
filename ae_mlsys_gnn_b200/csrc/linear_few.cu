// The linear layer for few rows (a generated token, a small batch), out = epilogue(x W^T).
//
// Bound by the bytes of W, each of which is used for M multiply-adds only: the kernel's whole task is
// to keep enough loads in flight on every SM.  Columns of the output (rows of W) are spread over the
// CTAs 16 at a time and the reduction axis over a CTA's eight warps and over the CTAs of a
// cluster; the partial sums meet in (distributed) shared memory and are added in a fixed order.
//
// 16-bit and 8-bit: warp-level MMAs with 16 rows of W as the 16-row operand and 8 rows of x as the
// 8-column operand.  The order of the reduction axis inside an MMA is free as long as both operands
// agree, so a lane loads 16 consecutive bytes of a row and feeds them to two MMAs as they lie: no
// shared memory, no shuffles between load and MMA.  (tcgen05 would need the operands in shared memory
// and 128 rows of output; its rate is not what bounds this shape.)
// fp32: multiply-adds, lanes along the reduction axis, 4 or 8 rows a CTA (the row groups beyond the
// first find W in L2).
//
// Measured on a B200 (event time, of which about 6 us are the events): 1 x 4096 -> 8192 bf16 (67 MB)
// 18.4 us, e4m3 14.3 us, fp32 30.7 us; 1 x 28672 -> 8192 bf16 (470 MB) 82 us, 5.7 TB/s = 0.88 of the
// copy bandwidth; 1 x 512 -> 512 bf16 at the floor of a launch.
#include <stdio.h>
#include "common.cuh"
#include "linear_epilogue.cuh"

namespace gnn {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxCluster = 8;

struct FewParams {
  const uint8_t* x;  // bytes, so that one kernel serves 8-bit and 16-bit elements
  const uint8_t* w;
  int64_t ldx, ldw;  // bytes from one row to the next
  int M, N;
  int64_t row_bytes; // bytes of a row that count (K elements)
  LinearEpilogue ep;
};

__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// Zeroes the bytes of a 16-byte piece from `left` on.
__device__ __forceinline__ uint4 cut(uint4 v, int64_t left) {
  auto word = [&](uint32_t w, int first) {
    const int64_t n = left - first;
    return n >= 4 ? w : n <= 0 ? 0u : w & (0xffffffffu >> (8 * (4 - (int)n)));
  };
  return make_uint4(word(v.x, 0), word(v.y, 4), word(v.z, 8), word(v.w, 12));
}

template <int KIND>  // GNN_BF16, GNN_F16 or GNN_E4M3
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
#define GNN_MMA(SHAPE_TYPES)                                                                                     \
  asm volatile("mma.sync.aligned." SHAPE_TYPES " {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};" \
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                                                  \
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
  if constexpr (KIND == GNN_BF16) GNN_MMA("m16n8k16.row.col.f32.bf16.bf16.f32");
  else if constexpr (KIND == GNN_F16) GNN_MMA("m16n8k16.row.col.f32.f16.f16.f32");
  else GNN_MMA("m16n8k32.row.col.f32.e4m3.e4m3.f32");
#undef GNN_MMA
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}
__device__ __forceinline__ float load_remote(const float* p, uint32_t rank) {
  float v;
  asm volatile(
      "{\n\t.reg .b32 r;\n\t"
      "mapa.shared::cluster.u32 r, %1, %2;\n\t"
      "ld.shared::cluster.f32 %0, [r];\n\t}" : "=f"(v) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank) : "memory");
  return v;
}

__device__ __forceinline__ void finish_any(const LinearEpilogue& ep, int64_t row, int col, int N, float v) {
  if (ep.out_type == GNN_BF16) finish_one<__nv_bfloat16>(ep, row, col, N, v);
  else if (ep.out_type == GNN_F16) finish_one<__half>(ep, row, col, N, v);
  else finish_one<float>(ep, row, col, N, v);
}

// parts[w][i], w < kWarps: the warps' sums of output i = row * cols + column.  Adds the warps, then
// the cluster's CTAs (each finishes its share of the outputs).
__device__ __forceinline__ void join_and_finish(const LinearEpilogue& ep, float* parts, int outputs, int cols, int M, int N,
                                                int row0, int col0) {
  const int S = gridDim.y, rank = blockIdx.y;  // the cluster spans the y axis of the grid
  __syncthreads();
  if (S == 1) {
    for (int i = threadIdx.x; i < outputs; i += blockDim.x) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += parts[w * outputs + i];
      const int m = row0 + i / cols, n = col0 + i % cols;
      if (m < M && n < N) finish_any(ep, m, n, N, v);
    }
    return;
  }
  for (int i = threadIdx.x; i < outputs; i += blockDim.x) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += parts[w * outputs + i];
    parts[i] = v;  // read by this thread alone so far
  }
  cluster_sync();
  const int share = (outputs + S - 1) / S;
  for (int i = rank * share + threadIdx.x; i < min((rank + 1) * share, outputs); i += blockDim.x) {
    float v = 0.f;
    for (int r = 0; r < S; ++r) v += load_remote(parts + i, r);
    const int m = row0 + i / cols, n = col0 + i % cols;
    if (m < M && n < N) finish_any(ep, m, n, N, v);
  }
  cluster_sync();  // nobody leaves while its sums are being read
}

// 16 columns and 8 rows a CTA; U pieces of 64 bytes of every row are requested at once.
template <int KIND>
__global__ void __launch_bounds__(32 * kWarps, 4) few_mma_kernel(const FewParams p) {
  constexpr int MG = 1, NT = 1, U = 4;  // groups of 8 rows, tiles of 16 columns
  __shared__ float parts[kWarps * MG * 8 * NT * 16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int col0 = blockIdx.x * (16 * NT);
  float acc[NT][MG][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MG; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][m][i] = 0.f;

  const uint8_t* w_row[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) w_row[n][h] = p.w + (int64_t)min(col0 + n * 16 + h * 8 + g, p.N - 1) * p.ldw + t * 16;
  const uint8_t* x_row[MG];
  bool x_in[MG];
#pragma unroll
  for (int m = 0; m < MG; ++m) {
    x_in[m] = m * 8 + g < p.M;
    x_row[m] = p.x + (int64_t)min(m * 8 + g, p.M - 1) * p.ldx + t * 16;
  }

  const int64_t step = (int64_t)gridDim.y * kWarps * (64 * U);
  for (int64_t k = ((int64_t)blockIdx.y * kWarps + warp) * (64 * U); k < p.row_bytes; k += step) {
    uint4 a[U][NT][2], b[U][MG];
    if (k + 64 * U <= p.row_bytes) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) a[u][n][h] = load_stream(w_row[n][h] + k + 64 * u);
#pragma unroll
        for (int m = 0; m < MG; ++m)
          b[u][m] = x_in[m] ? __ldg(reinterpret_cast<const uint4*>(x_row[m] + k + 64 * u)) : make_uint4(0, 0, 0, 0);
      }
    } else {
      // the rows' end: pieces behind it are not read, the one it lies in is cut on both sides
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t left = p.row_bytes - (k + 64 * u + t * 16);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            a[u][n][h] = left > 0 ? cut(load_stream(w_row[n][h] + k + 64 * u), left) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < MG; ++m)
          b[u][m] = left > 0 && x_in[m] ? cut(__ldg(reinterpret_cast<const uint4*>(x_row[m] + k + 64 * u)), left)
                                        : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MG; ++m) {
          mma<KIND>(acc[n][m], a[u][n][0].x, a[u][n][1].x, a[u][n][0].y, a[u][n][1].y, b[u][m].x, b[u][m].y);
          mma<KIND>(acc[n][m], a[u][n][0].z, a[u][n][1].z, a[u][n][0].w, a[u][n][1].w, b[u][m].z, b[u][m].w);
        }
  }
  // lane (g, t) holds columns g, g + 8 of rows 2t, 2t + 1
  constexpr int kCols = NT * 16, kOut = MG * 8 * kCols;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MG; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        parts[warp * kOut + (m * 8 + 2 * t + (i & 1)) * kCols + n * 16 + g + (i >> 1) * 8] = acc[n][m][i];
  join_and_finish(p.ep, parts, kOut, kCols, p.M, p.N, 0, col0);
}

// fp32: COLS columns x ROWS rows a CTA (32 sums a lane), lanes along the reduction axis.
template <int COLS, int ROWS>
__global__ void __launch_bounds__(32 * kWarps) few_fma_kernel(const FewParams p) {
  static_assert(COLS * ROWS == 32, "32 sums a lane");
  const int first = blockIdx.z * ROWS, rows = min(ROWS, p.M - first);
  __shared__ float parts[kWarps * 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col0 = blockIdx.x * COLS;
  float acc[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i] = 0.f;
  const int64_t step = (int64_t)gridDim.y * kWarps * 512;
#pragma unroll 2
  for (int64_t k = ((int64_t)blockIdx.y * kWarps + warp) * 512 + lane * 16; k < p.row_bytes; k += step) {
    float4 w[COLS], x[ROWS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const uint4 v = load_stream(p.w + (int64_t)min(col0 + c, p.N - 1) * p.ldw + k);
      w[c] = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
    }
#pragma unroll
    for (int m = 0; m < ROWS; ++m) x[m] = __ldg(reinterpret_cast<const float4*>(p.x + (int64_t)(first + min(m, rows - 1)) * p.ldx + k));
#pragma unroll
    for (int m = 0; m < ROWS; ++m)
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        float& s = acc[m * COLS + c];
        s = fmaf(w[c].x, x[m].x, s); s = fmaf(w[c].y, x[m].y, s);
        s = fmaf(w[c].z, x[m].z, s); s = fmaf(w[c].w, x[m].w, s);
      }
  }
  warp_multi_sum<32>(acc, lane);  // lane i holds sum i
  parts[warp * 32 + lane] = acc[0];
  join_and_finish(p.ep, parts, 32, COLS, p.M, p.N, first, col0);
}

// CTAs along the reduction axis (a cluster): enough of them that the GPU is full, as long as every
// warp has a block of its own.
int cluster_for(int64_t col_ctas, int64_t blocks) {
  int s = 1;
  while (s < kMaxCluster && col_ctas * s < 148 * 2 && blocks >= (int64_t)kWarps * s * 2) s *= 2;
  return s;
}

template <class Kernel>
bool launch(Kernel kernel, int64_t col_ctas, int cluster, const FewParams& p, cudaStream_t stream, int row_groups = 1) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)col_ctas, (unsigned)cluster, (unsigned)row_groups);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = (unsigned)cluster;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess;
}

template <int KIND>
void launch_kind(const FewParams& p, cudaStream_t stream) {
  const int64_t ctas = (p.N + 15) / 16;
  launch(few_mma_kernel<KIND>, ctas, cluster_for(ctas, (p.row_bytes + 255) / 256), p, stream);
}

}  // namespace

// fp32: the 3xTF32 kernel splits W into a workspace first, three passes over it, which pays from about
// 64 rows on (33 rows, N = 8192, K = 4096: 222 us against 47 us per 8 rows here).
bool linear_few_wanted(int64_t M, int64_t N, int64_t K, int in_type) { return M <= (in_type == GNN_F32 ? 32 : 8); }

int launch_linear_few(const TcOperand& a, const TcOperand& b, int in_type, int64_t M, int64_t N, int64_t K,
                      const LinearEpilogue& ep, cudaStream_t stream, const char* what) {
  const int elt = in_type == GNN_F32 ? 4 : in_type == GNN_E4M3 ? 1 : 2;
  const FewParams p{(const uint8_t*)a.p, (const uint8_t*)b.p, a.ld * elt, b.ld * elt, (int)M, (int)N, K * elt, ep};
  if (in_type == GNN_BF16) launch_kind<GNN_BF16>(p, stream);
  else if (in_type == GNN_F16) launch_kind<GNN_F16>(p, stream);
  else if (in_type == GNN_E4M3) launch_kind<GNN_E4M3>(p, stream);
  else if (M <= 4) {
    const int64_t ctas = (N + 7) / 8;
    launch(few_fma_kernel<8, 4>, ctas, cluster_for(ctas, (p.row_bytes + 511) / 512), p, stream);
  } else {
    const int64_t ctas = (N + 3) / 4;
    const int groups = (int)((M + 7) / 8);
    launch(few_fma_kernel<4, 8>, ctas, cluster_for(ctas * groups, (p.row_bytes + 511) / 512), p, stream, groups);
  }
  return check_launch(what);
}

}  // namespace gnn
