// The linear layer for up to 64 rows of 16-bit or 8-bit elements: out = epilogue(x W^T), bound by the
// bytes of W.
//
// W is the 128-row operand of the tcgen05 MMA and the few rows of x are its N side, so a stage of the
// TMA pipeline is 128 rows of W and only as many rows of x as there are (padded to 16, 32 or 64), and
// two CTAs of an SM keep up to 192 KB of W in flight.  One CTA computes 128 columns of the output for all
// rows; where N / 128 leaves SMs idle, a cluster of CTAs divides the reduction axis and its partial
// sums meet in distributed shared memory, added in a fixed order.  In the accumulator a lane of
// tensor memory is a column of the output: consecutive lanes store consecutive columns, bias and the
// weights' scale are one value per thread.
//
// Measured on a B200 (event time, of which about 6 us are the events): 19 x 4096 -> 8192 e4m3 (33.6
// MB) 16.4 us, 64 rows 20.5 us; 64 x 4096 -> 32768 bf16 (268 MB) 57 us, 4.7 TB/s.  What is left is the
// start of the pipeline, the join and the row-by-row epilogue.
//
// Waits are bounded as in linear_tc.cu.
#include <stdio.h>
#include "linear_epilogue.cuh"
#include "tc_ptx.cuh"

namespace gnn {
namespace {

constexpr int BM = 128;  // rows of W per CTA
constexpr int kATile = BM * kStageK;
constexpr int kThreads = 32 * 6;  // TMA, MMA, four epilogue warps
constexpr int kMaxStages = 6;
constexpr int kHalfSm = 114 * 1024;  // shared memory of a CTA when two share an SM
constexpr int kNumBars = 2 * kMaxStages + 1;
constexpr int kBarBytes = (8 * kNumBars + 16 + 127) / 128 * 128;
constexpr int kMaxCluster = 8;

struct NarrowParams {
  int M, N;          // rows of x, rows of W
  int total_kb;      // stages along the reduction axis
  int kb_per_cta, cluster;
  int k_elems, stages;
  uint32_t idesc;
  LinearEpilogue ep;
  int* status;
};

__device__ __forceinline__ float load_remote(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile(
      "{\n\t.reg .b32 r;\n\t"
      "mapa.shared::cluster.u32 r, %1, %2;\n\t"
      "ld.shared::cluster.f32 %0, [r];\n\t}" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
  return v;
}

template <int BN, bool FP8, class T>
__global__ void __launch_bounds__(kThreads, 2)
linear_narrow_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const NarrowParams p) {
  constexpr int kStageBytes = kATile + BN * kStageK;
  constexpr int kTmemCols = BN < 32 ? 32 : BN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (base - raw_addr);
  const int stages = p.stages;
  const uint32_t bar_off = stages * kStageBytes, bars = base + bar_off;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kMaxStages + s); };
  const uint32_t done_bar = bars + 8u * (2 * kMaxStages);
  const uint32_t tmem_slot = bars + 8u * kNumBars;

  __shared__ volatile int s_failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % p.cluster, n0 = blockIdx.x / p.cluster * BM;
  const int kb0 = rank * p.kb_per_cta, num_kb = max(0, min(p.kb_per_cta, p.total_kb - kb0));

  if (threadIdx.x == 0) {
    s_failed = 0;
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done_bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(base_ptr + bar_off + 8 * kNumBars);

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t phase = 1;  // a fresh barrier lets the wait for parity 1 through
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(empty_bar(s), phase, &s_failed)) { s_failed = 1; break; }
        const uint32_t st = base + s * kStageBytes;
        mbar_expect_tx(full_bar(s), kStageBytes);
        tma_load<false>(st, &map_w, (kb0 + kb) * p.k_elems, n0, full_bar(s));
        tma_load<false>(st + kATile, &map_x, (kb0 + kb) * p.k_elems, 0, full_bar(s));
        if (++s == stages) { s = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = p.idesc | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
      int s = 0;
      uint32_t phase = 0;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(full_bar(s), phase, &s_failed)) { s_failed = 1; ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t st = base + s * kStageBytes;
        const uint64_t da = operand_desc(st, false), db = operand_desc(st + kATile, false);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma<false, FP8>(tmem, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
        umma_commit<false>(empty_bar(s));
        if (++s == stages) { s = 0; phase ^= 1; }
      }
      if (ok) umma_commit<false>(done_bar);
    }
  } else {
    if (!warp_wait(done_bar, 0, &s_failed)) s_failed = 1;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  }
  // all copies have landed and all MMAs have read them: the stages are free for the partial sums
  const int lg = warp & 3, n = n0 + lg * 32 + lane;
  float* const mine = reinterpret_cast<float*>(base_ptr) + lg * 32 + lane;  // [m][128]
  if (warp >= 2 && !s_failed) {
#pragma unroll 1
    for (int c = 0; c < BN && c < p.M; c += 16) {
      uint32_t r[16];
      tmem_load16(tmem + ((uint32_t)(lg * 32) << 16) + (uint32_t)c, r);
      tmem_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) mine[(c + j) * BM] = num_kb ? __uint_as_float(r[j]) : 0.f;  // an empty range adds nothing
    }
  }
  if (p.cluster > 1) cluster_sync();
  if (warp >= 2 && n < p.N) {
    const int share = (p.M + p.cluster - 1) / p.cluster, lo = rank * share, hi = min(lo + share, p.M);
    const uint32_t at = smem_u32(mine);
    const LinearEpilogue& ep = p.ep;
    const float bias = ep.bias ? to_f32(static_cast<const T*>(ep.bias)[n]) : 0.f;
    const float scale = FP8 ? __ldg(ep.col_scale + n) : 1.f;
    // kRows rows at a time: their residuals and all partial sums of up to four CTAs are under way together
    constexpr int kRows = 8;
#pragma unroll 1
    for (int m0 = lo; m0 < hi; m0 += kRows) {
      float v[kRows], res[kRows], rs[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        v[j] = res[j] = 0.f;
        if (m0 + j < hi) {
          if (ep.residual) res[j] = to_f32(static_cast<const T*>(ep.residual)[(int64_t)(m0 + j) * p.N + n]);
          if constexpr (FP8) rs[j] = __ldg(ep.row_scale + m0 + j);
        }
      }
      if (p.cluster == 1) {
#pragma unroll
        for (int j = 0; j < kRows; ++j)
          if (m0 + j < hi) v[j] = mine[(m0 + j) * BM];  // this thread's own
      } else {
#pragma unroll 1
        for (int r0 = 0; r0 < p.cluster; r0 += 4) {
          float part[4][kRows];
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < kRows; ++j)
              part[r][j] = r0 + r < p.cluster && m0 + j < hi ? load_remote(at + (m0 + j) * BM * 4, r0 + r) : 0.f;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < kRows; ++j) v[j] += part[r][j];
        }
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        if constexpr (FP8) v[j] *= rs[j] * scale;
        v[j] += bias;
        if (ep.z && m0 + j < hi) static_cast<T*>(ep.z)[(int64_t)(m0 + j) * p.N + n] = from_f32<T>(v[j]);
      }
      apply_act<sizeof(T) == 4>(v, ep.act, ep.slope);
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        if (m0 + j < hi) static_cast<T*>(ep.out)[(int64_t)(m0 + j) * p.N + n] = from_f32<T>(v[j] + res[j]);
    }
  }
  if (p.cluster > 1) cluster_sync();  // nobody leaves while its sums are being read

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (s_failed) {
    // something expired: give the copies still in flight a bounded time to land
    if (threadIdx.x == 0) {
      *p.status = 1;
      for (int s = 0; s < stages; ++s) {
        mbar_wait(full_bar(s), 0, nullptr, kDrainCycles);
        mbar_wait(full_bar(s), 1, nullptr, kDrainCycles);
      }
    }
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

template <int BN, bool FP8, class T>
int launch_instance(const CUtensorMap& mw, const CUtensorMap& mx, NarrowParams p, cudaStream_t stream) {
  constexpr int kStageBytes = kATile + BN * kStageK;
  auto kernel = linear_narrow_kernel<BN, FP8, T>;
  const int fixed = 1024 + kBarBytes;
  p.stages = (kHalfSm - fixed) / kStageBytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  const int smem = fixed + p.stages * kStageBytes;
  static SmemGrant grant;
  grant.allow(kernel, kHalfSm);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.N + BM - 1) / BM * p.cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, mw, mx, p) == cudaSuccess ? 0 : 1;
}
template <bool FP8, class T>
int launch_shape(int bn, const CUtensorMap& mw, const CUtensorMap& mx, const NarrowParams& p, cudaStream_t stream) {
  switch (bn) {
    case 16: return launch_instance<16, FP8, T>(mw, mx, p, stream);
    case 32: return launch_instance<32, FP8, T>(mw, mx, p, stream);
    default: return launch_instance<64, FP8, T>(mw, mx, p, stream);
  }
}

}  // namespace

int launch_linear_narrow(const TcOperand& a, const TcOperand& b, int in_type, int64_t M, int64_t N, int64_t K,
                         const LinearEpilogue& ep, int* status, cudaStream_t stream, const char* what) {
  const int bn = M <= 16 ? 16 : M <= 32 ? 32 : 64;
  const bool fp8 = in_type == GNN_E4M3;
  CUtensorMap mw, mx;
  if (!encode_operand(&mw, b, in_type, N, K, BM) || !encode_operand(&mx, a, in_type, M, K, bn)) {
    char msg[200];
    snprintf(msg, sizeof msg, "%s: cuTensorMapEncodeTiled failed", what);
    set_last_error(msg);
    return GNN_ERR_CUDA;
  }
  NarrowParams p = {};
  p.M = (int)M;
  p.N = (int)N;
  p.k_elems = fp8 ? kStageK : kStageK / 2;
  p.total_kb = (int)((K + p.k_elems - 1) / p.k_elems);
  // CTAs of a cluster divide the reduction axis until the SMs hold two each, 4 stages at least
  const int64_t tiles = (N + BM - 1) / BM;
  p.cluster = 1;
  while (p.cluster < kMaxCluster &&
         ((tiles * p.cluster * 2 <= 2 * 148 && p.total_kb >= 8 * p.cluster) || p.total_kb > max_chain(in_type) * p.cluster))
    p.cluster *= 2;
  p.kb_per_cta = (p.total_kb + p.cluster - 1) / p.cluster;
  const uint32_t type = in_type == GNN_BF16 ? 1u : 0u;  // see launch_linear_tc
  p.idesc = (1u << 4) | (type << 7) | (type << 10);
  p.ep = ep;
  p.status = status;
  if (fp8) {
    if (ep.out_type == GNN_F32) launch_shape<true, float>(bn, mw, mx, p, stream);
    else if (ep.out_type == GNN_BF16) launch_shape<true, __nv_bfloat16>(bn, mw, mx, p, stream);
    else launch_shape<true, __half>(bn, mw, mx, p, stream);
  } else if (in_type == GNN_BF16) {
    launch_shape<false, __nv_bfloat16>(bn, mw, mx, p, stream);
  } else {
    launch_shape<false, __half>(bn, mw, mx, p, stream);
  }
  return check_launch(what);
}

// From 65 rows on the row-by-row epilogue costs what the wide tile of linear_tc.cu costs (128 x 4096 x
// 4096 bf16: 22 us both) and more for short reductions (128 x 1024 x 8192 e4m3: 31 against 19 us).
// Reductions of more than 8 of the longest chains go there too, to be split further.
bool linear_narrow_wanted(int64_t M, int64_t K, int in_type) {
  const int elt = in_type == GNN_E4M3 ? 1 : 2;
  return in_type != GNN_F32 && M <= 64 && K * elt <= kMaxCluster * max_chain(in_type) * kStageK;
}

}  // namespace gnn
