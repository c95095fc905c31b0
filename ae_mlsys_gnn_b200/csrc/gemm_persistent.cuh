// Host-side interface of the persistent 3xTF32 tcgen05 GEMM (gemm_persistent.cu), used by
// the C entry points in gemm_tf32x3.cu.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace gnn {

// How one operand of the product reaches the kernel.
enum OperandMode : int {
  // fp32 matrix [rows][K], K contiguous; the kernel splits it into hi/lo in shared memory
  kKMajorRaw = 0,
  // hi and lo given separately, each [rows][K] (prepared by a pre-pass; for small operands)
  kKMajorSplit = 1,
  // hi and lo given separately, K-blocked [ceil(K/32)][rows][32]
  kKMajorSplitBlocked = 2,
  // fp32 matrix [K][rows], rows contiguous (the reduction axis is the slow one); split in the kernel
  kMnMajorRaw = 3,
};

struct GemmOperand {
  OperandMode mode;
  const float* p0;  // raw matrix, or hi
  const float* p1;  // lo (split modes)
  int64_t rows;     // extent along the output dimension (M for A, N for B)
};

// Attention scores formed in the epilogue (splits == 1): C rows are `heads` heads of `head_w` floats.
struct GemmScores {
  const float* attn_l;  // [heads][head_w]
  const float* attn_r;
  float* score_l;       // [M][heads]
  float* score_r;
  int heads, head_w;
};

// Bias, activation and residual in the epilogue (splits == 1): with v the sum at (m, n),
//   v += bias[n];  z[m,n] = v;  v = act(v);  v += residual[m,n]        (null pointers, act 0: nothing)
// bias is [N], z and residual have C's layout.  With splits > 1 every member is null and act 0.
struct GemmFinish {
  const float* bias;
  float* z;
  int act;
  float slope;
  const float* residual;
};

// Shapes for which the epilogue can form the scores: every head inside one 128-column tile and
// starting on a 32-column chunk.
inline bool gemm_scores_ok(int heads, int head_w) {
  return (heads == 1 && head_w <= 128) || head_w == 32 || head_w == 64 || head_w == 128;
}

// C[z][M][N] (z < splits) = sum over the z-th range of K blocks of A * B^T.
// chain_kb: K blocks accumulated in tensor memory before the sum moves to registers (0: the default).
// Returns 0, or a negative GNN_ERR_* after set_last_error.
int launch_gemm_persistent(const GemmOperand& a, const GemmOperand& b, int64_t K, float* C, int64_t ldc,
                           int splits, int64_t split_stride, int* status, cudaStream_t stream,
                           const GemmScores* scores = nullptr, const GemmFinish* finish = nullptr, int chain_kb = 0);

// gnn_gemm_tf32x3 and gnn_gemm_tf32x3_tn (gemm_tf32x3.cu) with a linear layer's epilogue and a
// chain length of choice; `what` names the entry point in error messages.  splits > 1 (without scores):
// the ranges' sums go to `planes` ([splits][M][N], the finish is not applied) instead of C.
int tf32x3_product(const float* A, const float* B, int b_is_n_by_k, float* C, int64_t M, int64_t N, int64_t K,
                   void* workspace, size_t workspace_bytes, int* status, cudaStream_t stream, const GemmScores* scores,
                   const GemmFinish* finish, int chain_kb, const char* what, int splits = 1, float* planes = nullptr);
int tf32x3_product_tn(const float* A, const float* B, float* C, int64_t M, int64_t K1, int64_t N1, void* workspace,
                      size_t workspace_bytes, int* status, cudaStream_t stream, int chain_kb);

// Whether an operand with `cols` contiguous floats per row and base pointer p can be read by TMA.
inline bool tma_rows_ok(const void* p, int64_t cols) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && cols % 4 == 0;
}

}  // namespace gnn
