// Host-side interface of the tcgen05 product with an epilogue (linear_tc.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include "../../include/gnn_b200.h"

namespace gnn {

// One operand of D[m,n] = sum_k A[m,k] * B[n,k].
struct TcOperand {
  const void* p;
  int64_t ld;    // elements from one stored row to the next
  bool mn_major; // false: stored [rows][K]; true: stored [K][rows]
};

// What happens to a finished sum v at (m, n), in this order; null pointers and act 0 do nothing.
struct LinearEpilogue {
  const float* row_scale;  // v *= row_scale[m]
  const float* col_scale;  // v *= col_scale[n]
  const void* bias;        // v += bias[n]
  void* z;                 // z[m,n] = v
  int act;                 // v = act(v)
  float slope;
  const void* residual;    // v += residual[m,n]
  void* out;               // out[m,n] = v
  int out_type;            // GNN_F32 / BF16 / F16: type of bias, z, residual and out
};

// Element type of the operands: GNN_BF16, GNN_F16 or GNN_E4M3.
int launch_linear_tc(const TcOperand& a, const TcOperand& b, int in_type, int64_t M, int64_t N, int64_t K,
                     const LinearEpilogue& ep, void* workspace, size_t workspace_bytes, int* status,
                     cudaStream_t stream, const char* what);
size_t linear_tc_workspace(int64_t M, int64_t N, int64_t K, int in_type);

// Sum of `parts` fp32 planes [M,N] followed by the epilogue.
int launch_split_epilogue(const float* planes, int parts, int64_t M, int64_t N, const LinearEpilogue& ep,
                          cudaStream_t stream);

// The same product for few rows (linear_few.cu), bound by the bytes of B: no workspace, no status.
// fp32 operands too (rows K elements apart, K % 4 == 0).
bool linear_few_wanted(int64_t M, int64_t N, int64_t K, int in_type);
int launch_linear_few(const TcOperand& a, const TcOperand& b, int in_type, int64_t M, int64_t N, int64_t K,
                      const LinearEpilogue& ep, cudaStream_t stream, const char* what);

// The same product for up to 64 rows of 16-bit or 8-bit operands (linear_narrow.cu), both K-major;
// no workspace.
bool linear_narrow_wanted(int64_t M, int64_t K, int in_type);
int launch_linear_narrow(const TcOperand& a, const TcOperand& b, int in_type, int64_t M, int64_t N, int64_t K,
                         const LinearEpilogue& ep, int* status, cudaStream_t stream, const char* what);

// Longest chain of stages (of 128 bytes) that one accumulator takes.  The tensor cores cut off what
// does not fit the running sum: sums of same-sign products come out low by about 2^-23 of their value
// per MMA step, four steps a stage (measured: 1.1e-4 after 1,094 steps of fp16).  The limits keep
// that below half a step of the result: 8e-4 in bf16 (2^-9), 1.1e-4 in fp16 (2^-12).
inline int64_t max_chain(int in_type) { return in_type == GNN_F16 ? 256 : 2048; }

// TMA reads an operand whose rows are a multiple of 16 bytes apart and 16-byte aligned.
inline bool tma_operand_ok(const TcOperand& o, int elt) {
  return (reinterpret_cast<uintptr_t>(o.p) & 15) == 0 && o.ld * elt % 16 == 0;
}

}  // namespace gnn
