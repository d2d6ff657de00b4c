// Products of bf16 matrices with fp32 accumulation, for the library's own use.
#pragma once
#include "mtx_common.h"

namespace mtx {

// C = sum over p < pieces of A_p B_p (+ bias[n]) (+ add[m][n]):  A_p (M x K) starts
// pa elements after A_(p-1), B_p (K x N) pb elements after B_(p-1) (0: the same
// matrix).  Each operand is contiguous along k (a_k, b_k) or along its rows m or n,
// ld elements from one row, or k, to the next.  Alignment: bases of 16 bytes, lda,
// ldb, pa and pb multiples of 8, and so K where an operand is contiguous along it.
// What lies between K and a whole 32 is not read; rows are read up to a whole 8.
// C and add are contiguous along n; add may be C itself.
struct GemmBf16 {
  const bf16_t* a;
  int64_t lda, pa;
  bool a_k;
  const bf16_t* b;
  int64_t ldb, pb;
  bool b_k;
  int pieces;
  void* c;  // float, or bf16_t with c_bf16
  int64_t ldc;
  bool c_bf16;
  const float* add;  // or nullptr
  int64_t ldadd;
  const float* bias;  // or nullptr
  int M, N, K;
  int kb;  // where b is contiguous along n: its k from here on read as zeros (0: K)
};
// Operands' and results' rows must lie less than this many elements apart (byte
// offsets within a tile are 32 bits).
constexpr int64_t kGemmBf16MaxLd = 1 << 22, kGemmBf16MaxLdc = 1 << 26;
size_t gemm_bf16_workspace_bytes(int M, int N, int K, int pieces);
int gemm_bf16(const GemmBf16& g, void* workspace, hipStream_t st);

// to (rows x ld) = from (rows x cols, row stride ldf), zeros behind cols
int pack_bf16(const bf16_t* from, int64_t ldf, int64_t rows, int cols, bf16_t* to, int64_t ld, hipStream_t st);

}  // namespace mtx
