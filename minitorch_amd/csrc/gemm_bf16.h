// Products of bf16 matrices with fp32 accumulation, for the library's own use.
#pragma once
#include "mtx_common.h"

namespace mtx {

// C = sum over p < pieces of A_p B_p (+ bias[n]) (+ add[m][n]):  A_p (M x K) starts
// pa elements after A_(p-1), B_p (K x N) pb elements after B_(p-1) (0: the same
// matrix).  One of sam, sak and one of sbk, sbn must be 1.  add may be C itself.
struct GemmBf16 {
  const bf16_t* a;
  int64_t sam, sak, pa;
  const bf16_t* b;
  int64_t sbk, sbn, pb;
  int pieces;
  void* c;  // float, or bf16_t with c_bf16
  int64_t scm, scn;
  bool c_bf16;
  const float* add;  // or nullptr
  int64_t sdm, sdn;
  const float* bias;  // or nullptr
  int M, N, K;
};
int gemm_bf16(const GemmBf16& g, hipStream_t st);

}  // namespace mtx
