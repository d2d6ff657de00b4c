// Products of bf16 matrices with fp32 accumulation, for the library's own use.
#pragma once
#include "mtx_common.h"

namespace mtx {

// An operand: element (r, c) of piece p lies at r * row + c / 32 * panel + c % 32 +
// p * piece.  Row by row: row = ld, panel = 32; in panels of 32 columns, each with its
// rows one after another (so that what a tile needs at a time is one run of memory):
// row = 32, panel = 32 * rows.  Alignment: p of 16 bytes, all strides multiples of 8.
struct Bf16Matrix {
  const bf16_t* p;
  int64_t row, panel, piece;
  int64_t size;  // elements of a piece, from its first to its last; a multiple of 8
};
inline Bf16Matrix bf16_rows(const bf16_t* p, int64_t rows, int64_t cols, int64_t ld) {
  return {p, ld, 32, 0, (rows - 1) * ld + (cols + 7) / 8 * 8};
}
inline Bf16Matrix bf16_panels(const bf16_t* p, int64_t rows, int64_t panels, int64_t piece) {
  return {p, 32, 32 * rows, piece, 32 * rows * panels};
}

// C = scale * sum over p < pieces of A_p B_p (+ bias[n]) (+ add[m][n]).  A is stored as
// (M, K) (a_k) or as (K, M), B as (N, K) (b_k) or (K, N).  An operand's columns are read
// up to K where they are k (K a multiple of 8), else up to whole 32; its rows up to
// whole tiles, as far as its size goes; what lies behind reads as zeros.  So where the
// one's columns are k, and K is rounded up over zeros, the other's rows may end earlier.
// C and add are contiguous along n; add (with A as (K, M) only) may be C itself.
struct GemmBf16 {
  Bf16Matrix a;
  bool a_k;
  Bf16Matrix b;
  bool b_k;
  int pieces;
  void* c;  // float, or bf16_t with c_bf16
  int64_t ldc;
  bool c_bf16;
  const float* add;  // or nullptr
  int64_t ldadd;
  const float* bias;   // or nullptr
  const float* scale;  // one value on the device, or nullptr
  int M, N, K;
  // Instead of C (c = nullptr): of each row and each 64 columns the maximum and the sum
  // of exp(C - maximum), stats[column / 64][m], and chosen[m] = C[m][columns[m]], for
  // columns within N.
  float2* stats;
  const int64_t* columns;
  float* chosen;
};
// Strides must be smaller than this (byte offsets within a tile are 32 bits): an
// operand's rows', its panels' and a result's.
constexpr int64_t kGemmBf16MaxLd = 1 << 22, kGemmBf16MaxPanel = (int64_t)1 << 28, kGemmBf16MaxLdc = 1 << 26;
// (0 for products that give statistics)
size_t gemm_bf16_workspace_bytes(int M, int N, int K, int pieces);
int gemm_bf16(const GemmBf16& g, void* workspace, hipStream_t st);

// to = the (rows x cols) matrix `from` in panels, zeros behind cols and in the rows from
// `rows` to rows32, a multiple of 32
int pack_bf16(const bf16_t* from, int64_t ldf, int64_t rows, int cols, bf16_t* to, int64_t rows32, hipStream_t st);

}  // namespace mtx
