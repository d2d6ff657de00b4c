// The projection with its cross entropy for small vocabularies, for the library's own use.
#pragma once
#include "mtx_common.h"

namespace mtx {

constexpr int kNarrowV = 96;  // the largest vocabulary
// the rows of x, W and dx must lie closer (byte offsets within 128 of them are 32 bits)
constexpr int64_t kNarrowLd = 1 << 22;

// One block of rows.  Strides as mtx_linear_xent's; dtypes MTX_F32 or MTX_BF16.
struct NarrowXent {
  int dtype;
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t swc, swv;
  const float* bias;  // or nullptr
  const int64_t* labels;
  const float* inv;  // 1 / labels, on the device
  float *row_loss, *lse;
  int rows, C, V;
  void* dx;  // or nullptr
  int64_t lddx;
  bool dx_bf16;
  float* dz;  // out: (softmax - onehot) / labels, rows of ldz, 0 behind V; or nullptr
  int64_t ldz;  // a multiple of 32, at least V
};
int narrow_xent(const NarrowXent& a, hipStream_t st);

// loss = the mean of the rows' losses over those that have a label, summed in a fixed
// order by one workgroup of 1024 threads.
struct MeanLoss {
  const float* row_loss;
  const int64_t* labels;
  int64_t n;
  int V;
  float* loss;
};
__device__ __forceinline__ void mean_loss(const MeanLoss& a) {
  __shared__ float part[16];
  __shared__ int count[16];
  float s = 0.f;
  int c = 0;
#pragma unroll 16
  for (int64_t i = threadIdx.x; i < a.n; i += 1024) {
    s += a.row_loss[i];
    c += (uint64_t)a.labels[i] < (uint64_t)a.V;
  }
  s = wave_sum(s);
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) c += __shfl_xor(c, m, 64);
  if ((threadIdx.x & 63) == 0) {
    part[threadIdx.x >> 6] = s;
    count[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
    int k = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      t += part[i];
      k += count[i];
    }
    *a.loss = t / (float)(k > 0 ? k : 1);
  }
}

// dw[c][v] = x^T dz and db[v] = the column sums of dz, each where wanted, + what the
// block before left in sum (dw) and db unless it is the first
struct NarrowGrad {
  int dtype;
  const void* x;
  int64_t ldx;
  const float* dz;
  int64_t ldz;
  int rows, C, V;
  void* dw;  // or nullptr
  int64_t sdc, sdv;
  bool dw_bf16;
  const float* sum;  // fp32, at sum_c and sum_v; nullptr: the first block
  int64_t sum_c, sum_v;
  float* db;  // or nullptr
  bool first;
  MeanLoss mean;  // worked out beside the sums, unless mean.loss is nullptr
};
size_t narrow_grad_workspace_bytes(int rows, int C, int V);
int narrow_grad(const NarrowGrad& a, void* workspace, hipStream_t st);

}  // namespace mtx
