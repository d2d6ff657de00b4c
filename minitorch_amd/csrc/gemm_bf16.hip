// Products of bf16 matrices on the matrix cores with fp32 accumulation.
#include "gemm_bf16.h"

namespace mtx {
namespace {

constexpr int BT = 64, BK = 32, LD = BK + 8;

__global__ __launch_bounds__(256) void gemm_bf16_kernel(const GemmBf16 g) {
  __shared__ __attribute__((aligned(16))) bf16_t sa[BT * LD], sb[BT * LD];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int m0 = blockIdx.y * BT, n0 = blockIdx.x * BT;
  f32x4 acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = zero4();
  for (int p = 0; p < g.pieces; ++p) {
    const bf16_t* a = g.a + p * g.pa;
    const bf16_t* b = g.b + p * g.pb;
    for (int k0 = 0; k0 < g.K; k0 += BK) {
      __syncthreads();
      for (int i = tid; i < BT * BK; i += 256) {
        const int r = g.sak == 1 ? i / BK : i % BT, k = g.sak == 1 ? i % BK : i / BT;
        sa[r * LD + k] = m0 + r < g.M && k0 + k < g.K ? a[(int64_t)(m0 + r) * g.sam + (int64_t)(k0 + k) * g.sak] : 0;
        const int q = g.sbk == 1 ? i / BK : i % BT, l = g.sbk == 1 ? i % BK : i / BT;
        sb[q * LD + l] = n0 + q < g.N && k0 + l < g.K ? b[(int64_t)(n0 + q) * g.sbn + (int64_t)(k0 + l) * g.sbk] : 0;
      }
      __syncthreads();
      const bf16x8 fa = *reinterpret_cast<const bf16x8*>(sa + (wid * 16 + lane % 16) * LD + 8 * (lane / 16));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bf16x8 fb = *reinterpret_cast<const bf16x8*>(sb + (j * 16 + lane % 16) * LD + 8 * (lane / 16));
        acc[j] = Mfma<bf16_t>::mma(fa, fb, acc[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + j * 16 + lane % 16;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = m0 + wid * 16 + 4 * (lane / 16) + r;
      if (m >= g.M || n >= g.N) continue;
      float v = acc[j][r] + (g.bias ? g.bias[n] : 0.f);
      if (g.add) v += g.add[(int64_t)m * g.sdm + (int64_t)n * g.sdn];
      const int64_t at = (int64_t)m * g.scm + (int64_t)n * g.scn;
      if (g.c_bf16) static_cast<bf16_t*>(g.c)[at] = f2bf(v);
      else static_cast<float*>(g.c)[at] = v;
    }
  }
}

}  // namespace

int gemm_bf16(const GemmBf16& g, hipStream_t st) {
  if (g.M == 0 || g.N == 0) return MTX_OK;
  hipLaunchKernelGGL(gemm_bf16_kernel, dim3(cdiv(g.N, BT), cdiv(g.M, BT)), dim3(256), 0, st, g);
  MTX_LAUNCHED();
  return MTX_OK;
}

}  // namespace mtx
