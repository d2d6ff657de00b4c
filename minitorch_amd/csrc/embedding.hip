// Embedding lookup with scaling, and its gradient (fp32 and bf16).
//
//   out[i][c] = scale * W[t_i][c]                      (0 where t_i is no token)
//   dW[v][c] (+)= scale * sum over i with t_i = v of g[i][c], in token order
//
// A token outside [0, V) is none: padding.  Its row comes out as zeros and its
// gradient goes nowhere.
#include "mtx_common.h"

namespace mtx {
namespace {

template <typename T, typename O>
__global__ __launch_bounds__(256) void lookup_kernel(const T* __restrict__ w, int64_t ldw, int64_t V,
                                                     const int64_t* __restrict__ ids, int64_t n, int C, float scale,
                                                     O* __restrict__ out, int64_t ldo) {
  const int64_t total = n * C;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
    const int64_t i = e / C;
    const int c = (int)(e - i * C);
    const int64_t t = ids[i];
    const bool some = t >= 0 && t < V;
    out[i * ldo + c] = Elem<O>::from_f(some ? Elem<T>::to_f(w[t * ldw + c]) * scale : 0.f);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void grad_kernel(const int64_t* __restrict__ ids, int64_t n,
                                                   const T* __restrict__ g, int64_t ldg, float scale,
                                                   float* __restrict__ dw, int64_t lddw, int C, int accumulate) {
  const int64_t v = blockIdx.x;
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c >= C) return;
  float acc = 0.f;
  for (int64_t i = 0; i < n; ++i)
    if (ids[i] == v) acc += Elem<T>::to_f(g[i * ldg + c]);
  float* p = dw + v * lddw + c;
  *p = accumulate ? *p + scale * acc : scale * acc;
}

template <typename T, typename O>
int lookup(const void* w, int64_t ldw, int64_t V, const int64_t* ids, int64_t n, int C, float scale, void* out,
           int64_t ldo, hipStream_t st) {
  const int blocks = (int)std::min<int64_t>((n * C + 255) / 256, 16384);
  hipLaunchKernelGGL((lookup_kernel<T, O>), dim3(blocks), dim3(256), 0, st, static_cast<const T*>(w), ldw, V, ids, n, C,
                     scale, static_cast<O*>(out), ldo);
  MTX_LAUNCHED();
  return MTX_OK;
}

bool known(int dtype) { return dtype == MTX_F32 || dtype == MTX_BF16; }

}  // namespace
}  // namespace mtx

using namespace mtx;

extern "C" int mtx_embedding_lookup(int dtype, int out_dtype, const void* weight, int64_t ldw, int64_t V,
                                    const int64_t* ids, int64_t n, int C, float scale, void* out, int64_t ldo,
                                    void* stream) {
  if (!known(dtype) || !known(out_dtype)) return fail(MTX_ERR_DTYPE, "embedding_lookup: unsupported dtype");
  MTX_CHECK_SHAPE(n >= 0 && n < (1LL << 31) && V >= 1 && V < (1LL << 24) && C >= 1,
                  "embedding_lookup: need 0 <= n < 2^31, 1 <= V < 2^24, C >= 1");
  MTX_CHECK_ARG(ldw >= C && ldo >= C, "embedding_lookup: rows of weight or out overlap");
  if (n == 0) return MTX_OK;
  MTX_CHECK_ARG(weight && ids && out, "embedding_lookup: null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MTX_F32)
    return out_dtype == MTX_F32 ? lookup<float, float>(weight, ldw, V, ids, n, C, scale, out, ldo, st)
                                : lookup<float, bf16_t>(weight, ldw, V, ids, n, C, scale, out, ldo, st);
  return out_dtype == MTX_F32 ? lookup<bf16_t, float>(weight, ldw, V, ids, n, C, scale, out, ldo, st)
                              : lookup<bf16_t, bf16_t>(weight, ldw, V, ids, n, C, scale, out, ldo, st);
}

extern "C" size_t mtx_embedding_grad_workspace_bytes(int64_t n, int64_t V, int C) { return 0; }

extern "C" int mtx_embedding_grad(int dtype, const int64_t* ids, int64_t n, const void* grad, int64_t ldg, float scale,
                                  float* dweight, int64_t lddw, int64_t V, int C, int accumulate, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (!known(dtype)) return fail(MTX_ERR_DTYPE, "embedding_grad: unsupported dtype %d", dtype);
  MTX_CHECK_SHAPE(n >= 0 && n < (1LL << 31) && V >= 1 && V < (1LL << 24) && C >= 1,
                  "embedding_grad: need 0 <= n < 2^31, 1 <= V < 2^24, C >= 1");
  MTX_CHECK_ARG(lddw >= C && (n == 0 || ldg >= C), "embedding_grad: rows of grad or dweight overlap");
  MTX_CHECK_ARG(dweight && (n == 0 || (ids && grad)), "embedding_grad: null pointer");
  const dim3 grid((unsigned)V, (C + 255) / 256);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MTX_F32)
    hipLaunchKernelGGL((grad_kernel<float>), grid, dim3(256), 0, st, ids, n, static_cast<const float*>(grad), ldg, scale,
                       dweight, lddw, C, accumulate);
  else
    hipLaunchKernelGGL((grad_kernel<bf16_t>), grid, dim3(256), 0, st, ids, n, static_cast<const bf16_t*>(grad), ldg,
                       scale, dweight, lddw, C, accumulate);
  MTX_LAUNCHED();
  return MTX_OK;
}
