// Log probabilities of given tokens, the entropy of their distributions, the
// most likely alternatives, and the gradient of the first two, for gfx950.
//
// With x = scale * logits and lse = log sum exp x: logprob = x_t - lse,
// entropy = -sum p log p.  With e = exp(x - max), l = sum e it is computed as
// log l + (sum e (max - x)) / l: both terms are >= 0, so nothing cancels where
// the distribution is nearly certain.  The reference has log_softmax
// (functional.py:81-97) and samples from softmax (transformer.py:93-104).
#include "mtx_common.h"

#include <algorithm>
#include <cmath>

namespace mtx {
namespace {

struct LpArgs {
  const void* x;
  int64_t ld;
  const int64_t* tok;
  float* logprob;
  float* lse;
  float* entropy;
  int64_t* ids;
  float* tops;
  int V, top;
  float scale;
};

// order of (value, lowest index first) as unsigned numbers: NaN above
// everything, -0 equal to 0
__device__ __forceinline__ uint64_t rank_key(float v, int i) {
  uint32_t u = __float_as_uint(v + 0.f);
  u = v != v ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~i;
}

template <typename T>
__global__ __launch_bounds__(256) void logprobs_kernel(const LpArgs a) {
  __shared__ float red[4];
  __shared__ uint64_t best[4];
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  const T* __restrict__ x = static_cast<const T*>(a.x) + r * a.ld;
  float m = -INFINITY;
  for (int i = tid; i < a.V; i += 256) m = fmaxf(m, Elem<T>::to_f(x[i]) * a.scale);
  m = wave_max(m);
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float m0 = m == -INFINITY ? 0.f : m;
  float l = 0.f, t = 0.f;
  for (int i = tid; i < a.V; i += 256) {
    const float d = Elem<T>::to_f(x[i]) * a.scale - m0, e = expf(d);
    l += e;
    t -= e == 0.f ? 0.f : e * d;
  }
  l = wave_sum(l);
  __syncthreads();
  if ((tid & 63) == 0) red[tid >> 6] = l;
  __syncthreads();
  l = (red[0] + red[1]) + (red[2] + red[3]);
  t = wave_sum(t);
  __syncthreads();
  if ((tid & 63) == 0) red[tid >> 6] = t;
  __syncthreads();
  t = (red[0] + red[1]) + (red[2] + red[3]);
  const float lse = m0 + logf(l);
  if (tid == 0) {
    const int64_t k = a.tok[r];
    float lp = 0.f;
    if (k >= 0 && k < a.V) lp = l == 0.f ? -INFINITY : Elem<T>::to_f(x[k]) * a.scale - lse;
    a.logprob[r] = lp;
    a.lse[r] = lse;
    a.entropy[r] = l == 0.f ? 0.f : logf(l) + t / l;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t mine = 0;
    for (int i = tid; i < a.V; i += 256) {
      const uint64_t key = rank_key(Elem<T>::to_f(x[i]), i);
      if (key < last || k == 0) mine = key > mine ? key : mine;
    }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) {
      const uint64_t o = __shfl_xor(mine, s, 64);
      mine = o > mine ? o : mine;
    }
    __syncthreads();
    if ((tid & 63) == 0) best[tid >> 6] = mine;
    __syncthreads();
    last = std::max(std::max(best[0], best[1]), std::max(best[2], best[3]));
    if (tid == 0) {
      const int i = (int)~(uint32_t)last;
      a.ids[r * a.top + k] = i;
      a.tops[r * a.top + k] = l == 0.f ? -INFINITY : Elem<T>::to_f(x[i]) * a.scale - lse;
    }
  }
}

struct LpBwdArgs {
  const void* x;
  int64_t ld;
  const int64_t* tok;
  const float* lse;
  const float* entropy;
  const float* g;
  const float* gh;
  float* dx;
  int64_t ldd;
  int V;
  float scale;
  int accumulate;
};

template <typename T>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(const LpBwdArgs a) {
  const int64_t r = blockIdx.x;
  const float lse = a.lse[r];
  const int64_t tok = a.tok[r];
  const float g = a.g != nullptr && tok >= 0 && tok < a.V ? a.g[r] : 0.f;
  const float gh = a.gh != nullptr ? a.gh[r] : 0.f;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < a.V; i += gridDim.y * 256) {
    const float lp = Elem<T>::to_f(static_cast<const T*>(a.x)[r * a.ld + i]) * a.scale - lse;
    const float p = lse == -INFINITY ? 0.f : expf(lp);
    float d = p == 0.f ? 0.f : -p * (g + gh * (lp + a.entropy[r]));
    if (i == tok && lse != -INFINITY) d += g;
    d *= a.scale;
    float* o = a.dx + r * a.ldd + i;
    *o = a.accumulate ? *o + d : d;
  }
}

int check_rows(int dtype, int64_t rows, int V, const void* logits, int64_t ld, const int64_t* tokens, float scale) {
  if (dtype != MTX_F32 && dtype != MTX_BF16) return fail(MTX_ERR_DTYPE, "unsupported dtype %d", dtype);
  MTX_CHECK_SHAPE(rows >= 1 && rows <= (1 << 30) && V >= 1 && V <= (1 << 28),
                  "token_logprobs: needs rows >= 1 and 1 <= V <= 2^28 (got %lld, %d)", (long long)rows, V);
  MTX_CHECK_ARG(logits != nullptr && tokens != nullptr, "logits, tokens: null pointer");
  MTX_CHECK_ARG(((uintptr_t)logits & (dtype == MTX_F32 ? 3u : 1u)) == 0, "logits: pointer must be aligned to its type");
  MTX_CHECK_ARG(ld >= V || (rows == 1 && ld >= 0), "logits: row stride %lld < V=%d", (long long)ld, V);
  MTX_CHECK_ARG(std::isfinite(scale) && scale > 0.f, "scale must be finite and > 0");
  return MTX_OK;
}

constexpr int kMostTop = 64;

}  // namespace
}  // namespace mtx

using namespace mtx;

extern "C" size_t mtx_token_logprobs_workspace_bytes(int64_t rows, int V, int top) { return 0; }

extern "C" int mtx_token_logprobs(int dtype, int64_t rows, int V, const void* logits, int64_t ld,
                                  const int64_t* tokens, float scale, float* logprob, float* lse, float* entropy,
                                  int top, int64_t* top_ids, float* top_logprobs, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_rows(dtype, rows, V, logits, ld, tokens, scale))) return rc;
  MTX_CHECK_ARG(logprob && lse && entropy, "logprob, lse, entropy: null pointer");
  MTX_CHECK_SHAPE(top >= 0 && top <= kMostTop && top <= V, "top=%d alternatives of %d tokens (at most %d)", top, V,
                  kMostTop);
  MTX_CHECK_ARG(top == 0 || (top_ids && top_logprobs), "top_ids, top_logprobs: null pointer");
  LpArgs a{logits, ld, tokens, logprob, lse, entropy, top_ids, top_logprobs, V, top, scale};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MTX_F32) hipLaunchKernelGGL(logprobs_kernel<float>, dim3((unsigned)rows), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(logprobs_kernel<bf16_t>, dim3((unsigned)rows), dim3(256), 0, st, a);
  MTX_LAUNCHED();
  return MTX_OK;
}

extern "C" int mtx_token_logprobs_bwd(int dtype, int64_t rows, int V, const void* logits, int64_t ld,
                                      const int64_t* tokens, const float* lse, const float* entropy,
                                      const float* g_logprob, const float* g_entropy, float scale, float* dlogits,
                                      int64_t ldd, int accumulate, void* stream) {
  int rc;
  if ((rc = check_rows(dtype, rows, V, logits, ld, tokens, scale))) return rc;
  MTX_CHECK_ARG(lse && entropy && dlogits, "lse, entropy, dlogits: null pointer");
  MTX_CHECK_ARG(((uintptr_t)dlogits & 3u) == 0 && (ldd >= V || (rows == 1 && ldd >= 0)),
                "dlogits: row stride %lld < V=%d", (long long)ldd, V);
  LpBwdArgs a{logits, ld, tokens, lse, entropy, g_logprob, g_entropy, dlogits, ldd, V, scale, accumulate};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)rows, std::min(cdiv(V, 1024), 65535));
  if (dtype == MTX_F32) hipLaunchKernelGGL(logprobs_bwd_kernel<float>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(logprobs_bwd_kernel<bf16_t>, grid, dim3(256), 0, st, a);
  MTX_LAUNCHED();
  return MTX_OK;
}
