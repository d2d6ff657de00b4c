// Dropout on the device from a counter-based generator: keep-masks for the
// fused attention, and dropout of activations without a mask.
//
// The reference draws its dropout masks on the host, `np.random.rand(*shape)
// > p` (layers.py:120).  A fused attention kernel cannot replay NumPy's
// stream, so the attention dropout here consumes an explicit uint8 keep-mask
// (mtx_attn_fwd_dropout / mtx_attn_bwd_dropout), which the caller either
// draws on the host exactly as the reference does or generates with this
// kernel: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC'11), keyed by a 64-bit seed, counter =
// offset + element/4, each 32-bit output w giving the uniform
// u = (w >> 8) * 2^-24 in [0, 1) of one element; the element is kept iff
// u > p, the reference's comparison.
#include "mtx_common.h"

namespace mtx {
namespace {

struct U4 {
  uint32_t x, y, z, w;
};

__device__ __forceinline__ U4 philox4x32_10(U4 c, uint32_t k0, uint32_t k1) {
  constexpr uint32_t kM0 = 0xD2511F53u, kM1 = 0xCD9E8D57u;  // round multipliers
  constexpr uint32_t kW0 = 0x9E3779B9u, kW1 = 0xBB67AE85u;  // key increments (Weyl sequence)
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    if (r > 0) {
      k0 += kW0;
      k1 += kW1;
    }
    const uint64_t p0 = (uint64_t)kM0 * c.x, p1 = (uint64_t)kM1 * c.z;
    c = U4{(uint32_t)(p1 >> 32) ^ c.y ^ k0, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k1, (uint32_t)p0};
  }
  return c;
}

// one Philox call per 4 consecutive elements of the logical rows x cols
// array; element (i, j) is stored at keep[i * ld + j]
__global__ __launch_bounds__(256) void keep_philox_kernel(uint8_t* __restrict__ keep, int64_t rows, int cols,
                                                          int64_t ld, float p, uint32_t k0, uint32_t k1,
                                                          uint64_t offset, uint32_t sub, const uint64_t* base) {
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t n = rows * (int64_t)cols;
  const int64_t e0 = 4 * t;
  if (e0 >= n) return;
  const uint64_t ctr = offset + (base ? *base : 0) + (uint64_t)t;
  const U4 r = philox4x32_10(U4{(uint32_t)ctr, (uint32_t)(ctr >> 32), sub, 0u}, k0, k1);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  int64_t row = e0 / cols;
  int col = (int)(e0 - row * cols);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (e0 + i < n) {
      const float u = (float)(w[i] >> 8) * 0x1p-24f;
      keep[row * ld + col] = u > p ? 1 : 0;
      if (++col == cols) {
        col = 0;
        ++row;
      }
    }
  }
}

// y = residual + (keep ? x * scale : 0): dropout whose mask is drawn where it is
// used, so that neither it nor the uniforms ever lie in memory; the gradient is
// the same call on the upstream gradient.  Element e of the logical rows x cols
// array has the word that keep_philox_kernel would give it.  The product and the
// sum are rounded one after the other, as separate operations would.
struct DropArgs {
  const void *x, *res;  // res: nullptr for none
  void* y;
  int64_t ldx, ldr, ldy, n, cols;  // n: values
  uint32_t below;  // kept: words above it
  bool all;        // p = 0: every value, where the uniform is 0 too
  float scale;
  uint32_t k0, k1, sub;
  uint64_t offset;
  const uint64_t* base;
};

__device__ __forceinline__ U4 draw(const DropArgs& a, uint64_t from, uint64_t call) {
  if (a.all) return U4{~0u, ~0u, ~0u, ~0u};
  const uint64_t ctr = from + call;
  return philox4x32_10(U4{(uint32_t)ctr, (uint32_t)(ctr >> 32), a.sub, 0u}, a.k0, a.k1);
}

template <typename T, bool RES>
__device__ __forceinline__ T drop_one(const DropArgs& a, uint32_t word, T x, T r) {
#pragma clang fp contract(off)
  float v = word > a.below ? Elem<T>::to_f(x) * a.scale : 0.f;
  if constexpr (RES) v = Elem<T>::to_f(r) + v;
  return Elem<T>::from_f(v);
}

// Any strides and addresses: four values a thread, one by one.
template <typename T, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(const DropArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, e0 = 4 * t;
  if (e0 >= a.n) return;
  const U4 r = draw(a, a.offset + (a.base ? *a.base : 0), t);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  int64_t row = e0 / a.cols, col = e0 - row * a.cols;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (e0 + i < a.n) {
      const T x = static_cast<const T*>(a.x)[row * a.ldx + col];
      const T q = RES ? static_cast<const T*>(a.res)[row * a.ldr + col] : T();
      static_cast<T*>(a.y)[row * a.ldy + col] = drop_one<T, RES>(a, w[i], x, q);
      if (++col == a.cols) {
        col = 0;
        ++row;
      }
    }
  }
}

// Rows of whole 16-byte vectors (all values as one row where they lie side by side), a
// vector a thread.  Memory bounds it: 16384 x 384 fp32 with a residual 11.8 us (6.4
// TB/s, one value at a time 25.0), 32768 x 2048 bf16 45 us (5.9 TB/s; 106); the
// generator's 20 wide products for four values run beside it.  Two and four vectors a
// thread took 53 and 58 us.
template <typename T, bool RES, bool FLAT>
__global__ __launch_bounds__(256) void dropout_vec_kernel(const DropArgs a) {
  constexpr int kVec = Elem<T>::kVec;
  struct __attribute__((aligned(16))) Vec {
    T v[kVec];
  };
  const uint64_t from = a.offset + (a.base ? *a.base : 0);
  const int64_t vecs = a.n / kVec, v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (v < vecs) {
    const uint32_t across = FLAT ? 1 : (uint32_t)(a.cols / kVec);
    const int64_t row = FLAT ? 0 : (uint32_t)v / across;
    const int64_t col = FLAT ? v * kVec : (int64_t)((uint32_t)v - (uint32_t)row * across) * kVec;
    const Vec x = *reinterpret_cast<const Vec*>(static_cast<const T*>(a.x) + row * a.ldx + col);
    Vec r{}, y;
    if constexpr (RES) r = *reinterpret_cast<const Vec*>(static_cast<const T*>(a.res) + row * a.ldr + col);
#pragma unroll
    for (int c = 0; c < kVec / 4; ++c) {
      const U4 u = draw(a, from, v * (kVec / 4) + c);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) y.v[4 * c + i] = drop_one<T, RES>(a, w[i], x.v[4 * c + i], r.v[4 * c + i]);
    }
    *reinterpret_cast<Vec*>(static_cast<T*>(a.y) + row * a.ldy + col) = y;
  }
  if constexpr (FLAT) {  // the values behind the last whole vector
    const int64_t e = vecs * kVec + threadIdx.x;
    if (blockIdx.x == 0 && e < a.n) {
      const U4 u = draw(a, from, e / 4);
      const uint32_t w = e % 4 == 0 ? u.x : e % 4 == 1 ? u.y : e % 4 == 2 ? u.z : u.w;
      const T q = RES ? static_cast<const T*>(a.res)[e] : T();
      static_cast<T*>(a.y)[e] = drop_one<T, RES>(a, w, static_cast<const T*>(a.x)[e], q);
    }
  }
}

template <typename T, bool RES>
void dropout(DropArgs a, int64_t rows, hipStream_t st) {
  constexpr int kVec = Elem<T>::kVec;
  const bool flat = rows == 1 || (a.ldx == a.cols && a.ldy == a.cols && (!RES || a.ldr == a.cols));
  const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.y | (RES ? (uintptr_t)a.res : 0);
  const int64_t strides = a.ldx | a.ldy | (RES ? a.ldr : 0) | a.cols;
  const bool vec = at % 16 == 0 && (flat || strides % kVec == 0);
  if (!vec) {
    hipLaunchKernelGGL((dropout_kernel<T, RES>), dim3((unsigned)((a.n + 1023) / 1024)), dim3(256), 0, st, a);
    return;
  }
  const dim3 grid((unsigned)((a.n + 256 * kVec - 1) / (256 * kVec)));
  if (flat) hipLaunchKernelGGL((dropout_vec_kernel<T, RES, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((dropout_vec_kernel<T, RES, false>), grid, dim3(256), 0, st, a);
}

}  // namespace
}  // namespace mtx

using namespace mtx;

extern "C" int mtx_dropout(int dtype, const void* x, int64_t ldx, const void* residual, int64_t ldr, void* y,
                           int64_t ldy, int64_t rows, int64_t cols, float p, float scale, uint64_t seed,
                           uint64_t offset, uint32_t subsequence, const uint64_t* base, void* stream) {
  if (dtype != MTX_F32 && dtype != MTX_BF16) return fail(MTX_ERR_DTYPE, "dropout: unsupported dtype %d", dtype);
  MTX_CHECK_SHAPE(rows >= 0 && cols >= 1, "dropout: rows=%lld, cols=%lld: need rows >= 0, cols >= 1", (long long)rows,
                  (long long)cols);
  MTX_CHECK_ARG(p >= 0.f && p < 1.f, "dropout: p=%g must be in [0, 1)", (double)p);
  MTX_CHECK_ARG(ldx >= cols && ldy >= cols && (!residual || ldr >= cols), "dropout: rows overlap");
  if (rows == 0) return MTX_OK;
  MTX_CHECK_ARG(x && y, "dropout: null pointer");
  MTX_CHECK_ARG((reinterpret_cast<uintptr_t>(base) & 7) == 0, "dropout: base must be 8-byte aligned");
  MTX_CHECK_SHAPE(rows <= ((int64_t)1 << 33) / cols, "dropout: more than 2^33 values");
  // u > p with u = (w >> 8) 2^-24: w >= 256 (floor(2^24 p) + 1)
  const uint32_t below = (uint32_t)((((uint64_t)((double)p * 0x1p24)) + 1) * 256 - 1);
  const DropArgs a{x, residual, y, ldx, ldr, ldy, rows * cols, cols, below, p == 0.f, scale,
                   (uint32_t)seed, (uint32_t)(seed >> 32), subsequence, offset, base};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MTX_F32) residual ? dropout<float, true>(a, rows, st) : dropout<float, false>(a, rows, st);
  else residual ? dropout<bf16_t, true>(a, rows, st) : dropout<bf16_t, false>(a, rows, st);
  MTX_LAUNCHED();
  return MTX_OK;
}

extern "C" int mtx_dropout_keep(uint8_t* keep, int64_t rows, int cols, int64_t ld, float p, uint64_t seed,
                                uint64_t offset, uint32_t subsequence, const uint64_t* base, void* stream) {
  MTX_CHECK_ARG(rows >= 0 && cols >= 1, "rows=%lld, cols=%d: need rows >= 0, cols >= 1", (long long)rows, cols);
  MTX_CHECK_ARG(ld >= cols, "ld=%lld must be >= cols=%d", (long long)ld, cols);
  MTX_CHECK_ARG(p >= 0.f && p < 1.f, "p=%g must be in [0, 1)", (double)p);
  if (rows == 0) return MTX_OK;
  MTX_CHECK_ARG(keep != nullptr, "keep: null pointer");
  MTX_CHECK_ARG((reinterpret_cast<uintptr_t>(base) & 7) == 0, "dropout_keep: base must be 8-byte aligned");
  MTX_CHECK_SHAPE(rows <= (int64_t)0x7fffffff * 1024 / cols, "mask too large");
  const int64_t calls = (rows * (int64_t)cols + 3) / 4;
  const unsigned blocks = (unsigned)((calls + 255) / 256);
  hipLaunchKernelGGL(keep_philox_kernel, dim3(blocks), dim3(256), 0, static_cast<hipStream_t>(stream), keep, rows,
                     cols, ld, p, (uint32_t)seed, (uint32_t)(seed >> 32), offset, subsequence, base);
  MTX_LAUNCHED();
  return MTX_OK;
}

extern "C" int mtx_dropout_keep_philox(uint8_t* keep, int64_t rows, int cols, int64_t ld, float p,
                                       uint64_t seed, uint64_t offset, void* stream) {
  return mtx_dropout_keep(keep, rows, cols, ld, p, seed, offset, 0, nullptr, stream);
}
