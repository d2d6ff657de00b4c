// A vocabulary projection with its softmax cross entropy and the gradients of
// both, without keeping the logits.
//
//   z = x W + b;  lse_n = log sum_v exp z_nv;  l_n = lse_n - z_n[y_n]
//   loss = 1/M sum_n l_n over the M rows that have a label
//   dz = (softmax(z) - onehot(y)) / M, 0 in the others
//   dx = dz W^T;  dW = x^T dz;  db = sum_n dz_n
//
// The rows are taken in blocks whose logits fit the workspace: a block's
// gradients are worked out while its logits are there, so each logit is computed
// once.
#include "gemm_bf16.h"

namespace mtx {
namespace {

// The number of rows that have a label, as 1 / max(1, number).
__global__ __launch_bounds__(1024) void count_kernel(const int64_t* __restrict__ labels, int64_t n, int V,
                                                     float* __restrict__ inv) {
  __shared__ int part[16];
  int c = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) c += labels[i] >= 0 && labels[i] < V;
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) c += __shfl_xor(c, m, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    int t = 0;
    for (int k = 0; k < 16; ++k) t += part[k];
    *inv = 1.0f / (float)(t > 0 ? t : 1);
  }
}

// loss = inv * sum of the rows' losses, in a fixed order.
__global__ __launch_bounds__(1024) void loss_kernel(const float* __restrict__ row_loss, int64_t n,
                                                    const float* __restrict__ inv, float* __restrict__ loss) {
  __shared__ float part[16];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += row_loss[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
    for (int k = 0; k < 16; ++k) t += part[k];
    *loss = t * *inv;
  }
}

// rows x cols values of `size` bytes = 0
__global__ __launch_bounds__(256) void zero_kernel(void* p, int size, int64_t sr, int64_t sc, int rows, int cols) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)rows * cols; i += (int64_t)gridDim.x * 256) {
    const int64_t at = i / cols * sr + i % cols * sc;
    if (size == 4) static_cast<float*>(p)[at] = 0.f;
    else static_cast<bf16_t*>(p)[at] = 0;
  }
}

// pieces: 0 no gradient, -1 dz in place of z (fp32), 1 or 3 bf16 pieces of dz.
struct RowArgs {
  float* z;
  int64_t ldz;
  const int64_t* labels;
  const float* inv;
  float *row_loss, *lse;
  bf16_t* dz;
  int64_t ldd, piece;
  float* db;  // partial column sums, a row of ldz per workgroup; or nullptr
  int rows, V, pieces;
  bool first;  // the partial sums start here
};

__global__ __launch_bounds__(256) void row_kernel(const RowArgs a) {
  __shared__ float part[8];
  const int tid = threadIdx.x;
  float* db = a.db ? a.db + (int64_t)blockIdx.x * a.ldz : nullptr;
  if (db && a.first)
    for (int v = tid; v < a.V; v += 256) db[v] = 0.f;
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
    float* z = a.z + r * a.ldz;
    float m = -INFINITY;
    for (int v = tid; v < a.V; v += 256) m = fmaxf(m, z[v]);
    m = wave_max(m);
    __syncthreads();
    if ((tid & 63) == 0) part[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    const float from = m == -INFINITY ? 0.f : m;
    float s = 0.f;
    for (int v = tid; v < a.V; v += 256) s += expf(z[v] - from);
    s = wave_sum(s);
    if ((tid & 63) == 0) part[4 + (tid >> 6)] = s;
    __syncthreads();
    s = (part[4] + part[5]) + (part[6] + part[7]);
    const int64_t y = a.labels[r];
    const bool some = y >= 0 && y < a.V;
    if (tid == 0) {
      const float l = m + logf(s);
      a.lse[r] = l;
      const float zy = some ? z[y] : 0.f;
      a.row_loss[r] = !some ? 0.f : zy == -INFINITY && l == -INFINITY ? INFINITY : l - zy;
    }
    if (a.pieces == 0) continue;
    __syncthreads();  // z[y] is read before it is overwritten
    const float inv = *a.inv, rs = s == 0.f ? 0.f : 1.0f / s;
    for (int v = tid; v < a.ldd; v += 256) {
      float d = 0.f;
      if (some && v < a.V) d = (expf(z[v] - from) * rs - (v == y ? 1.f : 0.f)) * inv;
      if (a.pieces < 0) {
        z[v] = d;
      } else {
        bf16_t* q = a.dz + r * a.ldd + v;
        float rest = d;
        for (int p = 0; p < a.pieces; ++p) {
          const bf16_t h = f2bf(rest);
          q[p * a.piece] = h;
          rest -= bf2f(h);
        }
      }
      if (db && v < a.V) db[v] += d;
    }
  }
}

// db = the column sums of the workgroups' partial ones, in their order
__global__ __launch_bounds__(256) void bias_kernel(const float* __restrict__ part, int64_t ld, int n, int V,
                                                   float* __restrict__ db) {
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= V) return;
  float s = 0.f;
  for (int i = 0; i < n; ++i) s += part[i * ld + v];
  db[v] = s;
}

constexpr int kRowWgs = 1024;

struct Plan {
  int64_t ldz;
  int rows, wgs, pieces;
  bool pack_x, pack_w;
  size_t z, dz, db, dw, x, w, gemm, bytes;  // offsets, and the whole
};

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

// Whether rows of `cols` bf16 values at p, ld values apart, are whole 16-byte vectors
// that the products can take as they are.
bool whole(const void* p, int64_t ld, int cols) {
  return cols % 8 == 0 && ld % 8 == 0 && ld < kGemmBf16MaxLd && ((uintptr_t)p & 15) == 0;
}

// The rows whose logits are kept at a time are as many as have logits_bytes of them.
// The query for the workspace's size does not know where the operands lie and counts
// their copies (pack_x, pack_w) in.
Plan plan(int dtype, int grads, int64_t n, int C, int V, bool bias, int64_t logits_bytes, bool pack_x, bool pack_w) {
  Plan p{};
  p.ldz = (V + 7) / 8 * 8;
  const int64_t fit = std::max<int64_t>(logits_bytes / (4 * p.ldz), 1);
  p.rows = (int)std::min(n, fit < 256 ? fit : fit / 256 * 256);
  p.wgs = std::min(p.rows, kRowWgs);
  p.pieces = grads < 0 ? 0 : dtype == MTX_F32 ? -1 : grads == MTX_F32 ? 3 : 1;
  size_t at = 256;  // 1 / labels
  p.z = at;
  at += up((size_t)p.rows * p.ldz * 4);
  p.dz = at;
  if (p.pieces > 0) at += up((size_t)p.pieces * p.rows * p.ldz * 2);
  p.db = at;
  if (p.pieces && bias) at += up((size_t)p.wgs * p.ldz * 4);
  p.dw = at;  // a bf16 gradient of the weights is summed over blocks of rows in fp32
  if (p.pieces == 1 && p.rows < n) at += up((size_t)C * V * 4);
  p.pack_x = dtype == MTX_BF16 && pack_x;
  p.pack_w = dtype == MTX_BF16 && pack_w;
  const int64_t c8 = (C + 7) / 8 * 8, longer = std::max<int64_t>(C * p.ldz, V * c8);
  p.x = at;
  if (p.pack_x) at += up((size_t)p.rows * c8 * 2);
  p.w = at;
  if (p.pack_w) at += up((size_t)longer * 2);
  p.gemm = at;
  size_t most = 0;
  for (int r : {p.rows, (int)(n % p.rows)}) {
    if (!r) continue;
    auto bytes = [&](int M, int N, int K) {
      most = std::max(most, dtype == MTX_F32 ? mtx_gemm_workspace_bytes(M, N, K, 1)
                                             : gemm_bf16_workspace_bytes(M, N, K, N == V && M == r ? 1 : p.pieces));
    };
    bytes(r, V, C);
    if (!p.pieces) continue;
    if (dtype == MTX_F32) {
      bytes(r, C, V);
      bytes(C, V, r);
      bytes(V, C, r);
    } else {
      most = std::max({most, gemm_bf16_workspace_bytes(r, C, (int)p.ldz, p.pieces),
                       gemm_bf16_workspace_bytes(C, V, r, p.pieces), gemm_bf16_workspace_bytes(V, C, r, p.pieces),
                       gemm_bf16_workspace_bytes(r, C, V, p.pieces)});
    }
  }
  p.bytes = at + up(most);
  return p;
}

bool known(int dtype) { return dtype == MTX_F32 || dtype == MTX_BF16; }

}  // namespace
}  // namespace mtx

using namespace mtx;

extern "C" size_t mtx_linear_xent_workspace_bytes(int dtype, int grad_dtype, int64_t n, int C, int V, int bias,
                                                  int64_t logits_bytes) {
  if (n < 0 || C < 1 || V < 1 || n >= (1LL << 31)) return 0;
  return plan(dtype, grad_dtype, std::max<int64_t>(n, 1), C, V, bias != 0, logits_bytes, true, true).bytes;
}

extern "C" int mtx_linear_xent(int dtype, int grad_dtype, int64_t n, int C, int V, const void* x, int64_t ldx,
                               const void* w, int64_t swc, int64_t swv, const float* bias, const int64_t* labels,
                               float* loss, float* row_loss, float* lse, void* dx, int64_t lddx, void* dw, int64_t sdc,
                               int64_t sdv, float* db, int64_t logits_bytes, void* workspace, size_t workspace_bytes,
                               void* stream) {
  if (!known(dtype)) return fail(MTX_ERR_DTYPE, "linear_xent: unsupported dtype %d", dtype);
  const bool grad = dx || dw || db;
  if (grad && (!known(grad_dtype) || (dtype == MTX_F32 && grad_dtype != MTX_F32)))
    return fail(MTX_ERR_DTYPE, "linear_xent: gradients must be fp32, or bf16 like the inputs (got %d)", grad_dtype);
  MTX_CHECK_SHAPE(n >= 0 && n < (1LL << 31) && C >= 1 && C <= (1 << 20) && V >= 1 && V <= (1 << 27),
                  "linear_xent: need 0 <= n < 2^31, 1 <= C <= 2^20, 1 <= V <= 2^27");
  MTX_CHECK_ARG(loss && w && (n == 0 || (x && labels && row_loss && lse)), "linear_xent: null pointer");
  MTX_CHECK_ARG(bias || !db, "linear_xent: db without a bias");
  MTX_CHECK_ARG(n == 0 || ldx >= C, "linear_xent: rows of x overlap");
  MTX_CHECK_ARG((swv == 1 && swc >= V) || (swc == 1 && swv >= C) , "linear_xent: w needs a unit stride and rows that do not overlap");
  MTX_CHECK_ARG(logits_bytes >= 1, "linear_xent: logits_bytes must be positive");
  MTX_CHECK_ARG(!dx || lddx >= C, "linear_xent: rows of dx overlap");
  MTX_CHECK_ARG(!dw || (sdv == 1 && sdc >= V) || (sdc == 1 && sdv >= C),
                "linear_xent: dw needs a unit stride and rows that do not overlap");
  MTX_CHECK_ARG(dtype == MTX_F32 || (V < kGemmBf16MaxLd && (!dx || lddx < kGemmBf16MaxLdc) &&
                                     (!dw || std::max(sdc, sdv) < kGemmBf16MaxLdc)),
                "linear_xent: bf16 needs V below 2^22 and gradients' rows less than 2^26 values apart");
  // W's rows in memory: of V values, or of C
  const bool wv = swv == 1 && swc >= V;
  const int64_t ldw = wv ? swc : swv;
  const Plan p = plan(dtype, grad ? grad_dtype : -1, std::max<int64_t>(n, 1), C, V, db != nullptr, logits_bytes,
                      !whole(x, ldx, C), !whole(w, ldw, wv ? V : C));
  MTX_CHECK_ARG(workspace && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0,
                "linear_xent: workspace of %zu bytes, need %zu aligned to 256", workspace_bytes, p.bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  float* inv = reinterpret_cast<float*>(ws);
  float* z = reinterpret_cast<float*>(ws + p.z);
  bf16_t* dz = reinterpret_cast<bf16_t*>(ws + p.dz);
  float* part = reinterpret_cast<float*>(ws + p.db);
  float* sum = reinterpret_cast<float*>(ws + p.dw);
  bf16_t* xp = reinterpret_cast<bf16_t*>(ws + p.x);
  bf16_t* wp = reinterpret_cast<bf16_t*>(ws + p.w);
  void* gws = ws + p.gemm;
  const size_t gbytes = workspace_bytes - p.gemm;
  const int64_t piece = (int64_t)p.rows * p.ldz;
  const int c8 = (C + 7) / 8 * 8;

  hipLaunchKernelGGL(count_kernel, dim3(1), dim3(1024), 0, st, labels, n, V, inv);
  MTX_LAUNCHED();
  if (n == 0) {
    if (dw) {
      hipLaunchKernelGGL(zero_kernel, dim3((unsigned)std::min<int64_t>(((int64_t)C * V + 255) / 256, 16384)), dim3(256), 0,
                         st, dw, grad_dtype == MTX_F32 ? 4 : 2, sdc, sdv, C, V);
      MTX_LAUNCHED();
    }
  }
  // the weights as the bf16 products take them
  const bf16_t* wb = static_cast<const bf16_t*>(w);
  int64_t ldwb = ldw;
  if (p.pack_w && n) {
    ldwb = wv ? p.ldz : c8;
    if (int rc = pack_bf16(wb, ldw, wv ? C : V, wv ? V : C, wp, ldwb, st)) return rc;
    wb = wp;
  }
  for (int64_t r0 = 0; r0 < n; r0 += p.rows) {
    const int r = (int)std::min<int64_t>(p.rows, n - r0);
    const bool first = r0 == 0, last = r0 + r == n;
    const float* xf = static_cast<const float*>(x) + r0 * ldx;
    const bf16_t* xb = static_cast<const bf16_t*>(x) + r0 * ldx;
    int64_t ldxb = ldx;
    int rc;
    if (p.pack_x) {
      ldxb = c8;
      if ((rc = pack_bf16(xb, ldx, r, C, xp, ldxb, st))) return rc;
      xb = xp;
    }
    if (dtype == MTX_F32) {
      rc = mtx_gemm_f32(r, V, C, 1, 1.f, xf, ldx, 1, 0, static_cast<const float*>(w), swc, swv, 0, 0.f, z, p.ldz, 1, 0,
                        bias, gws, gbytes, stream);
    } else {
      GemmBf16 g{};
      g.a = xb;
      g.lda = ldxb;
      g.a_k = true;
      g.b = wb;
      g.ldb = ldwb;
      g.b_k = !wv;
      g.pieces = 1;
      g.c = z;
      g.ldc = p.ldz;
      g.bias = bias;
      g.M = r;
      g.N = V;
      g.K = c8;  // behind C: zeros in x
      g.kb = wv ? C : 0;
      rc = gemm_bf16(g, gws, st);
    }
    if (rc) return rc;
    const RowArgs a{z, p.ldz, labels + r0, inv, row_loss + r0, lse + r0, dz, p.ldz, piece, db ? part : nullptr, r, V,
                    p.pieces, first};
    hipLaunchKernelGGL(row_kernel, dim3(first ? p.wgs : std::min(r, p.wgs)), dim3(256), 0, st, a);
    MTX_LAUNCHED();
    if (dx) {
      if (dtype == MTX_F32) {
        rc = mtx_gemm_f32(r, C, V, 1, 1.f, z, p.ldz, 1, 0, static_cast<const float*>(w), swv, swc, 0, 0.f,
                          static_cast<float*>(dx) + r0 * lddx, lddx, 1, 0, nullptr, gws, gbytes, stream);
      } else {
        GemmBf16 g{};
        g.a = dz;
        g.lda = p.ldz;
        g.pa = piece;
        g.a_k = true;
        g.b = wb;
        g.ldb = ldwb;
        g.b_k = wv;
        g.pieces = p.pieces;
        g.c = static_cast<char*>(dx) + r0 * lddx * (grad_dtype == MTX_F32 ? 4 : 2);
        g.ldc = lddx;
        g.c_bf16 = grad_dtype == MTX_BF16;
        g.M = r;
        g.N = C;
        g.K = (int)p.ldz;  // behind V: zeros in dz, and zeros or nothing in W
        g.kb = wv ? 0 : V;
        rc = gemm_bf16(g, gws, st);
      }
      if (rc) return rc;
    }
    if (dw) {
      // the product whose result has contiguous rows: dW = x^T dz, or its
      // transpose dz^T x
      const bool rows = sdv == 1;
      const int M = rows ? C : V, N = rows ? V : C;
      const int64_t ld = rows ? sdc : sdv;
      if (dtype == MTX_F32) {
        const float *a = rows ? xf : z, *b = rows ? z : xf;
        const int64_t lda = rows ? ldx : p.ldz, ldb = rows ? p.ldz : ldx;
        rc = mtx_gemm_f32(M, N, r, 1, 1.f, a, 1, lda, 0, b, ldb, 1, 0, first ? 0.f : 1.f, static_cast<float*>(dw), ld, 1,
                          0, nullptr, gws, gbytes, stream);
      } else {
        GemmBf16 g{};
        g.a = rows ? xb : dz;
        g.lda = rows ? ldxb : p.ldz;
        g.pa = rows ? 0 : piece;
        g.b = rows ? dz : xb;
        g.ldb = rows ? p.ldz : ldxb;
        g.pb = rows ? piece : 0;
        g.pieces = p.pieces;
        g.M = M;
        g.N = N;
        g.K = r;
        // blocks of rows are added up in fp32, the sum is rounded once
        const bool narrow = grad_dtype == MTX_BF16;
        g.c_bf16 = narrow && last;
        g.c = narrow && !last ? static_cast<void*>(sum) : dw;
        g.ldc = narrow && !last ? N : ld;
        if (!first) {
          g.add = narrow ? sum : static_cast<const float*>(dw);
          g.ldadd = narrow ? N : ld;
        }
        rc = gemm_bf16(g, gws, st);
      }
      if (rc) return rc;
    }
  }
  if (db) {
    hipLaunchKernelGGL(bias_kernel, dim3(cdiv(V, 256)), dim3(256), 0, st, part, p.ldz, n ? p.wgs : 0, V, db);
    MTX_LAUNCHED();
  }
  hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, st, row_loss, n, inv, loss);
  MTX_LAUNCHED();
  return MTX_OK;
}
