// A vocabulary projection with its softmax cross entropy and the gradients of
// both, a block of rows' logits at a time.
//
//   z = x W + b;  lse_n = log sum_v exp z_nv;  l_n = lse_n - z_n[y_n]
//   loss = 1/M sum_n l_n over the M rows that have a label
//   dz = (softmax(z) - onehot(y)) / M, 0 in the others
//   dx = dz W^T;  dW = x^T dz;  db = sum_n dz_n
//
// The rows are taken in blocks whose logits fit the workspace: a block's
// gradients are worked out while its logits are there, so each logit is computed
// once.  Three ways, by sizes and types:
//   many rows and a small vocabulary: the logits stay in registers (narrow_xent.hip);
//   bf16 without gradients: the product's epilogue keeps a row's statistics of 64
//     columns each, and no logit is stored;
//   else: the product z, a pass over its rows that puts dz in z's place (fp32) or
//     beside it as bf16 pieces, the products dx and dW.  fp32 products are those of
//     mtx_gemm_f32, bf16 ones gemm_bf16's.
// (8192, 1024) x (1024, 50021) in bf16 with bf16 gradients, 5.1 ms: z 0.96-1.1, the rows'
// pass 0.87 (3.3 GB, 3.8 TB/s), dx 1.5 and dW 1.6 of two pieces each: bound by the products,
// at 1.0 PFLOP/s.  Of one piece, 3.1 ms: 0.55 (2.5 GB), 0.82 and 0.80.
#include "gemm_bf16.h"
#include "narrow_xent.h"

namespace mtx {
namespace {

// The number of rows that have a label, as 1 / max(1, number).
__global__ __launch_bounds__(1024) void count_kernel(const int64_t* __restrict__ labels, int64_t n, int V,
                                                     float* __restrict__ inv) {
  __shared__ int part[16];
  int c = 0;
#pragma unroll 16
  for (int64_t i = threadIdx.x; i < n; i += 1024) c += (uint64_t)labels[i] < (uint64_t)V;
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) c += __shfl_xor(c, m, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    int t = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += part[k];
    *inv = 1.0f / (float)(t > 0 ? t : 1);
  }
}

__global__ __launch_bounds__(1024) void loss_kernel(const MeanLoss a) { mean_loss(a); }

// rows x cols values of `size` bytes = 0
__global__ __launch_bounds__(256) void zero_kernel(void* p, int size, int64_t sr, int64_t sc, int rows, int cols) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)rows * cols; i += (int64_t)gridDim.x * 256) {
    const int64_t at = i / cols * sr + i % cols * sc;
    if (size == 4) static_cast<float*>(p)[at] = 0.f;
    else static_cast<bf16_t*>(p)[at] = 0;
  }
}

// to = the (rows x cols) matrix `from`, and zeros in the rows behind it
__global__ __launch_bounds__(256) void pad_kernel(const float* __restrict__ from, int64_t ldf, int rows, int cols,
                                                  float* __restrict__ to, int64_t ldt, int all) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, r = e / cols, c = e - r * cols;
  if (r < all) to[r * ldt + c] = r < rows ? from[r * ldf + c] : 0.f;
}

// ---------------------------------------------------------------------------
// The rows' statistics and losses and, in place of the logits or beside them, their
// gradients.
//
// MODE: 0 no gradient; 1 dz = (p - onehot) / labels in place of z, fp32; 2, 3 and 4 p -
// onehot as one, two or three bf16 pieces (of 8 bits each: three hold all 24), in panels
// of 32 columns, the factor 1 / labels left to the products: rounded to bf16, it would be
// off by the same amount in every row.
//
// bf16 gradients take two pieces: what these lack, 2^-18 of a term, is less than the fp32
// sums lose, so that the rounding of the result is all that counts.  One piece costs 2^-9
// more in every term: of 8192 x 1024 and a vocabulary of 50021, 1.86e-3 of the gradients'
// norm in place of 1.66e-3; it is what a caller asks for who wants the time (kOnePiece),
// 3.1 ms in place of 5.1.
// ---------------------------------------------------------------------------
struct RowArgs {
  float* z;
  int64_t ldz;  // a multiple of 32; what lies behind V is anything
  const int64_t* labels;
  const float* inv;
  float *row_loss, *lse;
  bf16_t* dz;
  int64_t rows32, piece;  // rows of a panel, values of a piece
  float* db;  // partial column sums of p - onehot, a row of ldz per workgroup; or nullptr
  int rows, V;
  bool first;  // the partial sums start here
};

// d = p - onehot of row r's columns v0 + 4 sub ..  + 3 (v0 a multiple of 32, the same
// for all lanes), where they lie before ldz
template <int MODE>
__device__ __forceinline__ void put_grad(const RowArgs& a, int64_t r, int v0, int sub, f32x4 d, float inv) {
  if (v0 + 4 * sub >= a.ldz) return;
  if constexpr (MODE == 1) {
    char* p = reinterpret_cast<char*>(a.z + r * a.ldz + v0);
    *reinterpret_cast<f32x4*>(p + 16u * sub) = f32x4{d[0] * inv, d[1] * inv, d[2] * inv, d[3] * inv};
  } else {
    // (32 bits: 2^18 rows of 128 panels)
    char* p = reinterpret_cast<char*>(a.dz + ((int64_t)(v0 >> 5) * a.rows32 + r) * 32);
    const uint32_t at = (uint32_t)(sub >> 3) * ((uint32_t)a.rows32 * 64u) + (sub & 7) * 8u;
    uint2 h, m, l;
    if constexpr (MODE == 2) {
      *reinterpret_cast<uint2*>(p + at) = make_uint2(pk_bf16(d[0], d[1]), pk_bf16(d[2], d[3]));
    } else if constexpr (MODE == 3) {
      split2(d, h, m);
      *reinterpret_cast<uint2*>(p + at) = h;
      *reinterpret_cast<uint2*>(p + 2 * a.piece + at) = m;
    } else {
      split3(d, h, m, l);
      *reinterpret_cast<uint2*>(p + at) = h;
      *reinterpret_cast<uint2*>(p + 2 * a.piece + at) = m;
      *reinterpret_cast<uint2*>(p + 4 * a.piece + at) = l;
    }
  }
}

// The rows' (m, s): maximum and sum of exp(z - m), to the label's loss, as the distance
// from the maximum and log s: their sum lse may be too large to hold log s
__device__ __forceinline__ void put_loss(const RowArgs& a, int64_t r, float m, float s, bool some, float zy) {
  const float l = logf(s);
  a.lse[r] = m + l;
  a.row_loss[r] = !some ? 0.f : zy == -INFINITY && m == -INFINITY ? INFINITY : (m - zy) + l;
}

// T threads a row, NV vectors of four columns each, all in registers: a row is read
// once.  T = 64: a wave a row, four of them a workgroup; else a workgroup a row, whose
// waves exchange their (maximum, sum) once.  Without column sums the next row is
// requested while one is worked on; with them their registers are taken.
template <int T, int NV, int MODE, bool DB>
__global__ __launch_bounds__(T < 256 ? 256 : T) void row_kernel(const RowArgs a) {
  constexpr int kRows = T == 64 ? 4 : 1, kW = T / 64;
  constexpr bool kNext = !DB && NV <= 8;
  __shared__ float part[2][2][kW];
  const int sub = threadIdx.x % T, lane = threadIdx.x & 63, w = threadIdx.x / 64 % kW;
  const int step = gridDim.x * kRows;
  f32x4 db[DB ? NV : 1];
  if constexpr (DB)
#pragma unroll
    for (int i = 0; i < NV; ++i) db[i] = zero4();
  int r = blockIdx.x * kRows + (T == 64 ? threadIdx.x / T : 0);
  if constexpr (T == 64) r = __builtin_amdgcn_readfirstlane(r);
  const float inv = MODE == 1 ? *a.inv : 1.f;
  f32x4 z[NV], next[kNext ? NV : 1];
  auto request = [&](int row, f32x4* to) {
#if defined(__HIP_DEVICE_COMPILE__)
    float* p = a.z + (int64_t)row * a.ldz;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int left = max(0, (int)a.ldz - 4 * T * i) * 4;  // what lies behind reads as zeros
      const auto rs = __builtin_amdgcn_make_buffer_rsrc(p + 4 * T * i, (short)0, left, 0x00020000);
      to[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, 16 * sub, 0, MODE >= 2 ? 2 : 0));
    }
#endif
  };
  if constexpr (kNext)
    if (r < a.rows) request(r, next);
  int par = 0;
  for (; r < a.rows; r += step, par ^= 1) {
    const int64_t y = a.labels[r];
    const bool some = (uint64_t)y < (uint64_t)a.V;
    const float zy = some ? a.z[(int64_t)r * a.ldz + y] : 0.f;
    if constexpr (kNext) {
#pragma unroll
      for (int i = 0; i < NV; ++i) z[i] = next[i];
    } else {
      request(r, z);
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (4 * T * (i + 1) > a.V)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * (sub + T * i) + j >= a.V) z[i][j] = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) m = fmaxf(m, z[i][j]);
    }
    m = wave_max(m);
    if constexpr (kNext)
      if (r + step < a.rows) request(r + step, next);
    // (the difference first: m log2(e) is infinite for a finite m beyond 2.36e38, as where a
    // row's entries all hold the type's lowest value)
    const float from = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        z[i][j] = __builtin_amdgcn_exp2f((z[i][j] - from) * kLog2e);
        s += z[i][j];
      }
    s = wave_sum(s);
    float mine = 1.f;  // what this wave's exponentials lack: exp(its maximum - the row's)
    if constexpr (kW > 1) {
      if (lane == 0) {
        part[par][0][w] = m;
        part[par][1][w] = s;
      }
      __syncthreads();
      float M = -INFINITY, S = 0.f;
#pragma unroll
      for (int k = 0; k < kW; ++k) M = fmaxf(M, part[par][0][k]);
      const float top = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int k = 0; k < kW; ++k) S += part[par][1][k] * __builtin_amdgcn_exp2f((part[par][0][k] - top) * kLog2e);
      mine = __builtin_amdgcn_exp2f((m - top) * kLog2e);
      m = M;
      s = S;
    }
    if (sub == 0) put_loss(a, r, m, s, some, zy);
    if constexpr (MODE != 0) {
      const float f = s == 0.f ? 0.f : mine / s;
      const int own = (int)y - 4 * sub;  // the label's column from this lane's first one
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        f32x4 d = zero4();
        if (some) {
#pragma unroll
          for (int j = 0; j < 4; ++j) d[j] = z[i][j] * f - (own == 4 * T * i + j ? 1.f : 0.f);
          // (behind V the exponentials are 0; if f is NaN, the products are not)
          if (4 * T * (i + 1) > a.V)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (4 * (sub + T * i) + j >= a.V) d[j] = 0.f;
          if constexpr (DB) db[i] += d;
        }
        put_grad<MODE>(a, r, 4 * T * i, sub, d, inv);
      }
    }
  }
  if constexpr (MODE >= 2) {  // the panels' rows behind the last one
    for (int64_t q = a.rows + r % step; q < a.rows32; q += step)
#pragma unroll
      for (int i = 0; i < NV; ++i) put_grad<MODE>(a, q, 4 * T * i, sub, zero4(), inv);
  }
  if constexpr (DB) {
    float* out = a.db + (int64_t)blockIdx.x * a.ldz;
    if constexpr (T == 64) {
      __shared__ f32x4 sums[3][NV * 64];
      const int k = threadIdx.x / 64;
      if (k)
#pragma unroll
        for (int i = 0; i < NV; ++i) sums[k - 1][sub + 64 * i] = db[i];
      __syncthreads();
      if (k) return;
#pragma unroll
      for (int i = 0; i < NV; ++i) db[i] = ((db[i] + sums[0][sub + 64 * i]) + sums[1][sub + 64 * i]) + sums[2][sub + 64 * i];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = 4 * (sub + T * i);
      if (v >= a.ldz) continue;
      f32x4* p = reinterpret_cast<f32x4*>(out + v);
      *p = a.first ? db[i] : *p + db[i];
    }
  }
}

// Rows that no workgroup's registers hold: read twice, by 1024 threads.
template <int MODE, bool DB>
__global__ __launch_bounds__(1024) void long_row_kernel(const RowArgs a) {
  __shared__ float part[2][16];
  const int tid = threadIdx.x;
  const float inv = MODE == 1 ? *a.inv : 1.f;
  float* db = DB ? a.db + (int64_t)blockIdx.x * a.ldz : nullptr;
  if constexpr (DB)
    if (a.first)
      for (int v = tid; v < a.ldz; v += 1024) db[v] = 0.f;
  for (int64_t r = blockIdx.x; r < (MODE >= 2 ? a.rows32 : a.rows); r += gridDim.x) {
    if (r >= a.rows) {
      for (int v0 = 0; v0 < a.ldz; v0 += 4096) put_grad<MODE>(a, r, v0, tid, zero4(), inv);
      continue;
    }
    const float* z = a.z + r * a.ldz;
    const int64_t y = a.labels[r];
    const bool some = (uint64_t)y < (uint64_t)a.V;
    const float zy = some ? z[y] : 0.f;
    float m = -INFINITY, s = 0.f;
    for (int v0 = tid; v0 < a.V; v0 += 8192) {
      float x[8], t = m;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = v0 + 1024 * j < a.V ? z[v0 + 1024 * j] : -INFINITY;
        t = fmaxf(t, x[j]);
      }
      const float from = t == -INFINITY ? 0.f : t;
      s *= __builtin_amdgcn_exp2f((m - from) * kLog2e);
      m = t;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += __builtin_amdgcn_exp2f((x[j] - from) * kLog2e);
    }
    const float wm = wave_max(m);
    s = wave_sum(s * __builtin_amdgcn_exp2f((m - (wm == -INFINITY ? 0.f : wm)) * kLog2e));
    __syncthreads();
    if ((tid & 63) == 0) {
      part[0][tid >> 6] = wm;
      part[1][tid >> 6] = s;
    }
    __syncthreads();
    m = -INFINITY;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) m = fmaxf(m, part[0][k]);
    const float top = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += part[1][k] * __builtin_amdgcn_exp2f((part[0][k] - top) * kLog2e);
    if (tid == 0) put_loss(a, r, m, s, some, zy);
    if constexpr (MODE == 0) continue;
    const float f = s == 0.f ? 0.f : 1.0f / s;
    for (int v0 = 0; v0 < a.ldz; v0 += 4096) {
      const int v = v0 + 4 * tid;
      f32x4 d = zero4();
      if (some && v < a.ldz) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(z + v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (v + j < a.V) d[j] = __builtin_amdgcn_exp2f((x[j] - top) * kLog2e) * f;
          if (v + j == (int)y) d[j] -= 1.f;
        }
        if constexpr (DB) *reinterpret_cast<f32x4*>(db + v) += d;
      }
      put_grad<MODE>(a, r, v0, tid, d, inv);
    }
  }
}

// The losses from the statistics of 64 columns each: 16 rows a workgroup, 64 threads a
// row.  (The logits themselves are never stored: 500 rows of 50021 took 88 us of
// products and 23 of the rows' pass with them.)
__global__ __launch_bounds__(1024) void stats_kernel(const float2* __restrict__ stats, int parts, const RowArgs a,
                                                     const float* __restrict__ chosen) {
  __shared__ float2 all[64][17];
  const int row = threadIdx.x % 16, k0 = threadIdx.x / 16, r = blockIdx.x * 16 + row;
  float m = -INFINITY, s = 0.f;
  auto join = [](float& m, float& s, float2 o) {
    const float top = fmaxf(m, o.x), from = top == -INFINITY ? 0.f : top;
    s = s * __builtin_amdgcn_exp2f((m - from) * kLog2e) + o.y * __builtin_amdgcn_exp2f((o.x - from) * kLog2e);
    m = top;
  };
  if (r < a.rows)
#pragma unroll 4
    for (int k = k0; k < parts; k += 64) join(m, s, stats[(int64_t)k * a.rows + r]);
  all[k0][row] = make_float2(m, s);
  __syncthreads();
  for (int h = 32; h >= 1; h >>= 1) {
    if (k0 < h) {
      join(m, s, all[k0 + h][row]);
      all[k0][row] = make_float2(m, s);
    }
    __syncthreads();
  }
  if (k0 || r >= a.rows) return;
  const bool some = (uint64_t)a.labels[r] < (uint64_t)a.V;
  put_loss(a, r, m, s, some, some ? chosen[r] : 0.f);
}

// db = scale times the column sums of the workgroups' partial ones, in a fixed order:
// 64 columns a workgroup, whose 16 waves take every 16th partial row
__global__ __launch_bounds__(1024) void bias_kernel(const float* __restrict__ part, int64_t ld, int n, int V,
                                                    const float* __restrict__ inv, float* __restrict__ db) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, v = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (v < V)
#pragma unroll 8
    for (int i = w; i < n; i += 16) s += part[i * ld + v];
  sums[w][lane] = s;
  __syncthreads();
  if (w || v >= V) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) s += sums[k][lane];
  db[v] = s * *inv;
}

// grad_dtype: bf16, from the logits' gradient in one piece
constexpr int kOnePiece = MTX_BF16 | MTX_GRAD_ONE_PIECE;

struct Plan {
  int64_t ldz, rows32;
  int rows, wgs, pieces;
  bool pack_x, pack_w, narrow;
  bool pad;  // fp32: x and dx in 128 rows
  size_t z, dz, db, dw, x, w, gemm, bytes;  // offsets, and the whole
};

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

// Whether x is copied into panels (gemm_bf16.h) where the products could take it as it is:
// a copy that is small beside them, for long vocabularies.  In us, as it is and with the
// copy, without gradients and with bf16 ones:
//   rows, C, V          none          bf16
//   8192, 1024, 50021   899   846     5183  5138
//   16384, 2048, 32768  2330  2106    12574 12254
//   2048, 1024, 32768   153   149     917   896
//   8192, 256, 32768    224   220     1566  1565
//   2048, 256, 50021    97    101     634   630
//   8192, 256, 16384    119   119     780   776
//   16384, 1024, 4096   159   159     850   843
//   8192, 1024, 4096    85    86      436   442
// (The copy of W, 62 us of the first, gains nothing.)
bool panels_pay(int64_t n, int C, int V) { return V >= 16384 && (double)n * C * V >= 0x1p36; }

// Whether rows of `cols` bf16 values at p, ld values apart, are whole 16-byte vectors
// that the products can take as they are.
bool whole(const void* p, int64_t ld, int cols) {
  return cols % 8 == 0 && ld % 8 == 0 && ld < kGemmBf16MaxLd && ((uintptr_t)p & 15) == 0;
}

// Whether a block of so many rows is faster in narrow_xent, where every wave goes through
// all of C for its 16 rows; bf16 values take the fp32 matrix cores there, so that wide rows
// are faster the general way however many they are.  Measured in us, the general way and
// narrow_xent; with gradients: bias and all of them, bf16 ones from bf16:
//   rows, C, V        fp32         fp32, none   bf16         bf16, none
//   16384, 384, 65    91    58     42    19     76    57     25    20
//   65536, 384, 65    263   154    114   57     153   152    51    57
//   16384, 1024, 65   184   101    87    34     95    103    34    35
//   4096, 1024, 65    73    82     32    33     62    86     30    34
//   2048, 384, 65     57    41     27    17     48    43     21    17
//   300, 384, 65      34    39     20    16     49    41     21    17
//   600, 256, 64      40    29     22    17     43    30     21    17
//   3000, 512, 80     59    50     29    20     54    52     20    21
//   3000, 768, 80     72    67     39    26     57    70     23    27
//   3000, 768, 64     48    58     22    22     55    60     23    24
//   6000, 512, 64     60    50     29    18     60    52     20    19
//   3000, 256, 96     48    39     20    17     49    41     20    18
//   4096, 384, 96     54    51     25    20     57    53     18    20
//   6000, 512, 96     71    64     32    24     63    67     20    25
//   1500, 1024, 32    49    42     22    18     52    45     26    19
//   3000, 2048, 32    66    76     27    30     62    80     39    32
//   12000, 2048, 32   128   92     56    33     103   96     43    35
//   30000, 2048, 32   294   212    129   57     167   158    52    56
bool narrow_is_faster(int dtype, bool grads, int rows, int C, int V) {
  if (V > kNarrowV) return false;
  const bool half = dtype == MTX_BF16;
  if (V <= 32) return C <= 1024 || (half && !grads ? C <= 2048 && rows <= 16384 : rows >= 4LL * C);
  const bool many = rows >= (grads && C > 512 ? 6LL : 4LL) * C;
  if (!half) return C <= (grads ? 256 : 512) || many;
  return C <= 256 || (V <= 80 && C <= 384 && (grads || rows <= 32768)) ||
         (C <= 512 && rows <= 16384 && (V <= 64 || (V <= 80 && many)));
}

// Row kernels' workgroups: about as many as the chip holds at once (as many partial
// column sums are added up at the end).
int row_wgs(int rows, int V) { return V <= 1024 ? std::min(cdiv(rows, 4), 1024) : std::min(rows, V <= 4096 ? 1024 : V <= 16384 ? 512 : 256); }

// The rows whose logits are kept at a time are as many as have logits_bytes of them.
// The query for the workspace's size does not know where the operands lie and counts
// their copies (pack_x, pack_w) in.
// near: strides that narrow_xent takes.
Plan plan(int dtype, int grads, int64_t n, int C, int V, bool bias, int64_t logits_bytes, bool pack_x, bool pack_w,
          bool near) {
  Plan p{};
  p.ldz = (V + 31) / 32 * 32;
  const int64_t fit = std::min<int64_t>(std::max<int64_t>(logits_bytes / (4 * p.ldz), 1), 1 << 18);
  p.rows = (int)std::min(n, fit < 256 ? fit : fit / 256 * 256);
  p.rows32 = (p.rows + 31) / 32 * 32;
  p.narrow = near && narrow_is_faster(dtype, grads >= 0, p.rows, C, V);
  // Below 128 rows the fp32 products leave the matrix cores; above 64 they pay for 128 on
  // the vector units.  With all gradients 72 rows, C = 1370, V = 37387: 556 us so, 308 as 128
  // rows; 100, 512, 20001: 138 and 107; but 65, 128, 5003: 48 and 78.
  p.pad = dtype == MTX_F32 && n > 64 && n < 128 && p.rows == n && C >= 128 && (int64_t)C * V >= 1 << 23;
  p.pieces = grads < 0 ? 0 : dtype == MTX_F32 ? -1 : grads == MTX_F32 ? 3 : grads == kOnePiece ? 1 : 2;
  // (rows of panels behind the last one are set to 0 by workgroups of their own: 2 rows, C =
  // 384, V = 27453, bf16 with fp32 dx: 99 us by two workgroups, 68 by 32)
  p.wgs = row_wgs(p.pieces > 0 ? (int)p.rows32 : p.rows, V);
  size_t at = 256;  // 1 / labels
  p.z = at;  // without gradients bf16 logits are never stored: their statistics are
  // narrow: dz alone, where the logits would be, and dW's ranges
  if (p.narrow) at += p.pieces ? up((size_t)p.rows * p.ldz * 4) : 0;
  else at += p.pieces == 0 && dtype == MTX_BF16 ? up((size_t)p.rows * (cdiv(V, 64) * 8 + 4)) : up((size_t)(p.pad ? 128 : p.rows) * p.ldz * 4);
  p.dz = at;
  if (p.pieces > 0 && !p.narrow) at += up((size_t)p.pieces * p.rows32 * p.ldz * 2);
  p.db = at;
  if (p.pieces && bias && !p.narrow) at += up((size_t)p.wgs * p.ldz * 4);
  p.dw = at;  // a bf16 gradient of the weights is summed over blocks of rows in fp32
  if ((p.pieces == 1 || p.pieces == 2) && p.rows < n) at += up((size_t)C * V * 4);
  p.pack_x = dtype == MTX_BF16 && !p.narrow && pack_x;
  p.pack_w = dtype == MTX_BF16 && !p.narrow && pack_w;
  const int64_t c32 = (C + 31) / 32 * 32;
  p.x = at;
  if (p.pack_x) at += up((size_t)p.rows32 * c32 * 2);
  if (p.pad) at += up((size_t)2 * 128 * C * 4);  // x, dx
  p.w = at;
  if (p.pack_w) at += up((size_t)c32 * p.ldz * 2);
  p.gemm = at;
  size_t most = 0;
  for (int r : {p.rows, (int)(n % p.rows)}) {
    if (!r) continue;
    if (p.narrow) {
      if (p.pieces) most = std::max(most, narrow_grad_workspace_bytes(r, C, V));
      continue;
    }
    auto bytes = [&](int M, int N, int K) {
      most = std::max(most, dtype == MTX_F32 ? gemm_room_bytes(M, N, K)
                                             : gemm_bf16_workspace_bytes(M, N, K, N == V && M == r ? 1 : p.pieces));
    };
    const int m = p.pad ? 128 : r;
    bytes(m, V, C);
    if (!p.pieces) continue;
    if (dtype == MTX_F32) {
      bytes(m, C, V);
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

template <int MODE, bool DB>
void rows(const RowArgs& a, int wgs, hipStream_t st) {
  auto go = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, dim3(wgs), dim3(threads), 0, st, a); };
  if (a.V <= 256) go(row_kernel<64, 1, MODE, DB>, 256);
  else if (a.V <= 512) go(row_kernel<64, 2, MODE, DB>, 256);
  else if (a.V <= 1024) go(row_kernel<64, 4, MODE, DB>, 256);
  else if (a.V <= 4096) go(row_kernel<256, 4, MODE, DB>, 256);
  else if (a.V <= 8192) go(row_kernel<256, 8, MODE, DB>, 256);
  else if (a.V <= 16384) go(row_kernel<512, 8, MODE, DB>, 512);
  else if (a.V <= 32768) go(row_kernel<1024, 8, MODE, DB>, 1024);
  else if (a.V <= (DB ? 40960 : 65536)) go(row_kernel<1024, DB ? 10 : 16, MODE, DB>, 1024);
  else go(long_row_kernel<MODE, DB>, 1024);
}

bool known(int dtype) { return dtype == MTX_F32 || dtype == MTX_BF16; }

}  // namespace
}  // namespace mtx

using namespace mtx;

extern "C" size_t mtx_linear_xent_workspace_bytes(int dtype, int grad_dtype, int64_t n, int C, int V, int bias,
                                                  int64_t logits_bytes) {
  if (n < 0 || C < 1 || V < 1 || n >= (1LL << 31)) return 0;
  auto bytes = [&](bool near) {
    return plan(dtype, grad_dtype, std::max<int64_t>(n, 1), C, V, bias != 0, logits_bytes, true, true, near).bytes;
  };
  return std::max(bytes(true), bytes(false));
}

extern "C" int mtx_linear_xent(int dtype, int grad_dtype, int64_t n, int C, int V, const void* x, int64_t ldx,
                               const void* w, int64_t swc, int64_t swv, const float* bias, const int64_t* labels,
                               float* loss, float* row_loss, float* lse, void* dx, int64_t lddx, void* dw, int64_t sdc,
                               int64_t sdv, float* db, int64_t logits_bytes, void* workspace, size_t workspace_bytes,
                               void* stream) {
  if (!known(dtype)) return fail(MTX_ERR_DTYPE, "linear_xent: unsupported dtype %d", dtype);
  const bool grad = dx || dw || db;
  if (grad && ((!known(grad_dtype) && grad_dtype != kOnePiece) || (dtype == MTX_F32 && grad_dtype != MTX_F32)))
    return fail(MTX_ERR_DTYPE, "linear_xent: gradients must be fp32, or bf16 like the inputs (got %d)", grad_dtype);
  const bool half = grad && grad_dtype != MTX_F32;  // bf16 gradients
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
  const bool near = std::max({n ? ldx : 0, ldw, dx ? lddx : 0}) < kNarrowLd;
  const Plan p = plan(dtype, grad ? grad_dtype : -1, std::max<int64_t>(n, 1), C, V, db != nullptr, logits_bytes,
                      panels_pay(n, C, V) || !whole(x, ldx, C), !whole(w, ldw, wv ? V : C), near);
  MTX_CHECK_ARG(workspace && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0,
                "linear_xent: workspace of %zu bytes, need %zu aligned to 256", workspace_bytes, p.bytes);
  {
    const void* in[] = {x, w, bias};
    const void* out[] = {dx, dw, db, loss, row_loss, lse};
    for (const void* o : out)
      for (const void* i : in) MTX_CHECK_ARG(!o || n == 0 || o != i, "linear_xent: an output is an input");
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  float* inv = reinterpret_cast<float*>(ws);
  float* z = reinterpret_cast<float*>(ws + p.z);
  bf16_t* dz = reinterpret_cast<bf16_t*>(ws + p.dz);
  // fp32: the bias' gradient comes with the weights', where their rows are contiguous
  const bool sums = dtype == MTX_F32 && db && dw && sdv == 1;
  float* part = db && !sums && !p.narrow ? reinterpret_cast<float*>(ws + p.db) : nullptr;
  float* sum = reinterpret_cast<float*>(ws + p.dw);
  bf16_t* xp = reinterpret_cast<bf16_t*>(ws + p.x);
  bf16_t* wp = reinterpret_cast<bf16_t*>(ws + p.w);
  float* padded = reinterpret_cast<float*>(ws + p.x);
  void* gws = ws + p.gemm;
  const size_t gbytes = workspace_bytes - p.gemm;
  const int64_t piece = p.rows32 * p.ldz;
  const int c8 = (C + 7) / 8 * 8, v8 = (V + 7) / 8 * 8, c32 = (C + 31) / 32 * 32;

  if (grad) {
    hipLaunchKernelGGL(count_kernel, dim3(1), dim3(1024), 0, st, labels, n, V, inv);
    MTX_LAUNCHED();
  }
  if (n == 0) {
    if (dw) {
      hipLaunchKernelGGL(zero_kernel, dim3((unsigned)std::min<int64_t>(((int64_t)C * V + 255) / 256, 16384)), dim3(256), 0,
                         st, dw, half ? 2 : 4, sdc, sdv, C, V);
      MTX_LAUNCHED();
    }
  }
  // the weights as the bf16 products take them
  Bf16Matrix wm = bf16_rows(static_cast<const bf16_t*>(w), wv ? C : V, wv ? V : C, ldw);
  if (p.pack_w && n) {
    const int64_t rows32 = wv ? c32 : p.ldz;
    if (int rc = pack_bf16(wm.p, ldw, wv ? C : V, wv ? V : C, wp, rows32, st)) return rc;
    wm = bf16_panels(wp, rows32, (wv ? p.ldz : c32) / 32, 0);
  }
  for (int64_t r0 = 0; r0 < n; r0 += p.rows) {
    const int r = (int)std::min<int64_t>(p.rows, n - r0);
    const bool first = r0 == 0, last = r0 + r == n;
    const float* xf = static_cast<const float*>(x) + r0 * ldx;
    const bf16_t* xb = static_cast<const bf16_t*>(x) + r0 * ldx;
    const int64_t r32 = (r + 31) / 32 * 32;
    int rc;
    Bf16Matrix xm = bf16_rows(xb, r, C, ldx);
    if (p.pack_x) {
      if ((rc = pack_bf16(xb, ldx, r, C, xp, r32, st))) return rc;
      xm = bf16_panels(xp, r32, c32 / 32, 0);
    }
    const Bf16Matrix dm = bf16_panels(dz, r32, p.ldz / 32, piece);
    if (p.narrow) {
      const void* xr = dtype == MTX_F32 ? static_cast<const void*>(xf) : xb;
      if ((rc = narrow_xent({dtype, xr, ldx, w, swc, swv, bias, labels + r0, inv, row_loss + r0, lse + r0, r, C, V,
                             dx ? static_cast<char*>(dx) + r0 * lddx * (half ? 2 : 4) : nullptr, lddx, half,
                             dw || db ? z : nullptr, p.ldz}, st)))
        return rc;
      if (!dw && !db) continue;
      // blocks of rows are added up in fp32, the sum is rounded once
      const bool apart = half && p.rows < n;
      NarrowGrad g{dtype, xr, ldx, z, p.ldz, r, C, V, dw, sdc, sdv, half, static_cast<const float*>(dw), sdc, sdv, db, first,
                   {row_loss, labels, n, V, last ? loss : nullptr}};
      if (apart) {
        g.sum = sum;
        g.sum_c = V;
        g.sum_v = 1;
        if (!last) {
          g.dw = dw ? sum : nullptr;
          g.sdc = V;
          g.sdv = 1;
          g.dw_bf16 = false;
        }
      }
      if ((rc = narrow_grad(g, gws, st))) return rc;
      continue;
    }
    if (dtype == MTX_F32) {
      if (p.pad) {
        hipLaunchKernelGGL(pad_kernel, dim3(cdiv(128 * C, 256)), dim3(256), 0, st, xf, ldx, r, C, padded, C, 128);
        MTX_LAUNCHED();
      }
      rc = mtx_gemm_f32(p.pad ? 128 : r, V, C, 1, 1.f, p.pad ? padded : xf, p.pad ? C : ldx, 1, 0,
                        static_cast<const float*>(w), swc, swv, 0, 0.f, z, p.ldz, 1, 0, bias, gws, gbytes, stream);
    } else {
      GemmBf16 g{};
      g.a = xm;
      g.a_k = true;
      g.b = wm;
      g.b_k = !wv;
      g.pieces = 1;
      g.c = z;
      g.ldc = p.ldz;
      g.bias = bias;
      g.M = r;
      g.N = V;
      g.K = c8;  // behind C: zeros in x
      if (!grad) {
        g.c = nullptr;
        g.stats = reinterpret_cast<float2*>(z);
        g.columns = labels + r0;
        g.chosen = z + (int64_t)r * cdiv(V, 64) * 2;
      }
      rc = gemm_bf16(g, gws, st);
    }
    if (rc) return rc;
    const RowArgs a{z, p.ldz, labels + r0, inv, row_loss + r0, lse + r0, dz, r32, piece, part, r, V, first};
    if (!grad && dtype == MTX_BF16) {
      hipLaunchKernelGGL(stats_kernel, dim3(cdiv(r, 16)), dim3(1024), 0, st, reinterpret_cast<const float2*>(z),
                         cdiv(V, 64), a, z + (int64_t)r * cdiv(V, 64) * 2);
      MTX_LAUNCHED();
      continue;
    }
    const int wgs = first ? p.wgs : std::min(p.wgs, row_wgs(p.pieces > 0 ? (int)r32 : r, V));
    if (p.pieces == 0) rows<0, false>(a, wgs, st);
    else if (p.pieces < 0) part ? rows<1, true>(a, wgs, st) : rows<1, false>(a, wgs, st);
    else if (p.pieces == 1) part ? rows<2, true>(a, wgs, st) : rows<2, false>(a, wgs, st);
    else if (p.pieces == 2) part ? rows<3, true>(a, wgs, st) : rows<3, false>(a, wgs, st);
    else part ? rows<4, true>(a, wgs, st) : rows<4, false>(a, wgs, st);
    MTX_LAUNCHED();
    if (dx) {
      if (dtype == MTX_F32) {
        float* to = p.pad ? padded + 128 * (int64_t)C : static_cast<float*>(dx) + r0 * lddx;
        rc = mtx_gemm_f32(p.pad ? 128 : r, C, V, 1, 1.f, z, p.ldz, 1, 0, static_cast<const float*>(w), swv, swc, 0, 0.f, to,
                          p.pad ? C : lddx, 1, 0, nullptr, gws, gbytes, stream);
        if (!rc && p.pad) {  // (what the rows behind give is left there)
          hipLaunchKernelGGL(pad_kernel, dim3(cdiv(r * C, 256)), dim3(256), 0, st, to, C, r, C, static_cast<float*>(dx), lddx, r);
          MTX_LAUNCHED();
        }
      } else {
        GemmBf16 g{};
        g.a = dm;
        g.a_k = true;
        g.b = wm;
        g.b_k = wv;
        g.pieces = p.pieces;
        g.c = static_cast<char*>(dx) + r0 * lddx * (half ? 2 : 4);
        g.ldc = lddx;
        g.c_bf16 = half;
        g.scale = inv;
        g.M = r;
        g.N = C;
        g.K = v8;  // behind V: zeros in dz
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
        float* out = static_cast<float*>(dw);
        if (sums)
          rc = mtx_gemm_wgrad_f32(M, N, r, a, 1, lda, b, ldb, 1, first ? 0.f : 1.f, out, ld, 1, db, !first, gws, gbytes,
                                  stream);
        else
          rc = mtx_gemm_f32(M, N, r, 1, 1.f, a, 1, lda, 0, b, ldb, 1, 0, first ? 0.f : 1.f, out, ld, 1, 0, nullptr, gws,
                            gbytes, stream);
      } else {
        GemmBf16 g{};
        g.a = rows ? xm : dm;
        g.b = rows ? dm : xm;
        g.scale = inv;
        g.pieces = p.pieces;
        g.M = M;
        g.N = N;
        g.K = r;
        // blocks of rows are added up in fp32, the sum is rounded once
        g.c_bf16 = half && last;
        g.c = half && !last ? static_cast<void*>(sum) : dw;
        g.ldc = half && !last ? N : ld;
        if (!first) {
          g.add = half ? sum : static_cast<const float*>(dw);
          g.ldadd = half ? N : ld;
        }
        rc = gemm_bf16(g, gws, st);
      }
      if (rc) return rc;
    }
  }
  if (part || (db && n == 0)) {
    hipLaunchKernelGGL(bias_kernel, dim3(cdiv(V, 64)), dim3(1024), 0, st, part, p.ldz, n ? p.wgs : 0, V, inv, db);
    MTX_LAUNCHED();
  }
  if (n && p.narrow && (dw || db)) return MTX_OK;  // (narrow_grad has it)
  hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, st, MeanLoss{row_loss, labels, n, V, loss});
  MTX_LAUNCHED();
  return MTX_OK;
}
