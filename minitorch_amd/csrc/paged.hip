// Keys and values kept in pages, for gfx950 (MI355X): writing new rows
// (mtx_kv_append_paged), attention of one new token per sequence over them
// (mtx_attn_decode_paged) and cutting a cache down to the rows that received
// the most attention (mtx_kv_evict_paged).
//
// A page holds `page` rows of every K/V head; a sequence's row j lies in page
// table[b][j / page] at row j % page.  Page ids come from device memory, so the
// kernels check each against the pool before using it: a row whose page id is
// outside [0, n_pages) is not there (attention does not see it, nothing is
// written to it).
//
// The reference recomputes the whole forward per token (GPT.generate,
// transformer.py:93-104) and has no cache; the attention is its sub-graph
// transformer.py:36-44 at the last position.
#include "mtx_common.h"

#include <algorithm>
#include <cmath>

namespace mtx {
namespace {

struct Pages {  // (n_pages, heads, page, D) view: element strides, d stride 1
  void* p;
  int64_t sp, sh, sr;
};

struct Table {
  const int* ids;
  int64_t ld;
  int width;        // pages per sequence
  int page;         // rows per page
  int64_t n_pages;  // pages in the pool
};

// page id of row j, or -1
__device__ __forceinline__ int page_of(const Table& t, int b, int j) {
  const int id = t.ids[b * t.ld + j / t.page];
  return (unsigned)id < (unsigned)t.n_pages ? id : -1;
}
__device__ __forceinline__ int64_t row_at(const Pages& g, const Table& t, int id, int h, int j) {
  return id * g.sp + h * g.sh + (j % t.page) * g.sr;
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct AppendArgs {
  const void* x[2];
  int64_t sb[2], sh[2], st[2];
  Pages g[2];
  Table tab;
  const int* lengths;
  const int* counts;
  int T, H, D, blocks;
};

template <typename TX, typename TC>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a) {
  const int z = blockIdx.y, b = blockIdx.x / a.blocks;
  const int c8 = a.D >> 3;  // chunks of 8 values a row
  const int i = (blockIdx.x % a.blocks) * 256 + threadIdx.x;
  if (i >= a.T * a.H * c8) return;
  const int c = i % c8, h = (i / c8) % a.H, t = i / (c8 * a.H);
  const int n = a.counts != nullptr ? min(a.counts[b], a.T) : a.T;
  const int j = a.lengths[b] - n + t;
  if (t >= n || j < 0 || j >= a.tab.width * a.tab.page) return;
  const int id = page_of(a.tab, b, j);
  if (id < 0) return;
  const TX* __restrict__ x = static_cast<const TX*>(a.x[z]) + b * a.sb[z] + h * a.sh[z] + t * a.st[z] + 8 * c;
  TC* __restrict__ y = static_cast<TC*>(a.g[z].p) + row_at(a.g[z], a.tab, id, h, j) + 8 * c;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (sizeof(TX) == sizeof(TC)) y[e] = x[e];
    else y[e] = Elem<TC>::from_f(Elem<TX>::to_f(x[e]));
  }
}

// ---------------------------------------------------------------------------
// decode
// ---------------------------------------------------------------------------
struct DecodeArgs {
  const void* q;
  int64_t qb, qh;
  Pages k, v;
  Table tab;
  const int* lengths;
  void* o;
  int64_t ob, oh;
  float* lse;
  const float* win;
  float* w;
  int64_t wld;
  float* ws;
  int B, H, Hkv, D, cap;
  float scale;
};

__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// one workgroup per sequence and query head, the scores in the workspace
template <typename TQ, typename TC>
__global__ __launch_bounds__(256) void decode_kernel(const DecodeArgs a) {
  __shared__ float q[128], red[4];
  const int b = blockIdx.x / a.H, h = blockIdx.x % a.H, hk = h / (a.H / a.Hkv);
  const int tid = threadIdx.x, len = min(max(a.lengths[b], 0), a.cap);
  const TQ* __restrict__ qp = static_cast<const TQ*>(a.q) + b * a.qb + h * a.qh;
  if (tid < a.D) q[tid] = Elem<TQ>::to_f(qp[tid]);
  __syncthreads();
  float* __restrict__ s = a.ws + (int64_t)blockIdx.x * a.cap;
  float m = -INFINITY;
  for (int j = tid; j < len; j += 256) {
    const int id = page_of(a.tab, b, j);
    float x = -INFINITY;
    if (id >= 0) {
      const TC* __restrict__ k = static_cast<const TC*>(a.k.p) + row_at(a.k, a.tab, id, hk, j);
      x = 0.f;
      for (int d = 0; d < a.D; ++d) x = fmaf(q[d], Elem<TC>::to_f(k[d]), x);
      x *= a.scale;
    }
    s[j] = x;
    m = fmaxf(m, x);
  }
  m = wave_max(m);
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  if (m == -INFINITY) m = 0.f;
  float l = 0.f;
  for (int j = tid; j < len; j += 256) l += expf(s[j] - m);
  l = block_sum(l, red);
  if (a.lse != nullptr && tid == 0) a.lse[blockIdx.x] = m + logf(l);
  __syncthreads();
  TQ* __restrict__ op = static_cast<TQ*>(a.o) + b * a.ob + h * a.oh;
  if (tid < a.D) {
    float acc = 0.f;
    for (int j = 0; j < len; ++j) {
      const int id = page_of(a.tab, b, j);
      if (id < 0) continue;
      acc = fmaf(expf(s[j] - m), Elem<TC>::to_f((static_cast<const TC*>(a.v.p) + row_at(a.v, a.tab, id, hk, j))[tid]),
                 acc);
    }
    op[tid] = Elem<TQ>::from_f(l > 0.f || l != l ? acc / l : 0.f);
  }
  if (a.w != nullptr) {
    __syncthreads();  // the scores are read above
    const float lse = m + logf(l);
    for (int j = tid; j < len; j += 256) s[j] = s[j] == -INFINITY ? 0.f : expf(s[j] - lse);
  }
}

__global__ __launch_bounds__(256) void weights_kernel(const DecodeArgs a) {
  const int bh = blockIdx.y, b = bh / a.Hkv, G = a.H / a.Hkv;
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= min(a.lengths[b], a.cap)) return;
  const float* __restrict__ s = a.ws + (int64_t)bh * G * a.cap + j;
  float w = 0.f;
  for (int g = 0; g < G; ++g) w += s[(int64_t)g * a.cap];
  if (a.win != nullptr) w += a.win[bh * a.wld + j];
  a.w[bh * a.wld + j] = w;
}

// ---------------------------------------------------------------------------
// evict
// ---------------------------------------------------------------------------
struct EvictArgs {
  Pages k, v;
  Table from, to;
  const int* lengths;
  const float* w;
  int64_t wld;
  int* lengths_out;
  float* w_out;
  int* slots;
  int B, H, D, cap, keep, recent;
};

// order of weights as unsigned numbers: NaN above everything, -0 equal to 0
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

__device__ __forceinline__ int block_count(int v, int* red) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// one workgroup per sequence and K/V head: the smallest key that is kept, bit
// by bit, then the kept slots in order
__global__ __launch_bounds__(256) void select_kernel(const EvictArgs a) {
  __shared__ int red[4], scan[256];
  const int bh = blockIdx.x, b = bh / a.H, tid = threadIdx.x;
  const int len = min(max(a.lengths[b], 0), a.cap);
  const float* __restrict__ w = a.w + bh * a.wld;
  int* __restrict__ slots = a.slots + (int64_t)bh * a.keep;
  float* __restrict__ wo = a.w_out + bh * a.wld;
  if (tid == 0 && bh % a.H == 0) a.lengths_out[b] = min(len, a.keep);
  const int cand = len > a.keep ? len - a.recent : 0, want = a.keep - a.recent;
  uint32_t bound = 0;
  if (cand > 0) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = bound | (1u << bit);
      int n = 0;
      for (int j = tid; j < cand; j += 256) n += weight_key(w[j]) >= t;
      if (block_count(n, red) >= want) bound = t;
    }
  }
  int above = 0;
  for (int j = tid; j < cand; j += 256) above += weight_key(w[j]) > bound;
  int ties = want - block_count(above, red);  // of those equal to the bound, the first ones
  int at = 0;
  for (int j0 = 0; j0 < len; j0 += 256) {
    const int j = j0 + tid;
    const uint32_t key = j < cand ? weight_key(w[j]) : 0u;
    const bool tie = j < cand && key == bound;
    scan[tid] = tie;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < 256; ++i) {
      before += i < tid ? scan[i] : 0;
      all += scan[i];
    }
    __syncthreads();
    const bool kept = j < len && (j >= cand || key > bound || (tie && before < ties));
    ties = max(0, ties - all);
    scan[tid] = kept;
    __syncthreads();
    before = 0, all = 0;
    for (int i = 0; i < 256; ++i) {
      before += i < tid ? scan[i] : 0;
      all += scan[i];
    }
    __syncthreads();
    if (kept && at + before < a.keep) {
      slots[at + before] = j;
      wo[at + before] = w[j];
    }
    at += all;
  }
  for (int j = at + tid; j < a.keep; j += 256) slots[j] = -1;
  for (int j = at + tid; j < a.cap; j += 256) wo[j] = 0.f;
}

template <typename TC>
__global__ __launch_bounds__(256) void gather_kernel(const EvictArgs a, int blocks) {
  const int bh = blockIdx.x / blocks, b = bh / a.H, h = bh % a.H;
  const int c8 = a.D >> 3, i = (blockIdx.x % blocks) * 256 + threadIdx.x;
  const int r = i / c8, c = i % c8;
  if (r >= a.keep) return;
  const int j = a.slots[(int64_t)bh * a.keep + r];
  if (j < 0) return;
  const int from = page_of(a.from, b, j), to = page_of(a.to, b, r);
  if (to < 0) return;
  const Pages& g = blockIdx.y ? a.v : a.k;
  const TC* __restrict__ x = static_cast<const TC*>(g.p) + row_at(g, a.from, from < 0 ? 0 : from, h, j) + 8 * c;
  TC* __restrict__ y = static_cast<TC*>(g.p) + row_at(g, a.to, to, h, r) + 8 * c;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = from < 0 ? (TC)0 : x[e];
}

// ---------------------------------------------------------------------------
// host checks
// ---------------------------------------------------------------------------
int check_dtypes(int dtype, int cache_dtype) {
  if (!((dtype == MTX_F32 && (cache_dtype == MTX_F32 || cache_dtype == MTX_BF16)) ||
        (dtype == MTX_BF16 && cache_dtype == MTX_BF16)))
    return fail(MTX_ERR_DTYPE, "dtypes %d over a cache of %d: fp32 over fp32 or bf16, or bf16 over bf16", dtype,
                cache_dtype);
  return MTX_OK;
}

// the three outer strides of a 4-d view whose d stride is 1
int check_view(const char* name, const void* p, const int64_t* s, int es) {
  MTX_CHECK_ARG(p != nullptr && s != nullptr, "%s: null pointer", name);
  MTX_CHECK_ARG(s[3] == 1, "%s: d stride must be 1 (got %lld)", name, (long long)s[3]);
  const int vec = 16 / es;
  for (int i = 0; i < 3; ++i)
    MTX_CHECK_ARG(s[i] >= 0 && s[i] % vec == 0, "%s: stride[%d]=%lld must be a non-negative multiple of %d elements",
                  name, i, (long long)s[i], vec);
  MTX_CHECK_ARG(((uintptr_t)p & 15u) == 0, "%s: pointer must be 16-byte aligned", name);
  return MTX_OK;
}

// no two rows of a view that is written may share memory
int check_apart(const char* name, const int64_t* s, int64_t n0, int64_t n1, int64_t n2, int D) {
  std::pair<int64_t, int64_t> d[3] = {{s[0], n0}, {s[1], n1}, {s[2], n2}};
  std::sort(d, d + 3);
  int64_t extent = D;
  for (auto& x : d) {
    if (x.second <= 1) continue;
    MTX_CHECK_ARG(x.first >= extent, "%s: rows overlap (strides %lld, %lld, %lld)", name, (long long)s[0],
                  (long long)s[1], (long long)s[2]);
    extent += x.first * (x.second - 1);
  }
  return MTX_OK;
}

int check_cache(int B, int H, int D, int64_t n_pages, int page, const int* table, int64_t table_ld, int width,
                const int* lengths) {
  MTX_CHECK_SHAPE(B >= 1 && H >= 1 && (int64_t)B * H <= (1 << 20), "B, H must be >= 1 and B*H <= 2^20 (got %d, %d)",
                  B, H);
  MTX_CHECK_SHAPE(D == 16 || D == 32 || D == 64 || D == 128, "head dim D=%d not in {16,32,64,128}", D);
  MTX_CHECK_SHAPE(page >= 1 && page <= 65536 && n_pages >= 1 && n_pages <= INT32_MAX,
                  "pages: 1 to 65536 rows each, 1 to 2^31-1 of them (got %d, %lld)", page, (long long)n_pages);
  MTX_CHECK_SHAPE(width >= 1 && (int64_t)width * page <= (1 << 28),
                  "a sequence's pages must hold 1 to 2^28 rows (got %d of %d)", width, page);
  MTX_CHECK_ARG(table != nullptr && lengths != nullptr, "table, lengths: null pointer");
  MTX_CHECK_ARG(table_ld >= 0, "table: negative row stride");
  return MTX_OK;
}

}  // namespace
}  // namespace mtx

using namespace mtx;

extern "C" int mtx_kv_append_paged(int dtype, int cache_dtype, int B, int T, int H, int D, const void* k,
                                   const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                   int64_t n_pages, int page, void* k_pages, const int64_t* kp_strides,
                                   void* v_pages, const int64_t* vp_strides, const int* table, int64_t table_ld,
                                   int max_pages, const int* lengths, const int* counts, void* stream) {
  int rc;
  if ((rc = check_dtypes(dtype, cache_dtype))) return rc;
  if ((rc = check_cache(B, H, D, n_pages, page, table, table_ld, max_pages, lengths))) return rc;
  MTX_CHECK_SHAPE(T >= 1 && (int64_t)T * H * (D / 8) <= (1 << 30), "T=%d new rows of %d heads: at least 1", T, H);
  const int es = dtype == MTX_F32 ? 4 : 2, ec = cache_dtype == MTX_F32 ? 4 : 2;
  if ((rc = check_view("k", k, k_strides, es))) return rc;
  if ((rc = check_view("v", v, v_strides, es))) return rc;
  if ((rc = check_view("k_pages", k_pages, kp_strides, ec))) return rc;
  if ((rc = check_view("v_pages", v_pages, vp_strides, ec))) return rc;
  if ((rc = check_apart("k_pages", kp_strides, n_pages, H, page, D))) return rc;
  if ((rc = check_apart("v_pages", vp_strides, n_pages, H, page, D))) return rc;
  AppendArgs a{{k, v},
               {k_strides[0], v_strides[0]},
               {k_strides[1], v_strides[1]},
               {k_strides[2], v_strides[2]},
               {{k_pages, kp_strides[0], kp_strides[1], kp_strides[2]},
                {v_pages, vp_strides[0], vp_strides[1], vp_strides[2]}},
               {table, table_ld, max_pages, page, n_pages},
               lengths,
               counts,
               T,
               H,
               D,
               cdiv(T * H * (D / 8), 256)};
  MTX_CHECK_SHAPE((int64_t)B * a.blocks <= INT32_MAX, "append: too many rows in one call");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(B * a.blocks, 2);
  if (cache_dtype == MTX_F32) hipLaunchKernelGGL((append_kernel<float, float>), grid, dim3(256), 0, st, a);
  else if (dtype == MTX_F32) hipLaunchKernelGGL((append_kernel<float, bf16_t>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((append_kernel<bf16_t, bf16_t>), grid, dim3(256), 0, st, a);
  MTX_LAUNCHED();
  return MTX_OK;
}

extern "C" size_t mtx_attn_decode_paged_workspace_bytes(int B, int H, int Hkv, int D, int page, int max_pages,
                                                        int with_weights) {
  if (B < 1 || H < 1 || page < 1 || max_pages < 1) return 0;
  return (size_t)B * H * page * max_pages * sizeof(float);
}

extern "C" int mtx_attn_decode_paged(int dtype, int cache_dtype, int B, int H, int Hkv, int D, const void* q,
                                     const int64_t* q_strides, int64_t n_pages, int page, const void* k_pages,
                                     const int64_t* kp_strides, const void* v_pages, const int64_t* vp_strides,
                                     const int* table, int64_t table_ld, int max_pages, const int* lengths, void* o,
                                     const int64_t* o_strides, float* lse, const float* weights_in, float* weights,
                                     int64_t weights_ld, void* workspace, size_t workspace_bytes, float scale,
                                     void* stream) {
  int rc;
  if ((rc = check_dtypes(dtype, cache_dtype))) return rc;
  if ((rc = check_cache(B, H, D, n_pages, page, table, table_ld, max_pages, lengths))) return rc;
  MTX_CHECK_SHAPE(Hkv >= 1 && H % Hkv == 0, "H=%d query heads must be a multiple of Hkv=%d K/V heads", H, Hkv);
  const int es = dtype == MTX_F32 ? 4 : 2, ec = cache_dtype == MTX_F32 ? 4 : 2;
  if ((rc = check_view("q", q, q_strides, es))) return rc;
  if ((rc = check_view("k_pages", k_pages, kp_strides, ec))) return rc;
  if ((rc = check_view("v_pages", v_pages, vp_strides, ec))) return rc;
  if ((rc = check_view("o", o, o_strides, es))) return rc;
  const int64_t os[4] = {o_strides[0], o_strides[1], 0, 1};
  if ((rc = check_apart("o", os, B, H, 1, D))) return rc;
  MTX_CHECK_ARG(std::isfinite(scale) && scale > 0.f, "scale must be finite and > 0");
  const int cap = max_pages * page;
  MTX_CHECK_ARG(weights != nullptr || weights_in == nullptr, "weights_in without weights");
  MTX_CHECK_ARG(weights == nullptr || weights_ld >= cap, "weights: rows of %lld values for %d cached rows",
                (long long)weights_ld, cap);
  const size_t need = mtx_attn_decode_paged_workspace_bytes(B, H, Hkv, D, page, max_pages, weights != nullptr);
  MTX_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need), "workspace too small (%zu < %zu)",
                workspace_bytes, need);
  DecodeArgs a{q, q_strides[0], q_strides[1],
               {const_cast<void*>(k_pages), kp_strides[0], kp_strides[1], kp_strides[2]},
               {const_cast<void*>(v_pages), vp_strides[0], vp_strides[1], vp_strides[2]},
               {table, table_ld, max_pages, page, n_pages},
               lengths, o, o_strides[0], o_strides[1], lse, weights_in, weights, weights_ld,
               static_cast<float*>(workspace), B, H, Hkv, D, cap, scale};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache_dtype == MTX_F32) hipLaunchKernelGGL((decode_kernel<float, float>), dim3(B * H), dim3(256), 0, st, a);
  else if (dtype == MTX_F32) hipLaunchKernelGGL((decode_kernel<float, bf16_t>), dim3(B * H), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((decode_kernel<bf16_t, bf16_t>), dim3(B * H), dim3(256), 0, st, a);
  MTX_LAUNCHED();
  if (weights != nullptr) {
    MTX_CHECK_SHAPE(B * Hkv <= 65535, "weights: at most 65535 sequences times K/V heads");
    hipLaunchKernelGGL(weights_kernel, dim3(cdiv(cap, 256), B * Hkv), dim3(256), 0, st, a);
    MTX_LAUNCHED();
  }
  return MTX_OK;
}

extern "C" int mtx_kv_evict_paged(int cache_dtype, int B, int H, int D, int64_t n_pages, int page, void* k_pages,
                                  const int64_t* kp_strides, void* v_pages, const int64_t* vp_strides,
                                  const int* table, int64_t table_ld, int max_pages, const int* lengths,
                                  const float* weights, int64_t weights_ld, const int* to_table, int64_t to_ld,
                                  int to_pages, int keep, int recent, int* lengths_out, float* weights_out,
                                  int* slots, void* stream) {
  int rc;
  if ((rc = check_dtypes(cache_dtype, cache_dtype))) return rc;
  if ((rc = check_cache(B, H, D, n_pages, page, table, table_ld, max_pages, lengths))) return rc;
  const int ec = cache_dtype == MTX_F32 ? 4 : 2;
  if ((rc = check_view("k_pages", k_pages, kp_strides, ec))) return rc;
  if ((rc = check_view("v_pages", v_pages, vp_strides, ec))) return rc;
  if ((rc = check_apart("k_pages", kp_strides, n_pages, H, page, D))) return rc;
  if ((rc = check_apart("v_pages", vp_strides, n_pages, H, page, D))) return rc;
  const int cap = max_pages * page;
  MTX_CHECK_SHAPE(keep >= 1 && recent >= 0 && recent <= keep && keep <= (1 << 28),
                  "evict: needs 1 <= keep and 0 <= recent <= keep (got %d, %d)", keep, recent);
  MTX_CHECK_SHAPE(to_pages >= 1 && (int64_t)to_pages * page >= std::min(keep, cap),
                  "evict: %d pages of %d rows do not hold keep=%d", to_pages, page, keep);
  MTX_CHECK_ARG(weights && to_table && lengths_out && weights_out && slots, "evict: null pointer");
  MTX_CHECK_ARG(to_ld >= 0 && weights_ld >= cap, "evict: rows of %lld weights for %d cached rows",
                (long long)weights_ld, cap);
  MTX_CHECK_ARG(weights_out != weights && lengths_out != lengths && to_table != table,
                "evict: the new weights, lengths and pages must be others than the old ones");
  const int rows = std::min(keep, cap);
  EvictArgs a{{k_pages, kp_strides[0], kp_strides[1], kp_strides[2]},
              {v_pages, vp_strides[0], vp_strides[1], vp_strides[2]},
              {table, table_ld, max_pages, page, n_pages},
              {to_table, to_ld, to_pages, page, n_pages},
              lengths, weights, weights_ld, lengths_out, weights_out, slots, B, H, D, cap, keep, recent};
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(select_kernel, dim3(B * H), dim3(256), 0, st, a);
  MTX_LAUNCHED();
  const int64_t blocks = ((int64_t)rows * (D / 8) + 255) / 256;
  MTX_CHECK_SHAPE(blocks * B * H <= INT32_MAX, "evict: too many rows in one call");
  const dim3 grid((unsigned)(blocks * B * H), 2);
  if (cache_dtype == MTX_F32) hipLaunchKernelGGL(gather_kernel<float>, grid, dim3(256), 0, st, a, (int)blocks);
  else hipLaunchKernelGGL(gather_kernel<bf16_t>, grid, dim3(256), 0, st, a, (int)blocks);
  MTX_LAUNCHED();
  return MTX_OK;
}
