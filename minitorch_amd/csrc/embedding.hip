// Embedding lookup with scaling, and its gradient without atomics on values (fp32, bf16).
//
//   out[i][c] = scale * W[t_i][c]                      (0 where t_i is no token)
//   dW[v][c] (+)= scale * sum over i with t_i = v of g[i][c], in token order
//
// A token outside [0, V) is none: padding.  Its row comes out as zeros and its
// gradient goes nowhere.
//
// The gradient's sums have one order, in one of three ways, by the sizes:
//   few tokens     one launch; a workgroup finds the tokens of its table rows by
//                  comparing (small_kernel)
//   small tables   the table in LDS, a chunk of the tokens a workgroup, then the
//                  chunks' tables added up (table_kernel, table_sum_kernel)
//   all others     one launch sorts the tokens (every workgroup takes a range of the
//                  table and looks through all ids for its own, so no workgroup waits
//                  for another) and sets rows without one to 0, one adds up (rows of
//                  more than kPiece tokens in pieces of the sorted order), one joins
//                  the pieces (sort_kernel, add_kernel, join_kernel)
// Bound by memory: the gradient's rows are read and the table written, once each.
#include "mtx_common.h"

#include <type_traits>

namespace mtx {
namespace {

// N values of T from or to memory, in 16-byte accesses where N values fill them
template <typename T, int N>
struct Pack {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ void load_f(const T* __restrict__ p, float (&f)[N]) {
  if constexpr (N == 1) {
    f[0] = Elem<T>::to_f(*p);
  } else {
    constexpr int K = 16 / sizeof(T);
    static_assert(N % K == 0, "whole 16-byte accesses");
#pragma unroll
    for (int i = 0; i < N / K; ++i) {
      const Pack<T, K> q = __builtin_bit_cast(Pack<T, K>, reinterpret_cast<const uint4*>(p)[i]);
#pragma unroll
      for (int j = 0; j < K; ++j) f[i * K + j] = Elem<T>::to_f(q.v[j]);
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_f(T* __restrict__ p, const float (&f)[N]) {
  if constexpr (N == 1) {
    *p = Elem<T>::from_f(f[0]);
  } else {
    constexpr int K = 16 / sizeof(T);
    static_assert(N % K == 0, "whole 16-byte accesses");
#pragma unroll
    for (int i = 0; i < N / K; ++i) {
      Pack<T, K> q;
#pragma unroll
      for (int j = 0; j < K; ++j) q.v[j] = Elem<T>::from_f(f[i * K + j]);
      reinterpret_cast<uint4*>(p)[i] = __builtin_bit_cast(uint4, q);
    }
  }
}

// LPR lanes take a row, VEC values at a time, and kLookRows rows one after another:
// their ids, then their values, are requested before the first is needed.  Bound by
// memory (32768 rows of 1024 bf16 values, words: 17 us, 67 MB written); where the rows
// are too few to fill the chip, the columns are dealt out too (5 rows of 1838 fp32
// values: 4.7 us a call, 11.5 by one workgroup).
constexpr int kLookRows = 4;
template <typename T, typename O, int VEC, int LPR>
__global__ __launch_bounds__(256) void lookup_kernel(const T* __restrict__ w, int64_t ldw, int64_t V,
                                                     const int64_t* __restrict__ ids, int64_t n, int C, float scale,
                                                     O* __restrict__ out, int64_t ldo) {
  constexpr int kRows = 256 / LPR * kLookRows;  // rows a workgroup
  const int sub = threadIdx.x % LPR, nv = C / VEC;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < n; r0 += (int64_t)gridDim.x * kRows) {
    const int64_t i0 = r0 + threadIdx.x / LPR;
    int64_t t[kLookRows];
#pragma unroll
    for (int k = 0; k < kLookRows; ++k) {
      const int64_t i = i0 + k * (256 / LPR);
      t[k] = i < n ? ids[i] : -1;
    }
    for (int c = sub + (int)blockIdx.y * LPR; c < nv; c += LPR * (int)gridDim.y) {
      float f[kLookRows][VEC];
#pragma unroll
      for (int k = 0; k < kLookRows; ++k) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[k][j] = 0.f;
        if (t[k] >= 0 && t[k] < V) load_f<T, VEC>(w + t[k] * ldw + c * VEC, f[k]);
      }
#pragma unroll
      for (int k = 0; k < kLookRows; ++k) {
        const int64_t i = i0 + k * (256 / LPR);
        if (i >= n) continue;
        // a row without a token stays 0 whatever the scale
        const float s = t[k] >= 0 && t[k] < V ? scale : 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[k][j] *= s;
        store_f<O, VEC>(out + i * ldo + c * VEC, f[k]);
      }
    }
  }
}

constexpr int kPiece = 32;  // sorted tokens a piece; rows of more are added in pieces

// ---------------------------------------------------------------------------
// Sorting.  Workgroup b owns the table rows [b R, (b + 1) R).  Its 16 waves take
// contiguous parts of the ids; every wave counts its part's ids per row, and how
// many lie below the range.  The counts' prefix sums, over rows and within a row
// over waves, are where each wave's ids go in the sorted order; a second look at
// the ids puts them there, in order.  Of 64 ids few belong to one workgroup (one
// in 256), so the loop over a group's distinct rows is short; where many do, a
// small table or one token everywhere, its rows are few.
// ---------------------------------------------------------------------------
constexpr int kWaves = 16, kMaxRows = 512;  // 32 KB of counts
constexpr int kAhead = 16, kHeld = 32;  // groups of 64 ids that a wave requests at once, and holds

struct SortArgs {
  const int64_t* ids;
  int64_t n, V;
  int R;            // rows of the table a workgroup
  uint2* span;      // [V] out: (first place in the sorted order, tokens)
  uint32_t* order;  // [tokens] out: the sorted tokens' places
  uint32_t* key;    // [tokens] out: and rows
  uint32_t* tokens;  // out: how many they are
  uint32_t* starts;  // [pieces] out: the row of more than a piece that begins there
  // Rows without a token are set to 0 here, while the sorting waits for its memory: of
  // 50021 x 1024 rows (205 MB) three quarters are, which makes this launch 43 us instead
  // of 16 and the adding up 30 instead of 66.  nullptr: they are left alone
  float* dw;
  int64_t lddw;
  int C, vec;
};

__global__ __launch_bounds__(64 * kWaves) void sort_kernel(const SortArgs a) {
  __shared__ uint32_t below[kWaves], sums[kWaves];
  extern __shared__ uint32_t cnt[];  // [wave][R], then the rows' tokens
  const int64_t* ids = a.ids;
  const int64_t n = a.n;
  const int R = a.R;
  uint32_t* count = cnt + kWaves * R;
  const int64_t v0 = (int64_t)blockIdx.x * R;
  const uint32_t rows = (uint32_t)min<int64_t>(R, a.V - v0);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t part = (n + 64 * kWaves - 1) / (64 * kWaves) * 64;
  const int64_t beg = min(n, w * part), end = min(n, beg + part);
  const bool once = part <= 64 * kHeld;  // the ids stay in registers for the second look
  uint32_t* mine = cnt + w * R;
  for (int i = tid; i < R * kWaves; i += 64 * kWaves) cnt[i] = 0;
  __syncthreads();

  uint32_t t[kHeld], less = 0;  // rows in the range, ~0 for others
  auto request = [&](int64_t i0) {
#pragma unroll
    for (int h = 0; h < kHeld; h += kAhead) {
      uint2 id[kAhead];
      const int64_t from = i0 + 64 * h;
      const int last = (int)min<int64_t>(end - 1 - from, 64 * kAhead);
      if (last < 0) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) t[h + k] = ~0u;
        continue;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) id[k] = reinterpret_cast<const uint2*>(ids + from)[min(64 * k + lane, last)];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const uint32_t v = id[k].y == 0 && 64 * k + lane <= last ? id[k].x : ~0u, off = v - (uint32_t)v0;
        less += v < (uint32_t)v0;
        t[h + k] = off < rows ? off : ~0u;
      }
    }
  };
  for (int64_t i0 = beg; i0 < end; i0 += 64 * kHeld) {
    request(i0);
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (t[k] != ~0u) atomicAdd(&mine[t[k]], 1u);
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) less += __shfl_xor(less, m, 64);
  if (lane == 0) below[w] = less;
  __syncthreads();

  // thread r has row r: its count, and the prefix sum over the rows before it
  uint32_t base = 0, total = 0;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) base += below[k];
  uint32_t c[kWaves];
  if (tid < R)
#pragma unroll
    for (int k = 0; k < kWaves; ++k) total += c[k] = cnt[k * R + tid];
  uint32_t run = total;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint32_t o = __shfl_up(run, m, 64);
    if (lane >= m) run += o;
  }
  if (lane == 63) sums[w] = run;
  __syncthreads();
  for (int k = 0; k < w; ++k) base += sums[k];
  uint32_t at = base + run - total;
  if (tid < (int)rows) {
    a.span[v0 + tid] = make_uint2(at, total);
    if (v0 + tid == a.V - 1) *a.tokens = at + total;
    if (total > kPiece) a.starts[at / kPiece] = (uint32_t)v0 + tid;  // at most one in a piece
    count[tid] = total;
  }
  if (tid < R)
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      cnt[k * R + tid] = at;
      at += c[k];
    }
  __syncthreads();
  if (a.dw)
    for (uint32_t r = w; r < rows; r += kWaves)
      if (count[r] == 0) {
        float* p = a.dw + (v0 + r) * a.lddw;
        if (a.vec)
          for (int k = 4 * lane; k < a.C; k += 256) *reinterpret_cast<f32x4*>(p + k) = zero4();
        else
          for (int k = lane; k < a.C; k += 64) p[k] = 0.f;
      }
  for (int64_t i0 = beg; i0 < end; i0 += 64 * kHeld) {
    if (!once) request(i0);
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      uint64_t left = __ballot(t[k] != ~0u);
      while (left) {
        const uint32_t r = __builtin_amdgcn_readlane(t[k], __builtin_ctzll(left));
        const uint64_t same = __ballot(t[k] == r);
        const uint32_t to = mine[r];
        if (t[k] == r) {
          const uint32_t place = to + __builtin_popcountll(same & ((1ull << lane) - 1));
          a.order[place] = (uint32_t)(i0 + 64 * k + lane);
          a.key[place] = (uint32_t)v0 + r;
        }
        mine[r] = to + __builtin_popcountll(same);  // by every lane, so that each reads its own write
        left &= ~same;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Adding up.  A group of LPR lanes, U vectors of VEC values a lane, takes a column
// slice of one table row, or of one piece of the sorted order.
// ---------------------------------------------------------------------------

struct GradArgs {
  const int64_t* ids;
  const void* g;
  int64_t ldg;
  float scale;
  float* dw;
  int64_t lddw, V, n;
  int C, slices, rows, accumulate;  // rows of the table a group takes
  const uint2* span;       // [V] (first place in the sorted order, tokens)
  const uint32_t* order;   // [tokens] the sorted tokens' places
  const uint32_t* key;     // [tokens] and rows
  const uint32_t* tokens;  // how many they are
  const uint32_t* starts;  // [pieces] the row of more than a piece that begins there, or anything
  float* part;             // [pieces][2][C] sums of pieces
};

// acc += the rows order[0 .. N), in order; all N are requested before the first is
// added.  Columns past C read the row's last ones.
template <typename T, int VEC, int LPR, int U, int N>
__device__ __forceinline__ void add_some(const GradArgs& a, const uint32_t* order, int c0, float (&acc)[U][VEC]) {
  const T* g = static_cast<const T*>(a.g);
  float f[N][U][VEC];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const T* row = g + order[k] * a.ldg;
#pragma unroll
    for (int u = 0; u < U; ++u) load_f<T, VEC>(row + min(c0 + u * LPR * VEC, a.C - VEC), f[k][u]);
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[u][j] += f[k][u][j];
}

// acc = the sum of the rows order[0 .. len)
template <typename T, int VEC, int LPR, int U, int AHEAD = 8>
__device__ __forceinline__ void add_rows(const GradArgs& a, const uint32_t* order, int len, int c0,
                                         float (&acc)[U][VEC]) {
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[u][j] = 0.f;
  if constexpr (LPR == 64) len = __builtin_amdgcn_readfirstlane(len);
  int k = 0;
  for (; k + AHEAD <= len; k += AHEAD) add_some<T, VEC, LPR, U, AHEAD>(a, order + k, c0, acc);
  if (AHEAD > 4 && len - k >= 4) {
    add_some<T, VEC, LPR, U, 4>(a, order + k, c0, acc);
    k += 4;
  }
  if (len - k >= 2) {
    add_some<T, VEC, LPR, U, 2>(a, order + k, c0, acc);
    k += 2;
  }
  if (len > k) add_some<T, VEC, LPR, U, 1>(a, order + k, c0, acc);
}

// dW[v] (+)= scale * acc
template <int VEC, int LPR, int U>
__device__ __forceinline__ void store_row(const GradArgs& a, int64_t v, int c0, float (&acc)[U][VEC]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = c0 + u * LPR * VEC;
    if (c >= a.C) continue;
    float* p = a.dw + v * a.lddw + c;
    float old[VEC];
    if (a.accumulate) load_f<float, VEC>(p, old);
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[u][j] = a.scale * acc[u][j] + (a.accumulate ? old[j] : 0.f);
    store_f<float, VEC>(p, acc[u]);
  }
}

// A wave's `rows` table rows from v0 on.  Their tokens follow each other in the sorted
// order: up to eight tokens' values are requested at once, whichever rows they are
// for, and a row is stored where its tokens end (one without a token was set to 0 by
// the sort).
template <typename T, int VEC, int U>
__device__ __forceinline__ void add_range(const GradArgs& a, int64_t v0, int rows, int c0) {
  const T* g = static_cast<const T*>(a.g);
  const int lane = threadIdx.x & 63;
  uint2 s = a.span[v0 + min(lane, rows - 1)];
  const uint32_t first = __builtin_amdgcn_readfirstlane(s.x);
  const int begins = (int)(s.x - first), ends = begins + (int)s.y;  // within the range's tokens
  const int total = __builtin_amdgcn_readlane(ends, rows - 1);
  const uint64_t longs = __ballot(lane < rows && s.y > kPiece);
  float acc[U][VEC];
  auto clear = [&] {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[u][j] = 0.f;
  };
  int r = 0, k = 0, held = -64;  // the row, the token, and the first token of those whose places are in o
  uint32_t o = 0;
  int end = __builtin_amdgcn_readlane(ends, 0);
  bool some = false;  // whether the row has tokens
  clear();
  // store the rows that end at token k
  auto flush = [&] {
    while (k == end && r < rows) {
      if (some) store_row<VEC, 64, U>(a, v0 + r, c0, acc);
      clear();
      some = false;
      ++r;
      end = r < rows ? __builtin_amdgcn_readlane(ends, r) : total;
    }
  };
  auto take = [&](auto count) {
    constexpr int N = decltype(count)::value;
    if (k + N > held + 64) {
      held = k;
      o = a.order[first + min(k + lane, total - 1)];
    }
    float f[N][U][VEC];
#pragma unroll
    for (int m = 0; m < N; ++m) {
      const T* row = g + (int64_t)__builtin_amdgcn_readlane(o, k - held + m) * a.ldg;
#pragma unroll
      for (int u = 0; u < U; ++u) load_f<T, VEC>(row + min(c0 + u * 64 * VEC, a.C - VEC), f[m][u]);
    }
#pragma unroll
    for (int m = 0; m < N; ++m) {
      flush();
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[u][j] += f[m][u][j];
      some = true;
      ++k;
    }
  };
  while (true) {
    flush();
    if (r >= rows) break;
    const uint64_t ahead = longs >> r;
    if (ahead & 1) {  // its pieces are added up elsewhere
      k = end;
      ++r;
      end = r < rows ? __builtin_amdgcn_readlane(ends, r) : total;
      continue;
    }
    const int to = ahead ? __builtin_amdgcn_readlane(begins, r + __builtin_ctzll(ahead)) : total;
    if (to - k >= 8) take(std::integral_constant<int, 8>());
    else if (to - k >= 4) take(std::integral_constant<int, 4>());
    else if (to - k >= 2) take(std::integral_constant<int, 2>());
    else take(std::integral_constant<int, 1>());
  }
}

template <typename T, int VEC, int LPR, int U>
__global__ __launch_bounds__(256) void add_kernel(const GradArgs a) {
  constexpr int kPer = 256 / LPR;
  const int64_t ranges = (a.V + a.rows - 1) / a.rows;
  const int64_t total = (ranges + (a.n + kPiece - 1) / kPiece) * a.slices;
  for (int64_t q = (int64_t)blockIdx.x * kPer + threadIdx.x / LPR; q < total; q += (int64_t)gridDim.x * kPer) {
    const int64_t item = q / a.slices;
    const int c0 = (int)(q - item * a.slices) * LPR * VEC * U + (threadIdx.x % LPR) * VEC;
    float acc[U][VEC];
    if (item < ranges) {
      if constexpr (LPR == 64) {
        const int64_t v0 = item * a.rows;
        add_range<T, VEC, U>(a, v0, (int)min<int64_t>(a.rows, a.V - v0), c0);
      } else {
        const uint2 s = a.span[item];
        if (s.y > kPiece || s.y == 0) continue;
        add_rows<T, VEC, LPR, U>(a, a.order + s.x, (int)s.y, c0, acc);
        store_row<VEC, LPR, U>(a, item, c0, acc);
      }
      continue;
    }
    // a piece: its first token's row, if long, from the piece's start, and its
    // last token's from where that one begins; rows in between are short
    const int64_t piece = item - ranges, p0 = piece * kPiece;
    const int64_t tokens = *a.tokens, p1 = min(p0 + kPiece, tokens);
    if (p0 >= tokens) continue;
    const uint2 s0 = a.span[a.key[p0]], s1 = a.span[a.key[p1 - 1]];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const uint2 s = side ? s1 : s0;
      if (s.y <= kPiece || (side && s.x == s0.x)) continue;
      const int64_t b = max<int64_t>(p0, s.x), e = min<int64_t>(p1, (int64_t)s.x + s.y);
      add_rows<T, VEC, LPR, U>(a, a.order + b, (int)(e - b), c0, acc);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * LPR * VEC;
        if (c < a.C) store_f<float, VEC>(a.part + (piece * 2 + side) * a.C + c, acc[u]);
      }
    }
  }
}

// Joining: a long row's pieces are added up by the workgroup that looks after the
// piece in which it begins.  Each of its 16 waves looks at one piece; the rows found
// are then taken by all of them, 64 columns a wave: `chunks` waves beside each
// other, and 16 / chunks contiguous parts of the row's pieces.
__global__ __launch_bounds__(64 * kWaves) void join_kernel(const GradArgs a, int chunks) {
  __shared__ float sums[kWaves][64];
  __shared__ uint32_t row[kWaves];
  __shared__ uint2 at[kWaves];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int parts = kWaves / chunks, chunk = w % chunks, pt = w / chunks;
  const int64_t pieces = (a.n + kPiece - 1) / kPiece;
  for (int64_t q0 = (int64_t)blockIdx.x * kWaves; q0 < pieces; q0 += (int64_t)gridDim.x * kWaves) {
    __syncthreads();
    if (lane == 0) {
      at[w] = make_uint2(0, 0);
      if (q0 + w < pieces) {
        // (nothing was written for a piece in which no long row begins)
        const uint32_t v = a.starts[q0 + w];
        if (v < a.V) {
          const uint2 s = a.span[v];
          row[w] = v;
          if (s.y > kPiece && s.x / kPiece == q0 + w) at[w] = s;
        }
      }
    }
    __syncthreads();
    for (int k = 0; k < kWaves; ++k) {
      const uint2 s = at[k];
      if (s.y == 0) continue;
      const int64_t piece = q0 + k, count = ((int64_t)s.x + s.y - 1) / kPiece - piece + 1;
      // a piece's first sum, but its second in the piece that the row begins inside
      const float* part = a.part + piece * 2 * a.C;
      const int64_t inside = (int64_t)s.x > piece * kPiece ? a.C : 0;
      const int64_t per = (count + parts - 1) / parts, b = pt * per, e = min(count, b + per);
      for (int c0 = blockIdx.y * 64 * chunks; c0 < a.C; c0 += gridDim.y * 64 * chunks) {
        const int c = c0 + 64 * chunk + lane;
        float t = 0.f;
        if (c < a.C)
#pragma unroll 8
          for (int64_t m = b; m < e; ++m) t += part[m * 2 * a.C + (m == 0 ? inside : 0) + c];
        __syncthreads();
        sums[w][lane] = t;
        __syncthreads();
        if (pt == 0 && c < a.C) {
          for (int m = 1; m < parts; ++m) t += sums[m * chunks + chunk][lane];
          float* p = a.dw + (int64_t)row[k] * a.lddw + c;
          *p = a.accumulate ? *p + a.scale * t : a.scale * t;
        }
      }
    }
  }
}

// The whole gradient in one launch, for few tokens.  A workgroup takes R rows of the
// table, a wave every 16th of them; the ids lie in LDS with the rows' counts, and a row's
// tokens are found by comparing 64 of them at a time.  Rows of more than kPiece tokens
// are left to the end: each wave takes a contiguous part of the ids, and the parts' sums
// are added in order.
// 300 tokens of 384 fp32 values, a table of 5003 rows (7.7 MB): 5.9 us (7.6 with all of a
// row's columns by one workgroup; 208 tokens of 2248, 4 rows: 6.3 and 34); 1339 bf16 tokens of
// 256, 42338 rows (43 MB): 19, and 29 sorted.
constexpr int kSmallTokens = 4096, kScan = 4;  // groups of ids looked at together
template <typename T, int VEC, int U>
__global__ __launch_bounds__(64 * kWaves) void small_kernel(const GradArgs a, int R) {
  constexpr int kCols = 64 * VEC * U;
  __shared__ uint32_t key[kSmallTokens];
  __shared__ float sums[kWaves][kCols];
  __shared__ uint32_t count[kMaxRows], longs[kSmallTokens / kPiece];
  __shared__ uint32_t many;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = (int)a.n;
  const int64_t v0 = (int64_t)blockIdx.x * R;
  const uint32_t rows = (uint32_t)min<int64_t>(R, a.V - v0);
  const int groups = (n + 63) / 64, from = (int)blockIdx.y * kCols + lane * VEC;
  if (threadIdx.x == 0) many = 0;
  if (threadIdx.x < kMaxRows) count[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSmallTokens / 1024; ++k) {
    const int i = threadIdx.x + 1024 * k;
    if (i >= 64 * groups) break;
    const uint2 id = i < n ? reinterpret_cast<const uint2*>(a.ids)[i] : make_uint2(~0u, ~0u);
    const uint32_t off = id.x - (uint32_t)v0;
    key[i] = id.y == 0 && off < rows ? off : ~0u;
    if (id.y == 0 && off < rows) atomicAdd(&count[off], 1u);
  }
  __syncthreads();
  const T* g = static_cast<const T*>(a.g);
  // acc = the tokens of row r among the ids of groups g0 to g1, for columns from c0 on
  auto add = [&](uint32_t r, int g0, int g1, int c0, float (&acc)[U][VEC]) {
    constexpr int N = sizeof(T);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[u][j] = 0.f;
    uint32_t o[N];
    int held = 0;
    auto put = [&](auto count) {
      constexpr int M = decltype(count)::value;
      add_some<T, VEC, 64, U, M>(a, o, c0, acc);
    };
    for (int q0 = g0; q0 < g1; q0 += kScan) {
      uint32_t keys[kScan];
#pragma unroll
      for (int h = 0; h < kScan; ++h) keys[h] = key[64 * min(q0 + h, g1 - 1) + lane];
#pragma unroll
      for (int h = 0; h < kScan; ++h) {
        uint64_t left = q0 + h < g1 ? __ballot(keys[h] == r) : 0;
        while (left) {
          const uint32_t i = 64 * (q0 + h) + __builtin_ctzll(left);
          left &= left - 1;
#pragma unroll
          for (int k = 0; k < N; ++k) o[k] = held == k ? i : o[k];
          if (++held == N) {
            put(std::integral_constant<int, N>());
            held = 0;
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k + 1 < N; ++k)
      if (k < held) {
        const uint32_t one[1] = {o[k]};
        add_some<T, VEC, 64, U, 1>(a, one, c0, acc);
      }
  };
  float acc[U][VEC];
  for (uint32_t r = w; r < rows; r += kWaves) {
    const uint32_t some = __builtin_amdgcn_readfirstlane(count[r]);
    if (some > kPiece) {
      if (lane == 0) longs[atomicAdd(&many, 1u)] = r;
      continue;
    }
    if (some == 0 && a.accumulate) continue;
    for (int c0 = from; c0 - lane * VEC < a.C; c0 += kCols * (int)gridDim.y) {
      add(r, 0, some ? groups : 0, c0, acc);
      store_row<VEC, 64, U>(a, v0 + r, c0, acc);
    }
  }
  __syncthreads();
  // (the order in which the long rows come does not matter: each is added up by itself)
  for (uint32_t k = 0; k < many; ++k) {
    const uint32_t r = longs[k];
    const int per = (groups + kWaves - 1) / kWaves, g0 = min(groups, w * per), g1 = min(groups, g0 + per);
    for (int c0 = from; c0 - lane * VEC < a.C; c0 += kCols * (int)gridDim.y) {
      add(r, g0, g1, c0, acc);
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[w][(u * 64 + lane) * VEC + j] = acc[u][j];
      __syncthreads();
      if (w != 0) continue;
#pragma unroll 1
      for (int m = 1; m < kWaves; ++m)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[u][j] += sums[m][(u * 64 + lane) * VEC + j];
      store_row<VEC, 64, U>(a, v0 + r, c0, acc);
    }
  }
}

// 16384 tokens of 384 fp32 values, V = 65: 15 us here (25 MB read, 25 MB of chunks' tables
// written) and 5 for their sum, where sorting and adding up took 30; bound by the chain of
// reads and writes of LDS that a column's tokens make.
//
// Small tables under many tokens: a workgroup holds a column slice of the whole table in
// LDS, a column a thread, and adds a chunk of the tokens to it one after another; a
// second launch adds the chunks' tables up in order.  Nothing is sorted.
template <typename T>
__global__ __launch_bounds__(512) void table_kernel(const GradArgs a, int chunk, float* __restrict__ part) {
  extern __shared__ float tab[];  // [V + 1][columns]
  const int W = blockDim.x, c = blockIdx.y * W + threadIdx.x, V = (int)a.V;
  const int i0 = blockIdx.x * chunk, i1 = (int)min<int64_t>(a.n, (int64_t)i0 + chunk);
  float* col = tab + threadIdx.x;
#pragma unroll 8
  for (int v = 0; v <= V; ++v) col[v * W] = 0.f;
  // (a thread reads and writes its own column alone: no barrier)
  const T* g = static_cast<const T*>(a.g) + min(c, a.C - 1);
  // Eight tokens at a time: their rows' sums are read at once (one after another they
  // wait 200 cycles each), a row that comes twice takes the sum of the time before, and
  // the last one to write it has it all.  Tokens that are none go to a row behind the
  // table.
  constexpr int N = 8;
  const int lane = threadIdx.x & 63;
  for (int b = i0; b < i1; b += 64) {
    const int64_t v = a.ids[min(b + lane, i1 - 1)];
    const int ids = b + lane < i1 && (uint64_t)v < (uint64_t)V ? (int)v : V;
    const int count = min(64, i1 - b);
    float all[64];  // requested at once: one wait for memory
#pragma unroll
    for (int k = 0; k < 64; ++k) all[k] = Elem<T>::to_f(g[(int64_t)(b + min(k, count - 1)) * a.ldg]);
#pragma unroll
    for (int k = 0; k < 64; ++k) asm volatile("" : "+v"(all[k]));  // (the loads stay where they are)
#pragma unroll
    for (int k0 = 0; k0 < 64; k0 += N) {
      if (k0 >= count) break;
      float x[N], t[N];
      int id[N];
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = all[k0 + k];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        id[k] = __builtin_amdgcn_readlane(ids, k0 + k);
        t[k] = col[id[k] * W];
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
#pragma unroll
        for (int m = 0; m < k; ++m) {
          float before = t[m];
          asm("" : "+v"(before));  // a plain select; from an array the compiler makes an index
          t[k] = id[m] == id[k] ? before : t[k];
        }
        t[k] += x[k];
      }
#pragma unroll
      for (int k = 0; k < N; ++k) col[id[k] * W] = t[k];
    }
  }
  if (c >= a.C) return;
  float* out = part + (int64_t)blockIdx.x * V * a.C + c;
#pragma unroll 8
  for (int v = 0; v < V; ++v) out[(int64_t)v * a.C] = col[v * W];
}

// dW (+)= scale times the sum of the chunks' tables: 64 values a workgroup, whose 16
// waves take contiguous runs of chunks
__global__ __launch_bounds__(64 * kWaves) void table_sum_kernel(const GradArgs a, int chunks, const float* __restrict__ part) {
  __shared__ float sums[kWaves][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, size = (int)a.V * a.C, e = blockIdx.x * 64 + lane;
  const int per = (chunks + kWaves - 1) / kWaves, b = w * per, end = min(chunks, b + per);
  float t = 0.f;
  if (e < size)
#pragma unroll 16
    for (int k = b; k < end; ++k) t += part[(int64_t)k * size + e];
  sums[w][lane] = t;
  __syncthreads();
  if (w || e >= size) return;
#pragma unroll
  for (int k = 1; k < kWaves; ++k) t += sums[k][lane];
  float* p = a.dw + (int64_t)(e / a.C) * a.lddw + e % a.C;
  *p = a.accumulate ? *p + a.scale * t : a.scale * t;
}

// (a launch has fewer than 2^32 threads: 1024 for kMaxRows rows of the table)
constexpr int64_t kMaxTable = (1LL << 31) - 2 * kMaxRows;

bool known(int dtype) { return dtype == MTX_F32 || dtype == MTX_BF16; }

// whether rows of C values at p, ld values apart, are whole 16-byte vectors of vec
// values each
bool whole(const void* p, int64_t ld, int C, int vec, int size) {
  return C % vec == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * size % 16 == 0;
}

// lanes per row for rows of nv vectors: the power of two from 8 to 64 that holds them
int lanes(int nv) {
  int l = 8;
  while (l < 64 && l < nv) l *= 2;
  return l;
}

template <typename T, typename O>
int lookup(const void* w, int64_t ldw, int64_t V, const int64_t* ids, int64_t n, int C, float scale, void* out,
           int64_t ldo, hipStream_t st) {
  constexpr int kVec = sizeof(T) + sizeof(O) == 8 ? 4 : 8;
  const bool vec = whole(w, ldw, C, kVec, sizeof(T)) && whole(out, ldo, C, kVec, sizeof(O));
  const int lpr = lanes(vec ? C / kVec : C);
  const int64_t rows = 256 / lpr * kLookRows;
  const unsigned blocks = (unsigned)std::min<int64_t>((n + rows - 1) / rows, 1 << 20);
  const unsigned slices = std::min<unsigned>(cdiv(vec ? C / kVec : C, lpr), std::max(1u, 512 / blocks));
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks, slices), dim3(256), 0, st, static_cast<const T*>(w), ldw, V, ids, n, C,
                       scale, static_cast<O*>(out), ldo);
  };
  switch ((vec ? 100 : 0) + lpr) {
    case 108: go(lookup_kernel<T, O, kVec, 8>); break;
    case 116: go(lookup_kernel<T, O, kVec, 16>); break;
    case 132: go(lookup_kernel<T, O, kVec, 32>); break;
    case 164: go(lookup_kernel<T, O, kVec, 64>); break;
    case 8: go(lookup_kernel<T, O, 1, 8>); break;
    case 16: go(lookup_kernel<T, O, 1, 16>); break;
    case 32: go(lookup_kernel<T, O, 1, 32>); break;
    default: go(lookup_kernel<T, O, 1, 64>); break;
  }
  MTX_LAUNCHED();
  return MTX_OK;
}

// How a gradient is worked out, its workspace's tables and size.
struct Plan {
  int R;           // table rows a sorting workgroup
  unsigned sorts;  // sorting workgroups
  bool small, table;
  int width, chunk, chunks;  // table: columns a workgroup, tokens a chunk
  size_t span, order, key, starts, part, bytes;
};

Plan plan(int dtype, int64_t n, int64_t V, int C) {
  Plan p{};
  const int size = dtype == MTX_F32 ? 4 : 2;
  p.R = (int)std::min<int64_t>((V + 255) / 256, kMaxRows);
  p.sorts = (unsigned)((V + p.R - 1) / p.R);
  // Few tokens, as long as one workgroup may have to read all their rows, 64 vectors or
  // 256 values of each at a time (1024 tokens of 1856 fp32 values, 9 rows: 8.1 us here, 25
  // sorted; of 1024, all of one row: 16 and 18; 600 bf16 tokens of 4096, 5003 rows: 26 and
  // 30)
  p.small = n <= 1024 || (n <= kSmallTokens && n * C * size <= (1 << 20));
  if (p.small) return p;
  auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
  // Small tables (64 columns of V + 1 rows in 64 KB of LDS, at most kTableValues values)
  // under tokens enough for 64 chunks of half the table or more: a chunk has 64 or 128 tokens,
  // and more where the workgroups would be more than the chip holds at once, whose tables
  // would only be written and read again.  In us, here and sorted:
  //     V, C        tokens    fp32            bf16
  //     65, 384     32768     24.8   36.3     24.5   31.9
  //                 131072    64.6   111      62.3   94.7
  //                 1048576   388    884      372    742
  //     255, 128    131072    51.4   82.7     50.5   78.5
  //     128, 256    131072    55.6   92.6     50.5   86.5
  //     200, 200    131072    82     92       81     86
  //     255, 160    131072    111    86       110    83
  //     128, 1024   131072    220    195      220    129
  // (131072 tokens of 384, V = 65, took 109 with 64 a chunk, and a workspace of 204 MB
  // where 34 do now.)  2^22 tokens at most: a column's sum of a chunk is one chain.
  constexpr int64_t kTableValues = 36864;
  p.chunk = V <= 128 ? 64 : 128;
  p.table = V < 256 && n / p.chunk >= 64 && n <= ((int64_t)1 << 22) && V * C <= kTableValues;
  if (p.table) {
    p.width = (int)std::min<int64_t>(512, (65536 / 4 / (V + 1)) / 64 * 64);
    const int slices = cdiv(C, p.width);
    p.width = (cdiv(C, slices) + 63) / 64 * 64;
    // (256 compute units of 160 KB of LDS)
    const int64_t held = 256 * std::min<int64_t>(8, 163840 / ((V + 1) * p.width * 4));
    p.chunk = (int)std::max<int64_t>(p.chunk, (n * slices / held + 63) / 64 * 64);
    p.chunks = (int)((n + p.chunk - 1) / p.chunk);
    p.bytes = up((size_t)p.chunks * V * C * 4);
    return p;
  }
  p.span = 256;
  p.order = p.span + up((size_t)V * sizeof(uint2));
  p.key = p.order + up((size_t)n * 4);
  p.starts = p.key + up((size_t)n * 4);
  p.part = p.starts + up((size_t)(n + kPiece - 1) / kPiece * 4);
  p.bytes = p.part + up((size_t)((n + kPiece - 1) / kPiece) * 2 * C * 4);
  return p;
}

template <typename T>
int grad(GradArgs a, const Plan& p, char* ws, hipStream_t st) {
  constexpr int kVec = 16 / sizeof(T), kU = sizeof(T) == 4 ? 2 : 1;
  const bool vec = whole(a.g, a.ldg, a.C, kVec, sizeof(T)) && whole(a.dw, a.lddw, a.C, kVec, 4);
  if (p.small) {
    // columns beside each other too (600 bf16 tokens of 4096, 5003 rows: 26 us with up to
    // 2048 workgroups, 43 with 512)
    const int cols = vec ? 64 * kVec : 256;
    const dim3 grid(p.sorts, std::min<unsigned>(cdiv(a.C, cols), std::max(1u, 2048 / p.sorts))), block(64 * kWaves);
    if (vec) hipLaunchKernelGGL((small_kernel<T, kVec, 1>), grid, block, 0, st, a, p.R);
    else hipLaunchKernelGGL((small_kernel<T, 1, 4>), grid, block, 0, st, a, p.R);
    MTX_LAUNCHED();
    return MTX_OK;
  }
  if (p.table) {
    float* part = reinterpret_cast<float*>(ws);
    hipLaunchKernelGGL((table_kernel<T>), dim3(p.chunks, cdiv(a.C, p.width)), dim3(p.width),
                       (size_t)(a.V + 1) * p.width * sizeof(float), st, a, p.chunk, part);
    MTX_LAUNCHED();
    hipLaunchKernelGGL(table_sum_kernel, dim3(cdiv((int)(a.V * a.C), 64)), dim3(64 * kWaves), 0, st, a, p.chunks, part);
    MTX_LAUNCHED();
    return MTX_OK;
  }
  uint32_t* tokens = reinterpret_cast<uint32_t*>(ws);
  uint2* span = reinterpret_cast<uint2*>(ws + p.span);
  uint32_t* order = reinterpret_cast<uint32_t*>(ws + p.order);
  uint32_t* key = reinterpret_cast<uint32_t*>(ws + p.key);
  uint32_t* starts = reinterpret_cast<uint32_t*>(ws + p.starts);
  const SortArgs sa{a.ids, a.n, a.V, p.R, span, order, key, tokens, starts, a.accumulate ? nullptr : a.dw, a.lddw, a.C,
                    whole(a.dw, a.lddw, a.C, 4, 4)};
  hipLaunchKernelGGL(sort_kernel, dim3(p.sorts), dim3(64 * kWaves), (size_t)(kWaves + 1) * p.R * 4, st, sa);
  MTX_LAUNCHED();
  a.tokens = tokens;
  a.span = span;
  a.order = order;
  a.key = key;
  a.starts = starts;
  a.part = reinterpret_cast<float*>(ws + p.part);
  const int lpr = lanes(vec ? a.C / kVec : a.C);
  auto go = [&](auto kernel, int columns) {
    a.slices = (a.C + columns - 1) / columns;
    a.rows = lpr < 64 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(8, a.V * a.slices / 8192));
    const int64_t items = ((a.V + a.rows - 1) / a.rows + (a.n + kPiece - 1) / kPiece) * a.slices;
    const int64_t blocks = (items * lpr + 255) / 256;
    hipLaunchKernelGGL(kernel, dim3((unsigned)std::min<int64_t>(blocks, 1 << 23)), dim3(256), 0, st, a);
  };
  switch ((vec ? 100 : 0) + lpr) {
    case 108: go(add_kernel<T, kVec, 8, 1>, 8 * kVec); break;
    case 116: go(add_kernel<T, kVec, 16, 1>, 16 * kVec); break;
    case 132: go(add_kernel<T, kVec, 32, 1>, 32 * kVec); break;
    case 164: go(add_kernel<T, kVec, 64, kU>, 64 * kVec * kU); break;
    case 8: go(add_kernel<T, 1, 8, 1>, 8); break;
    case 16: go(add_kernel<T, 1, 16, 1>, 16); break;
    case 32: go(add_kernel<T, 1, 32, 1>, 32); break;
    default: go(add_kernel<T, 1, 64, 4>, 256); break;
  }
  MTX_LAUNCHED();
  const int64_t wgs = (a.n + kPiece * kWaves - 1) / (kPiece * kWaves);
  const int chunks = a.C <= 64 ? 1 : a.C <= 128 ? 2 : 4;
  hipLaunchKernelGGL(join_kernel, dim3((unsigned)std::min<int64_t>(wgs, 4096), std::min(cdiv(a.C, 64 * chunks), 64)),
                     dim3(64 * kWaves), 0, st, a, chunks);
  MTX_LAUNCHED();
  return MTX_OK;
}

}  // namespace
}  // namespace mtx

using namespace mtx;

extern "C" int mtx_embedding_lookup(int dtype, int out_dtype, const void* weight, int64_t ldw, int64_t V,
                                    const int64_t* ids, int64_t n, int C, float scale, void* out, int64_t ldo,
                                    void* stream) {
  if (!known(dtype) || !known(out_dtype)) return fail(MTX_ERR_DTYPE, "embedding_lookup: unsupported dtype");
  MTX_CHECK_SHAPE(n >= 0 && n < (1LL << 31) && V >= 1 && V < (1LL << 31) && C >= 1 && C <= (1 << 30),
                  "embedding_lookup: need 0 <= n < 2^31, 1 <= V < 2^31, 1 <= C <= 2^30");
  MTX_CHECK_ARG(ldw >= C && ldo >= C, "embedding_lookup: rows of weight or out overlap");
  if (n == 0) return MTX_OK;
  MTX_CHECK_ARG(weight && ids && out, "embedding_lookup: null pointer");
  MTX_CHECK_ARG(out != weight, "embedding_lookup: out is the table");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MTX_F32)
    return out_dtype == MTX_F32 ? lookup<float, float>(weight, ldw, V, ids, n, C, scale, out, ldo, st)
                                : lookup<float, bf16_t>(weight, ldw, V, ids, n, C, scale, out, ldo, st);
  return out_dtype == MTX_F32 ? lookup<bf16_t, float>(weight, ldw, V, ids, n, C, scale, out, ldo, st)
                              : lookup<bf16_t, bf16_t>(weight, ldw, V, ids, n, C, scale, out, ldo, st);
}

extern "C" size_t mtx_embedding_grad_workspace_bytes(int dtype, int64_t n, int64_t V, int C) {
  if (n < 0 || n >= (1LL << 31) || V < 1 || V > kMaxTable || C < 1) return 0;
  return plan(dtype, n, V, C).bytes;
}

extern "C" int mtx_embedding_grad(int dtype, const int64_t* ids, int64_t n, const void* grad_, int64_t ldg, float scale,
                                  float* dweight, int64_t lddw, int64_t V, int C, int accumulate, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (!known(dtype)) return fail(MTX_ERR_DTYPE, "embedding_grad: unsupported dtype %d", dtype);
  MTX_CHECK_SHAPE(n >= 0 && n < (1LL << 31) && V >= 1 && V <= kMaxTable && C >= 1 && C <= (1 << 30),
                  "embedding_grad: need 0 <= n < 2^31, 1 <= V <= 2^31 - 1024, 1 <= C <= 2^30");
  MTX_CHECK_ARG(lddw >= C && (n == 0 || ldg >= C), "embedding_grad: rows of grad or dweight overlap");
  MTX_CHECK_ARG(dweight && (n == 0 || (ids && grad_)), "embedding_grad: null pointer");
  const Plan p = plan(dtype, n, V, C);
  MTX_CHECK_ARG(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0),
                "embedding_grad: workspace of %zu bytes, need %zu aligned to 256", workspace_bytes, p.bytes);
  MTX_CHECK_ARG(n == 0 || dweight != grad_, "embedding_grad: dweight is grad");
  GradArgs a{};
  a.ids = ids;
  a.g = grad_;
  a.ldg = ldg;
  a.scale = scale;
  a.dw = dweight;
  a.lddw = lddw;
  a.V = V;
  a.n = n;
  a.C = C;
  a.accumulate = accumulate ? 1 : 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MTX_F32 ? grad<float>(a, p, static_cast<char*>(workspace), st)
                          : grad<bf16_t>(a, p, static_cast<char*>(workspace), st);
}
