// Log probabilities of given tokens, the entropy of their distributions, the
// most likely alternatives, and the gradient of the first two, for gfx950.
//
// With x = scale * logits and lse = log sum exp x: logprob = x_t - lse,
// entropy = -sum p log p.  With e = exp(x - max), l = sum e it is computed as
// log l + (sum e (max - x)) / l: both terms are >= 0, so nothing cancels where
// the distribution is nearly certain.  All sums are fp32.  Long rows are bound by
// the memory (fp32: 5.2 to 6 TB/s; bf16, with ten instructions a value beside the
// loads, 4.2 to 4.7), short ones by the reductions and the ranking of a row's
// candidates.  The reference has log_softmax (functional.py:81-97)
// and samples from softmax (transformer.py:93-104).
#include "mtx_common.h"

#include <algorithm>
#include <cfloat>
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

// E values from any address that their type allows: global loads need no more
// alignment than that
template <typename T, int E>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned {
  T x[E];
};
template <int E>
__device__ __forceinline__ void load_values(const float* p, float (&x)[E]) {
  const auto u = *reinterpret_cast<const Unaligned<float, E>*>(p);
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = u.x[i];
}
template <int E>
__device__ __forceinline__ void load_values(const bf16_t* p, float (&x)[E]) {
  const auto u = *reinterpret_cast<const Unaligned<bf16_t, E>*>(p);
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = bf2f(u.x[i]);
}

// the same of the `left` values from p on, -inf behind them
template <int E, typename T>
__device__ __forceinline__ void load_left(const T* p, int left, float (&x)[E]) {
  if (left >= E) {
    load_values<E>(p, x);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = i < left ? Elem<T>::to_f(p[i]) : -INFINITY;
  }
}

// values of -inf add 0, not 0 * inf; NaN stays.  exp(kFarBelow * scale) is 0 for every
// scale that is taken, from kLeastScale on
constexpr float kFarBelow = -1e30f, kLeastScale = 1e-27f, kMostScale = 1e38f;
__device__ __forceinline__ float below(float d) { return __builtin_elementwise_maximum(d, kFarBelow); }

// The value of lane `lane ^ M` without the LDS pipe that a shuffle takes (a row of
// 65 logits needs some 40 of them): DPP within 16 lanes, for 16 and 32 the row
// swaps, of which pair() gives both partners' values to both, the lower lane's first
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int M>
__device__ __forceinline__ float lane_xor(float v) {
  if constexpr (M == 1) return dpp<0xB1>(v);          // quad_perm 1 0 3 2
  else if constexpr (M == 2) return dpp<0x4E>(v);     // quad_perm 2 3 0 1
  else if constexpr (M == 4) return dpp<0x1B>(dpp<0x141>(v));  // mirror of 8, then of 4
  else return dpp<0x128>(v);                          // 8: rotation of 16 by 8
}
template <int M>
__device__ __forceinline__ void pair(float v, float& a, float& b) {
  const uint32_t u = __float_as_uint(v);
  if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
  }
}
template <int N, typename F>
__device__ __forceinline__ float all_lanes(float v, F f) {  // over groups of N >= 16 lanes
  v = f(v, lane_xor<1>(v));
  v = f(v, lane_xor<2>(v));
  v = f(v, lane_xor<4>(v));
  v = f(v, lane_xor<8>(v));
  float a, b;
  if constexpr (N >= 32) {
    pair<16>(v, a, b);
    v = f(a, b);
  }
  if constexpr (N >= 64) {
    pair<32>(v, a, b);
    v = f(a, b);
  }
  return v;
}
template <int N = 64>
__device__ __forceinline__ float all_sum(float v) {
  return all_lanes<N>(v, [](float a, float b) { return a + b; });
}
template <int N = 64>
__device__ __forceinline__ float all_max(float v) {
  return all_lanes<N>(v, [](float a, float b) { return fmaxf(a, b); });
}

// one step of a bitonic network: the larger of lanes l and l ^ M to the lower lane,
// or, where `up`, to the upper one
template <int M>
__device__ __forceinline__ float exchange(float v, int lane, bool up) {
  float a = v, b;
  if constexpr (M >= 16) pair<M>(v, a, b);
  else b = lane_xor<M>(v);
  return ((lane & M) != 0) == up ? fmaxf(a, b) : fminf(a, b);
}
template <int M>
__device__ __forceinline__ float bitonic(float v, int lane, bool up) {
  v = exchange<M>(v, lane, up);
  if constexpr (M > 1) v = bitonic<M / 2>(v, lane, up);
  return v;
}
// N values of N lanes, largest in the first
template <int N>
__device__ __forceinline__ float lanes_sort(float v, int lane) {
  v = bitonic<1>(v, lane, lane & 2);
  v = bitonic<2>(v, lane, lane & 4);
  v = bitonic<4>(v, lane, lane & 8);
  v = bitonic<8>(v, lane, N > 16 && (lane & 16));
  if constexpr (N >= 32) v = bitonic<16>(v, lane, N > 32 && (lane & 32));
  if constexpr (N >= 64) v = bitonic<32>(v, lane, false);
  return v;
}
// the 64 largest of two sorted waves' values, sorted; w is read backwards
__device__ __forceinline__ float wave_merge(float v, float w_backwards, int lane) {
  return bitonic<32>(fmaxf(v, w_backwards), lane, false);
}

__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

// A row's outputs but the alternatives, by one thread: maximum m (at least
// -FLT_MAX), sums l of exp((x - m) scale) and t of that times (x - m)
template <typename T>
__device__ __forceinline__ void row_result(const LpArgs& a, int64_t r, const T* x, float m, float l, float t) {
  const float logl = logf(l);
  const int64_t k = a.tok[r];
  float lp = 0.f;
  if (k >= 0 && k < a.V) lp = l == 0.f ? -INFINITY : fmaf(Elem<T>::to_f(x[k]) - m, a.scale, -logl);
  a.logprob[r] = lp;
  a.lse[r] = l == 0.f ? -INFINITY : fmaf(m, a.scale, logl);
  a.entropy[r] = l == 0.f ? 0.f : fmaf(-t / l, a.scale, logl);
}
__device__ __forceinline__ void put_top(const LpArgs& a, int64_t r, int rank, uint64_t key, float v, float m, float l) {
  a.ids[r * a.top + rank] = (int)~(uint32_t)key;
  a.tops[r * a.top + rank] = l == 0.f ? -INFINITY : fmaf(v - m, a.scale, -logf(l));
}

// Alternatives of a row: the top-th largest of the lanes' (threads') largest
// values bounds the wanted ones from below, so only values from that bound on,
// about `top` of them, are collected and ranked by counting.  Rows that hold NaN,
// and rows where too many values reach the bound (ties), take `top` rounds over
// all values instead.

// ---- rows of up to LPR VPL values: LPR lanes each, the row in registers, 64 / LPR
// rows a wave (16384 rows of 65: one row a wave would spend its time on reductions
// over lanes that hold one value) ----
constexpr int kSmallCap = 256;  // candidates a row
template <typename T, int LPR, int VPL>
__global__ __launch_bounds__(256) void logprobs_small_kernel(const LpArgs a, int64_t rows) {
  constexpr int RPW = 64 / LPR, CAP = RPW == 1 ? kSmallCap : LPR * VPL;
  __shared__ uint64_t cands[4 * RPW][CAP];
  const int lane = threadIdx.x & 63, sub = lane % LPR, row = threadIdx.x / LPR;
  const int64_t r = (int64_t)blockIdx.x * (4 * RPW) + row;
  const bool in = r < rows;
  const T* __restrict__ x = static_cast<const T*>(a.x) + (in ? r : 0) * a.ld;
  float v[VPL], best = -INFINITY;
#pragma unroll
  for (int i = 0; i < VPL; ++i) v[i] = sub + LPR * i < a.V ? Elem<T>::to_f(x[sub + LPR * i]) : -INFINITY;
#pragma unroll
  for (int i = 0; i < VPL; ++i) best = fmaxf(best, v[i]);
  const float m = fmaxf(all_max<LPR>(best), -FLT_MAX), c = a.scale * kLog2e;
  float l = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const float d = below(v[i] - m), e = __builtin_amdgcn_exp2f(d * c);
    l += e;
    t = fmaf(e, d, t);
  }
  l = all_sum<LPR>(l);
  t = all_sum<LPR>(t);
  if (sub == 0 && in) row_result(a, r, x, m, l, t);
  if (a.top == 0) return;
  uint64_t* buf = cands[row];
  int n = 0;
  // the top-th largest of the lanes' largest values; all values where there are
  // fewer lanes than that
  float bound = -INFINITY;
  if (a.top <= LPR) bound = __shfl(lanes_sort<LPR>(best, lane), (lane & ~(LPR - 1)) + a.top - 1, 64);
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const bool good = v[i] >= bound && sub + LPR * i < a.V;
    const uint64_t mask = __ballot(good) >> (lane & ~(LPR - 1)) & (LPR == 64 ? ~0ull : (1ull << LPR % 64) - 1);
    const int at = n + __popcll(mask & ((1ull << sub) - 1));
    if (good && at < CAP) buf[at] = rank_key(v[i], sub + LPR * i);
    n += __popcll(mask);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const bool slow = l != l || n < a.top || n > CAP;  // alike in a row's lanes
  if (!slow && in) {
    for (int i = sub; i < n; i += LPR) {
      const uint64_t mine = buf[i];
      int rank = 0;
      for (int k = 0; k < n; ++k) rank += buf[k] > mine;
      if (rank < a.top) put_top(a, r, rank, mine, key_value(mine), m, l);
    }
  }
  if (!__ballot(slow)) return;
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const uint64_t key = rank_key(v[i], sub + LPR * i);
      if (sub + LPR * i < a.V && (key < last || k == 0) && key > mine) mine = key;
    }
#pragma unroll
    for (int s = LPR / 2; s >= 1; s >>= 1) {
      const uint64_t o = __shfl_xor(mine, s, 64);
      mine = o > mine ? o : mine;
    }
    last = mine;
    if (sub == 0 && slow && in) put_top(a, r, k, last, Elem<T>::to_f(x[(int)~(uint32_t)last]), m, l);
  }
}

// ---- longer rows: a workgroup of NT threads each, E values (16 bytes) a load, U of
// them in flight.  WHOLE: the row fits U loads a thread and stays in registers;
// otherwise one pass with the running maximum and sums, and what is collected for
// the alternatives is read again ----
template <typename T, int NT, int U, bool WHOLE>
__global__ __launch_bounds__(NT) void logprobs_kernel(const LpArgs a) {
  // kCap candidates: with 1024 LDS would leave half the place for single waves (16384 x
  // 700 bf16 20.3 us, 24.7)
  constexpr int E = Elem<T>::kVec, W = NT / 64, STEP = NT * E, kCap = NT == 64 ? 256 : 1024;
  __shared__ uint64_t cands[kCap];
  __shared__ float sorted[W][64], red[3][W];
  __shared__ int count;
  __shared__ uint64_t bests[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x;
  const T* __restrict__ row = static_cast<const T*>(a.x) + r * a.ld;
  // loads at odd bf16 addresses are slower than at even ones (2048 x 50021: 54 us, 47): the
  // first value of such a row is thread 0's
  const int odd = !WHOLE && sizeof(T) == 2 ? (int)((uintptr_t)row >> 1 & 1) : 0, V = a.V - odd;
  const T* __restrict__ x = row + odd;
  const float head = odd && tid == 0 ? Elem<T>::to_f(*row) : -INFINITY;
  const float c = a.scale * kLog2e;
  float v[U][E], m = -FLT_MAX, l = 0.f, t = 0.f;
  auto raise = [&](float top) {  // the sums relative to a larger maximum
    const float n = fmaxf(m, top), d = fmaxf(m - n, kFarBelow), f = __builtin_amdgcn_exp2f(d * c);
    t = f * fmaf(l, d, t);
    l *= f;
    m = n;
  };
  // whether the wave has values in round u of a whole row
  const int first = __builtin_amdgcn_readfirstlane(wave) * 64 * E;
  auto some = [&](int u) { return !WHOLE || first + u * STEP < V; };
  auto largest = [&] {
    float top = WHOLE ? -INFINITY : v[0][0];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (some(u)) {
#pragma unroll
        for (int e = 0; e < E; ++e) top = fmaxf(top, v[u][e]);
      }
    return top;
  };
  auto add = [&] {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (some(u)) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float d = below(v[u][e] - m), p = __builtin_amdgcn_exp2f(d * c);
          l += p;
          t = fmaf(p, d, t);
        }
      }
  };
  int i = tid * E;
  if (!WHOLE) {
    for (; i + (U - 1) * STEP + E <= V; i += U * STEP) {
#pragma unroll
      for (int u = 0; u < U; ++u) load_values<E>(x + i + u * STEP, v[u]);
      raise(largest());
      add();
    }
  }
  if (WHOLE || i < V) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (some(u)) load_left<E>(x + i + u * STEP, V - i - u * STEP, v[u]);
    if (WHOLE) {
      m = fmaxf(m, largest());
    } else {
      raise(largest());
      add();
    }
  }
  if (odd && tid == 0) {
    raise(head);
    const float d = below(head - m), p = __builtin_amdgcn_exp2f(d * c);
    l += p;
    t = fmaf(p, d, t);
  }
  const float mine = m;  // the thread's largest value
  if (WHOLE) {
    m = all_max(m);
    if (W > 1) {
      if (lane == 0) red[0][wave] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W; ++w) m = fmaxf(m, red[0][w]);
    }
    add();
  } else {
    raise(all_max(m));
  }
  l = all_sum(l);
  t = all_sum(t);
  if (lane == 0) {
    if (!WHOLE) red[0][wave] = m;
    red[1][wave] = l, red[2][wave] = t;
  }
  if (a.top) {
    sorted[wave][lane] = lanes_sort<64>(mine, lane);
    if (tid == 0) count = 0;
  }
  __syncthreads();
  // every thread joins the waves' sums in the same order
  if (W > 1) {
    const int w0 = lane % W;
    float all = m;
    if (!WHOLE) {
      m = red[0][w0], all = red[0][0];
#pragma unroll
      for (int w = 1; w < W; ++w) all = fmaxf(all, red[0][w]);
    }
    l = red[1][w0], t = red[2][w0];
    if (!WHOLE) raise(all);
#pragma unroll
    for (int s = 1; s < W; s <<= 1) {
      l += __shfl_xor(l, s, 64);
      t += __shfl_xor(t, s, 64);
    }
  }
  if (tid == 0) row_result(a, r, row, m, l, t);
  if (a.top == 0) return;
#pragma unroll
  for (int s = 1; s < W; s <<= 1) {
    if (wave % (2 * s) == 0) sorted[wave][lane] = wave_merge(sorted[wave][lane], sorted[wave + s][63 - lane], lane);
    __syncthreads();
  }
  const float bound = sorted[0][a.top - 1];
  auto collect = [&](const float (&w)[E], int at) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (w[e] >= bound && at + e < V) {
        const int k = atomicAdd(&count, 1);
        if (k < kCap) cands[k] = rank_key(w[e], at + e + odd);
      }
  };
  const bool look = l == l && mine >= bound;
  if (WHOLE) {
    if (look) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (some(u)) collect(v[u], i + u * STEP);
    }
  } else {
    // a thread's values are read again by lanes of its wave, a load each, and where
    // they are few those of several threads at once (8 x 20000 bf16 7.6 us, one thread
    // at a time 9.3)
    int per = 64;
    while (per > 8 && (per / 2) * STEP >= V) per /= 2;
    for (uint64_t mask = __ballot(look); mask;) {
      int from = -1;
      for (int k = 0; k < 64 && mask; k += per, mask &= mask - 1)
        if (lane >= k && lane < k + per) from = __ffsll((unsigned long long)mask) - 1;
      if (from < 0) continue;
      for (int j = (wave * 64 + from) * E + (lane & (per - 1)) * STEP; j < V; j += per * STEP) {
        float w[E];
        load_left<E>(x + j, V - j, w);
        collect(w, j);
      }
    }
    if (odd && tid == 0 && look && head >= bound) {
      const int k = atomicAdd(&count, 1);
      if (k < kCap) cands[k] = rank_key(head, 0);
    }
  }
  __syncthreads();
  const int n = count;
  if (n >= a.top && n <= kCap) {
    for (int k = tid; k < n; k += NT) {
      const uint64_t key = cands[k];
      int rank = 0;
      for (int o = 0; o < n; ++o) rank += cands[o] > key;
      if (rank < a.top) put_top(a, r, rank, key, key_value(key), m, l);
    }
    return;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t best = 0;
    for (int j = tid; j < a.V; j += NT) {
      const uint64_t key = rank_key(Elem<T>::to_f(row[j]), j);
      if ((key < last || k == 0) && key > best) best = key;
    }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) {
      const uint64_t o = __shfl_xor(best, s, 64);
      best = o > best ? o : best;
    }
    __syncthreads();
    if (lane == 0) bests[wave] = best;
    __syncthreads();
    last = bests[0];
#pragma unroll
    for (int w = 1; w < W; ++w) last = bests[w] > last ? bests[w] : last;
    if (tid == 0) put_top(a, r, k, last, Elem<T>::to_f(row[(int)~(uint32_t)last]), m, l);
  }
}

// The gradient reads the logits once more and writes as many fp32 values: bound by
// the memory, 4096 x 50021 fp32 in 313 us (5.2 TB/s; a large copy reaches 5.2).  The
// forward's pass over the same logits takes 137 us (6.0 TB/s) by itself, 179 behind
// the gradient's, whose last writes are then still on their way.
struct LpBwdArgs {
  const void* x;
  int64_t ld;
  const int64_t* tok;
  const float* lse;
  const float* entropy;
  const float* g;
  const float* gh;
  float* dx;
  int64_t ldd, rows;
  int V, per;  // threads per row
  float scale;
  int accumulate;
};

// dx = p (A + B log p) with A = -scale (g + gh H), B = -scale gh, and scale g at
// the token: one pass, 4 values a load and store, up to kUnroll of them a thread.
// log p is taken for kLeastLog at least, whose p is 0 already, so that B log p does
// not overflow where p is 0 (0 * inf)
constexpr int kUnroll = 4;
constexpr float kLeastLog = -128.f;
template <typename T>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(const LpBwdArgs a) {
  const int64_t r = (int64_t)blockIdx.x * (256 / a.per) + threadIdx.x / a.per;
  if (r >= a.rows) return;
  const T* __restrict__ x = static_cast<const T*>(a.x) + r * a.ld;
  float* __restrict__ o = a.dx + r * a.ldd;
  const float lse = a.lse[r];
  const int64_t tok = a.tok[r];
  const bool none = lse == -INFINITY;
  const float g = a.g != nullptr && tok >= 0 && tok < a.V && !none ? a.g[r] : 0.f;
  const float gh = a.gh != nullptr && !none ? a.gh[r] : 0.f;
  const float A = -a.scale * fmaf(gh, none ? 0.f : a.entropy[r], g), Bf = -a.scale * gh, own = a.scale * g;
  const float off = none ? 0.f : lse;
  const int step = 4 * a.per;
  const int i0 = (int)(blockIdx.y * kUnroll * step + 4 * (threadIdx.x % a.per));
  float v[kUnroll][4];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int i = i0 + u * step;
    if (i + 4 <= a.V) {
      load_values<4>(x + i, v[u]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[u][e] = i + e < a.V ? Elem<T>::to_f(x[i + e]) : 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int i = i0 + u * step;
    if (i >= a.V) break;
    float d[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float lp = __builtin_elementwise_maximum(fmaf(v[u][e], a.scale, -off), kLeastLog);
      const float p = __builtin_amdgcn_exp2f(lp * kLog2e);
      d[e] = p * fmaf(Bf, lp, A);
      if (i + e == tok) d[e] += own;
    }
    if (i + 4 <= a.V) {
      auto* q = reinterpret_cast<Unaligned<float, 4>*>(o + i);
      Unaligned<float, 4> w;
      if (a.accumulate) {
        w = *q;
#pragma unroll
        for (int e = 0; e < 4; ++e) w.x[e] += d[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) w.x[e] = d[e];
      }
      *q = w;
    } else {
      for (int e = 0; e < 4 && i + e < a.V; ++e) o[i + e] = a.accumulate ? o[i + e] + d[e] : d[e];
    }
  }
}

int check_rows(int dtype, int64_t rows, int V, const void* logits, int64_t ld, const int64_t* tokens, float scale) {
  if (dtype != MTX_F32 && dtype != MTX_BF16) return fail(MTX_ERR_DTYPE, "unsupported dtype %d", dtype);
  // a launch's threads, up to 512 a row, are counted in 32 bits
  MTX_CHECK_SHAPE(rows >= 1 && rows < (1 << 23) && V >= 1 && V <= (1 << 27),
                  "token_logprobs: needs 1 <= rows < 2^23 and 1 <= V <= 2^27 (got %lld, %d)", (long long)rows, V);
  MTX_CHECK_ARG(logits != nullptr && tokens != nullptr, "logits, tokens: null pointer");
  MTX_CHECK_ARG(((uintptr_t)logits & (dtype == MTX_F32 ? 3u : 1u)) == 0, "logits: pointer must be aligned to its type");
  MTX_CHECK_ARG(ld >= V || (rows == 1 && ld >= 0), "logits: row stride %lld < V=%d", (long long)ld, V);
  MTX_CHECK_ARG(scale >= kLeastScale && scale <= kMostScale, "scale=%g must be between 1e-27 and 1e38", scale);
  return MTX_OK;
}

constexpr int kMostTop = 64;

template <typename T>
int launch_logprobs(const LpArgs& a, int64_t rows, hipStream_t st) {
  constexpr int E = Elem<T>::kVec;
  // measured with 10 alternatives, us: 16384 x 65 (5 alternatives) 5.5 by 16 lanes a
  // row, 12.3 by 64; 16384 x 1500 fp32 26 whole in a wave, 43 in one pass, 60 by 256
  // threads; 8192 x 3000 fp32 29 whole in 256 threads, 35 in one pass; 4096 x 9000 32
  // by 256 threads, 39 by 512, 64 by 1024; 2048 x 50021 fp32 88 by 256, 79 by 512;
  // 8 x 50021 bf16 11.4 by 256, 9.1 by 512, 10.6 by 1024
#define SMALL(LPR, VPL)                                                                                        \
  hipLaunchKernelGGL((logprobs_small_kernel<T, LPR, VPL>), dim3((unsigned)((rows * LPR + 255) / 256)), dim3(256), 0, \
                     st, a, rows)
  if (a.V <= 16) SMALL(16, 1);
  else if (a.V <= 48) SMALL(16, 3);
  else if (a.V <= 80) SMALL(16, 5);
  else if (a.V <= 128) SMALL(16, 8);
  else if (a.V <= 256) SMALL(32, 8);
  else if (a.V <= 512) SMALL(64, 8);
#define ROW(NT, U, WHOLE) \
  hipLaunchKernelGGL((logprobs_kernel<T, NT, U, WHOLE>), dim3((unsigned)rows), dim3(NT), 0, st, a)
  else if (sizeof(T) == 2 && a.V <= 64 * E * 2) ROW(64, sizeof(T) == 2 ? 2 : 4, true);
  else if (a.V <= 64 * E * 4) ROW(64, 4, true);
  else if (a.V <= 64 * E * 8) ROW(64, 8, true);
  else if (a.V <= 256 * E * 4) ROW(256, 4, true);
  else if (rows >= 256 && a.V * sizeof(T) <= (128 << 10)) ROW(256, 4, false);
  else ROW(512, 4, false);
#undef ROW
#undef SMALL
  MTX_LAUNCHED();
  return MTX_OK;
}

}  // namespace
}  // namespace mtx

using namespace mtx;

extern "C" int mtx_token_logprobs(int dtype, int64_t rows, int V, const void* logits, int64_t ld,
                                  const int64_t* tokens, float scale, float* logprob, float* lse, float* entropy,
                                  int top, int64_t* top_ids, float* top_logprobs, void*, size_t, void* stream) {
  int rc;
  if ((rc = check_rows(dtype, rows, V, logits, ld, tokens, scale))) return rc;
  MTX_CHECK_ARG(logprob && lse && entropy, "logprob, lse, entropy: null pointer");
  MTX_CHECK_SHAPE(top >= 0 && top <= kMostTop && top <= V, "top=%d alternatives of %d tokens (at most %d)", top, V,
                  kMostTop);
  MTX_CHECK_ARG(top == 0 || (top_ids && top_logprobs), "top_ids, top_logprobs: null pointer");
  LpArgs a{logits, ld, tokens, logprob, lse, entropy, top_ids, top_logprobs, V, top, scale};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MTX_F32 ? launch_logprobs<float>(a, rows, st) : launch_logprobs<bf16_t>(a, rows, st);
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
  int per = 16;
  while (per < 256 && per * 4 < V) per *= 2;
  LpBwdArgs a{logits, ld, tokens, lse, entropy, g_logprob, g_entropy, dlogits, ldd, rows, V, per, scale, accumulate};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t groups = (rows + 256 / per - 1) / (256 / per);
  const dim3 grid((unsigned)groups, (unsigned)cdiv(V, 4 * per * kUnroll));
  if (dtype == MTX_F32) hipLaunchKernelGGL(logprobs_bwd_kernel<float>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(logprobs_bwd_kernel<bf16_t>, grid, dim3(256), 0, st, a);
  MTX_LAUNCHED();
  return MTX_OK;
}
