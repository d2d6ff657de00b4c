// The projection with its cross entropy and gradients for many rows and vocabularies of at
// most kNarrowV entries, as character models have: z = x W + b, dz = (softmax(z) - onehot) /
// labels, dx = dz W^T, dW = x^T dz, db = column sums of dz.
//
// A wave takes 16 rows and all of the vocabulary, so that a row's logits, its softmax and
// its gradient stay in the registers of 16 lanes: x is read once and dx written once by
// one launch, and only dz (for the second launch, dW) passes through memory.  All products
// are fp32 ones (mfma_f32_16x16x4f32): nothing of the operands is cut.  (16384, 384) x
// (384, 65), fp32: 30 us (16 of them before dx), dW 21, and 57.5 with the count and the
// sums, where products, softmax and gradients in five launches took 91.  Bound by the
// matrix cores, half busy (7 us a product at their fp32 rate): a SIMD has but one wave.
// A wave's rows are worked on one chunk of k after another, so few rows of many k are slow:
// 300 x 2048 takes 124 us, the general way 50.
#include "narrow_xent.h"

#include <algorithm>
#include <type_traits>

namespace mtx {
namespace {

constexpr int kRows = 64;  // rows a workgroup, 16 a wave

// Four k of a row, as one request
template <typename T>
struct Four;
template <>
struct Four<float> {
  typedef f32x4 type;
  __device__ __forceinline__ static f32x4 to_f(f32x4 v) { return v; }
};
template <>
struct Four<bf16_t> {
  typedef uint2 type;
  __device__ __forceinline__ static f32x4 to_f(uint2 v) {
    return f32x4{__builtin_bit_cast(float, v.x << 16), __builtin_bit_cast(float, v.x & 0xffff0000u),
                 __builtin_bit_cast(float, v.y << 16), __builtin_bit_cast(float, v.y & 0xffff0000u)};
  }
};

constexpr uint32_t kNone = 0xfffffff0u;  // an offset behind every operand's end
template <typename T>
__device__ __forceinline__ T load_one(__amdgpu_buffer_rsrc_t rs, uint32_t off) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(rs, (int)off, 0, 0));
  else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(rs, (int)off, 0, 0));
}

// memory from p on, `bytes` of it (the same for all lanes: scalar registers hold it)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t memory(const void* p, int64_t bytes) {
  const uint64_t from = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)from), hi = __builtin_amdgcn_readfirstlane((uint32_t)(from >> 32));
  const uint32_t size = __builtin_amdgcn_readfirstlane(bytes > 0xffffff00ll ? 0xffffff00u : bytes < 0 ? 0u : (uint32_t)bytes);
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)hi << 32 | lo), (short)0, (int)size, 0x00020000);
}

// f(x of another lane) until f has seen all 16 lanes that have a row
template <typename F>
__device__ __forceinline__ void row16(F f) {
  f([](float x) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xb1, 0xf, 0xf, true)); });   // lane ^ 1
  f([](float x) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4e, 0xf, 0xf, true)); });   // lane ^ 2
  f([](float x) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xf, 0xf, true)); });  // 7 - lane
  f([](float x) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x140, 0xf, 0xf, true)); });  // 15 - lane
}

// n products, and what else stands beside them, by turns: an instruction that does not need
// the matrix core is issued while it is busy
__device__ __forceinline__ void interleave(int n) {
#pragma unroll
  for (int i = 0; i < n; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // product
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
    __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // LDS write
    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // memory read
    __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);  // vector arithmetic
  }
  __builtin_amdgcn_sched_barrier(0);
}

// NT: tiles of 16 vocabulary entries.  VEC: x's rows are whole groups of four k that one
// request can take.
//
// W passes through LDS in chunks of KC k, twice: forward for z, backward for dx (whose
// first two chunks are there still).  A chunk's requests are under way while the one
// before is multiplied.  Rows of VS = 16 NT + 4 floats: the reads of W[k][v .. v + 15] for
// four k of a wave cover all banks, as do 16-byte reads of 16 rows.
//
// MFMA operands: lane l has row (or column) l % 16 and, of every 16 k, those from 4 (l / 16)
// on: step s of four multiplies the k = 4 (l / 16) + s of both operands.
template <typename T, int NT, bool VEC>
__global__ __launch_bounds__(256, 2) void narrow_kernel(const NarrowXent a) {
  constexpr int KC = NT <= 5 ? 64 : 32, VS = 16 * NT + 4, KT = KC / 16;
  constexpr int PER = KC * NT / 16;  // values of a chunk that a thread copies
  __shared__ float wt[2][KC * VS];
  __shared__ float dzs[4][16 * VS];
  typedef typename Four<T>::type V4;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int C = a.C, V = a.V, chunks = (C + KC - 1) / KC;
  const int row0 = blockIdx.x * kRows + 16 * w;
  const T* W = static_cast<const T*>(a.w);
  const T* x = static_cast<const T*>(a.x) + (int64_t)min(row0 + c, a.rows - 1) * a.ldx;
  const bool rowwise = a.swv == 1 && a.swc >= V;

  // A chunk's values: neighbouring threads' are neighbours in memory.  What lies behind
  // W's end, or gets an offset behind it, reads as 0.  Chunks that there are none of are
  // requested as well, of no bytes: were they left out by a branch, the compiler could not
  // count the requests in flight and would wait for all of them.
  uint32_t off[PER];
  int at[PER];
  auto places = [&](auto by_rows) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      constexpr int N = decltype(by_rows)::value ? 16 * NT : KC;
      const int e = threadIdx.x + 256 * i, k = decltype(by_rows)::value ? e / N : e % N,
                v = decltype(by_rows)::value ? e % N : e / N;
      off[i] = ((uint32_t)k * (uint32_t)a.swc + (uint32_t)v * (uint32_t)a.swv) * (uint32_t)sizeof(T);
      off[i] = v < V ? off[i] : kNone;
      at[i] = k * VS + v;
    }
  };
  if (rowwise) places(std::true_type());
  else places(std::false_type());
  const int64_t size = (C - 1) * a.swc + (V - 1) * a.swv + 1;
  // (two chunks' requests are under way: sets of registers by turns)
  T wr[2][PER];
  auto fetch = [&](int ch, T (&to)[PER], int i0, int i1) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int64_t left = size - (int64_t)ch * KC * a.swc;
    const auto rs = memory(W + (int64_t)ch * KC * a.swc, ch < 0 ? 0 : left * (int64_t)sizeof(T));
    // by columns, other entries' values lie behind the last k (256 is a multiple of KC)
    const uint32_t least = !rowwise && ch * KC + (int)threadIdx.x % KC >= C ? kNone : 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i >= i0 && i < i1) to[i] = load_one<T>(rs, max(off[i], least));
#endif
  };
  // (where there is no chunk to put, its place is that of dz, which comes later)
  auto put = [&](int ch, const T (&from)[PER], int i0, int i1) {
    float* to = ch < chunks ? wt[ch & 1] : dzs[0];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i >= i0 && i < i1) to[at[i]] = Elem<T>::to_f(from[i]);
  };
  V4 xr[2][KT];
  auto request = [&](int ch, V4 (&to)[KT], int j0, int j1) {
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      if (j < j0 || j >= j1) continue;
      const int k = ch * KC + 16 * j + 4 * g;
      if constexpr (VEC) {
        to[j] = *reinterpret_cast<const V4*>(x + min(k, C - 4));
      } else {
        T one[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) one[s] = x[min(k + s, C - 1)];
        __builtin_memcpy(&to[j], one, sizeof(V4));
      }
    }
  };

  int y[4];  // this lane's rows' labels; -1: none
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + 4 * g + i;
    const int64_t label = a.labels[min(row, a.rows - 1)];
    y[i] = row < a.rows && (uint64_t)label < (uint64_t)V ? (int)label : -1;
  }
  fetch(0, wr[0], 0, PER);
  request(0, xr[0], 0, KT);
  fetch(1, wr[1], 0, PER);
  request(1, xr[1], 0, KT);
  put(0, wr[0], 0, PER);
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = zero4();
  auto forward = [&](int ch, auto set) {
    constexpr int S = decltype(set)::value;
    f32x4 now[KT];
#pragma unroll
    for (int j = 0; j < KT; ++j) now[j] = Four<T>::to_f(xr[S][j]);
    if ((ch + 1) * KC > C)
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int s = 0; s < 4; ++s) now[j][s] = ch * KC + 16 * j + 4 * g + s < C ? now[j][s] : 0.f;
    __syncthreads();
    // the operands of 16 k are read while those before are multiplied
    const float* b = wt[ch & 1] + 4 * g * VS + c;
    float bv[2][4][NT];
    auto read = [&](int j) {
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int t = 0; t < NT; ++t) bv[j & 1][s][t] = b[(16 * j + s) * VS + 16 * t];
    };
    read(0);
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      if (j + 1 < KT) read(j + 1);
      // (the other buffer is free: all waves are past the chunk before)
      put(ch + 1, wr[1 - S], j * PER / KT, (j + 1) * PER / KT);
      fetch(ch + 2, wr[S], j * PER / KT, (j + 1) * PER / KT);
      request(ch + 2, xr[S], j, j + 1);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(now[j][s], bv[j & 1][s][t], acc[t], 0, 0, 0);
      interleave(4 * NT);
    }
  };
  constexpr std::integral_constant<int, 0> first;
  constexpr std::integral_constant<int, 1> second;
  int ch = 0;
  for (; ch + 1 < chunks; ch += 2) {
    forward(ch, first);
    forward(ch + 1, second);
  }
  if (ch < chunks) forward(ch, first);
  __syncthreads();  // dzs is each wave's own from here on
  if (a.dx) {  // for the way back, which finds the last two chunks in LDS
    fetch(chunks - 3, wr[0], 0, PER);
    fetch(chunks - 4, wr[1], 0, PER);
  }

  // acc[t][i]: row row0 + 4 g + i, entry 16 t + c
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int v = 16 * t + c;
    const float bias = a.bias ? a.bias[min(v, V - 1)] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[t][i] = v < V ? acc[t][i] + bias : -INFINITY;
  }
  // the four rows side by side: their reductions do not wait for each other
  float m[4], sum[4], zy[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    zy[i] = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[i] = fmaxf(m[i], acc[t][i]);
      zy[i] = y[i] == 16 * t + c ? acc[t][i] : zy[i];  // one lane's
    }
  }
  row16([&](auto dpp) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = fmaxf(m[i], dpp(m[i]));
      zy[i] += dpp(zy[i]);
    }
  });
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // (the difference first: m log2(e) may be infinite for a finite m)
    const float from = m[i] == -INFINITY ? 0.f : m[i];
    sum[i] = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
      sum[i] += acc[t][i] = __builtin_amdgcn_exp2f((acc[t][i] - from) * kLog2e);
  }
  row16([&](auto dpp) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += dpp(sum[i]);
  });
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + 4 * g + i;
    if (c != i || row >= a.rows) continue;  // (a lane a row)
    const float l = logf(sum[i]);
    a.lse[row] = m[i] + l;
    a.row_loss[row] = y[i] < 0 ? 0.f : zy[i] == -INFINITY && m[i] == -INFINITY ? INFINITY : (m[i] - zy[i]) + l;
  }
  if (!a.dx && !a.dz) return;
  const float inv = *a.inv;
  float* mine = dzs[w];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = sum[i] == 0.f ? 0.f : 1.f / sum[i];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int v = 16 * t + c;
      acc[t][i] = y[i] >= 0 && v < V ? (acc[t][i] * f - (y[i] == v ? 1.f : 0.f)) * inv : 0.f;
      mine[(4 * g + i) * VS + v] = acc[t][i];
    }
  }
  if (a.dz)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + 4 * g + i;
      if (row >= a.rows) continue;
      float* p = a.dz + (int64_t)row * a.ldz + c;
#pragma unroll
      for (int t = 0; t < NT; ++t) p[16 * t] = acc[t][i];
    }
  if (!a.dx) return;

  // dx: this wave's dz as operands (its own writes, which need no barrier)
  f32x4 dv[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) dv[t] = *reinterpret_cast<const f32x4*>(mine + c * VS + 16 * t + 4 * g);
  uint32_t row_at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) row_at[i] = (uint32_t)(4 * g + i) * (uint32_t)a.lddx;
#if defined(__HIP_DEVICE_COMPILE__)
  const int size_x = sizeof(T) == 2 && a.dx_bf16 ? 2 : 4;
  const auto dxs = memory(static_cast<const char*>(a.dx) + row0 * a.lddx * size_x,
                          row0 < a.rows ? ((min(a.rows - row0, 16) - 1) * a.lddx + C) * size_x : 0);
#endif
  auto back = [&](int ch, auto set, auto refill) {
    constexpr int S = decltype(set)::value;
    __syncthreads();
    f32x4 out[KT];
#pragma unroll
    for (int j = 0; j < KT; ++j) out[j] = zero4();
    f32x4 bv[2][KT];
    auto read = [&](int t) {
#pragma unroll
      for (int j = 0; j < KT; ++j)
        bv[t & 1][j] = *reinterpret_cast<const f32x4*>(wt[ch & 1] + (16 * j + c) * VS + 16 * t + 4 * g);
    };
    read(0);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t + 1 < NT) read(t + 1);
      if constexpr (decltype(refill)::value) {
        // in place of the chunk after this one, whose turn is over
        put(ch - 1, wr[S], t * PER / NT, (t + 1) * PER / NT);
        fetch(ch - 3, wr[S], t * PER / NT, (t + 1) * PER / NT);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int j = 0; j < KT; ++j)
          out[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(dv[t][s], bv[t & 1][j][s], out[j], 0, 0, 0);
      interleave(4 * KT);
    }
#if defined(__HIP_DEVICE_COMPILE__)
    // (rows behind the last one and columns behind C get places behind the end)
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      const int k = ch * KC + 16 * j + c;
      const uint32_t least = k < C ? 0u : kNone;
      if (sizeof(T) == 2 && a.dx_bf16) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          __builtin_amdgcn_raw_buffer_store_b16(f2bf(out[j][i]), dxs, (int)max((row_at[i] + k) * 2u, least), 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(out[j][i]), dxs, (int)max((row_at[i] + k) * 4u, least), 0, 0);
      }
    }
#endif
  };
  back(chunks - 1, second, std::false_type());
  for (ch = chunks - 2; ch >= 1; ch -= 2) {
    back(ch, first, std::true_type());
    back(ch - 1, second, std::true_type());
  }
  if (ch == 0) back(0, first, std::true_type());
}

// Partial sums of dW over a range of rows: a workgroup takes 64 columns of x, a wave a
// quarter of the range, straight from memory into the matrix cores (of every x value and
// every dz value 64 bytes beside it are used, and each is used 4 NT or 64 times).  The
// waves' sums are added in order.  part: [range][C + 1][V], the last row dz's own sums.
constexpr int kGradCols = 64;
template <typename T, int NT>
__global__ __launch_bounds__(256, 2) void narrow_grad_kernel(const NarrowGrad a, int per, float* __restrict__ part) {
  constexpr int VS = 16 * NT + 4, U = NT <= 5 ? 4 : 2, CT = kGradCols / 16;
  __shared__ float sums[kGradCols * VS];
  __shared__ float bsum[16 * NT];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int c0 = blockIdx.x * kGradCols, V = a.V;
  const int r0 = __builtin_amdgcn_readfirstlane((int)min<int64_t>(a.rows, ((int64_t)blockIdx.y * 4 + w) * per));
  const int r1 = min(a.rows, r0 + per);
  const T* x = static_cast<const T*>(a.x);
  // two sets of registers by turns: one's requests are under way while the other is worked on
  T ax[2][U][CT];
  float bz[2][U][NT];
  uint32_t xo[U], zo[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    xo[u] = ((uint32_t)(4 * u + g) * (uint32_t)a.ldx + c0 + c) * (uint32_t)sizeof(T);
    zo[u] = ((uint32_t)(4 * u + g) * (uint32_t)a.ldz + c) * 4u;
  }
  // (rows behind the range read as 0; columns behind C, which no sum that is kept takes in,
  // as what stands there)
  auto request = [&](int r, auto set) {
    constexpr int S = decltype(set)::value;
#if defined(__HIP_DEVICE_COMPILE__)
    int left = r1 - r;
    asm("" : "+s"(left));  // (the compiler would make the loop's exits of it, and copy all sums)
    const auto xs = memory(x + r * a.ldx, ((left - 1) * a.ldx + a.C) * (int64_t)sizeof(T));
    const auto zs = memory(a.dz + r * a.ldz, left * a.ldz * 4);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < CT; ++j) ax[S][u][j] = load_one<T>(xs, xo[u] + 16 * j * sizeof(T));
#pragma unroll
      for (int t = 0; t < NT; ++t) bz[S][u][t] = load_one<float>(zs, zo[u] + 64 * t);
    }
#endif
  };
  f32x4 acc[CT][NT];
  float db[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    db[t] = 0.f;
#pragma unroll
    for (int j = 0; j < CT; ++j) acc[j][t] = zero4();
  }
  auto add = [&](auto set) {
    constexpr int S = decltype(set)::value;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int t = 0; t < NT; ++t) db[t] += bz[S][u][t];
#pragma unroll
      for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          acc[j][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(Elem<T>::to_f(ax[S][u][j]), bz[S][u][t], acc[j][t], 0, 0, 0);
    }
  };
  constexpr std::integral_constant<int, 0> first;
  constexpr std::integral_constant<int, 1> second;
  // (each request where it stands: its registers are those of the set just added)
  request(r0, first);
#pragma unroll 1
  for (int r = r0; r < r1; r += 8 * U) {
    request(r + 4 * U, second);
    __builtin_amdgcn_sched_barrier(0);
    add(first);
    __builtin_amdgcn_sched_barrier(0);
    request(r + 8 * U, first);
    __builtin_amdgcn_sched_barrier(0);
    add(second);
    __builtin_amdgcn_sched_barrier(0);
  }
  float* out = part + (int64_t)blockIdx.y * (a.C + 1) * V;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    db[t] += __shfl_xor(db[t], 16, 64);
    db[t] += __shfl_xor(db[t], 32, 64);
  }
  float* own = sums + 4 * g * VS + c;
  auto join = [&] {  // reads of four tiles together: one after another they wait for each other
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      db[t] += bsum[16 * t + c];
      f32x4 old[CT];
#pragma unroll
      for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) old[j][i] = own[(16 * j + i) * VS + 16 * t];
#pragma unroll
      for (int j = 0; j < CT; ++j) acc[j][t] += old[j];
      __builtin_amdgcn_sched_barrier(0);  // (not all tiles at once: their registers are not there)
    }
  };
#pragma unroll 1
  for (int k = 0; k < 3; ++k) {
    if (w == k) {
      if (k) join();
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (g == 0) bsum[16 * t + c] = db[t];
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) own[(16 * j + i) * VS + 16 * t] = acc[j][t][i];
      }
    }
    __syncthreads();
  }
  if (w != 3) return;
  join();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int v = 16 * t + c;
    if (v >= V) continue;
    if (g == 0 && blockIdx.x == 0) out[(int64_t)a.C * V + v] = db[t];
#pragma unroll
    for (int j = 0; j < CT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = c0 + 16 * j + 4 * g + i;
        if (row < a.C) out[(int64_t)row * V + v] = acc[j][t][i];
      }
  }
}

// The ranges' sums, added in order: 64 values a workgroup, whose 16 waves take contiguous
// runs of ranges.  The mean of the losses by one more, if wanted: its 4 us pass beside.
__global__ __launch_bounds__(1024) void narrow_sum_kernel(const NarrowGrad a, int ranges, const float* __restrict__ part) {
  __shared__ float sums[16][64];
  if (a.mean.loss && blockIdx.x == gridDim.x - 1) {
    mean_loss(a.mean);
    return;
  }
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t size = (int64_t)(a.C + 1) * a.V, e = (a.dw ? 0 : (int64_t)a.C * a.V) + (int64_t)blockIdx.x * 64 + lane;
  const int per = (ranges + 15) / 16, b = w * per, end = min(ranges, b + per);
  float t = 0.f;
  if (e < size)
#pragma unroll 8
    for (int k = b; k < end; ++k) t += part[k * size + e];
  sums[w][lane] = t;
  __syncthreads();
  if (w || e >= size) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) t += sums[k][lane];
  const int64_t c = e / a.V, v = e % a.V;
  if (c == a.C) {
    if (a.db) a.db[v] = a.first ? t : a.db[v] + t;
    return;
  }
  if (!a.first) t += a.sum[c * a.sum_c + v * a.sum_v];
  const int64_t at = c * a.sdc + v * a.sdv;
  if (a.dw_bf16) static_cast<bf16_t*>(a.dw)[at] = f2bf(t);
  else static_cast<float*>(a.dw)[at] = t;
}

// Ranges of rows, each of four waves' parts of whole 32 rows: as many as make about
// kGradWgs workgroups
constexpr int kGradWgs = 512;
int grad_part(int rows, int C) {
  const int want = std::max(1, std::min(cdiv(rows, 128), kGradWgs / cdiv(C, kGradCols)));
  return cdiv(cdiv(rows, 4 * want), 32) * 32;
}
int grad_ranges(int rows, int C) { return cdiv(rows, 4 * grad_part(rows, C)); }

template <typename F>
void with_tiles(int V, F f) {
  if (V <= 32) f(std::integral_constant<int, 2>());
  else if (V <= 64) f(std::integral_constant<int, 4>());
  else if (V <= 80) f(std::integral_constant<int, 5>());
  else f(std::integral_constant<int, 6>());
}

template <typename T>
void run(const NarrowXent& a, hipStream_t st) {
  const bool vec = a.C % 4 == 0 && a.ldx % 4 == 0 && (uintptr_t)a.x % (4 * sizeof(T)) == 0;
  const dim3 grid(cdiv(a.rows, kRows)), block(256);
  with_tiles(a.V, [&](auto nt) {
    constexpr int NT = decltype(nt)::value;
    if (vec) hipLaunchKernelGGL((narrow_kernel<T, NT, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((narrow_kernel<T, NT, false>), grid, block, 0, st, a);
  });
}

template <typename T>
void run(const NarrowGrad& a, int per, const dim3& grid, float* part, hipStream_t st) {
  with_tiles(a.V, [&](auto nt) {
    hipLaunchKernelGGL((narrow_grad_kernel<T, decltype(nt)::value>), grid, dim3(256), 0, st, a, per, part);
  });
}

}  // namespace

int narrow_xent(const NarrowXent& a, hipStream_t st) {
  if (a.dtype == MTX_F32) run<float>(a, st);
  else run<bf16_t>(a, st);
  MTX_LAUNCHED();
  return MTX_OK;
}

size_t narrow_grad_workspace_bytes(int rows, int C, int V) {
  return (size_t)grad_ranges(rows, C) * (C + 1) * V * sizeof(float);
}

int narrow_grad(const NarrowGrad& a, void* workspace, hipStream_t st) {
  float* part = static_cast<float*>(workspace);
  const int ranges = grad_ranges(a.rows, a.C), per = grad_part(a.rows, a.C);
  const dim3 grid(a.dw ? cdiv(a.C, kGradCols) : 1, ranges);
  if (a.dtype == MTX_F32) run<float>(a, per, grid, part, st);
  else run<bf16_t>(a, per, grid, part, st);
  MTX_LAUNCHED();
  const int64_t values = a.dw ? (int64_t)(a.C + 1) * a.V : a.V;
  const unsigned wgs = (unsigned)((values + 63) / 64) + (a.mean.loss ? 1 : 0);
  hipLaunchKernelGGL(narrow_sum_kernel, dim3(wgs), dim3(1024), 0, st, a, ranges, part);
  MTX_LAUNCHED();
  return MTX_OK;
}

}  // namespace mtx
