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
#include <cfloat>
#include <cmath>

namespace mtx {
namespace {

struct Pages {  // (n_pages, heads, page, D) view: element strides, d stride 1
  void* p;
  int64_t sp, sh, sr;
};

// Division by a number that the host knows: j / d = (mulhi(j, mul) + j) >> shift for
// j < 2^31, the smallest shift with 2^shift >= d, and mul = 2^32 (2^shift - d) / d + 1
// (Granlund and Montgomery's division by an invariant integer)
struct Divisor32 {
  uint32_t mul;
  int shift;
  __device__ __forceinline__ int quotient(int j) const {
    return (int)((__umulhi((uint32_t)j, mul) + (uint32_t)j) >> shift);
  }
};
Divisor32 divisor32(int d) {
  int shift = 0;
  while (((int64_t)1 << shift) < d) ++shift;
  return Divisor32{(uint32_t)(((((uint64_t)1 << shift) - d) << 32) / d + 1), shift};
}

struct Table {
  const int* ids;
  int64_t ld;
  int width;        // pages per sequence
  int page;         // rows per page
  int64_t n_pages;  // pages in the pool
  Divisor32 by;     // page

  // the index of the page that holds row j
  __device__ __forceinline__ int div(int j) const { return by.quotient(j); }
  // the id at index i of sequence b's pages, or -1
  __device__ __forceinline__ int id(int b, int i) const {
    const int x = ids[b * ld + i];
    return (unsigned)x < (unsigned)n_pages ? x : -1;
  }
};

Table make_table(const int* ids, int64_t ld, int width, int page, int64_t n_pages) {
  return Table{ids, ld, width, page, n_pages, divisor32(page)};
}

// offset of row j, whose page's index is i and id is `id`
__device__ __forceinline__ int64_t row_at(const Pages& g, const Table& t, int id, int i, int j) {
  return id * g.sp + (j - i * t.page) * g.sr;
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
  int T, H, C, blocks;  // C: 16-byte chunks of a cached row
};

// 16 bytes of a cached row from the values of a new one
__device__ __forceinline__ uint4 cache_chunk(const float* x, float*) { return *reinterpret_cast<const uint4*>(x); }
__device__ __forceinline__ uint4 cache_chunk(const bf16_t* x, bf16_t*) { return *reinterpret_cast<const uint4*>(x); }
__device__ __forceinline__ uint4 cache_chunk(const float* x, bf16_t*) {
  const f32x4 u = reinterpret_cast<const f32x4*>(x)[0], v = reinterpret_cast<const f32x4*>(x)[1];
  return make_uint4(pack_bf2(u[0], u[1]), pack_bf2(u[2], u[3]), pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
}

// A thread writes 16 bytes of a row's key and of its value, found by one lookup
template <typename TX, typename TC>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a) {
  constexpr int E = 16 / sizeof(TC);
  const int b = blockIdx.x / a.blocks;
  const int i = (blockIdx.x % a.blocks) * 256 + threadIdx.x;
  const int c = i & (a.C - 1), row = i / a.C, h = row % a.H, t = row / a.H;
  if (t >= a.T) return;
  const int n = a.counts != nullptr ? min(a.counts[b], a.T) : a.T;
  const int64_t j = (int64_t)a.lengths[b] - n + t;
  if (t >= n || j < 0 || j >= (int64_t)a.tab.width * a.tab.page) return;
  const int pi = a.tab.div((int)j), id = a.tab.id(b, pi);
  if (id < 0) return;
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    const TX* x = static_cast<const TX*>(a.x[z]) + b * a.sb[z] + h * a.sh[z] + t * a.st[z] + E * c;
    TC* y = static_cast<TC*>(a.g[z].p) + row_at(a.g[z], a.tab, id, pi, (int)j) + h * a.g[z].sh + E * c;
    *reinterpret_cast<uint4*>(y) = cache_chunk(x, y);
  }
}

// ---------------------------------------------------------------------------
// decode
// ---------------------------------------------------------------------------
// One query against n cached rows reads 2 n D values a K/V head and does 4 G n D
// flops on them (G = H / Hkv heads share the rows): 2 G flops a value, bound by
// the memory for every G here.  So K and V go from memory straight into the
// registers the matrix instructions read, each value once:
//
//   scores, S^T = K Q^T: A = K (16 keys, lane l holds key l % 16 and the d values
//   of its quarter l / 16), B = Q (16 heads, the same d values); lane l then has
//   the scores of head l % 16 and keys 4 (l / 16) + r;
//   output, O^T = V^T P^T: B = P is those registers as they are, keys
//   16 t + 4 (l / 16) + r for k; A = V^T takes the same keys' rows, of which lane
//   l loads values VD (l % 16) .. + VD - 1 (VD = D / 16): its matrix row of
//   product n is d = VD (l % 16) + n.
//
// Nothing passes through LDS or across lanes but the rare update of the running
// maximum: it is raised only when a score exceeds it by more than 2^8 in the
// exponent (probabilities stay below 2^8, the sums in fp32), which in practice
// happens in a wave's first tile.
//
// fp32 pools use fp32 matrix instructions.  Over bf16 pools the weights, and fp32 rows'
// q, enter the products as three bf16 pieces (24 bits, as fp32 has).
//
// Measured, 16 sequences of 8000 to 16384 rows, 8 K/V heads of 128 in bf16 (797
// MB), 32 query heads: 140 us, 5.7 TB/s (a plain read of the same pages: 136 us); one of
// 131071 rows (67 MB): 18 us, of which 11 at the memory's rate.  The third piece of the
// weights costs no time there and more the smaller the heads are (64 sequences of 1000 to
// 3000 rows, 8 K/V heads of 16, 32 query heads: 28.1 us, 24.5 with two).
//
// A workgroup takes some rows of one sequence and K/V head (make_plan), its four
// waves in turn tiles of 16 NT of them, and joins them in LDS; several workgroups'
// results for a sequence are joined by finish_kernel.
constexpr int kMaxIds = 4096;  // page ids of a chunk, in LDS
constexpr float kRaise = 8.f;

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
  float* part_o;  // [B H][S][D] or [P][H][D] sums, relative to part_ml's maximum
  float* part_ml; // [B H][S][2] or [P][H][2] maximum (log2 units) and sum
  float* s;       // [B H][sld] scores (log2 units), with weights
  int64_t sld;
  int* cuts;      // [B][2] with P: first piece of a sequence, how many
  int B, H, Hkv, G, S, HT, chunk, cap;
  int P, most;    // pieces the sequences are cut into, by their lengths, of at most 64 `most` rows (0: S chunks each)
  int lines;      // heads' rows share 128-byte lines
  int direct;     // the workgroup's result is final: no finish_kernel
  float c;        // scale * log2(e)
  Divisor32 by_ht, by_hkv, by_s;
};

template <typename TQ, typename TC, int D> struct DecodeTile;

// bf16 pools
template <typename TQ, int D>
struct DecodeTile<TQ, bf16_t, D> {
  static constexpr int NT = 2, VD = D / 16, NC = D >= 32 ? D / 32 : 1, VW = VD >= 2 ? VD / 2 : 1;
  static constexpr int QP = sizeof(TQ) == 4 ? 3 : 1, PP = 3;
  bf16x8 q[QP][NC];
  uint4 k[NT][NC];
  uint32_t v[4 * NT][VW];

  __device__ __forceinline__ void load_q(const TQ* row, int quarter) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const bool in = row != nullptr && 32 * c + 8 * quarter < D;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = in ? Elem<TQ>::to_f(row[32 * c + 8 * quarter + e]) : 0.f;
#pragma unroll
      for (int p = 0; p < QP; ++p) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = pk_bf16(x[2 * i], x[2 * i + 1]);
          x[2 * i] -= __uint_as_float(w[i] << 16);
          x[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
        }
        q[p][c] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
      }
    }
  }
  __device__ __forceinline__ void load_k(int t, const bf16_t* row, int quarter) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      k[t][c] = *reinterpret_cast<const uint4*>(row + 32 * c + (D >= 32 ? 8 * quarter : 8 * (quarter & 1)));
  }
  __device__ __forceinline__ void load_v(int e, const bf16_t* row) {
    if constexpr (VD == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(row);
      v[e][0] = u.x, v[e][1] = u.y, v[e][2] = u.z, v[e][3] = u.w;
    } else if constexpr (VD == 4) {
      const uint2 u = *reinterpret_cast<const uint2*>(row);
      v[e][0] = u.x, v[e][1] = u.y;
    } else if constexpr (VD == 2) {
      v[e][0] = *reinterpret_cast<const uint32_t*>(row);
    } else {
      v[e][0] = *row;
    }
  }
  __device__ __forceinline__ void clear_v(int e) {
#pragma unroll
    for (int i = 0; i < VW; ++i) v[e][i] = 0;
  }
  __device__ __forceinline__ f32x4 scores(int t, int quarter) const {
    f32x4 s = zero4();
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint4 u = k[t][c];
      if (D < 32 && quarter >= 2) u = make_uint4(0, 0, 0, 0);  // 16 values fill half the product
      const bf16x8 a = __builtin_bit_cast(bf16x8, u);
#pragma unroll
      for (int p = QP - 1; p >= 0; --p) s = Mfma<bf16_t>::mma(a, q[p][c], s);
    }
    return s;
  }
  __device__ __forceinline__ void add_v(float (&p)[4 * NT], f32x4 (&o)[VD]) const {
    bf16x8 b[PP];
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = pk_bf16(p[2 * j], p[2 * j + 1]);
        p[2 * j] -= __uint_as_float(w[j] << 16);
        p[2 * j + 1] -= __uint_as_float(w[j] & 0xffff0000u);
      }
      b[i] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
    }
#pragma unroll
    for (int n = 0; n < VD; ++n) {
      uint32_t w[4];  // column n of the eight rows
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = __builtin_amdgcn_perm(v[2 * j + 1][n / 2], v[2 * j][n / 2], n & 1 ? 0x07060302 : 0x05040100);
      const bf16x8 a = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
      for (int i = PP - 1; i >= 0; --i) o[n] = Mfma<bf16_t>::mma(a, b[i], o[n]);
    }
  }
};

// fp32 pools
template <typename TQ, int D>
struct DecodeTile<TQ, float, D> {
  static constexpr int NT = D >= 128 ? 1 : 2, VD = D / 16, NC = D / 16;
  f32x4 q[NC];
  f32x4 k[NT][NC];
  float v[4 * NT][VD];

  __device__ __forceinline__ void load_q(const TQ* row, int quarter) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      q[c] = row != nullptr ? *reinterpret_cast<const f32x4*>(row + 16 * c + 4 * quarter) : zero4();
  }
  __device__ __forceinline__ void load_k(int t, const float* row, int quarter) {
#pragma unroll
    for (int c = 0; c < NC; ++c) k[t][c] = *reinterpret_cast<const f32x4*>(row + 16 * c + 4 * quarter);
  }
  __device__ __forceinline__ void load_v(int e, const float* row) {
    if constexpr (VD >= 4) {
#pragma unroll
      for (int i = 0; i < VD; i += 4) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(row + i);
        v[e][i] = x[0], v[e][i + 1] = x[1], v[e][i + 2] = x[2], v[e][i + 3] = x[3];
      }
    } else if constexpr (VD == 2) {
      const f32x2 x = *reinterpret_cast<const f32x2*>(row);
      v[e][0] = x[0], v[e][1] = x[1];
    } else {
      v[e][0] = *row;
    }
  }
  __device__ __forceinline__ void clear_v(int e) {
#pragma unroll
    for (int i = 0; i < VD; ++i) v[e][i] = 0.f;
  }
  __device__ __forceinline__ f32x4 scores(int t, int) const {
    f32x4 s = zero4();
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = Mfma<float>::mma(k[t][c][e], q[c][e], s);
    return s;
  }
  __device__ __forceinline__ void add_v(float (&p)[4 * NT], f32x4 (&o)[VD]) const {
#pragma unroll
    for (int e = 0; e < 4 * NT; ++e)
#pragma unroll
      for (int n = 0; n < VD; ++n) o[n] = Mfma<float>::mma(v[e][n], p[e], o[n]);
  }
};

__device__ __forceinline__ float lane_max4(float v) {  // over the four quarters
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float lane_sum4(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// Cutting up to 128 sequences into at most P pieces, by their lengths: the size (a
// multiple of 64 rows, 256 or more) that needs no more than P, from 64 sizes tried at
// once, a lane each.  Every wave of every workgroup comes to the same: false if there is
// no piece q, otherwise its sequence, its number in it, its rows [c0, c1), the sequence's
// length n and how many pieces it has.  It costs 1 to 1.5 us before the first load of a
// page id
struct Cut {
  int b, split, count, c0, c1, n;
};
// u > 0 units in pieces of m, exact for u < 2^21: u - 1/2 is half a piece's unit away
// from where the result changes, which is more than the product's rounding
__device__ __forceinline__ int pieces(int u, float inv) { return u ? (int)(((float)u - 0.5f) * inv) + 1 : 0; }
// f over the lanes up to each, in the wave's last lane over all of them
template <typename F>
__device__ __forceinline__ int wave_scan(int x, F f) {
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));  // row_shr 1, 2, 4, 8
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // row_bcast 15, 31
  return f(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
}
__device__ __forceinline__ bool cut_rows(const DecodeArgs& a, int q, int lane, Cut& x) {
  if (a.B == 1) {  // no trying: 0.7 us less
    x.n = min(max(a.lengths[0], 0), a.cap);
    const int size = min(max((x.n + a.P - 1) / a.P + 63 & ~63, 256), 64 * a.most);
    x.b = 0;
    x.split = q;
    x.count = (x.n + size - 1) / size;
    x.c0 = q * size;
    x.c1 = min(x.n, x.c0 + size);
    return q < x.count;
  }
  int len[2], u[2], sum = 0, top = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    len[i] = 2 * lane + i < a.B ? a.lengths[2 * lane + i] : 0;
    len[i] = min(max(len[i], 0), a.cap);
    u[i] = (len[i] + 63) >> 6;
    sum += u[i];
    top = max(top, u[i]);
  }
  const auto add = [](int x, int y) { return x + y; };
  sum = __builtin_amdgcn_readlane(wave_scan(sum, add), 63);
  top = __builtin_amdgcn_readlane(wave_scan(top, [](int x, int y) { return max(x, y); }), 63);
  const float hi = (float)min(max(top, 4), a.most), lo = fminf(fmaxf(ceilf((float)sum / (float)a.P), 4.f), hi);
  const float f = __builtin_amdgcn_exp2f(__builtin_amdgcn_logf(hi / lo) * ((float)lane * (1.f / 63.f)));
  const float m = lane == 0 ? lo : lane == 63 ? hi : fminf(ceilf(lo * f), hi), inv = 1.f / m;
  int need = 0;
  for (int s = 0; 2 * s < a.B; ++s)
    need += pieces(__builtin_amdgcn_readlane(u[0], s), inv) + pieces(__builtin_amdgcn_readlane(u[1], s), inv);
  const uint64_t fits = __ballot(need <= a.P);
  const int pick = fits ? __ffsll((unsigned long long)fits) - 1 : 63;
  const int size = 64 * (int)__uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(m), pick));
  const float by = __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(inv), pick));
  const int c0 = pieces(u[0], by), mine = c0 + pieces(u[1], by), upto = wave_scan(mine, add);
  const uint64_t in = __ballot(q < upto && q >= upto - mine);
  if (!in) return false;
  const int at = __ffsll((unsigned long long)in) - 1;
  const int first = __builtin_amdgcn_readlane(c0, at);
  x.split = q - __builtin_amdgcn_readlane(upto - mine, at);
  const int i = x.split >= first;
  x.b = 2 * at + i;
  x.split -= i ? first : 0;
  x.count = i ? __builtin_amdgcn_readlane(mine, at) - first : first;
  x.n = __builtin_amdgcn_readlane(i ? len[1] : len[0], at);
  x.c0 = x.split * size;
  x.c1 = min(x.n, x.c0 + size);
  return true;
}

// RUN consecutive rows (aligned to RUN) lie in one page, at row strides that fit
// 32-bit offsets: 16, a tile's rows have one uniform address; 4, a lane looks up
// its four V rows at once (64 sequences in pages of 20: 13.8 us a call, 15.8 with
// RUN 1); 1, each by itself
template <typename TQ, typename TC, int D, int RUN>
__global__ __launch_bounds__(256, 2) void decode_kernel(const DecodeArgs a) {
  using Tile = DecodeTile<TQ, TC, D>;
  constexpr int NT = Tile::NT, VD = Tile::VD, KT = 16 * NT, LD = D + 4;
  __shared__ union {
    int ids[kMaxIds];
    struct { float o[4][16][LD], m[4][16], l[4][16]; } j;
  } sh;
  __shared__ float lse2[16];

  // the HT workgroups that read the same rows are 8 apart: on one XCD, sharing its L2
  const int group = blockIdx.x / 8, eight = a.by_ht.quotient(group), ht = group - eight * a.HT;
  const int piece = 8 * eight + blockIdx.x % 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quarter = lane >> 4;
  // piece `slot` of all heads' rows (with P of cut_rows, else chunk r = slot mod S of
  // sequence slot / S) and K/V head hk of it
  Cut x;
  int hk, slot;
  if (__builtin_expect(a.lines != 0, 0)) {
    // a piece's heads 8 workgroups apart too
    const int e = a.by_hkv.quotient(eight);
    hk = eight - e * a.Hkv;
    slot = 8 * e + blockIdx.x % 8;
    if (!a.P) x.b = a.by_s.quotient(slot);
  } else if (__builtin_expect(a.P != 0, 0)) {
    // the pieces that there are come first, so that the GPU's compute units get one each,
    // and a piece's heads on another XCD each time (an XCD's L2 has its channels by
    // address: one head's rows of a pool stored by rows lie in few of them)
    slot = a.by_hkv.quotient(piece);
    hk = piece + slot;
    hk -= a.by_hkv.quotient(hk) * a.Hkv;
  } else {
    const int bh = a.by_s.quotient(piece);
    x.b = a.by_hkv.quotient(bh);
    hk = bh - x.b * a.Hkv;
    slot = piece - (bh - x.b) * a.S;
  }
  if (__builtin_expect(a.P != 0, 0)) {
    if (slot >= a.P || !cut_rows(a, slot, lane, x)) return;
    if (x.split == 0 && hk == 0 && ht == 0 && tid == 0) a.cuts[2 * x.b] = slot, a.cuts[2 * x.b + 1] = x.count;
  } else {
    if (x.b >= a.B) return;
    // the first chunks, which most sequences have, lie on all XCDs in turn, also where S
    // is a multiple of 8
    const int t = slot + (a.lines ? x.b : x.b * a.Hkv + hk);
    x.split = t - a.by_s.quotient(t) * a.S;
    x.c0 = x.split * a.chunk;
    x.c1 = min(a.cap, x.c0 + a.chunk);
  }
  const int b = x.b, c0 = x.c0, bh = b * a.Hkv + hk;
  const int heads = min(16, a.G - 16 * ht), h0 = hk * a.G + 16 * ht;
  // the page ids of the whole chunk, without P whatever the length, so that neither
  // load waits for the other
  const int p0 = a.tab.div(c0), np = a.tab.div(x.c1 - 1) - p0 + 1;
  if (!a.P) x.n = a.lengths[b];
  for (int i = tid; i < np; i += 256) sh.ids[i] = a.tab.id(b, p0 + i);
  Tile tile;
  tile.load_q(col < heads ? static_cast<const TQ*>(a.q) + b * a.qb + (h0 + col) * a.qh : nullptr, quarter);
  const int n = min(max(x.n, 0), a.cap), c1 = min(n, x.c1);
  if (c0 >= n && !(a.direct && c0 == 0)) return;  // finish_kernel knows which chunks there are
  __syncthreads();

  const TC* __restrict__ kp = static_cast<const TC*>(a.k.p) + hk * a.k.sh;
  const TC* __restrict__ vp = static_cast<const TC*>(a.v.p) + hk * a.v.sh;
  uint32_t there = 0;  // which of the lane's rows 16 t + 4 quarter + r (bit 4 t + r) are seen

  // offset in a pool of row j, of the pool's first row where j is not there, and
  // whether it is; without branches, for the waits on the loads in flight
  auto look = [&](const Pages& g, int j, bool& in) -> int64_t {
    const int pi = a.tab.div(min(j, c1 - 1)), id = sh.ids[pi - p0];
    in = j < c1 && id >= 0;
    return in ? row_at(g, a.tab, id, pi, j) : 0;
  };
  // the same of a row that is one for the whole wave
  auto look1 = [&](const Pages& g, int j, bool& in) -> int64_t {
    const int pi = a.tab.div(min(j, c1 - 1)), id = __builtin_amdgcn_readfirstlane(sh.ids[pi - p0]);
    in = j < c1 && id >= 0;
    return in ? row_at(g, a.tab, id, pi, j) : 0;
  };
  auto load_k = [&](int j0) {
    bool in;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (RUN == 16)
        tile.load_k(t, kp + look1(a.k, j0 + 16 * t, in) + col * (int)a.k.sr, quarter);
      else
        tile.load_k(t, kp + look(a.k, j0 + 16 * t + col, in), quarter);
    }
  };
  auto load_v = [&](int j0) {
    bool in;
    there = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (RUN == 16) {
        const TC* base = vp + look1(a.v, j0 + 16 * t, in);
        const int seen = in ? c1 - j0 - 16 * t : 0;  // rows from j0 + 16 t on
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          tile.load_v(4 * t + r, base + (4 * quarter + r) * (int)a.v.sr + VD * col);
          there |= (uint32_t)(4 * quarter + r < seen) << (4 * t + r);
        }
      } else if constexpr (RUN == 4) {
        const int j = j0 + 16 * t + 4 * quarter;
        const TC* base = vp + look(a.v, j, in) + VD * col;
        const int seen = in ? c1 - j : 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          tile.load_v(4 * t + r, base + r * (int)a.v.sr);
          there |= (uint32_t)(r < seen) << (4 * t + r);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          tile.load_v(4 * t + r, vp + look(a.v, j0 + 16 * t + 4 * quarter + r, in) + VD * col);
          there |= (uint32_t)in << (4 * t + r);
        }
      }
    }
  };

  f32x4 o[VD];
#pragma unroll
  for (int i = 0; i < VD; ++i) o[i] = zero4();
  float mu = -FLT_MAX, l = 0.f;
  int j0 = c0 + KT * wave;
  if (j0 < c1) {
    load_k(j0);
    load_v(j0);
  }
  for (; j0 < c1; j0 += 4 * KT) {
    const int next = j0 + 4 * KT;
    float p[4 * NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const f32x4 s = tile.scores(t, quarter);
#pragma unroll
      for (int r = 0; r < 4; ++r) p[4 * t + r] = s[r] * a.c;
    }
    // unconditional, or the wait for V would have to wait for these loads too: behind
    // the last tile they read the pool's first rows
    load_k(next);
    if (__ballot(there != (1u << (4 * NT)) - 1)) {  // a hidden row: no weight, and its V is not used
#pragma unroll
      for (int e = 0; e < 4 * NT; ++e)
        if (!((there >> e) & 1)) {
          p[e] = -INFINITY;
          tile.clear_v(e);
        }
    }
    if (a.w != nullptr && col < heads) {
      float* s = a.s + (int64_t)(b * a.H + h0 + col) * a.sld + j0 + 4 * quarter;
#pragma unroll
      for (int t = 0; t < NT; ++t)
        *reinterpret_cast<f32x4*>(s + 16 * t) = f32x4{p[4 * t], p[4 * t + 1], p[4 * t + 2], p[4 * t + 3]};
    }
    float mx = p[0];
#pragma unroll
    for (int e = 1; e < 4 * NT; ++e) mx = fmaxf(mx, p[e]);
    if (__ballot(mx > mu + kRaise)) {
      const float m = fmaxf(mu, lane_max4(mx)), f = __builtin_amdgcn_exp2f(mu - m);
      mu = m;
      l *= f;
#pragma unroll
      for (int i = 0; i < VD; ++i) o[i] *= f;
    }
#pragma unroll
    for (int e = 0; e < 4 * NT; ++e) {
      p[e] = __builtin_amdgcn_exp2f(p[e] - mu);
      l += p[e];
    }
    tile.add_v(p, o);
    load_v(next);
  }

  // join the waves: head col's values VD (4 quarter + r) + n in o[n][r]
  l = lane_sum4(l);
  __syncthreads();  // the page ids are read
  if (col < heads) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < VD; ++i) sh.j.o[wave][col][VD * (4 * quarter + r) + i] = o[i][r];
    if (quarter == 0) {
      sh.j.m[wave][col] = mu;
      sh.j.l[wave][col] = l;
    }
  }
  __syncthreads();
  for (int i = tid; i < heads * D; i += 256) {
    const int h = i / D, d = i % D;
    const float m = fmaxf(fmaxf(sh.j.m[0][h], sh.j.m[1][h]), fmaxf(sh.j.m[2][h], sh.j.m[3][h]));
    float value = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(sh.j.m[w][h] - m);
      value += f * sh.j.o[w][h][d];
      sum += f * sh.j.l[w][h];
    }
    const int64_t row = (int64_t)b * a.H + h0 + h;
    if (a.direct) {
      const bool some = sum > 0.f || sum != sum;
      static_cast<TQ*>(a.o)[b * a.ob + (h0 + h) * a.oh + d] = Elem<TQ>::from_f(some ? value / sum : 0.f);
      if (d == 0) {
        if (a.lse != nullptr) a.lse[row] = some ? m * kLn2 + logf(sum) : -INFINITY;
        lse2[h] = some ? m + log2f(sum) : 0.f;
      }
    } else {
      const int64_t at = a.P ? (int64_t)slot * a.H + h0 + h : row * a.S + x.split;
      a.part_o[at * D + d] = value;
      if (d == 0) {
        a.part_ml[at * 2] = m;
        a.part_ml[at * 2 + 1] = sum;
      }
    }
  }
  if (a.direct && a.w != nullptr) {
    __syncthreads();  // this workgroup's scores and lse2 are written
    const float* s = a.s + ((int64_t)b * a.H + h0) * a.sld;
    for (int j = tid; j < n; j += 256) {
      float w = 0.f;
      for (int g = 0; g < heads; ++g) w += __builtin_amdgcn_exp2f(s[g * a.sld + j] - lse2[g]);
      if (a.win != nullptr) w += a.win[bh * a.wld + j];
      a.w[bh * a.wld + j] = w;
    }
  }
}

// a sequence's chunks: how many of `n` rows, the place of head h's first in part_o
// and part_ml, and how far apart they are
struct Chunks {
  int count, step;
  int64_t first;
  __device__ __forceinline__ Chunks(const DecodeArgs& a, int b, int h, int n) {
    if (a.P) {
      count = n ? a.cuts[2 * b + 1] : 0;
      step = a.H;
      first = n ? (int64_t)a.cuts[2 * b] * a.H + h : 0;
    } else {
      count = (n + a.chunk - 1) / a.chunk;
      step = 1;
      first = ((int64_t)b * a.H + h) * a.S;
    }
  }
};
// maximum and sum of one head over its chunks, by one wave
__device__ __forceinline__ void chunk_total(const float* ml, const Chunks& c, int lane, float& m, float& l) {
  m = -FLT_MAX;
  l = 0.f;
  for (int i = lane; i < c.count; i += 64) {
    const f32x2 x = reinterpret_cast<const f32x2*>(ml)[(int64_t)i * c.step];
    const float n = fmaxf(m, x[0]);
    l = l * __builtin_amdgcn_exp2f(m - n) + x[1] * __builtin_amdgcn_exp2f(x[0] - n);
    m = n;
  }
  const float all = wave_max(m);
  l = wave_sum(l * __builtin_amdgcn_exp2f(m - all));
  m = all;
}

// Joins the chunks of decode_kernel: the first workgroups each FD values of one
// head's output, the others kFinishRows rows' weights of one sequence and K/V
// head.  FD is 16 where there are few heads, whose chunks may be hundreds (8 heads
// of 256 chunks: 4.7 us, 22 with D), and D where there are many (512 heads of 16:
// 4.7 us, 9 with 16)
constexpr int kFinishRows = 1024;
template <typename TQ, int D, int FD>
__global__ __launch_bounds__(256) void finish_kernel(const DecodeArgs a) {
  constexpr int DL = FD / 4, NG = 256 / DL, ND = D / FD;  // lanes over d, groups of chunks
  __shared__ union {
    f32x4 x[4][DL];
    float lse2[256];
  } sh;
  const int tid = threadIdx.x, lane = tid & 63, outs = a.B * a.H * ND;
  if ((int)blockIdx.x < outs) {
    const int64_t row = blockIdx.x / ND;
    const int b = (int)row / a.H, h = (int)row % a.H;
    const Chunks chunks(a, b, h, min(max(a.lengths[b], 0), a.cap));
    const float* ml = a.part_ml + chunks.first * 2;
    float m, l;
    chunk_total(ml, chunks, lane, m, l);
    const int d = tid % DL, g = tid / DL, d0 = blockIdx.x % ND * FD;
    const float* po = a.part_o + chunks.first * D + d0 + 4 * d;
    f32x4 x = zero4();
    for (int i = g; i < chunks.count; i += NG) {
      const int64_t at = (int64_t)i * chunks.step;
      x += *reinterpret_cast<const f32x4*>(po + at * D) * __builtin_amdgcn_exp2f(ml[2 * at] - m);
    }
#pragma unroll
    for (int s = DL; s < 64; s <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], s, 64);
    if (lane < DL) sh.x[tid >> 6][lane] = x;
    __syncthreads();
    const bool some = l > 0.f || l != l;
    if (tid < FD) {
      const float* y = reinterpret_cast<const float*>(sh.x) + tid;
      const float sum = (y[0] + y[FD]) + (y[2 * FD] + y[3 * FD]);
      static_cast<TQ*>(a.o)[b * a.ob + h * a.oh + d0 + tid] = Elem<TQ>::from_f(some ? sum / l : 0.f);
    }
    if (tid == 0 && d0 == 0 && a.lse != nullptr) a.lse[row] = some ? m * kLn2 + logf(l) : -INFINITY;
    return;
  }
  const int i = blockIdx.x - outs, blocks = (a.cap + kFinishRows - 1) / kFinishRows;
  const int bh = i / blocks, b = bh / a.Hkv, hk = bh % a.Hkv;
  const int n = min(max(a.lengths[b], 0), a.cap), j0 = (i % blocks) * kFinishRows, j1 = min(n, j0 + kFinishRows);
  if (j0 >= n) return;
  const int64_t row = (int64_t)b * a.H + hk * a.G;
  for (int g = tid >> 6; g < a.G; g += 4) {
    const Chunks chunks(a, b, hk * a.G + g, n);
    float m, l;
    chunk_total(a.part_ml + chunks.first * 2, chunks, lane, m, l);
    if (lane == 0) sh.lse2[g] = l > 0.f || l != l ? m + log2f(l) : 0.f;
  }
  __syncthreads();
  const float* s = a.s + row * a.sld;
  for (int j = j0 + tid; j < j1; j += 256) {
    float w = 0.f;
    for (int g = 0; g < a.G; ++g) w += __builtin_amdgcn_exp2f(s[g * a.sld + j] - sh.lse2[g]);
    if (a.win != nullptr) w += a.win[bh * a.wld + j];
    a.w[bh * a.wld + j] = w;
  }
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
  int B, H, cap, keep, recent;
  int C, es;  // 16-byte chunks of a row, bytes of a value
};

// order of weights as unsigned numbers: NaN above everything, -0 equal to 0
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// Selection, one workgroup of NT threads per sequence and K/V head: the key of
// the last kept row (of the cand rows that are not recent, `want` are kept), then
// the kept rows in order.  The range of keys [lo, hi] is cut into up to 2048 equal
// bins, counted in LDS; the bin in which the want-th largest key lies is the next
// range, and once it holds NT / 2 rows or fewer they are ranked among themselves:
// mostly after one round, three at most.  A sample of long sequences says first where
// the key lies, mostly in a list of some thousand.  Rows are held in registers, R a
// thread, where they fit (SINGLE); otherwise each step reads them again.  Bound by its
// vector instructions, some 30 a row, on as many compute units as there are sequences
// and heads (64 of 30000 to 40000 rows: 24 us).
constexpr int kBins = 2048;

template <int NT, int R, bool SINGLE>
__device__ __forceinline__ void select_rows(const EvictArgs& a, int bh, int len, int* slots) {
  constexpr int W = NT / 64;
  __shared__ int bins[kBins], part[W], gts[W], ties[W];
  __shared__ uint32_t mins[W], maxs[W], found[4], few[NT / 2], list[4 * NT];
  __shared__ int nfew;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float* __restrict__ w = a.w + bh * a.wld;
  const int cand = len > a.keep ? len - a.recent : 0;
  int want = a.keep - a.recent;

  // wave w has rows `per` w .. and takes them 64 R at a time: row 64 i + lane of
  // those in key[i], 0 (which no weight has) behind the last
  const int per = SINGLE ? 64 * R : (cand + 64 * R * W - 1) / (64 * R * W) * (64 * R);
  const int first = per * wave, last = min(cand, first + per);
  uint32_t key[R];
  auto load = [&](int base) {
    if (!SINGLE && base + 64 * R <= last) {
      float x[R];
#pragma unroll
      for (int i = 0; i < R; ++i) x[i] = w[base + lane + 64 * i];
#pragma unroll
      for (int i = 0; i < R; ++i) key[i] = weight_key(x[i]);
      return;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int j = base + lane + 64 * i;
      key[i] = j < last ? __float_as_uint(w[j]) : 0xffffffffu;
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
      key[i] = base + lane + 64 * i < last ? weight_key(__uint_as_float(key[i])) : 0u;
  };
  if (SINGLE) load(first);
  auto each = [&](auto f) {
    if (SINGLE) {
#pragma unroll
      for (int i = 0; i < R; ++i) f(key[i]);
    } else {
      for (int base = first; base < last; base += 64 * R) {
        load(base);
#pragma unroll
        for (int i = 0; i < R; ++i) f(key[i]);
      }
    }
  };

  uint32_t bound = 0xffffffffu;  // smallest kept key; `want` of the rows that have it are kept
  if (cand > 0 && want > 0) {
    uint32_t lo = 0xffffffffu, hi = 0;
    // the least and largest of the workgroup's keys, of which a thread has lo + 1 and hi
    auto range = [&] {
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) {
        lo = min(lo, (uint32_t)__shfl_xor((int)lo, m, 64));
        hi = max(hi, (uint32_t)__shfl_xor((int)hi, m, 64));
      }
      if (lane == 0) mins[wave] = lo, maxs[wave] = hi;
      for (int i = tid; i < kBins; i += NT) bins[i] = 0;
      __syncthreads();
      for (int i = 0; i < W; ++i) lo = min(lo, mins[i]), hi = max(hi, maxs[i]);
      lo = __builtin_amdgcn_readfirstlane(lo + 1), hi = __builtin_amdgcn_readfirstlane(hi);
    };
    constexpr int PB = kBins / NT;
    const int top = kBins - 1 - PB * tid;
    // with the bins counted: this thread's, and those from the top down to them
    auto scan = [&](int& n, int& upto) {
      n = 0;
#pragma unroll
      for (int i = 0; i < PB; ++i) n += bins[top - i];
      upto = n;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const int x = __shfl_up(upto, m, 64);
        if (lane >= m) upto += x;
      }
      if (lane == 63) part[wave] = upto;
      __syncthreads();
      for (int i = 0; i < wave; ++i) upto += part[i];
    };
    auto clear = [&] {
      for (int i = tid; i < kBins; i += NT) bins[i] = 0;
    };
    bool known = false;  // lo and hi hold the bound between them
    int listed = -1;     // the keys between them are in the list, if not negative
    if (NT * 8 < cand) {
      // 4 NT rows spread over all say between which keys the bound lies (three
      // deviations of such a sample's median to either side); if the count confirms it
      // only the rows between them are looked at below, in a list where they fit
      constexpr int S = 4 * NT, MARGIN = 3 * 32;
      static_assert(S <= 4096, "the margin is three times half the root of 4096");
      uint32_t some[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) some[i] = weight_key(w[(int64_t)(tid + NT * i) * cand / S]);
#pragma unroll
      for (int i = 0; i < 4; ++i) lo = min(lo, some[i] - 1u), hi = max(hi, some[i]);
      range();
      const int shift = max(0, 21 - __clz((int)(hi - lo)));
#pragma unroll
      for (int i = 0; i < 4; ++i) atomicAdd(&bins[(some[i] - lo) >> shift], 1);
      if (tid == 0) found[0] = 1, found[1] = 0xffffffffu;
      __syncthreads();
      int n, upto;
      scan(n, upto);
      const int rank = (int)((int64_t)want * S / cand);
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const int x = side ? rank - MARGIN : rank + MARGIN;
        if (x >= 1 && upto - n < x && upto >= x) {
          int above = upto - n, i = 0;
          while (above + bins[top - i] < x) above += bins[top - i++];
          const uint32_t l = lo + ((uint32_t)(top - i) << shift);
          found[side] = side ? l + min(hi - l, (1u << shift) - 1) : l;
        }
      }
      __syncthreads();
      const uint32_t l = __builtin_amdgcn_readfirstlane(found[0]), h = __builtin_amdgcn_readfirstlane(found[1]);
      clear();
      int gt = 0, in = 0;  // of the lane
      each([&](uint32_t k) {
        gt += k > h;
        in += k - l <= h - l;
      });
      int upin = wave_scan(in, [](int x, int y) { return x + y; }), upgt = wave_scan(gt, [](int x, int y) { return x + y; });
      if (lane == 63) gts[wave] = upgt, ties[wave] = upin;
      __syncthreads();
      int all = 0, before = upin - in;
      gt = 0;
      for (int i = 0; i < W; ++i) {
        gt += gts[i];
        if (i == wave) before += all;
        all += ties[i];
      }
      gt = __builtin_amdgcn_readfirstlane(gt), all = __builtin_amdgcn_readfirstlane(all);
      if (gt < want && want <= gt + all) {
        known = true;
        lo = l, hi = h, want -= gt;
        if (lo < hi && all <= 4 * NT) {
          listed = all;
          asm("" : "+s"(lo));  // compared again, as below
          each([&](uint32_t k) {
            if (k - lo <= h - lo) list[before++] = k;
          });
          __syncthreads();
        }
      } else {
        lo = 0xffffffffu, hi = 0;
        __syncthreads();  // mins and maxs may still be read
      }
    }
    if (!known) {
      each([&](uint32_t k) {
        lo = min(lo, k - 1u);
        hi = max(hi, k);
      });
      range();
    }
    auto between = [&](auto f) {
      if (listed >= 0) {
        for (int i = tid; i < listed; i += NT) f(list[i]);
      } else {
        each(f);
      }
    };
    while (lo < hi) {
      const int shift = max(0, 21 - __clz((int)(hi - lo)));  // (hi - lo) >> shift < kBins
      between([&](uint32_t k) {
        if (k - lo <= hi - lo) atomicAdd(&bins[(k - lo) >> shift], 1);
      });
      if (tid == 0) nfew = 0;
      __syncthreads();
      // from the top bin down, to that of the want-th largest
      int n, upto;
      scan(n, upto);
      if (upto - n < want && upto >= want) {
        int above = upto - n, i = 0;
        while (above + bins[top - i] < want) above += bins[top - i++];
        const uint32_t l = lo + ((uint32_t)(top - i) << shift);
        found[0] = l;
        found[1] = l + min(hi - l, (1u << shift) - 1);
        found[2] = (uint32_t)(want - above);
        found[3] = (uint32_t)bins[top - i];
      }
      __syncthreads();
      lo = __builtin_amdgcn_readfirstlane(found[0]), hi = __builtin_amdgcn_readfirstlane(found[1]);
      want = __builtin_amdgcn_readfirstlane((int)found[2]);
      const int in = __builtin_amdgcn_readfirstlane((int)found[3]);
      if (lo == hi) break;
      if (in > NT / 2) {
        clear();
        __syncthreads();
        continue;
      }
      between([&](uint32_t k) {
        if (k - lo <= hi - lo) few[atomicAdd(&nfew, 1)] = k;
      });
      __syncthreads();
      if (tid < in) {
        const uint32_t k = few[tid];
        int gt = 0, ge = 0;
        for (int i = 0; i < in; ++i) {
          const uint32_t o = few[i];
          gt += o > k;
          ge += o >= k;
        }
        if (gt < want && ge >= want) found[0] = k, found[2] = (uint32_t)(want - gt);
      }
      __syncthreads();
      lo = __builtin_amdgcn_readfirstlane(found[0]);
      want = __builtin_amdgcn_readfirstlane((int)found[2]);
      break;
    }
    bound = lo;
  } else {
    want = 0;  // no candidate, or none of them
  }

  // places: how many rows above the bound come before a row, and of those at the
  // bound the first `want`
  bound = __builtin_amdgcn_readfirstlane(bound);
  __syncthreads();  // gts and ties may still be read, for the sample
  int g = 0, t = 0;
  each([&](uint32_t k) {
    g += __popcll(__ballot(k > bound));
    t += __popcll(__ballot(k == bound));
  });
  if (lane == 0) gts[wave] = g, ties[wave] = t;
  __syncthreads();
  g = lane < wave ? gts[lane] : 0, t = lane < wave ? ties[lane] : 0;
#pragma unroll
  for (int m = 1; m < W; m <<= 1) g += __shfl_xor(g, m, 64), t += __shfl_xor(t, m, 64);
  g = __builtin_amdgcn_readfirstlane(g), t = __builtin_amdgcn_readfirstlane(t);
  asm("" : "+s"(bound));  // the comparisons are made again, not kept (R pairs of masks)
  int j = first + lane;
  each([&](uint32_t k) {
    const bool isg = k > bound, ist = k == bound;
    const uint64_t bg = __ballot(isg), bt = __ballot(ist);
    if (bt == 0) {  // mostly
      const int at = g + min(t, want);
      const int pos = __builtin_amdgcn_mbcnt_hi((uint32_t)(bg >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bg, at));
      if (isg) slots[pos] = j;
    } else {
      const int ga = __builtin_amdgcn_mbcnt_hi((uint32_t)(bg >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bg, g));
      const int ta = __builtin_amdgcn_mbcnt_hi((uint32_t)(bt >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bt, t));
      if (isg | (ist & (ta < want))) slots[ga + min(ta, want)] = j;
      t += __popcll(bt);
    }
    g += __popcll(bg);
    j += 64;
  });
  // and the recent ones, or all
  for (int j = cand + tid; j < len; j += NT) slots[min(len, a.keep) - len + j] = j;
}

template <int NT, int R, bool SINGLE>
__global__ __launch_bounds__(NT) void select_kernel(const EvictArgs a) {
  const int bh = blockIdx.x, b = bh / a.H, len = min(max(a.lengths[b], 0), a.cap);
  if (threadIdx.x == 0 && bh % a.H == 0) a.lengths_out[b] = min(len, a.keep);
  select_rows<NT, R, SINGLE>(a, bh, len, a.slots + (int64_t)bh * a.keep);
}

// The same of up to 64 R rows by one wave, with nothing but ballots.  The last kept
// key is found bit by bit: the largest with `want` or more rows at or above it
template <int R>
__device__ __forceinline__ void select_few(const EvictArgs& a, int bh, int len, int* slots) {
  const int lane = threadIdx.x & 63, cand = len > a.keep ? len - a.recent : 0;
  const float* __restrict__ w = a.w + bh * a.wld;
  uint32_t key[R];
#pragma unroll
  for (int i = 0; i < R; ++i) key[i] = lane + 64 * i < a.cap ? weight_key(w[lane + 64 * i]) : 0u;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (lane + 64 * i >= cand) key[i] = 0u;
  int want = cand > 0 ? a.keep - a.recent : 0;
  uint32_t bound = 0xffffffffu;
  if (want > 0) {
    bound = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = bound | (1u << bit);
      int n = 0;
#pragma unroll
      for (int i = 0; i < R; ++i) n += __popcll(__ballot(key[i] >= t));
      if (n >= want) bound = t;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) want -= __popcll(__ballot(key[i] > bound));
  }
  int at = 0, ties = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const bool tie = key[i] == bound;
    const uint64_t tm = __ballot(tie);
    const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(tm >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)tm, ties));
    const bool kept = key[i] > bound || (tie && before < want);
    const uint64_t km = __ballot(kept);
    const int pos = __builtin_amdgcn_mbcnt_hi((uint32_t)(km >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)km, at));
    if (kept) slots[pos] = lane + 64 * i;
    ties += __popcll(tm);
    at += __popcll(km);
  }
  for (int j = cand + lane; j < len; j += 64) slots[min(len, a.keep) - len + j] = j;
}

// Copying the kept rows: a thread takes 16 bytes (number c) of the keys and the
// values of the rows r0 + per i, i < kRows, which are the old rows j[i] (-1: none),
// and the first of a row's threads its weight.  A row without a new page is not read
constexpr int kRows = 2;
struct RowCopy {
  int c, per, r0, j[kRows], from[kRows], to[kRows], ti[kRows];

  __device__ __forceinline__ RowCopy(const EvictArgs& a, int block) {
    c = threadIdx.x & (a.C - 1);
    per = 256 / a.C;
    r0 = block * per * kRows + threadIdx.x / a.C;
  }
  __device__ __forceinline__ void copy(const EvictArgs& a, int bh, int h) const {
    if (c == 0) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (j[i] >= 0) a.w_out[bh * a.wld + r0 + per * i] = a.w[bh * a.wld + j[i]];
    }
    uint4 x[kRows], y[kRows];
    const int64_t es = a.es;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      x[i] = y[i] = make_uint4(0, 0, 0, 0);
      if (from[i] < 0) continue;
      const int fi = a.from.div(j[i]);
      x[i] = reinterpret_cast<const uint4*>(static_cast<const char*>(a.k.p) +
                                            es * (row_at(a.k, a.from, from[i], fi, j[i]) + h * a.k.sh))[c];
      y[i] = reinterpret_cast<const uint4*>(static_cast<const char*>(a.v.p) +
                                            es * (row_at(a.v, a.from, from[i], fi, j[i]) + h * a.v.sh))[c];
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (to[i] < 0) continue;
      const int r = r0 + per * i;
      reinterpret_cast<uint4*>(static_cast<char*>(a.k.p) +
                               es * (row_at(a.k, a.to, to[i], ti[i], r) + h * a.k.sh))[c] = x[i];
      reinterpret_cast<uint4*>(static_cast<char*>(a.v.p) +
                               es * (row_at(a.v, a.to, to[i], ti[i], r) + h * a.v.sh))[c] = y[i];
    }
  }
};

// Selection and copy in one launch, of caches of up to N rows: each of a sequence
// and head's `blocks` workgroups selects the rows, into LDS, and copies its share
template <int N>
__global__ __launch_bounds__(256) void evict_kernel(const EvictArgs a, int blocks) {
  __shared__ int rows[N], ids[N];
  const int bh = blockIdx.x / blocks, block = blockIdx.x % blocks, b = bh / a.H, tid = threadIdx.x;
  const int length = a.lengths[b];
  RowCopy copy(a, block);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = copy.r0 + copy.per * i;
    copy.ti[i] = a.to.div(r);
    copy.to[i] = r < min(a.keep, a.cap) ? a.to.id(b, copy.ti[i]) : -1;
  }
  const int len = min(max(length, 0), a.cap), new_len = min(len, a.keep);
  constexpr bool few = N <= 256;  // by the first wave alone, the others read the page ids
  if (!few || tid >= 64)
    for (int i = few ? tid - 64 : tid; i < a.from.width; i += few ? 192 : 256) ids[i] = a.from.id(b, i);
  if constexpr (few) {
    if (tid < 64) select_few<N / 64>(a, bh, len, rows);
  } else {
    select_rows<256, N / 256, true>(a, bh, len, rows);
  }
  __syncthreads();
  int* slots = a.slots + (int64_t)bh * a.keep;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = copy.r0 + copy.per * i;
    copy.j[i] = r < new_len ? rows[r] : -1;
    if (r >= new_len) copy.to[i] = -1;
    else if (copy.c == 0) slots[r] = copy.j[i];
    copy.from[i] = copy.to[i] < 0 ? -1 : ids[a.from.div(copy.j[i])];
  }
  copy.copy(a, bh, bh % a.H);
  if (block) return;
  if (tid == 0 && bh % a.H == 0) a.lengths_out[b] = new_len;
  for (int j = new_len + tid; j < max(a.cap, a.keep); j += 256) {
    if (j < a.cap) a.w_out[bh * a.wld + j] = 0.f;
    if (j < a.keep) slots[j] = -1;
  }
}

// The copy behind select_kernel; the last blocks of a sequence and head clear the
// weights behind its rows
__global__ __launch_bounds__(256) void gather_kernel(const EvictArgs a, int blocks, int fills) {
  const int bh = blockIdx.x / (blocks + fills), block = blockIdx.x % (blocks + fills);
  const int b = bh / a.H;
  const int new_len = min(min(max(a.lengths[b], 0), a.cap), a.keep);
  if (block >= blocks) {
    float* wo = a.w_out + bh * a.wld;
    int* slots = a.slots + (int64_t)bh * a.keep;
    for (int j = new_len + (block - blocks) * 256 + threadIdx.x; j < max(a.cap, a.keep); j += fills * 256) {
      if (j < a.cap) wo[j] = 0.f;
      if (j < a.keep) slots[j] = -1;
    }
    return;
  }
  const int* __restrict__ slots = a.slots + (int64_t)bh * a.keep;
  RowCopy copy(a, block);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = copy.r0 + copy.per * i;
    copy.j[i] = r < new_len ? slots[r] : -1;
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    copy.ti[i] = a.to.div(copy.r0 + copy.per * i);
    copy.from[i] = copy.j[i] < 0 ? -1 : a.from.id(b, a.from.div(copy.j[i]));
    copy.to[i] = copy.j[i] < 0 ? -1 : a.to.id(b, copy.ti[i]);
    if (copy.to[i] < 0) copy.from[i] = -1;
  }
  copy.copy(a, bh, bh % a.H);
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

// a launch's threads are counted in 32 bits
constexpr int64_t kMaxGroups = (1 << 24) - 1;

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

// How a decode call is cut, and its workspace [part_o | part_ml | scores | cuts].
//
// Whole sequences, with no second launch, where the rows are few (1280 rows of 64
// values, 640 of 128: 8.6 us in one workgroup, 12.5 in several) or the workgroups
// enough for the GPU (B = 32, 4 K/V heads of 128, 1500 rows: 21 us, 23 to 25 in chunks;
// 64 sequences of 100 to 3000 rows, 8 of 128: 85, 97).
//
// Else up to 128 sequences and K/V heads: P pieces by the lengths (cut_rows), one for each
// compute unit, or for each HT workgroups' where there are many (30 sequences of 1000 to
// 9000 rows, 3 K/V heads of 128, 96 query heads: 77 us, in chunks 102).  16 sequences of
// 8000 to 16384 rows, 8 heads: 144 us, in chunks of 1024 rows 156; one of 16384 and 15 of
// 300: 25, 38; 7 sequences of 9000, 2 heads, 21.0, 20.0.
//
// Else chunks alike, 512 to 1024 rows each, some 768 or more: they come to the compute
// units as those get free, which P pieces of unequal size would not (20 sequences of
// 10000 rows, 8 heads of 64: 83 us, 90 by pieces)
struct DecodePlan {
  int chunk, S, HT, P, most, direct;
  int64_t n_o, n_ml, n_s, n_cuts, sld;
  size_t bytes() const { return (size_t)(n_o + n_ml + n_s + n_cuts) * sizeof(float); }
};
DecodePlan make_plan(int B, int H, int Hkv, int D, int page, int max_pages, bool weights) {
  const int cap = page * max_pages;
  DecodePlan p{};
  p.HT = cdiv(H / Hkv, 16);
  const int64_t segments = (int64_t)B * Hkv * p.HT;
  p.most = (int)(std::min<int64_t>((int64_t)(kMaxIds - 2) * page, 1 << 27) / 64);
  const int one = (segments >= 384 ? 4096 : 2048) / (D >= 64 ? 1 : 2);
  if (cap <= one && (segments >= 128 || cap * std::max(D, 64) <= 81920)) {
    p.chunk = cap;
  } else if (B * Hkv <= 128 && cap <= (1 << 27)) {
    // two a compute unit where a tile is small (32 sequences of 30000 rows, 4 heads of 32:
    // 96 us, 121 with one; 5 of 43000, 8 heads of 16: 36, 54); the HT workgroups of a piece
    // lie on one XCD: each of the 8 has place for 32 / HT
    const int n = 8 * (D < 64 ? 2 : 1) * (segments <= 128 ? 32 / p.HT : 32) / Hkv;
    p.P = (int)std::max<int64_t>(std::min<int64_t>(n, (int64_t)B * cdiv(cap, 256)),
                                 (int64_t)B * cdiv(cap, 64 * p.most));
    p.chunk = cap;
  } else {
    const int64_t want = std::min<int64_t>(std::max<int64_t>(cap * segments / 768, 512), 1024);
    p.chunk = (cdiv(cap, cdiv(cap, (int)want)) + 63) / 64 * 64;
  }
  p.S = cdiv(cap, p.chunk);
  p.direct = !p.P && p.S == 1 && (!weights || p.HT == 1);
  p.sld = ((int64_t)cap + 31) / 32 * 32;
  const int64_t parts = p.direct ? 0 : p.P ? (int64_t)p.P * H : (int64_t)B * H * p.S;
  p.n_o = parts * D;
  p.n_ml = (parts * 2 + 3) / 4 * 4;
  p.n_s = weights ? (int64_t)B * H * p.sld : 0;
  p.n_cuts = p.P ? (2 * B + 3) / 4 * 4 : 0;
  return p;
}

template <typename TQ, typename TC, int D>
int launch_decode(int run, unsigned groups, unsigned finish, const DecodeArgs& a, hipStream_t st) {
  if (run == 16) hipLaunchKernelGGL((decode_kernel<TQ, TC, D, 16>), dim3(groups), dim3(256), 0, st, a);
  else if (run == 4) hipLaunchKernelGGL((decode_kernel<TQ, TC, D, 4>), dim3(groups), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((decode_kernel<TQ, TC, D, 1>), dim3(groups), dim3(256), 0, st, a);
  MTX_LAUNCHED();
  if (!a.direct) {
    const unsigned heads = (unsigned)(a.B * a.H);
    if (heads * (D / 16) <= 1024)
      hipLaunchKernelGGL((finish_kernel<TQ, D, 16>), dim3(heads * (D / 16) + finish), dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((finish_kernel<TQ, D, D>), dim3(heads + finish), dim3(256), 0, st, a);
    MTX_LAUNCHED();
  }
  return MTX_OK;
}
template <typename TQ, typename TC>
int dispatch_decode(int D, int run, unsigned groups, unsigned finish, const DecodeArgs& a, hipStream_t st) {
  switch (D) {
    case 16: return launch_decode<TQ, TC, 16>(run, groups, finish, a, st);
    case 32: return launch_decode<TQ, TC, 32>(run, groups, finish, a, st);
    case 64: return launch_decode<TQ, TC, 64>(run, groups, finish, a, st);
    default: return launch_decode<TQ, TC, 128>(run, groups, finish, a, st);
  }
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
  const int es = dtype == MTX_F32 ? 4 : 2, ec = cache_dtype == MTX_F32 ? 4 : 2;
  const int64_t chunks = (int64_t)T * H * (D * ec / 16), blocks = (chunks + 255) / 256;
  MTX_CHECK_SHAPE(T >= 1 && chunks <= (1 << 30) && blocks * B <= kMaxGroups,
                  "append: %d new rows of %d heads for %d sequences: at least 1, and fewer in one call", T, H, B);
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
               make_table(table, table_ld, max_pages, page, n_pages),
               lengths,
               counts,
               T,
               H,
               D * ec / 16,
               (int)blocks};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(B * a.blocks);
  if (cache_dtype == MTX_F32) hipLaunchKernelGGL((append_kernel<float, float>), grid, dim3(256), 0, st, a);
  else if (dtype == MTX_F32) hipLaunchKernelGGL((append_kernel<float, bf16_t>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((append_kernel<bf16_t, bf16_t>), grid, dim3(256), 0, st, a);
  MTX_LAUNCHED();
  return MTX_OK;
}

extern "C" size_t mtx_attn_decode_paged_workspace_bytes(int B, int H, int Hkv, int D, int page, int max_pages,
                                                        int with_weights) {
  if (B < 1 || H < 1 || Hkv < 1 || H % Hkv || D < 1 || page < 1 || max_pages < 1 ||
      (int64_t)page * max_pages > (1 << 28))
    return 0;
  return make_plan(B, H, Hkv, D, page, max_pages, with_weights != 0).bytes();
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
  MTX_CHECK_SHAPE(Hkv >= 1 && H % Hkv == 0 && H / Hkv <= 256,
                  "H=%d query heads must be a multiple of Hkv=%d K/V heads, at most 256 times", H, Hkv);
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
  const DecodePlan plan = make_plan(B, H, Hkv, D, page, max_pages, weights != nullptr);
  const size_t need = plan.bytes();
  MTX_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need && ((uintptr_t)workspace & 15u) == 0),
                "workspace: %zu bytes, 16-byte aligned, needed (got %zu)", need, workspace_bytes);
  // one XCD reads the lines that heads share, where its pieces are about as many as
  // another's (64 sequences of 1000 to 3000 rows, 8 heads of 16 bf16 stored by rows:
  // 27 us, else 50)
  const int64_t slots = plan.P ? plan.P : (int64_t)B * plan.S;
  const int lines = Hkv > 1 && std::max(kp_strides[1], vp_strides[1]) * (cache_dtype == MTX_F32 ? 4 : 2) < 128 &&
                    (slots % 8 == 0 || slots >= 64);
  const int64_t groups = (lines ? (slots + 7) / 8 * 8 * Hkv : (slots * Hkv + 7) / 8 * 8) * plan.HT;
  const int64_t finish = (weights != nullptr ? (int64_t)B * Hkv * cdiv(cap, kFinishRows) : 0);
  MTX_CHECK_SHAPE(groups <= kMaxGroups && finish + (int64_t)B * H <= kMaxGroups,
                  "decode: too many sequences, heads and rows in one call");
  float* ws = static_cast<float*>(workspace);
  DecodeArgs a{q, q_strides[0], q_strides[1],
               {const_cast<void*>(k_pages), kp_strides[0], kp_strides[1], kp_strides[2]},
               {const_cast<void*>(v_pages), vp_strides[0], vp_strides[1], vp_strides[2]},
               make_table(table, table_ld, max_pages, page, n_pages),
               lengths, o, o_strides[0], o_strides[1], lse, weights_in, weights, weights_ld,
               ws, ws + plan.n_o, ws + plan.n_o + plan.n_ml, plan.sld,
               reinterpret_cast<int*>(ws + plan.n_o + plan.n_ml + plan.n_s),
               B, H, Hkv, H / Hkv, plan.S, plan.HT, plan.chunk, cap, plan.P, plan.most, lines, plan.direct, scale * kLog2e,
               divisor32(plan.HT), divisor32(Hkv), divisor32(plan.S)};
  const bool near = std::max(kp_strides[2], vp_strides[2]) < (1 << 24);
  const int run = !near || page % 4 ? 1 : page % 16 ? 4 : 16;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache_dtype == MTX_F32) return dispatch_decode<float, float>(D, run, (unsigned)groups, (unsigned)finish, a, st);
  if (dtype == MTX_F32) return dispatch_decode<float, bf16_t>(D, run, (unsigned)groups, (unsigned)finish, a, st);
  return dispatch_decode<bf16_t, bf16_t>(D, run, (unsigned)groups, (unsigned)finish, a, st);
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
              make_table(table, table_ld, max_pages, page, n_pages),
              make_table(to_table, to_ld, to_pages, page, n_pages),
              lengths, weights, weights_ld, lengths_out, weights_out, slots, B, H, cap, keep, recent,
              D * ec / 16, ec};
  const int64_t blocks = cdiv(rows, kRows * (256 / a.C)), fills = std::min(cdiv(std::max(cap, keep), 4096), 64);
  MTX_CHECK_SHAPE((blocks + fills) * B * H <= kMaxGroups, "evict: too many rows in one call");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(B * H);
  // in one launch, us, against two: 192 sequences and heads of 256 rows 11.5, 15.9; 768
  // of 37.5, 37.0; 1000 rows by 1024 workgroups 12.1, 14.9, by 2048 20.4, 19.8 (each
  // selects for itself); 4000 rows by 448 14.3, 14.6, by 832 23.7, 16.9
#define FUSED(N) hipLaunchKernelGGL(evict_kernel<N>, dim3((unsigned)(blocks * B * H)), dim3(256), 0, st, a, (int)blocks)
  if (cap <= 256 || (cap <= 4096 && blocks * B * H <= (cap <= 1024 ? 1536 : 512))) {
    if (cap <= 256) FUSED(256);
    else if (cap <= 1024) FUSED(1024);
    else FUSED(4096);
    MTX_LAUNCHED();
    return MTX_OK;
  }
#undef FUSED
  // else measured for 64 sequences and heads, us: 4000 rows 11.2 by 1024 threads, 9.2
  // by 256; 32768 rows 18 held in registers, 35 read again each step; 49152 rows
  // 24 and 40; with 64 rows a thread registers spill: 48
#define SELECT(NT, R, SINGLE) hipLaunchKernelGGL((select_kernel<NT, R, SINGLE>), grid, dim3(NT), 0, st, a)
  if (cap <= 256 * 4) SELECT(256, 4, true);
  else if (cap <= 256 * 16) SELECT(256, 16, true);
  else if (cap <= 1024 * 16) SELECT(1024, 16, true);
  else if (cap <= 1024 * 32) SELECT(1024, 32, true);
  else if (cap <= 1024 * 48) SELECT(1024, 48, true);
  else SELECT(1024, 16, false);
#undef SELECT
  MTX_LAUNCHED();
  hipLaunchKernelGGL(gather_kernel, dim3((unsigned)((blocks + fills) * B * H)), dim3(256), 0, st, a, (int)blocks,
                     (int)fills);
  MTX_LAUNCHED();
  return MTX_OK;
}
