// Products of bf16 matrices on the matrix cores with fp32 accumulation.
//
// Tiling: 256 threads = 4 waves; a wave owns MI x NI MFMA tiles of 32 x 32 and the
// waves form a 2 x 2 grid; k is taken 32 at a time.  A stage of both operands goes
// from global memory straight into LDS (16 bytes a lane), two stages ahead of the
// one that is multiplied; one barrier a stage.  Two workgroups fit a compute unit:
// one's epilogue runs beside the other's products.
//
// (8192, 1024) x (1024, 50021), 839 GFLOP: 0.96 ms with 1.6 GB of fp32 results, 0.80 for
// the product over 8192 rows, 0.82 for the one over 50021 columns, of one piece each; 1.6 and
// 1.5 of two (a library's products of
// these shapes, with bf16 results: 0.70, 0.84, 0.68 ms).  The matrix cores are 60 % busy
// (42 % in the first, whose results' way out is what bounds it), at a clock that falls to
// 1.5 GHz under this load.
//
// LDS layouts, free of bank conflicts with the lanes' order that the direct loads
// impose, by permuting which 16 bytes of global memory a lane asks for:
//   contiguous along k: [row][32 k], chunk c (8 k) of row r at c ^ (r / 4 & 3), read
//     with ds_read_b128: 16 rows cover the 16 bank groups once;
//   contiguous along rows: [32 rows][k][row], read with the transposing
//     ds_read_b64_tr_b16: four k of a panel cover them.
#include "gemm_bf16.h"

#include <algorithm>
#include <type_traits>

namespace mtx {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

constexpr int BK = 32, kStages = 3, kThreads = 256, kWaves = 4;
constexpr uint32_t kNone = 0xfffffff0u;  // an offset behind every operand's end

struct Args {
  GemmBf16 g;
  int gx, gy;            // tiles along n and m
  int whole, split;      // the first tiles are taken whole, each of the others in so many ranges of k
  int units, ksteps, per;  // units of work, k stages of a tile, and of a range
  float* part;           // [range][tile - whole][BM][BN]
};

// One operand's tile of R rows and BK k.
template <bool KC, int R>
struct Tile {
  static constexpr int NI = R * BK / 512;  // direct loads of 64 x 16 bytes
  static constexpr int PW = NI / kWaves;   // of one wave
  uint32_t off[PW];
  int ck;  // KC: the lane's first k in a stage

  __device__ __forceinline__ void init(const Bf16Matrix& m, int wid, int lane) {
#pragma unroll
    for (int j = 0; j < PW; ++j) {
      const int at = (wid * PW + j) * 64 + lane;
      if constexpr (KC) {
        const int row = at / 4, c = (at & 3) ^ ((row >> 2) & 3);
        off[j] = (uint32_t)row * (uint32_t)(m.row * 2) + c * 16;
        ck = c * 8;  // (row / 4 & 3 is the same for all j)
      } else {
        const int panel = at / 128, k = at / 4 % 32, c = at & 3;
        off[j] = (uint32_t)panel * (uint32_t)(m.panel * 2) + (uint32_t)k * (uint32_t)(m.row * 2) + c * 16;
      }
    }
  }
  // Request the stage that begins at p, `left` bytes before the operand's end, and
  // holds kleft more k.
  __device__ __forceinline__ void request(const char* p, int64_t left, int kleft, bf16_t* lds, int wid) const {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint32_t bytes = left < 0 ? 0u : left > (int64_t)0xffffff00 ? 0xffffff00u : (uint32_t)left;
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), (short)0, (int)bytes, 0x00020000);
    const bool edge = KC && kleft < BK;
#pragma unroll
    for (int j = 0; j < PW; ++j) {
      const uint32_t o = edge && ck >= kleft ? kNone : off[j];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(lds + (wid * PW + j) * 512), 16, (int)o, 0, 0, 0);
    }
#endif
  }
  // Where a lane reads MFMA operands, in bytes from the tile's begin: of rows rb + 32 x
  // .. and k = 16 kk .., lane l needs row l % 32 and k = 8 (l / 32) + 0..7.
  // KC: at[kk] + 2048 x.  Else the lane of a group of 16 addresses four rows of k row
  // j / 4 and receives one row's four k: at[0] + 2048 x + 1024 kk, + 256 for the second
  // four.
  static constexpr int NA = KC ? 2 : 1;
  __device__ __forceinline__ static void places(uint32_t (&at)[NA], int rb, int lane) {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      if constexpr (KC) {
        const int row = rb + (lane & 31), c = 2 * i + (lane >> 5);
        at[i] = row * BK * 2 + ((c ^ ((row >> 2) & 3)) * 16);
      } else {
        const int G = lane >> 4, j = lane & 15, k = 8 * (G >> 1) + (j >> 2);
        at[i] = rb * BK * 2 + k * 64 + (16 * (G & 1) + 4 * (j & 3)) * 2;
      }
    }
  }
};

// The MFMA operands of one k = 16 kk: MI of A and two of B.  The reads and the wait for
// them are one block of assembly: for the reads it sees the compiler would wait until
// every direct load in flight has landed, the next stages' too.
struct Half {
  uint2 lo, hi;
  __device__ __forceinline__ bf16x8 both() const {
    return __builtin_bit_cast(bf16x8, make_uint4(lo.x, lo.y, hi.x, hi.y));
  }
};
#define MTX_RK(d, p, off) "ds_read_b128 " d ", " p " offset:" off "\n\t"
#define MTX_RR(d, p, off) "ds_read_b64_tr_b16 " d ", " p " offset:" off "\n\t"
#define MTX_DONE "s_waitcnt lgkmcnt(0)"

template <int MI, bool AK, bool BKC, int KK>
__device__ __forceinline__ void frags(const uint32_t* pa, const uint32_t* pb, uint32_t la, uint32_t lb, bf16x8 (&fa)[MI],
                                      bf16x8 (&fb)[2]) {
  const uint32_t a = la + pa[AK ? KK : 0], b = lb + pb[BKC ? KK : 0];
  if constexpr (AK && BKC) {
    if constexpr (MI == 4)
      asm volatile(MTX_RK("%4", "%7", "0") MTX_RK("%0", "%6", "0") MTX_RK("%5", "%7", "2048") MTX_RK("%1", "%6", "2048")
                       MTX_RK("%2", "%6", "4096") MTX_RK("%3", "%6", "6144") MTX_DONE
                   : "=&v"(fa[0]), "=&v"(fa[1]), "=&v"(fa[2]), "=&v"(fa[3]), "=&v"(fb[0]), "=&v"(fb[1])
                   : "v"(a), "v"(b)
                   : "memory");
    else
      asm volatile(MTX_RK("%2", "%5", "0") MTX_RK("%0", "%4", "0") MTX_RK("%3", "%5", "2048") MTX_RK("%1", "%4", "2048")
                       MTX_DONE
                   : "=&v"(fa[0]), "=&v"(fa[1]), "=&v"(fb[0]), "=&v"(fb[1])
                   : "v"(a), "v"(b)
                   : "memory");
  } else {
    constexpr int k = 1024 * KK;
    Half ha[MI], hb[2];
    if constexpr (AK) {
      if constexpr (MI == 4)
        asm volatile(MTX_RR("%4", "%9", "%c10") MTX_RR("%5", "%9", "%c11") MTX_RK("%0", "%8", "0")
                         MTX_RR("%6", "%9", "%c12") MTX_RR("%7", "%9", "%c13") MTX_RK("%1", "%8", "2048")
                             MTX_RK("%2", "%8", "4096") MTX_RK("%3", "%8", "6144") MTX_DONE
                     : "=&v"(fa[0]), "=&v"(fa[1]), "=&v"(fa[2]), "=&v"(fa[3]), "=&v"(hb[0].lo), "=&v"(hb[0].hi),
                       "=&v"(hb[1].lo), "=&v"(hb[1].hi)
                     : "v"(a), "v"(b), "n"(k), "n"(k + 256), "n"(k + 2048), "n"(k + 2304)
                     : "memory");
      else
        asm volatile(MTX_RR("%2", "%7", "%c8") MTX_RR("%3", "%7", "%c9") MTX_RK("%0", "%6", "0")
                         MTX_RR("%4", "%7", "%c10") MTX_RR("%5", "%7", "%c11") MTX_RK("%1", "%6", "2048") MTX_DONE
                     : "=&v"(fa[0]), "=&v"(fa[1]), "=&v"(hb[0].lo), "=&v"(hb[0].hi), "=&v"(hb[1].lo), "=&v"(hb[1].hi)
                     : "v"(a), "v"(b), "n"(k), "n"(k + 256), "n"(k + 2048), "n"(k + 2304)
                     : "memory");
    } else {
      if constexpr (MI == 4)
        asm volatile(MTX_RR("%8", "%13", "%c14") MTX_RR("%9", "%13", "%c15") MTX_RR("%0", "%12", "%c14")
                         MTX_RR("%1", "%12", "%c15") MTX_RR("%10", "%13", "%c16") MTX_RR("%11", "%13", "%c17")
                             MTX_RR("%2", "%12", "%c16") MTX_RR("%3", "%12", "%c17") MTX_RR("%4", "%12", "%c18")
                                 MTX_RR("%5", "%12", "%c19") MTX_RR("%6", "%12", "%c20") MTX_RR("%7", "%12", "%c21")
                                     MTX_DONE
                     : "=&v"(ha[0].lo), "=&v"(ha[0].hi), "=&v"(ha[1].lo), "=&v"(ha[1].hi), "=&v"(ha[2].lo),
                       "=&v"(ha[2].hi), "=&v"(ha[3].lo), "=&v"(ha[3].hi), "=&v"(hb[0].lo), "=&v"(hb[0].hi),
                       "=&v"(hb[1].lo), "=&v"(hb[1].hi)
                     : "v"(a), "v"(b), "n"(k), "n"(k + 256), "n"(k + 2048), "n"(k + 2304), "n"(k + 4096), "n"(k + 4352),
                       "n"(k + 6144), "n"(k + 6400)
                     : "memory");
      else
        asm volatile(MTX_RR("%4", "%9", "%c10") MTX_RR("%5", "%9", "%c11") MTX_RR("%0", "%8", "%c10")
                         MTX_RR("%1", "%8", "%c11") MTX_RR("%6", "%9", "%c12") MTX_RR("%7", "%9", "%c13")
                             MTX_RR("%2", "%8", "%c12") MTX_RR("%3", "%8", "%c13") MTX_DONE
                     : "=&v"(ha[0].lo), "=&v"(ha[0].hi), "=&v"(ha[1].lo), "=&v"(ha[1].hi), "=&v"(hb[0].lo),
                       "=&v"(hb[0].hi), "=&v"(hb[1].lo), "=&v"(hb[1].hi)
                     : "v"(a), "v"(b), "n"(k), "n"(k + 256), "n"(k + 2048), "n"(k + 2304)
                     : "memory");
#pragma unroll
      for (int x = 0; x < MI; ++x) fa[x] = ha[x].both();
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) fb[y] = hb[y].both();
  }
}

// a lane number whose uses are computed where they stand: the epilogue's addresses
// otherwise stay in registers across the k loop, which needs them all
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// OUT: 0 fp32, 1 fp32 plus add, 2 bf16, 3 bf16 of the sum with add; 4 the rows'
// statistics: there the products are taken transposed, so that a lane holds 32 columns
// of a row and only two lanes have to meet
template <int MI, bool AK, bool BKC, int OUT>
__global__ __launch_bounds__(kThreads, 2) void gemm_bf16_kernel(const Args a) {
  constexpr int BM = 64 * MI, BN = 128, NI = 2;
  using TA = Tile<AK, BM>;
  using TB = Tile<BKC, BN>;
  constexpr int kA = BM * BK, kStage = (BM + BN) * BK;
  constexpr int kLoads = TA::PW + TB::PW;  // of a wave and stage
  __shared__ __attribute__((aligned(1024))) bf16_t smem[kStages * kStage];
  const GemmBf16& g = a.g;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = (wid >> 1) * 32 * MI, wn = (wid & 1) * 32 * NI;
  TA ta;
  TB tb;
  ta.init(g.a, wid, lane);
  tb.init(g.b, wid, lane);
  uint32_t pa[TA::NA], pb[TB::NA];
  TA::places(pa, wm, lane);
  TB::places(pb, wn, lane);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)smem;

  // A unit: a whole tile, or a range of one's k stages.
  struct Unit {
    int m0, n0, s0, s1, range, tile;
  };
  auto unit = [&](int u) {
    Unit q;
    q.tile = u;
    q.s0 = 0;
    q.s1 = a.ksteps;
    q.range = -1;
    if (u >= a.whole) {
      // a range of all tiles after the other: units that run side by side share their rows
      const int v = u - a.whole, tiles = a.gx * a.gy - a.whole;
      q.tile = a.whole + v % tiles;
      q.range = v / tiles;
      q.s0 = q.range * a.per;
      q.s1 = min(a.ksteps, q.s0 + a.per);
    }
    // tiles in panels of 8 rows of tiles, column by column
    const int panel = 8 * a.gx, first = q.tile / panel * 8, high = min(8, a.gy - first), in = q.tile % panel;
    q.m0 = (first + in % high) * BM;
    q.n0 = in / high * BN;
    return q;
  };
  // Workgroups are dealt round-robin over the 8 XCDs: an XCD's take a run of units, whose
  // tiles are neighbours and read their rows through one L2
  const int wgs = gridDim.x;
  const int w0 = (blockIdx.x & 7) * (wgs >> 3) + (blockIdx.x >> 3);
  const int kpiece = (g.K + BK - 1) / BK;  // stages of a piece

  // the requests run two stages ahead of the products, across units
  struct Ahead {
    int u, left, k0;  // the unit, its stages left, k
    const char *a, *b;
    int64_t la, lb;  // bytes to the operands' ends
  } r;
  auto enter = [&](int u) {
    r.u = u;
    const Unit q = unit(u);
    r.left = q.s1 - q.s0;
    const int p = q.s0 / kpiece;
    r.k0 = (q.s0 - p * kpiece) * BK;
    const int64_t fa = AK ? q.m0 * g.a.row + r.k0 / 32 * g.a.panel : r.k0 * g.a.row + q.m0 / 32 * g.a.panel;
    const int64_t fb = BKC ? q.n0 * g.b.row + r.k0 / 32 * g.b.panel : r.k0 * g.b.row + q.n0 / 32 * g.b.panel;
    r.a = reinterpret_cast<const char*>(g.a.p + p * g.a.piece + fa);
    r.b = reinterpret_cast<const char*>(g.b.p + p * g.b.piece + fb);
    r.la = 2 * (g.a.size - fa);
    r.lb = 2 * (g.b.size - fb);
  };
  // a stage's bytes along k
  const int64_t sa = 2 * (AK ? g.a.panel : BK * g.a.row), sb = 2 * (BKC ? g.b.panel : BK * g.b.row);
  int rbuf = 0;
  bool more = true;
  auto request = [&] {
    bf16_t* to = smem + rbuf * kStage;
    rbuf = rbuf == kStages - 1 ? 0 : rbuf + 1;
    if (!more) return;
    ta.request(r.a, r.la, g.K - r.k0, to, wid);
    tb.request(r.b, r.lb, g.K - r.k0, to + kA, wid);
    if (--r.left == 0) {
      more = r.u + wgs < a.units;
      if (more) enter(r.u + wgs);
      return;
    }
    r.k0 += BK;
    r.a += sa;
    r.b += sb;
    r.la -= sa;
    r.lb -= sb;
    if (r.k0 >= g.K) {  // the next piece begins
      r.a += 2 * g.a.piece - kpiece * sa;
      r.b += 2 * g.b.piece - kpiece * sb;
      r.la += kpiece * sa;
      r.lb += kpiece * sb;
      r.k0 = 0;
    }
  };
  if (w0 >= a.units) return;
  enter(w0);
  request();
  request();
  int buf = 0;
  // Stages whose loads are older than a tile's MI * NI * 16 stores: these need not have
  // reached memory when those have landed
  int fresh = 0;
  for (int u = w0; u < a.units; u += wgs) {
    const Unit q = unit(u);
    f32x16 acc[MI][NI];
#pragma unroll
    for (int x = 0; x < MI; ++x)
#pragma unroll
      for (int y = 0; y < NI; ++y)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;
#pragma unroll 1
    for (int s = q.s0; s < q.s1; ++s) {
      // this stage's loads have landed (the next one's may be in flight), for every
      // wave; and every wave is done with the stage before, whose place the next
      // request takes
      if (!more) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      else if (fresh) asm volatile("s_waitcnt vmcnt(63)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
      fresh = max(fresh - 1, 0);
      __builtin_amdgcn_s_barrier();
      request();
      const uint32_t la = lds0 + buf * kStage * 2, lb = la + kA * 2;
      buf = buf == kStages - 1 ? 0 : buf + 1;
      auto products = [&](auto kk) {
        bf16x8 fa[MI], fb[NI];
        frags<MI, AK, BKC, decltype(kk)::value>(pa, pb, la, lb, fa, fb);
#pragma unroll
        for (int x = 0; x < MI; ++x)
#pragma unroll
          for (int y = 0; y < NI; ++y)
            acc[x][y] = OUT == 4 ? __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[y], fa[x], acc[x][y], 0, 0, 0)
                                 : __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[x], fb[y], acc[x][y], 0, 0, 0);
      };
      products(std::integral_constant<int, 0>());
      products(std::integral_constant<int, 1>());
    }

    // acc[x][y][e] = row 32 x + 8 (e / 4) + 4 (lane / 32) + e % 4, column 32 y + lane % 32
    const int lv = here(lane), lr = lv & 31, lh = lv >> 5;
    const bool part = q.range >= 0;
    const int mw = q.m0 + wm, nw = q.n0 + wn;
    if (part) {
      float* p = a.part + ((int64_t)q.range * (a.gx * a.gy - a.whole) + q.tile - a.whole) * (BM * BN) + wm * BN + wn;
#pragma unroll
      for (int x = 0; x < MI; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
          for (int y = 0; y < NI; ++y) p[(32 * x + 8 * (e / 4) + 4 * lh + e % 4) * BN + 32 * y + lr] = acc[x][y][e];
      continue;
    }
    if constexpr (OUT == 4) {
      // acc[x][y][e] = row 32 x + lane % 32, column 32 y + 8 (e / 4) + 4 (lane / 32) + e % 4
      float bias[NI][16];
#pragma unroll
      for (int y = 0; y < NI; ++y)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int n = nw + 32 * y + 8 * (e / 4) + 4 * lh + e % 4;
          bias[y][e] = g.bias && n < g.N ? g.bias[n] : 0.f;
        }
#pragma unroll
      for (int x = 0; x < MI; ++x) {
        const int m = mw + 32 * x + lr;
        const int64_t t = m < g.M ? g.columns[m] : -1;
        const int at = t >= nw && t < nw + 64 && t < g.N ? (int)(t - nw) : -1;
        const int own = at >= 0 && ((at >> 2) & 1) == lh ? (at >> 5) * 16 + ((at & 31) >> 3) * 4 + (at & 3) : -1;
        float top = -INFINITY, sum = 0.f, pick = 0.f;
#pragma unroll
        for (int y = 0; y < NI; ++y)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            acc[x][y][e] += bias[y][e];
            // (behind N there may be anything)
            if (nw + 64 > g.N && nw + 32 * y + 8 * (e / 4) + 4 * lh + e % 4 >= g.N) acc[x][y][e] = -INFINITY;
            top = fmaxf(top, acc[x][y][e]);
            pick = own == 16 * y + e ? acc[x][y][e] : pick;
          }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        // (the difference first: top log2(e) may be infinite for a finite top)
        const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int y = 0; y < NI; ++y)
#pragma unroll
          for (int e = 0; e < 16; ++e) sum += __builtin_amdgcn_exp2f((acc[x][y][e] - from) * kLog2e);
        sum += __shfl_xor(sum, 32, 64);
        if (m < g.M && nw < g.N && lh == 0) g.stats[(int64_t)(nw / 64) * g.M + m] = make_float2(top, sum);
        if (own >= 0) g.chosen[m] = pick;
      }
      continue;
    }
#if defined(__HIP_DEVICE_COMPILE__)
    // rows through a resource that begins at the pair's first row and ends with the
    // output: rows behind it are dropped, a column behind it has an offset that is
    // (fp32 results are large and not read again here: they pass the caches. The 1.6 GB
    // of 8192 x 50021: 1120 -> 1060 us)
    constexpr int kSize = OUT >= 2 ? 2 : 4, kNt = 2;
    uint32_t oo[NI], ao[NI];
    float bias[NI];
    const float scale = g.scale ? *g.scale : 1.f;
#pragma unroll
    for (int y = 0; y < NI; ++y) {
      const int n = 32 * y + lr;
      const bool ok = nw + n < g.N;
      oo[y] = ok ? (uint32_t)(4 * lh * g.ldc + n) * kSize : kNone;
      ao[y] = ok ? (uint32_t)(4 * lh * g.ldadd + n) * 4u : kNone;
      bias[y] = g.bias && ok ? g.bias[nw + n] : 0.f;
    }
    // (stepped from row to row, not worked out for each: 8192 x 50021 1020 -> 962 us)
    struct Row {
      char* p;
      int64_t left, step;
      __device__ __forceinline__ Row(const void* base, int64_t ld, int size, const GemmBf16& g, int m, int n)
          : p(const_cast<char*>(static_cast<const char*>(base)) + ((int64_t)m * ld + n) * size),
            left(n < g.N ? ((int64_t)(g.M - 1 - m) * ld + g.N - n) * size : -1), step(ld * size) {}
      __device__ __forceinline__ __amdgpu_buffer_rsrc_t here() const {
        const uint32_t bytes = left < 0 ? 0u : left >> 32 ? 0xffffff00u : (uint32_t)left;
        return __builtin_amdgcn_make_buffer_rsrc(p, (short)0, (int)bytes, 0x00020000);
      }
      __device__ __forceinline__ void on(int rows) {
        p += rows * step;
        left -= rows * step;
      }
    };
    Row cr(g.c, g.ldc, kSize, g, mw, nw), ar(g.add, g.ldadd, 4, g, mw, nw);
#pragma unroll
    for (int x = 0; x < MI; ++x)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        __builtin_amdgcn_sched_barrier(0);
        float v[4][NI];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const auto ra = ar.here();
#pragma unroll
          for (int y = 0; y < NI; ++y) {
            v[i][y] = scale * acc[x][y][e + i] + bias[y];
            if constexpr (OUT & 1) v[i][y] += __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ra, (int)ao[y], 0, 0));
          }
          ar.on(i < 3 ? 1 : 5);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const auto rc = cr.here();
          cr.on(i < 3 ? 1 : 5);
#pragma unroll
          for (int y = 0; y < NI; ++y) {
            if constexpr (OUT >= 2) __builtin_amdgcn_raw_buffer_store_b16(f2bf(v[i][y]), rc, (int)oo[y], 0, 0);
            else __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[i][y]), rc, (int)oo[y], 0, kNt);
          }
        }
      }
    static_assert(MI * NI * 16 >= 63, "stores of a tile");
    fresh = 2;
#endif
  }
}

// The tiles that were taken in ranges of k: the ranges' sums in order, then the
// epilogue.
template <int BM, int BN>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
  const GemmBf16& g = a.g;
  const int t = blockIdx.x, tiles = gridDim.x;
  const float scale = g.scale ? *g.scale : 1.f;
  const int tile = a.whole + t;
  const int panel = 8 * a.gx, first = tile / panel * 8, high = min(8, a.gy - first), in = tile % panel;
  const int m0 = (first + in % high) * BM, n0 = in / high * BN;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < BM * BN / 4; i += gridDim.y * 256) {
    const int m = m0 + i * 4 / BN, n = n0 + i * 4 % BN;
    if (m >= g.M || n >= g.N) continue;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 16
    for (int r = 0; r < a.split; ++r)
      v += *reinterpret_cast<const f32x4*>(a.part + ((int64_t)r * tiles + t) * (BM * BN) + 4 * (int64_t)i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (n + j >= g.N) break;
      float x = scale * v[j] + (g.bias ? g.bias[n + j] : 0.f);
      if (g.add) x += g.add[(int64_t)m * g.ldadd + n + j];
      if (g.c_bf16) static_cast<bf16_t*>(g.c)[(int64_t)m * g.ldc + n + j] = f2bf(x);
      else static_cast<float*>(g.c)[(int64_t)m * g.ldc + n + j] = x;
    }
  }
}

// 64 rows x 128 columns a workgroup and step, four rows' eight columns a thread: whole 16
// bytes of a panel.  (Rows that are not aligned are read in 16 bytes all the same.)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
__global__ __launch_bounds__(256) void pack_kernel(const bf16_t* __restrict__ from, int64_t ldf, int64_t rows, int cols,
                                                   bf16_t* __restrict__ to, int64_t rows32, int panels) {
  const int across = (panels + 3) / 4;
  const int64_t blocks = (rows32 + 63) / 64 * across;
  for (int64_t i = blockIdx.x; i < blocks; i += gridDim.x) {
    const int64_t r0 = i / across * 64, r = r0 + threadIdx.x / 16;
    const int c0 = (int)(i % across) * 128, panel = c0 / 32 + threadIdx.x % 16 / 4, in = threadIdx.x % 4 * 8;
    const int c = panel * 32 + in;
    const bf16_t* p = from + r * ldf + c;
    u32x4 q[4];
    if (c0 + 128 <= cols && r0 + 64 <= rows) {
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = *reinterpret_cast<const u32x4_any*>(p + 16 * k * ldf);
    } else {
#pragma unroll 1
      for (int k = 0; k < 4; ++k) {
        bf16_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = r + 16 * k < rows && c + j < cols ? p[16 * k * ldf + j] : 0;
        const u32x4 x = {v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16, v[4] | (uint32_t)v[5] << 16,
                         v[6] | (uint32_t)v[7] << 16};
        q[0] = k == 0 ? x : q[0];
        q[1] = k == 1 ? x : q[1];
        q[2] = k == 2 ? x : q[2];
        q[3] = x;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (panel < panels && r + 16 * k < rows32)
        *reinterpret_cast<u32x4*>(to + (panel * rows32 + r + 16 * k) * 32 + in) = q[k];
  }
}

constexpr int kWgs = 512;  // two workgroups a compute unit

struct Plan {
  bool wide;  // tiles of 256 x 128, or 128 x 128
  int gx, gy, whole, split, per, units, ksteps;
  size_t bytes;
};
// Tiles that fill whole rounds of the chip are taken whole; those of the last round,
// where it is not full, in ranges of k that fill it.
Plan plan(int M, int N, int K, int pieces, bool stats = false) {
  Plan p{};
  p.ksteps = (K + BK - 1) / BK * pieces;
  p.wide = (int64_t)cdiv(M, 256) * cdiv(N, 128) >= kWgs / 2;
  const int bm = p.wide ? 256 : 128;
  p.gx = cdiv(N, 128);
  p.gy = cdiv(M, bm);
  const int tiles = p.gx * p.gy;
  const int rest = tiles % kWgs;
  p.whole = tiles - rest;
  // the number of ranges, of at least 8 stages each, after which the last round ends
  // soonest, in us: 0.5 a stage, 0.05 for a partial tile's way to memory and back, 5 for
  // the launch that joins them (linear cross entropy of 2 rows, C = 384, over 27453 columns, dx
  // in three pieces: 113 us in 16 ranges, 68 in 64)
  p.split = 1;
  double best = 1e30;
  for (int s = 1; rest && !stats && s <= std::min(64, std::max(1, p.ksteps / 8)); ++s) {
    const double cost = 0.5 * p.ksteps / s * cdiv(rest * s, kWgs) + (s > 1 ? 0.05 * rest * s + 5 : 0.0);
    if (cost < best) {
      best = cost;
      p.split = s;
    }
  }
  p.per = std::max(1, cdiv(p.ksteps, p.split));
  p.split = std::max(1, cdiv(p.ksteps, p.per));
  if (p.split == 1) p.whole = tiles;
  p.units = p.whole + (tiles - p.whole) * p.split;
  p.bytes = (size_t)(tiles - p.whole) * p.split * bm * 128 * 4;
  return p;
}

template <int MI, int OUT>
void launch_out(const Args& a, int wgs, hipStream_t st) {
  const dim3 grid(wgs), block(kThreads);
  if constexpr (OUT == 0 || OUT == 2 || OUT == 4) {  // (only products over rows are added up)
    if (a.g.a_k) {
      if (a.g.b_k) hipLaunchKernelGGL((gemm_bf16_kernel<MI, true, true, OUT>), grid, block, 0, st, a);
      else hipLaunchKernelGGL((gemm_bf16_kernel<MI, true, false, OUT>), grid, block, 0, st, a);
      return;
    }
  }
  if constexpr (OUT != 4) hipLaunchKernelGGL((gemm_bf16_kernel<MI, false, false, OUT>), grid, block, 0, st, a);
}
template <int MI>
void launch(const Args& a, int wgs, hipStream_t st) {
  if (a.g.stats) launch_out<MI, 4>(a, wgs, st);
  else if (a.g.c_bf16) a.g.add ? launch_out<MI, 3>(a, wgs, st) : launch_out<MI, 2>(a, wgs, st);
  else a.g.add ? launch_out<MI, 1>(a, wgs, st) : launch_out<MI, 0>(a, wgs, st);
}

}  // namespace

size_t gemm_bf16_workspace_bytes(int M, int N, int K, int pieces) {
  return M < 1 || N < 1 ? 0 : plan(M, N, K, pieces).bytes;
}

int gemm_bf16(const GemmBf16& g, void* workspace, hipStream_t st) {
  if (g.M == 0 || g.N == 0) return MTX_OK;
  const Plan p = plan(g.M, g.N, g.K, g.pieces, g.stats != nullptr);
  auto bad = [](const Bf16Matrix& m) {
    return ((uintptr_t)m.p & 15) || (m.row | m.panel | m.piece | m.size) % 8 || m.row >= kGemmBf16MaxLd ||
           m.panel >= kGemmBf16MaxPanel;
  };
  MTX_CHECK_ARG(g.K > 0 && (g.a_k ? !g.add : !g.b_k && !g.stats) && (!g.a_k || g.K % 8 == 0) && !bad(g.a) && !bad(g.b) &&
                    g.ldc < kGemmBf16MaxLdc && g.ldadd < kGemmBf16MaxLdc,
                "bf16 product: operand layout");
  const Args a{g, p.gx, p.gy, p.whole, p.split, p.units, p.ksteps, p.per, static_cast<float*>(workspace)};
  // (a multiple of 8: every XCD has as many workgroups)
  const int wgs = std::min(kWgs, cdiv(p.units, 8) * 8);
  if (p.wide) launch<4>(a, wgs, st);
  else launch<2>(a, wgs, st);
  MTX_LAUNCHED();
  const int joins = p.gx * p.gy - p.whole;
  if (joins) {
    if (p.wide) hipLaunchKernelGGL((join_kernel<256, 128>), dim3(joins, 8), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((join_kernel<128, 128>), dim3(joins, 8), dim3(256), 0, st, a);
    MTX_LAUNCHED();
  }
  return MTX_OK;
}

int pack_bf16(const bf16_t* from, int64_t ldf, int64_t rows, int cols, bf16_t* to, int64_t rows32, hipStream_t st) {
  const int panels = cdiv(cols, 32);
  const int64_t blocks = (rows32 + 63) / 64 * cdiv(panels, 4);
  hipLaunchKernelGGL(pack_kernel, dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), dim3(256), 0, st, from, ldf, rows,
                     cols, to, rows32, panels);
  MTX_LAUNCHED();
  return MTX_OK;
}

}  // namespace mtx
