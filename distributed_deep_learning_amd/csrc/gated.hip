// Gated feed-forward block (gfx950):   h = act(x Wg^T) * (x Wu^T),   y = h Wd^T        x [M][D], Wg and Wu [F][D], Wd [D][F], bf16
//
// Forward, two products:   up    both projections in one product: a block's columns are gate and up rows of the same features side by
//                                side, so that one lane holds g and u of a feature and the activation and the product are the epilogue;
//                                training also keeps P = u act'(g) and Q = act(g);
//                          down  y = h Wd^T.
// Backward, three:         dh    dy Wd, epilogue  dg = dh P,  du = dh Q  (dh itself is never written);
//                          dx    dg Wg + du Wu, one reduction over both pairs;
//                          dw    dg^T x, du^T x and dy^T h, one launch.
// A product is one launch, two where large tiles leave a rest to small ones, and one more where blocks share a tile's reduction (cut_of).
// All on the tiles of gemm_tile.h, which take the tensors as they lie: no transposed copy of a weight or an activation exists.
//
// Numbers.  Products accumulate in fp32.  h, dg and du are rounded to bf16 once, being operands of the next product at the bf16 rate.  P and Q
// only scale dh, so they need not be rounded twice as coarsely as that: they are kept in 24 bits (the upper 16 bits of the fp32 value in
// one plane, the next 8 in another; half-step 2^-17), 2 bytes more per feature and token than bf16 copies of g and u, which would add
// two more roundings of 2^-9 to every gradient (measured: relative error of dx, dWg, dWu 0.0031 with g and u in bf16, 0.0024 so).
// Few tokens leave few roundings to average over, and little work: up to 64 tokens h, dg and du are pairs of bf16 values (16 bits; what the
// rounding left is a second plane) and their products run over both planes, so that results have no rounding but their own (0.0017).
#include "common.h"
#include "host_util.h"
#include "gemm_tile.h"

namespace {

enum { SILU = 0, GELU = 1, RELU = 2 };

// a = act(g), d = act'(g)
template <int ACT> __device__ __forceinline__ void act_and_slope(float g, float& a, float& d) {
  if (ACT == SILU) {
    const float s = 1.f / (1.f + __expf(-g));
    a = g * s;
    d = s + a * (1.f - s);
  } else if (ACT == GELU) {
    const float c = 0.5f * (1.f + erff(g * 0.70710678f));
    a = g * c;
    d = c + g * __expf(-0.5f * g * g) * 0.39894228f;
  } else {
    a = g > 0.f ? g : (g != g ? g : 0.f);
    d = g > 0.f ? 1.f : (g != g ? g : 0.f);
  }
}

// fp32 values to 24 bits (round half up in the magnitude; NaN stays NaN) and back: upper 16 bits, next 8 bits
__device__ __forceinline__ unsigned round24(float v) { return v != v ? 0x7fc00000u : __float_as_uint(v) + 0x80u; }
template <int N> __device__ __forceinline__ void keep24(unsigned short* hi, unsigned char* lo, const float* v) {
  unsigned h[N / 2], l[N / 4];
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const unsigned r0 = round24(v[e]), r1 = round24(v[e + 1]), r2 = round24(v[e + 2]), r3 = round24(v[e + 3]);
    h[e / 2] = (r0 >> 16) | (r1 & 0xffff0000u);
    h[e / 2 + 1] = (r2 >> 16) | (r3 & 0xffff0000u);
    l[e / 4] = ((r0 >> 8) & 0xffu) | (r1 & 0xff00u) | ((r2 << 8) & 0xff0000u) | ((r3 << 16) & 0xff000000u);
  }
  if (N == 8) {
    *reinterpret_cast<u32x4*>(hi) = u32x4{h[0], h[1], h[2], h[3]};
    *reinterpret_cast<u32x2*>(lo) = u32x2{l[0], l[1]};
  } else {
    *reinterpret_cast<u32x2*>(hi) = u32x2{h[0], h[1]};
    *reinterpret_cast<unsigned*>(lo) = l[0];
  }
}
struct Kept { u32x4 h; u32x2 l; };
__device__ __forceinline__ Kept load24(const unsigned short* hi, const unsigned char* lo) {
  return Kept{*reinterpret_cast<const u32x4*>(hi), *reinterpret_cast<const u32x2*>(lo)};
}
__device__ __forceinline__ void get24(const Kept& k, float* v) {
  const u32x4 h = k.h;
  const u32x2 l = k.l;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const unsigned top = (e & 1) ? h[e / 2] & 0xffff0000u : h[e / 2] << 16;
    v[e] = __uint_as_float(top | (((l[e / 4] >> (8 * (e & 3))) & 0xffu) << 8));
  }
}

// Tile order: XCD-contiguous runs (t counts blocks that way) that sweep 8 tile rows column by column, so that the operand panels a run shares
// stay in that L2.
__device__ __forceinline__ void tile_of(unsigned t, int tm, int tn, int& i, int& j) {
  const unsigned per = 8u * (unsigned)tn, grp = t / per, in = t - grp * per;
  const unsigned rows = min(8u, (unsigned)tm - grp * 8u);
  j = (int)(in / rows);
  i = (int)(grp * 8u + in - (unsigned)j * rows);
}

// B operand of the up product: K-contiguous rows of two matrices, alternating by half the columns of a wave.
template <int BN> struct PairStager {
  static constexpr int NP = BN / 32, HALF = BN / 4, PJ = HALF / 32;      // HALF: features of a wave
  unsigned voff[NP];
  const unsigned short *gate, *up;
  int k, kdone, kchunk;
  __device__ __forceinline__ void init(const unsigned short* wg, const unsigned short* wu, long long ld, int f0, int feats, int K, int wid, int lane) {
    const int chunk = (lane & 7) ^ ((4 * (wid & 1) + (lane >> 4)) & 7);
    kchunk = chunk * 8; k = K; kdone = 0;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int f = (j / (2 * PJ)) * HALF + (j % PJ) * 32 + wid * 8 + (lane >> 3);
      voff[j] = f0 + f < feats ? (unsigned)(((long long)f * ld + chunk * 8) * 2) : gt::OOB;
    }
    gate = wg + (long long)f0 * ld;
    up = wu + (long long)f0 * ld;
  }
  u32x4 rg, ru;
  unsigned kill;
  __device__ __forceinline__ void begin() {
    rg = gt::make_rsrc(gate, 0xFFFFFFE0ull);
    ru = gt::make_rsrc(up, 0xFFFFFFE0ull);
    kill = kdone + kchunk >= k ? gt::OOB : 0u;
  }
  __device__ __forceinline__ void piece(int j, unsigned lds, int wid) const {
    gt::dma16(((j / PJ) & 1) ? ru : rg, lds + (unsigned)((j * 4 + wid) * 1024), voff[j] | kill);
  }
  __device__ __forceinline__ void end() { kdone += 64; gate += 64; up += 64; }
  __device__ __forceinline__ void part(int first, int n) {
    kdone = first * 64; gate += kdone; up += kdone;
    k = min(k, (first + n) * 64);
  }
};

// N operands of the same shape one after the other along the reduction: p0, p1, p0 + step, p1 + step.
template <class S, int N> struct Series {
  static constexpr int NP = S::NP;
  S s;
  const unsigned short *p0, *p1;
  long long step;
  int stages, left, seg;                          // stages of each;  of this one to come;  this one
  __device__ __forceinline__ void start(const unsigned short* a, const unsigned short* b, long long st, int nk) {
    p0 = a; p1 = b; step = st; stages = left = nk; seg = 0;
  }
  __device__ __forceinline__ const unsigned short* base() const { return ((seg & 1) ? p1 : p0) + (N > 2 && seg >= 2 ? step : 0); }
  __device__ __forceinline__ void part(int first, int) {
    seg = first / stages;
    first -= seg * stages;
    s.base = base();
    s.part(first, stages - first);
    left = stages - first;
  }
  __device__ __forceinline__ void begin() {
    if (left == 0) {
      if (seg + 1 < N) { ++seg; left = stages; s.base = base(); s.kdone = 0; }       // behind the last: zeros (kdone >= k)
      else left = 1 << 30;
    }
    --left;
    s.begin();
  }
  __device__ __forceinline__ void piece(int j, unsigned lds, int wid) const { s.piece(j, lds, wid); }
  __device__ __forceinline__ void end() { s.end(); }
};

struct GatedArgs {
  const unsigned short *x, *wg, *wu, *wd, *dy;
  unsigned short *h, *dg, *du, *y;
  unsigned short *hlo, *dglo, *dulo;               // null, or what the rounding of h, dg and du left: few tokens only
  void* dx;
  unsigned short* keep16; unsigned char* keep8;    // P then Q, [2][M][Fp]
  void *dwg, *dwu, *dwd;
  float* slabs;
  int M, D, F, Dp, Fp;                            // Dp, Fp: D and F padded to 8, the row lengths of all operands (the padding is zero)
  int dx32, dw;                                   // dx fp32 instead of bf16;  weight gradients: 0 bf16, 1 fp32 added to, 2 fp32
  int splits, per;                                // blocks that share the reduction of a tile, stages of each
  int first;                                      // 256 x 256 tiles that another launch does (Block::place)
};

__device__ __forceinline__ void store8(unsigned short* p, const float* v) { *reinterpret_cast<u32x4*>(p) = pack8(v); }
// what rounding to bf16 leaves of v; nothing of what is or becomes infinite (inf - inf would make it NaN)
__device__ __forceinline__ float lower(float v) {
  const float h = bf16_to_f32(f32_to_bf16(v));
  return __builtin_isinf(h) ? 0.f : v - h;
}
__device__ __forceinline__ void lower8(unsigned short* p, const float* v) {     // what store8 leaves
  float l[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) l[e] = lower(v[e]);
  store8(p, l);
}
// results have rows of their own length n: columns c .. c + 7 of row r
__device__ __forceinline__ void result16(unsigned short* p, long long r, int c, int n, const float* v) {
  p += r * n + c;
  if ((n & 7) == 0) { store8(p, v); return; }
#pragma unroll
  for (int e = 0; e < 8; ++e) if (c + e < n) p[e] = f32_to_bf16(v[e]);
}
__device__ __forceinline__ void result32(float* p, long long r, int c, int n, const float* v) {
  p += r * n + c;
  if ((n & 7) == 0) {
    *reinterpret_cast<f32x4*>(p) = *reinterpret_cast<const f32x4*>(v);
    *reinterpret_cast<f32x4*>(p + 4) = *reinterpret_cast<const f32x4*>(v + 4);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) if (c + e < n) p[e] = v[e];
}

// What a block of a product does.  The reduction of a tile may be shared by several blocks (few tiles, long reductions): each leaves its fp32
// partial tile in a slab, and the launch with JOIN adds them in order, a block per 16-row group, and does the epilogue.
template <int BT, int NST, bool JOIN> struct Block {
  using T = gt::Tile<BT, BT, NST>;
  static constexpr int NJ = JOIN ? 1 : T::FM;
  static constexpr bool SPLIT = BT == 128 && !JOIN;
  T tile;
  int tid, lane, wid, t, part;                    // t: the tile;  part: of its reduction (JOIN: its row group)
  // Tiles are dealt to the XCDs in runs, within `window` blocks at a time (0: all)
  __device__ __forceinline__ void begin(const GatedArgs& a, unsigned window = 0) {
    tid = threadIdx.x; lane = tid & 63; wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned before = window == 0 ? 0u : blockIdx.x / window * window, left = gridDim.x - before;
    t = (int)(before + xcd_remap(blockIdx.x - before, window == 0 ? left : min(window, left))); part = 0;
    if (JOIN) { part = t % T::FM; t /= T::FM; }
    else if (SPLIT && a.splits > 1) { part = t % a.splits; t /= a.splits; }
  }
  // Where tile `index` of a rows x cols result lies, COLS columns a tile; false: it is empty.  After a.first tiles of twice the size that another
  // launch does, index counts the quarters of tiles of that size.
  template <int COLS = BT> __device__ __forceinline__ bool place(const GatedArgs& a, int index, int rows, int cols, int& ti, int& tj) const {
    if (BT == 128 && a.first > 0) {
      tile_of((unsigned)index >> 2, (rows + 2 * BT - 1) / (2 * BT), (cols + 2 * COLS - 1) / (2 * COLS), ti, tj);
      ti = 2 * ti + ((index >> 1) & 1);
      tj = 2 * tj + (index & 1);
      return ti * BT < rows && tj * COLS < cols;
    }
    tile_of((unsigned)index, (rows + BT - 1) / BT, (cols + COLS - 1) / COLS, ti, tj);
    return true;
  }
  __device__ __forceinline__ int index(const GatedArgs& a) const { return BT == 128 ? t + 4 * a.first : t; }
  // true: the tile's epilogue is this block's
  template <int AM, int BMD, class SA, class SB> __device__ __forceinline__ bool product(const GatedArgs& a, SA& sa, SB& sb, int nk, char* smem) {
    float* const slab = a.slabs + (long long)t * a.splits * T::SLAB;
    if (JOIN) { tile.sum_slabs(slab, a.splits, part, tid); return true; }
    if (SPLIT && a.splits > 1) {
      const int first = part * a.per;
      nk = min(a.per, nk - first);
      sa.part(first, nk);
      sb.part(first, nk);
    }
    tile.zero();
    tile.template mul<gt::Bf16, AM, BMD, 1>(sa, sb, nk, smem, wid, lane);
    if (SPLIT && a.splits > 1) { tile.put_slab(slab + (long long)part * T::SLAB, tid); return false; }
    return true;
  }
  template <class LD, class F> __device__ __forceinline__ void store(char* smem, LD&& load, F&& f) {
    tile.template store<false, NJ>(smem, wid, lane, load, f, [](int, int, float*) {}, JOIN ? part : 0);
  }
};
// Measured at 8192 tokens, 4096 x 12288 (256 x 256 tiles): up 1.37 ms (1.20 PFLOP/s), down 0.65 (1.26), dh 0.82 (1.00), dx 1.38 (1.20), dw 2.08 (1.19).
// The clock is at 2.0 to 2.15 GHz and the matrix units are busy 53, 55, 43, 52 and 52 % of its cycles; schedules with 10 to 16 % fewer cycles ran at
// 1.8 GHz, no faster.  A library's plain products of these sizes reach 1.55, 1.59, 1.30, 1.39 and 1.14 PFLOP/s, without the epilogues.
// Measured at 517 tokens, 2048 x 5632 (128 x 128 tiles): up 37 us (440 blocks; 0.65 PFLOP/s), down 22 us in 240 parts and 4.5 us to join them,
// 53 us in 80 whole tiles.
#define GATED_BOUNDS __launch_bounds__(256, BT == 256 || NST > 2 ? 1 : 2)

// g and u of a feature in one lane: half of a wave's columns are gate rows, half up rows (PairStager).  SAVE adds 6 bytes a feature to write.
template <int BT, int NST, bool JOIN, int ACT, bool SAVE> __global__ GATED_BOUNDS void gated_up_kernel(const GatedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Block<BT, NST, JOIN> b;
  b.begin(a);
  int ti, tj;
  if (!b.template place<BT / 2>(a, b.index(a), a.M, a.F, ti, tj)) return;
  const int m0 = ti * BT, f0 = tj * (BT / 2);
  gt::Stager<BT, gt::CONTIG, 1> sa;
  PairStager<BT> sb;
  sa.init(gt::Operand{a.x, a.Dp, m0, a.M, a.D}, b.wid, b.lane);
  sb.init(a.wg, a.wu, a.Dp, f0, a.F, a.D, b.wid, b.lane);
  if (!b.template product<gt::CONTIG, gt::CONTIG>(a, sa, sb, (a.D + 63) / 64, smem)) return;
  b.tile.template store_pairs<b.NJ>(smem, b.wid, b.lane, [&](int r, int f, const float* g, const float* u) {
    r += m0; f += f0;
    if (r >= a.M || f >= a.Fp) return;
    const long long o = (long long)r * a.Fp + f;
    float h[8], p[8], q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float d;
      act_and_slope<ACT>(g[e], q[e], d);
      p[e] = u[e] * d;
      h[e] = q[e] * u[e];
    }
    store8(a.h + o, h);
    if (SAVE) {
      const long long plane = (long long)a.M * a.Fp;
      keep24<8>(a.keep16 + o, a.keep8 + o, p);
      keep24<8>(a.keep16 + plane + o, a.keep8 + plane + o, q);
    }
  }, JOIN ? b.part : 0);
}

// Both operands as they lie, K-contiguous.  Few tiles and a long reduction in small batches: the first to be shared by blocks.
template <int BT, int NST, bool JOIN> __global__ GATED_BOUNDS void gated_down_kernel(const GatedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Block<BT, NST, JOIN> b;
  b.begin(a);
  int ti, tj;
  if (!b.place(a, b.index(a), a.M, a.D, ti, tj)) return;
  const int m0 = ti * BT, n0 = tj * BT;
  gt::Stager<BT, gt::CONTIG, 1> sa, sb;
  sa.init(gt::Operand{a.h, a.Fp, m0, a.M, a.F}, b.wid, b.lane);
  sb.init(gt::Operand{a.wd, a.Fp, n0, a.D, a.F}, b.wid, b.lane);
  if (!b.template product<gt::CONTIG, gt::CONTIG>(a, sa, sb, (a.F + 63) / 64, smem)) return;
  b.store(smem, gt::NoLoad{}, [&](int r, int c, const float* v, gt::None) {
    r += m0; c += n0;
    if (r < a.M && c < a.D) result16(a.y, r, c, a.D, v);
  });
}

// Wd is K-slow here.  The shortest reduction and the widest epilogue (6 bytes read, 4 written per element, read a row group ahead): the lowest rate.
template <int BT, int NST, bool JOIN, bool LO> __global__ GATED_BOUNDS void gated_dh_kernel(const GatedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Block<BT, NST, JOIN> b;
  b.begin(a);
  int ti, tj;
  if (!b.place(a, b.index(a), a.M, a.F, ti, tj)) return;
  const int m0 = ti * BT, n0 = tj * BT;
  gt::Stager<BT, gt::CONTIG, 1> sa;
  gt::Stager<BT, gt::SLOW, 1> sb;
  sa.init(gt::Operand{a.dy, a.Dp, m0, a.M, a.D}, b.wid, b.lane);
  sb.init(gt::Operand{a.wd, a.Fp, n0, a.Fp, a.D}, b.wid, b.lane);
  if (!b.template product<gt::CONTIG, gt::SLOW>(a, sa, sb, (a.D + 63) / 64, smem)) return;
  const long long plane = (long long)a.M * a.Fp;
  struct Factors { Kept p, q; };
  auto load = [&](int r, int c) {
    r += m0; c += n0;
    const long long o = (long long)r * a.Fp + c;
    Factors k{};
    if (r < a.M && c < a.Fp) { k.p = load24(a.keep16 + o, a.keep8 + o); k.q = load24(a.keep16 + plane + o, a.keep8 + plane + o); }
    return k;
  };
  b.store(smem, load, [&](int r, int c, const float* v, const Factors& k) {
    r += m0; c += n0;
    if (r >= a.M || c >= a.Fp) return;
    const long long o = (long long)r * a.Fp + c;
    float p[8], q[8], dg[8], du[8];
    get24(k.p, p);
    get24(k.q, q);
#pragma unroll
    for (int e = 0; e < 8; ++e) { dg[e] = v[e] * p[e]; du[e] = v[e] * q[e]; }
    store8(a.dg + o, dg);
    store8(a.du + o, du);
    if (LO) { lower8(a.dglo + o, dg); lower8(a.dulo + o, du); }
  });
}

// dg Wg + du Wu as one reduction of twice the length: dx is written once and never read back.
template <int BT, int NST, bool JOIN, bool LO> __global__ GATED_BOUNDS void gated_dx_kernel(const GatedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Block<BT, NST, JOIN> b;
  b.begin(a);
  int ti, tj;
  if (!b.place(a, b.index(a), a.M, a.D, ti, tj)) return;
  const int m0 = ti * BT, n0 = tj * BT, nk = (a.F + 63) / 64;
  constexpr int N = LO ? 4 : 2;
  Series<gt::Stager<BT, gt::CONTIG, 1>, N> sa;
  Series<gt::Stager<BT, gt::SLOW, 1>, N> sb;
  const long long row = (long long)m0 * a.Fp;
  sa.s.init(gt::Operand{a.dg, a.Fp, m0, a.M, a.F}, b.wid, b.lane);
  sa.start(a.dg + row, a.du + row, LO ? a.dglo - a.dg : 0, nk);
  sb.s.init(gt::Operand{a.wg, a.Dp, n0, a.Dp, a.F}, b.wid, b.lane);
  sb.start(a.wg, a.wu, 0, nk);
  if (!b.template product<gt::CONTIG, gt::SLOW>(a, sa, sb, N * nk, smem)) return;
  b.store(smem, gt::NoLoad{}, [&](int r, int c, const float* v, gt::None) {
    r += m0; c += n0;
    if (r >= a.M || c >= a.D) return;
    if (a.dx32) result32((float*)a.dx, r, c, a.D, v);
    else result16((unsigned short*)a.dx, r, c, a.D, v);
  });
}

// Three products of one size in one launch, all operands K-slow (transposing LDS reads), one after the other over the whole chip: spread over the
// XCDs at the same time they took 2.15 ms.
template <int BT, int NST, bool JOIN, bool LO> __global__ GATED_BOUNDS void gated_dw_kernel(const GatedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Block<BT, NST, JOIN> b;
  const bool rest = BT == 128 && a.first > 0;
  const int size = rest ? 256 : BT, each = ((a.F + size - 1) / size) * ((a.D + size - 1) / size) * (rest ? 4 : 1);
  b.begin(a, rest ? 0u : (unsigned)(each * (JOIN ? gt::Tile<BT, BT>::FM : BT == 128 ? a.splits : 1)));
  const int which = b.index(a) / each, rows = which == 2 ? a.D : a.F, cols = which == 2 ? a.F : a.D;
  int ti, tj;
  if (!b.place(a, b.index(a) - which * each, rows, cols, ti, tj)) return;
  const int lda = which == 2 ? a.Dp : a.Fp, ldb = which == 2 ? a.Fp : a.Dp;
  const unsigned short* const pa = which == 0 ? a.dg : which == 1 ? a.du : a.dy;
  const unsigned short* const pb = which == 2 ? a.h : a.x;
  void* const out = which == 0 ? a.dwg : which == 1 ? a.dwu : a.dwd;
  if (out == nullptr) return;
  const int m0 = ti * BT, n0 = tj * BT;
  if constexpr (LO) {
    Series<gt::Stager<BT, gt::SLOW, 1>, 2> sa, sb;
    const int nk = (a.M + 63) / 64;
    sa.s.init(gt::Operand{pa, lda, m0, lda, a.M}, b.wid, b.lane);
    sb.s.init(gt::Operand{pb, ldb, n0, ldb, a.M}, b.wid, b.lane);
    sa.start(pa, which == 0 ? a.dglo : which == 1 ? a.dulo : a.dy, 0, nk);
    sb.start(pb, which == 2 ? a.hlo : a.x, 0, nk);
    if (!b.template product<gt::SLOW, gt::SLOW>(a, sa, sb, 2 * nk, smem)) return;
  } else {
    gt::Stager<BT, gt::SLOW, 1> sa, sb;
    sa.init(gt::Operand{pa, lda, m0, lda, a.M}, b.wid, b.lane);
    sb.init(gt::Operand{pb, ldb, n0, ldb, a.M}, b.wid, b.lane);
    if (!b.template product<gt::SLOW, gt::SLOW>(a, sa, sb, (a.M + 63) / 64, smem)) return;
  }
  struct Sum { f32x4 lo, hi; };
  auto load = [&](int r, int c) {
    r += m0; c += n0;
    Sum q{};
    if (a.dw == 1 && r < rows && c < cols) {
      const float* const p = (const float*)out + (long long)r * cols + c;
      if ((cols & 7) == 0) {
        q = Sum{*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 4)};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (c + e < cols) q.lo[e] = p[e];
          if (c + e + 4 < cols) q.hi[e] = p[e + 4];
        }
      }
    }
    return q;
  };
  b.store(smem, load, [&](int r, int c, float* v, const Sum& q) {
    r += m0; c += n0;
    if (r >= rows || c >= cols) return;
    if (a.dw == 0) { result16((unsigned short*)out, r, c, cols, v); return; }
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] += q.lo[e]; v[e + 4] += q.hi[e]; }
    result32((float*)out, r, c, cols, v);
  });
}

// Operands as the products take them: bf16, rows padded with zeros to 8 elements (16 bytes), contiguous.  What is so already is used as it lies;
// the rest (fp32, other widths or row strides) is copied here, all in one launch.
struct PadJob { const void* src; unsigned short* dst; long long stride, first; int rows, cols, is32, wide; };
struct PadArgs { PadJob job[4]; int n; long long total; };
__global__ __launch_bounds__(256) void gated_pad_kernel(const PadArgs a) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < a.total; i += (long long)gridDim.x * 256) {
    int j = 0;
    while (j + 1 < a.n && i >= a.job[j + 1].first) ++j;
    const PadJob& q = a.job[j];
    const int per = (q.cols + 7) / 8;
    const long long in = i - q.first, row = in / per;
    const int c = (int)(in - row * per) * 8;
    const long long at = row * q.stride + c;
    float v[8];
    if (q.wide && q.is32) {
      *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>((const float*)q.src + at);
      *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>((const float*)q.src + at + 4);
    } else if (q.wide) {
      *reinterpret_cast<u32x4*>(q.dst + in * 8) = *reinterpret_cast<const u32x4*>((const unsigned short*)q.src + at);
      continue;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = c + e >= q.cols ? 0.f : q.is32 ? ((const float*)q.src)[at + e] : bf16_to_f32(((const bf16_t*)q.src)[at + e]);
    }
    store8(q.dst + in * 8, v);
  }
}

// ---- few tokens (serving): bound by reading the weights once.  A block owns 16 features (their gate and up rows, or 16 rows of Wd); its waves
// share the reduction in steps of 64 (one 128-byte line of each row; wave w takes steps w, w + WAVES, ...), load the weights straight into
// matrix-instruction operands - nothing is staged, every byte is used once - several steps ahead, and add their fp32 tiles in LDS in a fixed order.
// 1 token, 4096 x 12288: up 36 us (201 MB of weights, 5.6 TB/s), down 19 us (5.3 TB/s); in 128 x 128 tiles the two took 231 us.  65 tokens and more
// are faster in tiles.
// TB: blocks of 16 columns.  LO: h goes from one product to the other as a pair of bf16 values; the lower ones take the second half of the columns
// (up to 8 tokens one block serves for both, at no cost).
template <int TB, int WAVES, bool PAIR, int ACT, bool SAVE, bool LO>
__global__ __launch_bounds__(64 * WAVES) void gated_few_kernel(const GatedArgs a) {
  constexpr int NM = PAIR ? 2 : 1, U = TB == 4 ? 2 : 4;                  // weight matrices; steps in flight
  constexpr bool TWO = LO && !PAIR;                                      // upper and lower values of h
  constexpr int COLS = TWO ? TB * 8 : TB * 16;                           // columns for tokens
  __shared__ f32x4 red[WAVES][NM * TB][64];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 15, kc = (lane >> 4) * 8;
  const int K = PAIR ? a.D : a.F, N = PAIR ? a.F : a.D, ld = PAIR ? a.Dp : a.Fp;   // reduction, rows of the weights, row length of both operands
  const int f0 = blockIdx.x * 16;
  const unsigned short* const in = PAIR ? a.x : a.h;
  const unsigned long long wbytes = (unsigned long long)(N - f0 < 16 ? N - f0 : 16) * (unsigned long long)ld * 2ull;
  const __amdgpu_buffer_rsrc_t w0 = __builtin_amdgcn_make_buffer_rsrc((void*)((PAIR ? a.wg : a.wd) + (long long)f0 * ld), 0, (int)wbytes, 0x00020000);
  const __amdgpu_buffer_rsrc_t w1 = __builtin_amdgcn_make_buffer_rsrc((void*)((PAIR ? a.wu : a.wd) + (long long)f0 * ld), 0, (int)wbytes, 0x00020000);
  const unsigned lo = TWO ? (unsigned)(a.hlo - a.h) : 0u;         // elements from the upper to the lower values
  const __amdgpu_buffer_rsrc_t xs = __builtin_amdgcn_make_buffer_rsrc((void*)in, 0, (int)(((unsigned long long)a.M * ld + lo) * 2ull), 0x00020000);
  f32x4 acc[NM][TB];
#pragma unroll
  for (int m = 0; m < NM; ++m)
#pragma unroll
    for (int t = 0; t < TB; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = (K + 63) / 64;
  for (int s = wid; s < steps; s += WAVES * U) {
    u32x4 w[U][2][NM], x[U][2][TB];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = (s + u * WAVES) * 64 + h * 32 + kc;
        const bool in_k = k < K;                                         // a last piece ends in the padding
        const unsigned off = in_k ? (unsigned)(row * ld + k) * 2u : gt::OOB;
        w[u][h][0] = __builtin_amdgcn_raw_buffer_load_b128(w0, (int)off, 0, 0);
        if (PAIR) w[u][h][NM - 1] = __builtin_amdgcn_raw_buffer_load_b128(w1, (int)off, 0, 0);
#pragma unroll
        for (int t = 0; t < TB; ++t) {
          const int col = t * 16 + row, tok = col % COLS;
          const unsigned xo = in_k && tok < a.M ? ((unsigned)(tok * ld + k) + (col >= COLS ? lo : 0u)) * 2u : gt::OOB;
          x[u][h][t] = __builtin_amdgcn_raw_buffer_load_b128(xs, (int)xo, 0, 0);
        }
      }
    __builtin_amdgcn_sched_barrier(0);                                   // all of them requested before the first is used
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
          for (int t = 0; t < TB; ++t)
            acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w[u][h][m]), __builtin_bit_cast(bf16x8, x[u][h][t]),
                                                                 acc[m][t], 0, 0, 0);
  }
#pragma unroll
  for (int m = 0; m < NM; ++m)
#pragma unroll
    for (int t = 0; t < TB; ++t) red[wid][m * TB + t][lane] = acc[m][t];
  __syncthreads();
  for (int i = tid; i < TB * 64; i += 64 * WAVES) {
    const int t = i >> 6, l = i & 63, tok = t * 16 + (l & 15), f = f0 + (l >> 4) * 4;
    if (tok >= a.M || tok >= COLS || f >= (PAIR ? a.Fp : N)) continue;
    f32x4 v[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      v[m] = red[0][m * TB + t][l];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) {
        const f32x4 o = red[w][m * TB + t][l];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[m][e] += o[e];
      }
      if (TWO) {                                                         // the same token's lower values: COLS columns further
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          const f32x4 o = TB == 1 ? red[w][0][(l + 8) & 63] : red[w][t + TB / 2][l];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[m][e] += o[e];
        }
      }
    }
    const long long o = (long long)tok * (PAIR ? a.Fp : N) + f;
    float y[4], p[4], q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (PAIR) {
        float d;
        act_and_slope<ACT>(v[0][e], q[e], d);
        p[e] = v[NM - 1][e] * d;
        y[e] = q[e] * v[NM - 1][e];
      } else {
        y[e] = v[0][e];
      }
    }
    if (LO && PAIR) {
      float l[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) l[e] = lower(y[e]);
      *reinterpret_cast<u32x2*>(a.hlo + o) = u32x2{pack_bf16x2(l[0], l[1]), pack_bf16x2(l[2], l[3])};
    }
    if (PAIR || (N & 3) == 0) {
      *reinterpret_cast<u32x2*>((PAIR ? a.h : a.y) + o) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) if (f + e < N) a.y[o + e] = f32_to_bf16(y[e]);
    }
    if (SAVE) {
      const long long plane = (long long)a.M * a.Fp;
      keep24<4>(a.keep16 + o, a.keep8 + o, p);
      keep24<4>(a.keep16 + plane + o, a.keep8 + plane + o, q);
    }
  }
}

inline long long tiles(int n, int t) { return ((long long)n + t - 1) / t; }

// one launch of a kernel that takes GatedArgs; opts in to its LDS once per device
template <int BT, int NST, auto KERNEL> int launch(long long blocks, const GatedArgs& a, void* stream) {
  static SmemAttrOnce once;
  if (blocks <= 0 || blocks > 0x7fffffffll) return -2;
  constexpr int smem = gt::Tile<BT, BT, NST>::SMEM;
  const int rc = once.ensure(reinterpret_cast<const void*>(KERNEL), smem);
  if (rc != 0) return rc;
  hipLaunchKernelGGL(KERNEL, dim3((unsigned)blocks), dim3(256), smem, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

// How `count` products of rows x cols over ks stages are cut, by estimated times in stages of a CU's pair of 128 x 128 tiles (about 1 us).  Measured
// rounds: 512 small tiles ks + 6;  256 large ones, four times the work of half as many blocks, 1.75 (ks + 7.5) (9 stages 30 us, 16 42, 32 73, 64 120).
// Large tiles may take whole rounds of the chip and leave the rest to small ones, whose reductions can be shared: 6000 x 4096 x 11008 forward and
// backward 4.79 -> 4.30 ms;  3000 x 2048 x 5632 0.85 -> 0.74.
struct Cut { int first, splits, per; long long tiles; };                    // large tiles;  then small ones
Cut cut_of(int count, int rows, int cols, int ks, bool small_only = false) {
  const long long big = count * tiles(rows, 256) * tiles(cols, 256), rounds = big / gt::CUS, rest = big - rounds * gt::CUS;
  const double round = 1.75 * (ks + 7.5);
  Cut c{0, 1, ks, count * tiles(rows, 128) * tiles(cols, 128)};
  double small = 0.0, ends = 0.0;
  c.per = gt::chunk_for(c.tiles, ks, &small);
  if (c.per == ks && c.tiles > gt::SLOTS) {               // several rounds overlap: a last one of single blocks is shorter, many drift apart
    const long long full = c.tiles / gt::SLOTS, left = c.tiles - full * gt::SLOTS;
    const double steps = (double)full + (left == 0 ? 0.0 : left <= gt::CUS ? 0.6 : 1.0), drift = (double)c.tiles / gt::SLOTS + 0.25;
    small = (steps < drift ? steps : drift) * (ks + 6);
  }
  if (!small_only && big < (1 << 28)) {
    const int per = rest > 0 ? gt::chunk_for(4 * rest, ks, &ends) : ks;
    const double whole = round * (double)(rounds + (rest > 0)), mixed = round * (double)rounds + ends + 8;      // 8: a launch more
    if (whole < small && whole <= mixed) c = Cut{(int)big, 1, ks, 0};
    else if (rounds > 0 && mixed < small) c = Cut{(int)(rounds * gt::CUS), 1, per, 4 * rest};
  }
  c.splits = (ks + c.per - 1) / c.per;
  return c;
}
long long slab_floats(const Cut& c) { return c.splits > 1 ? c.tiles * c.splits * gt::Tile<128, 128>::SLAB : 0; }

// P::at<BT, NST, JOIN>: the kernel
template <class P> int product(const Cut& c, GatedArgs a, void* st) {
  a.splits = c.splits; a.per = c.per;
  if (c.splits > 1 && a.slabs == nullptr) return -1;
  int rc = 0;
  if constexpr (P::LARGE) {
    if (c.first > 0) rc = launch<256, 2, P::template at<256, 2, false>>(c.first, a, st);
  }
  if (rc != 0 || c.tiles == 0) return rc;
  a.first = c.first;
  const long long blocks = c.tiles * c.splits;
  rc = blocks <= gt::CUS ? launch<128, 4, P::template at<128, 4, false>>(blocks, a, st)
                         : launch<128, 2, P::template at<128, 2, false>>(blocks, a, st);
  if (rc == 0 && c.splits > 1) rc = launch<128, 2, P::template at<128, 2, true>>(c.tiles * gt::Tile<128, 128>::FM, a, st);
  return rc;
}
template <int ACT, bool SAVE> struct Up {
  static constexpr bool LARGE = true;
  template <int BT, int NST, bool JOIN> static constexpr auto at = &gated_up_kernel<BT, NST, JOIN, ACT, SAVE>;
};
struct Down { static constexpr bool LARGE = true; template <int BT, int NST, bool JOIN> static constexpr auto at = &gated_down_kernel<BT, NST, JOIN>; };
template <bool LO> struct Dh {
  static constexpr bool LARGE = !LO;
  template <int BT, int NST, bool JOIN> static constexpr auto at = &gated_dh_kernel<BT, NST, JOIN, LO>;
};
template <bool LO> struct Dx {
  static constexpr bool LARGE = !LO;
  template <int BT, int NST, bool JOIN> static constexpr auto at = &gated_dx_kernel<BT, NST, JOIN, LO>;
};
template <bool LO> struct Dw {
  static constexpr bool LARGE = !LO;
  template <int BT, int NST, bool JOIN> static constexpr auto at = &gated_dw_kernel<BT, NST, JOIN, LO>;
};

int stages(int k) { return (int)tiles(k, 64); }
inline int pad8(int n) { return (n + 7) & ~7; }

// A lane addresses its rows of a tile with 32-bit byte offsets: up to 2^24 elements a row in 128-row tiles (127 * 2^25 bytes), 2^23 in 256-row ones.
constexpr int WIDEST = 1 << 24, WIDEST_LARGE = 1 << 23;
bool sizes_ok(int M, int D, int F) { return M > 0 && D > 0 && F > 0 && M <= 0x7fffff00 && D <= WIDEST && F <= WIDEST; }
bool long_rows(int D, int F) { return pad8(D) > WIDEST_LARGE || pad8(F) > WIDEST_LARGE; }

Cut cut_up(int M, int D, int F) { return cut_of(1, M, 2 * F, stages(D), long_rows(D, F)); }
Cut cut_down(int M, int D, int F) { return cut_of(1, M, D, stages(F), long_rows(D, F)); }
Cut cut_dh(int M, int D, int F, bool lo) { return cut_of(1, M, F, stages(D), lo || long_rows(D, F)); }
Cut cut_dx(int M, int D, int F, bool lo) { return cut_of(1, M, D, (lo ? 4 : 2) * stages(F), lo || long_rows(D, F)); }
Cut cut_dw(int M, int D, int F, bool lo) { return cut_of(3, F, D, (lo ? 2 : 1) * stages(M), lo || long_rows(D, F)); }

constexpr int FEW = 64;                            // tokens up to which gated_few_kernel is used

template <int TB, bool PAIR, int ACT, bool SAVE, bool LO> int launch_few_t(const GatedArgs& a, void* st) {
  constexpr int WAVES = PAIR ? 8 : 16;             // Wd has fewer rows (a third of the blocks) and a longer reduction
  hipLaunchKernelGGL(HIP_KERNEL_NAME(gated_few_kernel<TB, WAVES, PAIR, ACT, SAVE, LO>), dim3((unsigned)tiles(PAIR ? a.F : a.D, 16)),
                     dim3(64 * WAVES), 0, (hipStream_t)st, a);
  return (int)hipGetLastError();
}
template <bool PAIR, int ACT, bool SAVE> int launch_few(const GatedArgs& a, void* st) {
  if (a.hlo != nullptr && PAIR)
    return a.M <= 16 ? launch_few_t<1, PAIR, ACT, SAVE, true>(a, st) : a.M <= 32 ? launch_few_t<2, PAIR, ACT, SAVE, true>(a, st)
                                                                                 : launch_few_t<4, PAIR, ACT, SAVE, true>(a, st);
  if (a.hlo != nullptr && a.M <= 32)               // twice the columns
    return a.M <= 8 ? launch_few_t<1, PAIR, ACT, SAVE, true>(a, st) : a.M <= 16 ? launch_few_t<2, PAIR, ACT, SAVE, true>(a, st)
                                                                                : launch_few_t<4, PAIR, ACT, SAVE, true>(a, st);
  return a.M <= 16 ? launch_few_t<1, PAIR, ACT, SAVE, false>(a, st) : a.M <= 32 ? launch_few_t<2, PAIR, ACT, SAVE, false>(a, st)
                                                                                : launch_few_t<4, PAIR, ACT, SAVE, false>(a, st);
}
template <int ACT> int few_up(const GatedArgs& a, bool save, void* st) {
  return save ? launch_few<true, ACT, true>(a, st) : launch_few<true, ACT, false>(a, st);
}
// 32-bit offsets inside 16 rows of a weight and inside the tokens
bool few(int M, int K) { return M <= FEW && (long long)FEW * K * 2 < 0x7fffffffll; }

// h, dg and du as pairs: offsets between the planes in 32 bits too
bool pairs(int M, int Dp, int Fp) { return few(M, Dp) && (long long)FEW * Fp * 10 < 0x7fffffffll; }

template <int ACT> int up(const GatedArgs& a, void* st) {
  const bool save = a.keep16 != nullptr;
  if (few(a.M, a.Dp)) return few_up<ACT>(a, save, st);
  const Cut c = cut_up(a.M, a.D, a.F);
  return save ? product<Up<ACT, true>>(c, a, st) : product<Up<ACT, false>>(c, a, st);
}

}  // namespace

// Floats of partial tiles that a forward (0) or backward pass (1: dh and dx, 2: weight gradients) needs
extern "C" long long ddl_gated_workspace(int M, int D, int F, int pass) {
  if (!sizes_ok(M, D, F) || pass < 0 || pass > 2) return -1;
  long long n = 0;
  auto most = [&](const Cut& c) { n = max(n, slab_floats(c)); };
  if (pass == 0) {
    if (!few(M, pad8(D))) most(cut_up(M, D, F));
    if (!few(M, pad8(F))) most(cut_down(M, D, F));
  }
  const bool lo = pairs(M, pad8(D), pad8(F));
  if (pass == 1) { most(cut_dh(M, D, F, lo)); most(cut_dx(M, D, F, lo)); }
  if (pass == 2) most(cut_dw(M, D, F, lo));
  return n;
}

// n <= 4 matrices [rows][cols] with the given row strides (elements) -> bf16 [rows][cols padded to 8]
extern "C" int ddl_gated_pad(const void* const* src, void* const* dst, const int* rows, const int* cols, const long long* stride, const int* is32,
                             int n, void* stream) {
  if (n < 1 || n > 4) return -1;
  PadArgs a{};
  a.n = n;
  for (int i = 0; i < n; ++i) {
    if (rows[i] < 0 || cols[i] <= 0) return -1;
    PadJob& j = a.job[i];
    j = PadJob{src[i], (unsigned short*)dst[i], stride[i], a.total, rows[i], cols[i], is32[i], 0};
    j.wide = cols[i] % 8 == 0 && stride[i] % (is32[i] ? 4 : 8) == 0 && (unsigned long long)src[i] % 16 == 0;
    a.total += (long long)rows[i] * (pad8(cols[i]) / 8);
  }
  if (a.total == 0) return 0;
  hipLaunchKernelGGL(gated_pad_kernel, dim3(grid_for(a.total, 256, 16384)), dim3(256), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

// x [M][Dp], wg and wu [F][Dp], wd [D][Fp], h [M][Fp], y [M][D];  keep16 [2][M][Fp] (16 bit) and keep8 [2][M][Fp] (8 bit), or both null: what
// the backward pass needs;  hlo [M][Fp] behind h in the same allocation, up to 64 tokens (else unused).  Dp and Fp: D and F padded to 8 with zeros.
extern "C" int ddl_gated_fwd(const void* x, const void* wg, const void* wu, const void* wd, void* h, void* hlo, void* keep16, void* keep8, void* y,
                             float* slabs, int M, int D, int F, int act, void* stream) {
  if (!sizes_ok(M, D, F) || (keep16 == nullptr) != (keep8 == nullptr)) return -1;
  GatedArgs a{};
  a.x = (const unsigned short*)x; a.wg = (const unsigned short*)wg; a.wu = (const unsigned short*)wu; a.wd = (const unsigned short*)wd;
  a.h = (unsigned short*)h; a.keep16 = (unsigned short*)keep16; a.keep8 = (unsigned char*)keep8; a.y = (unsigned short*)y;
  a.slabs = slabs;
  a.M = M; a.D = D; a.F = F; a.Dp = pad8(D); a.Fp = pad8(F);
  if (pairs(M, a.Dp, a.Fp) && (M <= 32 || keep16 != nullptr)) a.hlo = (unsigned short*)hlo;
  int rc = -1;
  if (act == SILU) rc = up<SILU>(a, stream);
  else if (act == GELU) rc = up<GELU>(a, stream);
  else if (act == RELU) rc = up<RELU>(a, stream);
  if (rc != 0) return rc;
  return few(M, a.Fp) ? launch_few<false, SILU, false>(a, stream) : product<Down>(cut_down(M, D, F), a, stream);
}

// pass: 1 dg and du (and dx, unless null), 2 weight gradients (those that are not null; they take dg and du).  dy [M][Dp], dgu: dg, du and,
// up to 64 tokens, what their rounding left, [M][Fp] each, dx [M][D] bf16 or (dx32) fp32, dwg and dwu [F][D], dwd [D][F]: dw 0 bf16, 1 fp32 that are added to, 2 fp32
extern "C" int ddl_gated_bwd(const void* x, const void* dy, const void* wg, const void* wu, const void* wd, const void* h, const void* hlo,
                             const void* keep16, const void* keep8, void* dgu, void* dx, int dx32, void* dwg, void* dwu, void* dwd, int dw, float* slabs,
                             int M, int D, int F, int pass, void* stream) {
  if (!sizes_ok(M, D, F) || pass < 1 || pass > 2 || dw < 0 || dw > 2) return -1;
  GatedArgs a{};
  a.x = (const unsigned short*)x; a.dy = (const unsigned short*)dy;
  a.wg = (const unsigned short*)wg; a.wu = (const unsigned short*)wu; a.wd = (const unsigned short*)wd;
  a.h = (unsigned short*)h; a.keep16 = (unsigned short*)keep16; a.keep8 = (unsigned char*)keep8;
  a.dx = dx; a.dx32 = dx32;
  a.dwg = dwg; a.dwu = dwu; a.dwd = dwd; a.dw = dw;
  a.slabs = slabs;
  a.M = M; a.D = D; a.F = F; a.Dp = pad8(D); a.Fp = pad8(F);
  const long long plane = (long long)M * a.Fp;
  a.dg = (unsigned short*)dgu;
  if (dgu != nullptr) { a.du = a.dg + plane; a.dglo = a.du + plane; a.dulo = a.dglo + plane; }
  a.hlo = (unsigned short*)hlo;
  const bool lo = pairs(M, a.Dp, a.Fp);
  if (pass == 2) return lo ? product<Dw<true>>(cut_dw(M, D, F, lo), a, stream) : product<Dw<false>>(cut_dw(M, D, F, lo), a, stream);
  const int rc = lo ? product<Dh<true>>(cut_dh(M, D, F, lo), a, stream) : product<Dh<false>>(cut_dh(M, D, F, lo), a, stream);
  if (rc != 0 || dx == nullptr) return rc;
  return lo ? product<Dx<true>>(cut_dx(M, D, F, lo), a, stream) : product<Dx<false>>(cut_dx(M, D, F, lo), a, stream);
}
