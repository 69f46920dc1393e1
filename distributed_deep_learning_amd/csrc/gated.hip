// Gated feed-forward block (gfx950):   h = act(x Wg^T) * (x Wu^T),   y = h Wd^T        x [M][D], Wg and Wu [F][D], Wd [D][F], bf16
//
// Forward, two launches:   up    both projections in one product: a block's columns are gate and up rows of the same features side by
//                                side, so that one lane holds g and u of a feature and the activation and the product are the epilogue
//                                (training also stores g and u, in bf16 like every saved activation);
//                          down  y = h Wd^T.
// Backward, three:         dh    dy Wd, epilogue  dg = dh u act'(g),  du = dh act(g)  (dh itself is never written);
//                          dx    dg Wg + du Wu, one reduction over both pairs;
//                          dw    dg^T x, du^T x and dy^T h, one launch.
// All on the tiles of gemm_tile.h, which take the tensors as they lie: no transposed copy of a weight or an activation exists.
// Products accumulate in fp32; h, g, u, dg and du are rounded to bf16 once, because they are operands of the next product (bf16 rate) and
// what training keeps; activations are evaluated in fp32 on unrounded projections in the forward pass.
#include "common.h"
#include "host_util.h"
#include "gemm_tile.h"

namespace {

enum { SILU = 0, GELU = 1, RELU = 2 };

template <int ACT> __device__ __forceinline__ float act_of(float g) {
  if (ACT == SILU) return g / (1.f + __expf(-g));
  if (ACT == GELU) return 0.5f * g * (1.f + erff(g * 0.70710678f));
  return g > 0.f ? g : (g != g ? g : 0.f);
}
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
    a = act_of<RELU>(g);
    d = g > 0.f ? 1.f : (g != g ? g : 0.f);
  }
}

// Tile order: XCD-contiguous runs that sweep 8 tile rows column by column, so that the operand panels a run shares stay in that L2.
__device__ __forceinline__ void tile_of(unsigned bid, unsigned nwg, int tm, int tn, int& i, int& j) {
  const unsigned t = xcd_remap(bid, nwg);
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
};

// Two operands of the same shape one after the other along the reduction.
template <class S> struct Twice {
  static constexpr int NP = S::NP;
  S s;
  const unsigned short* second;
  int left;                                       // stages of the first
  __device__ __forceinline__ void begin() {
    if (left == 0) { s.base = second; s.kdone = 0; }
    --left;
    s.begin();
  }
  __device__ __forceinline__ void piece(int j, unsigned lds, int wid) const { s.piece(j, lds, wid); }
  __device__ __forceinline__ void end() { s.end(); }
};

struct GatedArgs {
  const unsigned short *x, *wg, *wu, *wd, *dy;
  unsigned short *h, *g, *u, *dg, *du, *y, *dx;
  void *dwg, *dwu, *dwd;
  int M, D, F, accumulate;                        // accumulate: weight gradients are fp32 and added to
};

__device__ __forceinline__ void store8(unsigned short* p, const float* v) { *reinterpret_cast<u32x4*>(p) = pack8(v); }

template <int BT, int ACT, bool SAVE>
__global__ __launch_bounds__(256, BT == 256 ? 1 : 2) void gated_up_kernel(const GatedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  int ti, tj;
  tile_of(blockIdx.x, gridDim.x, (a.M + BT - 1) / BT, (a.F + BT / 2 - 1) / (BT / 2), ti, tj);
  const int m0 = ti * BT, f0 = tj * (BT / 2);
  gt::Tile<BT, BT> tile;
  tile.zero();
  gt::Stager<BT, gt::CONTIG, 1> sa;
  PairStager<BT> sb;
  sa.init(gt::Operand{a.x, a.D, m0, a.M, a.D}, wid, lane);
  sb.init(a.wg, a.wu, a.D, f0, a.F, a.D, wid, lane);
  tile.template mul<gt::Bf16, gt::CONTIG, gt::CONTIG, 1>(sa, sb, (a.D + 63) / 64, smem, wid, lane);
  tile.store_pairs(smem, wid, lane, [&](int r, int f, const float* g, const float* u) {
    r += m0; f += f0;
    if (r >= a.M || f >= a.F) return;
    const long long o = (long long)r * a.F + f;
    float h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = act_of<ACT>(g[e]) * u[e];
    store8(a.h + o, h);
    if (SAVE) { store8(a.g + o, g); store8(a.u + o, u); }
  });
}

template <int BT>
__global__ __launch_bounds__(256, BT == 256 ? 1 : 2) void gated_down_kernel(const GatedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  int ti, tj;
  tile_of(blockIdx.x, gridDim.x, (a.M + BT - 1) / BT, (a.D + BT - 1) / BT, ti, tj);
  const int m0 = ti * BT, n0 = tj * BT;
  gt::Tile<BT, BT> tile;
  tile.zero();
  gt::Stager<BT, gt::CONTIG, 1> sa, sb;
  sa.init(gt::Operand{a.h, a.F, m0, a.M, a.F}, wid, lane);
  sb.init(gt::Operand{a.wd, a.F, n0, a.D, a.F}, wid, lane);
  tile.template mul<gt::Bf16, gt::CONTIG, gt::CONTIG, 1>(sa, sb, (a.F + 63) / 64, smem, wid, lane);
  tile.template store<false>(smem, wid, lane, [&](int r, int c, const float* v) {
    r += m0; c += n0;
    if (r < a.M && c < a.D) store8(a.y + (long long)r * a.D + c, v);
  }, [](int, int, float*) {});
}

template <int BT, int ACT>
__global__ __launch_bounds__(256, BT == 256 ? 1 : 2) void gated_dh_kernel(const GatedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  int ti, tj;
  tile_of(blockIdx.x, gridDim.x, (a.M + BT - 1) / BT, (a.F + BT - 1) / BT, ti, tj);
  const int m0 = ti * BT, n0 = tj * BT;
  gt::Tile<BT, BT> tile;
  tile.zero();
  gt::Stager<BT, gt::CONTIG, 1> sa;
  gt::Stager<BT, gt::SLOW, 1> sb;
  sa.init(gt::Operand{a.dy, a.D, m0, a.M, a.D}, wid, lane);
  sb.init(gt::Operand{a.wd, a.F, n0, a.F, a.D}, wid, lane);
  tile.template mul<gt::Bf16, gt::CONTIG, gt::SLOW, 1>(sa, sb, (a.D + 63) / 64, smem, wid, lane);
  tile.template store<false>(smem, wid, lane, [&](int r, int c, const float* v) {
    r += m0; c += n0;
    if (r >= a.M || c >= a.F) return;
    const long long o = (long long)r * a.F + c;
    float g[8], u[8], dg[8], du[8];
    unpack8(*reinterpret_cast<const u32x4*>(a.g + o), g);
    unpack8(*reinterpret_cast<const u32x4*>(a.u + o), u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float av, dv;
      act_and_slope<ACT>(g[e], av, dv);
      dg[e] = v[e] * u[e] * dv;
      du[e] = v[e] * av;
    }
    store8(a.dg + o, dg);
    store8(a.du + o, du);
  }, [](int, int, float*) {});
}

template <int BT>
__global__ __launch_bounds__(256, BT == 256 ? 1 : 2) void gated_dx_kernel(const GatedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  int ti, tj;
  tile_of(blockIdx.x, gridDim.x, (a.M + BT - 1) / BT, (a.D + BT - 1) / BT, ti, tj);
  const int m0 = ti * BT, n0 = tj * BT, nk = (a.F + 63) / 64;
  gt::Tile<BT, BT> tile;
  tile.zero();
  Twice<gt::Stager<BT, gt::CONTIG, 1>> sa;
  Twice<gt::Stager<BT, gt::SLOW, 1>> sb;
  sa.s.init(gt::Operand{a.dg, a.F, m0, a.M, a.F}, wid, lane);
  sa.second = a.du + (long long)m0 * a.F;
  sb.s.init(gt::Operand{a.wg, a.D, n0, a.D, a.F}, wid, lane);
  sb.second = a.wu;
  sa.left = sb.left = nk;
  tile.template mul<gt::Bf16, gt::CONTIG, gt::SLOW, 1>(sa, sb, 2 * nk, smem, wid, lane);
  tile.template store<false>(smem, wid, lane, [&](int r, int c, const float* v) {
    r += m0; c += n0;
    if (r < a.M && c < a.D) store8(a.dx + (long long)r * a.D + c, v);
  }, [](int, int, float*) {});
}

template <int BT>
__global__ __launch_bounds__(256, BT == 256 ? 1 : 2) void gated_dw_kernel(const GatedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tf = (a.F + BT - 1) / BT, td = (a.D + BT - 1) / BT, per = tf * td, which = (int)blockIdx.x / per;
  int ti, tj;
  tile_of(blockIdx.x - (unsigned)(which * per), (unsigned)per, which == 2 ? td : tf, which == 2 ? tf : td, ti, tj);
  const int rows = which == 2 ? a.D : a.F, cols = which == 2 ? a.F : a.D;
  const unsigned short* const pa = which == 0 ? a.dg : which == 1 ? a.du : a.dy;
  const unsigned short* const pb = which == 2 ? a.h : a.x;
  void* const out = which == 0 ? a.dwg : which == 1 ? a.dwu : a.dwd;
  if (out == nullptr) return;
  const int m0 = ti * BT, n0 = tj * BT;
  gt::Tile<BT, BT> tile;
  tile.zero();
  gt::Stager<BT, gt::SLOW, 1> sa, sb;
  sa.init(gt::Operand{pa, rows, m0, rows, a.M}, wid, lane);
  sb.init(gt::Operand{pb, cols, n0, cols, a.M}, wid, lane);
  tile.template mul<gt::Bf16, gt::SLOW, gt::SLOW, 1>(sa, sb, (a.M + 63) / 64, smem, wid, lane);
  tile.template store<false>(smem, wid, lane, [&](int r, int c, const float* v) {
    r += m0; c += n0;
    if (r >= rows || c >= cols) return;
    const long long o = (long long)r * cols + c;
    if (a.accumulate) {
      float* const p = (float*)out + o;
      f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { lo[e] += v[e]; hi[e] += v[4 + e]; }
      *reinterpret_cast<f32x4*>(p) = lo;
      *reinterpret_cast<f32x4*>(p + 4) = hi;
    } else {
      store8((unsigned short*)out + o, v);
    }
  }, [](int, int, float*) {});
}

inline long long tiles(int n, int t) { return ((long long)n + t - 1) / t; }

// one launch of a kernel that takes GatedArgs; opts in to its LDS once per device
template <int BT, auto KERNEL> int launch(long long blocks, const GatedArgs& a, void* stream) {
  static SmemAttrOnce once;
  if (blocks <= 0 || blocks > 0x7fffffffll) return -2;
  constexpr int smem = gt::Tile<BT, BT>::SMEM;
  const int rc = once.ensure(reinterpret_cast<const void*>(KERNEL), smem);
  if (rc != 0) return rc;
  hipLaunchKernelGGL(KERNEL, dim3((unsigned)blocks), dim3(256), smem, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

template <int BT, int ACT> int launch_up(const GatedArgs& a, bool save, void* st) {
  const long long nb = tiles(a.M, BT) * tiles(a.F, BT / 2);
  return save ? launch<BT, &gated_up_kernel<BT, ACT, true>>(nb, a, st) : launch<BT, &gated_up_kernel<BT, ACT, false>>(nb, a, st);
}
template <int BT> int up_act(const GatedArgs& a, int act, bool save, void* st) {
  return act == SILU ? launch_up<BT, SILU>(a, save, st) : act == GELU ? launch_up<BT, GELU>(a, save, st) : launch_up<BT, RELU>(a, save, st);
}
template <int BT> int dh_act(const GatedArgs& a, int act, void* st) {
  const long long nb = tiles(a.M, BT) * tiles(a.F, BT);
  return act == SILU ? launch<BT, &gated_dh_kernel<BT, SILU>>(nb, a, st)
       : act == GELU ? launch<BT, &gated_dh_kernel<BT, GELU>>(nb, a, st) : launch<BT, &gated_dh_kernel<BT, RELU>>(nb, a, st);
}

// 256 x 256 tiles where they fill the chip
bool large(int m, int n) { return tiles(m, 256) * tiles(n, 256) >= 256; }

bool sizes_ok(int M, int D, int F) { return M > 0 && D > 0 && F > 0 && D % 8 == 0 && F % 8 == 0; }

}  // namespace

// h [M][F];  g, u [M][F] or null (both): what the backward pass needs
extern "C" int ddl_gated_up(const void* x, const void* wg, const void* wu, void* h, void* g, void* u, int M, int D, int F, int act, void* stream) {
  if (!sizes_ok(M, D, F) || (g == nullptr) != (u == nullptr)) return -1;
  GatedArgs a{};
  a.x = (const unsigned short*)x; a.wg = (const unsigned short*)wg; a.wu = (const unsigned short*)wu;
  a.h = (unsigned short*)h; a.g = (unsigned short*)g; a.u = (unsigned short*)u;
  a.M = M; a.D = D; a.F = F;
  if (act < SILU || act > RELU) return -1;
  return large(M, 2 * F) ? up_act<256>(a, act, g != nullptr, stream) : up_act<128>(a, act, g != nullptr, stream);
}

extern "C" int ddl_gated_down(const void* h, const void* wd, void* y, int M, int D, int F, void* stream) {
  if (!sizes_ok(M, D, F)) return -1;
  GatedArgs a{};
  a.h = (unsigned short*)h; a.wd = (const unsigned short*)wd; a.y = (unsigned short*)y;
  a.M = M; a.D = D; a.F = F;
  return large(M, D) ? launch<256, &gated_down_kernel<256>>(tiles(M, 256) * tiles(D, 256), a, stream)
                     : launch<128, &gated_down_kernel<128>>(tiles(M, 128) * tiles(D, 128), a, stream);
}

extern "C" int ddl_gated_dh(const void* dy, const void* wd, const void* g, const void* u, void* dg, void* du, int M, int D, int F, int act,
                            void* stream) {
  if (!sizes_ok(M, D, F)) return -1;
  GatedArgs a{};
  a.dy = (const unsigned short*)dy; a.wd = (const unsigned short*)wd;
  a.g = (unsigned short*)g; a.u = (unsigned short*)u; a.dg = (unsigned short*)dg; a.du = (unsigned short*)du;
  a.M = M; a.D = D; a.F = F;
  if (act < SILU || act > RELU) return -1;
  return large(M, F) ? dh_act<256>(a, act, stream) : dh_act<128>(a, act, stream);
}

extern "C" int ddl_gated_dx(const void* dg, const void* du, const void* wg, const void* wu, void* dx, int M, int D, int F, void* stream) {
  if (!sizes_ok(M, D, F)) return -1;
  GatedArgs a{};
  a.dg = (unsigned short*)dg; a.du = (unsigned short*)du; a.wg = (const unsigned short*)wg; a.wu = (const unsigned short*)wu;
  a.dx = (unsigned short*)dx;
  a.M = M; a.D = D; a.F = F;
  return large(M, D) ? launch<256, &gated_dx_kernel<256>>(tiles(M, 256) * tiles(D, 256), a, stream)
                     : launch<128, &gated_dx_kernel<128>>(tiles(M, 128) * tiles(D, 128), a, stream);
}

// weight gradients: bf16, written (accumulate 0), or fp32, added to (accumulate 1); a null one is left out
extern "C" int ddl_gated_dw(const void* x, const void* dy, const void* h, const void* dg, const void* du, void* dwg, void* dwu, void* dwd, int M,
                            int D, int F, int accumulate, void* stream) {
  if (!sizes_ok(M, D, F)) return -1;
  GatedArgs a{};
  a.x = (const unsigned short*)x; a.dy = (const unsigned short*)dy; a.h = (unsigned short*)h;
  a.dg = (unsigned short*)dg; a.du = (unsigned short*)du;
  a.dwg = dwg; a.dwu = dwu; a.dwd = dwd;
  a.M = M; a.D = D; a.F = F; a.accumulate = accumulate;
  return large(3 * F, D) ? launch<256, &gated_dw_kernel<256>>(3 * tiles(F, 256) * tiles(D, 256), a, stream)
                         : launch<128, &gated_dw_kernel<128>>(3 * tiles(F, 128) * tiles(D, 128), a, stream);
}
