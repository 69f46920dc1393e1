// Gated feed-forward block (gfx950):   h = act(x Wg^T) * (x Wu^T),   y = h Wd^T        x [M][D], Wg and Wu [F][D], Wd [D][F], bf16
//
// Forward, two launches:   up    both projections in one product: a block's columns are gate and up rows of the same features side by
//                                side, so that one lane holds g and u of a feature and the activation and the product are the epilogue;
//                                training also keeps P = u act'(g) and Q = act(g);
//                          down  y = h Wd^T.
// Backward, three:         dh    dy Wd, epilogue  dg = dh P,  du = dh Q  (dh itself is never written);
//                          dx    dg Wg + du Wu, one reduction over both pairs;
//                          dw    dg^T x, du^T x and dy^T h, one launch.
// All on the tiles of gemm_tile.h, which take the tensors as they lie: no transposed copy of a weight or an activation exists.
//
// Numbers.  Products accumulate in fp32.  h, dg and du are rounded to bf16 once, being operands of the next product at the bf16 rate.  P and Q
// only scale dh, so they need not be rounded twice as coarsely as that: they are kept in 24 bits (the upper 16 bits of the fp32 value in
// one plane, the next 8 in another; half-step 2^-17), 2 bytes more per feature and token than bf16 copies of g and u, which would add
// two more roundings of 2^-9 to every gradient (measured: relative error of dx, dWg, dWu 0.0031 with g and u in bf16, 0.0024 so).
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
  unsigned short *h, *dg, *du, *y, *dx;
  unsigned short* keep16; unsigned char* keep8;    // P then Q, [2][M][F]
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
      const long long plane = (long long)a.M * a.F;
      keep24<8>(a.keep16 + o, a.keep8 + o, p);
      keep24<8>(a.keep16 + plane + o, a.keep8 + plane + o, q);
    }
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
  tile.template store<false>(smem, wid, lane, gt::NoLoad{}, [&](int r, int c, const float* v, gt::None) {
    r += m0; c += n0;
    if (r < a.M && c < a.D) store8(a.y + (long long)r * a.D + c, v);
  }, [](int, int, float*) {});
}

template <int BT>
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
  const long long plane = (long long)a.M * a.F;
  struct Factors { Kept p, q; };
  auto load = [&](int r, int c) {
    r += m0; c += n0;
    const long long o = (long long)r * a.F + c;
    Factors k{};
    if (r < a.M && c < a.F) { k.p = load24(a.keep16 + o, a.keep8 + o); k.q = load24(a.keep16 + plane + o, a.keep8 + plane + o); }
    return k;
  };
  tile.template store<false>(smem, wid, lane, load, [&](int r, int c, const float* v, const Factors& k) {
    r += m0; c += n0;
    if (r >= a.M || c >= a.F) return;
    const long long o = (long long)r * a.F + c;
    float p[8], q[8], dg[8], du[8];
    get24(k.p, p);
    get24(k.q, q);
#pragma unroll
    for (int e = 0; e < 8; ++e) { dg[e] = v[e] * p[e]; du[e] = v[e] * q[e]; }
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
  tile.template store<false>(smem, wid, lane, gt::NoLoad{}, [&](int r, int c, const float* v, gt::None) {
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
  struct Sum { f32x4 lo, hi; };
  auto load = [&](int r, int c) {
    r += m0; c += n0;
    Sum q{};
    if (a.accumulate && r < rows && c < cols) {
      const float* const p = (const float*)out + (long long)r * cols + c;
      q = Sum{*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 4)};
    }
    return q;
  };
  tile.template store<false>(smem, wid, lane, load, [&](int r, int c, const float* v, const Sum& q) {
    r += m0; c += n0;
    if (r >= rows || c >= cols) return;
    const long long o = (long long)r * cols + c;
    if (a.accumulate) {
      float* const p = (float*)out + o;
      *reinterpret_cast<f32x4*>(p) = f32x4{q.lo[0] + v[0], q.lo[1] + v[1], q.lo[2] + v[2], q.lo[3] + v[3]};
      *reinterpret_cast<f32x4*>(p + 4) = f32x4{q.hi[0] + v[4], q.hi[1] + v[5], q.hi[2] + v[6], q.hi[3] + v[7]};
    } else {
      store8((unsigned short*)out + o, v);
    }
  }, [](int, int, float*) {});
}

// ---- few tokens (serving): bound by reading the weights once.  A block owns 16 features (their gate and up rows, or 16 rows of Wd); its waves
// share the reduction in steps of 64 (one 128-byte line of each row; wave w takes steps w, w + WAVES, ...), load the weights straight into
// matrix-instruction operands - nothing is staged, every byte is used once - several steps ahead, and add their fp32 tiles in LDS in a fixed order.
// TB: blocks of 16 tokens.
template <int TB, int WAVES, bool PAIR, int ACT, bool SAVE>
__global__ __launch_bounds__(64 * WAVES) void gated_few_kernel(const GatedArgs a) {
  constexpr int NM = PAIR ? 2 : 1, U = TB == 4 ? 2 : 4;                  // weight matrices; steps in flight
  __shared__ f32x4 red[WAVES][NM * TB][64];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 15, kc = (lane >> 4) * 8;
  const int K = PAIR ? a.D : a.F, N = PAIR ? a.F : a.D;                  // reduction, rows of the weights
  const int f0 = blockIdx.x * 16;
  const unsigned short* const in = PAIR ? a.x : a.h;
  const unsigned long long wbytes = (unsigned long long)(N - f0 < 16 ? N - f0 : 16) * (unsigned long long)K * 2ull;
  const __amdgpu_buffer_rsrc_t w0 = __builtin_amdgcn_make_buffer_rsrc((void*)((PAIR ? a.wg : a.wd) + (long long)f0 * K), 0, (int)wbytes, 0x00020000);
  const __amdgpu_buffer_rsrc_t w1 = __builtin_amdgcn_make_buffer_rsrc((void*)((PAIR ? a.wu : a.wd) + (long long)f0 * K), 0, (int)wbytes, 0x00020000);
  const __amdgpu_buffer_rsrc_t xs = __builtin_amdgcn_make_buffer_rsrc((void*)in, 0, (int)((unsigned long long)a.M * K * 2ull), 0x00020000);
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
        const bool in_k = k < K;                                         // K % 8 == 0: whole pieces
        const unsigned off = in_k ? (unsigned)(row * K + k) * 2u : gt::OOB;
        w[u][h][0] = __builtin_amdgcn_raw_buffer_load_b128(w0, (int)off, 0, 0);
        if (PAIR) w[u][h][NM - 1] = __builtin_amdgcn_raw_buffer_load_b128(w1, (int)off, 0, 0);
#pragma unroll
        for (int t = 0; t < TB; ++t) {
          const unsigned xo = in_k && t * 16 + row < a.M ? (unsigned)((t * 16 + row) * K + k) * 2u : gt::OOB;
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
    if (tok >= a.M || f >= N) continue;
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
    }
    const long long o = (long long)tok * N + f;
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
    *reinterpret_cast<u32x2*>((PAIR ? a.h : a.y) + o) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
    if (SAVE) {
      const long long plane = (long long)a.M * a.F;
      keep24<4>(a.keep16 + o, a.keep8 + o, p);
      keep24<4>(a.keep16 + plane + o, a.keep8 + plane + o, q);
    }
  }
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
constexpr int FEW = 64;                            // tokens up to which gated_few_kernel is used

template <int TB, bool PAIR, int ACT, bool SAVE> int launch_few_t(const GatedArgs& a, void* st) {
  constexpr int WAVES = PAIR ? 8 : 16;             // Wd has fewer rows (a third of the blocks) and a longer reduction
  hipLaunchKernelGGL(HIP_KERNEL_NAME(gated_few_kernel<TB, WAVES, PAIR, ACT, SAVE>), dim3((unsigned)tiles(PAIR ? a.F : a.D, 16)), dim3(64 * WAVES),
                     0, (hipStream_t)st, a);
  return (int)hipGetLastError();
}
template <bool PAIR, int ACT, bool SAVE> int launch_few(const GatedArgs& a, void* st) {
  return a.M <= 16 ? launch_few_t<1, PAIR, ACT, SAVE>(a, st) : a.M <= 32 ? launch_few_t<2, PAIR, ACT, SAVE>(a, st)
                                                                         : launch_few_t<4, PAIR, ACT, SAVE>(a, st);
}
template <int ACT> int few_up(const GatedArgs& a, bool save, void* st) {
  return save ? launch_few<true, ACT, true>(a, st) : launch_few<true, ACT, false>(a, st);
}
// 32-bit offsets inside 16 rows of a weight and inside the tokens
bool few(int M, int K) { return M <= FEW && (long long)FEW * K * 2 < 0x7fffffffll; }

// 256 x 256 tiles where they fill the chip
bool large(int m, int n) { return tiles(m, 256) * tiles(n, 256) >= 256; }

bool sizes_ok(int M, int D, int F) { return M > 0 && D > 0 && F > 0 && D % 8 == 0 && F % 8 == 0; }

}  // namespace

// h [M][F];  keep16 [2][M][F] (16 bit) and keep8 [2][M][F] (8 bit), or both null: what the backward pass needs
extern "C" int ddl_gated_up(const void* x, const void* wg, const void* wu, void* h, void* keep16, void* keep8, int M, int D, int F, int act,
                            void* stream) {
  if (!sizes_ok(M, D, F) || (keep16 == nullptr) != (keep8 == nullptr)) return -1;
  GatedArgs a{};
  a.x = (const unsigned short*)x; a.wg = (const unsigned short*)wg; a.wu = (const unsigned short*)wu;
  a.h = (unsigned short*)h; a.keep16 = (unsigned short*)keep16; a.keep8 = (unsigned char*)keep8;
  a.M = M; a.D = D; a.F = F;
  if (act < SILU || act > RELU) return -1;
  const bool save = keep16 != nullptr;
  if (few(M, D)) return act == SILU ? few_up<SILU>(a, save, stream) : act == GELU ? few_up<GELU>(a, save, stream) : few_up<RELU>(a, save, stream);
  return large(M, 2 * F) ? up_act<256>(a, act, save, stream) : up_act<128>(a, act, save, stream);
}

extern "C" int ddl_gated_down(const void* h, const void* wd, void* y, int M, int D, int F, void* stream) {
  if (!sizes_ok(M, D, F)) return -1;
  GatedArgs a{};
  a.h = (unsigned short*)h; a.wd = (const unsigned short*)wd; a.y = (unsigned short*)y;
  a.M = M; a.D = D; a.F = F;
  if (few(M, F)) return launch_few<false, SILU, false>(a, stream);
  return large(M, D) ? launch<256, &gated_down_kernel<256>>(tiles(M, 256) * tiles(D, 256), a, stream)
                     : launch<128, &gated_down_kernel<128>>(tiles(M, 128) * tiles(D, 128), a, stream);
}

extern "C" int ddl_gated_dh(const void* dy, const void* wd, const void* keep16, const void* keep8, void* dg, void* du, int M, int D, int F,
                            void* stream) {
  if (!sizes_ok(M, D, F)) return -1;
  GatedArgs a{};
  a.dy = (const unsigned short*)dy; a.wd = (const unsigned short*)wd;
  a.keep16 = (unsigned short*)keep16; a.keep8 = (unsigned char*)keep8; a.dg = (unsigned short*)dg; a.du = (unsigned short*)du;
  a.M = M; a.D = D; a.F = F;
  return large(M, F) ? launch<256, &gated_dh_kernel<256>>(tiles(M, 256) * tiles(F, 256), a, stream)
                     : launch<128, &gated_dh_kernel<128>>(tiles(M, 128) * tiles(F, 128), a, stream);
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
