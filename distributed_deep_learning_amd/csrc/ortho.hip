// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step built on it (gfx950).
//
//   X0 = G / (|G|_F + eps);   `steps` times:  S = X X^T (X^T X when X is taller than wide),  X <- a X + (b S + c S S) X
// drives every singular value of X to about one while the singular vectors stay.  Per step 2 m^2 n (S, symmetric: half is
// computed, half mirrored: m^2 n) + 2 m^3 (S S, likewise m^3) + 2 m^2 n operations, m the thin side: all of it matrix products,
// run on the tiles of gemm_tile.h.  A tall X is never transposed: its gram matrix takes both operands K-slow, its update is X B.
//
// Chains.  All factors P_i = a I + b S_i + c S_i S_i are polynomials of the first S and commute, and S_(i+1) = P_i S_i P_i, so up to three
// steps can be taken on m x m matrices before X is touched again:  X <- (P_2 P_1 P_0) X.  Five steps then cost 6 m^2 n + 14 m^3 (3 + 2 steps)
// instead of 15 m^2 n + 5 m^3.  What the first S has lost of a small singular value is not found again inside a chain; with 22-bit
// operands chains of three leave the result as exact as single steps (a chain of five does not: 1e-4 on a spectrum that falls like 1/k^2),
// with 11-bit operands they do not, so PROD = 1 takes single steps.  Chosen for wide matrices (use_chains below).
//
// Numbers.  The polynomial has slope a = 3.4 at zero, so five steps amplify what a rounding leaves in a small singular direction
// by up to a^5 = 485.  Therefore
//   * all values are scaled by 2^12 and held in fp16, whose 11 bits cost the same matrix rate as bf16's 8: the entries of X, S
//     and B = b S + c S S are at most a few units in size (the host checks the polynomial's range), so neither end of fp16 is met;
//   * X itself, the state of the iteration, is carried in 22 bits (fp16 hi + lo) in every mode;
//   * PROD = 1 multiplies the hi parts only (one product, 11-bit operands): bf16 matrices, 0.2 % of the result's norm, about the
//     rounding of a bf16 result;   PROD = 3 holds S and B in 22 bits too and multiplies hi*hi + hi*lo + lo*hi: fp32 matrices,
//     1e-6 of the norm, the same as fp32 products, at a third of the fp16 rate instead of a sixteenth.
// The Frobenius norm is summed in fp64, in a fixed order.
//
// Measured, 8192 x 2048 fp32 (two chains): norm 13 us, X0 23, gram 2 x (115 + join 12; 0.95 PFLOP/s of fp16 products), m x m products 14 x (33 + 12;
// 0.85, few tiles), X 2 x 170 (1.22): bound by the matrix rate.  8 x 512 x 4608 bf16, five steps: gram 20 + 5.5, square 11, X 42 us (190 MB, 4.5 TB/s:
// bandwidth).  ResNet-50's Muon step: norm and momentum 51 us, X0 57 (both 5.5 TB/s), gram 2 x 70, m x m 14 x 32, X 95 + 123.
//
// Many matrices share every launch: blocks find their matrix through maps of (matrix, block) pairs, so an optimizer step over a whole
// network is 2 launches and 3 to 6 for every step of the iteration (joins of split reductions, two tile sizes), whatever it has of them.
#include "common.h"
#include "host_util.h"
#include "gemm_tile.h"
#include <math.h>
#include <algorithm>

namespace {

constexpr float SCALE = 4096.f, UNSCALE = 1.f / 4096.f;
constexpr int MAX_PARTS = 1024;                  // partial sums of squares per matrix
constexpr int INIT_CHUNKS = 1024;                // 8-element pieces of X0 per block of the init kernel

struct NsMat {                                   // one matrix of a step (device table, or the one of a plain call)
  long long elem;                                // Muon: element offset in the arena;  plain: 0
  long long ws;                                  // fp16 offset of its workspace: X, X', S, B
  long long slab;                                // float offset of its partial tiles
  int rows, cols, seg;
  float scale;                                   // Muon: factor of the update
  int gram_splits, square_splits;                // blocks that share the reduction of one tile
};

struct NsArgs {
  const NsMat* table;                            // null: every matrix is `one`, at strides
  const int2* map;                               // with a table: (matrix, block) of every block
  int per;                                       // without: blocks per matrix
  NsMat one;
  long long g_stride, ws_stride, slab_stride;
  unsigned short* ws;
  float* slabs;
  double* parts;                                 // [matrix][MAX_PARTS]
  float eps;
  // source / destination
  const float* g32; const bf16_t* g16;           // plain gradient, or
  float* grad; float* mom; float* master; bf16_t* shadow; const float* seg_wd; const float* hyper;   // Muon's arena
  int zero_grad;
  float* out32; bf16_t* out16;
};

__host__ __device__ constexpr long long up(long long n, long long m) { return (n + m - 1) / m * m; }

// Layout of one matrix's workspace (fp16 elements).  PROD 1: X is a hi plane and a lo plane of [rows][ld], S and B are hi planes.
// PROD 3: rows of interleaved groups (32 hi, 32 lo).
template <int PROD> struct Lay {
  enum { MATS = PROD == 3 ? 5 : 2 };             // m x m matrices: S, P (or B = P - a I); chains also T = P S and two for the product of the P
  long long ldx, lds, x0, x1, s, size, lo;       // lo: distance from a hi value to its lo value
  long long mat;                                 // size of an m x m matrix, S the first
  __host__ __device__ Lay(int rows, int cols) {
    const int thin = rows < cols ? rows : cols;
    if (PROD == 3) {
      ldx = 2 * up(cols, 32); lds = 2 * up(thin, 32);
      x0 = 0; x1 = (long long)rows * ldx; s = 2 * x1;
      lo = 32;
    } else {
      ldx = up(cols, 64); lds = up(thin, 64);
      x0 = 0; lo = (long long)rows * ldx; x1 = 2 * lo; s = 4 * lo;
    }
    mat = (long long)thin * lds;
    size = s + MATS * mat;
  }
  __host__ __device__ static long long at(long long row, long long ld, int col) {
    return PROD == 3 ? row * ld + (col >> 5) * 64 + (col & 31) : row * ld + col;
  }
};

__device__ __forceinline__ NsMat locate(const NsArgs& a, unsigned bid, int& mat, int& idx) {
  if (a.table != nullptr) {
    const int2 e = a.map[bid];
    mat = __builtin_amdgcn_readfirstlane(e.x);
    idx = __builtin_amdgcn_readfirstlane(e.y);
    return a.table[mat];
  }
  mat = (int)(bid / (unsigned)a.per);
  idx = (int)(bid - (unsigned)mat * (unsigned)a.per);
  NsMat m = a.one;
  m.elem = (long long)mat * a.g_stride;
  m.ws = (long long)mat * a.ws_stride;
  m.slab = (long long)mat * a.slab_stride;
  return m;
}

__device__ __forceinline__ void f16_store8(unsigned short* p, const float* v) {
  f16x8 h;
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = (_Float16)v[e];
  *reinterpret_cast<f16x8*>(p) = h;
}
__device__ __forceinline__ void split_store8(unsigned short* hi, long long lo, const float* v) {
  f16x8 h, l;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    // The value is pinned in a register first: left to itself the compiler folds the caller's last multiply into the conversion (one
    // rounding) for the stored hi and not into the one the residual is taken from, and near a tie of fp16 the two differ by a step.
    float x = v[e];
    asm("" : "+v"(x));
    h[e] = (_Float16)x;
    l[e] = (_Float16)(x - (float)h[e]);
  }
  *reinterpret_cast<f16x8*>(hi) = h;
  *reinterpret_cast<f16x8*>(hi + lo) = l;
}

// parts of a matrix: slices of `slice` elements (a multiple of 1024), at most MAX_PARTS
__host__ __device__ inline long long slice_of(long long n) { return up((n + MAX_PARTS - 1) / MAX_PARTS, 1024); }

// Muon's gradient of one element: momentum already updated
__device__ __forceinline__ float muon_update(float g, float m, float mu, float nesterov) { return nesterov != 0.f ? g + mu * m : m; }

// ---- sums of squares; with Muon also the momentum update.  One block per slice.
template <bool MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(const NsArgs a) {
  __shared__ double red[4];
  int mat, idx;
  const NsMat m = locate(a, blockIdx.x, mat, idx);
  const long long n = (long long)m.rows * m.cols, slice = slice_of(n);
  const long long lo = (long long)idx * slice, hi = lo + slice < n ? lo + slice : n;
  double s = 0.0;
  if (MUON) {
    const float mu = a.hyper[1], nest = a.hyper[2], gs = a.hyper[4];
    float* const gp = a.grad + m.elem;
    float* const mp = a.mom + m.elem;
    // tensors start and end on 1024-element boundaries of the arena, whose padding is zero: whole 16-byte pieces
    for (long long i = lo + threadIdx.x * 4; i < hi; i += 1024) {
      const f32x4 g = *reinterpret_cast<const f32x4*>(gp + i);
      f32x4 v = *reinterpret_cast<const f32x4*>(mp + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float ge = gs * g[e];
        v[e] = mu * v[e] + ge;
        const float u = muon_update(ge, v[e], mu, nest);
        s += (double)u * (double)u;
      }
      *reinterpret_cast<f32x4*>(mp + i) = v;
    }
  } else {
    const bool wide = (((unsigned long long)(a.g32 != nullptr ? (const void*)(a.g32 + m.elem) : (const void*)(a.g16 + m.elem))) & 15) == 0;
    long long i = lo + threadIdx.x * 8;
    if (wide) {
      auto piece = [&](long long at, float* v) {
        if (a.g32 != nullptr) {
          *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(a.g32 + m.elem + at);
          *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(a.g32 + m.elem + at + 4);
        } else {
          unpack8(*reinterpret_cast<const u32x4*>(a.g16 + m.elem + at), v);
        }
      };
#pragma unroll 4
      for (; i + 8 <= hi; i += 2048) {
        float v[8];
        piece(i, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += (double)v[e] * (double)v[e];
      }
    }
    for (; i < hi; i += 2048) {                             // the last elements, or a matrix of a batch that starts off a 16-byte boundary
      for (int e = 0; e < 8 && i + e < hi; ++e) {
        const float g = a.g32 != nullptr ? a.g32[m.elem + i + e] : bf16_to_f32(a.g16[m.elem + i + e]);
        s += (double)g * (double)g;
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) a.parts[(long long)mat * MAX_PARTS + idx] = red[0] + red[1] + red[2] + red[3];
}

// ---- X0 = 2^12 G / (|G| + eps), split into fp16 hi + lo, rows padded with zeros.  With Muon the gradient is cleared behind the read.
template <int PROD, bool MUON>
__global__ __launch_bounds__(256) void ns_init_kernel(const NsArgs a) {
  __shared__ double red[4];
  int mat, idx;
  const NsMat m = locate(a, blockIdx.x, mat, idx);
  const Lay<PROD> L(m.rows, m.cols);
  const long long n = (long long)m.rows * m.cols, slice = slice_of(n);
  const int parts = (int)((n + slice - 1) / slice);
  double s = 0.0;
  for (int i = (int)threadIdx.x; i < parts; i += 256) s += a.parts[(long long)mat * MAX_PARTS + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  const float inv = (float)((double)SCALE / (sqrt(red[0] + red[1] + red[2] + red[3]) + (double)a.eps));
  const int width = (int)(PROD == 3 ? L.ldx / 2 : L.ldx), w8 = width / 8;      // padded row in 8-element pieces
  const long long total = (long long)m.rows * w8;
  float mu = 0.f, nest = 0.f, gs = 1.f;
  if (MUON) { mu = a.hyper[1]; nest = a.hyper[2]; gs = a.hyper[4]; }
  const bool wide8 = (m.cols & 7) == 0;
  const long long end = (long long)(idx + 1) * INIT_CHUNKS < total ? (long long)(idx + 1) * INIT_CHUNKS : total;
  for (long long t = (long long)idx * INIT_CHUNKS + threadIdx.x; t < end; t += 256) {
    const int row = (int)(t / w8), col = (int)(t - (long long)row * w8) * 8;
    const long long src = m.elem + (long long)row * m.cols + col;
    float v[8];
    if (wide8 && col < m.cols) {
      if (MUON) {
        float mm[8];
        *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(a.grad + src);
        *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(a.grad + src + 4);
        *reinterpret_cast<f32x4*>(mm) = *reinterpret_cast<const f32x4*>(a.mom + src);
        *reinterpret_cast<f32x4*>(mm + 4) = *reinterpret_cast<const f32x4*>(a.mom + src + 4);
        if (a.zero_grad) {
          *reinterpret_cast<f32x4*>(a.grad + src) = f32x4{0.f, 0.f, 0.f, 0.f};
          *reinterpret_cast<f32x4*>(a.grad + src + 4) = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = muon_update(gs * v[e], mm[e], mu, nest);
      } else if (a.g32 != nullptr) {
        *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(a.g32 + src);
        *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(a.g32 + src + 4);
      } else {
        unpack8(*reinterpret_cast<const u32x4*>(a.g16 + src), v);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = 0.f;
        if (col + e < m.cols) {
          if (MUON) {
            v[e] = muon_update(gs * a.grad[src + e], a.mom[src + e], mu, nest);
            if (a.zero_grad) a.grad[src + e] = 0.f;
          } else {
            v[e] = a.g32 != nullptr ? a.g32[src + e] : bf16_to_f32(a.g16[src + e]);
          }
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= inv;
    split_store8(a.ws + m.ws + L.x0 + Lay<PROD>::at(row, L.ldx, col), L.lo, v);
  }
}

// ---- the products.  KIND 0: S = X X^T;  1: an m x m product;  2: X' = beta X + F X;  3: the same, last step, to the destination.
enum { MAT_S = 0, MAT_P = 1, MAT_T = 2, MAT_Q = 3, MAT_R = 4 };
struct Op {
  int a, b, dst;                                 // SQUARE: mats[dst] = alpha mats[a] mats[b] + beta mats[a] + diag I;  APPLY: F = mats[a]
  int flip;                                      // X is in the second of its two places
  float alpha, beta, diag;
};
enum { GRAM = 0, SQUARE = 1, APPLY = 2, FINAL = 3 };

// A tile's reduction may be shared by several blocks (few tiles, long reductions: the gram matrix of a wide X): each leaves its fp32
// partial tile, and the launch with JOIN adds them in order and does the epilogue.
template <int PROD, int KIND, int BT, int NST, bool MUON, bool JOIN>
__global__ __launch_bounds__(256, BT == 256 || NST > 2 ? 1 : 2) void ns_product_kernel(const NsArgs a, const Op op) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  int mat, idx;
  const NsMat m = locate(a, xcd_remap(blockIdx.x, gridDim.x), mat, idx);
  const Lay<PROD> L(m.rows, m.cols);
  const bool tall = m.rows > m.cols;
  const int thin = tall ? m.cols : m.rows;
  unsigned short* const ws = a.ws + m.ws;
  unsigned short* const X = ws + (op.flip ? L.x1 : L.x0);
  unsigned short* const A = ws + L.s + op.a * L.mat;
  unsigned short* const B = ws + L.s + op.b * L.mat;

  using T = gt::Tile<BT, BT, NST>;
  int ti, tj, split = 0, splits = 1, which = 0;
  if (KIND <= SQUARE) {                                   // lower triangle, row by row
    splits = KIND == GRAM ? m.gram_splits : m.square_splits;
    if (JOIN) { which = idx / T::FM; split = idx - which * T::FM; }   // split: the row group this block joins
    else { which = idx / splits; split = idx - which * splits; }
    ti = (int)((sqrtf(8.f * (float)which + 1.f) - 1.f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= which) ++ti;
    while (ti * (ti + 1) / 2 > which) --ti;
    tj = which - ti * (ti + 1) / 2;
  } else {
    const int tm = (m.rows + BT - 1) / BT;
    tj = idx / tm;
    ti = idx - tj * tm;
  }
  const int m0 = ti * BT, n0 = tj * BT;

  T tile;
  float* const slab = a.slabs + m.slab + (long long)which * splits * T::SLAB;
  if (JOIN) {
    tile.sum_slabs(slab, splits, split, tid);
  } else {
    tile.zero();
    auto run = [&](auto am, auto bm, const unsigned short* pa, long long lda, int ra, const unsigned short* pb, long long ldb, int rb, int k) {
      constexpr int AM = decltype(am)::value, BMD = decltype(bm)::value;
      using SA = gt::Stager<BT, AM, PROD>;
      using SB = gt::Stager<BT, BMD, PROD>;
      SA sa;
      SB sb;
      if (KIND <= SQUARE && splits > 1) {                 // this block's part of the reduction, whole stages
        const int per = ((k + SA::KSTEP - 1) / SA::KSTEP + splits - 1) / splits * SA::KSTEP, k0 = min(k, split * per);
        pa += AM == gt::SLOW ? k0 * lda : (PROD == 3 ? 2 : 1) * k0;
        pb += BMD == gt::SLOW ? k0 * ldb : (PROD == 3 ? 2 : 1) * k0;
        k = min(k - k0, per);
      }
      sa.init(gt::Operand{pa, lda, m0, ra, k}, wid, lane);
      sb.init(gt::Operand{pb, ldb, n0, rb, k}, wid, lane);
      tile.template mul<gt::Fp16, AM, BMD, PROD>(sa, sb, (k + SA::KSTEP - 1) / SA::KSTEP, smem, wid, lane);
    };
    struct C { enum { value = gt::CONTIG }; };
    struct W { enum { value = gt::SLOW }; };
    if (KIND == GRAM) {
      if (tall) run(W{}, W{}, X, L.ldx, m.cols, X, L.ldx, m.cols, m.rows);
      else      run(C{}, C{}, X, L.ldx, m.rows, X, L.ldx, m.rows, m.cols);
    } else if (KIND == SQUARE) {
      run(C{}, C{}, A, L.lds, thin, B, L.lds, thin, thin);
    } else {
      if (tall) run(C{}, C{}, X, L.ldx, m.rows, A, L.lds, thin, thin);
      else      run(C{}, W{}, A, L.lds, thin, X, L.ldx, m.cols, thin);
    }
    if (KIND <= SQUARE && splits > 1) { tile.put_slab(slab + (long long)split * T::SLAB, tid); return; }
  }

  if (KIND <= SQUARE) {
    unsigned short* const dst = ws + L.s + op.dst * L.mat;
    const int ncol = (int)(PROD == 3 ? L.lds / 2 : L.lds);
    struct Old { f16x8 h, l; };
    auto load = [&](int r, int c) {                       // A(r, c), 8 columns
      Old o{};
      r += m0; c += n0;
      if (KIND == SQUARE && op.beta != 0.f && r < thin && c < ncol) {
        const unsigned short* q = A + Lay<PROD>::at(r, L.lds, c);
        o.h = *reinterpret_cast<const f16x8*>(q);
        if (PROD == 3) o.l = *reinterpret_cast<const f16x8*>(q + 32);
      }
      return o;
    };
    auto put = [&](int r, int c, const float* v) {
      if (r >= thin || c >= ncol) return;
      unsigned short* q = dst + Lay<PROD>::at(r, L.lds, c);
      if (PROD == 3) split_store8(q, 32, v); else f16_store8(q, v);
    };
    auto straight = [&](int r, int c, float* v, const Old& o) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] *= op.alpha;
        if (KIND == SQUARE) v[e] += op.beta * (PROD == 3 ? (float)o.h[e] + (float)o.l[e] : (float)o.h[e]) + (m0 + r == n0 + c + e ? op.diag : 0.f);
      }
      put(m0 + r, n0 + c, v);
    };
    constexpr int NJ = JOIN ? 1 : T::FM;
    const int j0 = JOIN ? split : 0;
    if (ti != tj)
      tile.template store<true, NJ>(smem, wid, lane, load, straight, [&](int r, int c, const float* v) { put(n0 + r, m0 + c, v); }, j0);
    else
      tile.template store<false, NJ>(smem, wid, lane, load, straight, [](int, int, float*) {}, j0);
  } else {
    unsigned short* const dst = ws + (op.flip ? L.x0 : L.x1);
    const int ncol = (int)(PROD == 3 ? L.ldx / 2 : L.ldx);
    float lr = 0.f, wd = 0.f;
    if (KIND == FINAL && MUON) { lr = a.hyper[0]; wd = a.seg_wd[m.seg]; }
    const bool wide8 = (m.cols & 7) == 0;
    struct Old { f16x8 h, l; f32x4 w[2]; };
    auto load = [&](int r, int c) {                       // X(r, c), 8 columns; Muon's last step: the weights too
      Old q{};
      r += m0; c += n0;
      if (r >= m.rows || c >= (KIND == FINAL ? m.cols : ncol)) return q;
      const long long at = Lay<PROD>::at(r, L.ldx, c);
      if (op.beta != 0.f) {
        q.h = *reinterpret_cast<const f16x8*>(X + at);
        q.l = *reinterpret_cast<const f16x8*>(X + at + L.lo);
      }
      if (KIND == FINAL && MUON && wide8) {
        const float* const wp = a.master + m.elem + (long long)r * m.cols + c;
        q.w[0] = *reinterpret_cast<const f32x4*>(wp);
        q.w[1] = *reinterpret_cast<const f32x4*>(wp + 4);
      }
      return q;
    };
    tile.template store<false>(smem, wid, lane, load, [&](int r, int c, float* v, const Old& q) {
      r += m0; c += n0;
      if (r >= m.rows || c >= (KIND == FINAL ? m.cols : ncol)) return;
      const long long at = Lay<PROD>::at(r, L.ldx, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = op.alpha * v[e] + op.beta * ((float)q.h[e] + (float)q.l[e]);
      if (KIND == APPLY) { split_store8(dst + at, L.lo, v); return; }
      const long long o = m.elem + (long long)r * m.cols + c;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= UNSCALE;
      if (MUON) {
        float* const wp = a.master + o;
        if (wide8) {
          float w[8];
          *reinterpret_cast<f32x4*>(w) = q.w[0];
          *reinterpret_cast<f32x4*>(w + 4) = q.w[1];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] -= lr * (m.scale * v[e] + wd * w[e]);
          *reinterpret_cast<f32x4*>(wp) = *reinterpret_cast<const f32x4*>(w);
          *reinterpret_cast<f32x4*>(wp + 4) = *reinterpret_cast<const f32x4*>(w + 4);
          if (a.shadow != nullptr) *reinterpret_cast<u32x4*>(a.shadow + o) = pack8(w);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < m.cols) {
              const float w = wp[e] - lr * (m.scale * v[e] + wd * wp[e]);
              wp[e] = w;
              if (a.shadow != nullptr) a.shadow[o + e] = f32_to_bf16(w);
            }
        }
      } else if (a.out32 != nullptr) {
        if (wide8) {
          *reinterpret_cast<f32x4*>(a.out32 + o) = *reinterpret_cast<const f32x4*>(v);
          *reinterpret_cast<f32x4*>(a.out32 + o + 4) = *reinterpret_cast<const f32x4*>(v + 4);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) if (c + e < m.cols) a.out32[o + e] = v[e];
        }
      } else {
        if (wide8) *reinterpret_cast<u32x4*>(a.out16 + o) = pack8(v);
        else {
#pragma unroll
          for (int e = 0; e < 8; ++e) if (c + e < m.cols) a.out16[o + e] = f32_to_bf16(v[e]);
        }
      }
    }, [](int, int, float*) {});
  }
}

// ---- matrices that fit one CU: thin side <= 128, wide side <= NT * 128.  One block of eight waves does everything in one launch: X stays in
// registers in fp32 (every lane holds fragments of all NT column tiles in the layout of the products' results), S, B and one tile of X at a
// time are in LDS as operands.  Such matrices are bound by latency: 17 launches of about 5 us each take longer than all their products.
// X is taken as [thin][wide] (a tall matrix is read and written transposed).
template <int PROD> struct Solo {
  static constexpr int KSTAGES = PROD == 3 ? 4 : 2, KSTEP = 128 / KSTAGES, BUF = KSTAGES * 16384;      // a 128 x 128 operand
  static constexpr int SMEM = 2 * BUF;
  // Byte offset of the elements (row, col .. col + 3) of an operand, for a lane's first fragment; its other fragments are 16 rows (ROWS16 or
  // SLOW16(j)) and 16 columns (^ COL16) away.  The lo part of split operands is half a row (^ 64) or 32 rows (+ 8192) away.
  static constexpr int ROWS16 = 2048, COL16 = 32;
  static __device__ __forceinline__ int contig(int row, int col) {
    const int st = PROD == 3 ? col >> 5 : col >> 6, c = PROD == 3 ? (col & 31) >> 3 : (col & 63) >> 3;
    return st * 16384 + row * 128 + ((c ^ ((row >> 1) & 7)) << 4) + (col & 7) * 2;
  }
  static __device__ __forceinline__ int slow(int row, int col) {
    const int st = PROD == 3 ? row >> 5 : row >> 6, r = PROD == 3 ? row & 31 : row & 63;
    return st * 16384 + r * 256 + (((col >> 3) ^ (((r & 3) << 2) | ((r >> 2) & 3))) << 4) + (col & 7) * 2;
  }
  static constexpr int SLOW16(int j) { return PROD == 3 ? (j >> 1) * 16384 + (j & 1) * 4096 : j * 4096; }
};

template <int PROD> __device__ __forceinline__ void solo_put(char* buf, int off, int lo, const f32x4& v) {
  f16x4 h, l;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x = v[e];
    asm("" : "+v"(x));                                                  // one rounding for both parts (split_store8)
    h[e] = (_Float16)x;
    l[e] = (_Float16)(x - (float)h[e]);
  }
  *reinterpret_cast<f16x4*>(buf + off) = h;
  if (PROD == 3) *reinterpret_cast<f16x4*>(buf + lo) = l;
}

// FULL (fp32 matrices): sums of 22-bit products as exact as fp32 products' (64 x 147: error 1.1e-6 -> 0.8e-6 at 45 -> 52 us).
template <int PROD, int NT, bool MUON, bool FULL>
__global__ __launch_bounds__(512, 2) void ns_solo_kernel(const NsArgs a, const int steps, const float ca, const float cb, const float cc) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ double red[8];
  using L = Solo<PROD>;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid & 1, wn = wid >> 1;                                // 64 rows x 32 columns of a tile: 4 x 2 fragments
  int mat, idx;
  const NsMat m = locate(a, blockIdx.x, mat, idx);
  const bool tall = m.rows > m.cols;
  const int thin = tall ? m.cols : m.rows, wide = tall ? m.rows : m.cols;
  const int row0 = wm * 64 + (lane & 15), col0 = wn * 32 + (lane >> 4) * 4;
  auto at = [&](int r, int c) { return m.elem + (tall ? (long long)c * m.cols + r : (long long)r * m.cols + c); };
  float mu = 0.f, nest = 0.f, gs = 1.f;
  if (MUON) { mu = a.hyper[1]; nest = a.hyper[2]; gs = a.hyper[4]; }

  f32x4 x[NT][4][2];
  double sq = 0.0;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = row0 + j * 16, c = t * 128 + col0 + i * 16;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = 0.f;
          if (r < thin && c + e < wide) {
            const long long o = at(r, c + e);
            if (MUON) {
              const float g = gs * a.grad[o], mm = mu * a.mom[o] + g;
              a.mom[o] = mm;
              if (a.zero_grad) a.grad[o] = 0.f;
              v = muon_update(g, mm, mu, nest);
            } else {
              v = a.g32 != nullptr ? a.g32[o] : bf16_to_f32(a.g16[o]);
            }
          }
          x[t][j][i][e] = v;
          sq += (double)v * (double)v;
        }
      }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sq += __shfl_xor(sq, o, 64);
  if (lane == 0) red[wid] = sq;
  __syncthreads();
  sq = 0.0;
#pragma unroll
  for (int w = 0; w < 8; ++w) sq += red[w];
  const float inv = (float)((double)SCALE / (sqrt(sq) + (double)a.eps));
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) x[t][j][i] *= inv;

  char* const buf0 = smem;
  char* const buf1 = smem + L::BUF;
  gt::Reader<128, gt::CONTIG> ra;                                       // 64 rows of the first operand
  gt::Reader<64, gt::CONTIG> rb;                                        // 32 rows of the second
  gt::Reader<64, gt::SLOW> rs;
  ra.init(wm, lane);
  rb.init(wn, lane);
  rs.init(wn, lane);
  f32x4 acc[4][2];
  auto clear = [&]() {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  // k: length of the reduction;  cols: of the result.  A wave whose part of the result is all padding keeps its zeros.
  auto mul = [&](const char* pa, const char* pb, auto slow, int k, int cols) {
    if (wm * 64 >= thin || wn * 32 >= cols) return;
    f32x4 cross[4][2];                                                  // FULL: hi lo, lo hi and lo lo apart, a third of the roundings of the large sums
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) cross[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int st = 0; st * L::KSTEP < k && st < L::KSTAGES; ++st, pa += 16384, pb += 16384) {
      s16x8 fa[4], fb[2][2];
      auto load_a = [&](int h) {
#pragma unroll
        for (int j = 0; j < 4; ++j) fa[j] = ra.get(pa, j, h);
      };
      auto load_b = [&](int h) {
#pragma unroll
        for (int i = 0; i < 2; ++i) fb[h][i] = decltype(slow)::value ? rs.get(pb, i, h) : rb.get(pb, i, h);
      };
      auto go = [&](int h, f32x4 (*sum)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[j][i] = gt::Fp16::mfma(fb[h][i], fa[j], sum[j][i]);
      };
      load_a(0); load_b(0); load_b(1);
      go(0, acc);
      if (PROD == 3) go(1, FULL ? cross : acc);
      load_a(1);
      if (PROD == 3) go(0, FULL ? cross : acc); else go(1, acc);
      if (FULL) go(1, cross);
    }
    if (FULL) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[j][i] += cross[j][i];
    }
  };
  const int off_c = L::contig(row0, col0), off_s = L::slow(row0, col0);
  // cols: of the operand.  What no product reads is not written (whole 64 x 32 parts; a product reads up to a multiple of KSTEP columns).
  auto put_contig = [&](char* buf, const f32x4 (*v)[2], int cols) {
    if (wm * 64 >= thin || wn * 32 >= (cols + L::KSTEP - 1) / L::KSTEP * L::KSTEP) return;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int off = off_c ^ (i * L::COL16);
        solo_put<PROD>(buf + j * L::ROWS16, off, off ^ 64, v[j][i]);
      }
  };
  auto put_slow = [&](char* buf, const f32x4 (*v)[2], int cols) {
    if (wm * 64 >= thin || wn * 32 >= cols) return;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int off = off_s ^ (i * L::COL16);
        solo_put<PROD>(buf + L::SLOW16(j), off, off + 8192, v[j][i]);
      }
  };
  struct No { enum { value = 0 }; };
  struct Yes { enum { value = 1 }; };

  for (int s = 0; s < steps; ++s) {
    clear();
#pragma unroll
    for (int t = 0; t < NT; ++t) {                                      // S = X X^T
      put_contig(t & 1 ? buf1 : buf0, x[t], wide - t * 128);
      __syncthreads();                                                  // the other buffer's readers passed the previous barrier
      mul(t & 1 ? buf1 : buf0, t & 1 ? buf1 : buf0, No{}, wide - t * 128, thin);
    }
    f32x4 sv[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) sv[j][i] = acc[j][i] * UNSCALE;
    char* const bs = NT & 1 ? buf1 : buf0;                              // not read since the last barrier
    char* const bb = NT & 1 ? buf0 : buf1;
    put_contig(bs, sv, thin);
    __syncthreads();
    clear();
    mul(bs, bs, No{}, thin, thin);                                                  // B = b S + c S S
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) sv[j][i] = sv[j][i] * cb + acc[j][i] * (cc * UNSCALE);
    put_contig(bb, sv, thin);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {                                      // X = a X + B X
      put_slow(bs, x[t], wide - t * 128);
      __syncthreads();
      clear();
      mul(bb, bs, Yes{}, thin, wide - t * 128);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) x[t][j][i] = x[t][j][i] * ca + acc[j][i] * UNSCALE;
      __syncthreads();
    }
  }

  float lr = 0.f, wd = 0.f;
  if (MUON) { lr = a.hyper[0]; wd = a.seg_wd[m.seg]; }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = row0 + j * 16, c = t * 128 + col0 + i * 16;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (r < thin && c + e < wide) {
            const long long o = at(r, c + e);
            const float v = x[t][j][i][e] * UNSCALE;
            if (MUON) {
              const float w = a.master[o] - lr * (m.scale * v + wd * a.master[o]);
              a.master[o] = w;
              if (a.shadow != nullptr) a.shadow[o] = f32_to_bf16(w);
            } else if (a.out32 != nullptr) {
              a.out32[o] = v;
            } else {
              a.out16[o] = f32_to_bf16(v);
            }
          }
        }
      }
}

using gt::CUS;
using gt::SLOTS;
using gt::chunk_for;
constexpr int SLAB = gt::Tile<128, 128>::SLAB;

inline int tri(int thin) { const int t = (thin + 127) / 128; return t * (t + 1) / 2; }
inline int full(int rows, int cols, int bt) { return ((rows + bt - 1) / bt) * ((cols + bt - 1) / bt); }
inline int stages(int k, int prod) { return prod == 3 ? (k + 31) / 32 : (k + 63) / 64; }

// X' = a X + B X in 256 x 256 tiles (half the staged bytes per operation) where they alone fill the chip and the reduction is long enough for
// one block on a CU to hide its ends: 8192 x 2048 fp32 164 us against 183;  8 x 512 x 4608 bf16 (8 stages) 70 us against 44.
inline bool large_apply(int rows, int cols, long long batch) { return min(rows, cols) >= 1024 && full(rows, cols, 256) * batch >= CUS; }

template <int PROD, int KIND, int BT, int NST, bool MUON, bool JOIN>
int launch_product(const NsArgs& a, int blocks, const Op& op, hipStream_t st) {
  if (blocks == 0) return 0;
  static SmemAttrOnce once;
  auto* fn = &ns_product_kernel<PROD, KIND, BT, NST, MUON, JOIN>;
  const int smem = gt::Tile<BT, BT, NST>::SMEM;
  const int rc = once.ensure(reinterpret_cast<const void*>(fn), smem);
  if (rc != 0) return rc;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(ns_product_kernel<PROD, KIND, BT, NST, MUON, JOIN>), dim3(blocks), dim3(256), smem, st, a, op);
  return (int)hipGetLastError();
}

// Launches: 0 norm, 1 init, 2 gram, 3 square, 4 joining gram, 5 joining square, 6 apply in 128 x 128, 7 apply in 256 x 256 tiles
enum { LAUNCHES = 8 };

template <int PROD, int KIND, bool MUON>
int symmetric(const NsArgs& a, const NsArgs& join, int blocks, int joins, const Op& op, hipStream_t st) {
  int rc = blocks <= CUS ? launch_product<PROD, KIND, 128, 4, MUON, false>(a, blocks, op, st)
                         : launch_product<PROD, KIND, 128, 2, MUON, false>(a, blocks, op, st);
  if (rc == 0) rc = launch_product<PROD, KIND, 128, 2, MUON, true>(join, joins, op, st);
  return rc;
}
template <int PROD, int KIND, bool MUON>
int apply(const NsArgs& small, const NsArgs& big, int nsmall, int nbig, const Op& op, hipStream_t st) {
  int rc = launch_product<PROD, KIND, 256, 2, MUON, false>(big, nbig, op, st);
  if (rc == 0)
    rc = nsmall <= CUS ? launch_product<PROD, KIND, 128, 4, MUON, false>(small, nsmall, op, st)
                       : launch_product<PROD, KIND, 128, 2, MUON, false>(small, nsmall, op, st);
  return rc;
}

// The largest value of |P(t)| = |a + b t + c t^2| over squared singular values t up to 1.6, with a little to spare.  The range check lets singular
// values reach 2.5, but none of them leaves a step above that either: beyond 1.6 |P(t)| <= 2.5 / sqrt(t) < 2, whose third power is in range at any scale
inline float factor_bound(const float* abc) {
  float f = 0.f;
  for (int i = 0; i <= 160; ++i) {
    const float t = 0.01f * (float)i, v = fabsf(abc[0] + abc[1] * t + abc[2] * t * t);
    f = v > f ? v : f;
  }
  return 1.05f * f;
}
// Scale of products of up to three factors in fp16 (4096 for the usual matrices): a power of two that keeps them in range.  0: out of range
inline float chain_scale(const float* abc) {
  const float f = factor_bound(abc);
  float q = 4096.f;
  while (q >= 256.f && f * f * f * q > 60000.f) q *= 0.5f;
  return f * 4096.f < 60000.f && q >= 256.f ? q : 0.f;
}
// A set of matrices: operations in chains (6 m^2 n + 14 m^3 each) against single steps (15 m^2 n + 5 m^3).  Chains are 18 launches instead of 15,
// and up to 4 more that join: some 35 us where all of them are short, what 1e10 operations take with split operands; and their m x m products
// fill the chip less.  (LeNet-5's Muon step 179 us in chains, 162 in single steps;  8192 x 2048 1205 us against 1760.)
// A plain call decides by one matrix, however many it has: chains would save a batch of smaller ones time and cost it accuracy, which nobody asked
// to trade (8 x 512 x 4608 fp32: 666 us and an error of 2.4e-6 in single steps, 507 us and 3.9e-6 in chains; 64 x 256 x 1024: 458 us and 2.2e-6, 406 us and 3.2e-6).
inline bool use_chains(double chained, double single) { return chained <= 0.8 * single && single - chained > 1e10; }
inline double chained_work(double thin, double wide) { return 6 * thin * thin * wide + 14 * thin * thin * thin; }
inline double single_work(double thin, double wide) { return 15 * thin * thin * wide + 5 * thin * thin * thin; }

// Measured: 16 x 16 20 us, 64 x 147 49 us, 128 x 256 94 us (bf16; fp32 22, 52, 108) against 100 to 170 us in 17 launches.  Four tiles (120 x 400 fp32) spill and run 257 us against 150: two at most.
constexpr int SOLO_TILES = 2;
inline bool solo(int rows, int cols) { return min(rows, cols) <= 128 && max(rows, cols) <= SOLO_TILES * 128; }

template <int PROD, int NT, bool MUON, bool FULL> int launch_solo_t(const NsArgs& a, int mats, int steps, const float* abc, hipStream_t st) {
  static SmemAttrOnce once;
  auto* fn = &ns_solo_kernel<PROD, NT, MUON, FULL>;
  const int smem = Solo<PROD>::SMEM, rc = once.ensure(reinterpret_cast<const void*>(fn), smem);
  if (rc != 0) return rc;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(ns_solo_kernel<PROD, NT, MUON, FULL>), dim3(mats), dim3(512), smem, st, a, steps, abc[0], abc[1], abc[2]);
  return (int)hipGetLastError();
}
// wide: the widest matrix
template <int PROD, bool MUON, bool FULL> int launch_solo(const NsArgs& a, int mats, int wide, int steps, const float* abc, hipStream_t st) {
  return wide <= 128 ? launch_solo_t<PROD, 1, MUON, FULL>(a, mats, steps, abc, st) : launch_solo_t<PROD, 2, MUON, FULL>(a, mats, steps, abc, st);
}

// What 32-bit counts and a lane's 32-bit byte offsets inside a tile hold: 128 K-contiguous rows of X, or a stage of its rows.  (Only the columns of wide
// matrices are long rows; 256-row tiles of X have rows as long as the thin side.)
template <int PROD> bool addressable(int rows, int cols) {
  const long long bytes = 2 * Lay<PROD>(rows, cols).ldx, most = 0xFFFFFFE0ll;
  return rows > 0 && cols > 0 && rows <= 0x7fffff00 && cols <= 0x7fffff00 && (min(rows, 128) - 1) * bytes + 128 <= most &&
         min(rows, PROD == 3 ? 32 : 64) * bytes <= most;
}
bool addressable(int rows, int cols, int prod) { return prod == 3 ? addressable<3>(rows, cols) : prod == 1 && addressable<1>(rows, cols); }

// blocks of every launch;  maps likewise (null for a plain call: `per` blocks a matrix);  chains: only with PROD = 3
template <int PROD, bool MUON>
int run_steps(NsArgs a, const int* blocks, const int2* const* maps, const int* per, int steps, const float* abc, bool chains, hipStream_t st) {
  auto with = [&](int i) { a.map = maps != nullptr ? maps[i] : nullptr; a.per = per != nullptr ? per[i] : 1; return a; };
  hipLaunchKernelGGL(HIP_KERNEL_NAME(ns_norm_kernel<MUON>), dim3(blocks[0]), dim3(256), 0, st, with(0));
  hipLaunchKernelGGL(HIP_KERNEL_NAME(ns_init_kernel<PROD, MUON>), dim3(blocks[1]), dim3(256), 0, st, with(1));
  int rc = (int)hipGetLastError();
  const float ca = abc[0], cb = abc[1], cc = abc[2];
  int flip = 0;
  auto gram = [&]() {
    if (rc == 0) rc = symmetric<PROD, GRAM, MUON>(with(2), with(4), blocks[2], blocks[4], Op{0, 0, MAT_S, flip, UNSCALE, 0.f, 0.f}, st);
  };
  auto mats = [&](int x, int y, int dst, float alpha, float beta, float diag) {
    if (rc == 0) rc = symmetric<PROD, SQUARE, MUON>(with(3), with(5), blocks[3], blocks[5], Op{x, y, dst, flip, alpha, beta, diag}, st);
  };
  auto applied = [&](int f, float alpha, float beta, bool last) {
    const Op op{f, f, 0, flip, alpha, beta, 0.f};
    if (rc == 0)
      rc = last ? apply<PROD, FINAL, MUON>(with(6), with(7), blocks[6], blocks[7], op, st) : apply<PROD, APPLY, MUON>(with(6), with(7), blocks[6], blocks[7], op, st);
    flip ^= 1;
  };
  const float q = chain_scale(abc);
  if (!chains || q == 0.f) {
    for (int s = 0; s < steps; ++s) {                     // B = b S + c S S;  X <- a X + B X
      gram();
      mats(MAT_S, MAT_S, MAT_P, cc * UNSCALE, cb, 0.f);
      applied(MAT_P, UNSCALE, ca, s + 1 == steps);
    }
    return rc;
  }
  for (int done = 0; done < steps;) {
    const int rest = steps - done, len = rest == 4 ? 2 : rest < 3 ? rest : 3;
    int f = MAT_Q, free = MAT_R;                          // where the product of the chain's factors is; the other place
    float scale = SCALE;
    gram();
    for (int i = 0; i < len; ++i) {
      const int p = i == 0 ? f : MAT_P;
      mats(MAT_S, MAT_S, p, cc * UNSCALE, cb, ca * SCALE);                     // P
      if (i > 0) {                                                             // product so far <- P times it, at scale q
        mats(MAT_P, f, free, q / (SCALE * scale), 0.f, 0.f);
        const int t = f; f = free; free = t;
        scale = q;
      }
      if (i + 1 < len) {                                                       // S <- P (P S)
        mats(p, MAT_S, MAT_T, UNSCALE, 0.f, 0.f);
        mats(p, MAT_T, MAT_S, UNSCALE, 0.f, 0.f);
      }
    }
    done += len;
    applied(f, 1.f / scale, 0.f, done == steps);
  }
  return rc;
}

// One matrix of `batch` like it, with the stages a block does of its gram and of its square product: its splits and the blocks of every launch.
struct Shape { int gram_splits, square_splits, blocks[LAUNCHES]; long long slabs; };
template <int PROD> Shape shape_of(int rows, int cols, long long batch, int gram_chunk, int square_chunk) {
  const long long n = (long long)rows * cols, slice = slice_of(n);
  const Lay<PROD> L(rows, cols);
  const long long pieces = (long long)rows * ((PROD == 3 ? L.ldx / 2 : L.ldx) / 8);
  const int thin = rows < cols ? rows : cols, wide = rows < cols ? cols : rows, t = tri(thin);
  Shape h{};
  auto splits = [](int ks, int chunk) { return (ks + chunk - 1) / chunk; };
  h.gram_splits = splits(stages(wide, PROD), gram_chunk);
  h.square_splits = splits(stages(thin, PROD), square_chunk);
  h.blocks[0] = (int)((n + slice - 1) / slice);
  h.blocks[1] = (int)((pieces + INIT_CHUNKS - 1) / INIT_CHUNKS);
  h.blocks[2] = t * h.gram_splits;
  h.blocks[3] = t * h.square_splits;
  h.blocks[4] = h.gram_splits > 1 ? t * gt::Tile<128, 128>::FM : 0;
  h.blocks[5] = h.square_splits > 1 ? t * gt::Tile<128, 128>::FM : 0;
  const bool big = large_apply(rows, cols, batch);
  h.blocks[6] = big ? 0 : full(rows, cols, 128);
  h.blocks[7] = big ? full(rows, cols, 256) : 0;
  const int most = h.gram_splits > h.square_splits ? h.gram_splits : h.square_splits;
  h.slabs = most > 1 ? (long long)t * most * SLAB : 0;
  return h;
}

Shape shape_of(int rows, int cols, int prod, long long batch, int gram_chunk, int square_chunk) {
  return prod == 3 ? shape_of<3>(rows, cols, batch, gram_chunk, square_chunk) : shape_of<1>(rows, cols, batch, gram_chunk, square_chunk);
}
Shape shape_of_batch(int rows, int cols, int prod, int batch) {
  const int thin = rows < cols ? rows : cols, wide = rows < cols ? cols : rows;
  const long long tiles = (long long)batch * tri(thin);
  return shape_of(rows, cols, prod, batch, chunk_for(tiles, stages(wide, prod)), chunk_for(tiles, stages(thin, prod)));
}
// Sets of different matrices: the stages that a block does at most, by the same measure as chunk_for.  `ks`: stages of matrix i's tiles.  Blocks of
// different lengths are handed out longest first: more than fit at once take their sum's share of the chip and half of the longest.
// (ResNet-50's Muon step, square products: parts of 8 stages 42 us, 16 36 us, 32 - no part, no join - 27 us.)
template <class KS> int set_chunk(const int* thin, int n, KS&& ks) {
  int most = 1, best = 1;
  for (int i = 0; i < n; ++i) most = max(most, ks(i));
  double least = 1e30;
  for (int c = min(8, most); ; c = min(c + 8, most)) {
    double blocks = 0, sum = 0, parts = 0, longest = 0;
    for (int i = 0; i < n; ++i) {
      const int s = (ks(i) + c - 1) / c, per = (ks(i) + s - 1) / s;
      blocks += (double)tri(thin[i]) * s;
      sum += (double)tri(thin[i]) * s * (per + 6);
      if (s > 1) parts += (double)tri(thin[i]) * s;
      longest = per + 6 > longest ? per + 6 : longest;
    }
    double t = blocks <= CUS ? 0.6 * longest : longest;
    if (blocks > SLOTS && sum / SLOTS + 0.5 * longest > t) t = sum / SLOTS + 0.5 * longest;
    if (parts > 0) t += 2.5 + parts / 60;
    if (t < least) { least = t; best = c; }
    if (c == most) break;
  }
  return best;
}

}  // namespace

// fp16 elements of workspace for one matrix (-1: it is too large, here and in the other calls)
extern "C" long long ddl_ns_workspace(int rows, int cols, int prod) {
  if (!addressable(rows, cols, prod)) return -1;
  return prod == 3 ? Lay<3>(rows, cols).size : Lay<1>(rows, cols).size;
}

// Products of a plain call.  bf16 results need no more than 11-bit operands in large matrices (relative error of the result 0.0018 to 0.0021,
// of which its rounding is 0.0017), but few products average less: 0.0023 to 0.0032 at thin sides of 128 to 16, 0.0017 with PROD = 3.
extern "C" int ddl_ns_prod(int rows, int cols, int is_bf16) { return is_bf16 && min(rows, cols) > 128 ? 1 : 3; }

// 1: one block does the whole matrix in one launch, which needs no workspace
extern "C" int ddl_ns_solo(int rows, int cols) { return rows > 0 && cols > 0 && solo(rows, cols) ? 1 : 0; }

extern "C" int ddl_ns_max_parts() { return MAX_PARTS; }

// A set of n matrices that share launches: out[0], out[1] the stages that a block of their gram and of their square products does at most
extern "C" int ddl_ns_chunks(const int* thin, const int* wide, int n, int prod, int* out) {
  if (n <= 0 || (prod != 1 && prod != 3)) return -1;
  out[0] = set_chunk(thin, n, [&](int i) { return stages(wide[i], prod); });
  out[1] = set_chunk(thin, n, [&](int i) { return stages(thin[i], prod); });
  return 0;
}

// For one of `batch` equal matrices (gram_chunk 0), or one of a set of matrices with the chunks of ddl_ns_chunks (batch 1): out[0..1] the splits
// of the gram and of the square product, out[2..9] blocks of every launch; returns the floats of partial tiles it needs.
extern "C" long long ddl_ns_shape(int rows, int cols, int prod, int batch, int gram_chunk, int square_chunk, int* out) {
  if (!addressable(rows, cols, prod) || batch <= 0 || gram_chunk < 0 || square_chunk < 0 || (gram_chunk == 0) != (square_chunk == 0)) return -1;
  const Shape h = gram_chunk == 0 ? shape_of_batch(rows, cols, prod, batch) : shape_of(rows, cols, prod, 1, gram_chunk, square_chunk);
  out[0] = h.gram_splits;
  out[1] = h.square_splits;
  for (int i = 0; i < LAUNCHES; ++i) out[2 + i] = h.blocks[i];
  return h.slabs;
}

// 1: matrices with these thin and wide sides take their steps in chains
extern "C" int ddl_ns_chains(const int* thin, const int* wide, int n) {
  double chained = 0.0, single = 0.0;
  for (int i = 0; i < n; ++i) {
    chained += chained_work(thin[i], wide[i]);
    single += single_work(thin[i], wide[i]);
  }
  return use_chains(chained, single) ? 1 : 0;
}

extern "C" int ddl_ns_mat_bytes() { return (int)sizeof(NsMat); }

// g, out: [batch][rows][cols], bf16 or fp32;  ws: batch * ddl_ns_workspace fp16;  parts: batch * MAX_PARTS doubles;  slabs: batch times what
// ddl_ns_shape(.., batch, 0, 0, ..) returns, floats;  abc on the host
extern "C" int ddl_orthogonalize(const void* g, int is_bf16, void* out, void* ws, double* parts, float* slabs, int batch, int rows, int cols,
                                 int prod, int steps, const float* abc, float eps, void* stream) {
  if (batch <= 0 || !addressable(rows, cols, prod) || steps <= 0) return -1;
  const Shape h = shape_of_batch(rows, cols, prod, batch);
  NsArgs a{};
  a.one.rows = rows; a.one.cols = cols;
  a.one.gram_splits = h.gram_splits; a.one.square_splits = h.square_splits;
  a.g_stride = (long long)rows * cols;
  a.ws_stride = ddl_ns_workspace(rows, cols, prod);
  a.slab_stride = h.slabs;
  a.ws = (unsigned short*)ws;
  a.slabs = slabs;
  a.parts = parts;
  a.eps = eps;
  if (is_bf16) { a.g16 = (const bf16_t*)g; a.out16 = (bf16_t*)out; } else { a.g32 = (const float*)g; a.out32 = (float*)out; }
  if (solo(rows, cols) && prod != 3) return -1;           // ddl_ns_prod
  const double thin = min(rows, cols), wide = max(rows, cols);
  const bool one = solo(rows, cols), chains = prod == 3 && use_chains(chained_work(thin, wide), single_work(thin, wide));
  // a launch has less than 2^32 threads: more matrices take several (of all kinds)
  const long long most = 0xffffffffll / 512 / (one ? 1 : *std::max_element(h.blocks, h.blocks + LAUNCHES));
  if (most < 1) return -2;
  int rc = 0;
  for (long long b = 0; b < batch && rc == 0; b += most) {
    const int n = (int)min(most, batch - b);
    a.per = 1;
    if (one) {
      rc = is_bf16 ? launch_solo<3, false, false>(a, n, max(rows, cols), steps, abc, (hipStream_t)stream)
                   : launch_solo<3, false, true>(a, n, max(rows, cols), steps, abc, (hipStream_t)stream);
    } else {
      int blocks[LAUNCHES];
      for (int i = 0; i < LAUNCHES; ++i) blocks[i] = h.blocks[i] * n;
      rc = prod == 3 ? run_steps<3, false>(a, blocks, nullptr, h.blocks, steps, abc, chains, (hipStream_t)stream)
                     : run_steps<1, false>(a, blocks, nullptr, h.blocks, steps, abc, false, (hipStream_t)stream);
      a.ws += n * a.ws_stride; a.slabs += n * a.slab_stride; a.parts += (long long)n * MAX_PARTS;
    }
    if (is_bf16) { a.g16 += n * a.g_stride; a.out16 += n * a.g_stride; } else { a.g32 += n * a.g_stride; a.out32 += n * a.g_stride; }
  }
  return rc;
}

// Muon over the matrices of an arena.  table: NsMat[], maps: one int2[] after the other for the 8 launches, on the device;  blocks[8] on the host.
// hyper (device): [0] lr [1] momentum [2] nesterov [4] gradient scale.  solo_wide > 0: every matrix is a ddl_ns_solo one, the widest has this many
// columns (rows, if tall), blocks[0] is the number of matrices and maps[] names each once.  chains: ddl_ns_chains of the set.
extern "C" int ddl_muon_step(const void* table, const void* maps, const int* blocks, float* master, float* grad, float* mom, void* shadow,
                             const float* seg_wd, const float* hyper, void* ws, double* parts, float* slabs, int prod, int steps, const float* abc,
                             float eps, int zero_grad, int solo_wide, int chains, void* stream) {
  if (steps <= 0 || (prod != 1 && prod != 3)) return -1;
  NsArgs a{};
  a.table = (const NsMat*)table;
  a.ws = (unsigned short*)ws;
  a.slabs = slabs;
  a.parts = parts;
  a.eps = eps;
  a.grad = grad; a.mom = mom; a.master = master; a.shadow = (bf16_t*)shadow; a.seg_wd = seg_wd; a.hyper = hyper;
  a.zero_grad = zero_grad;
  if (solo_wide > 0) {
    a.map = (const int2*)maps;
    return prod == 3 ? launch_solo<3, true, true>(a, blocks[0], solo_wide, steps, abc, (hipStream_t)stream)
                     : launch_solo<1, true, false>(a, blocks[0], solo_wide, steps, abc, (hipStream_t)stream);
  }
  const int2* list[LAUNCHES];
  const int2* at = (const int2*)maps;
  for (int i = 0; i < LAUNCHES; ++i) { list[i] = at; at += blocks[i]; }
  return prod == 3 ? run_steps<3, true>(a, blocks, list, nullptr, steps, abc, chains != 0, (hipStream_t)stream)
                   : run_steps<1, true>(a, blocks, list, nullptr, steps, abc, false, (hipStream_t)stream);
}
