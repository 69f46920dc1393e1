// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step built on it (gfx950).
//
//   X0 = G / (|G|_F + eps);   `steps` times:  S = X X^T (X^T X when X is taller than wide),  X <- a X + (b S + c S S) X
// drives every singular value of X to about one while the singular vectors stay.  Per step 2 m^2 n (S, symmetric: half is
// computed, half mirrored: m^2 n) + 2 m^3 (S S, likewise m^3) + 2 m^2 n operations, m the thin side: all of it matrix products,
// run on the tiles of gemm_tile.h.  A tall X is never transposed: its gram matrix takes both operands K-slow, its update is X B.
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
// Many matrices share every launch: blocks find their matrix through maps of (matrix, block) pairs, so an optimizer step over a whole
// network is 2 + 3 * steps launches.
#include "common.h"
#include "host_util.h"
#include "gemm_tile.h"
#include <math.h>

namespace {

constexpr float SCALE = 4096.f, UNSCALE = 1.f / 4096.f;
constexpr int MAX_PARTS = 256;                   // partial sums of squares per matrix
constexpr int INIT_CHUNKS = 1024;                // 8-element pieces of X0 per block of the init kernel

struct NsMat {                                   // one matrix of a step (device table, or the one of a plain call)
  long long elem;                                // Muon: element offset in the arena;  plain: 0
  long long ws;                                  // fp16 offset of its workspace: X, X', S, B
  int rows, cols, seg;
  float scale;                                   // Muon: factor of the update
};

struct NsArgs {
  const NsMat* table;                            // null: every matrix is `one`, at strides
  const int2* map;                               // with a table: (matrix, block) of every block
  int per;                                       // without: blocks per matrix
  NsMat one;
  long long g_stride, ws_stride;
  unsigned short* ws;
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
  long long ldx, lds, x0, x1, s, b, size, lo;    // lo: distance from a hi value to its lo value
  __host__ __device__ Lay(int rows, int cols) {
    const int thin = rows < cols ? rows : cols;
    if (PROD == 3) {
      ldx = 2 * up(cols, 32); lds = 2 * up(thin, 32);
      x0 = 0; x1 = (long long)rows * ldx; s = 2 * x1; b = s + (long long)thin * lds; size = up(b + (long long)thin * lds, 64);
      lo = 32;
    } else {
      ldx = up(cols, 64); lds = up(thin, 64);
      x0 = 0; lo = (long long)rows * ldx; x1 = 2 * lo; s = 4 * lo; b = s + (long long)thin * lds;
      size = up(b + (long long)thin * lds, 64);
    }
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
      float q = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float ge = gs * g[e];
        v[e] = mu * v[e] + ge;
        const float u = muon_update(ge, v[e], mu, nest);
        s += (double)u * (double)u;
      }
      (void)q;
      *reinterpret_cast<f32x4*>(mp + i) = v;
    }
  } else {
    for (long long i = lo + threadIdx.x; i < hi; i += 256) {
      const float g = a.g32 != nullptr ? a.g32[m.elem + i] : bf16_to_f32(a.g16[m.elem + i]);
      s += (double)g * (double)g;
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
  double s = (int)threadIdx.x < parts ? a.parts[(long long)mat * MAX_PARTS + threadIdx.x] : 0.0;
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

// ---- the products.  KIND 0: S = X X^T;  1: B = b S + c S S;  2: X' = a X + B X;  3: the same, last step, to the destination.
enum { GRAM = 0, SQUARE = 1, APPLY = 2, FINAL = 3 };

template <int PROD, int KIND, int BT, bool MUON>
__global__ __launch_bounds__(256, 2) void ns_product_kernel(const NsArgs a, const int flip, const float alpha, const float beta) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  int mat, idx;
  const NsMat m = locate(a, xcd_remap(blockIdx.x, gridDim.x), mat, idx);
  const Lay<PROD> L(m.rows, m.cols);
  const bool tall = m.rows > m.cols;
  const int thin = tall ? m.cols : m.rows;
  unsigned short* const ws = a.ws + m.ws;
  unsigned short* const X = ws + (flip ? L.x1 : L.x0);
  unsigned short* const S = ws + L.s;
  unsigned short* const B = ws + L.b;

  int ti, tj;
  if (KIND <= SQUARE) {                                   // lower triangle, row by row
    ti = (int)((sqrtf(8.f * (float)idx + 1.f) - 1.f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= idx) ++ti;
    while (ti * (ti + 1) / 2 > idx) --ti;
    tj = idx - ti * (ti + 1) / 2;
  } else {
    const int tm = (m.rows + BT - 1) / BT;
    tj = idx / tm;
    ti = idx - tj * tm;
  }
  const int m0 = ti * BT, n0 = tj * BT;

  gt::Tile<BT, BT> tile;
  tile.zero();
  auto run = [&](auto am, auto bm, const unsigned short* pa, long long lda, int ra, const unsigned short* pb, long long ldb, int rb, int k) {
    constexpr int AM = decltype(am)::value, BMD = decltype(bm)::value;
    gt::Stager<BT, AM, PROD> sa;
    gt::Stager<BT, BMD, PROD> sb;
    sa.init(gt::Operand{pa, lda, m0, ra, k}, wid, lane);
    sb.init(gt::Operand{pb, ldb, n0, rb, k}, wid, lane);
    tile.template mul<gt::Fp16, AM, BMD, PROD>(sa, sb, (k + sa.KSTEP - 1) / sa.KSTEP, smem, wid, lane);
  };
  struct C { enum { value = gt::CONTIG }; };
  struct W { enum { value = gt::SLOW }; };
  if (KIND == GRAM) {
    if (tall) run(W{}, W{}, X, L.ldx, m.cols, X, L.ldx, m.cols, m.rows);
    else      run(C{}, C{}, X, L.ldx, m.rows, X, L.ldx, m.rows, m.cols);
  } else if (KIND == SQUARE) {
    run(C{}, C{}, S, L.lds, thin, S, L.lds, thin, thin);
  } else {
    if (tall) run(C{}, C{}, X, L.ldx, m.rows, B, L.lds, thin, thin);
    else      run(C{}, W{}, B, L.lds, thin, X, L.ldx, m.cols, thin);
  }

  if (KIND <= SQUARE) {
    unsigned short* const dst = KIND == GRAM ? S : B;
    auto value = [&](int r, int c, float* v) {            // v <- alpha v + beta S(r, c), 8 columns
      if (KIND == SQUARE) {
        const unsigned short* q = S + Lay<PROD>::at(r, L.lds, c);
        const f16x8 h = *reinterpret_cast<const f16x8*>(q);
        if (PROD == 3) {
          const f16x8 l = *reinterpret_cast<const f16x8*>(q + 32);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = alpha * v[e] + beta * ((float)h[e] + (float)l[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = alpha * v[e] + beta * (float)h[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= alpha;
      }
    };
    const int ncol = (int)(PROD == 3 ? L.lds / 2 : L.lds);
    auto put = [&](int r, int c, float* v) {
      if (r >= thin || c >= ncol) return;
      value(r, c, v);
      unsigned short* q = dst + Lay<PROD>::at(r, L.lds, c);
      if (PROD == 3) split_store8(q, 32, v); else f16_store8(q, v);
    };
    if (ti != tj)
      tile.template store<true>(smem, wid, lane, [&](int r, int c, float* v) { put(m0 + r, n0 + c, v); },
                                [&](int r, int c, float* v) { put(n0 + r, m0 + c, v); });
    else
      tile.template store<false>(smem, wid, lane, [&](int r, int c, float* v) { put(m0 + r, n0 + c, v); }, [](int, int, float*) {});
  } else {
    unsigned short* const dst = ws + (flip ? L.x0 : L.x1);
    const int ncol = (int)(PROD == 3 ? L.ldx / 2 : L.ldx);
    float lr = 0.f, wd = 0.f;
    if (KIND == FINAL && MUON) { lr = a.hyper[0]; wd = a.seg_wd[m.seg]; }
    const bool wide8 = (m.cols & 7) == 0;
    tile.template store<false>(smem, wid, lane, [&](int r, int c, float* v) {
      r += m0; c += n0;
      if (r >= m.rows || c >= (KIND == FINAL ? m.cols : ncol)) return;
      const long long at = Lay<PROD>::at(r, L.ldx, c);
      const f16x8 h = *reinterpret_cast<const f16x8*>(X + at), l = *reinterpret_cast<const f16x8*>(X + at + L.lo);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = alpha * v[e] + beta * ((float)h[e] + (float)l[e]);
      if (KIND == APPLY) { split_store8(dst + at, L.lo, v); return; }
      const long long o = m.elem + (long long)r * m.cols + c;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= UNSCALE;
      if (MUON) {
        float* const wp = a.master + o;
        if (wide8) {
          float w[8];
          *reinterpret_cast<f32x4*>(w) = *reinterpret_cast<const f32x4*>(wp);
          *reinterpret_cast<f32x4*>(w + 4) = *reinterpret_cast<const f32x4*>(wp + 4);
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

constexpr int BT = 128;

struct Grids { int norm, init, tri, full; };

template <int PROD> Grids grids_of(int rows, int cols) {
  const long long n = (long long)rows * cols, slice = slice_of(n);
  const Lay<PROD> L(rows, cols);
  const long long pieces = (long long)rows * ((PROD == 3 ? L.ldx / 2 : L.ldx) / 8);
  const int thin = rows < cols ? rows : cols, t = (thin + BT - 1) / BT;
  Grids g;
  g.norm = (int)((n + slice - 1) / slice);
  g.init = (int)((pieces + INIT_CHUNKS - 1) / INIT_CHUNKS);
  g.tri = t * (t + 1) / 2;
  g.full = ((rows + BT - 1) / BT) * ((cols + BT - 1) / BT);
  return g;
}

template <int PROD, int KIND, bool MUON>
int launch_product(const NsArgs& a, int blocks, int flip, float alpha, float beta, hipStream_t st) {
  static SmemAttrOnce once;
  auto* fn = &ns_product_kernel<PROD, KIND, BT, MUON>;
  const int smem = gt::Tile<BT, BT>::SMEM;
  const int rc = once.ensure(reinterpret_cast<const void*>(fn), smem);
  if (rc != 0) return rc;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(ns_product_kernel<PROD, KIND, BT, MUON>), dim3(blocks), dim3(256), smem, st, a, flip, alpha, beta);
  return (int)hipGetLastError();
}

// blocks[4]: norm, init, triangle, full;  maps[4] likewise (null for a plain call)
template <int PROD, bool MUON>
int run_steps(NsArgs a, const int* blocks, const int2* const* maps, const int* per, int steps, const float* abc, hipStream_t st) {
  auto with = [&](int i) { a.map = maps != nullptr ? maps[i] : nullptr; a.per = per != nullptr ? per[i] : 1; return a; };
  hipLaunchKernelGGL(HIP_KERNEL_NAME(ns_norm_kernel<MUON>), dim3(blocks[0]), dim3(256), 0, st, with(0));
  hipLaunchKernelGGL(HIP_KERNEL_NAME(ns_init_kernel<PROD, MUON>), dim3(blocks[1]), dim3(256), 0, st, with(1));
  int rc = (int)hipGetLastError();
  if (rc != 0) return rc;
  for (int s = 0; s < steps; ++s) {
    const float ca = abc[0], cb = abc[1], cc = abc[2];
    rc = launch_product<PROD, GRAM, MUON>(with(2), blocks[2], s & 1, UNSCALE, 0.f, st);
    if (rc == 0) rc = launch_product<PROD, SQUARE, MUON>(with(2), blocks[2], s & 1, cc * UNSCALE, cb, st);
    if (rc != 0) return rc;
    rc = s + 1 < steps ? launch_product<PROD, APPLY, MUON>(with(3), blocks[3], s & 1, UNSCALE, ca, st)
                       : launch_product<PROD, FINAL, MUON>(with(3), blocks[3], s & 1, UNSCALE, ca, st);
    if (rc != 0) return rc;
  }
  return 0;
}

}  // namespace

// fp16 elements of workspace for one matrix
extern "C" long long ddl_ns_workspace(int rows, int cols, int prod) {
  if (rows <= 0 || cols <= 0 || (prod != 1 && prod != 3)) return -1;
  return prod == 3 ? Lay<3>(rows, cols).size : Lay<1>(rows, cols).size;
}

extern "C" int ddl_ns_max_parts() { return MAX_PARTS; }

// blocks of one matrix in the four launches: norm, init, triangle, full
extern "C" int ddl_ns_blocks(int rows, int cols, int prod, int* out) {
  if (rows <= 0 || cols <= 0 || (prod != 1 && prod != 3)) return -1;
  const Grids g = prod == 3 ? grids_of<3>(rows, cols) : grids_of<1>(rows, cols);
  out[0] = g.norm; out[1] = g.init; out[2] = g.tri; out[3] = g.full;
  return 0;
}

extern "C" int ddl_ns_mat_bytes() { return (int)sizeof(NsMat); }

// g, out: [batch][rows][cols], bf16 or fp32;  ws: batch * ddl_ns_workspace fp16;  parts: batch * MAX_PARTS doubles;  abc on the host
extern "C" int ddl_orthogonalize(const void* g, int is_bf16, void* out, void* ws, double* parts, int batch, int rows, int cols,
                                 int prod, int steps, const float* abc, float eps, void* stream) {
  if (batch <= 0 || rows <= 0 || cols <= 0 || steps <= 0 || (prod != 1 && prod != 3)) return -1;
  NsArgs a{};
  a.one.rows = rows; a.one.cols = cols;
  a.g_stride = (long long)rows * cols;
  a.ws_stride = ddl_ns_workspace(rows, cols, prod);
  a.ws = (unsigned short*)ws;
  a.parts = parts;
  a.eps = eps;
  if (is_bf16) { a.g16 = (const bf16_t*)g; a.out16 = (bf16_t*)out; } else { a.g32 = (const float*)g; a.out32 = (float*)out; }
  int per[4], blocks[4];
  ddl_ns_blocks(rows, cols, prod, per);
  for (int i = 0; i < 4; ++i) {
    if ((long long)per[i] * batch > 0x7fffffffll) return -2;
    blocks[i] = per[i] * batch;
  }
  return prod == 3 ? run_steps<3, false>(a, blocks, nullptr, per, steps, abc, (hipStream_t)stream)
                   : run_steps<1, false>(a, blocks, nullptr, per, steps, abc, (hipStream_t)stream);
}

// Muon over the matrices of an arena.  table: NsMat[] and maps: int2[] on the device, blocks[4] on the host.
// hyper (device): [0] lr [1] momentum [2] nesterov [4] gradient scale.
extern "C" int ddl_muon_step(const void* table, const void* map0, const void* map1, const void* map2, const void* map3,
                             const int* blocks, float* master, float* grad, float* mom, void* shadow, const float* seg_wd,
                             const float* hyper, void* ws, double* parts, int prod, int steps, const float* abc, float eps,
                             int zero_grad, void* stream) {
  if (steps <= 0 || (prod != 1 && prod != 3)) return -1;
  NsArgs a{};
  a.table = (const NsMat*)table;
  a.ws = (unsigned short*)ws;
  a.parts = parts;
  a.eps = eps;
  a.grad = grad; a.mom = mom; a.master = master; a.shadow = (bf16_t*)shadow; a.seg_wd = seg_wd; a.hyper = hyper;
  a.zero_grad = zero_grad;
  const int2* maps[4] = {(const int2*)map0, (const int2*)map1, (const int2*)map2, (const int2*)map3};
  return prod == 3 ? run_steps<3, true>(a, blocks, maps, nullptr, steps, abc, (hipStream_t)stream)
                   : run_steps<1, true>(a, blocks, maps, nullptr, steps, abc, (hipStream_t)stream);
}
