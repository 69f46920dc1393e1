// Output tiles of matrix products with 16-bit operands on the matrix cores (gfx950), shared by the orthogonalisation and
// the gated feed-forward kernels.
//
//   C[m][n] = sum_k A(m, k) B(n, k)          one block of four waves (2 x 2) per BM x BN tile, fp32 accumulators
//
// An operand is K-CONTIGUOUS (stored [rows][ld], reduction index fastest) or K-SLOW (stored [K][ld], its own index fastest), so
// that X X^T, B X, dY W, dY^T X ... all run on the tensors as they lie in memory, with no transposed copies:
//   * both kinds go global -> LDS with 16-byte LDS-DMA, 1 KiB per wave instruction, a stage of 64 reduction steps = 128 bytes of
//     LDS per tile row;
//   * K-contiguous tiles keep 128-byte rows; the 16-byte chunk c of row r lies at c ^ ((r >> 1) & 7), fragments are ds_read_b128;
//   * K-slow tiles keep their natural [64 k][128 columns] order (256-byte rows, chunk c of row r at
//     c ^ (((r & 3) << 2) | ((r >> 2) & 3))), fragments are pairs of transposing reads (ds_read_b64_tr_b16).
// Both give lane (g = lane >> 4, r = lane & 15) the reduction steps 8g..8g+7 of row r, so the kinds mix freely.
//
// Split operands (PROD = 3): a value is held as fp16 hi + fp16 lo (22 bits).  Rows then hold groups of 32 hi followed by their 32
// lo values, so a 128-byte LDS row is 32 reduction steps of both parts, the staging is the same, and the stage multiplies
// hi*hi + hi*lo + lo*hi (lo*lo is below 2^-22 of the product).
//
// The second argument of the MFMA takes A: a lane ends up with FOUR CONSECUTIVE n of one m, rows of C are stored through a wave's
// own LDS window as 16-byte pieces.
//
// Addresses: an operand's buffer descriptor is moved along the reduction by scalar adds in 64 bits, the per-lane 32-bit offsets
// only span one tile (rows x ld, or 64 k x ld), so tensors may exceed 4 GiB.  What lies outside reads as zero.
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

namespace gt {

constexpr unsigned OOB = 0xFFFFFFF0u;      // beyond any descriptor: the lane reads zero

// Tied forms (dst == src C, AGPR file): through the builtin the compiler gives the unrolled products rotating destinations and, for the large
// tile, moves half of the 256 accumulators back at every stage.  The waits for the fragments stay the
// compiler's (it sees the operands); nothing else touches the accumulators between settle() before and after the loop.
struct Bf16 {
  static __device__ __forceinline__ void mfma_tied(const s16x8& a, const s16x8& b, f32x4& c) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ f32x4 mfma(const s16x8 a, const s16x8 b, const f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
struct Fp16 {
  static __device__ __forceinline__ void mfma_tied(const s16x8& a, const s16x8& b, f32x4& c) {
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ f32x4 mfma(const s16x8 a, const s16x8 b, const f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// wait states between a matrix instruction the compiler does not see and other accesses of its registers
__device__ __forceinline__ void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

__device__ __forceinline__ u32x4 make_rsrc(const void* base, unsigned long long bytes) {
  const unsigned long long a = (unsigned long long)base;
  const unsigned n = bytes > 0xFFFFFFE0ull ? 0xFFFFFFE0u : (unsigned)bytes;
  u32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((unsigned)a);
  r[1] = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32) & 0xffffu);
  r[2] = __builtin_amdgcn_readfirstlane(n);
  r[3] = 0x00020000u;
  return r;
}

// Hidden from the compiler's wait insertion: it would drain every LDS-DMA it can see in front of the next transposing read.
// The waits are the explicit ones below.  M0 (the LDS address) has no other user in these kernels.
__device__ __forceinline__ void dma16(const u32x4 rsrc, unsigned lds_addr, unsigned voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds_addr), "v"(voff), "s"(rsrc) : "memory");
}

// One operand of one tile.  `rows`: valid rows (m or n) from row0 on; `k`: reduction length in elements; `ld`: elements per stored
// row (the hi/lo pairs of split operands counted singly: ld = 2 * padded width).
struct Operand {
  const unsigned short* base;
  long long ld;
  int row0, rows;        // first row of the tile, number of valid rows of the whole operand
  int k;
};

enum { CONTIG = 0, SLOW = 1 };

template <int ROWS, int MODE, int PROD>
struct Stager {
  static constexpr int NP = ROWS / 32;             // 1 KiB pieces per wave and stage
  unsigned voff[NP];
  const unsigned short* base;
  long long ld;
  int k, kdone;                                    // reduction steps left to stage: k - kdone
  int kchunk;                                      // CONTIG: first reduction step of this lane's chunk

  __device__ __forceinline__ void init(const Operand& o, int wid, int lane) {
    base = o.base; ld = o.ld; k = o.k; kdone = 0;
    if (MODE == CONTIG) {
      const int chunk = (lane & 7) ^ ((4 * (wid & 1) + (lane >> 4)) & 7);
      kchunk = PROD == 3 ? 0 : chunk * 8;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int r = o.row0 + j * 32 + wid * 8 + (lane >> 3);
        voff[j] = r < o.rows ? (unsigned)(((long long)(r - o.row0) * ld + chunk * 8) * 2) : OOB;
      }
      base += (long long)o.row0 * ld;
    } else {
      const int chunk = (lane & 15) ^ (((lane >> 4) << 2) | wid);
      kchunk = 0;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int q = j * 4 + wid, sub = q >> 4, row = (q & 15) * 4 + (lane >> 4);
        const int col = o.row0 + sub * 128 + chunk * 8;
        const bool ok = col < o.rows;
        if (PROD == 3)
          voff[j] = ok ? (unsigned)(((long long)(row & 31) * ld + (col >> 5) * 64 + (row >> 5) * 32 + (col & 31)) * 2) : OOB;
        else
          voff[j] = ok ? (unsigned)(((long long)row * ld + col) * 2) : OOB;
      }
    }
  }
  static constexpr int KSTEP = PROD == 3 ? 32 : 64;

  // only stages [first, first + n) of the reduction
  __device__ __forceinline__ void part(int first, int n) {
    const int end = (first + n) * KSTEP;
    kdone = first * KSTEP;
    base += MODE == SLOW ? kdone * ld : (long long)first * 64;
    k = end < k ? end : k;
  }

  // Staging of one stage: begin, every piece, end.  Stages behind the end of the reduction come out as zeros.
  u32x4 rsrc;
  unsigned kill;
  __device__ __forceinline__ void begin() {
    // bytes the descriptor may reach: K-slow tiles end behind the last reduction step; K-contiguous ones check per chunk
    if (MODE == SLOW) {
      const int left = k - kdone;
      rsrc = make_rsrc(base, left > 0 ? (unsigned long long)left * (unsigned long long)ld * 2ull : 0ull);
    } else {
      rsrc = make_rsrc(base, 0xFFFFFFE0ull);
    }
    kill = MODE == CONTIG && kdone + kchunk >= k ? OOB : 0u;
  }
  __device__ __forceinline__ void piece(int j, unsigned lds, int wid) const {
    dma16(rsrc, lds + (unsigned)((j * 4 + wid) * 1024), voff[j] | kill);
  }
  __device__ __forceinline__ void end() {
    kdone += KSTEP;
    base += MODE == SLOW ? (long long)KSTEP * ld : 64;
  }
};

template <class S> __device__ __forceinline__ void issue(S& s, unsigned lds, int wid) {
  s.begin();
#pragma unroll
  for (int j = 0; j < S::NP; ++j) s.piece(j, lds, wid);
  s.end();
}

template <int ROWS, int MODE>
struct Reader {                                    // fragments of a wave's ROWS / 2 rows
  int off_a, off_b;
  __device__ __forceinline__ void init(int w, int lane) {
    if (MODE == CONTIG) {
      off_a = (w * (ROWS / 2) + (lane & 15)) * 128 + (((lane >> 4) ^ ((lane >> 1) & 7)) << 4);
      off_b = off_a ^ 64;                          // second half of the stage: chunk + 4
    } else {
      const int g = lane >> 4, q4 = (lane & 15) >> 2, pp = lane & 3;
      const int c0 = w * (ROWS / 2), ch = ((c0 & 127) >> 3) + (pp >> 1);
      const int row = 8 * g + q4, swz = (q4 << 2) | ((2 * g) & 3);
      off_a = (c0 >> 7) * 16384 + row * 256 + ((ch ^ swz) << 4) + (pp & 1) * 8;
      off_b = (off_a ^ 16) + 4 * 256;              // rows + 4: the swizzle flips the chunk's lowest bit
    }
  }
  // fragment i (16 rows), half h of the stage
  __device__ __forceinline__ s16x8 get(const char* tile, int i, int h) const {
    if (MODE == CONTIG) return *reinterpret_cast<const s16x8*>(tile + (h ? off_b : off_a) + i * 2048);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(tile + (off_a ^ (i << 5)) + h * 8192));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(tile + (off_b ^ (i << 5)) + h * 8192));
    return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
};

struct None {};                                    // epilogues that read nothing
struct NoLoad { __device__ __forceinline__ None operator()(int, int) const { return None{}; } };

template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory"); }

// 128 x 128 with NST = 2 stages: 64 KiB of LDS, two blocks on a CU; with NST = 4: one block, three stages on their way, for launches of no more
// blocks than CUs.  256 x 256 (NST = 2, 128 KiB, one wave per SIMD, 128 x 128 a wave) asks the L2 -> LDS path, which sits at its ~25 bytes per
// clock and CU with 128 x 128, for half the bytes per operation.
template <int BM, int BN, int NST = 2> struct Tile {
  static constexpr int WM = BM / 2, WN = BN / 2;           // rows / columns of a wave
  static constexpr int FM = WM / 16, FN = WN / 16;
  static constexpr int STAGE = (BM + BN) * 128;
  static constexpr int WPITCH = WN + 4;                    // floats per row of a wave's output window
  static constexpr int WBYTES = 16 * WPITCH * 4;
  static constexpr int SMEM = NST * STAGE;
  static constexpr int SLAB = FN * FM * 1024;                // floats of a partial tile (all four waves)
  static_assert(4 * WBYTES <= SMEM, "output windows reuse the stages");
  f32x4 acc[FN][FM];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Partial tiles of a split reduction: every lane's accumulators as they are, 16-byte stores that are contiguous over the block.
  __device__ __forceinline__ void put_slab(float* slab, int tid) const {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) *reinterpret_cast<f32x4*>(slab + ((i * FM + j) * 256 + tid) * 4) = acc[i][j];
  }
  // Only the wave's 16-row group j, so that a tile is joined by FM blocks.  In order: the result does not depend on timing.
  __device__ __forceinline__ void sum_slabs(const float* slab, int n, int j, int tid) {
#pragma unroll
    for (int i = 0; i < FN; ++i) acc[i][0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
#pragma unroll
      for (int i = 0; i < FN; ++i) acc[i][0] += *reinterpret_cast<const f32x4*>(slab + (long long)s * SLAB + ((i * FM + j) * 256 + tid) * 4);
    }
  }

  // acc += product over nk stages.
  //
  // A wave reads the fragments of the next half stage between the products of this one (a[0], b[0]: first halves; a[1], b[1]: second), and there
  // is one barrier per stage, between the halves: behind it every wave has read all of stage t (its second half is in registers) and all
  // pieces of stage t+1 have landed; stage t+NST is then requested into t's place and the first half of t+1 is read.
  template <class E, int AM, int BMD, int PROD, class SA, class SB>
  __device__ __forceinline__ void mul(SA& sa, SB& sb, int nk, char* smem, int wid, int lane) {
    static_assert(FM == FN && SA::NP == FM && SB::NP == FN, "square tiles of a 2 x 2 block of waves");
    constexpr int H = FN / 2, PER = SA::NP + SB::NP, BOFF = BM * 128;
    const unsigned lds = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)smem;
    Reader<BM, AM> ra;
    Reader<BN, BMD> rb;
    ra.init(wid & 1, lane);
    rb.init(wid >> 1, lane);
#pragma unroll
    for (int q = 0; q < NST; ++q) {                        // behind the end: zeros, so that the counted waits stay uniform
      issue(sa, lds + q * STAGE, wid);
      issue(sb, lds + q * STAGE + BOFF, wid);
    }
    wait_vm<(NST - 1) * PER>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    s16x8 a0[FM], b0[FN], a1[FM], b1[FN], b2[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) a0[i] = ra.get(smem, i, 0);
#pragma unroll
    for (int i = 0; i < FN; ++i) b0[i] = rb.get(smem + BOFF, i, 0);
    settle();
    int cur = 0;
    for (int t = 0; t < nk; ++t) {
      const int nxt = cur + STAGE == SMEM ? 0 : cur + STAGE;
      const char* const ta = smem + cur;
      const char* const tb = ta + BOFF;
      const char* const na = smem + nxt;
      const char* const nb = na + BOFF;
      const unsigned refill = lds + (unsigned)cur;
      // first half: hi x hi of split operands
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        if (i < H) { a1[2 * i] = ra.get(ta, 2 * i, 1); a1[2 * i + 1] = ra.get(ta, 2 * i + 1, 1); }
        else       { b1[2 * (i - H)] = rb.get(tb, 2 * (i - H), 1); b1[2 * (i - H) + 1] = rb.get(tb, 2 * (i - H) + 1, 1); }
#pragma unroll
        for (int j = 0; j < FM; ++j) E::mfma_tied(b0[i], a0[j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
      wait_vm<(NST - 2) * PER>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      sa.begin();
      sb.begin();
#pragma unroll
      for (int i = 0; i < FN; ++i) {                       // second half;  split operands: lo x hi
        if (i < H) {
          sa.piece(2 * i, refill, wid); sa.piece(2 * i + 1, refill, wid);
          sb.piece(2 * i, refill + BOFF, wid); sb.piece(2 * i + 1, refill + BOFF, wid);
          if (PROD == 1) { a0[2 * i] = ra.get(na, 2 * i, 0); a0[2 * i + 1] = ra.get(na, 2 * i + 1, 0); }
        } else if (PROD == 1) {
          b0[2 * (i - H)] = rb.get(nb, 2 * (i - H), 0); b0[2 * (i - H) + 1] = rb.get(nb, 2 * (i - H) + 1, 0);
        }
#pragma unroll
        for (int j = 0; j < FM; ++j) {
          if (PROD == 1) E::mfma_tied(b1[i], a1[j], acc[i][j]);
          else           E::mfma_tied(b1[i], a0[j], acc[i][j]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (PROD == 3) {
#pragma unroll
        for (int i = 0; i < FN; ++i) {                     // hi x lo;  the hi fragments of A are free, those of B are not yet
          if (i < H) { a0[2 * i] = ra.get(na, 2 * i, 0); a0[2 * i + 1] = ra.get(na, 2 * i + 1, 0); }
          else       { b2[2 * (i - H)] = rb.get(nb, 2 * (i - H), 0); b2[2 * (i - H) + 1] = rb.get(nb, 2 * (i - H) + 1, 0); }
#pragma unroll
          for (int j = 0; j < FM; ++j) E::mfma_tied(b0[i], a1[j], acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < FN; ++i) b0[i] = b2[i];
      }
      sa.end();
      sb.end();
      cur = nxt;
    }
    settle();
    wait_vm<0>();
    __builtin_amdgcn_s_barrier();                          // every wave has read its last fragments: windows may be written
    asm volatile("" ::: "memory");
  }

  // Rows of the wave's part, 16 at a time through its own window: f(m, n, v[8], aux) with tile-relative m and n (n a multiple of 8), where
  // aux = load(m, n) was requested one row group earlier (what an epilogue reads would otherwise cost a memory latency per group).
  // With COLS the window gets f's values back and is walked down its columns: ft(n, m, v[8]), m a multiple of 8 - the transposed tile.
  // NJ = 1: the one group that sum_slabs() left, which is group j0 of the tile.
  template <bool COLS, int NJ = FM, class LD, class F, class FT>
  __device__ __forceinline__ void store(char* smem, int wid, int lane, LD&& load, F&& f, FT&& ft, int j0 = 0) {
    constexpr int NC = WN / 32;
    float* const win = reinterpret_cast<float*>(smem + wid * WBYTES);
    const int wm0 = (wid & 1) * WM + j0 * 16, wn0 = (wid >> 1) * WN;
    auto row = [&](int c) { return (c * 64 + lane) / (WN / 8); };
    auto chunk = [&](int c) { return (c * 64 + lane) % (WN / 8) * 8; };
    decltype(load(0, 0)) aux[2][NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) aux[0][c] = load(wm0 + row(c), wn0 + chunk(c));
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if (j + 1 < NJ) {
#pragma unroll
        for (int c = 0; c < NC; ++c) aux[(j + 1) & 1][c] = load(wm0 + (j + 1) * 16 + row(c), wn0 + chunk(c));
      }
#pragma unroll
      for (int i = 0; i < FN; ++i)
        *reinterpret_cast<f32x4*>(win + (lane & 15) * WPITCH + i * 16 + (lane >> 4) * 4) = acc[i][j];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float* const at = win + row(c) * WPITCH + chunk(c);
        float v[8];
        *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(at);
        *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(at + 4);
        f(wm0 + j * 16 + row(c), wn0 + chunk(c), v, aux[j & 1][c]);
        if (COLS) {
          *reinterpret_cast<f32x4*>(at) = *reinterpret_cast<const f32x4*>(v);
          *reinterpret_cast<f32x4*>(at + 4) = *reinterpret_cast<const f32x4*>(v + 4);
        }
      }
      if (COLS) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int idx = c * 64 + lane, col = idx >> 1, half = idx & 1;
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = win[(half * 8 + e) * WPITCH + col];
          ft(wn0 + col, wm0 + j * 16 + half * 8, v);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }

  // Gate / up pairs: columns [0, WN/2) of a wave are gate features, the rest the up features of the same index:
  // f(m, feature, gate[8], up[8]) with tile-relative m and feature.
  template <int NJ = FM, class F>
  __device__ __forceinline__ void store_pairs(char* smem, int wid, int lane, F&& f, int j0 = 0) {
    float* const win = reinterpret_cast<float*>(smem + wid * WBYTES);
    const int wm0 = (wid & 1) * WM + j0 * 16, wf0 = (wid >> 1) * (WN / 2);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int i = 0; i < FN; ++i)
        *reinterpret_cast<f32x4*>(win + (lane & 15) * WPITCH + i * 16 + (lane >> 4) * 4) = acc[i][j];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int c = 0; c < WN / 64; ++c) {
        const int idx = c * 64 + lane, row = idx / (WN / 16), ch = idx % (WN / 16);
        float g[8], u[8];
        const float* src = win + row * WPITCH + ch * 8;
        *reinterpret_cast<f32x4*>(g) = *reinterpret_cast<const f32x4*>(src);
        *reinterpret_cast<f32x4*>(g + 4) = *reinterpret_cast<const f32x4*>(src + 4);
        *reinterpret_cast<f32x4*>(u) = *reinterpret_cast<const f32x4*>(src + WN / 2);
        *reinterpret_cast<f32x4*>(u + 4) = *reinterpret_cast<const f32x4*>(src + WN / 2 + 4);
        f(wm0 + j * 16 + row, wf0 + ch * 8, g, u);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
};

constexpr int CUS = 256, SLOTS = 2 * CUS;         // two 128 x 128 blocks run on a CU

// Stages of its reduction that a block does when `tiles` equal 128 x 128 tiles have `ks` stages each: the split with the least rounds of blocks
// times stages.  A block's start and end cost about 6 stages; partial tiles are 64 KiB each to write and to read again (joining 240 takes
// 4.4 us, 408 13 us, 952 18 us, where a stage is about 1 us); a block alone on its CU runs its stages in 0.6 of the time it needs beside another.  `time`, if wanted: of the choice, in stages of a full CU.
inline int chunk_for(long long tiles, int ks, double* time = nullptr) {
  int best = ks;
  double least = 1e30;
  for (int s = 1; s == 1 || s <= ks / 8; ++s) {
    const long long blocks = tiles * s;
    if (s > 1 && blocks > 4 * SLOTS) break;
    const int per = (ks + s - 1) / s;
    const double t = (double)((blocks + SLOTS - 1) / SLOTS) * (per + 6) * (blocks <= CUS ? 0.6 : 1.0) + (s > 1 ? 2.5 + (double)blocks / 60.0 : 0.0);
    if (t < least) { least = t; best = per; }
  }
  if (time != nullptr) *time = least;
  return best;
}

}  // namespace gt
