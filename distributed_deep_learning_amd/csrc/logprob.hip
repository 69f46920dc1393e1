// Log probabilities of given tokens, entropy and the most likely tokens of every row of logits, and their gradient (gfx950).
//
//   lse = log sum_j exp z_j      logp = z_t - lse      H = lse - sum_j p_j z_j      top: the k largest z_j - lse
//
// One pass over the logits: every thread carries the maximum m, s = sum e^(z - m) and q = sum e^(z - m) (z - m) of what it
// has seen (joining to a larger m' rescales: s' = f s, q' = f (q + (m - m') s), f = e^(m - m')); H = log s - q / s.  The kernel is
// bound by reading z once.  A row is cut into parts when there are too few rows to fill the chip, and a second launch joins
// (m, s, q) and the candidate lists of the parts.
//
// Top k in the same pass: the part's logits stay in registers (packed as loaded).  The threads form k' >= k disjoint groups (k' a power
// of two); the smallest of the groups' maxima is a bound that at least k elements reach and only about k' ln k' of them, whatever the
// part's length.  Those are gathered in LDS and ordered by counting.  Where very many elements tie with the bound: k rounds of a
// block-wide maximum.  Candidates are
// 64-bit keys, an order-preserving image of the value above the inverted index: equal values go to the lowest index.
//
// Measured: 8192 x 32000 bf16 without a list 90 us (5.8 TB/s: bandwidth), backward 185 us (5.7 TB/s);  2048 x 131072 bf16 with the top five 119 us and
// 7 us to join the parts (4.5 TB/s: the vector unit is as busy as the memory);  1 x 50257 fp32 with the top twenty 8 + 5 us (latency).
//
// Masked logits (-inf) have probability zero.  A row without any logit above -inf has logp = top = -inf, entropy 0, gradient 0.  A NaN
// or +inf in a row makes its results NaN; in the order of the top list NaN counts as the largest value.
//
// Backward, one pass (read z, write dz):  with G = g_logp + sum_k g_top[k]
//   dz_j = -p_j (G + g_H (z_j - lse + H)) + g_logp [j = t] + sum_k g_top[k] [j = idx_k]
#include "common.h"
#include "host_util.h"
#include <float.h>

namespace {

typedef unsigned long long u64;
constexpr int NT = 256;                           // threads per block
constexpr int CAP = 1024;                         // gathered candidates per part
constexpr int TOP_MAX = 64;

template <typename T> struct Io;
template <> struct Io<float> {
  static constexpr int ALIGN = 4;                 // elements per 16 bytes
  struct Raw { f32x4 a, b; };
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ Raw load(const float* p) {
    return Raw{*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 4)};
  }
  static __device__ __forceinline__ Raw stream(const float* p) {
    return Raw{__builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p)), __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + 4))};
  }
  static __device__ __forceinline__ Raw pack(const float* f) { return Raw{f32x4{f[0], f[1], f[2], f[3]}, f32x4{f[4], f[5], f[6], f[7]}}; }
  static __device__ __forceinline__ void unpack(const Raw& r, float* f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[e] = r.a[e]; f[4 + e] = r.b[e]; }
  }
  static __device__ __forceinline__ void store(float* p, const float* f) {
    *reinterpret_cast<f32x4*>(p) = f32x4{f[0], f[1], f[2], f[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{f[4], f[5], f[6], f[7]};
  }
  static __device__ __forceinline__ void put_stream(float* p, const float* f) {
    __builtin_nontemporal_store(f32x4{f[0], f[1], f[2], f[3]}, reinterpret_cast<f32x4*>(p));
    __builtin_nontemporal_store(f32x4{f[4], f[5], f[6], f[7]}, reinterpret_cast<f32x4*>(p + 4));
  }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
  static __device__ __forceinline__ void pin(Raw& r) { asm volatile("" : "+v"(r.a), "+v"(r.b)); }
};
template <> struct Io<bf16_t> {
  static constexpr int ALIGN = 8;
  typedef u32x4 Raw;
  static __device__ __forceinline__ float one(const bf16_t* p) { return bf16_to_f32(*p); }
  static __device__ __forceinline__ Raw load(const bf16_t* p) { return *reinterpret_cast<const u32x4*>(p); }
  static __device__ __forceinline__ Raw stream(const bf16_t* p) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)); }
  static __device__ __forceinline__ Raw pack(const float* f) { return pack8(f); }     // exact: the values came from bf16
  static __device__ __forceinline__ void unpack(const Raw& r, float* f) { unpack8(r, f); }
  static __device__ __forceinline__ void store(bf16_t* p, const float* f) { *reinterpret_cast<u32x4*>(p) = pack8(f); }
  static __device__ __forceinline__ void put_stream(bf16_t* p, const float* f) { __builtin_nontemporal_store(pack8(f), reinterpret_cast<u32x4*>(p)); }
  static __device__ __forceinline__ void put(bf16_t* p, float v) { *p = f32_to_bf16(v); }
  static __device__ __forceinline__ void pin(Raw& r) { asm volatile("" : "+v"(r)); }
};

// A row is a run of whole 16-byte aligned pieces of 8 elements, whatever its address, with up to 7 elements in front and behind that belong
// to part 0: its thread e < 16 holds one of them (e < 8: in front, else behind).
struct Split { int first, pieces, head, tail; };          // first: element of the first piece;  head, tail: elements in front and behind
template <typename T> __device__ __forceinline__ Split split_row(const T* row, int V) {
  const int mis = (int)(((u64)row / sizeof(T)) & (Io<T>::ALIGN - 1));
  const int first = mis == 0 ? 0 : Io<T>::ALIGN - mis;
  Split s;
  s.first = first < V ? first : V;
  s.pieces = (V - s.first) / 8;
  s.head = s.first;
  s.tail = V - s.first - 8 * s.pieces;
  return s;
}
__device__ __forceinline__ int edge_element(const Split& s, int tid) {       // -1: none
  if (tid < s.head) return tid;
  if (tid >= 8 && tid < 8 + s.tail) return s.first + 8 * s.pieces + tid - 8;
  return -1;
}
template <typename T> __device__ __forceinline__ typename Io<T>::Raw nothing() {
  const float f[8] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY};
  return Io<T>::pack(f);
}

struct Stat { float m, s, q; };

__device__ __forceinline__ void stat_rescale(Stat& a, float m) {       // to a maximum m >= a.m
  const float d = a.m - m, f = __expf(d);
  a.q = a.s == 0.f ? 0.f : f * (a.q + fmaxf(d, -200.f) * a.s);        // f is zero long before -200
  a.s = a.s == 0.f ? 0.f : f * a.s;
  a.m = m;
}
// Ignores quiet NaNs.  In assembly because fmaxf of values that came out of integer operations is compiled to two more operations each that
// quiet signalling NaNs (such a row is NaN by its sum in any case): 2 instead of 0.5 per element in a kernel whose vector unit is 88 % busy.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}
__device__ __forceinline__ float max8(const float* z) { return max3(max3(max3(z[0], z[1], z[2]), z[3], z[4]), max3(z[5], z[6], z[7]), z[7]); }

constexpr float LOG2E = 1.44269504f, LN2 = 0.69314718f;
__device__ __forceinline__ void stat_add8(Stat& a, const float* z) {     // a.m is at least the largest of z
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = z[e] - a.m, p = __expf(d);
    a.s += p;                                                            // a NaN (or inf - inf) stays in s
    a.q += p * fmaxf(d, -200.f);                                         // p is zero below about -104: no 0 * inf
  }
}
// The same sums with base-2 exponents, one operation less per element: z log2(e) - c is one fused operation, c = m log2(e) rounded, and what the
// rounding left, e = m log2(e) - c, is put right in the sums once (Base2::into).  For |m| < 2^20, where |e| < 1/16.
struct Base2 {
  float c, e, s, q;
  __device__ __forceinline__ void begin(float m) { c = m * LOG2E; e = fmaf(m, LOG2E, -c); s = q = 0.f; }
  __device__ __forceinline__ void add8(const float* z) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = fmaf(z[i], LOG2E, -c), p = __builtin_amdgcn_exp2f(d);
      s += p;
      q += p * fmaxf(d, -300.f);
    }
  }
  __device__ __forceinline__ void into(Stat& a) const {
    const float f = __builtin_amdgcn_exp2f(-e);
    a.s += f * s;
    a.q += f * LN2 * (q - e * s);
  }
};
__device__ __forceinline__ void stat_add1(Stat& a, float z) {
  if (z > a.m) stat_rescale(a, z);
  const float d = z - a.m, p = __expf(d);
  a.s += p;
  a.q += p * fmaxf(d, -200.f);
}
__device__ __forceinline__ Stat stat_join(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  stat_rescale(a, m);
  stat_rescale(b, m);
  return Stat{m, a.s + b.s, a.q + b.q};
}
__device__ __forceinline__ Stat stat_wave(Stat a) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) a = stat_join(a, Stat{__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.q, o, 64)});
  return a;
}

constexpr unsigned NAN_KEY = 0xfffffffeu;                               // one below the top: a candidate is always below ~0, where lists begin
__device__ __forceinline__ unsigned key_of(float z) {                    // order-preserving; -0 and 0 equal, NaN on top; 0 = absent
  const unsigned b = __float_as_uint(z + 0.f);
  if (z != z) return NAN_KEY;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) {
  if (k == NAN_KEY) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ u64 cand(unsigned key, int j) { return ((u64)key << 32) | (u64)(0xffffffffu - (unsigned)j); }
__device__ __forceinline__ u64 wave_max(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 w = __shfl_xor(v, o, 64);
    v = w > v ? w : v;
  }
  return v;
}
__device__ __forceinline__ u64 block_max(u64 v, u64* red) {              // red[4]; result in every thread
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 r = red[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) r = red[w] > r ? red[w] : r;
  return r;
}

// norm (null: not wanted): (m, log s) of every row; their sum is lse, but far from zero it would swallow log s
struct Outs { float* logp; float* ent; float* norm; float* top; long long* idx; };

// thread 0 writes the row's scalars, threads < k its list
template <typename T>
__device__ __forceinline__ void finish_row(const Stat& st, const T* row, long long token, int V, long long r, int k, u64 mine, const Outs& o) {
  const bool empty = st.s == 0.f;
  const float ls = __logf(st.s);
  if (threadIdx.x == 0) {
    const bool in = token >= 0 && token < V;
    const float zt = in ? Io<T>::one(row + token) : 0.f;
    o.logp[r] = in ? (empty ? -INFINITY : (zt - st.m) - ls) : 0.f;
    o.ent[r] = empty ? 0.f : ls - st.q / st.s;
    if (o.norm != nullptr) {
      o.norm[2 * r] = st.m;
      o.norm[2 * r + 1] = empty ? -INFINITY : ls;
    }
  }
  if ((int)threadIdx.x < k) {
    const float z = value_of((unsigned)(mine >> 32));
    o.top[r * k + threadIdx.x] = empty ? -INFINITY : (z - st.m) - ls;
    o.idx[r * k + threadIdx.x] = (long long)(0xffffffffu - (unsigned)mine);
  }
}

// The k largest of `n` gathered candidates, in order, by counting: list[n] -> best[k].
__device__ __forceinline__ void order_list(const u64* list, unsigned n, int k, u64* best) {
  for (unsigned i = threadIdx.x; i < n; i += NT) {
    const u64 me = list[i];
    int rank = 0;
    for (unsigned j = 0; j < n; ++j) rank += list[j] > me ? 1 : 0;
    if (rank < k) best[rank] = me;
  }
}

// ---- one part of one row.  NCH pieces a thread are in registers at a time; without TOP a part may be longer and is taken in turns.
// `groups`: a power of two >= k, disjoint sets of threads.
template <typename T, int NCH, bool TOP, bool STREAM>
__global__ __launch_bounds__(NT, 4) void logprob_kernel(const T* __restrict__ z, const long long* __restrict__ tokens, int V, int parts, int per,
                                                        int k, int groups, Stat* __restrict__ pstat, u64* __restrict__ ptop, const Outs o) {
  __shared__ Stat red[4];
  const int tid = threadIdx.x;
  const long long r = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x - (unsigned)r * (unsigned)parts);
  const T* const row = z + r * V;
  const Split sp = split_row(row, V);
  const T* const body = row + sp.first;
  const int c0 = part * per, c1 = min(sp.pieces, c0 + per);
  const int je = part == 0 ? edge_element(sp, tid) : -1;
  const float ze = je >= 0 ? Io<T>::one(row + je) : -INFINITY;
  Stat st{-FLT_MAX, 0.f, 0.f};
  typename Io<T>::Raw raw[NCH];
  float tm = ze == ze ? ze : -INFINITY;                                  // this thread's largest
  int mine = c0 + tid;                                                   // its pieces: mine + u * NT
  for (;; mine += NCH * NT) {
#pragma unroll
    for (int u = 0; u < NCH; ++u) {
      raw[u] = nothing<T>();
      const T* const at = body + (long long)(mine + u * NT) * 8;
      if (mine + u * NT < c1) raw[u] = STREAM ? Io<T>::stream(at) : Io<T>::load(at);
    }
    // the maximum first, then the sums about it: one rescaling.  (Pinned before every pass: else the compiler keeps what one pass
    // unpacked for the next, four times the registers.)
#pragma unroll
    for (int u = 0; u < NCH; ++u) {
      float f[8];
      Io<T>::pin(raw[u]);
      Io<T>::unpack(raw[u], f);
      tm = fmaxf(tm, max8(f));
    }
    if (tm > st.m) stat_rescale(st, tm);
    if (fabsf(st.m) < 1048576.f) {
      Base2 b;
      b.begin(st.m);
#pragma unroll
      for (int u = 0; u < NCH; ++u) {
        float f[8];
        Io<T>::pin(raw[u]);
        Io<T>::unpack(raw[u], f);
        b.add8(f);
      }
      b.into(st);
    } else {
#pragma unroll
      for (int u = 0; u < NCH; ++u) {
        float f[8];
        Io<T>::pin(raw[u]);
        Io<T>::unpack(raw[u], f);
        stat_add8(st, f);
      }
    }
    if (TOP || mine - tid + NCH * NT >= c1) break;
  }
  if (je >= 0) stat_add1(st, ze);
  if (!TOP) {
    st = stat_wave(st);
    if ((tid & 63) == 0) red[tid >> 6] = st;
    __syncthreads();
    st = stat_join(stat_join(red[0], red[1]), stat_join(red[2], red[3]));
    if (parts == 1) finish_row(st, row, tokens[r], V, r, 0, 0ull, o);
    else if (tid == 0) pstat[r * parts + part] = st;
    return;
  }
  __shared__ u64 ured[4];
  __shared__ float gmax[4][64];
  __shared__ u64 list[CAP];
  __shared__ u64 best[TOP_MAX];
  __shared__ unsigned count;
  // a bound that at least k elements reach: the smallest of `groups` maxima over disjoint sets
  float gm = tm;
  for (int off = 32; off >= groups; off >>= 1) gm = fmaxf(gm, __shfl_xor(gm, off, 64));
  gmax[tid >> 6][tid & 63] = gm;
  st = stat_wave(st);
  if ((tid & 63) == 0) red[tid >> 6] = st;
  if (tid == 0) count = 0u;
  if (tid < TOP_MAX) best[tid] = 0ull;
  __syncthreads();
  st = stat_join(stat_join(red[0], red[1]), stat_join(red[2], red[3]));
  float bound = fmaxf(fmaxf(gmax[0][tid & 63], gmax[1][tid & 63]), fmaxf(gmax[2][tid & 63], gmax[3][tid & 63]));
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) bound = fminf(bound, __shfl_xor(bound, off, 64));
  const bool odd = !(st.s < INFINITY);                                   // a NaN or inf somewhere: no piece may be skipped
#pragma unroll
  for (int u = 0; u < NCH; ++u) {
    float f[8];
    Io<T>::pin(raw[u]);
    Io<T>::unpack(raw[u], f);
    if ((max8(f) >= bound || odd) && mine + u * NT < c1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!(f[e] < bound)) {                                           // a NaN counts as the largest
          const unsigned at = atomicAdd(&count, 1u);
          if (at < CAP) list[at] = cand(key_of(f[e]), sp.first + (mine + u * NT) * 8 + e);
        }
      }
    }
  }
  if (je >= 0 && !(ze < bound)) {
    const unsigned at = atomicAdd(&count, 1u);
    if (at < CAP) list[at] = cand(key_of(ze), je);
  }
  __syncthreads();
  const unsigned n = count;
  if (n <= CAP) {
    order_list(list, n, k, best);
  } else {                                                               // many elements tie with the bound
    u64 prev = ~0ull;
    for (int t = 0; t < k; ++t) {
      u64 mx = je >= 0 ? cand(key_of(ze), je) : 0ull;
      mx = mx < prev ? mx : 0ull;
      for (int c = mine; c < c1; c += NT) {                              // read again: rare, and 64-bit keys of registers would spill
        float f[8];
        Io<T>::unpack(Io<T>::load(body + (long long)c * 8), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const u64 v = cand(key_of(f[e]), sp.first + c * 8 + e);
          mx = v < prev && v > mx ? v : mx;
        }
      }
      prev = block_max(mx, ured);
      if (tid == 0) best[t] = prev;
    }
  }
  __syncthreads();
  if (parts == 1) {
    finish_row(st, row, tokens[r], V, r, k, tid < k ? best[tid] : 0ull, o);
  } else {
    if (tid == 0) pstat[r * parts + part] = st;
    if (tid < k) ptop[(r * parts + part) * k + tid] = best[tid];
  }
}

// ---- joins the parts of a row: one block per row
template <typename T>
__global__ __launch_bounds__(NT) void logprob_join_kernel(const T* __restrict__ z, const long long* __restrict__ tokens, int V, int parts, int k, int groups,
                                                          const Stat* __restrict__ pstat, const u64* __restrict__ ptop, const Outs o) {
  __shared__ Stat red[4];
  const int tid = threadIdx.x;
  const long long r = blockIdx.x;
  Stat st{-FLT_MAX, 0.f, 0.f};
  for (int p = tid; p < parts; p += NT) st = stat_join(st, pstat[r * parts + p]);
  st = stat_wave(st);
  if ((tid & 63) == 0) red[tid >> 6] = st;
  __syncthreads();
  st = stat_join(stat_join(red[0], red[1]), stat_join(red[2], red[3]));
  if (k == 0) { finish_row(st, z + r * V, tokens[r], V, r, 0, 0ull, o); return; }
  // the same bound over the parts' lists (keys here: a NaN counts)
  __shared__ u64 ured[4];
  __shared__ unsigned gmax[4][64];
  __shared__ u64 list[CAP];
  __shared__ u64 best[TOP_MAX];
  __shared__ unsigned count;
  const u64* const src = ptop + r * parts * k;
  const int total = parts * k;
  unsigned mk = 0u;
  for (int i = tid; i < total; i += NT) mk = max(mk, (unsigned)(src[i] >> 32));
  for (int off = 32; off >= groups; off >>= 1) mk = max(mk, (unsigned)__shfl_xor((int)mk, off, 64));
  gmax[tid >> 6][tid & 63] = mk;
  if (tid == 0) count = 0u;
  __syncthreads();
  unsigned bound = max(max(gmax[0][tid & 63], gmax[1][tid & 63]), max(gmax[2][tid & 63], gmax[3][tid & 63]));
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) bound = min(bound, (unsigned)__shfl_xor((int)bound, off, 64));
  bound = max(bound, 1u);                                                // 0 marks what a short part left empty
  for (int i = tid; i < total; i += NT) {
    const u64 v = src[i];
    if ((unsigned)(v >> 32) >= bound) {
      const unsigned at = atomicAdd(&count, 1u);
      if (at < CAP) list[at] = v;
    }
  }
  __syncthreads();
  if (count <= CAP) {
    order_list(list, count, k, best);
  } else {
    u64 prev = ~0ull;
    for (int t = 0; t < k; ++t) {
      u64 mx = 0ull;
      for (int i = tid; i < total; i += NT) {
        const u64 v = src[i];
        mx = v < prev && v > mx ? v : mx;
      }
      prev = block_max(mx, ured);
      if (tid == 0) best[t] = prev;
    }
  }
  __syncthreads();
  const u64 mine = tid < k ? best[tid] : 0ull;
  finish_row(st, z + r * V, tokens[r], V, r, k, mine, o);
}

// ---- gradient: one part of one row
template <typename T, bool STREAM>
__global__ __launch_bounds__(NT) void logprob_bwd_kernel(const T* __restrict__ z, const long long* __restrict__ tokens,
                                                         const float* __restrict__ norm, const float* __restrict__ ent,
                                                         const float* __restrict__ glogp, const float* __restrict__ gent,
                                                         const float* __restrict__ gtop, const long long* __restrict__ idx, int k,
                                                         T* __restrict__ dz, int V, int parts, int per) {
  const unsigned bid = gridDim.x - 1 - blockIdx.x;                        // the last rows first (beyond_cache)
  const long long r = bid / (unsigned)parts;
  const int part = (int)(bid - (unsigned)r * (unsigned)parts);
  const T* const row = z + r * V;
  T* const drow = dz + r * V;
  const Split sp = split_row(row, V);
  const bool vec = (((u64)(drow + sp.first)) & 15) == 0;
  const int c0 = part * per, c1 = min(sp.pieces, c0 + per);
  const float mx = norm[2 * r], ls = norm[2 * r + 1], H = ent[r];
  const bool empty = ls == -INFINITY;
  const long long tok = tokens[r];
  const int t = tok >= 0 && tok < V ? (int)tok : -1;
  const float gl = (glogp != nullptr && t >= 0) ? glogp[r] : 0.f, gh = gent != nullptr ? gent[r] : 0.f;
  float G = gl;
  if (gtop != nullptr)
    for (int i = 0; i < k; ++i) G += gtop[r * k + i];
  auto grad = [&](float zj) {
    const float d = (zj - mx) - ls, p = __expf(d);
    return -p * (G + (p == 0.f ? 0.f : gh * (d + H)));
  };
  auto piece = [&](int c, typename Io<T>::Raw raw) {
    float f[8];
    const int j0 = sp.first + c * 8;
    Io<T>::unpack(raw, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = empty ? 0.f : grad(f[e]);
    if (!empty && t >= j0 && t < j0 + 8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += t - j0 == e ? gl : 0.f;
    }
    if (vec && STREAM) Io<T>::put_stream(drow + j0, f);
    else if (vec) Io<T>::store(drow + j0, f);
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) Io<T>::put(drow + j0 + e, f[e]);
    }
  };
  const T* const body = row + sp.first;
  auto get = [&](int c) { return STREAM ? Io<T>::stream(body + (long long)c * 8) : Io<T>::load(body + (long long)c * 8); };
  int c = c0 + (int)threadIdx.x;
  for (; c + NT < c1; c += 2 * NT) {
    const typename Io<T>::Raw r0 = get(c), r1 = get(c + NT);
    piece(c, r0);
    piece(c + NT, r1);
  }
  if (c < c1) piece(c, get(c));
  const int je = part == 0 ? edge_element(sp, threadIdx.x) : -1;
  if (je >= 0) Io<T>::put(drow + je, empty ? 0.f : grad(Io<T>::one(row + je)) + (je == t ? gl : 0.f));
  if (gtop == nullptr || empty) return;
  __syncthreads();                                                        // this block's dense values are written: replace the listed ones
  for (int i = threadIdx.x; i < k; i += NT) {
    const int j = (int)idx[r * k + i], body_j = j - sp.first, pc = body_j >> 3;
    if ((body_j >= 0 && pc < sp.pieces) ? (pc >= c0 && pc < c1) : part == 0) {
      float v = grad(Io<T>::one(row + j)) + gtop[r * k + i];
      if (j == t) v += gl;
      Io<T>::put(drow + j, v);
    }
  }
}

// Pieces (of 8 elements) per part.  A block streams a whole row when there are rows enough for two blocks on each of the 256 CUs; fewer
// rows are cut so that about 512 blocks run, down to one piece a thread.
int plan(long long rows, int V, int most) {
  const int pieces = V / 8;
  long long parts = (512 + rows - 1) / rows;
  if (parts < 1) parts = 1;
  long long per = (pieces + parts - 1) / parts;
  per = (per + NT - 1) / NT * NT;
  if (per < NT) per = NT;
  if (per > most) per = most;
  return (int)per;
}

// Rows begin at any alignment: a row has V / 8 pieces at most (fewer behind an unaligned start).
int parts_of(int V, int per) { const int pieces = V / 8; return pieces == 0 ? 1 : (pieces + per - 1) / per; }

// Rows of one launch, which has less than 2^32 threads: more rows take several.
long long rows_of_launch(long long parts) { const long long n = 0xffffffffll / NT / parts; return n > 0 ? n : 1; }

// Most pieces a thread keeps in registers: 64 registers of logits, of the 128 that four waves per SIMD have.
template <typename T> struct MaxPieces { static constexpr int value = sizeof(T) == 2 ? 16 : 8; };

template <typename T, int NCH, bool STREAM>
void launch(dim3 grid, hipStream_t st, const T* z, const long long* tokens, int V, int parts, int per, int k, int groups,
            Stat* ps, u64* pt, const Outs& o) {
  if (k > 0) hipLaunchKernelGGL(HIP_KERNEL_NAME(logprob_kernel<T, NCH, true, STREAM>), grid, dim3(NT), 0, st, z, tokens, V, parts, per, k, groups, ps, pt, o);
  else hipLaunchKernelGGL(HIP_KERNEL_NAME(logprob_kernel<T, NCH, false, STREAM>), grid, dim3(NT), 0, st, z, tokens, V, parts, per, k, groups, ps, pt, o);
}

template <typename T, bool STREAM>
int forward(const T* z, const long long* tokens, long long rows, int V, int k, int per, int parts, void* ws, const Outs& o, hipStream_t st) {
  Stat* ps = (Stat*)ws;
  u64* pt = (u64*)((char*)ws + ((size_t)rows * parts * sizeof(Stat) + 15) / 16 * 16);
  int groups = 1;
  while (groups < k) groups *= 2;
  const long long most = rows_of_launch(parts);
  int rc = 0;
  for (long long r = 0; r < rows && rc == 0; r += most) {
    const long long n = min(most, rows - r);
    const dim3 grid((unsigned)(n * parts));
    const Outs p{o.logp + r, o.ent + r, o.norm == nullptr ? nullptr : o.norm + 2 * r, o.top + r * k, o.idx + r * k};
    if (per <= NT) launch<T, 1, STREAM>(grid, st, z, tokens, V, parts, per, k, groups, ps, pt, p);
    else if (per <= 4 * NT) launch<T, 4, STREAM>(grid, st, z, tokens, V, parts, per, k, groups, ps, pt, p);
    else launch<T, MaxPieces<T>::value, STREAM>(grid, st, z, tokens, V, parts, per, k, groups, ps, pt, p);
    if (parts > 1)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(logprob_join_kernel<T>), dim3((unsigned)n), dim3(NT), 0, st, z, tokens, V, parts, k, groups, ps, pt, p);
    rc = (int)hipGetLastError();
    z += n * V; tokens += n; ps += n * parts; pt += n * parts * k;
  }
  return rc;
}

int parts_for(long long rows, int V, int is_bf16, int k, int* per) {
  *per = plan(rows, V, k > 0 ? NT * (is_bf16 ? MaxPieces<bf16_t>::value : MaxPieces<float>::value) : 0x7fffff00);
  return parts_of(V, *per);
}

// Logits that the memory-side cache (256 MiB) does not hold.  Read once (no gradient asked) they are loaded past the caches: 8192 x 32000 bf16
// 94 us against 116.  In training the end of the forward pass stays in that cache and the backward pass, which streams, starts there, with
// the last rows: 183 us against 205 (streamed forward, first rows first).
bool beyond_cache(long long rows, int V, int is_bf16) { return rows * V * (is_bf16 ? 2 : 4) > (256ll << 20); }

}  // namespace

// bytes of workspace of a forward call
extern "C" long long ddl_logprob_workspace(long long rows, int V, int is_bf16, int k) {
  if (rows <= 0 || V <= 0 || k < 0 || k > TOP_MAX) return -1;
  int per;
  const long long parts = parts_for(rows, V, is_bf16, k, &per);
  if (parts <= 1) return 0;
  return (rows * parts * (long long)sizeof(Stat) + 15) / 16 * 16 + rows * parts * k * 8;
}

// ws: null where ddl_logprob_workspace is 0;  train: norm is wanted, a backward call follows
extern "C" int ddl_logprob_fwd(const void* z, int is_bf16, const long long* tokens, long long rows, int V, int k, int train, void* ws, float* logp,
                               float* ent, float* norm, float* top, long long* idx, void* stream) {
  if (rows <= 0 || V <= 0 || V > 0x7fffff00 || k < 0 || k > TOP_MAX || k > V) return -1;
  int per;
  const int parts = parts_for(rows, V, is_bf16, k, &per);
  const Outs o{logp, ent, norm, top, idx};
  hipStream_t st = (hipStream_t)stream;
  if (!train && beyond_cache(rows, V, is_bf16))
    return is_bf16 ? forward<bf16_t, true>((const bf16_t*)z, tokens, rows, V, k, per, parts, ws, o, st)
                   : forward<float, true>((const float*)z, tokens, rows, V, k, per, parts, ws, o, st);
  return is_bf16 ? forward<bf16_t, false>((const bf16_t*)z, tokens, rows, V, k, per, parts, ws, o, st)
                 : forward<float, false>((const float*)z, tokens, rows, V, k, per, parts, ws, o, st);
}

// glogp, gent [rows], gtop [rows][k] (null: no gradient through that output); idx as the forward call left it
extern "C" int ddl_logprob_bwd(const void* z, int is_bf16, const long long* tokens, const float* norm, const float* ent, const float* glogp,
                               const float* gent, const float* gtop, const long long* idx, long long rows, int V, int k, void* dz, void* stream) {
  if (rows <= 0 || V <= 0 || V > 0x7fffff00 || k < 0 || k > TOP_MAX || (gtop != nullptr && idx == nullptr)) return -1;
  const int per = plan(rows, V, 0x7fffff00), parts = parts_of(V, per);
  hipStream_t st = (hipStream_t)stream;
  const long long most = rows_of_launch(parts);
  int rc = 0;
  auto run = [&](auto* kernel, auto* in, auto* out) {
    auto at = [](auto* p, long long i) { return p == nullptr ? p : p + i; };
    for (long long r = (rows - 1) / most * most; r >= 0 && rc == 0; r -= most) {           // the last rows first (beyond_cache)
      hipLaunchKernelGGL(kernel, dim3((unsigned)(min(most, rows - r) * parts)), dim3(NT), 0, st, in + r * V, tokens + r, norm + 2 * r, ent + r,
                         at(glogp, r), at(gent, r), at(gtop, r * k), at(idx, r * k), k, out + r * V, V, parts, per);
      rc = (int)hipGetLastError();
    }
  };
  const bool large = beyond_cache(rows, V, is_bf16);
  if (is_bf16) run(large ? &logprob_bwd_kernel<bf16_t, true> : &logprob_bwd_kernel<bf16_t, false>, (const bf16_t*)z, (bf16_t*)dz);
  else run(large ? &logprob_bwd_kernel<float, true> : &logprob_bwd_kernel<float, false>, (const float*)z, (float*)dz);
  return rc;
}
