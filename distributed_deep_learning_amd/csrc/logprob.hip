// Log probabilities of given tokens, entropy and the most likely tokens of every row of logits, and their gradient (gfx950).
//
//   lse = log sum_j exp z_j      logp = z_t - lse      H = lse - sum_j p_j z_j      top: the k largest z_j - lse
//
// One pass over the logits: every thread carries the running maximum m, s = sum e^(z - m) and q = sum e^(z - m) (z - m) of what it
// has seen (a larger maximum m' rescales: s' = f s, q' = f (q + (m - m') s), f = e^(m - m')); H = log s - q / s.  The kernel is
// bound by reading z once.  A row is cut into parts when there are too few rows to fill the chip, and a second launch joins
// (m, s, q) and the candidate lists of the parts.
//
// Top k in the same pass: the part's logits stay in registers (packed as loaded).  The k-th largest of the 256 per-thread maxima is
// a lower bound of the part's k-th largest value that only a few elements beside the k reach; those are gathered in LDS and ordered by
// counting.  Rows where very many elements tie with the bound fall back to k rounds of a block-wide maximum.  Candidates are
// 64-bit keys, an order-preserving image of the value above the inverted index: equal values go to the lowest index.
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
  static __device__ __forceinline__ Raw pack(const float* f) { return Raw{f32x4{f[0], f[1], f[2], f[3]}, f32x4{f[4], f[5], f[6], f[7]}}; }
  static __device__ __forceinline__ void unpack(const Raw& r, float* f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[e] = r.a[e]; f[4 + e] = r.b[e]; }
  }
  static __device__ __forceinline__ void store(float* p, const float* f) {
    *reinterpret_cast<f32x4*>(p) = f32x4{f[0], f[1], f[2], f[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{f[4], f[5], f[6], f[7]};
  }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <> struct Io<bf16_t> {
  static constexpr int ALIGN = 8;
  typedef u32x4 Raw;
  static __device__ __forceinline__ float one(const bf16_t* p) { return bf16_to_f32(*p); }
  static __device__ __forceinline__ Raw load(const bf16_t* p) { return *reinterpret_cast<const u32x4*>(p); }
  static __device__ __forceinline__ Raw pack(const float* f) { return pack8(f); }     // exact: the values came from bf16
  static __device__ __forceinline__ void unpack(const Raw& r, float* f) { unpack8(r, f); }
  static __device__ __forceinline__ void store(bf16_t* p, const float* f) { *reinterpret_cast<u32x4*>(p) = pack8(f); }
  static __device__ __forceinline__ void put(bf16_t* p, float v) { *p = f32_to_bf16(v); }
};

// Pieces of 8 elements start on 16-byte boundaries whatever the row's address: piece c holds elements 8c - shift .. 8c - shift + 7.
template <typename T> __device__ __forceinline__ int shift_of(const T* row) {
  return (int)(((u64)row / sizeof(T)) & (Io<T>::ALIGN - 1));
}
__host__ __device__ inline int pieces_of(int V, int align) { return (V + align - 1 + 7) / 8; }      // for any shift < align

// elements outside the row read as -inf and are marked absent in `valid`
template <typename T> __device__ __forceinline__ typename Io<T>::Raw load_piece(const T* row, int j0, int V, unsigned& valid) {
  if (j0 >= 0 && j0 + 8 <= V) { valid = 0xffu; return Io<T>::load(row + j0); }
  float f[8];
  valid = 0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int j = j0 + e;
    const bool in = j >= 0 && j < V;
    f[e] = in ? Io<T>::one(row + j) : -INFINITY;
    valid |= in ? 1u << e : 0u;
  }
  return Io<T>::pack(f);
}

struct Stat { float m, s, q; };

__device__ __forceinline__ void stat_rescale(Stat& a, float m) {       // to a maximum m >= a.m
  const float d = a.m - m, f = __expf(d);
  a.q = a.s == 0.f ? 0.f : f * (a.q + fmaxf(d, -200.f) * a.s);        // f is zero long before -200
  a.s = a.s == 0.f ? 0.f : f * a.s;
  a.m = m;
}
__device__ __forceinline__ void stat_add8(Stat& a, const float* z) {
  float mx = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7])));
  if (mx > a.m) stat_rescale(a, mx);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = z[e] - a.m, p = __expf(d);
    a.s += p;                                                            // a NaN (or inf - inf) stays in s
    a.q += p * fmaxf(d, -200.f);                                         // p is zero below about -104: no 0 * inf
  }
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

__device__ __forceinline__ unsigned key_of(float z) {                    // order-preserving; -0 and 0 equal, NaN on top; 0 = absent
  const unsigned b = __float_as_uint(z + 0.f);
  if (z != z) return 0xffffffffu;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
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

// norm: (m, log s) of every row; their sum is lse, but far from zero it would swallow log s
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
    o.norm[2 * r] = st.m;
    o.norm[2 * r + 1] = empty ? -INFINITY : ls;
  }
  if ((int)threadIdx.x < k) {
    const float z = value_of((unsigned)(mine >> 32));
    o.top[r * k + threadIdx.x] = empty ? -INFINITY : (z - st.m) - ls;
    o.idx[r * k + threadIdx.x] = (long long)(0xffffffffu - (unsigned)mine);
  }
}

// ---- one part of one row, nothing but the statistics
template <typename T>
__global__ __launch_bounds__(NT) void logprob_stats_kernel(const T* __restrict__ z, const long long* __restrict__ tokens, int V, int parts,
                                                           int per, Stat* __restrict__ pstat, const Outs o) {
  __shared__ Stat red[4];
  const long long r = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x - (unsigned)r * (unsigned)parts);
  const T* const row = z + r * V;
  const int shift = shift_of(row);
  const int pieces = (V + shift + 7) / 8, c0 = part * per, c1 = min(pieces, c0 + per);
  Stat st{-FLT_MAX, 0.f, 0.f};
  int c = c0 + (int)threadIdx.x;
  for (; c + 3 * NT < c1; c += 4 * NT) {                               // four 16-byte loads in flight
    typename Io<T>::Raw raw[4];
    unsigned valid;
#pragma unroll
    for (int u = 0; u < 4; ++u) raw[u] = load_piece(row, (c + u * NT) * 8 - shift, V, valid);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float f[8];
      Io<T>::unpack(raw[u], f);
      stat_add8(st, f);
    }
  }
  for (; c < c1; c += NT) {
    unsigned valid;
    float f[8];
    Io<T>::unpack(load_piece(row, c * 8 - shift, V, valid), f);
    stat_add8(st, f);
  }
  st = stat_wave(st);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = st;
  __syncthreads();
  st = stat_join(stat_join(red[0], red[1]), stat_join(red[2], red[3]));
  if (parts == 1) finish_row(st, row, tokens[r], V, r, 0, 0ull, o);
  else if (threadIdx.x == 0) pstat[r * parts + part] = st;
}

// ---- the same with the k largest; at most NCH pieces a thread
template <typename T, int NCH>
__global__ __launch_bounds__(NT) void logprob_top_kernel(const T* __restrict__ z, const long long* __restrict__ tokens, int V, int parts,
                                                         int per, int k, Stat* __restrict__ pstat, u64* __restrict__ ptop, const Outs o) {
  __shared__ Stat red[4];
  __shared__ u64 ured[4];
  __shared__ u64 tmax[NT];
  __shared__ u64 list[CAP];
  __shared__ u64 best[TOP_MAX];
  __shared__ unsigned bound, count;
  const int tid = threadIdx.x;
  const long long r = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x - (unsigned)r * (unsigned)parts);
  const T* const row = z + r * V;
  const int shift = shift_of(row);
  const int pieces = (V + shift + 7) / 8, c0 = part * per, c1 = min(pieces, c0 + per);
  Stat st{-FLT_MAX, 0.f, 0.f};
  typename Io<T>::Raw raw[NCH];
  unsigned valid[NCH];
#pragma unroll
  for (int u = 0; u < NCH; ++u) {
    const int c = c0 + tid + u * NT;
    raw[u] = load_piece(row, c < c1 ? c * 8 - shift : V, V, valid[u]);
  }
  unsigned mk = 0u;                                                      // largest key of this thread
#pragma unroll
  for (int u = 0; u < NCH; ++u) {
    float f[8];
    Io<T>::unpack(raw[u], f);
    if (valid[u] != 0u) stat_add8(st, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned key = (valid[u] >> e) & 1u ? key_of(f[e]) : 0u;
      mk = key > mk ? key : mk;
    }
  }
  st = stat_wave(st);
  if ((tid & 63) == 0) red[tid >> 6] = st;
  tmax[tid] = ((u64)mk << 32) | (u64)(NT - 1 - tid);
  if (tid == 0) count = 0u;
  if (tid < TOP_MAX) best[tid] = 0ull;
  __syncthreads();
  st = stat_join(stat_join(red[0], red[1]), stat_join(red[2], red[3]));
  {
    const u64 me = tmax[tid];
    int rank = 0;
    for (int i = 0; i < NT; ++i) rank += tmax[i] > me ? 1 : 0;
    if (rank == k - 1) bound = mk;
  }
  __syncthreads();
  const unsigned lim = bound > 0u ? bound : 1u;
#pragma unroll
  for (int u = 0; u < NCH; ++u) {
    float f[8];
    Io<T>::unpack(raw[u], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned key = (valid[u] >> e) & 1u ? key_of(f[e]) : 0u;
      if (key >= lim) {
        const unsigned at = atomicAdd(&count, 1u);
        if (at < CAP) list[at] = cand(key, (c0 + tid + u * NT) * 8 - shift + e);
      }
    }
  }
  __syncthreads();
  const unsigned n = count;
  if (n <= CAP) {
    for (unsigned i = tid; i < n; i += NT) {
      const u64 me = list[i];
      int rank = 0;
      for (unsigned j = 0; j < n; ++j) rank += list[j] > me ? 1 : 0;
      if (rank < k) best[rank] = me;
    }
  } else {                                                               // many elements tie with the bound
    u64 prev = ~0ull;
    for (int t = 0; t < k; ++t) {
      u64 mx = 0ull;
#pragma unroll
      for (int u = 0; u < NCH; ++u) {
        float f[8];
        Io<T>::unpack(raw[u], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if ((valid[u] >> e) & 1u) {
            const u64 v = cand(key_of(f[e]), (c0 + tid + u * NT) * 8 - shift + e);
            mx = v < prev && v > mx ? v : mx;
          }
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
__global__ __launch_bounds__(NT) void logprob_join_kernel(const T* __restrict__ z, const long long* __restrict__ tokens, int V, int parts, int k,
                                                          const Stat* __restrict__ pstat, const u64* __restrict__ ptop, const Outs o) {
  __shared__ Stat red[4];
  __shared__ u64 ured[4];
  const int tid = threadIdx.x;
  const long long r = blockIdx.x;
  Stat st{-FLT_MAX, 0.f, 0.f};
  for (int p = tid; p < parts; p += NT) st = stat_join(st, pstat[r * parts + p]);
  st = stat_wave(st);
  if ((tid & 63) == 0) red[tid >> 6] = st;
  __syncthreads();
  st = stat_join(stat_join(red[0], red[1]), stat_join(red[2], red[3]));
  u64 prev = ~0ull, mine = 0ull;
  for (int t = 0; t < k; ++t) {
    u64 mx = 0ull;
    for (int i = tid; i < parts * k; i += NT) {
      const u64 v = ptop[r * parts * k + i];
      mx = v < prev && v > mx ? v : mx;
    }
    prev = block_max(mx, ured);
    if (tid == t) mine = prev;
  }
  finish_row(st, z + r * V, tokens[r], V, r, k, mine, o);
}

// ---- gradient: one part of one row
template <typename T>
__global__ __launch_bounds__(NT) void logprob_bwd_kernel(const T* __restrict__ z, const long long* __restrict__ tokens,
                                                         const float* __restrict__ norm, const float* __restrict__ ent,
                                                         const float* __restrict__ glogp, const float* __restrict__ gent,
                                                         const float* __restrict__ gtop, const long long* __restrict__ idx, int k,
                                                         T* __restrict__ dz, int V, int parts, int per) {
  const long long r = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x - (unsigned)r * (unsigned)parts);
  const T* const row = z + r * V;
  T* const drow = dz + r * V;
  const int shift = shift_of(row);
  const bool vec = shift_of(drow) == shift;
  const int pieces = (V + shift + 7) / 8, c0 = part * per, c1 = min(pieces, c0 + per);
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
  for (int c = c0 + (int)threadIdx.x; c < c1; c += NT) {
    unsigned valid;
    float f[8];
    const int j0 = c * 8 - shift;
    Io<T>::unpack(load_piece(row, j0, V, valid), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = empty ? 0.f : grad(f[e]);
    if (!empty && (unsigned)(t - j0) < 8u && t >= 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += t - j0 == e ? gl : 0.f;
    }
    if (valid == 0xffu && vec) Io<T>::store(drow + j0, f);
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) if ((valid >> e) & 1u) Io<T>::put(drow + j0 + e, f[e]);
    }
  }
  if (gtop == nullptr || empty) return;
  __syncthreads();                                                        // this block's dense values are written: replace the listed ones
  for (int i = threadIdx.x; i < k; i += NT) {
    const int j = (int)idx[r * k + i], c = (j + shift) / 8;
    if (c >= c0 && c < c1) {
      float v = grad(Io<T>::one(row + j)) + gtop[r * k + i];
      if (j == t) v += gl;
      Io<T>::put(drow + j, v);
    }
  }
}

// Pieces (of 8 elements) per part.  A block streams a whole row when there are rows enough for two blocks on each of the 256 CUs; fewer
// rows are cut so that about 512 blocks run, down to one piece a thread.
int plan(long long rows, int V, int align, int most) {
  const int pieces = pieces_of(V, align);
  long long parts = (512 + rows - 1) / rows;
  if (parts < 1) parts = 1;
  long long per = (pieces + parts - 1) / parts;
  per = (per + NT - 1) / NT * NT;
  if (per > most) per = most;
  return (int)per;
}

template <typename T, int NCH>
void launch_top(dim3 grid, hipStream_t st, const T* z, const long long* tokens, int V, int parts, int per, int k, Stat* ps, u64* pt, const Outs& o) {
  hipLaunchKernelGGL(HIP_KERNEL_NAME(logprob_top_kernel<T, NCH>), grid, dim3(NT), 0, st, z, tokens, V, parts, per, k, ps, pt, o);
}

template <typename T>
int forward(const T* z, const long long* tokens, long long rows, int V, int k, int per, int parts, void* ws, const Outs& o, hipStream_t st) {
  Stat* const ps = (Stat*)ws;
  u64* const pt = (u64*)((char*)ws + ((size_t)rows * parts * sizeof(Stat) + 15) / 16 * 16);
  const dim3 grid((unsigned)(rows * parts));
  if (k == 0) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(logprob_stats_kernel<T>), grid, dim3(NT), 0, st, z, tokens, V, parts, per, ps, o);
  } else {
    const int nch = (per + NT - 1) / NT;
    if (nch <= 1) launch_top<T, 1>(grid, st, z, tokens, V, parts, per, k, ps, pt, o);
    else if (nch <= 4) launch_top<T, 4>(grid, st, z, tokens, V, parts, per, k, ps, pt, o);
    else launch_top<T, 16>(grid, st, z, tokens, V, parts, per, k, ps, pt, o);
  }
  if (parts > 1)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(logprob_join_kernel<T>), dim3((unsigned)rows), dim3(NT), 0, st, z, tokens, V, parts, k, ps, pt, o);
  return (int)hipGetLastError();
}

constexpr int TOP_PIECES = 16 * NT;               // most pieces of a part that keeps its logits in registers

int parts_for(long long rows, int V, int is_bf16, int k, int* per) {
  const int align = is_bf16 ? 8 : 4;
  *per = plan(rows, V, align, k > 0 ? TOP_PIECES : 0x7fffff00);
  return (pieces_of(V, align) + *per - 1) / *per;
}

}  // namespace

extern "C" int ddl_logprob_top_max() { return TOP_MAX; }

// bytes of workspace of a forward call
extern "C" long long ddl_logprob_workspace(long long rows, int V, int is_bf16, int k) {
  if (rows <= 0 || V <= 0 || k < 0 || k > TOP_MAX) return -1;
  int per;
  const long long parts = parts_for(rows, V, is_bf16, k, &per);
  if (parts <= 1) return 16;
  return (rows * parts * (long long)sizeof(Stat) + 15) / 16 * 16 + rows * parts * k * 8;
}

extern "C" int ddl_logprob_fwd(const void* z, int is_bf16, const long long* tokens, long long rows, int V, int k, void* ws, float* logp, float* ent,
                               float* norm, float* top, long long* idx, void* stream) {
  if (rows <= 0 || V <= 0 || V > 0x7fffff00 || k < 0 || k > TOP_MAX || k > V) return -1;
  int per;
  const int parts = parts_for(rows, V, is_bf16, k, &per);
  if (rows * parts > 0x7fffffffll) return -2;
  const Outs o{logp, ent, norm, top, idx};
  return is_bf16 ? forward((const bf16_t*)z, tokens, rows, V, k, per, parts, ws, o, (hipStream_t)stream)
                 : forward((const float*)z, tokens, rows, V, k, per, parts, ws, o, (hipStream_t)stream);
}

// glogp, gent [rows], gtop [rows][k] (null: no gradient through that output); idx as the forward call left it
extern "C" int ddl_logprob_bwd(const void* z, int is_bf16, const long long* tokens, const float* norm, const float* ent, const float* glogp,
                               const float* gent, const float* gtop, const long long* idx, long long rows, int V, int k, void* dz, void* stream) {
  if (rows <= 0 || V <= 0 || V > 0x7fffff00 || k < 0 || k > TOP_MAX || (gtop != nullptr && idx == nullptr)) return -1;
  const int align = is_bf16 ? 8 : 4;
  const int per = plan(rows, V, align, 0x7fffff00), parts = (pieces_of(V, align) + per - 1) / per;
  if (rows * parts > 0x7fffffffll) return -2;
  const dim3 grid((unsigned)(rows * parts));
  hipStream_t st = (hipStream_t)stream;
  if (is_bf16)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(logprob_bwd_kernel<bf16_t>), grid, dim3(NT), 0, st, (const bf16_t*)z, tokens, norm, ent, glogp, gent, gtop,
                       idx, k, (bf16_t*)dz, V, parts, per);
  else
    hipLaunchKernelGGL(HIP_KERNEL_NAME(logprob_bwd_kernel<float>), grid, dim3(NT), 0, st, (const float*)z, tokens, norm, ent, glogp, gent, gtop, idx, k,
                       (float*)dz, V, parts, per);
  return (int)hipGetLastError();
}
