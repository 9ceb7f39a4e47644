// Log probabilities of given tokens, with the entropy of each row's
// distribution and its most likely alternatives, and the gradient of the
// first two.  For a row z of V logits with m = max z, e_j = exp(z_j - m):
//   lse = m + log sum e       lp = z_t - lse      H = log sum e - sum e_j (z_j - m) / sum e
//   dz_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H)
// Sums are kept in fp32.  The elements at the maximum count one each: they
// are counted apart from the others, so that log sum e = log1p(..) keeps its
// digits where one token has nearly all of the probability.
// A row of -inf only has no distribution: lse and lp are -inf, H 0, and its
// gradient is 0.
//
// Both directions are bound by the read (and write) of the logits: one pass,
// each thread with a running maximum that moves its sums, 16 elements a step
// as 16-byte loads whose next ones are in flight.  Few rows are split over
// blocks, whose states a second launch merges.  Measured: 2047 x 50257 fp32
// with 20 alternatives 85 us (4.84 TB/s), in bf16 67 us (bound by its
// instructions, an exponential and some eight others a value); 8 rows in f16
// 8 us and 6 for the merge; the gradient in bf16 86 us (4.8 TB/s, read and
// written).
#include "device.hpp"

namespace agpu {
namespace k {
using namespace dev;

namespace {

constexpr int kNT = 512, kNW = kNT / 64;  // threads and waves of a block
constexpr int kCh = 16;                   // elements of a thread's step
constexpr int kCap = 2560;                // alternatives that a block sorts at most
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;
constexpr float kLowest = -3.402823466e38f;

struct LpArgs {
  TokenLogprobs a;
  int splits;
  int64_t chunk;    // logits of a split
  float4* stats;    // [R][splits]: maximum, elements at it, sum of the others, sum of e d
  uint64_t* keys;   // [R][splits][top_k]
};

// Unsigned integers in the order of the floats, -0 as 0, NaN above all.
__device__ __forceinline__ uint32_t order_of(float z) {
  if (z != z) return 0xffffffffu;
  const uint32_t u = __float_as_uint(z + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// A logit and its index as one number: larger logits first, then lower indices.
__device__ __forceinline__ uint64_t key_of(float z, uint32_t j) {
  return ((uint64_t)order_of(z) << 32) | (0xffffffffu - j);
}
__device__ __forceinline__ uint32_t index_of(uint64_t k) { return 0xffffffffu - (uint32_t)k; }

__device__ __forceinline__ int64_t token_at(const TokenLogprobs& a, int64_t r) {
  return a.idx_dt == DType::I64 ? ((const int64_t*)a.tokens)[r] : (int64_t)((const int32_t*)a.tokens)[r];
}

// Part of a row as 16-byte vectors at 16-byte boundaries, and the few elements
// before the first and behind the last of them, one each for the first threads.
template <typename T>
struct Span {
  static constexpr int VE = 16 / (int)sizeof(T), NV = kCh / VE;
  const T* z;      // the first vector
  int head, vecs;  // elements before it; vectors
  int edge;        // index of this thread's single element, or -1
  __device__ __forceinline__ Span(const T* p, int n) {
    const int mis = (int)(((uintptr_t)p & 15) / sizeof(T));
    head = mis ? VE - mis : 0;
    head = head < n ? head : n;
    z = p + head;
    vecs = (n - head) / VE;
    const int tid = (int)threadIdx.x, tail = n - head - vecs * VE;
    edge = tid < head ? tid : tid < head + tail ? vecs * VE + tid : -1;
  }
  __device__ __forceinline__ int steps() const { return (vecs + kNT * NV - 1) / (kNT * NV); }
  // this thread's vector u of step c
  static __device__ __forceinline__ int vec(int c, int u) { return (c * NV + u) * kNT + (int)threadIdx.x; }
  // index of element i of its step c
  __device__ __forceinline__ int at(int c, int i) const { return head + vec(c, i / VE) * VE + i % VE; }
  __device__ __forceinline__ void load(int c, uint4 (&raw)[NV]) const {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int v = vec(c, u);
      T e[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) e[i] = from_f<T>(-INFINITY);
      __builtin_memcpy(&raw[u], e, 16);
      if (v < vecs) raw[u] = *(const uint4*)(z + (int64_t)v * VE);
    }
  }
  static __device__ __forceinline__ void floats(const uint4 (&raw)[NV], float (&f)[kCh]) {
    T e[kCh];
    __builtin_memcpy(e, raw, sizeof(e));
#pragma unroll
    for (int i = 0; i < kCh; ++i) f[i] = to_f(e[i]);
  }
};

struct Stats {
  float m, ones, rest, dot;  // maximum; number of elements at it; sums over the others, dot in log2 units
};

// One more part of the row.
__device__ __forceinline__ void add_stats(Stats& s, const Stats& o) {
  const float M = fmaxf(s.m, o.m);
  const float d1 = s.m == M ? 0.f : fmaxf((s.m - M) * kLog2e, -200.f), d2 = o.m == M ? 0.f : fmaxf((o.m - M) * kLog2e, -200.f);
  const float f1 = __builtin_amdgcn_exp2f(d1), f2 = __builtin_amdgcn_exp2f(d2);
  const float l1 = s.ones + s.rest, l2 = o.ones + o.rest;
  s.dot = f1 * (s.dot + l1 * d1) + f2 * (o.dot + l2 * d2);
  s.rest = (d1 == 0.f ? s.rest : f1 * l1) + (d2 == 0.f ? o.rest : f2 * l2);
  s.ones = (d1 == 0.f ? s.ones : 0.f) + (d2 == 0.f ? o.ones : 0.f);
  s.m = M;
}

__device__ __forceinline__ Stats wave_stats(Stats s) {
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) {
    const Stats o{__shfl_xor(s.m, x, 64), __shfl_xor(s.ones, x, 64), __shfl_xor(s.rest, x, 64), __shfl_xor(s.dot, x, 64)};
    add_stats(s, o);
  }
  return s;
}

// The outputs of row r from the whole row's statistics; returns what is
// taken from a logit for its log probability.
__device__ __forceinline__ void finish_row(const TokenLogprobs& a, int64_t r, float z_t, int64_t t, const Stats& s,
                                           float* m_out, float* logl_out) {
  const bool none = s.ones + s.rest == 0.f;  // every logit is -inf
  const float m = none ? -INFINITY : s.m;
  const float logl = none ? 0.f : log1pf((s.ones - 1.f) + s.rest);
  if (threadIdx.x == 0) {
    a.lp[r] = t < 0 || t >= a.V ? 0.f : none ? m : (z_t - m) - logl;
    a.entropy[r] = none ? 0.f : logl - s.dot * kLn2 / (s.ones + s.rest);
    a.lse[r] = m + logl;
  }
  *m_out = m;
  *logl_out = logl;
}

__device__ __forceinline__ float logp_of(float z, float m, float logl) { return m == -INFINITY ? m : (z - m) - logl; }

// The logit of a key.
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return o == 0xffffffffu ? NAN : __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o);
}

// log p of a key's element: z - lse in the form that lp has.
__device__ __forceinline__ float logp_of(uint64_t key, float m, float logl) {
  return m == -INFINITY ? m : (value_of(key) - m) - logl;
}

constexpr int kSlots = 8;  // maxima of a thread's steps that are kept, step c in slot c % kSlots

struct TopShared {
  uint64_t list[kCap];
  float top[kSlots][kNT];
  uint64_t group[kNW][64], red[kNW], floor;
  int rank[64];
  int count;
};

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int x) {
  return ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), x, 64) << 32) | (uint32_t)__shfl_xor((int)(uint32_t)v, x, 64);
}

// The n keys in list, sorted: those of rank < k go to put(rank, key).
template <typename F>
__device__ __forceinline__ void rank_keys(const uint64_t* list, int n, int k, F&& put) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const uint64_t me = list[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += list[j] > me ? 1 : 0;
    if (rank < k) put(rank, me);
  }
}

// f(key) for each element of this thread's step c that is not below `least`.
template <typename T, typename F>
__device__ __forceinline__ void keys_of_step(const Span<T>& sp, uint32_t j0, int c, float least, F&& f) {
  uint4 raw[Span<T>::NV];
  float x[kCh];
  sp.load(c, raw);
  Span<T>::floats(raw, x);
  float top = x[0];
#pragma unroll
  for (int i = 1; i < kCh; ++i) top = fmaxf(top, x[i]);
  if (top < least) return;
#pragma unroll
  for (int i = 0; i < kCh; ++i) {
    if (!(x[i] < least) && sp.vec(c, i / Span<T>::VE) < sp.vecs) f(key_of(x[i], (uint32_t)sp.at(c, i) + j0));
  }
}

// In sh.floor the k-th largest of the keys that 64 groups of threads have, a
// group being the threads of one lane of each wave (mine: the largest of this
// thread); ends with a barrier.
__device__ __forceinline__ void group_floor(TopShared& sh, uint64_t mine, int k) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  sh.group[wave][lane] = mine;
  if (tid < 64) sh.rank[tid] = 0;
  if (tid == 0) sh.count = 0;
  __syncthreads();
  uint64_t v = sh.group[0][lane];
#pragma unroll
  for (int w = 1; w < kNW; ++w) v = sh.group[w][lane] > v ? sh.group[w][lane] : v;
  int rank = 0;   // this wave's share of the groups
#pragma unroll
  for (int i = 0; i < 64 / kNW; ++i) {
    const int at = wave * (64 / kNW) + i;
    const uint64_t o = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), at) << 32) |
                       (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, at);
    rank += o > v || (o == v && at < lane) ? 1 : 0;
  }
  if (rank) atomicAdd(&sh.rank[lane], rank);
  __syncthreads();
  if (wave == 0 && sh.rank[lane] == k - 1) sh.floor = v;
  __syncthreads();
}

// The k largest keys of the span (indices from j0) in order, by put(rank,
// key).  edge: the thread's single element; best: its largest (the maxima of
// its steps are in sh.top); plain: no NaN or +inf among the elements.
//
// A lower bound of the k-th largest is the k-th largest of the maxima of 64
// groups of threads.  Only the steps whose own maximum reaches it are looked
// at again, and what reaches it, little more than k elements of an ordinary
// row, is sorted by counting.  Rows in which more than kCap elements do are
// those with many equal to the bound: they are bounded once more, with the
// index as part of the order.  Where that leaves too many as well (the
// largest of a row gathered in a few threads' elements), and in rows that are
// not plain, one maximum after another is searched.
template <typename T, typename F>
__device__ __forceinline__ void top_keys(const Span<T>& sp, uint32_t j0, int k, float edge, float best, bool plain,
                                         TopShared& sh, F&& put) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int steps = sp.steps();
  bool one_by_one = !plain;
  const uint64_t edge_key = sp.edge >= 0 ? key_of(edge, (uint32_t)sp.edge + j0) : 0;
  auto add = [&](uint64_t key) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < kCap) sh.list[at] = key;
  };
  if (plain) {
    group_floor(sh, key_of(best, 0xffffffffu), k);
    const float least = value_of(sh.floor);
    if (best >= least) {
      if (edge_key && edge >= least) add(edge_key);
      for (int c = 0; c < steps; ++c)
        if (sh.top[c % kSlots][tid] >= least) keys_of_step(sp, j0, c, least, add);
    }
    __syncthreads();
    int n = sh.count;
    if (n > kCap) {
      uint64_t mine = edge_key;
      for (int c = 0; c < steps; ++c)
        keys_of_step(sp, j0, c, best, [&](uint64_t key) { mine = key > mine ? key : mine; });
      __syncthreads();
      group_floor(sh, mine, k);
      const uint64_t floor = sh.floor;
      if (mine >= floor) {
        if (edge_key && edge_key >= floor) add(edge_key);
        for (int c = 0; c < steps; ++c)
          keys_of_step(sp, j0, c, floor ? value_of(floor) : -INFINITY, [&](uint64_t key) {
            if (key >= floor) add(key);
          });
      }
      __syncthreads();
      n = sh.count;
    }
    if (n <= kCap) {
      rank_keys(sh.list, n, k, put);
      for (int i = n + tid; i < k; i += kNT) put(i, 0);  // a span of fewer than k elements
    } else {
      one_by_one = true;
    }
  }
  if (one_by_one) {
    uint64_t last = ~0ull;
    for (int i = 0; i < k; ++i) {
      uint64_t next = edge_key < last ? edge_key : 0;
      if (last)
        for (int c = 0; c < steps; ++c)
          keys_of_step(sp, j0, c, -INFINITY, [&](uint64_t key) {
            if (key < last && key > next) next = key;
          });
#pragma unroll
      for (int x = 32; x >= 1; x >>= 1) {
        const uint64_t o = shfl64(next, x);
        next = o > next ? o : next;
      }
      __syncthreads();
      if (lane == 0) sh.red[wave] = next;
      __syncthreads();
      last = sh.red[0];
      for (int x = 1; x < kNW; ++x) last = sh.red[x] > last ? sh.red[x] : last;
      if (tid == 0) put(i, last);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kNT, 4) token_logprobs_kernel(LpArgs g) {
  const TokenLogprobs& a = g.a;
  __shared__ TopShared sh;
  __shared__ Stats wave_s[kNW];
  const int tid = threadIdx.x;
  const int split = (int)(blockIdx.x % (unsigned)g.splits);
  const int64_t r = blockIdx.x / (unsigned)g.splits, j0 = split * g.chunk;
  const int64_t n = j0 + g.chunk < a.V ? g.chunk : a.V - j0;
  const T* z = (const T*)a.z + r * a.ld;
  const Span<T> sp(z + j0, (int)n);
  const int steps = sp.steps();

  float m = kLowest, l = 0.f, rest = 0.f, dot = 0.f;
  // (a NaN stays one; -inf gives e = 0 and 0 to the sum of e d)
  auto sum = [&](float x) __attribute__((always_inline)) {
    const float d = __builtin_elementwise_maximum((x - m) * kLog2e, -200.f);
    const float e = __builtin_amdgcn_exp2f(d);
    l += e;
    rest += __builtin_amdgcn_fractf(e);  // 0 for the elements at the maximum
    dot += e * d;
  };
  const float edge = sp.edge >= 0 ? to_f(z[j0 + sp.edge]) : -INFINITY;
  uint4 cur[Span<T>::NV], nxt[Span<T>::NV];
  sp.load(0, cur);
  if (a.top_k)
    for (int i = 0; i < kSlots; ++i) sh.top[i][tid] = -INFINITY;
  float best = edge == edge ? edge : -INFINITY;
  m = fmaxf(m, best);
  sum(edge);
  for (int c = 0; c < steps; ++c) {
    if (c + 1 < steps) sp.load(c + 1, nxt);
    float x[kCh];
    Span<T>::floats(cur, x);
    float top = x[0];
#pragma unroll
    for (int i = 1; i < kCh; ++i) top = fmaxf(top, x[i]);
    if (a.top_k) {
      float* at = &sh.top[c % kSlots][tid];
      *at = c < kSlots ? top : fmaxf(*at, top);
      best = fmaxf(best, top);
    }
    if (top > m) {
      const float d = fmaxf((m - top) * kLog2e, -200.f), f = __builtin_amdgcn_exp2f(d);
      dot = f * (dot + l * d);
      l *= f;
      rest = l;
      m = top;
    }
#pragma unroll
    for (int i = 0; i < kCh; ++i) sum(x[i]);
#pragma unroll
    for (int u = 0; u < Span<T>::NV; ++u) cur[u] = nxt[u];
  }
  Stats s = wave_stats(Stats{m, rintf(l - rest), rest, dot});
  if ((tid & 63) == 0) wave_s[tid >> 6] = s;
  __syncthreads();
  s = wave_s[0];
#pragma unroll
  for (int w = 1; w < kNW; ++w) add_stats(s, wave_s[w]);
  const bool plain = s.dot == s.dot && s.rest == s.rest;

  const int64_t at = r * g.splits + split;
  float mm = 0.f, logl = 0.f;
  if (g.splits == 1) {
    const int64_t t = token_at(a, r);
    finish_row(a, r, t >= 0 && t < a.V ? to_f(z[t]) : 0.f, t, s, &mm, &logl);
  } else if (tid == 0) {
    g.stats[at] = float4{s.m, s.ones, s.rest, s.dot};
  }
  if (a.top_k)
    top_keys(sp, (uint32_t)j0, a.top_k, edge, best, plain, sh, [&](int rank, uint64_t key) {
      const int64_t to = at * a.top_k + rank;
      if (g.splits > 1) {
        g.keys[to] = key;
      } else {
        a.top_ids[to] = (int32_t)index_of(key);
        a.top_lp[to] = logp_of(key, mm, logl);
      }
    });
}

// One block per row: its splits' statistics in order, and the largest of
// their keys.
template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_merge(LpArgs g) {
  const TokenLogprobs& a = g.a;
  __shared__ uint64_t list[64 * kTopKMax];
  const int64_t r = blockIdx.x, t = token_at(a, r);
  Stats s{kLowest, 0.f, 0.f, 0.f};
  for (int i = 0; i < g.splits; ++i) {
    const float4 x = g.stats[r * g.splits + i];
    add_stats(s, Stats{x.x, x.y, x.z, x.w});
  }
  const T* z = (const T*)a.z + r * a.ld;
  float mm, logl;
  finish_row(a, r, t >= 0 && t < a.V ? to_f(z[t]) : 0.f, t, s, &mm, &logl);
  if (!a.top_k) return;
  const int n = g.splits * a.top_k;
  for (int i = threadIdx.x; i < n; i += 256) list[i] = g.keys[r * n + i];
  __syncthreads();
  rank_keys(list, n, a.top_k, [&](int rank, uint64_t key) {
    if (key == 0) return;  // (a row has at least top_k elements)
    a.top_ids[r * a.top_k + rank] = (int32_t)index_of(key);
    a.top_lp[r * a.top_k + rank] = logp_of(key, mm, logl);
  });
}

constexpr float kSure = 0.75f;  // (at most one element of a row is past it)

// This thread's share (of 256) of the sum of f(z_i) over the row but for z_j,
// by 16-byte vectors at 16-byte boundaries.
template <typename T, typename F>
__device__ __forceinline__ float sum_of_others(const T* z, int V, int j, F&& f) {
  constexpr int VE = 16 / (int)sizeof(T), U = 4;
  const int tid = (int)threadIdx.x, mis = (int)(((uintptr_t)z & 15) / sizeof(T));
  const int head = mis ? (VE - mis < V ? VE - mis : V) : 0, vecs = (V - head) / VE;
  float sum = 0.f;
  if (tid < head && tid != j) sum += f(to_f(z[tid]));
  for (int i = head + vecs * VE + tid; i < V; i += 256) sum += i != j ? f(to_f(z[i])) : 0.f;
  const T* at = z + head;
  for (int v = tid; v < vecs; v += 256 * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = *(const uint4*)(at + (int64_t)(v + 256 * u < vecs ? v + 256 * u : v) * VE);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v + 256 * u >= vecs) break;
      T e[VE];
      __builtin_memcpy(e, &raw[u], 16);
#pragma unroll
      for (int i = 0; i < VE; ++i) sum += head + (v + 256 * u) * VE + i != j ? f(to_f(e[i])) : 0.f;
    }
  }
  return sum;
}

// A row to g.splits blocks, 16-byte vectors (VEC: the rows of z and dz are
// aligned alike) to threads in turn.
//
// 1 - p_t and log p + H lose their digits where one element has nearly all of
// the probability, since lse is known to half its last place only.  So the
// others' probabilities are summed, on the way where the row has one block, else
// by the block that meets an element past kSure in a second read: with T = sum
// p_i / p_j, p = 1 / (1 + T), 1 - p = T p and log p = -log1p(T).  2047 x 50257
// bf16 86 us with no such row, 102 with half, 121 with all of them; 8 rows 5.0
// and 11.4.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) token_logprobs_grad(LpArgs g, const float* __restrict__ g_lp,
                                                           const float* __restrict__ g_h, T* __restrict__ dz) {
  const TokenLogprobs& a = g.a;
  constexpr int VE = VEC ? 16 / (int)sizeof(T) : 1;
  const uint32_t gy = (uint32_t)g.splits, part_of = blockIdx.x % gy;
  const int64_t r = blockIdx.x / gy, t = token_at(a, r);
  const T* z = (const T*)a.z + r * a.ld;
  T* out = dz + r * a.V;
  const float lse = a.lse[r];
  const bool none = lse == -INFINITY;
  const float gl = t >= 0 && t < a.V ? g_lp[r] : 0.f, gh = g_h ? g_h[r] : 0.f, H = g_h ? a.entropy[r] : 0.f;
  const float c0 = gl + gh * H, c1 = gh * kLn2;
  const int mis = VEC ? (int)(((uintptr_t)z & 15) / sizeof(T)) : 0;
  const int V = (int)a.V, vecs = (V + mis + VE - 1) / VE, tid = (int)threadIdx.x;
  auto prob = [&](float x) __attribute__((always_inline)) {
    return __builtin_amdgcn_exp2f(__builtin_elementwise_maximum((x - lse) * kLog2e, -200.f));
  };
  // f(x, j) of vector v's elements in the row
  auto each = [&](int v, auto&& f) __attribute__((always_inline)) {
    const int j = v * VE - mis;
    if (VEC && j >= 0 && j + VE <= V) {
      const uint4 raw = *(const uint4*)(z + j);
      T e[VE];
      __builtin_memcpy(e, &raw, sizeof(e));
#pragma unroll
      for (int i = 0; i < VE; ++i) f(to_f(e[i]), j + i);
    } else {
      for (int i = 0; i < VE; ++i)
        if (j + i >= 0 && j + i < V) f(to_f(z[j + i]), j + i);
    }
  };
  float sum = 0.f;
  int at = -1;
  for (int v = (int)part_of * 256 + tid; v < vecs; v += (int)gy * 256) {
    float top = 0.f, part = 0.f;
    // -p (g_lp + g_H (log p + H)), + g_lp at the token
    auto grad = [&](float x, int j) __attribute__((always_inline)) {
      const float d = __builtin_elementwise_maximum((x - lse) * kLog2e, -200.f);
      const float p = __builtin_amdgcn_exp2f(d), w = -p * (c0 + c1 * d);
      top = fmaxf(top, p);
      part += p;
      return none ? 0.f : j == t ? w + gl : w;
    };
    const int j = v * VE - mis;
    if (VEC && j >= 0 && j + VE <= V) {
      const uint4 raw = *(const uint4*)(z + j);
      T e[VE];
      __builtin_memcpy(e, &raw, sizeof(e));
#pragma unroll
      for (int i = 0; i < VE; ++i) e[i] = from_f<T>(grad(to_f(e[i]), j + i));
      uint4 o;
      __builtin_memcpy(&o, e, sizeof(e));
      *(uint4*)(out + j) = o;
    } else {
      for (int i = 0; i < VE; ++i)
        if (j + i >= 0 && j + i < V) out[j + i] = from_f<T>(grad(to_f(z[j + i]), j + i));
    }
    if (top > kSure) {
      part = 0.f;
      each(v, [&](float x, int i) {
        const float p = prob(x);
        if (p > kSure) at = i;
        else part += p;
      });
    }
    sum += part;
  }

  __shared__ int sure[4];
  __shared__ float parts[4];
  const int lane = tid & 63, wave = tid >> 6;
  const uint64_t who = __ballot(at >= 0);
  if (lane == (who ? __ffsll((long long)who) - 1 : 0)) sure[wave] = at;
  __syncthreads();
  const int j = max(max(sure[0], sure[1]), max(sure[2], sure[3]));
  if (j < 0) return;
  if (gy > 1) sum = sum_of_others(z, V, j, prob);
  sum = wave_sum(sum);
  if (lane == 0) parts[wave] = sum;
  __syncthreads();  // (and the stores to dz before the last one)
  if (tid) return;
  sum = ((parts[0] + parts[1]) + (parts[2] + parts[3])) / prob(to_f(z[j]));
  const float p = 1.f / (1.f + sum);
  out[j] = from_f<T>((j == t ? gl * (sum * p) : -gl * p) - gh * p * (H - log1pf(sum)));
}

LpArgs plan(const TokenLogprobs& a) {
  LpArgs g{};
  g.a = a;
  // rows that fill the CUs take a block each; fewer are split, in equal parts
  // of at least 4096 logits
  int64_t want = a.R > 0 && a.R < 512 ? (512 + a.R - 1) / a.R : 1;
  const int64_t most = a.V / 4096 > 0 ? a.V / 4096 : 1;
  if (want > most) want = most;
  if (want > 64) want = 64;
  g.chunk = ((a.V + want - 1) / want + 63) / 64 * 64;
  g.splits = (int)((a.V + g.chunk - 1) / g.chunk);
  return g;
}

}  // namespace

size_t token_logprobs_ws_bytes(const TokenLogprobs& a) {
  const LpArgs g = plan(a);
  return g.splits <= 1 ? 0 : (size_t)a.R * g.splits * (sizeof(float4) + a.top_k * sizeof(uint64_t));
}

void token_logprobs(const TokenLogprobs& a, void* ws, hipStream_t s) {
  if (a.R == 0) return;
  LpArgs g = plan(a);
  if (a.R * g.splits > 0x7fffffffLL) fail("token_logprobs: too many rows");
  if (g.splits > 1) {
    if (!ws) fail("token_logprobs: workspace missing");
    g.stats = (float4*)ws;
    g.keys = (uint64_t*)(g.stats + a.R * g.splits);
  }
  AGPU_FLOAT_SWITCH(a.dt, {
    hipLaunchKernelGGL((token_logprobs_kernel<T>), dim3((unsigned)(a.R * g.splits)), dim3(kNT), 0, s, g);
    if (g.splits > 1) hipLaunchKernelGGL((token_logprobs_merge<T>), dim3((unsigned)a.R), dim3(256), 0, s, g);
  });
  check_launch("token_logprobs");
}

void token_logprobs_backward(const TokenLogprobs& a, const float* g_lp, const float* g_H, void* dz, hipStream_t s) {
  if (a.R == 0) return;
  if (a.R > 0x7fffffffLL) fail("token_logprobs_backward: too many rows");
  LpArgs g{};
  g.a = a;
  const int64_t es = (int64_t)dtype_size(a.dt);
  const bool vec = ((uintptr_t)a.z & 15) == ((uintptr_t)dz & 15) && (a.ld - a.V) * es % 16 == 0;
  // blocks of a row, one after another: what an element past kSure has its
  // block read again is in the caches then, and writes are in a row (2047 x
  // 50257 fp32 150 us; a part of every row first 177)
  const int64_t per = 256 * 16 / es * 2, most = a.R < (1 << 23) ? (1 << 23) / a.R : 1;
  int64_t parts = (a.V + per - 1) / per;
  if (parts > most) parts = most;
  g.splits = (int)parts;
  const dim3 grid((unsigned)(a.R * parts));
  AGPU_FLOAT_SWITCH(a.dt, {
    if (vec) hipLaunchKernelGGL((token_logprobs_grad<T, true>), grid, dim3(256), 0, s, g, g_lp, g_H, (T*)dz);
    else hipLaunchKernelGGL((token_logprobs_grad<T, false>), grid, dim3(256), 0, s, g, g_lp, g_H, (T*)dz);
  });
  check_launch("token_logprobs_backward");
}

}  // namespace k
}  // namespace agpu
