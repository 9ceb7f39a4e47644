// Softmax cross entropy of a linear layer over a vocabulary, and its gradient,
// without the logits in memory.
//
//   z = x w^T,  lse_r = log sum_v exp z_rv,  loss_r = lse_r - z_rt
//   d_rv = g_r (p_rv - [v = t]) + h_r p_rv,  dx = d w,  dw = d^T x
//
// Forward: one product whose epilogue keeps, of each row of a tile, the
// maximum and the sum of exponentials without the target's own, and the
// target's logit; a second launch joins the tiles of a row.  With the others'
// sum apart, a nearly certain word's loss is log1p(sum exp(z_v - z_t)) and
// keeps its digits, where lse - z_t would have lost them.
//
// Backward: the logits of a piece of the vocabulary are formed again, their
// epilogue writes d (16-bit, or the two fp16 planes of fp32 operands), and two
// products read it: dx over the piece's words, in parts that are summed in
// order, and dw over the rows.  No sum goes through atomics.
//
// Roundings: d is rounded once to the operands' 16 bits before its products,
// as the logits' gradient of any 16-bit program is, times a factor that takes
// the largest of them to 255 2^6 (planes of fp32: a power of two, to 2^13 and
// more), so that in fp16 what is 2^-37 of it still counts, in bf16 2^-139.  That
// value has 8 bits: rows of one weight, whose targets' d are all nearly the
// largest, are then held without an error that their sums would keep (96 rows
// of weight 1.0035 in bf16: error of dw 3.6e-3 with a power of two, so 1.7e-3,
// its own rounding).  fp32 operands are scaled by a power of two, from their
// largest magnitude, and split into fp16 planes (22 bits); where an operand's rows
// lie too far apart for one power, its products are of the fp32 values themselves.
#include "tile16.hpp"

namespace agpu {
namespace k {
using namespace dev;
using namespace t16;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();

__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// A sum of exponentials as {m, s}: s exp(m), m the largest logit; no term:
// {-inf, 0}.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x), ref = m == -kInf ? 0.f : m;
  return make_float2(m, a.y * exp_fast(a.x - ref) + b.y * exp_fast(b.x - ref));
}
// Logits past this are subtracted before they are multiplied by log2(e).  Up to
// it z log2(e) - c is one fused operation, for c = m log2(e) rounded, and the sum
// is multiplied by what c was rounded by (a step of c is 2^-3 here; it is 512 at
// 2^33, and 2 to that power no number).
constexpr float kFused = 0x1p20f;

// ── powers of two that bring values into fp16's range ─────────────────────
// {2^s, 2^-s} with the largest magnitude times 2^s in [2^13, 2^14); {1, 1}
// where there is none.
__device__ __forceinline__ float2 power_for(float most) {
  if (!(most > 0.f)) return make_float2(1.f, 1.f);
  int e;
  frexpf(most, &e);  // most in [2^(e-1), 2^e)
  int s = 14 - e;
  s = s > 126 ? 126 : s;
  return make_float2(ldexpf(1.f, s), ldexpf(1.f, -s));
}
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a < kInf ? a : 0.f;
}
__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (unsigned i = 1; i < blockDim.x / 64; ++i) v = fmaxf(v, red[i]);
  return v;
}

constexpr int kParts = 512;  // blocks of the largest magnitudes' first pass
struct Rows32 {
  const float* x;
  int64_t rows, n, ld;
  int team;  // threads of a row: a power of two up to 64, or 256
};
// Of a part of an operand's rows: the largest magnitude, and the least that is
// any row's largest (rows of zeros aside).
struct Span {
  float most, least;
};
// part[y][b]: of the rows of operand y that block b has; infinite with an
// infinity among them.  (50257 x 768: 28 us, 26 without the rows' own.)
__global__ void __launch_bounds__(256) most_kernel(Rows32 x0, Rows32 x1, Span* part) {
  __shared__ float red[4];
  const Rows32 o = blockIdx.y ? x1 : x0;
  const bool fours = o.n % 4 == 0 && o.ld % 4 == 0 && ((uintptr_t)o.x & 15) == 0;
  auto size4 = [](float4 v) { return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))); };
  Span s{0.f, kInf};
  if (o.rows == 1) {  // a row of its own scale, by all blocks
    const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, apart = (int64_t)kParts * 256;
    if (fours)
      for (int64_t i = first * 4; i < o.n; i += apart * 4) s.most = fmaxf(s.most, size4(*(const float4*)(o.x + i)));
    else
      for (int64_t i = first; i < o.n; i += apart) s.most = fmaxf(s.most, fabsf(o.x[i]));
  } else {
    const int team = o.team, member = threadIdx.x & (team - 1), each = 256 / team;
    const int64_t apart = (int64_t)kParts * each;
    constexpr int kAtOnce = 4;
    for (int64_t r0 = (int64_t)blockIdx.x * each; r0 < o.rows; r0 += apart * kAtOnce) {
      float m[kAtOnce] = {};
      const float* at[kAtOnce];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {  // (the last row again behind it)
        const int64_t r = r0 + threadIdx.x / team + q * apart;
        at[q] = o.x + (r < o.rows ? r : o.rows - 1) * o.ld;
      }
      if (fours) {
#pragma unroll 1
        for (int64_t i = member * 4; i < o.n; i += team * 4)
#pragma unroll
          for (int q = 0; q < kAtOnce; ++q) m[q] = fmaxf(m[q], size4(*(const float4*)(at[q] + i)));
      } else {
        for (int64_t i = member; i < o.n; i += team)
#pragma unroll
          for (int q = 0; q < kAtOnce; ++q) m[q] = fmaxf(m[q], fabsf(at[q][i]));
      }
      for (int k = team == 256 ? 32 : team / 2; k; k >>= 1)
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) m[q] = fmaxf(m[q], __shfl_xor(m[q], k));
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        if (team == 256) m[q] = block_max(m[q], red);
        s.most = fmaxf(s.most, m[q]);
        if (m[q] > 0.f) s.least = fminf(s.least, m[q]);
      }
    }
  }
  s.most = block_max(s.most, red);
  s.least = -block_max(-s.least, red);
  if (threadIdx.x == 0) part[blockIdx.y * kParts + blockIdx.x] = s;
}
// The operands' powers, and whether fp16 planes do not hold them: a row whose
// largest value is 2^-14 of the operand's is held to 2^-24 of that value (the
// low plane's smallest step is 2^-38 of the operand's largest), but beside a row
// of 2^40 times the others nothing is left of them.  Where rows are further apart
// than 2^14, or hold an infinity or nothing that a power and its inverse reach
// (2^90: products of up to 2^47 times one operand's power stay finite), products
// are of the fp32 values themselves and the powers are 1.  (In planes / of the values, us: loss of 61 x 50257 x 1280
// 101 / 231, of 1023 x 50257 x 768 313 / 962; gradients 307 / 558, 733 / 2738.)
struct Scales {
  float2 x, w;  // {2^s, 2^-s}
  int full;
};
// From all parts, for a block of 256.
__device__ __forceinline__ Scales scales_of(const Span* part) {
  static_assert(kParts == 512, "two parts a thread");
  __shared__ Span red[2][4];
  Span t[2];
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const Span a = part[y * kParts + threadIdx.x], b = part[y * kParts + threadIdx.x + 256];
    t[y] = {wave_max(fmaxf(a.most, b.most)), -wave_max(-fminf(a.least, b.least))};
    if ((threadIdx.x & 63) == 0) red[y][threadIdx.x >> 6] = t[y];
  }
  __syncthreads();
  Scales s;
  s.full = 0;
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    Span a = red[y][0];
#pragma unroll
    for (int q = 1; q < 4; ++q) a = {fmaxf(a.most, red[y][q].most), fminf(a.least, red[y][q].least)};
    if (!(a.most <= 0x1p90f && a.most <= a.least * 0x1p14f) || (a.most > 0.f && a.most < 0x1p-90f)) s.full = 1;
    (y ? s.w : s.x) = power_for(a.most);
  }
  if (s.full) s.x = s.w = make_float2(1.f, 1.f);
  return s;
}
// Rows [rows, n] as 16-bit rows of ld values, zeros behind n: fp32 as planes of
// x times its power of two, 16-bit values as they are.  The first operand's
// launch (with the parts) finds both powers and leaves them in *scales for what
// follows.
template <typename TI, typename T, int PL>
__global__ void __launch_bounds__(256) pack_kernel(const TI* x, int64_t rows, int64_t n, int64_t ldi, const Span* part,
                                                   Scales* scales, T* out, int64_t ld) {
  float s = 1.f;
  if constexpr (PL == 2) {
    Scales c;
    if (part) {
      c = scales_of(part);
      if (blockIdx.x == 0 && threadIdx.x == 0) *scales = c;
      s = c.x.x;
    } else {
      c = *scales;
      s = c.w.x;
    }
    if (c.full) return;
  }
  const int chunks = (int)(ld / (8 * PL));
  const int64_t total = rows * chunks, apart = (int64_t)gridDim.x * 256;
  struct V { TI e[8]; };
  for (int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x; i0 < total; i0 += 2 * apart) {
    V t[2] = {};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t i = i0 + q * apart;
      if (i >= total) continue;
      const int64_t r = i / chunks, c = (i - r * chunks) * 8;
      const TI* at = x + r * ldi + c;
      if (c + 8 <= n) __builtin_memcpy(&t[q], at, sizeof(V));  // (at any alignment)
      else
        for (int e = 0; e < 8; ++e)
          if (c + e < n) t[q].e[e] = at[e];
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t i = i0 + q * apart;
      if (i >= total) continue;
      const int64_t r = i / chunks, c = (i - r * chunks) * 8;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = to_f(t[q].e[e]) * s;
      put_planes<T, PL>(out + r * ld, c, v);
    }
  }
}

// ── forward ───────────────────────────────────────────────────────────────
__device__ __forceinline__ int64_t target_of(const void* t, bool wide, int64_t r, int64_t V) {
  const int64_t v = wide ? ((const int64_t*)t)[r] : ((const int32_t*)t)[r];
  return v >= 0 && v < V ? v : -1;
}

// Of each row of the tile: the sum of exponentials of the logits but the
// target's, and the target's logit.
struct EpiLoss {
  float2* part;  // [tiles_n][R]
  float* zt;
  const void* targets;
  bool wide;
  const Scales* scales;  // fp32
  static constexpr bool kFull = true;
  // the accumulators' first registers take a row's {m, s}
  template <class TL>
  __device__ __forceinline__ void form(const Args& p, const Place& c, typename TL::Acc& acc) const {
    constexpr int TM = TL::TM, TN = TL::TN;
    float ux = 1.f, uw = 1.f;
    if constexpr (TL::PL == 2) { ux = scales->x.y; uw = scales->w.y; }
    const int64_t cols = c.n0 + c.wn * 32 * TN;
    const bool ragged = cols + 32 * TN > p.N;
    const int hi = c.lane >> 5;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int64_t row = c.m0 + TL::row_of(c, i);
      const int64_t t = row < p.M ? target_of(targets, wide, row, p.N) : -1;
      const int64_t far = t - cols;
      const int rel = far >= 0 && far < 32 * TN && ((far >> 2) & 1) == hi ? (int)far - 4 * hi : -1;
      float z[TN * 16];
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float v = acc[i][j][e];
          if constexpr (TL::PL == 2) v = v * ux * uw;
          z[j * 16 + e] = v;
        }
      if (ragged) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (c.n0 + TL::col_of(c, j, e) >= p.N) z[j * 16 + e] = -kInf;
      }
      if (rel >= 0) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (rel == j * 32 + 8 * (e >> 2) + (e & 3)) {
              zt[row] = z[j * 16 + e];
              z[j * 16 + e] = -kInf;
            }
      }
      float m = z[0];
#pragma unroll
      for (int e = 1; e < TN * 16; ++e) m = fmaxf(m, z[e]);
      m = fmaxf(m, __shfl_xor(m, 32));
      // (a NaN is no maximum but makes the sum NaN, and so does +inf)
      if (!(m > -kInf)) m = -kInf;
      const bool large = m > -kInf && fabsf(m) > kFused, fused = m > -kInf && !large;
      const float c2 = fused ? m * kLog2e : 0.f, lost = fused ? fmaf(m, kLog2e, -c2) : 0.f;
      if (__any(large)) {
        const float ref = large ? m : 0.f;
#pragma unroll
        for (int e = 0; e < TN * 16; ++e) z[e] -= ref;
      }
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < TN * 16; ++e) s += __builtin_amdgcn_exp2f(fmaf(z[e], kLog2e, -c2));
      s += __shfl_xor(s, 32);
      s *= __builtin_amdgcn_exp2f(-lost);
      acc[i][0][0] = m;
      acc[i][0][1] = s;
    }
  }
  template <class TL>
  __device__ __forceinline__ void store(const Args& p, const Place& c, typename TL::T* lds, typename TL::Acc& acc) const {
    float2* pair = (float2*)lds;  // [BM][WN]
#pragma unroll
    for (int i = 0; i < TL::TM; ++i)
      if (c.lane < 32) pair[TL::row_of(c, i) * TL::WN + c.wn] = make_float2(acc[i][0][0], acc[i][0][1]);
    __syncthreads();
    for (int r = threadIdx.x; r < TL::BM; r += 64 * TL::NW) {
      if (c.m0 + r >= p.M) break;
      float2 v = pair[r * TL::WN];
#pragma unroll
      for (int q = 1; q < TL::WN; ++q) v = join(v, pair[r * TL::WN + q]);
      part[(int64_t)c.tn * p.M + c.m0 + r] = v;
    }
  }
};

// Joins a row's parts: 256 threads as `rx` rows by 256 / rx parts.
__global__ void __launch_bounds__(256) loss_kernel(const float2* part, int64_t parts, const float* zt,
                                                   const void* targets, bool wide, int64_t R, int64_t V, int rx,
                                                   float* loss, float* lse) {
  __shared__ float2 red[256];
  const int x = threadIdx.x % rx, y = threadIdx.x / rx, ny = 256 / rx;
  const int64_t row = (int64_t)blockIdx.x * rx + x;
  float2 a = make_float2(-kInf, 0.f);
  if (row < R)
    for (int64_t q = y; q < parts; q += ny) a = join(a, part[q * R + row]);
  red[threadIdx.x] = a;
  for (int h = ny >> 1; h; h >>= 1) {
    __syncthreads();
    if (y < h) red[threadIdx.x] = a = join(a, red[threadIdx.x + h * rx]);
  }
  if (y != 0 || row >= R) return;
  float out = 0.f, sum;
  if (target_of(targets, wide, row, V) < 0) {
    sum = a.x + logf(a.y);
  } else {
    // log(exp z_t + the others), from the larger of the two
    const float z = zt[row];
    if (z == kInf) {
      out = sum = kInf - z;  // an infinite sum has no certain word: NaN
    } else if (z >= a.x) {
      out = log1pf(a.y * expf(a.x - z));
      sum = z + out;
    } else {
      const float others = logf(a.y + expf(z - a.x));
      out = (a.x - z) + others;
      sum = a.x + others;
    }
  }
  loss[row] = out;
  lse[row] = sum;
}

// ── backward ──────────────────────────────────────────────────────────────
// What a row of d is made of: {lse, weight of p, d of the target in 16 bits,
// what that rounding lost}.  The weight and d hold the factor from the largest
// |d| that any row can have: of words other than the target |g + h| (1 - p_t),
// of all |h| where there is none.  A row's largest part is its target's, alone in
// its size, so its rounding would be dx's: dx gets back what it lost times the
// target's weights (fp16, 30 rows: error of dx 3.3e-4, so 2.2e-4), and dw likewise
// where rows are few.  Every block finds the factor from all rows.
struct RowPart {
  float g, h, dt, most;
};
__device__ __forceinline__ RowPart row_part(const float* g, const float* h, const float* loss, bool there, int64_t r) {
  RowPart o;
  o.g = there ? g[r] : 0.f;
  o.h = h ? h[r] : 0.f;
  o.dt = o.most = 0.f;
  if (o.g == 0.f && o.h == 0.f) return o;  // without weight: nothing, whatever its loss is
  // 1 - p of the target from its loss, which keeps its digits
  const float left = there ? -expm1f(-loss[r]) : 1.f;
  o.dt = there ? o.h * expf(-loss[r]) - o.g * left : 0.f;
  o.most = fmaxf(finite_abs(o.dt), finite_abs((o.g + o.h) * left));
  return o;
}
__device__ __forceinline__ float2 factor_for(float most) {
  constexpr float kLargest = 16320.f;  // 255 2^6
  return most >= 0x1p-100f ? make_float2(kLargest / most, most / kLargest) : power_for(most);
}
// The largest of rows' parts and weights: of many rows by blocks of 1024 first
// (every block over all rows / in a launch of its own, whole gradients: 4096 x
// 1000 x 64 bf16 36 / 37 us, 16384 x 256 x 128 48 / 38).
struct Most {
  float part, weight;
};
__device__ __forceinline__ Most most_of_rows(const float* g, const float* h, const float* loss, const void* targets,
                                             bool wide, int64_t R, int64_t V, int64_t i, int64_t apart, float* red) {
  Most m{0.f, 0.f};
#pragma unroll 4
  for (; i < R; i += apart) {
    const RowPart o = row_part(g, h, loss, target_of(targets, wide, i, V) >= 0, i);
    m.part = fmaxf(m.part, o.most);
    m.weight = fmaxf(m.weight, finite_abs(o.g + o.h));
  }
  m.part = block_max(m.part, red);
  m.weight = block_max(m.weight, red);
  return m;
}
constexpr int kMostBlocks = 128;
__global__ void __launch_bounds__(1024) rows_most_kernel(const float* g, const float* h, const float* loss,
                                                         const void* targets, bool wide, int64_t R, int64_t V, Most* out) {
  __shared__ float red[16];
  const Most m = most_of_rows(g, h, loss, targets, wide, R, V, (int64_t)blockIdx.x * 1024 + threadIdx.x,
                              (int64_t)gridDim.x * 1024, red);
  if (threadIdx.x == 0) out[blockIdx.x] = m;
}

template <typename T, int PL>
__global__ void __launch_bounds__(1024) rows_kernel(const float* g, const float* h, const float* loss, const float* lse,
                                                    const void* targets, bool wide, int64_t R, int64_t V, float2* power,
                                                    float4* rows, const Most* most, int mosts, const Scales* scales) {
  __shared__ float red[16];
  Most all;
  if (most) {
    const Most mine = (int)threadIdx.x < mosts ? most[threadIdx.x] : Most{0.f, 0.f};
    all = {block_max(mine.part, red), block_max(mine.weight, red)};
  } else {
    all = most_of_rows(g, h, loss, targets, wide, R, V, threadIdx.x, 1024, red);
  }
  // (a weight of p times the factor stays finite where every row is certain)
  const float m = fmaxf(all.part, all.weight * 0x1p-106f);
  const float2 pw = PL == 1 ? factor_for(m) : scales->full ? make_float2(1.f, 1.f) : power_for(m);
  if (blockIdx.x == 0 && threadIdx.x == 0) *power = pw;
  const float up = pw.x;
  const int64_t r = (int64_t)blockIdx.x * 1024 + threadIdx.x;
  if (r >= R) return;
  const RowPart o = row_part(g, h, loss, target_of(targets, wide, r, V) >= 0, r);
  float held = o.dt * up, lost = 0.f;
  if constexpr (PL == 1) {
    held = to_f(from_f<T>(o.dt * up));
    lost = (o.dt * up - held) * pw.y;
    if (!(fabsf(lost) < kInf)) lost = 0.f;
  }
  rows[r] = make_float4(lse[r], (o.g + o.h) * up, held, lost);
}

// d of the tile's logits, in panels; zeros behind the words up to the last
// panel's end.  Formed where the accumulators are, from the few rows that a lane
// has.
template <typename T>
struct EpiGrad {
  T* d;
  int64_t panel, len;  // values of a panel; the piece's words
  int64_t v0, V;  // the piece's first word; all words
  const void* targets;
  bool wide;
  const float4* rows;
  const Scales* scales;  // fp32
  static constexpr bool kFull = true;
  template <class TL>
  __device__ __forceinline__ void form(const Args& p, const Place& c, typename TL::Acc& acc) const {
    constexpr int PL = TL::PL, TM = TL::TM, TN = TL::TN;
    float ux = 1.f, uw = 1.f;
    if constexpr (PL == 2) { ux = scales->x.y; uw = scales->w.y; }
    const int64_t cols = c.n0 + c.wn * 32 * TN;
    const bool ragged = cols + 32 * TN > p.N;
    const int hi = c.lane >> 5;
    float4 of[TM];
    int rel[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int64_t row = c.m0 + TL::row_of(c, i), at = row < p.M ? row : p.M - 1;
      const int64_t t = row < p.M ? target_of(targets, wide, at, V) : -1, far = t - v0 - cols;
      of[i] = rows[at];
      rel[i] = t >= 0 && far >= 0 && far < 32 * TN && ((far >> 2) & 1) == hi ? (int)far - 4 * hi : -1;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const bool none = of[i].y == 0.f && of[i].z == 0.f;  // without weight: no gradient, whatever the logits are
      auto p_times_weight = [&](float at, float most) {
        float z = at;
        if constexpr (PL == 2) z = z * ux * uw;
        z -= of[i].x;
        return exp_fast(z > most ? most : z) * of[i].y;
      };
      // a logit may pass a large sum by what either was rounded by, but p is no
      // more than 1
      const bool large = fabsf(of[i].x) > kFused;
      if (__any(large)) {
        const float most = large ? 0.f : kInf;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] = none ? 0.f : p_times_weight(acc[i][j][e], most);
      } else {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] = none ? 0.f : p_times_weight(acc[i][j][e], kInf);
      }
      if (rel[i] >= 0 && !none) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (rel[i] == j * 32 + 8 * (e >> 2) + (e & 3)) acc[i][j][e] = of[i].z;
      }
      if (ragged) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (c.n0 + TL::col_of(c, j, e) >= p.N) acc[i][j][e] = 0.f;
      }
    }
  }
  template <class TL>
  __device__ __forceinline__ void store(const Args& p, const Place& c, typename TL::T* lds, typename TL::Acc& acc) const {
    constexpr int PL = TL::PL;
    const bool full = PL == 2 && scales->full;  // (as they are: fp32 values take the planes' place)
    TL::template runs<false>(
        c, lds, acc, false,
        [&](int64_t row, int64_t col, float (&v)[8]) {
          constexpr int W = 64 / PL;  // words of a panel
          if (row >= p.M || col >= (len + W - 1) / W * W) return;
          T* at = d + col / W * panel + row * 64;
          if (full) {
            struct alignas(16) V { float e[4]; } o[2];
            __builtin_memcpy(o, v, 32);
            put_past((float*)at + col % W, o[0]);
            put_past((float*)at + col % W + 4, o[1]);
          } else {
            put_planes<T, PL>(at, col % W, v);
          }
        },
        [](int64_t, int64_t, float (&)[8]) {});
  }
};

// What dx gets back of its targets' parts (rows null: nothing).
template <typename TO>
struct Lost {
  const TO* w = nullptr;
  int64_t ldw = 0, V = 0;
  const void* targets = nullptr;
  bool wide = false;
  const float4* rows = nullptr;
  // the factor, and the weights it applies to from column k on
  __device__ __forceinline__ float of(int64_t row, int64_t k, const TO** at) const {
    if (!rows) return 0.f;
    const int64_t t = target_of(targets, wide, row, V);
    *at = w + t * ldw + k;
    return t < 0 ? 0.f : rows[row].w;
  }
};
// What dw gets back of its words' rows, in the units of the accumulators, for few
// rows: there one row's rounding can be most of the error (1 to 5 rows in bf16: up
// to 3.9e-3 beside the result's own 1.7e-3), where that of many evens out (61: 1.3
// times the result's, 8191: 1.35) and looking the targets up takes 7 us of 102.
constexpr int kFewRows = 32;
template <typename TO>
struct LostOfRows {
  int count = 0;
  const float4* rows = nullptr;
  const TO* x = nullptr;
  int64_t ldx = 0, v0 = 0;
  const void* targets = nullptr;
  bool wide = false;
  const float2* up = nullptr;
  template <class TL>
  __device__ __forceinline__ void add(const Args& p, const Place& c, typename TL::Acc& acc) const {
    const int64_t t = c.lane < count ? target_of(targets, wide, c.lane, v0 + p.M) : -1;
    const int64_t far = t - v0 - c.m0 - c.wm * TL::TM * 32;
    const int in = t >= 0 && far >= 0 && far < TL::TM * 32 ? (int)far : -1;
    const int cols = (int)(p.N - c.n0);
    for (uint64_t left = __ballot(in >= 0); left; left &= left - 1) {
      const int r = __builtin_ctzll(left), word = __builtin_amdgcn_readlane(in, r);
      const float back = rows[r].w * up->x;
      if (back == 0.f || (c.lane & 31) != (word & 31)) continue;
      const TO* at = x + r * ldx + c.n0;
#pragma unroll
      for (int i = 0; i < TL::TM; ++i)
        if (word >> 5 == i) {
#pragma unroll
          for (int j = 0; j < TL::TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int col = TL::col_of(c, j, e);  // (columns behind the last are not stored)
              acc[i][j][e] += back * to_f(at[col < cols ? col : 0]);
            }
        }
    }
  }
};

// The inverse powers of a product's operands (null: 1), the smaller first: what is
// between them is not past the result.
__device__ __forceinline__ float2 unscale(const float2* pa, const float2* pb) {
  const float a = pa ? pa->y : 1.f, b = pb ? pb->y : 1.f;
  return make_float2(fminf(a, b), fmaxf(a, b));
}
// acc times the inverse powers, as outputs or as fp32 parts of a sum.
template <typename TO, bool FEW = false>
struct EpiOut {
  static constexpr bool kFull = true;
  TO* out;
  float* part;   // [splits][M][N], or null
  bool more;     // parts are added to what is there
  const float2 *pa, *pb;
  Lost<TO> lost;
  LostOfRows<TO> back;
  template <class TL>
  __device__ __forceinline__ void form(const Args& p, const Place& c, typename TL::Acc& acc) const {
    if constexpr (FEW && TL::PL == 1) back.template add<TL>(p, c, acc);
  }
  template <class TL>
  __device__ __forceinline__ void store(const Args& p, const Place& c, typename TL::T* lds, typename TL::Acc& acc) const {
    const float2 u = unscale(pa, pb);
    float* sums = part ? part + (int64_t)c.split * p.M * p.N : nullptr;
    TL::template runs<false>(
        c, lds, acc, false,
        [&](int64_t row, int64_t col, float (&v)[8]) {
          if (row >= p.M || col >= p.N) return;
          const int64_t at = row * p.N + col;
          const int n = p.N - col < 8 ? (int)(p.N - col) : 8;
          if (sums) {
            if (n == 8) {
              struct F4 { float e[4]; } t[2] = {};
              if (more) __builtin_memcpy(t, sums + at, 32);
#pragma unroll
              for (int e = 0; e < 8; ++e) t[e >> 2].e[e & 3] += v[e];
              put_past(sums + at, t[0]);
              put_past(sums + at + 4, t[1]);
            } else {
              for (int e = 0; e < 8; ++e)
                if (e < n) sums[at + e] = v[e] + (more ? sums[at + e] : 0.f);
            }
            return;
          }
          const TO* wt = nullptr;
          const float back = lost.of(row, col, &wt);
          constexpr int W = 16 / sizeof(TO);  // a store
          struct V { TO e[W]; } o[8 / W];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = v[e] * u.x * u.y;
            if (back != 0.f && e < n) v[e] += back * to_f(wt[e]);
            o[e / W].e[e % W] = from_f<TO>(v[e]);
          }
          if (n == 8) {
#pragma unroll
            for (int q = 0; q < 8 / W; ++q) put_past(out + at + q * W, o[q]);
          } else {
            for (int e = 0; e < 8; ++e)
              if (e < n) out[at + e] = o[e / W].e[e % W];
          }
        },
        [](int64_t, int64_t, float (&)[8]) {});
  }
};

// out [.., K] = the parts' sum times the inverse powers, and what they lost.  G
// threads take the parts of 4 values in turn and their sums are added in order:
// many parts behind one another are a chain of loads (32 parts of 61 x 1280, one
// thread / eight: 10.4 / 6.5 us).
template <typename TO, int G>
__global__ void __launch_bounds__(256) sum_parts_kernel(const float* part, int splits, int64_t n, int64_t K,
                                                        const float2* pa, const float2* pb, Lost<TO> lost, TO* out) {
  __shared__ float4 red[256];
  constexpr int X = 256 / G;
  const int x = threadIdx.x % X, y = threadIdx.x / X;
  const int64_t i = ((int64_t)blockIdx.x * X + x) * 4;
  const int m = n - i < 4 ? (int)(n - i) : 4;  // (none behind the end)
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (n % 4 == 0) {
    if (m > 0)
#pragma unroll 8
      for (int s = y; s < splits; s += G) {
        const float4 b = *(const float4*)(part + s * n + i);
        a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
      }
  } else {
    for (int s = y; s < splits; s += G) {
      const float* b = part + s * n + i;
      if (m > 0) a.x += b[0];
      if (m > 1) a.y += b[1];
      if (m > 2) a.z += b[2];
      if (m > 3) a.w += b[3];
    }
  }
  if constexpr (G > 1) {
    red[threadIdx.x] = a;
    __syncthreads();
    if (y != 0) return;
#pragma unroll
    for (int g = 1; g < G; ++g) {
      const float4 b = red[g * X + x];
      a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
    }
  }
  if (m <= 0) return;
  const float2 u = unscale(pa, pb);
  float v[4] = {a.x * u.x * u.y, a.y * u.x * u.y, a.z * u.x * u.y, a.w * u.x * u.y};
  const TO* wt = nullptr;
  if (K % 4 == 0) {
    const int64_t r = i / K;
    const float back = lost.of(r, i - r * K, &wt);
    struct V { TO e[4]; } o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (back != 0.f) v[e] += back * to_f(wt[e]);
      o.e[e] = from_f<TO>(v[e]);
    }
    __builtin_memcpy(out + i, &o, sizeof(o));
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (e >= m) break;
    const float back = lost.of((i + e) / K, (i + e) % K, &wt);
    if (back != 0.f) v[e] += back * to_f(*wt);
    out[i + e] = from_f<TO>(v[e]);
  }
}

// ── host side ─────────────────────────────────────────────────────────────
// Parts of a workspace; without one, only their sizes.
struct Carver {
  char* base;
  size_t used = 0;
  template <typename P> P* take(size_t n) {
    P* at = base ? (P*)(base + used) : nullptr;
    used += (n * sizeof(P) + 255) / 256 * 256;
    return at;
  }
};

bool direct(const void* p, int64_t ld, int64_t K) {
  return K % 8 == 0 && ld % 8 == 0 && ((uintptr_t)p & 15) == 0 && ld < (1 << 21);
}

// The operands x and w as a product takes them: in place, packed into the
// workspace, or (raw) w as the fp32 rows that it is; fp32: with their powers.
struct Both {
  Operand x, w;
  Scales* scales = nullptr;
  const float2 *px = nullptr, *pw = nullptr;
  const int* full = nullptr;
};
template <typename TI, typename T, int PL>
Both ready(const LinearCE& a, bool raw, Carver& ws, hipStream_t s) {
  Both b;
  Span* part = nullptr;
  if constexpr (PL == 2) {
    part = ws.take<Span>(2 * kParts);
    b.scales = ws.take<Scales>(1);
    if (ws.base) {
      b.px = &b.scales->x;
      b.pw = &b.scales->w;
      b.full = &b.scales->full;
      auto rows = [&](const void* x, int64_t rows, int64_t ld) {
        int team = 256;
        if (a.K <= 4096 && rows > 1)
          for (team = 1; team < 64 && team * 4 < a.K;) team *= 2;
        return Rows32{(const float*)x, rows, a.K, ld, team};
      };
      hipLaunchKernelGGL(most_kernel, dim3(kParts, 2), dim3(256), 0, s, rows(a.x, a.R, a.ldx), rows(a.w, a.V, a.ldw),
                         part);
      check_launch("linear_cross_entropy");
    }
  }
  auto pack = [&](Operand& o, const void* x, int64_t rows, int64_t ld, const Span* parts) {
    if (PL == 1 && direct(x, ld, a.K)) {
      o = {x, ld, 0};
      return;
    }
    const int64_t kp = (a.K + 31) / 32 * 32 * PL;
    T* out = ws.take<T>((size_t)(rows * kp));
    o = {out, kp, 0};
    if (!ws.base) return;
    const unsigned blocks = (unsigned)std::min<int64_t>(blocks_for(rows * (kp / (8 * PL)), 512), 4096);
    hipLaunchKernelGGL((pack_kernel<TI, T, PL>), dim3(blocks), dim3(256), 0, s, (const TI*)x, rows, a.K, ld, parts,
                       b.scales, out, kp);
    check_launch("linear_cross_entropy");
  };
  pack(b.x, a.x, a.R, a.ldx, part);
  if (raw) b.w = {a.w, 2 * a.ldw, 0};
  else pack(b.w, a.w, a.V, a.ldw, nullptr);
  return b;
}

// Tiles of 8 wavefronts: 256 x 256, 128 x 128, 64 x 128; of 4: 32 x 128.
enum { kBig, kMid, kThin, kFew };
// Forward in us, 256 / 128 / 64 / 32 rows a tile:
//   1 x 50257 x 1280 fp16     35 / 25 / 25 / 24
//   61 x 50257 x 1280 fp16    37 / 27 / 26 / 31
//   509 x 50257 x 768 bf16    52 / 54 / 60       (394 and 1572 tiles)
//   1111 x 10007 x 515 fp16   38 / 42 / 46       (200 and 711)
//   1000 x 2000 x 512 bf16    22 / 12 / 11       (32 and 128)
// A round of 128-wide tiles, two a compute unit, takes 0.53 times a round of
// 256-wide ones.  (Splitting fp32 words takes registers that 256 x 256 does not
// have.)
int pick(int64_t M, int64_t N, bool raw, int cus) {
  if (M <= 32) return kFew;
  if (M <= 64) return kThin;
  const double big = (double)ceil_div(ceil_div(M, 256) * ceil_div(N, 256), cus);
  const double mid = (double)ceil_div(ceil_div(M, 128) * ceil_div(N, 128), 2 * cus);
  return !raw && big <= 0.53 * mid ? kBig : kMid;
}
int bn_of(int tile) { return tile == kBig ? 256 : 128; }

template <typename T, int PL, Layout BL, class Epi>
void run(int tile, const Args& p, const Epi& e, hipStream_t s, const char* what) {
  if (tile == kBig && BL == kRows) launch<Tile<T, 4, 2, 2, 4, PL, kRows, kRows>>(p, e, s, what);
  else if (tile == kMid) launch<Tile<T, 2, 1, 2, 4, PL, kRows, BL>>(p, e, s, what);
  else if (tile == kThin) launch<Tile<T, 1, 1, 2, 4, PL, kRows, BL>>(p, e, s, what);
  else launch<Tile<T, 1, 1, 1, 4, PL, kRows, BL>>(p, e, s, what);
}

// The fp32 operands of the logits of the words from v0 on, as they are.
void full_rows(Args& p, const Both& b, const LinearCE& a, int64_t v0) {
  p.full = b.full;
  p.fa = (const float*)a.x;
  p.lda = a.ldx;
  p.fb = (const float*)a.w + v0 * a.ldw;
  p.ldb = a.ldw;
}

template <typename TI, typename T, int PL>
size_t forward(const LinearCE& a, void* wsp, int cus, hipStream_t s) {
  const char* what = "linear_cross_entropy";
  Carver ws{(char*)wsp};
  // fp32 words of few rows are split where they are multiplied (packed, each is
  // written and read once more), by every block that multiplies them: 50257 x
  // 768, us, packed / split at 20 rows 119 / 62, 61: 122 / 72, 255: 145 / 129,
  // 1023: 311 / 345
  const bool raw = PL == 2 && a.R <= 320 && a.K % 4 == 0 && a.ldw % 4 == 0 && a.ldw < (1 << 20) &&
                   ((uintptr_t)a.w & 15) == 0;
  const Both b = ready<TI, T, PL>(a, raw, ws, s);
  const int tile = pick(a.R, a.V, raw, cus);
  const int64_t parts = ceil_div(a.V, bn_of(tile));
  float2* part = ws.take<float2>((size_t)(parts * a.R));
  float* zt = ws.take<float>((size_t)a.R);
  if (!wsp) return ws.used;
  Args p;
  p.a = b.x; p.b = b.w;
  p.M = a.R; p.N = a.V; p.K = a.K;
  const bool wide = a.idx_dt == DType::I64;
  p.b_power = b.pw;
  if (PL == 2) full_rows(p, b, a, 0);
  const EpiLoss e{part, zt, a.targets, wide, b.scales};
  if (PL == 2 && raw) run<T, PL, PL == 2 ? kRaw : kRows>(tile, p, e, s, what);
  else run<T, PL, kRows>(tile, p, e, s, what);
  const int rx = a.R >= 64 * cus ? 64 : a.R >= 16 * cus ? 16 : a.R >= 4 * cus ? 4 : 1;
  hipLaunchKernelGGL(loss_kernel, dim3(blocks_for(a.R, rx)), dim3(256), 0, s, part, parts, zt, a.targets, wide, a.R,
                     a.V, rx, a.loss, a.lse);
  check_launch(what);
  return ws.used;
}

// Values of d that are held at once: 2^29 (1 GB of 16 bits).
constexpr int64_t kHeld = (int64_t)1 << 29;

// When n1 blocks of l1 stages and then n2 of l2 have all ended, one after
// another on `slots` places.
double ends(int64_t n1, double l1, int64_t n2, double l2, int64_t slots) {
  const double whole = (double)(n1 / slots) * l1;  // by then every place is free of whole rounds
  const int64_t late = n1 % slots;                 // places that take one more of the first
  const double least = late ? whole + l1 : whole;
  auto fit = [&](double t) {
    return (int64_t)((t - whole) / l2 + 1e-6) * (slots - late) + (int64_t)((t - whole - l1) / l2 + 1e-6) * late >= n2;
  };
  double t = least;
  for (int64_t k = n2 / slots; !fit(t) && k <= n2 + 1; ++k) {
    const double a = whole + (double)k * l2, b = whole + l1 + (double)k * l2;
    if (a >= least && fit(a)) t = a;
    else if (b >= least && fit(b)) t = b;
  }
  return t;
}

// The products dx (over the words, in parts) and dw (over the rows, in parts
// where the vocabulary is one piece) in one launch: tiles and parts by the time
// they end, in us.  A stage of 64 k takes 1.75 us in
// 256 x 256 tiles, 0.95 in 128 x 128 ones (two blocks a compute unit); a block's
// start and end count as 4 stages; parts are written and read back at 6 TB/s
// and summed by a launch of their own.  us at 2 / 4 / 8 / 16 / 32 parts, 256:
// 61 x 50257 x 1280 fp16 536 / 287 / 165 / 114 / 106, 2047 x 10007 x 768 bf16
// 187 / 138 / 163 / 171 / 219; 128: 275 / 155 / 103 / 103 / 100, 135 / 138 / 148
// / 163 / 201.  The whole gradient with dw in one part / in those chosen: bf16,
// 16384 x 100 x 768 206 / 57, 16384 x 5000 x 64 233 / 125; fp32, 4096 x 1000 x 64
// 120 / 49.
struct Plan {
  bool big;
  int parts, wparts;
};
Plan plan_products(int64_t R, int64_t K, int64_t words, bool one_piece, int ks, int cus) {
  Plan best{false, 1, 1};
  double least = 1e300;
  const int64_t stages = ceil_div(words, ks), row_stages = ceil_div(R, ks);
  constexpr int kMany[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48};
  auto join = [&](int parts, int64_t values) { return parts > 1 ? 4 + parts * (double)values * 8 / 6e6 : 0; };
  for (int big = R > 32 ? 1 : 0; big >= 0; --big) {
    const int64_t side = big ? 256 : 128, xside = R <= 32 ? 32 : side;
    const int64_t xtiles = ceil_div(R, xside) * ceil_div(K, side), wtiles = ceil_div(words, side) * ceil_div(K, side);
    for (int w : kMany) {
      if (w > 1 && (!one_piece || w * 4 > row_stages)) break;
      const double wlen = (double)ceil_div(row_stages, w) + 4;
      for (int s : kMany) {
        if (s > 1 && s * 4 > stages) break;
        const double len = (double)ceil_div(stages, s) + 4;
        const double t = ends(xtiles * s, len, wtiles * w, wlen, big ? cus : 2 * cus) * (big ? 1.75 : 0.95) +
                         join(s, R * K) + join(w, words * K);
        if (t < least) {
          least = t;
          best = {big != 0, s, w};
        }
      }
    }
  }
  return best;
}

template <typename TI, typename T, int PL>
size_t backward(const LinearCE& a, void* wsp, int cus, hipStream_t s) {
  const char* what = "linear_cross_entropy_backward";
  Carver ws{(char*)wsp};
  const Both b = ready<TI, T, PL>(a, false, ws, s);
  const bool wide = a.idx_dt == DType::I64;
  // pieces of the vocabulary, whole tiles of it
  const int64_t most = std::max<int64_t>(kHeld / PL / a.R / 256 * 256, 256);
  const int64_t pieces = ceil_div(a.V, most), each = ceil_div(ceil_div(a.V, pieces), 256) * 256;
  // d lies in panels of 128 bytes a row: dx reads it along its rows, dw down
  // them, both in long runs (as rows as long as the piece / in panels, us: 8191 x
  // 50257 x 768 bf16 2057 / 1993, 1023 x 50257 x 768 fp32 and 61 x 50257 x 1280
  // fp16 within 1 % of one another)
  const int64_t len = std::min(each, a.V), panel = a.R * 64;
  T* d = ws.take<T>((size_t)(panel * ceil_div(len, 64 / PL)));
  float2* pg = ws.take<float2>(1);
  float4* rows = ws.take<float4>((size_t)a.R);
  const int mosts = a.R > 4096 ? (int)std::min<int64_t>(ceil_div(a.R, 1024), kMostBlocks) : 0;
  Most* most_of = mosts ? ws.take<Most>((size_t)mosts) : nullptr;
  const Plan plan = plan_products(a.R, a.K, len, pieces == 1, 64 / PL, cus);
  const int splits = plan.parts;
  const bool parted = splits > 1 || pieces > 1;
  float* part = parted ? ws.take<float>((size_t)(splits * a.R * a.K)) : nullptr;
  float* wpart = plan.wparts > 1 ? ws.take<float>((size_t)(plan.wparts * a.V * a.K)) : nullptr;
  if (!wsp) return ws.used;
  if (mosts) {
    hipLaunchKernelGGL(rows_most_kernel, dim3((unsigned)mosts), dim3(1024), 0, s, a.g_loss, a.g_lse, a.loss, a.targets,
                       wide, a.R, a.V, most_of);
    check_launch(what);
  }
  hipLaunchKernelGGL((rows_kernel<T, PL>), dim3(blocks_for(a.R, 1024)), dim3(1024), 0, s, a.g_loss, a.g_lse, a.loss,
                     a.lse, a.targets, wide, a.R, a.V, pg, rows, most_of, mosts, b.scales);
  check_launch(what);
  const Lost<TI> lost{(const TI*)a.w, a.ldw, a.V, a.targets, wide, PL == 1 ? rows : nullptr};
  for (int64_t v0 = 0; v0 < a.V; v0 += each) {
    const int64_t n = std::min(each, a.V - v0);
    const Operand wp{(const T*)b.w.p + v0 * b.w.ld, b.w.ld, 0}, dp{d, panel, 0};
    Args p;
    p.a = b.x; p.b = wp;
    p.M = a.R; p.N = n; p.K = a.K;
    if (PL == 2) full_rows(p, b, a, v0);
    run<T, PL, kRows>(pick(a.R, n, false, cus), p,
                      EpiGrad<T>{d, panel, len, v0, a.V, a.targets, wide, rows, b.scales}, s, what);
    Args px, pw;
    px.full = pw.full = p.full;
    px.fa = pw.fa = (const float*)d;
    px.lda = pw.lda = a.R * 32;
    px.fb = p.fb; px.ldb = p.ldb;
    pw.fb = p.fa; pw.ldb = p.lda;
    px.a = pw.a = dp;
    px.b = wp;
    px.M = a.R; px.N = a.K; px.K = n; px.splits = splits;
    pw.b = b.x;
    pw.M = n; pw.N = a.K; pw.K = a.R; pw.splits = plan.wparts;
    const EpiOut<TI> ex{(TI*)a.dx, part, v0 > 0, pg, b.pw, lost, {}},
        ew{(TI*)a.dw + v0 * a.K, wpart, false, pg, b.px, {}, {}};
    typedef Tile<T, 2, 2, 2, 2, PL, kPanelCols, kCols> WFew;  // (of four wavefronts, as dx's)
    if (plan.big)
      launch_pair<Tile<T, 4, 2, 2, 4, PL, kPanelRows, kCols>, Tile<T, 4, 2, 2, 4, PL, kPanelCols, kCols>>(px, ex, pw, ew, s, what);
    else if (a.R > kFewRows)
      launch_pair<Tile<T, 2, 1, 2, 4, PL, kPanelRows, kCols>, Tile<T, 2, 1, 2, 4, PL, kPanelCols, kCols>>(px, ex, pw, ew, s, what);
    else
      launch_pair<Tile<T, 1, 1, 1, 4, PL, kPanelRows, kCols>, WFew>(
          px, ex, pw,
          EpiOut<TI, true>{ew.out, nullptr, false, pg, b.px, {},
                           {(int)a.R, rows, (const TI*)a.x, a.ldx, v0, a.targets, wide, pg}}, s, what);
  }
  auto sum = [&](const float* of, int parts, int64_t n, const float2* power, const Lost<TI>& back, void* out) {
    auto go = [&](auto kernel, int threads) {
      hipLaunchKernelGGL(kernel, dim3(blocks_for(n * threads, 1024)), dim3(256), 0, s, of, parts, n, a.K, pg, power, back,
                         (TI*)out);
    };
    if (parts >= 8) go(sum_parts_kernel<TI, 8>, 8);
    else go(sum_parts_kernel<TI, 1>, 1);
    check_launch(what);
  };
  if (parted) sum(part, splits, a.R * a.K, b.pw, lost, a.dx);
  if (wpart) sum(wpart, plan.wparts, a.V * a.K, b.px, {}, a.dw);
  return ws.used;
}

}  // namespace

size_t linear_ce_ws_bytes(const LinearCE& a, int cus) {
  if (a.dt == DType::F16) return forward<half_t, half_t, 1>(a, nullptr, cus, nullptr);
  if (a.dt == DType::BF16) return forward<bf16_t, bf16_t, 1>(a, nullptr, cus, nullptr);
  return forward<float, half_t, 2>(a, nullptr, cus, nullptr);
}
void linear_ce(const LinearCE& a, void* ws, int cus, hipStream_t s) {
  if (a.dt == DType::F16) forward<half_t, half_t, 1>(a, ws, cus, s);
  else if (a.dt == DType::BF16) forward<bf16_t, bf16_t, 1>(a, ws, cus, s);
  else forward<float, half_t, 2>(a, ws, cus, s);
}
size_t linear_ce_backward_ws_bytes(const LinearCE& a, int cus) {
  if (a.dt == DType::F16) return backward<half_t, half_t, 1>(a, nullptr, cus, nullptr);
  if (a.dt == DType::BF16) return backward<bf16_t, bf16_t, 1>(a, nullptr, cus, nullptr);
  return backward<float, half_t, 2>(a, nullptr, cus, nullptr);
}
void linear_ce_backward(const LinearCE& a, void* ws, int cus, hipStream_t s) {
  if (a.dt == DType::F16) backward<half_t, half_t, 1>(a, ws, cus, s);
  else if (a.dt == DType::BF16) backward<bf16_t, bf16_t, 1>(a, ws, cus, s);
  else backward<float, half_t, 2>(a, ws, cus, s);
}

}  // namespace k
}  // namespace agpu
