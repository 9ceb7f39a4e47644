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
// as the logits' gradient of any 16-bit program is; fp16 (and the planes of
// fp32) hold d times a power of two that takes the largest |g| + |h| to 2^13,
// so that words of probability 2^-37 still count.  fp32 operands are scaled
// alike by their largest magnitude and split into fp16 planes (22 bits).
#include "tile16.hpp"

namespace agpu {
namespace k {
using namespace dev;
using namespace t16;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();

__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// A sum of exponentials as {c, s}: s 2^c, c the largest exponent; no term:
// {-inf, 0}.  An exponent is z log2(e) - c in one fused operation, whatever c
// was rounded to.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x), ref = m == -kInf ? 0.f : m;
  return make_float2(m, a.y * __builtin_amdgcn_exp2f(a.x - ref) + b.y * __builtin_amdgcn_exp2f(b.x - ref));
}

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

constexpr int kParts = 512;  // blocks of the largest magnitude's first pass
// part[b] = the largest finite magnitude of every kParts-th run of x [rows, n].
__global__ void __launch_bounds__(256) most_kernel(const float* x, int64_t rows, int64_t n, int64_t ld, float* part) {
  __shared__ float red[4];
  float m = 0.f;
  if (ld == n && n % 4 == 0 && ((uintptr_t)x & 15) == 0) {
    const int64_t q = rows * n / 4;
#pragma unroll 4
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < q; i += (int64_t)gridDim.x * 256) {
      const float4 v = ((const float4*)x)[i];
      m = fmaxf(fmaxf(m, fmaxf(finite_abs(v.x), finite_abs(v.y))), fmaxf(finite_abs(v.z), finite_abs(v.w)));
    }
  } else {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
      for (int64_t i = threadIdx.x; i < n; i += 256) m = fmaxf(m, finite_abs(x[r * ld + i]));
  }
  m = block_max(m, red);
  if (threadIdx.x == 0) part[blockIdx.x] = m;
}
// The power of the largest |g| + |h|.
__global__ void __launch_bounds__(1024) grad_power_kernel(const float* g, const float* h, int64_t R, float2* power) {
  __shared__ float red[16];
  float m = 0.f;
  for (int64_t i = threadIdx.x; i < R; i += 1024) m = fmaxf(m, finite_abs(g[i]) + (h ? finite_abs(h[i]) : 0.f));
  m = block_max(m, red);
  if (threadIdx.x == 0) *power = power_for(m);
}

// Rows [rows, n] as 16-bit rows of ld values, zeros behind n: fp32 as planes of
// x times its power of two (from part), 16-bit values as they are.
template <typename TI, typename T, int PL>
__global__ void __launch_bounds__(256) pack_kernel(const TI* x, int64_t rows, int64_t n, int64_t ldi, const float* part,
                                                   float2* power, T* out, int64_t ld) {
  __shared__ float red[4];
  float s = 1.f;
  if constexpr (PL == 2) {
    const float2 pw = power_for(block_max(fmaxf(part[threadIdx.x], part[threadIdx.x + 256]), red));
    s = pw.x;
    if (blockIdx.x == 0 && threadIdx.x == 0) *power = pw;
  }
  const int64_t chunks = ld / (8 * PL), total = rows * chunks;
  const bool whole = ldi % 8 == 0 && ((uintptr_t)x & 15) == 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / chunks, c = (i - r * chunks) * 8;
    float v[8];
    const TI* at = x + r * ldi + c;
    if (whole && c + 8 <= n) {
      struct alignas(16) V { TI e[8]; };
      const V t = *(const V*)at;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = to_f(t.e[e]) * s;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < n ? to_f(at[e]) * s : 0.f;
    }
    put_planes<T, PL>(out + r * ld, c, v);
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
  const float2 *px, *pw;  // fp32: the operands' powers
  // the accumulators' first registers take a row's {c, s}
  template <class TL>
  __device__ __forceinline__ void form(const Args& p, const Place& c, typename TL::Acc& acc) const {
    constexpr int TM = TL::TM, TN = TL::TN;
    float ux = 1.f, uw = 1.f;
    if constexpr (TL::PL == 2) { ux = px->y; uw = pw->y; }
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
      m = m > -kInf ? m * kLog2e : -kInf;
      const float ref = m > -kInf ? m : 0.f;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < TN * 16; ++e) s += __builtin_amdgcn_exp2f(fmaf(z[e], kLog2e, -ref));
      s += __shfl_xor(s, 32);
      acc[i][0][0] = m;
      acc[i][0][1] = s;
    }
  }
  template <class TL>
  __device__ __forceinline__ void store(const Args& p, const Place& c, typename TL::T* lds, typename TL::Acc& acc) const {
    float2* pair = (float2*)(lds + TL::STAGE);  // [BM][WN]
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
  constexpr float kLn2 = 0.69314718055994531f;
  float out = 0.f, sum;
  if (target_of(targets, wide, row, V) < 0) {
    sum = (a.x + log2f(a.y)) * kLn2;
  } else {
    // log(exp z_t + the others), from the larger of the two
    const float z = zt[row], q = z * kLog2e;
    if (q >= a.x) {
      out = log1pf(a.y * exp2f(fmaf(-z, kLog2e, a.x)));
      sum = z + out;
    } else {
      const float others = log2f(a.y + exp2f(fmaf(z, kLog2e, -a.x)));
      out = (fmaf(-z, kLog2e, a.x) + others) * kLn2;
      sum = (a.x + others) * kLn2;
    }
  }
  loss[row] = out;
  lse[row] = sum;
}

// ── backward ──────────────────────────────────────────────────────────────
// d of the tile's logits, times the power of the rows' gradients; zeros behind
// the words up to the row's end.  Formed where the accumulators are, from the
// few rows that a lane has.
template <typename T>
struct EpiGrad {
  T* d;
  int64_t ldd;
  int64_t v0, V;  // the piece's first word; all words
  const void* targets;
  bool wide;
  const float *loss, *lse, *g, *h;
  const float2 *px, *pw, *pg;
  template <class TL>
  __device__ __forceinline__ void form(const Args& p, const Place& c, typename TL::Acc& acc) const {
    constexpr int PL = TL::PL, TM = TL::TM, TN = TL::TN;
    float ux = 1.f, uw = 1.f, up = 1.f;
    if constexpr (PL == 2) { ux = px->y; uw = pw->y; }
    if (pg) up = pg->x;
    const int64_t cols = c.n0 + c.wn * 32 * TN;
    const bool ragged = cols + 32 * TN > p.N;
    const int hi = c.lane >> 5;
    float l[TM], all[TM], gr[TM], hr[TM];
    int rel[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int64_t row = c.m0 + TL::row_of(c, i), at = row < p.M ? row : p.M - 1;
      const int64_t t = row < p.M ? target_of(targets, wide, at, V) : -1, far = t - v0 - cols;
      gr[i] = t >= 0 ? g[at] : 0.f;
      hr[i] = h ? h[at] : 0.f;
      all[i] = (gr[i] + hr[i]) * up;
      l[i] = lse[at];
      rel[i] = t >= 0 && far >= 0 && far < 32 * TN && ((far >> 2) & 1) == hi ? (int)far - 4 * hi : -1;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      // a row without weight has no gradient, whatever its logits are
      const bool none = gr[i] == 0.f && hr[i] == 0.f;
      float zt = 0.f;
      if (rel[i] >= 0) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (rel[i] == j * 32 + 8 * (e >> 2) + (e & 3)) zt = acc[i][j][e];
        if constexpr (PL == 2) zt = zt * ux * uw;
      }
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float z = acc[i][j][e];
          if constexpr (PL == 2) z = z * ux * uw;
          acc[i][j][e] = none ? 0.f : exp_fast(z - l[i]) * all[i];
        }
      // p - 1 of the target from its loss, which keeps the digits of 1 - p
      if (rel[i] >= 0 && !none) {
        const float dt = (gr[i] * expm1f(-loss[c.m0 + TL::row_of(c, i)]) + hr[i] * exp_fast(zt - l[i])) * up;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (rel[i] == j * 32 + 8 * (e >> 2) + (e & 3)) acc[i][j][e] = dt;
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
    TL::template runs<false>(
        c, lds, acc, false,
        [&](int64_t row, int64_t col, float (&v)[8]) {
          if (row < p.M && col * PL < ldd) put_planes<T, PL>(d + row * ldd, col, v);
        },
        [](int64_t, int64_t, float (&)[8]) {});
  }
};

// acc times the inverse powers, as outputs or as fp32 parts of a sum.
template <typename TO>
struct EpiOut {
  TO* out;
  float* part;   // [splits][M][N], or null
  bool more;     // parts are added to what is there
  const float2 *pa, *pb;
  template <class TL>
  __device__ __forceinline__ void form(const Args&, const Place&, typename TL::Acc&) const {}
  template <class TL>
  __device__ __forceinline__ void store(const Args& p, const Place& c, typename TL::T* lds, typename TL::Acc& acc) const {
    const float ua = pa ? pa->y : 1.f, ub = pb ? pb->y : 1.f;
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
          constexpr int W = 16 / sizeof(TO);  // a store
          struct V { TO e[W]; } o[8 / W];
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e / W].e[e % W] = from_f<TO>(v[e] * ua * ub);
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

// out = the parts' sum times the inverse powers.
template <typename TO>
__global__ void __launch_bounds__(256) sum_parts_kernel(const float* part, int splits, int64_t n, const float2* pa,
                                                        const float2* pb, TO* out) {
  const float ua = pa ? pa->y : 1.f, ub = pb ? pb->y : 1.f;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  if (i + 4 <= n && n % 4 == 0) {
    float4 a = *(const float4*)(part + i);
    for (int s = 1; s < splits; ++s) {
      const float4 b = *(const float4*)(part + s * n + i);
      a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
    }
    struct V { TO e[4]; } o = {from_f<TO>(a.x * ua * ub), from_f<TO>(a.y * ua * ub), from_f<TO>(a.z * ua * ub),
                               from_f<TO>(a.w * ua * ub)};
    __builtin_memcpy(out + i, &o, sizeof(o));
    return;
  }
  for (int64_t j = i; j < n && j < i + 4; ++j) {
    float a = part[j];
    for (int s = 1; s < splits; ++s) a += part[s * n + j];
    out[j] = from_f<TO>(a * ua * ub);
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

// x [rows, K] as an operand: in place, or packed into the workspace.
struct Packed {
  Operand o;
  float2* power = nullptr;
};
template <typename TI, typename T, int PL>
Packed ready(const void* x, int64_t rows, int64_t K, int64_t ld, Carver& ws, hipStream_t s) {
  Packed r;
  if (PL == 1 && direct(x, ld, K)) {
    r.o = {x, ld, 0};
    return r;
  }
  const int64_t kp = (K + 31) / 32 * 32 * PL;
  T* out = ws.take<T>((size_t)(rows * kp));
  float* part = nullptr;
  if (PL == 2) {
    part = ws.take<float>(kParts);
    r.power = ws.take<float2>(1);
  }
  r.o = {out, kp, 0};
  if (!ws.base) return r;
  if constexpr (PL == 2) {
    hipLaunchKernelGGL(most_kernel, dim3(kParts), dim3(256), 0, s, (const float*)x, rows, K, ld, part);
    check_launch("linear_cross_entropy");
  }
  const int64_t chunks = rows * (kp / (8 * PL));
  const unsigned blocks = (unsigned)std::min<int64_t>(blocks_for(chunks, 256), 4096);
  hipLaunchKernelGGL((pack_kernel<TI, T, PL>), dim3(blocks), dim3(256), 0, s, (const TI*)x, rows, K, ld, part, r.power,
                     out, kp);
  check_launch("linear_cross_entropy");
  return r;
}

// Tiles: 256 x 256 (8 wavefronts), 128 x 128 (4), 32 x 128 (4).
enum { kBig, kMid, kFew };
int pick(int64_t M, int64_t N, int64_t splits, int cus) {
  if (M <= 32) return kFew;
  return ceil_div(M, 256) * ceil_div(N, 256) * splits * 4 >= 3 * cus ? kBig : kMid;
}
int bn_of(int tile) { return tile == kBig ? 256 : 128; }

template <typename T, int PL, bool AC, bool BC, class Epi>
void run(int tile, const Args& p, const Epi& e, hipStream_t s, const char* what) {
  if (tile == kBig) launch<Tile<T, 4, 2, 2, 4, PL, AC, BC>>(p, e, s, what);
  else if (tile == kMid) launch<Tile<T, 2, 2, 2, 2, PL, AC, BC>>(p, e, s, what);
  else launch<Tile<T, 1, 1, 1, 4, PL, AC, BC>>(p, e, s, what);
}

template <typename TI, typename T, int PL>
size_t forward(const LinearCE& a, void* wsp, int cus, hipStream_t s) {
  const char* what = "linear_cross_entropy";
  Carver ws{(char*)wsp};
  const Packed x = ready<TI, T, PL>(a.x, a.R, a.K, a.ldx, ws, s), w = ready<TI, T, PL>(a.w, a.V, a.K, a.ldw, ws, s);
  const int tile = pick(a.R, a.V, 1, cus);
  const int64_t parts = ceil_div(a.V, bn_of(tile));
  float2* part = ws.take<float2>((size_t)(parts * a.R));
  float* zt = ws.take<float>((size_t)a.R);
  if (!wsp) return ws.used;
  Args p;
  p.a = x.o; p.b = w.o;
  p.M = a.R; p.N = a.V; p.K = a.K;
  const bool wide = a.idx_dt == DType::I64;
  run<T, PL, false, false>(tile, p, EpiLoss{part, zt, a.targets, wide, x.power, w.power}, s, what);
  const int rx = a.R >= 64 * cus ? 64 : a.R >= 16 * cus ? 16 : a.R >= 4 * cus ? 4 : 1;
  hipLaunchKernelGGL(loss_kernel, dim3(blocks_for(a.R, rx)), dim3(256), 0, s, part, parts, zt, a.targets, wide, a.R,
                     a.V, rx, a.loss, a.lse);
  check_launch(what);
  return ws.used;
}

// Values of d that are held at once: 2^29 (1 GB of 16 bits).
constexpr int64_t kHeld = (int64_t)1 << 29;

// Parts of dx's sum over the words, with the blocks of dw beside them: the
// least of what a compute unit has to do, in stages of 64 k (a block's start
// and end count as 4, half of a last block's length as waiting, a part's
// writing and reading back by its bytes).
int dx_parts(int64_t xtiles, int64_t stages, int64_t wtiles, int64_t wstages, int64_t values, int slots) {
  int best = 1;
  double least = 1e300;
  for (int s = 1; s <= 64 && s * 4 <= std::max<int64_t>(stages, 4); ++s) {
    const double len = (double)ceil_div(stages, s) + 4, last = std::min<double>(len, (double)wstages + 4);
    const double work = ((double)xtiles * s * len + (double)wtiles * ((double)wstages + 4)) / slots;
    const double t = std::max(work, len) + 0.5 * last + (s > 1 ? s * (double)values * 8 / 8e6 : 0);
    if (t < least) {
      least = t;
      best = s;
    }
  }
  return best;
}

template <typename TI, typename T, int PL>
size_t backward(const LinearCE& a, void* wsp, int cus, hipStream_t s) {
  const char* what = "linear_cross_entropy_backward";
  Carver ws{(char*)wsp};
  const Packed x = ready<TI, T, PL>(a.x, a.R, a.K, a.ldx, ws, s), w = ready<TI, T, PL>(a.w, a.V, a.K, a.ldw, ws, s);
  const bool wide = a.idx_dt == DType::I64;
  // pieces of the vocabulary, whole tiles of it
  const int64_t most = std::min<int64_t>(std::max<int64_t>(kHeld / PL / a.R / 256 * 256, 256), 1 << 19);
  const int64_t pieces = ceil_div(a.V, most), each = ceil_div(ceil_div(a.V, pieces), 256) * 256;
  const int64_t len = std::min(each, a.V), ldd = (len + 31) / 32 * 32 * PL;
  T* d = ws.take<T>((size_t)(a.R * ldd));
  constexpr bool scaled = !std::is_same<T, bf16_t>::value;
  float2* pg = scaled ? ws.take<float2>(1) : nullptr;
  // both products of a piece in one launch: large tiles where they fill the
  // chip at one block a compute unit
  const bool big = a.R > 32 && ceil_div(len, 256) * ceil_div(a.K, 256) >= cus / 2;
  const int64_t b = big ? 256 : 128, xb = a.R <= 32 ? 32 : b;
  const int splits = dx_parts(ceil_div(a.R, xb) * ceil_div(a.K, b), ceil_div(len, 64 / PL),
                              ceil_div(len, b) * ceil_div(a.K, b), ceil_div(a.R, 64 / PL), a.R * a.K, big ? cus : 2 * cus);
  const bool parted = splits > 1 || pieces > 1;
  float* part = parted ? ws.take<float>((size_t)(splits * a.R * a.K)) : nullptr;
  if (!wsp) return ws.used;
  if (scaled) {
    hipLaunchKernelGGL(grad_power_kernel, dim3(1), dim3(1024), 0, s, a.g_loss, a.g_lse, a.R, pg);
    check_launch(what);
  }
  for (int64_t v0 = 0; v0 < a.V; v0 += each) {
    const int64_t n = std::min(each, a.V - v0);
    const Operand wp{(const T*)w.o.p + v0 * w.o.ld, w.o.ld, 0}, dp{d, ldd, 0};
    Args p;
    p.a = x.o; p.b = wp;
    p.M = a.R; p.N = n; p.K = a.K;
    run<T, PL, false, false>(pick(a.R, n, 1, cus), p,
                             EpiGrad<T>{d, ldd, v0, a.V, a.targets, wide, a.loss, a.lse, a.g_loss, a.g_lse, x.power,
                                        w.power, pg}, s, what);
    Args px, pw;
    px.a = pw.a = dp;
    px.b = wp;
    px.M = a.R; px.N = a.K; px.K = n; px.splits = splits;
    pw.b = x.o;
    pw.M = n; pw.N = a.K; pw.K = a.R;
    const EpiOut<TI> ex{(TI*)a.dx, part, v0 > 0, pg, w.power}, ew{(TI*)a.dw + v0 * a.K, nullptr, false, pg, x.power};
    typedef Tile<T, 2, 2, 2, 2, PL, true, true> WMid;
    if (big)
      launch_pair<Tile<T, 4, 2, 2, 4, PL, false, true>, Tile<T, 4, 2, 2, 4, PL, true, true>>(px, ex, pw, ew, s, what);
    else if (a.R > 32)
      launch_pair<Tile<T, 2, 2, 2, 2, PL, false, true>, WMid>(px, ex, pw, ew, s, what);
    else
      launch_pair<Tile<T, 1, 1, 1, 4, PL, false, true>, WMid>(px, ex, pw, ew, s, what);
  }
  if (parted) {
    const int64_t n = a.R * a.K;
    hipLaunchKernelGGL((sum_parts_kernel<TI>), dim3(blocks_for(n, 1024)), dim3(256), 0, s, part, splits, n, pg, w.power,
                       (TI*)a.dx);
    check_launch(what);
  }
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
