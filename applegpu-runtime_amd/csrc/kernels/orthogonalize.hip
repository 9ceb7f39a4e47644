// Orthogonalised updates by Newton-Schulz products:
//
//   X = U / (|U|_F + eps);  five times  A = X X^T,  X = a X + (b A + c A A) X
//
// which takes every singular value of X towards 1 (a matrix taller than wide
// works with X^T X instead, from the other side).  A step is three products:
//   gram    A = X X^T          symmetric: tiles on and below the diagonal,
//                              each stored as its mirror image too
//   poly    B = b A + c A A    symmetric too (A's rows are its columns)
//   update  X = a X + B X      X read as columns, so no transpose is kept
// with one launch each for all matrices of a batch (two, where tiles are cut).
//
// Precision: products are of fp16 with fp32 sums, of one plane or of two (22
// bits), see planes_of.  With singular values s of X below 1.2 the entries of X
// and A stay below 1.2 and 1.5, those of B below 2.81 (b s^2 + c s^4 is -b^2 / 4c
// at most in size, at s = 1.08): X, A and B are held times 2^14, where fp16 ends
// at 4.0 and keeps 11 bits of everything down to 2^-28.  X itself
// keeps more beside its planes, 22 bits for 16-bit matrices and fp32 for fp32
// ones: a X is what carries the small singular values, multiplied by 3.4 in
// each step, and would carry a rounding of X along (256 x 512 of rank 8 and 3 %
// noise: relative error 9.5e-3 with X in 11 bits, 3.8e-4 in 22); what fp16 loses
// of X inside B X is B's small share of that direction.
#include "tile16.hpp"

namespace agpu {
namespace k {
using namespace dev;
using namespace t16;

namespace {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kUnit = 16384.f, kPerUnit = 1.f / 16384.f;

template <typename T>
__device__ __forceinline__ T* mat(const Mats& t, int64_t i) {
  return t.apart ? (T*)t.p[0] + i * t.apart : (T*)t.p[i];
}

// 8 values or the first n of them, at any alignment.
template <typename E>
struct Run { E e[8]; };
template <typename E>
__device__ __forceinline__ Run<E> get_run(const E* at, int n) {
  Run<E> r{};
  if (n >= 8) __builtin_memcpy(&r, at, sizeof(r));
  else
    for (int e = 0; e < 8; ++e)
      if (e < n) r.e[e] = at[e];
  return r;
}
template <typename E>
__device__ __forceinline__ void put_run(E* at, const Run<E>& r, int n) {
  if (n >= 8) {
    struct Half { E e[4]; } h[2];
    __builtin_memcpy(h, &r, sizeof(r));
    if constexpr (sizeof(E) == 4) {
      put_past(at, h[0]);
      put_past(at + 4, h[1]);
    } else {
      put_past(at, r);
    }
  } else {
    for (int e = 0; e < 8; ++e)
      if (e < n) at[e] = r.e[e];
  }
}

// U times `pre` over `by` is X: |U| + eps, from the sum of U's squares, and a
// power of two where that has no float32 or few bits of one.
struct Norm {
  float pre, by;
};
__device__ __forceinline__ Norm norm_of(double squares, float eps) {
  const double root = sqrt(squares);
  const float norm = (float)root + eps;
  Norm n{1.f, norm > 0.f || norm != norm ? norm : 1.f};  // a matrix of zeros stays one
  if (norm > 0.f && norm < 0x1p-100f) n.pre = 0x1p64f;
  else if (norm == __builtin_inff() && root < __builtin_inf()) n.pre = 0x1p-64f;
  if (n.pre != 1.f) n.by = (float)((root + (double)eps) * (double)n.pre);
  return n;
}

constexpr int kNormParts = 128;  // blocks a matrix for its norm

// Of matrix blockIdx.y: the sum of U's squares in kNormParts parts, and with
// momentum the new momentum.  Four runs' loads are under way at a time.
template <typename TI, bool MOM>
__global__ void __launch_bounds__(256) norm_kernel(Mats in, Mats mom, float beta, bool nesterov, int64_t n, double* part) {
  __shared__ double red[4];
  const int64_t i = blockIdx.y;
  const TI* __restrict__ g = mat<TI>(in, i);
  float* __restrict__ b = MOM ? mat<float>(mom, i) : nullptr;
  constexpr int kAtOnce = 4;
  double sum = 0.0;
  const int64_t apart = (int64_t)kNormParts * 256 * 8;
  for (int64_t j0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; j0 < n; j0 += apart * kAtOnce) {
    Run<TI> gv[kAtOnce];
    Run<float> bv[kAtOnce];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      const int64_t j = j0 + q * apart, left = n - j;
      const int m = left < 0 ? 0 : left < 8 ? (int)left : 8;
      gv[q] = get_run(g + j, m);
      if constexpr (MOM) bv[q] = get_run(b + j, m);
    }
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      const int64_t j = j0 + q * apart, left = n - j;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = to_f(gv[q].e[e]);
        if constexpr (MOM) {
          const float m = beta * bv[q].e[e] + v;
          bv[q].e[e] = m;
          v = nesterov ? v + beta * m : m;
        }
        sum += (double)v * (double)v;  // (nothing where nothing was read)
      }
      if constexpr (MOM)
        if (left > 0) put_run(b + j, bv[q], left < 8 ? (int)left : 8);
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) part[i * kNormParts + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// What X keeps beside the planes of a step's factor, in units of 2^-14: fp32
// (F32), or with one plane the low half, rows as long as the plane's.
struct Kept {
  float* x = nullptr;     // [count][m][n]
  half_t* low = nullptr;  // [count][m][ld]
};

// X = U / (|U| + eps) and its planes, rows of ld values.
template <typename TI, bool MOM, int PL>
__global__ void __launch_bounds__(256) start_kernel(Mats in, Mats mom, float beta, bool nesterov, int64_t m, int64_t n,
                                                   const double* part, float eps, Kept keep, half_t* planes, int64_t ld) {
  constexpr bool F32 = sizeof(TI) == 4;
  __shared__ double red[2];
  const int64_t i = blockIdx.y;
  const TI* __restrict__ g = mat<TI>(in, i);
  const float* __restrict__ b = MOM ? mat<float>(mom, i) : nullptr;
  if (threadIdx.x < kNormParts) {
    double s = part[i * kNormParts + threadIdx.x];
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) s += __shfl_xor(s, k);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  }
  __syncthreads();
  const Norm norm = norm_of(red[0] + red[1], eps);
  const int chunks = (int)(ld / (8 * PL));
  constexpr int kAtOnce = 2;
  const int64_t total = m * chunks, apart = (int64_t)gridDim.x * 256;
  for (int64_t t0 = (int64_t)blockIdx.x * 256 + threadIdx.x; t0 < total; t0 += apart * kAtOnce) {
    Run<TI> gv[kAtOnce];
    Run<float> bv[kAtOnce];
    int64_t row[kAtOnce];
    int col[kAtOnce], len[kAtOnce];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      const int64_t t = t0 + q * apart;
      row[q] = t < total ? t / chunks : -1;
      col[q] = (int)(t - row[q] * chunks) * 8;
      const int64_t left = n - col[q];
      len[q] = row[q] < 0 || left < 0 ? 0 : left < 8 ? (int)left : 8;
      gv[q] = get_run(g + row[q] * n + col[q], len[q]);
      if constexpr (MOM) bv[q] = get_run(b + row[q] * n + col[q], len[q]);
    }
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      if (row[q] < 0) continue;
      const int64_t r = i * m + row[q];
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float u = to_f(gv[q].e[e]);
        if constexpr (MOM) u = nesterov ? u + beta * bv[q].e[e] : bv[q].e[e];
        v[e] = u * norm.pre / norm.by * kUnit;
      }
      put_planes<half_t, PL>(planes + r * ld, col[q], v);
      if constexpr (F32) {
        Run<float> x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x.e[e] = v[e];
        put_run(keep.x + r * n + col[q], x, len[q]);
      } else if constexpr (PL == 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] -= (float)(half_t)v[e];
        put_planes<half_t, 1>(keep.low + r * ld, col[q], v);
      }
    }
  }
}

// A (or B = b A + c A A) of a tile, and its mirror image.
template <bool POLY>
struct EpiGram {
  static constexpr bool kFull = false;
  const half_t* a;  // POLY
  half_t* out;
  int64_t ld, batch;  // rows ld apart, matrices batch apart
  template <class TL>
  __device__ __forceinline__ void form(const Args& p, const Place& c, typename TL::Acc& acc) const {
    constexpr int PL = TL::PL;
    typedef typename TL::template Places<half_t, PL> From;
    const From from(c, POLY ? a + c.batch * batch : out, ld, p.M);
    // zeros behind the matrix, where what was summed is not
    const bool whole = c.m0 + TL::BM <= p.M && c.n0 + TL::BN <= p.N;
    const int rows = (int)(p.M - c.m0), cols = (int)(p.N - c.n0);
    TL::fours(acc, [&](int i, int j, int g, float (&v)[4]) {
      float t[4] = {};
      if constexpr (POLY) {
        from.load(i, j, g, t);
        if constexpr (PL == 2) {
          float l[4];
          from.load(i, j, g, l, 1);
#pragma unroll
          for (int e = 0; e < 4; ++e) t[e] += l[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float s = v[e] * kPerUnit;
        v[e] = POLY ? kB * t[e] + kC * s : s;
        if (!whole && (TL::row_of(c, i) >= rows || TL::col_of(c, j, 4 * g + e) >= cols)) v[e] = 0.f;
      }
    });
  }
  template <class TL>
  __device__ __forceinline__ void store(const Args& p, const Place& c, typename TL::T* lds, typename TL::Acc& acc) const {
    constexpr int PL = TL::PL;
    half_t* to = out + c.batch * batch;
    auto put = [&](int64_t r, int64_t q, float (&v)[8]) {
      if (r < p.M && q * PL < ld) put_planes<half_t, PL>(to + r * ld, q, v);
    };
    TL::template runs<true>(
        c, lds, acc, c.tm != c.tn, [&](int64_t row, int64_t col, float (&v)[8]) { put(row, col, v); },
        [&](int64_t row, int64_t col, float (&v)[8]) { put(col, row, v); });
  }
};

// X = a X + B X, as the next step's NEXT planes and what is kept beside them;
// after the last step (NEXT = 0) the result instead.  X is read where the
// accumulators are, eight loads under way at a time (a load and its use after
// one another, run by run, took 18 us more a tile of 256 x 256); fp32 X and
// the weights run by run where a tile reaches past the columns or their rows
// are not aligned.
template <typename TO, bool F32, int NEXT>
struct EpiUpdate {
  static constexpr bool kFull = false;
  const half_t* from;  // the step's planes, rows ld apart
  int64_t ld;
  Kept keep;
  half_t* planes;      // the next step's, rows ld_next apart
  int64_t ld_next;
  Mats out;
  bool step;           // out = keep out - rate X
  float hold, rate;
  __device__ __forceinline__ float result(float v, float was) const {
    const float s = v * kPerUnit;
    return step ? hold * was - rate * s : s;
  }
  template <class TL>
  __device__ __forceinline__ bool near(const Args& p, const Place& c) const {
    return c.n0 + TL::BN <= p.N && p.N % 4 == 0 &&
           (NEXT != 0 || ((uintptr_t)mat<TO>(out, c.batch) % (4 * sizeof(TO))) == 0);
  }
  template <class TL>
  __device__ __forceinline__ void form(const Args& p, const Place& c, typename TL::Acc& acc) const {
    constexpr int PL = TL::PL;
    if constexpr (F32) {
      if (!near<TL>(p, c)) return;
    }
    const bool weights = NEXT == 0 && step && near<TL>(p, c);
    const int64_t b = c.batch;
    const TO* o = NEXT ? nullptr : mat<TO>(out, b);
    const typename TL::template Places<float> xs(c, F32 ? keep.x + b * p.M * p.N : nullptr, p.N, F32 ? p.M : c.m0);
    const typename TL::template Places<half_t, PL> hs(c, from + b * p.M * ld, ld, p.M);
    const typename TL::template Places<half_t> ls(c, PL == 1 && !F32 ? keep.low + b * p.M * ld : from, ld, p.M);
    const typename TL::template Places<TO> os(c, NEXT ? (const TO*)from : o, p.N, weights ? p.M : c.m0);
    TL::fours(acc, [&](int i, int j, int g, float (&v)[4]) {
      float t[4];
      if constexpr (F32) {
        xs.load(i, j, g, t);
      } else {
        float l[4];
        hs.load(i, j, g, t);
        if constexpr (PL == 2) hs.load(i, j, g, l, 1);
        else ls.load(i, j, g, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] += l[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = kA * t[e] + v[e] * kPerUnit;
      if constexpr (NEXT == 0) {
        if (weights) {
          os.load(i, j, g, t);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = result(v[e], t[e]);
        } else if (!step) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = result(v[e], 0.f);
        }
      }
    });
  }
  template <class TL>
  __device__ __forceinline__ void store(const Args& p, const Place& c, typename TL::T* lds, typename TL::Acc& acc) const {
    float* xb = F32 ? keep.x + (int64_t)c.batch * p.M * p.N : nullptr;
    TO* o = NEXT ? nullptr : mat<TO>(out, c.batch);
    const bool close = near<TL>(p, c), ragged = c.n0 + TL::BN > p.N;
    TL::template runs<false>(
        c, lds, acc, false,
        [&](int64_t row, int64_t col, float (&v)[8]) {
          if (row >= p.M || (col >= p.N && (NEXT == 0 || col * NEXT >= ld_next))) return;
          // (none behind the columns, where planes hold zeros)
          const int n = p.N - col < 8 ? (int)(p.N - col) : 8;
          const int64_t at = row * p.N + col;
          if constexpr (F32) {
            if (!close) {
              const Run<float> t = get_run(xb + at, n);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = kA * t.e[e] + v[e] * kPerUnit;
              if constexpr (NEXT == 0)
                if (!step)
#pragma unroll
                  for (int e = 0; e < 8; ++e) v[e] = result(v[e], 0.f);
            }
          }
          if constexpr (NEXT != 0) {
            if (ragged) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = e < n ? v[e] : 0.f;
            }
            const int64_t r = (int64_t)c.batch * p.M + row;
            put_planes<half_t, NEXT>(planes + r * ld_next, col, v);
            if constexpr (F32) {
              Run<float> x;
#pragma unroll
              for (int e = 0; e < 8; ++e) x.e[e] = v[e];
              put_run(xb + at, x, n);
            } else if constexpr (NEXT == 1) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] -= (float)(half_t)v[e];
              put_planes<half_t, 1>(keep.low + r * ld_next, col, v);
            }
          } else {
            if (step && !close) {
              const Run<TO> w = get_run(o + at, n);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = result(v[e], to_f(w.e[e]));
            }
            Run<TO> q;
#pragma unroll
            for (int e = 0; e < 8; ++e) q.e[e] = from_f<TO>(v[e]);
            put_run(o + at, q, n);
          }
        },
        [](int64_t, int64_t, float (&)[8]) {});
  }
};

// Square tiles of 256 (one block a compute unit), 128 (both 8 wavefronts) or 64
// (4).  Large ones where they fill whole rounds of the chip, else the next size
// that makes enough blocks.  Gram, poly (both uncut) and update in us, 256 / 128
// / 64:
//   2 x 4096 x 4096 fp32      526/419/572  520/393/575  635/692/889  (272 and 512 tiles of 256)
//   12 x 768 x 2304           56/28/30     32/13/14     83/66/74
//   12 x 768 x 768            28/12/13     33/14/14     41/25/28
//   1280 x 1280               36/14/9.5    42/15/10     50/20/16
//   200 x 400                 22/9/6       18/7.5/5.4   20/8.4/5.5
enum { kBig, kMid, kSmall };
int pick(int64_t M, int64_t N, int64_t count, int cus) {
  const int64_t big = ceil_div(M, 256) * ceil_div(N, 256) * count;
  if (big * 10 >= ceil_div(big, cus) * cus * 9) return kBig;
  return ceil_div(M, 128) * ceil_div(N, 128) * count * 8 >= 5 * cus ? kMid : kSmall;
}

// The same of a symmetric product, whose tiles behind the last whole round of
// the chip may be cut along k, their parts joined by a launch of its own.  By
// the time its rounds take, in us: a stage 1.75 in tiles of 256 and 0.95 in
// tiles of 128 (two planes: 2 and 1.3), 0.4 in tiles of 64 (0.5), of which four
// blocks share a compute unit and which small products take; a block's start and
// end 4 stages, the parts' way through memory at 4 TB/s.  Blocks alone on their compute unit are
// faster than that, so a cut has to win by 15 %.  Whole / cut, us:
//   2 x 4096 x 4096 fp32              435 / 372 + 13   (256 tiles of 256 and 16 in 12 parts)
//   4 x 1280 x 1280 over 5120 fp16    81 / 63 + 10     (220 tiles of 128 in 2 parts)
//   of two planes                     162 / 121 + 17   (60 tiles of 256 in 4)
//   4 x 1280 x 1280 over 1280 of two  49 / 40 + 15     (not cut)
// and all launches of a matrix in tiles of 64, bf16: 64 x 4096 211 / 118, 768 x
// 2304 273 / 217, 16 x 100000 3844 / 320; fp32: 340 / 159, 480 / 321, 7976 / 364.
struct Cut {
  int tile;
  int splits;     // of the tiles from `whole` on
  int64_t whole;
  size_t bytes;   // of their parts
};
Cut cut(int64_t side, int64_t k, int64_t count, int planes, int cus) {
  auto tiles = [&](int64_t b) {
    const int64_t m = ceil_div(side, b);
    return m * (m + 1) / 2 * count;
  };
  const bool few = tiles(128) * 8 < 5 * cus;
  const int64_t stages = ceil_div(k, 64 / planes);
  Cut best{};
  double least = 1e300;
  for (int tile : {kBig, kMid, kSmall}) {
    if (few != (tile == kSmall)) continue;
    const int64_t b = tile == kBig ? 256 : tile == kMid ? 128 : 64, all = tiles(b);
    const int64_t slots = (tile == kBig ? 1 : tile == kMid ? 2 : 4) * cus;
    static const double kStage[2][3] = {{1.75, 0.95, 0.4}, {2.0, 1.3, 0.5}};
    const double stage = kStage[planes - 1][tile];
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
      if (s > 1 && s * 4 > stages) break;
      const int64_t whole = s > 1 ? all / slots * slots : all, rest = all - whole;
      const size_t bytes = (size_t)(rest * s * b * b * 4);
      const double t = ((double)ceil_div(whole, slots) * (double)(stages + 4) +
                        (double)ceil_div(rest * s, slots) * (double)(ceil_div(stages, s) + 4)) * stage +
                       (rest ? 6 + (double)bytes * 2 / 4e6 : 0);
      if (t * (rest ? 1.15 : 1.0) < least) {
        least = t * (rest ? 1.15 : 1.0);
        best = {tile, s, whole, bytes};
      }
    }
  }
  return best;
}

template <int PL, Layout AL, Layout BL, class Epi>
void run(int tile, const Args& p, const Epi& e, hipStream_t s, const char* what) {
  if (tile == kBig) launch<Tile<half_t, 4, 2, 2, 4, PL, AL, BL>>(p, e, s, what);
  else if (tile == kMid) launch<Tile<half_t, 2, 1, 2, 4, PL, AL, BL>>(p, e, s, what);
  else launch<Tile<half_t, 1, 1, 2, 2, PL, AL, BL>>(p, e, s, what);
}
template <int PL, Layout L, class Epi>
void run_symmetric(const Cut& c, const Args& p, const Epi& e, float* part, hipStream_t s, const char* what) {
  typedef Tile<half_t, 1, 1, 2, 2, PL, kRows, kRows, true> Join;
  if (c.tile == kBig) launch_tail<Tile<half_t, 4, 2, 2, 4, PL, L, L, true>, Join>(p, e, c.whole, c.splits, part, s, what);
  else if (c.tile == kMid) launch_tail<Tile<half_t, 2, 1, 2, 4, PL, L, L, true>, Join>(p, e, c.whole, c.splits, part, s, what);
  else launch_tail<Tile<half_t, 1, 1, 2, 2, PL, L, L, true>, Join>(p, e, c.whole, c.splits, part, s, what);
}

// fp16 planes of a step's factors.  What a step rounds is passed on by the
// steps behind it, so the last ones set the result's error: relative to the
// result (160 x 640 with a few strong directions, oracle with roundings) 1.4e-3
// with one plane throughout, 1.2e-4 with two in the last three steps, 1e-6 with
// two throughout.  Against the rounding of the result itself, 1.7e-3 in bf16,
// 2.1e-4 in fp16 and 3e-8 in fp32, that is one plane, two in the last three
// steps, and two.  Matrices of a short side take two in fp16 throughout: their
// error is larger (64 x 128: 2.5e-4) and their time is the launches'.
int planes_of(const Orthogonalize& a, int step) {
  if (a.dt == DType::F32) return 2;
  if (a.dt == DType::BF16) return 1;
  return step + 3 >= a.steps || std::min(a.m, a.n) <= 256 ? 2 : 1;
}
int64_t row_of(int64_t n, int planes) { return (n + 31) / 32 * 32 * planes; }

struct Space {
  double* part;
  Kept keep;
  half_t *planes[2], *a, *b;
  float* split;
  size_t bytes;
};
Space space(const Orthogonalize& a, int cus, char* base) {
  Space w;
  size_t used = 0;
  auto take = [&](size_t n) {
    char* at = base ? base + used : nullptr;
    used += (n + 255) / 256 * 256;
    return at;
  };
  const int pl = planes_of(a, a.steps - 1);  // the most of all steps
  const int64_t side = std::min(a.m, a.n);
  w.part = (double*)take((size_t)a.count * kNormParts * 8);
  if (a.dt == DType::F32) w.keep.x = (float*)take((size_t)(a.count * a.m * a.n) * 4);
  else if (planes_of(a, 0) == 1) w.keep.low = (half_t*)take((size_t)(a.count * a.m * row_of(a.n, 1)) * 2);
  for (auto& q : w.planes) q = (half_t*)take((size_t)(a.count * a.m * row_of(a.n, pl)) * 2);
  w.a = (half_t*)take((size_t)(a.count * side * row_of(side, pl)) * 2);
  w.b = (half_t*)take((size_t)(a.count * side * row_of(side, pl)) * 2);
  size_t split = 0;
  for (int planes : {planes_of(a, 0), pl})
    for (int64_t k : {std::max(a.m, a.n), side}) split = std::max(split, cut(side, k, a.count, planes, cus).bytes);
  w.split = (float*)take(split);
  w.bytes = used;
  return w;
}

template <typename TI, bool MOM>
void start(const Orthogonalize& a, const Space& w, hipStream_t s, const char* what) {
  hipLaunchKernelGGL((norm_kernel<TI, MOM>), dim3(kNormParts, (unsigned)a.count), dim3(256), 0, s, a.in, a.mom, a.beta,
                     a.nesterov, a.m * a.n, w.part);
  check_launch(what);
  const int pl = planes_of(a, 0);
  const int64_t ld = row_of(a.n, pl);
  const dim3 grid((unsigned)std::min<int64_t>(blocks_for(a.m * (ld / (8 * pl)), 512), 512), (unsigned)a.count);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a.in, a.mom, a.beta, a.nesterov, a.m, a.n, w.part, a.eps, w.keep,
                       w.planes[0], ld);
  };
  if constexpr (sizeof(TI) == 4) go(start_kernel<TI, MOM, 2>);
  else pl == 1 ? go(start_kernel<TI, MOM, 1>) : go(start_kernel<TI, MOM, 2>);
  check_launch(what);
}

// Step i on PL planes, the next on NEXT (0: none follows).
template <typename TO, bool F32, int PL, int NEXT>
void step(const Orthogonalize& a, const Space& w, int i, int cus, hipStream_t s, const char* what) {
  const int64_t m = a.m, n = a.n, side = std::min(m, n), ld = row_of(n, PL), lda = row_of(side, PL);
  const bool tall = m > n;
  const int upd = pick(m, n, a.count, cus);
  const Operand xo{w.planes[i & 1], ld, m * ld}, ao{w.a, lda, side * lda}, bo{w.b, lda, side * lda};
  Args p;
  p.batches = (int)a.count;
  p.a = p.b = xo;
  p.M = p.N = side;
  p.K = tall ? m : n;
  const EpiGram<false> eg{nullptr, w.a, lda, side * lda};
  const Cut gram = cut(side, p.K, a.count, PL, cus);
  if (tall) run_symmetric<PL, kCols>(gram, p, eg, w.split, s, what);
  else run_symmetric<PL, kRows>(gram, p, eg, w.split, s, what);
  p.a = p.b = ao;
  p.K = side;
  run_symmetric<PL, kRows>(cut(side, side, a.count, PL, cus), p, EpiGram<true>{w.a, w.b, lda, side * lda}, w.split, s,
                           what);
  p.M = m;
  p.N = n;
  p.a = tall ? xo : bo;
  p.b = tall ? bo : xo;
  const EpiUpdate<TO, F32, NEXT> eu{w.planes[i & 1], ld, w.keep, w.planes[(i + 1) & 1], row_of(n, NEXT), a.out,
                                    a.momentum, a.keep, a.rate};
  if (tall) run<PL, kRows, kRows>(upd, p, eu, s, what);
  else run<PL, kRows, kCols>(upd, p, eu, s, what);
}

// ── small matrices: everything in one block ───────────────────────────────
// A matrix of at most kSmallValues values (sides rounded up to 32), the shorter
// side at most 128, stays in one block's LDS and registers from its norm to its
// result: one launch where the products of a step would be three of 4.5 us each
// (128 x 64 fp32, five steps: 73 us, so 27).  X and the Gram matrix (then the
// polynomial in its place) are two fp16 planes each; a wavefront holds two 32 x
// 32 tiles of X in fp32.
constexpr int kSmallValues = 16384, kSmallWaves = 8;

// Rows of a plane in LDS, 8 values apart from being multiples of 32: a
// fragment's 16 rows lie in different banks.
struct Flat {
  half_t *high, *low;
  int ld;
};
typedef typename Mfma<half_t>::vec H8;
template <bool COLS>
__device__ __forceinline__ H8 flat_read(const half_t* plane, int ld, int blk, int kk, int lane) {
  if constexpr (COLS) {
    const int i = lane & 15, k = kk * 16 + 8 * (lane >> 5) + (i >> 2);
    const half_t* at = plane + k * ld + blk * 32 + (lane & 16) + 4 * (i & 3);
    union {
      i16x4 h[2];
      H8 v;
    } u;
    u.h[0] = read_transposed((lds_i16x4)at);
    u.h[1] = read_transposed((lds_i16x4)(at + 4 * ld));
    return u.v;
  } else {
    return *(const H8*)(plane + (blk * 32 + (lane & 31)) * ld + kk * 16 + 8 * (lane >> 5));
  }
}
// Tile (ra, rb) of the product over k: rows of a, columns of b.
template <bool AC, bool BC>
__device__ __forceinline__ f32x16 flat_product(const Flat& a, int ra, const Flat& b, int rb, int k, int lane) {
  f32x16 high, cross;
#pragma unroll
  for (int e = 0; e < 16; ++e) high[e] = cross[e] = 0.f;
  // the next step's fragments are read meanwhile
  H8 f[2][4];
  auto read = [&](int set, int kk) __attribute__((always_inline)) {
    f[set][0] = flat_read<AC>(a.high, a.ld, ra, kk, lane);
    f[set][1] = flat_read<AC>(a.low, a.ld, ra, kk, lane);
    f[set][2] = flat_read<BC>(b.high, b.ld, rb, kk, lane);
    f[set][3] = flat_read<BC>(b.low, b.ld, rb, kk, lane);
  };
  auto mul = [&](int set) __attribute__((always_inline)) {
    high = Mfma<half_t>::run(f[set][2], f[set][0], high);
    cross = Mfma<half_t>::run(f[set][3], f[set][0], cross);
    cross = Mfma<half_t>::run(f[set][2], f[set][1], cross);
  };
  read(0, 0);
  for (int kk = 0; kk < k / 16; kk += 2) {  // (an even number of steps)
    read(1, kk + 1);
    mul(0);
    if (kk + 2 < k / 16) read(0, kk + 2);
    mul(1);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) high[e] += cross[e];
  return high;
}
// 4 values of a row as planes.
__device__ __forceinline__ void flat_put(const Flat& f, int row, int col, const float (&v)[4]) {
  typedef _Float16 h4 __attribute__((ext_vector_type(4)));
  h4 h, l;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = (_Float16)v[e];
    l[e] = (_Float16)(v[e] - (float)h[e]);
  }
  *(h4*)(f.high + row * f.ld + col) = h;
  *(h4*)(f.low + row * f.ld + col) = l;
}
__device__ __forceinline__ void flat_get(const Flat& f, int row, int col, float (&v)[4]) {
  typedef _Float16 h4 __attribute__((ext_vector_type(4)));
  const h4 h = *(const h4*)(f.high + row * f.ld + col), l = *(const h4*)(f.low + row * f.ld + col);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (float)h[e] + (float)l[e];
}

template <typename TI, bool MOM, bool TALL>
__global__ void __launch_bounds__(64 * kSmallWaves, 2) small_kernel(Orthogonalize a) {
  __shared__ __attribute__((aligned(16))) half_t lds[69632];  // 2 x 128 x 136 of X and of A
  __shared__ double red[kSmallWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = (int)a.m, n = (int)a.n, mp = (m + 31) & ~31, np = (n + 31) & ~31, side = TALL ? np : mp;
  const Flat x{lds, lds + mp * (np + 8), np + 8};
  const Flat g{lds + 2 * mp * (np + 8), lds + 2 * mp * (np + 8) + side * (side + 8), side + 8};
  const TI* in = mat<TI>(a.in, blockIdx.x);
  const int xt = np / 32, xtiles = mp / 32 * xt, gt = side / 32;
  // this lane's places of tile t (of `wide` tiles a row): row, and column of 4
  // values for each i
  auto row_at = [&](int t, int wide) { return t / wide * 32 + (lane & 31); };
  auto col_at = [&](int t, int wide, int i) { return t % wide * 32 + 8 * i + 4 * (lane >> 5); };
  float v[2][16];
  double sum = 0.0;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int t = wave + kSmallWaves * q;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      v[q][e] = 0.f;
      const int r = row_at(t, xt), c = col_at(t, xt, e >> 2) + (e & 3);
      if (t < xtiles && r < m && c < n) {
        float u = to_f(in[r * n + c]);
        if constexpr (MOM) {
          float* b = mat<float>(a.mom, blockIdx.x) + r * n + c;
          const float mv = a.beta * *b + u;
          *b = mv;
          u = a.nesterov ? u + a.beta * mv : mv;
        }
        v[q][e] = u;
        sum += (double)u * (double)u;
      }
    }
  }
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) sum += __shfl_xor(sum, k);
  if (lane == 0) red[wave] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int w = 0; w < kSmallWaves; ++w) sum += red[w];
  const Norm norm = norm_of(sum, a.eps);
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int e = 0; e < 16; ++e) v[q][e] = v[q][e] * norm.pre / norm.by * kUnit;
  auto put = [&](const Flat& f, const float (&w)[16], int t, int wide) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p[4] = {w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
      flat_put(f, row_at(t, wide), col_at(t, wide, i), p);
    }
  };
#pragma unroll
  for (int q = 0; q < 2; ++q)
    if (wave + kSmallWaves * q < xtiles) put(x, v[q], wave + kSmallWaves * q, xt);
  __syncthreads();
  for (int s = 0; s < a.steps; ++s) {
    float w[2][16];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int t = wave + kSmallWaves * q;
      if (t >= gt * gt) break;
      const f32x16 p = flat_product<TALL, TALL>(x, t / gt, x, t % gt, TALL ? mp : np, lane);
#pragma unroll
      for (int e = 0; e < 16; ++e) w[q][e] = p[e] * kPerUnit;
      put(g, w[q], t, gt);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int t = wave + kSmallWaves * q;
      if (t >= gt * gt) break;
      const f32x16 p = flat_product<false, false>(g, t / gt, g, t % gt, side, lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float was[4];
        flat_get(g, row_at(t, gt), col_at(t, gt, i), was);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[q][4 * i + e] = kB * was[e] + kC * (p[4 * i + e] * kPerUnit);
      }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (wave + kSmallWaves * q < gt * gt) put(g, w[q], wave + kSmallWaves * q, gt);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int t = wave + kSmallWaves * q;
      if (t >= xtiles) break;
      const f32x16 p = TALL ? flat_product<false, false>(x, t / xt, g, t % xt, side, lane)
                            : flat_product<false, true>(g, t / xt, x, t % xt, side, lane);
#pragma unroll
      for (int e = 0; e < 16; ++e) v[q][e] = kA * v[q][e] + p[e] * kPerUnit;
    }
    if (s + 1 == a.steps) break;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (wave + kSmallWaves * q < xtiles) put(x, v[q], wave + kSmallWaves * q, xt);
    __syncthreads();
  }
  TI* out = mat<TI>(a.out, blockIdx.x);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int t = wave + kSmallWaves * q;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int r = row_at(t, xt), c = col_at(t, xt, e >> 2) + (e & 3);
      if (t < xtiles && r < m && c < n) {
        const float o = v[q][e] * kPerUnit;
        out[r * n + c] = from_f<TI>(MOM ? a.keep * to_f(out[r * n + c]) - a.rate * o : o);
      }
    }
  }
}

bool small_ok(const Orthogonalize& a) {
  const int64_t mp = (a.m + 31) / 32 * 32, np = (a.n + 31) / 32 * 32;
  return mp * np <= kSmallValues && std::min(mp, np) <= 128;
}

template <typename TI>
void small(const Orthogonalize& a, hipStream_t s, const char* what) {
  const dim3 grid((unsigned)a.count), block(64 * kSmallWaves);
  const bool tall = a.m > a.n;
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, a); };
  if (a.momentum) tall ? go(small_kernel<TI, true, true>) : go(small_kernel<TI, true, false>);
  else tall ? go(small_kernel<TI, false, true>) : go(small_kernel<TI, false, false>);
  check_launch(what);
}

}  // namespace

size_t orthogonalize_ws_bytes(const Orthogonalize& a, int cus) {
  return small_ok(a) ? 0 : space(a, cus, nullptr).bytes;
}

void orthogonalize(const Orthogonalize& a, void* ws, int cus, hipStream_t s) {
  const char* what = a.momentum ? "muon_step" : "orthogonalize";
  if (small_ok(a)) {
    AGPU_FLOAT_SWITCH(a.dt, small<T>(a, s, what));
    return;
  }
  const Space w = space(a, cus, (char*)ws);
  AGPU_FLOAT_SWITCH(a.dt, if (a.momentum) start<T, true>(a, w, s, what); else start<T, false>(a, w, s, what));
  const bool f32 = a.dt == DType::F32;
  for (int i = 0; i + 1 < a.steps; ++i) {
    // (the type of a 16-bit result matters to the last step alone)
    const int pl = planes_of(a, i), next = planes_of(a, i + 1);
    if (f32) step<float, true, 2, 2>(a, w, i, cus, s, what);
    else if (pl == 2) step<half_t, false, 2, 2>(a, w, i, cus, s, what);
    else if (next == 2) step<half_t, false, 1, 2>(a, w, i, cus, s, what);
    else step<half_t, false, 1, 1>(a, w, i, cus, s, what);
  }
  if (f32) step<float, true, 2, 0>(a, w, a.steps - 1, cus, s, what);
  else if (a.dt == DType::F16) step<half_t, false, 2, 0>(a, w, a.steps - 1, cus, s, what);
  else step<bf16_t, false, 1, 0>(a, w, a.steps - 1, cus, s, what);
}

}  // namespace k
}  // namespace agpu
