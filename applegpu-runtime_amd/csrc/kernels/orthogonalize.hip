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
// with one launch each for all matrices of a batch.
//
// Precision: products are of fp16 with fp32 sums, of one plane for 16-bit
// matrices and of two (22 bits) for fp32 ones.  All entries are at most about
// 1.3 in magnitude (singular values stay below 1.2), so X, A and B are held
// times 2^14, where fp16 keeps 11 bits of everything down to 2^-28.  X itself
// stays in fp32 beside its planes: a X is what carries the small singular
// values, multiplied by 3.4 in each step, and would carry a rounding of X
// along; what fp16 loses of X inside B X is B's small share of that direction.
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

constexpr int kNormParts = 128;  // blocks a matrix for its norm

// Of matrix blockIdx.y: the squares' sum in kNormParts parts, and with
// momentum the new momentum and U (fp32, contiguous).
template <typename TI, bool MOM>
__global__ void __launch_bounds__(256) norm_kernel(Mats in, Mats mom, float beta, bool nesterov, int64_t n,
                                                   double* part, float* u) {
  __shared__ double red[4];
  const int64_t i = blockIdx.y;
  const TI* g = mat<TI>(in, i);
  float* b = MOM ? mat<float>(mom, i) : nullptr;
  double sum = 0.0;
  auto one = [&](int64_t j, float gv) {
    float v = gv;
    if constexpr (MOM) {
      const float mv = beta * b[j] + gv;
      b[j] = mv;
      v = nesterov ? gv + beta * mv : mv;
      u[i * n + j] = v;
    }
    sum += (double)v * (double)v;
  };
  struct alignas(4 * sizeof(TI)) V { TI e[4]; };
  if (n % 4 == 0 && ((uintptr_t)g % sizeof(V)) == 0) {
#pragma unroll 2
    for (int64_t j = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; j < n; j += (int64_t)kNormParts * 1024) {
      const V v = *(const V*)(g + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) one(j + e, to_f(v.e[e]));
    }
  } else {
    for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < n; j += (int64_t)kNormParts * 256) one(j, to_f(g[j]));
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) part[i * kNormParts + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// X = U / (|U| + eps) in units of 2^-14: fp32 [m, n] and planes with rows of
// ld values.  TI: what U is held as (the matrices, or fp32 at u).
template <typename TI, int PL>
__global__ void __launch_bounds__(256) start_kernel(Mats in, const float* u, int64_t m, int64_t n, const double* part,
                                                    float eps, float* x, half_t* planes, int64_t ld) {
  __shared__ double red[2];
  const int64_t i = blockIdx.y;
  const TI* g = u ? (const TI*)(u + i * m * n) : mat<TI>(in, i);
  if (threadIdx.x < kNormParts) {
    double s = part[i * kNormParts + threadIdx.x];
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) s += __shfl_xor(s, k);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  }
  __syncthreads();
  const float norm = (float)sqrt(red[0] + red[1]) + eps;
  const float by = norm > 0.f || norm != norm ? norm : 1.f;  // a matrix of zeros stays one
  const int64_t chunks = ld / (8 * PL), total = m * chunks;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t r = t / chunks, c = (t - r * chunks) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < n ? to_f(g[r * n + c + e]) / by * kUnit : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < n) x[(i * m + r) * n + c + e] = v[e];
    put_planes<half_t, PL>(planes + (i * m + r) * ld, c, v);
  }
}

// A (or B = b A + c A A) of a tile, and its mirror image.
template <bool POLY>
struct EpiGram {
  const half_t* a;  // POLY
  half_t* out;
  int64_t ld, batch;  // rows ld apart, matrices batch apart
  template <class TL>
  __device__ void store(const Args& p, const Place& c, typename TL::T* lds, typename TL::Acc& acc) const {
    constexpr int PL = TL::PL;
    half_t* to = out + c.batch * batch;
    const half_t* from = POLY ? a + c.batch * batch : nullptr;
    // 8 values of row r from column q on
    auto put = [&](int64_t r, int64_t q, float (&v)[8]) {
      if (r >= p.M || q * PL >= ld) return;
      float t[8] = {};
      if constexpr (POLY) get_planes<half_t, PL>(from + r * ld, q, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float s = v[e] * kPerUnit;
        v[e] = q + e < p.N ? (POLY ? kB * t[e] + kC * s : s) : 0.f;
      }
      put_planes<half_t, PL>(to + r * ld, q, v);
    };
    TL::template runs<true>(
        c, lds, acc, c.tm != c.tn, [&](int64_t row, int64_t col, float (&v)[8]) { put(row, col, v); },
        [&](int64_t row, int64_t col, float (&v)[8]) { put(col, row, v); });
  }
};

// X = a X + B X, in fp32 and planes; at the end the result instead.
template <typename TO, bool LAST>
struct EpiUpdate {
  float* x;        // [count][m][n]
  half_t* planes;  // rows ld apart
  int64_t ld;
  Mats out;
  bool step;       // out = keep out - rate X
  float keep, rate;
  template <class TL>
  __device__ void store(const Args& p, const Place& c, typename TL::T* lds, typename TL::Acc& acc) const {
    constexpr int PL = TL::PL;
    float* xb = x + (int64_t)c.batch * p.M * p.N;
    half_t* to = LAST ? nullptr : planes + (int64_t)c.batch * p.M * ld;
    TO* o = LAST ? mat<TO>(out, c.batch) : nullptr;
    TL::template runs<false>(
        c, lds, acc, false,
        [&](int64_t row, int64_t col, float (&v)[8]) {
          if (row >= p.M || col >= p.N) {
            if (LAST || row >= p.M || col * PL >= ld) return;
          }
          const int64_t at = row * p.N + col;
          const int n = p.N - col < 8 ? (int)(p.N - col) : 8;
          float t[8] = {};
          if (n == 8) {
            __builtin_memcpy(t, xb + at, 32);
          } else {
            for (int e = 0; e < 8; ++e)
              if (e < n) t[e] = xb[at + e];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = e < n ? kA * t[e] + v[e] * kPerUnit : 0.f;
          if constexpr (!LAST) {
            if (n == 8) {
              __builtin_memcpy(xb + at, v, 32);
            } else {
              for (int e = 0; e < 8; ++e)
                if (e < n) xb[at + e] = v[e];
            }
            put_planes<half_t, PL>(to + row * ld, col, v);
          } else {
            struct V { TO e[8]; } q;
            if (step) {
              if (n == 8) {
                __builtin_memcpy(&q, o + at, sizeof(q));
              } else {
                for (int e = 0; e < 8; ++e)
                  if (e < n) q.e[e] = o[at + e];
              }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float s = v[e] * kPerUnit;
              q.e[e] = from_f<TO>(step ? keep * to_f(q.e[e]) - rate * s : s);
            }
            if (n == 8) {
              __builtin_memcpy(o + at, &q, sizeof(q));
            } else {
              for (int e = 0; e < 8; ++e)
                if (e < n) o[at + e] = q.e[e];
            }
          }
        },
        [](int64_t, int64_t, float (&)[8]) {});
  }
};

// Square tiles of 256 (8 wavefronts), 128 or 64 (4).
enum { kBig, kMid, kSmall };
int pick(int64_t M, int64_t N, int64_t count, bool sym, int cus) {
  auto tiles = [&](int64_t b) {
    const int64_t m = ceil_div(M, b), n = ceil_div(N, b);
    return (sym ? m * (m + 1) / 2 : m * n) * count;
  };
  return tiles(256) * 4 >= 3 * cus ? kBig : tiles(128) * 4 >= 3 * cus ? kMid : kSmall;
}

template <int PL, bool AC, bool BC, bool SYM, class Epi>
void run(int tile, const Args& p, const Epi& e, hipStream_t s, const char* what) {
  if (tile == kBig) launch<Tile<half_t, 4, 2, 2, 4, PL, AC, BC, SYM>>(p, e, s, what);
  else if (tile == kMid) launch<Tile<half_t, 2, 2, 2, 2, PL, AC, BC, SYM>>(p, e, s, what);
  else launch<Tile<half_t, 1, 1, 2, 2, PL, AC, BC, SYM>>(p, e, s, what);
}

struct Space {
  double* part;
  float* x;
  half_t *planes[2], *a, *b;
  size_t bytes;
};
Space space(const Orthogonalize& a, int pl, char* base) {
  Space w;
  size_t used = 0;
  auto take = [&](size_t n) {
    char* at = base ? base + used : nullptr;
    used += (n + 255) / 256 * 256;
    return at;
  };
  const int64_t side = std::min(a.m, a.n), ld = (a.n + 31) / 32 * 32 * pl, lda = (side + 31) / 32 * 32 * pl;
  w.part = (double*)take((size_t)a.count * kNormParts * 8);
  w.x = (float*)take((size_t)(a.count * a.m * a.n) * 4);
  for (auto& q : w.planes) q = (half_t*)take((size_t)(a.count * a.m * ld) * 2);
  w.a = (half_t*)take((size_t)(a.count * side * lda) * 2);
  w.b = (half_t*)take((size_t)(a.count * side * lda) * 2);
  w.bytes = used;
  return w;
}

template <typename TI, int PL>
void ortho(const Orthogonalize& a, void* wsp, int cus, hipStream_t s) {
  const char* what = a.momentum ? "muon_step" : "orthogonalize";
  const Space w = space(a, PL, (char*)wsp);
  const int64_t m = a.m, n = a.n, side = std::min(m, n);
  const int64_t ld = (n + 31) / 32 * 32 * PL, lda = (side + 31) / 32 * 32 * PL;
  const dim3 parts(kNormParts, (unsigned)a.count);
  if (a.momentum)
    hipLaunchKernelGGL((norm_kernel<TI, true>), parts, dim3(256), 0, s, a.in, a.mom, a.beta, a.nesterov, m * n, w.part,
                       w.x);
  else
    hipLaunchKernelGGL((norm_kernel<TI, false>), parts, dim3(256), 0, s, a.in, a.mom, a.beta, a.nesterov, m * n, w.part,
                       (float*)nullptr);
  check_launch(what);
  const dim3 grid((unsigned)std::min<int64_t>(blocks_for(m * (ld / (8 * PL)), 256), 1024), (unsigned)a.count);
  if (a.momentum)  // U and X share their place: each value is read before it is written, by the same thread
    hipLaunchKernelGGL((start_kernel<float, PL>), grid, dim3(256), 0, s, a.in, w.x, m, n, w.part, a.eps, w.x,
                       w.planes[0], ld);
  else
    hipLaunchKernelGGL((start_kernel<TI, PL>), grid, dim3(256), 0, s, a.in, (const float*)nullptr, m, n, w.part, a.eps,
                       w.x, w.planes[0], ld);
  check_launch(what);
  const bool tall = m > n;
  const int gram = pick(side, side, a.count, true, cus), upd = pick(m, n, a.count, false, cus);
  const Operand ao{w.a, lda, side * lda}, bo{w.b, lda, side * lda};
  for (int i = 0; i < a.steps; ++i) {
    const Operand xo{w.planes[i & 1], ld, m * ld};
    Args p;
    p.batches = (int)a.count;
    p.a = p.b = xo;
    p.M = p.N = side;
    p.K = tall ? m : n;
    const EpiGram<false> eg{nullptr, w.a, lda, side * lda};
    if (tall) run<PL, true, true, true>(gram, p, eg, s, what);
    else run<PL, false, false, true>(gram, p, eg, s, what);
    p.a = p.b = ao;
    p.K = side;
    run<PL, false, false, true>(gram, p, EpiGram<true>{w.a, w.b, lda, side * lda}, s, what);
    p.M = m;
    p.N = n;
    p.a = tall ? xo : bo;
    p.b = tall ? bo : xo;
    auto update = [&](const auto& e) {
      if (tall) run<PL, false, false, false>(upd, p, e, s, what);
      else run<PL, false, true, false>(upd, p, e, s, what);
    };
    if (i + 1 < a.steps) update(EpiUpdate<TI, false>{w.x, w.planes[(i + 1) & 1], ld, a.out, false, 1.f, 1.f});
    else update(EpiUpdate<TI, true>{w.x, nullptr, ld, a.out, a.momentum, a.keep, a.rate});
  }
}

}  // namespace

size_t orthogonalize_ws_bytes(const Orthogonalize& a, int) {
  return space(a, a.dt == DType::F32 ? 2 : 1, nullptr).bytes;
}

void orthogonalize(const Orthogonalize& a, void* ws, int cus, hipStream_t s) {
  if (a.dt == DType::F32) ortho<float, 2>(a, ws, cus, s);
  else if (a.dt == DType::F16) ortho<half_t, 1>(a, ws, cus, s);
  else ortho<bf16_t, 1>(a, ws, cus, s);
}

}  // namespace k
}  // namespace agpu
