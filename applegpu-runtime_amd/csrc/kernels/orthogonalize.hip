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
// Precision: products are of fp16 with fp32 sums, of one plane or of two (22
// bits), see planes_of.  All entries are at most about
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
  if (n >= 8) __builtin_memcpy(at, &r, sizeof(r));
  else
    for (int e = 0; e < 8; ++e)
      if (e < n) at[e] = r.e[e];
}

// X = a X + B X, in fp32 and as the next step's NEXT planes; after the last
// step (NEXT = 0) the result instead.  Tiles within the columns of a matrix
// whose rows stay aligned read X and the weights where the accumulators are,
// eight loads under way at a time; others run by run (a load and its use after
// one another: 18 us more a tile of 256 x 256).
template <typename TO, int NEXT>
struct EpiUpdate {
  float* x;        // [count][m][n]
  half_t* planes;  // rows ld apart
  int64_t ld;
  Mats out;
  bool step;       // out = keep out - rate X
  float keep, rate;
  __device__ __forceinline__ float result(float v, float was) const {
    const float s = v * kPerUnit;
    return step ? keep * was - rate * s : s;
  }
  template <class TL>
  __device__ __forceinline__ bool near(const Args& p, const Place& c) const {
    return c.n0 + TL::BN <= p.N && p.N % 4 == 0 &&
           (NEXT != 0 || ((uintptr_t)mat<TO>(out, c.batch) % (4 * sizeof(TO))) == 0);
  }
  template <class TL>
  __device__ __forceinline__ void form(const Args& p, const Place& c, typename TL::Acc& acc) const {
    const float* xb = x + (int64_t)c.batch * p.M * p.N;
    const TO* o = NEXT ? nullptr : mat<TO>(out, c.batch);
    if (near<TL>(p, c)) {
      const typename TL::template Places<float> xs(c, xb, p.N, p.M);
      const typename TL::template Places<TO> os(c, NEXT ? (const TO*)xb : o, p.N, p.M);
      TL::fours(acc, [&](int i, int j, int g, float (&v)[4]) {
        float t[4];
        xs.load(i, j, g, t);
        if (NEXT == 0 && step) {
          float w[4];
          os.load(i, j, g, w);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = result(kA * t[e] + v[e] * kPerUnit, w[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = kA * t[e] + v[e] * kPerUnit;
            if constexpr (NEXT == 0) v[e] = result(v[e], 0.f);
          }
        }
      });
    }
  }
  template <class TL>
  __device__ __forceinline__ void store(const Args& p, const Place& c, typename TL::T* lds, typename TL::Acc& acc) const {
    float* xb = x + (int64_t)c.batch * p.M * p.N;
    TO* o = NEXT ? nullptr : mat<TO>(out, c.batch);
    const bool near = this->near<TL>(p, c);
    TL::template runs<false>(
        c, lds, acc, false,
        [&](int64_t row, int64_t col, float (&v)[8]) {
          if (row >= p.M || (col >= p.N && col * NEXT >= ld * (NEXT != 0))) return;
          const int n = p.N - col < 8 ? (int)(p.N - col) : 8;  // (none behind the columns, where planes hold zeros)
          const int64_t at = row * p.N + col;
          if (near) {
            if constexpr (NEXT != 0) {
              float4* to = (float4*)(xb + at);
              to[0] = make_float4(v[0], v[1], v[2], v[3]);
              to[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
          } else {
            Run<float> t = get_run(xb + at, n);
            Run<TO> w{};
            if (NEXT == 0 && step) w = get_run(o + at, n);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              v[e] = e < n ? kA * t.e[e] + v[e] * kPerUnit : 0.f;
              t.e[e] = v[e];
              if constexpr (NEXT == 0) v[e] = result(v[e], to_f(w.e[e]));
            }
            if constexpr (NEXT != 0) put_run(xb + at, t, n);
          }
          if constexpr (NEXT != 0) {
            put_planes<half_t, NEXT>(planes + ((int64_t)c.batch * p.M + row) * ld, col, v);
          } else {
            Run<TO> q;
#pragma unroll
            for (int e = 0; e < 8; ++e) q.e[e] = from_f<TO>(v[e]);
            put_run(o + at, q, n);
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

// fp16 planes of a step's factors.  What a step rounds is passed on by the
// steps behind it, so the last ones set the result's error: relative to the
// result (160 x 640 with a few strong directions, oracle with roundings) 1.4e-3
// with one plane throughout, 1.2e-4 with two in the last three steps, 1e-6 with
// two throughout.  Against the rounding of the result itself, 1.7e-3 in bf16,
// 2.1e-4 in fp16 and 3e-8 in fp32, that is one plane, two in the last three
// steps, and two.  Small matrices take two in fp16 throughout: their error is
// larger (64 x 128: 2.5e-4) and their time is the launches'.
int planes_of(const Orthogonalize& a, int step) {
  if (a.dt == DType::F32) return 2;
  if (a.dt == DType::BF16) return 1;
  return step + 3 >= a.steps || std::min(a.m, a.n) <= 256 ? 2 : 1;
}
int64_t row_of(int64_t n, int planes) { return (n + 31) / 32 * 32 * planes; }

struct Space {
  double* part;
  float* x;
  half_t *planes[2], *a, *b;
  size_t bytes;
};
Space space(const Orthogonalize& a, char* base) {
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
  w.x = (float*)take((size_t)(a.count * a.m * a.n) * 4);
  for (auto& q : w.planes) q = (half_t*)take((size_t)(a.count * a.m * row_of(a.n, pl)) * 2);
  w.a = (half_t*)take((size_t)(a.count * side * row_of(side, pl)) * 2);
  w.b = (half_t*)take((size_t)(a.count * side * row_of(side, pl)) * 2);
  w.bytes = used;
  return w;
}

template <typename TI>
void start(const Orthogonalize& a, const Space& w, hipStream_t s, const char* what) {
  const int64_t n = a.m * a.n;
  const dim3 parts(kNormParts, (unsigned)a.count);
  if (a.momentum)
    hipLaunchKernelGGL((norm_kernel<TI, true>), parts, dim3(256), 0, s, a.in, a.mom, a.beta, a.nesterov, n, w.part, w.x);
  else
    hipLaunchKernelGGL((norm_kernel<TI, false>), parts, dim3(256), 0, s, a.in, a.mom, a.beta, a.nesterov, n, w.part,
                       (float*)nullptr);
  check_launch(what);
  const int pl = planes_of(a, 0);
  const int64_t ld = row_of(a.n, pl);
  const dim3 grid((unsigned)std::min<int64_t>(blocks_for(a.m * (ld / (8 * pl)), 256), 1024), (unsigned)a.count);
  // (U and X share their place: a value is read before it is written, by the
  // same thread)
  auto go = [&](auto kernel, const float* u) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a.in, u, a.m, a.n, w.part, a.eps, w.x, w.planes[0], ld);
  };
  if (a.momentum) pl == 1 ? go(start_kernel<float, 1>, w.x) : go(start_kernel<float, 2>, w.x);
  else pl == 1 ? go(start_kernel<TI, 1>, nullptr) : go(start_kernel<TI, 2>, nullptr);
  check_launch(what);
}

// Step i on PL planes, the next on NEXT (0: none follows).
template <typename TO, int PL, int NEXT>
void step(const Orthogonalize& a, const Space& w, int i, int cus, hipStream_t s, const char* what) {
  const int64_t m = a.m, n = a.n, side = std::min(m, n), ld = row_of(n, PL), lda = row_of(side, PL);
  const bool tall = m > n;
  const int gram = pick(side, side, a.count, true, cus), upd = pick(m, n, a.count, false, cus);
  const Operand xo{w.planes[i & 1], ld, m * ld}, ao{w.a, lda, side * lda}, bo{w.b, lda, side * lda};
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
  const EpiUpdate<TO, NEXT> eu{w.x, w.planes[(i + 1) & 1], row_of(n, NEXT), a.out, a.momentum, a.keep, a.rate};
  if (tall) run<PL, false, false, false>(upd, p, eu, s, what);
  else run<PL, false, true, false>(upd, p, eu, s, what);
}

}  // namespace

size_t orthogonalize_ws_bytes(const Orthogonalize& a, int) { return space(a, nullptr).bytes; }

void orthogonalize(const Orthogonalize& a, void* ws, int cus, hipStream_t s) {
  const char* what = a.momentum ? "muon_step" : "orthogonalize";
  const Space w = space(a, (char*)ws);
  AGPU_FLOAT_SWITCH(a.dt, start<T>(a, w, s, what));
  for (int i = 0; i + 1 < a.steps; ++i) {
    // (the type of a result matters to the last step alone)
    const int pl = planes_of(a, i), next = planes_of(a, i + 1);
    if (pl == 2) step<float, 2, 2>(a, w, i, cus, s, what);
    else if (next == 2) step<float, 1, 2>(a, w, i, cus, s, what);
    else step<float, 1, 1>(a, w, i, cus, s, what);
  }
  if (a.dt == DType::F32) step<float, 2, 0>(a, w, a.steps - 1, cus, s, what);
  else if (a.dt == DType::F16) step<half_t, 2, 0>(a, w, a.steps - 1, cus, s, what);
  else step<bf16_t, 1, 0>(a, w, a.steps - 1, cus, s, what);
}

}  // namespace k
}  // namespace agpu
