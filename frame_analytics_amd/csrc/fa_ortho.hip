// The orthogonalised update: X <- a X + (b A + c A^2) X with A = X X^T, from X =
// g / (|g| + eps), which drives every singular value of g towards one.
//
// All the work is matrix products, on the matrix cores in float16 with float32
// accumulators.  Matrices are held times a power of two (X and A 2^11, the polynomial
// 2^10) so that float16's range serves them: an entry is at most the largest singular
// value, for which the default coefficients keep 1.2 (1.4 of A, 2.8 of the polynomial).
// Coefficients for which X, A or the polynomial would pass 65504, or fade into float16's
// smallest, are refused (fits).  Two precisions:
//
//   single (bfloat16 input of more than 64 rows): one float16 per entry.  Rounding X to 11 bits is noise
//     in every direction, and a step multiplies a small singular direction by a, so X
//     is also kept in float32 for the a X term while three or more steps follow; the
//     result is within 1.5e-3 of exact before it is rounded to bfloat16 (1.7e-3).
//   pair (the rest): hi + lo, 22 bits, three products hi hi + hi lo +
//     lo hi; the result is within 3e-6, as with float32 products.
//
// A and its square are symmetric: only tiles on and above the diagonal are computed.
// Products are rows times rows (both operands contiguous along k), so X is kept both
// ways round.  The norm's factor is a power of two, exact, in the operands and the rest
// (in (1, 2]) in the first step's epilogues: 16-bit input enters unrounded.
#include "fa_matrix.h"
#include "fa_train_abi.h"

#include <utility>

namespace fa {
namespace {

typedef _Float16 f16;
constexpr int NT = 256;
constexpr int SUMS = 512;                    // most partial sums of squares per matrix
constexpr int MOST_BATCH = 65535;            // matrices at a time: a grid's height
constexpr float SX = 2048.0f, SP = 1024.0f;  // scale of X and A, of the polynomial

template <typename T> __device__ inline float widen(T v) { return static_cast<float>(v); }

struct Poly {
  float a, b, c;
};

// Where the matrices of a call stand: batch after batch in each.
struct Bufs {
  f16 *x[2], *a[2], *p[2];  // hi, lo (lo null in single precision)
  // X^T, an operand of the step that overwrites X: read from one buffer and written to
  // the other (X itself is read only where the same thread then writes it)
  f16 *xt[2], *xt_out[2];
  float* xf;                         // X in float32 (single precision only)
  float* f;                          // [batch] the first step's factor
  double* sums;                      // [batch][SUMS]
};

// ---------------------------------------------------------------------------
// |g|^2, then X and its transpose
// ---------------------------------------------------------------------------
// Eight elements a thread, 16 bytes (or twice) at once where the matrix is aligned for
// it; the sums are float64, in a fixed order.
template <typename T>
__global__ __launch_bounds__(NT) void ortho_norm_kernel(const T* g, int64_t count, bool wide, double* sums) {
  const T* p = g + blockIdx.y * count;
  double acc = 0.0;
  for (int64_t i = (blockIdx.x * static_cast<int64_t>(NT) + threadIdx.x) * 8; i < count;
       i += static_cast<int64_t>(gridDim.x) * NT * 8) {
    float v[8];
    if (wide && i + 8 <= count) {
      constexpr int W = 16 / sizeof(T);
      typedef typename std::conditional<W == 8, typename Mat<T>::V8, typename Mat<T>::V4>::type V;
#pragma unroll
      for (int e = 0; e < 8; e += W) {
        const V x = *reinterpret_cast<const V*>(p + i + e);
#pragma unroll
        for (int k = 0; k < W; ++k) v[e + k] = widen(x[k]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = i + e < count ? widen(p[i + e]) : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) acc += static_cast<double>(v[e]) * v[e];
  }
  __shared__ double smem[WAVES_PER_BLOCK];
  const double s = block_sum(acc, smem);
  if (threadIdx.x == 0) sums[blockIdx.y * SUMS + blockIdx.x] = s;
}

__device__ inline void put(f16* hi, f16* lo, int64_t at, float v) {
  const f16 h = f16(v);
  hi[at] = h;
  if (lo) lo[at] = f16(v - float(h));
}

// Four neighbours, 8-byte aligned.
__device__ inline void put4(f16* hi, f16* lo, int64_t at, const float* v) {
  f16x4 h, l;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = f16(v[e]);
    l[e] = f16(v[e] - float(h[e]));
  }
  *reinterpret_cast<f16x4*>(hi + at) = h;
  if (lo) *reinterpret_cast<f16x4*>(lo + at) = l;
}

constexpr int PT = 64;  // side of a transposed piece
template <typename T>
__global__ __launch_bounds__(NT) void ortho_prep_kernel(const T* g, int rows, int cols, int m, int n,
                                                        int mp, int np, int parts, double eps,
                                                        Bufs w) {
  __shared__ float tile[PT][PT + 1];
  __shared__ double smem[WAVES_PER_BLOCK];
  __shared__ int exponent;
  const int b = blockIdx.z;
  {
    double own = 0.0;
    for (int t = threadIdx.x; t < parts; t += NT) own += w.sums[b * SUMS + t];
    const double s = block_sum(own, smem);
    if (threadIdx.x == 0) {
      const double norm = sqrt(s) + eps;
      int ex = 0;
      const double mant = frexp(norm, &ex);
      const bool fine = norm < __builtin_inf();  // not inf, not NaN: the result is NaN there
      exponent = fine ? ex : 0;
      if (blockIdx.x == 0 && blockIdx.y == 0)
        w.f[b] = fine ? static_cast<float>(1.0 / mant) : __builtin_nanf("");
    }
    __syncthreads();
  }
  const int shift = 11 - exponent;  // SX is 2^11
  const int i0 = blockIdx.y * PT, j0 = blockIdx.x * PT;  // of X, m x n
  const T* src = g + static_cast<int64_t>(b) * rows * cols;
  const bool tall = rows > cols;
  for (int t = threadIdx.x; t < PT * PT; t += NT) {
    // consecutive threads along the input's rows
    const int u = t / PT, v = t % PT;
    const int i = tall ? v : u, j = tall ? u : v;
    float x = 0.0f;
    if (i0 + i < m && j0 + j < n)
      x = widen(src[tall ? static_cast<int64_t>(j0 + j) * cols + i0 + i
                         : static_cast<int64_t>(i0 + i) * cols + j0 + j]);
    tile[i][j] = ldexpf(x, shift);
  }
  __syncthreads();
  const int64_t base = static_cast<int64_t>(b) * mp * np;
  f16* xl = w.x[1] ? w.x[1] + base : nullptr;
  f16* tl = w.xt[1] ? w.xt[1] + base : nullptr;
  for (int t = threadIdx.x; t < PT * PT; t += NT) {
    const int u = t / PT, v = t % PT;
    put(w.x[0] + base, xl, static_cast<int64_t>(i0 + u) * np + j0 + v, tile[u][v]);
    put(w.xt[0] + base, tl, static_cast<int64_t>(j0 + u) * mp + i0 + v, tile[v][u]);
  }
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
enum Mode : int { GRAM = 0, SQUARE = 1, STEP = 2 };

struct Step {
  int m, n, mp, np;
  Poly poly;
  bool first, last;     // of the steps
  bool read_f, write_f;  // X in float32
  bool tall;
  int tiles_i, tiles_j;
};

// Tile t of the tiles on and above the diagonal of a k x k grid, row by row.
__device__ inline void upper(int t, int k, int* ti, int* tj) {
  int i = static_cast<int>((2 * k + 1 - sqrtf(static_cast<float>((2 * k + 1) * (2 * k + 1) - 8 * t))) * 0.5f);
  auto before = [k](int r) { return r * k - r * (r - 1) / 2; };
  while (i > 0 && before(i) > t) --i;
  while (before(i + 1) <= t) ++i;
  *ti = i;
  *tj = i + t - before(i);
}

// The KG groups of four waves of a workgroup take every KG-th piece of k, each with LDS
// of its own; their sums are added in order of the groups.
template <int TM, int KG, bool PAIR, int MODE, typename T>
__global__ __launch_bounds__(NT * KG) void ortho_product_kernel(Bufs w, Step st, T* out) {
  constexpr int BK = PAIR ? 32 : 64, PARTS = PAIR ? 2 : 1, WT = TM / 2, NB = WT / 32;
  constexpr int BUFS = KG > 1 ? 1 : 2;
  using TL = Tile<f16, BK>;
  using M = Mat<f16>;
  constexpr int PIECE = TM * TL::LD;
  extern __shared__ __align__(16) unsigned char smem[];
  const int kg = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0;
  // [KG][BUFS][A, B][PARTS][TM][LD]
  f16* lds = reinterpret_cast<f16*>(smem) + kg * BUFS * 2 * PARTS * PIECE;
  const int tid = threadIdx.x & (NT - 1), lane = tid & 63, wave = tid >> 6, hh = lane >> 5, col = lane & 31;
  const int per = MODE == STEP ? st.tiles_i * st.tiles_j : st.tiles_i * (st.tiles_i + 1) / 2;
  const unsigned wg = xcd_tile(blockIdx.x, gridDim.x);
  const int b = wg / per, t = wg % per;
  int ti, tj;
  if (MODE == STEP) {
    ti = t / st.tiles_j;
    tj = t % st.tiles_j;
  } else {
    upper(t, st.tiles_i, &ti, &tj);
  }
  const int K = MODE == GRAM ? st.np : st.mp;
  const int64_t xs = static_cast<int64_t>(st.mp) * st.np, as = static_cast<int64_t>(st.mp) * st.mp;
  f16* const* A = MODE == GRAM ? w.x : MODE == SQUARE ? w.a : w.p;
  f16* const* B = MODE == GRAM ? w.x : MODE == SQUARE ? w.a : w.xt;
  const int64_t abase = b * (MODE == GRAM ? xs : as), bbase = b * (MODE == SQUARE ? as : xs);
  const f16 *ap[PARTS], *bp[PARTS];
#pragma unroll
  for (int s = 0; s < PARTS; ++s) {
    ap[s] = A[s] + abase + static_cast<int64_t>(ti) * TM * K;
    bp[s] = B[s] + bbase + static_cast<int64_t>(tj) * TM * K;
  }
  // 128-wide tiles have two pieces of k on their way at a time (2 x 4096^2 4.44 -> 4.42 ms);
  // 64-wide ones, more of which share a compute unit, one (two: 139 -> 153 us, 6 x 180^2)
  constexpr bool TWO = TM == 128;
  TileLoad<f16, BK, TM, NT, true> al[2][PARTS], bl[2][PARTS];
  auto load = [&](auto stage, int piece) {  // past the end: zeros
    constexpr int S = decltype(stage)::value;
    const int rows = piece * BK < K ? TM : 0, k = rows ? piece * BK : 0;
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
      al[S][s].load(ap[s] + k, K, rows, BK, 8, tid);
      bl[S][s].load(bp[s] + k, K, rows, BK, 8, tid);
    }
  };
  auto store = [&](auto stage, int buf) {
    constexpr int S = decltype(stage)::value;
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
      al[S][s].store(lds + ((buf * 2 + 0) * PARTS + s) * PIECE, tid);
      bl[S][s].store(lds + ((buf * 2 + 1) * PARTS + s) * PIECE, tid);
    }
  };
  const int wi = (wave >> 1) * WT, wj = (wave & 1) * WT;
  f32x16 acc[NB][NB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  const int rounds = (K / BK + KG - 1) / KG;
  typedef std::integral_constant<int, 0> Even;
  typedef std::integral_constant<int, 1> Odd;
  load(Even(), kg);
  if (TWO) load(Odd(), KG + kg);
  store(Even(), 0);
  auto round = [&](int k, auto stage, auto other) {
    __syncthreads();
    if (TWO) load(stage, (k + 2) * KG + kg);
    else if (k + 1 < rounds) load(other, (k + 1) * KG + kg);
    const f16* la = lds + ((k % BUFS) * 2 + 0) * PARTS * PIECE;
    const f16* lb = lds + ((k % BUFS) * 2 + 1) * PARTS * PIECE;
#pragma unroll
    for (int c = 0; c < BK / 16; ++c) {
      f16x8 af[PARTS][NB], bf[PARTS][NB];
#pragma unroll
      for (int s = 0; s < PARTS; ++s)
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          af[s][i] = TL::straight(la + s * PIECE, wi + 32 * i + col, 16 * c + 8 * hh);
          bf[s][i] = TL::straight(lb + s * PIECE, wj + 32 * i + col, 16 * c + 8 * hh);
        }
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          acc[i][j] = M::mma(af[0][i], bf[0][j], acc[i][j]);
          if constexpr (PAIR) {
            acc[i][j] = M::mma(af[0][i], bf[1][j], acc[i][j]);
            acc[i][j] = M::mma(af[1][i], bf[0][j], acc[i][j]);
          }
        }
    }
    if (k + 1 < rounds) {
      if (BUFS == 1) __syncthreads();
      store(other, (k + 1) % BUFS);
    }
  };
  for (int k = 0; k < rounds; k += 2) {
    round(k, Even(), Odd());
    if (k + 1 < rounds) round(k + 1, Odd(), Even());
  }
  if constexpr (KG > 1) {
    // group g finishes the registers r with (r / 4) % KG = g
    static_assert(KG == 4, "a group for each four registers");
    float* part = reinterpret_cast<float*>(smem);  // [KG][4 waves][NB * NB][64 lanes][16]
    constexpr int GROUP = 4 * NB * NB * 1024;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
          *reinterpret_cast<f32x4*>(part + kg * GROUP + ((wave * NB + i) * NB + j) * 1024 + r4 * 256 + lane * 4) =
              f32x4{acc[i][j][4 * r4], acc[i][j][4 * r4 + 1], acc[i][j][4 * r4 + 2], acc[i][j][4 * r4 + 3]};
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(part + g * GROUP + ((wave * NB + i) * NB + j) * 1024 +
                                                          kg * 256 + lane * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += x[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = v[e];  // (read below as register 4 r4 + e, r4 = 0)
      }
  }

  const float f = st.first ? w.f[b] : 1.0f;
#pragma unroll
  for (int bi = 0; bi < NB; ++bi)
#pragma unroll
    for (int bj = 0; bj < NB; ++bj) {
      const int j = tj * TM + wj + 32 * bj + col;
#pragma unroll
      for (int q4 = 0; q4 < (KG > 1 ? 1 : 4); ++q4) {
        const int r4 = KG > 1 ? kg : q4;
        const int i = ti * TM + wi + 32 * bi + 8 * r4 + 4 * hh;  // four rows from here
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[bi][bj][4 * q4 + e];
        if constexpr (MODE == GRAM || MODE == SQUARE) {
          f16* const* dst = MODE == GRAM ? w.a : w.p;
          const int64_t o = b * as;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t at = o + static_cast<int64_t>(i + e) * st.mp + j;
            if constexpr (MODE == GRAM) {
              v[e] *= f * f / SX;  // SX A of (SX X)(SX X)^T
            } else {
              float x = float(w.a[0][at]);
              if constexpr (PAIR) x += float(w.a[1][at]);
              v[e] = (SP / SX) * st.poly.b * x + (SP / SX / SX) * st.poly.c * v[e];
            }
            put(dst[0], PAIR ? dst[1] : nullptr, at, v[e]);
          }
          if (ti != tj) put4(dst[0], PAIR ? dst[1] : nullptr, o + static_cast<int64_t>(j) * st.mp + i, v);
        } else {
          const int64_t o = b * xs;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t at = o + static_cast<int64_t>(i + e) * st.np + j;
            float x;
            if (!PAIR && st.read_f) {
              x = w.xf[at];
            } else {
              x = float(w.x[0][at]);
              if constexpr (PAIR) x += float(w.x[1][at]);
            }
            v[e] = f * (st.poly.a * x + v[e] / SP);
          }
          if (st.last) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (i + e < st.m && j < st.n) {
                const int64_t at = st.tall ? static_cast<int64_t>(j) * st.m + i + e
                                           : static_cast<int64_t>(i + e) * st.n + j;
                out[static_cast<int64_t>(b) * st.m * st.n + at] = T(v[e] / SX);
              }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int64_t at = o + static_cast<int64_t>(i + e) * st.np + j;
              put(w.x[0], PAIR ? w.x[1] : nullptr, at, v[e]);
              if (!PAIR && st.write_f) w.xf[at] = v[e];
            }
            put4(w.xt_out[0], PAIR ? w.xt_out[1] : nullptr, o + static_cast<int64_t>(j) * st.mp + i, v);
          }
        }
      }
    }
}

struct Plan {
  int m, n, mp, np, tile, parts;
  int64_t off_x, off_xt0, off_xt1, off_a, off_p, off_xf, off_f, off_sums, bytes;
};

// Whether float16 holds every iterate of these coefficients.  A step takes each singular
// value s of X to p(s) = a s + b s^3 + c s^5 by itself, from (0, 1] on, so the largest
// that any input can have after k steps is the largest |p| over the range before: at its
// end, or where p' = a + 3 b s^2 + 5 c s^4 is zero.  The polynomial's eigenvalues are
// b s^2 + c s^4.  Each range is widened by what rounding may add.
inline bool fits(double a, double b, double c, int steps) {
  constexpr double MOST = 65504.0 * 0.99, NOISE = 1.0 + 1.0 / 512, LEAST = 1.0 / 64;
  double top = NOISE, before = 0.0;
  for (int k = 0; k < steps; ++k) {
    const double t = top * top;
    // (the negated form refuses NaN)
    if (!(top * SX <= MOST && t * SX <= MOST && top >= LEAST)) return false;
    auto poly = [&](double u) { return fabs(b * u + c * u * u); };  // of u = s^2
    auto step = [&](double u) { return fabs(sqrt(u) * (a + b * u + c * u * u)); };
    double most = poly(t), next = step(t);
    auto at = [&](double u) {
      if (u > 0.0 && u < t) most = fmax(most, poly(u)), next = fmax(next, step(u));
    };
    if (c != 0.0) {
      at(-b / (2.0 * c));
      const double disc = 9.0 * b * b - 20.0 * a * c;
      if (disc >= 0.0) at((-3.0 * b + sqrt(disc)) / (10.0 * c)), at((-3.0 * b - sqrt(disc)) / (10.0 * c));
    } else if (b != 0.0) {
      at(-a / (3.0 * b));
    }
    if (!(most * SP <= MOST) || !(next < 1e30)) return false;
    if (next == before) return true;  // so will every further step's
    before = next;
    top = next * NOISE;
  }
  return true;  // (what the last step leaves is held in float32)
}

inline int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

inline int plan(int dtype, int batch, int rows, int cols, Plan* p) {
  if (dtype != FA_F16 && dtype != FA_BF16 && dtype != FA_F32) return FA_E_DTYPE;
  if (batch < 1 || rows < 1 || cols < 1 || rows > (1 << 20) || cols > (1 << 20)) return FA_E_SHAPE;
  if (batch > MOST_BATCH) batch = MOST_BATCH;
  p->m = rows < cols ? rows : cols;
  p->n = rows < cols ? cols : rows;
  // up to 64 rows a product is a launch's time whatever its precision, and little
  // averages the noise of single float16
  p->parts = dtype == FA_BF16 && p->m > 64 ? 1 : 2;
  // rows and columns are padded to the tile: 128 where such tiles of X make two workgroups
  // for every compute unit (the card's 256: the workspace's size depends on it; 288 of 128 took
  // 31 us where 1152 of 64 took 27), and 64 where a matrix has no more rows (4096
  // of 16 x 27 padded to 128 took 5.1 ms, and 0.78 padded to 64)
  const int64_t tiles = static_cast<int64_t>(batch) * ((p->m + 127) / 128) * ((p->n + 127) / 128);
  p->tile = tiles >= 512 && p->m > 64 ? 128 : 64;
  p->mp = (p->m + p->tile - 1) / p->tile * p->tile;
  p->np = (p->n + p->tile - 1) / p->tile * p->tile;
  const int64_t xs = static_cast<int64_t>(batch) * p->mp * p->np, as = static_cast<int64_t>(batch) * p->mp * p->mp;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += align256(bytes);
    return o;
  };
  p->off_x = take(xs * 2 * p->parts);
  p->off_xt0 = take(xs * 2 * p->parts);
  p->off_xt1 = take(xs * 2 * p->parts);
  p->off_a = take(as * 2 * p->parts);
  p->off_p = take(as * 2 * p->parts);
  p->off_xf = take(p->parts == 1 ? xs * 4 : 0);
  p->off_f = take(batch * 4);
  p->off_sums = take(static_cast<int64_t>(batch) * SUMS * 8);
  p->bytes = at;
  return FA_OK;
}

template <int TM, int KG, bool PAIR, int MODE, typename T>
int launch_tiles(const Bufs& w, const Step& st, int64_t wgs, T* out, hipStream_t s) {
  constexpr int BK = PAIR ? 32 : 64, PARTS = PAIR ? 2 : 1, BUFS = KG > 1 ? 1 : 2;
  constexpr size_t tiles = size_t(KG) * BUFS * 2 * PARTS * TM * Tile<f16, BK>::LD * sizeof(f16);
  constexpr size_t sums = KG > 1 ? size_t(KG) * TM * TM * sizeof(float) : 0;
  constexpr size_t lds = tiles > sums ? tiles : sums;
  auto kernel = ortho_product_kernel<TM, KG, PAIR, MODE, T>;
  if (lds > 64 * 1024)
    FA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
  kernel<<<static_cast<unsigned>(wgs), NT * KG, lds, s>>>(w, st, out);
  FA_LAUNCH_CHECK();
  return FA_OK;
}

template <bool PAIR, int MODE, typename T>
int launch_product(const Bufs& w, Step st, int tile, int batch, int device, T* out, hipStream_t s) {
  // of the padded size's tiles, unless they leave compute units without a workgroup
  auto count = [&](int t) {
    const int64_t ti = st.mp / t, tj = st.np / t;
    return batch * (MODE == STEP ? ti * tj : ti * (ti + 1) / 2);
  };
  int64_t wgs = count(tile);
  if (wgs > 0x7fffffff / 4) return FA_E_SHAPE;
  if (tile == 128 && wgs < cu_count(device)) tile = 64, wgs = count(64);
  st.tiles_i = st.mp / tile;
  st.tiles_j = st.np / tile;
  if (tile == 128) return launch_tiles<128, 1, PAIR, MODE, T>(w, st, wgs, out, s);
  // few workgroups: k is split between four groups of waves
  if (wgs < cu_count(device)) return launch_tiles<64, 4, PAIR, MODE, T>(w, st, wgs, out, s);
  return launch_tiles<64, 1, PAIR, MODE, T>(w, st, wgs, out, s);
}

template <typename T, bool PAIR>
int orthogonalize(const void* g, int batch, int rows, int cols, int steps, const Poly& poly, double eps,
                  void* out, char* ws, const Plan& p, int device, hipStream_t s) {
  const int64_t xs = static_cast<int64_t>(batch) * p.mp * p.np, as = static_cast<int64_t>(batch) * p.mp * p.mp;
  auto set = [&](f16** dst, int64_t off, int64_t count) {
    dst[0] = reinterpret_cast<f16*>(ws + off);
    dst[1] = PAIR ? dst[0] + count : nullptr;
  };
  Bufs w{};
  set(w.x, p.off_x, xs);
  set(w.xt, p.off_xt0, xs);
  set(w.a, p.off_a, as);
  set(w.p, p.off_p, as);
  w.xf = PAIR ? nullptr : reinterpret_cast<float*>(ws + p.off_xf);
  w.f = reinterpret_cast<float*>(ws + p.off_f);
  w.sums = reinterpret_cast<double*>(ws + p.off_sums);
  const int64_t count = static_cast<int64_t>(rows) * cols;
  const int64_t want = (count + 8 * NT - 1) / (8 * NT);
  const int parts = static_cast<int>(want < SUMS ? want : SUMS);
  const bool wide = reinterpret_cast<uintptr_t>(g) % 16 == 0 && count * sizeof(T) % 16 == 0;
  ortho_norm_kernel<T><<<dim3(parts, batch), NT, 0, s>>>(static_cast<const T*>(g), count, wide, w.sums);
  FA_LAUNCH_CHECK();
  ortho_prep_kernel<T><<<dim3(p.np / PT, p.mp / PT, batch), NT, 0, s>>>(
      static_cast<const T*>(g), rows, cols, p.m, p.n, p.mp, p.np, parts, eps, w);
  FA_LAUNCH_CHECK();
  Step st{};
  st.m = p.m;
  st.n = p.n;
  st.mp = p.mp;
  st.np = p.np;
  st.poly = poly;
  st.tall = rows > cols;
  set(w.xt_out, p.off_xt1, xs);
  T* o = static_cast<T*>(out);
  for (int k = 0; k < steps; ++k) {
    st.first = k == 0;
    st.last = k == steps - 1;
    st.read_f = k >= 1 && steps - k >= 3;
    st.write_f = steps - (k + 1) >= 3;
    if (const int e = launch_product<PAIR, GRAM, T>(w, st, p.tile, batch, device, o, s)) return e;
    if (const int e = launch_product<PAIR, SQUARE, T>(w, st, p.tile, batch, device, o, s)) return e;
    if (const int e = launch_product<PAIR, STEP, T>(w, st, p.tile, batch, device, o, s)) return e;
    std::swap(w.xt, w.xt_out);
  }
  return FA_OK;
}

}  // namespace
}  // namespace fa

extern "C" {

FA_API int fa_gpu_orthogonalize_workspace(int dtype, int batch, int rows, int cols,
                                          int64_t* out_bytes) {
  if (!out_bytes) return FA_E_ARG;
  fa::Plan p;
  if (const int e = fa::plan(dtype, batch, rows, cols, &p)) return e;
  *out_bytes = p.bytes;
  return FA_OK;
}

FA_API int fa_gpu_orthogonalize(const void* g, int dtype, int batch, int rows, int cols, int steps,
                                double a, double b, double c, double eps, void* out,
                                void* workspace, int64_t workspace_bytes, int device,
                                void* stream) {
  using namespace fa;
  if (!g || !out || !workspace) return FA_E_ARG;
  Plan p;
  if (const int e = plan(dtype, batch, rows, cols, &p)) return e;
  if (steps < 1 || !(eps > 0.0) || workspace_bytes < p.bytes || !fits(a, b, c, steps)) return FA_E_ARG;
  DeviceScope scope(device);
  if (scope.status != hipSuccess) return -static_cast<int>(scope.status);
  const Poly poly{static_cast<float>(a), static_cast<float>(b), static_cast<float>(c)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  auto some = [&](const void* from, void* to, int count) {
    switch (dtype) {
      case FA_BF16:
        return p.parts == 1
                   ? orthogonalize<__bf16, false>(from, count, rows, cols, steps, poly, eps, to, ws, p, device, s)
                   : orthogonalize<__bf16, true>(from, count, rows, cols, steps, poly, eps, to, ws, p, device, s);
      case FA_F16: return orthogonalize<f16, true>(from, count, rows, cols, steps, poly, eps, to, ws, p, device, s);
      default: return orthogonalize<float, true>(from, count, rows, cols, steps, poly, eps, to, ws, p, device, s);
    }
  };
  const int64_t each = static_cast<int64_t>(rows) * cols * (dtype == FA_F32 ? 4 : 2);
  for (int64_t b0 = 0; b0 < batch; b0 += MOST_BATCH) {
    const int count = static_cast<int>(batch - b0 < MOST_BATCH ? batch - b0 : MOST_BATCH);
    if (const int e = some(static_cast<const char*>(g) + b0 * each, static_cast<char*>(out) + b0 * each, count))
      return e;
  }
  return FA_OK;
}

}  // extern "C"
