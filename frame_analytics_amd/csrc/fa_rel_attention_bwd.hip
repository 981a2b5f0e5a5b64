// Attention with a relative position bias, backward.
//
// With P the weights (formed again from the scores and what the forward pass kept) and D_i =
// dout_i . out_i:  dS = P (dout V^T - D);  dQ = scale dS K;  dK = scale dS^T Q;
// dV = P^T dout;  dtable[r] = the sum of dS over the pairs of row r.
//
// Two kernels, so that every sum has one owner and a fixed order: one whose waves own
// queries (dQ, and the table's sums by difference), one whose waves own keys (dK, dV,
// over the query heads that share them).  Each forms S and dout V^T again: seven
// products in place of five, against atomic sums of dQ in memory in no fixed order.
#include "fa_rel_attention.h"

namespace fa {

namespace {

enum : int { ANY, FAR, WINDOW };  // the pairs of a tile

struct Grads {
  const void *out, *dout;
  View os, gs;
  const float* lse;  // [2][B, H, Lq]: shifts and factors, see keep_row
  float* dsum;       // [B, H, Lq]: D_i times the row's factor
  void *dq, *dk, *dv;
  View dqs, dks, dvs;
  int dqvec, dkvec;
  float* parts;  // [H][B * q_tiles][n], or null: the table needs no gradient
  float* joint;  // [splits][dk, dv][B, Hk, Lk, D] where heads that share a key are split
};

template <typename T, int DP> struct Shape {
  static constexpr int BN = sizeof(T) == 2 && DP <= 64 ? 64 : 32;
  static constexpr int BUFS = sizeof(T) == 4 && DP == 128 ? 1 : 2;
  static constexpr size_t TILE = size_t(BN) * Tile<T, DP>::LD * sizeof(T);
};

// Elements that are not finite become 0.  K of a pair that is seen and not finite has
// made that pair's dS NaN already; one that is hidden must not turn 0 x K into NaN.
template <typename T> __device__ inline typename Mat<T>::V8 finite(typename Mat<T>::V8 v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __builtin_fabsf(widen(v[i])) < INF ? v[i] : T(0);
  return v;
}

// A row's factor (rarely any but 1: read where it is used), and dout times it.
__device__ inline float factor_of(const RelAttn& a, const Grads& g, int64_t row, float shift) {
  return has_factor(shift) ? g.lse[static_cast<int64_t>(a.B) * a.H * a.Lq + row] : 1.0f;
}
template <typename T, int N> __device__ inline void scale_row(typename Mat<T>::V8 (&v)[N], float f) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = T(widen(v[i][e]) * f);
}

// ---------------------------------------------------------------------------
// dQ and the table
// ---------------------------------------------------------------------------
// Windows of up to 256 tokens (KEYS blocks of 32 keys, KEYS > 0): a workgroup takes one
// tile of queries of every `chunks`-th batch entry, and its dS by pair is summed over
// them in registers, to reach the table's differences once at the end.  (By LDS atomics
// for each window: 1617 us of 2270 for 512 windows of 16 x 16, 8 heads.)  On a line most
// blocks are far from the wave's queries and are one sum.
// KG groups of NW waves take every KG-th tile of keys, as in the forward pass.
template <typename T, int DP, int NW, int KG, bool TABLE, bool WIDE, int KEYS>
__global__ __launch_bounds__(NW * 64 * KG, sizeof(T) == 2 && DP <= 64 && KEYS / KG < 8 ? 2 : 1) void rel_attention_dq_kernel(
    RelAttn a, Grads g, int q_tiles, int chunks) {
  constexpr int NT = NW * 64;
  using M = Mat<T>;
  using TL = Tile<T, DP>;
  constexpr int BN = Shape<T, DP>::BN, NB = BN / 32, CH = DP / 16, OB = DP / 32;
  constexpr int BUFS = Shape<T, DP>::BUFS;
  extern __shared__ __align__(16) unsigned char smem[];
  static_assert(KG == 1 || BUFS == 2, "a second group");
  const int kg = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0;
  T* kt = reinterpret_cast<T*>(smem) + kg * 2 * BUFS * BN * TL::LD;
  T* vt = kt + BUFS * BN * TL::LD;
  float* eb = reinterpret_cast<float*>(reinterpret_cast<T*>(smem) + KG * 2 * BUFS * BN * TL::LD);
  const int np = a.pos.n + 2 * PAD;
  float* sums = eb + np;  // [KG * NW][np]: the table's sums by slot, one copy for each wave
  int* codes = reinterpret_cast<int*>(eb + ((TABLE ? 1 + KG * NW : 1) * np + 3) / 4 * 4);  // of a window's keys
  const int tid = threadIdx.x - kg * NT, lane = tid & 63, hh = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned wg = xcd_tile(blockIdx.x, gridDim.x);
  const int tile = q_tiles - 1 - int(wg % q_tiles);
  const int h = int(wg / q_tiles) % a.H, chunk = int(wg / q_tiles) / a.H, hk = h / (a.H / a.Hk);
  const int qw = tile * (NW * 32) + wave * 32;
  const int q = qw + col, qc = min(q, a.Lq - 1);
  const float c = a.scale * LOG2E;

  load_bias<T>(eb, a, h, 1, threadIdx.x, NT * KG);
  if (a.pos.grid_w) load_codes(codes, a.pos, a.Lk, threadIdx.x, NT * KG);
  constexpr int TOTALS = KEYS > 0 ? KEYS / KG : 1;
  f32x16 total[TOTALS];
#pragma unroll
  for (int i = 0; i < TOTALS; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) total[i][r] = 0.0f;
  if (TABLE && KEYS == 0)
    for (int t = threadIdx.x; t < KG * NW * np; t += KG * NT) sums[t] = 0.0f;
  float* mine = sums + (kg * NW + wave) * np;
  float far_lo = 0.0f, far_hi = 0.0f;
  bool far_below = false;

  for (int b = chunk; b < a.B; b += chunks) {
  const int s0 = a.start(b), len = a.keys(b), qpos = s0 + q, cq = s0 + a.pos.code(qc);
  const uint8_t* mask = a.mask_of(b, h);
  typename M::V8 qf[CH], gf[CH];
  const int64_t row = (static_cast<int64_t>(b) * a.H + h) * a.Lq + qc;
  // a row that sees no key: its weights are 2^(s - inf) = 0 whatever dout holds
  const float lse = g.lse[row];
  const bool on = q < a.Lq && lse != INF;
  // D_i by the matrix instructions, in the order that dout V^T is summed in (the
  // diagonal of dout out^T): a row that sees one key has out = v, and dS exactly 0
  f32x16 dd;
#pragma unroll
  for (int r = 0; r < 16; ++r) dd[r] = 0.0f;
  {
    const int f = tile * (NW * 32);  // the workgroup's first query
    auto rows = [&](const void* p, const View& s) {
      return Rows<T>(static_cast<const T*>(p) + b * s.b + h * s.h + f * s.t, s.t);
    };
    typename M::V8 of[CH];
    load_row<T, WIDE>(qf, rows(a.q, a.qs), q - f, 8 * hh, a.D, a.vec, on);
    load_row<T, WIDE>(gf, rows(g.dout, g.gs), q - f, 8 * hh, a.D, a.vec, on);
    load_row<T, WIDE>(of, rows(g.out, g.os), q - f, 8 * hh, a.D, a.vec, on);
    // a row's factor goes into dout, and so into dP and D_i: such a row's weights without it
    // are nearly all 0 or 1, which round to no fewer bits
    if (__ballot(has_factor(lse))) scale_row<T>(gf, factor_of(a, g, row, lse));
#pragma unroll
    for (int i = 0; i < CH; ++i) dd = M::mma(of[i], gf[i], dd);
    if (sizeof(T) == 2 && KEYS == 0 && a.pos.grid_w == 0) {  // and what the output's rounding left
      const T* low = low_of<T>(g.lse, static_cast<int64_t>(a.B) * a.H * a.Lq);
      load_row<T, WIDE>(of, Rows<T>(low + ((static_cast<int64_t>(b) * a.H + h) * a.Lq + f) * a.D, a.D), q - f,
                        8 * hh, a.D, a.vec, on);
#pragma unroll
      for (int i = 0; i < CH; ++i) dd = M::mma(of[i], gf[i], dd);
    }
  }
  float dsum = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (8 * (r / 4) + 4 * hh + r % 4 == col) dsum = dd[r];
  dsum = both_sum(dsum);
  if (kg == 0 && q < a.Lq && hh == 0) g.dsum[row] = dsum;

  f32x16 dq[OB];
#pragma unroll
  for (int i = 0; i < OB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[i][r] = 0.0f;

  int end = len;
  if (a.causal) {
    const int64_t last = int64_t(s0) + min(tile * (NW * 32) + NW * 32, a.Lq);
    end = static_cast<int>(max<int64_t>(0, min<int64_t>(end, last)));
  }
  const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  TileLoad<T, DP, BN, NT, WIDE> kl, vl;
  const int tiles = (end + BN - 1) / BN;
  if (KEYS > 0) __syncthreads();  // the window before is done with the tiles
  bool far_on = false;
  if (kg < tiles) {
    const int k1 = kg * BN;
    kl.load(kb + k1 * a.ks.t, a.ks.t, len - k1, a.D, a.vec, tid);
    vl.load(vb + k1 * a.vs.t, a.vs.t, len - k1, a.D, a.vec, tid);
    kl.store(kt, tid);
    vl.store(vt, tid);
  }
  // One tile of keys, as in the forward pass: FAR and WINDOW have no hidden pair and run
  // without a branch.
  auto work = [&](int t, f32x16* pairs, auto mode, float far) {
    constexpr int MODE = decltype(mode)::value;
    const T* kk = kt + (t / KG % BUFS) * BN * TL::LD;
    const T* vv = vt + (t / KG % BUFS) * BN * TL::LD;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int k0 = t * BN + nb * 32;
      if (MODE == ANY) {
        const bool hidden = a.causal && k0 > s0 + qw + 31;  // nothing for this wave
        if (hidden || k0 >= len || qw >= a.Lq) continue;
      }
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        s = M::mma(TL::straight(kk, nb * 32 + col, 16 * i + 8 * hh), qf[i], s);
        dp = M::mma(TL::straight(vv, nb * 32 + col, 16 * i + 8 * hh), gf[i], dp);
      }
      const bool partial = MODE == ANY && (mask || k0 + 32 > len || (a.causal && k0 + 31 > s0 + qw));
      int kind = MODE == FAR ? ALL_BELOW : NEAR;
      int slot[16];  // of each pair, where it has one of its own
      if (MODE == WINDOW || (MODE == ANY && a.pos.grid_w)) {
        // (codes are those of the window's keys, the last one's past its end)
        const int at = afresh(cq - a.pos.lo + PAD);
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int4 ck = *reinterpret_cast<const int4*>(codes + k0 + 4 * hh + 8 * r4);
          slot[4 * r4] = at - ck.x;
          slot[4 * r4 + 1] = at - ck.y;
          slot[4 * r4 + 2] = at - ck.z;
          slot[4 * r4 + 3] = at - ck.w;
        }
      } else if (MODE == ANY) {
        kind = block_kind(a.pos, s0 + qw - (k0 + 31), s0 + qw + 31 - k0);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          slot[r] = s0 + q - k0 - 4 * hh - a.pos.lo + PAD - (8 * (r / 4) + r % 4);
      }
      if (MODE == FAR) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = s[r] * c + (far - lse);
      } else if (MODE == WINDOW || kind == NEAR) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = s[r] * c + eb[slot[r]] - lse;
      } else {
        const float e = kind == ALL_BELOW ? eb[0] : eb[np - 1];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = s[r] * c + e - lse;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r]) * (dp[r] - dsum);
      if (partial) {
        const uint32_t seen = seen_keys(a, mask, qc, qpos, k0 + 4 * hh, len);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = seen >> r & 1 ? s[r] : 0.0f;
      }
      if (TABLE && KEYS > 0) {
#pragma unroll
        for (int r = 0; r < 16; ++r) pairs[nb][r] += s[r];
      } else if (TABLE) {
        if (MODE != FAR && kind == NEAR) {
          // within one half of the lanes one key meets 32 queries: 32 slots.  The
          // halves add one after the other, so the order of every slot's sum is fixed.
          if (hh == 0) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (q < a.Lq) unsafeAtomicAdd(mine + slot[r], s[r]);
          }
          __builtin_amdgcn_wave_barrier();
          if (hh == 1) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (q < a.Lq) unsafeAtomicAdd(mine + slot[r], s[r]);
          }
          __builtin_amdgcn_wave_barrier();
        } else {
          float acc = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) acc += s[r];
          acc = q < a.Lq ? acc : 0.0f;
          if (MODE == FAR ? far_below : kind == ALL_BELOW) far_lo += acc;
          else far_hi += acc;
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        typename M::V8 ds;
#pragma unroll
        for (int i = 0; i < 8; ++i) ds[i] = T(s[8 * half + i]);
#pragma unroll
        for (int i = 0; i < OB; ++i) {
          typename M::V8 kf = TL::transposed(kk, nb * 32 + 16 * half, 32 * i, lane);
          if (partial) kf = finite<T>(kf);
          dq[i] = M::mma(kf, ds, dq[i]);
        }
      }
    }
  };
  auto step = [&](int t, f32x16* pairs) {
    __syncthreads();
    if (KG > 1 && t >= tiles) return;  // (in the last round)
    const bool more = t + KG < tiles;
    const int k0 = t * BN, k1 = k0 + KG * BN;
    if (more) {
      kl.load(kb + k1 * a.ks.t, a.ks.t, len - k1, a.D, a.vec, tid);
      vl.load(vb + k1 * a.vs.t, a.vs.t, len - k1, a.D, a.vec, tid);
    }
    const bool all = !mask && k0 + BN <= len && (!a.causal || k0 + BN - 1 <= s0 + qw) && qw < a.Lq;
    const int kind = block_kind(a.pos, s0 + qw - (k0 + BN - 1), s0 + qw + 31 - k0);
    far_below = kind == ALL_BELOW;
    if (KEYS > 0 && all)
      work(t, pairs, std::integral_constant<int, WINDOW>(), 0.0f);
    else if (KEYS == 0 && all && a.pos.grid_w == 0 && kind != NEAR && far_on)
      work(t, pairs, std::integral_constant<int, KEYS == 0 ? FAR : ANY>(), far_below ? eb[0] : eb[np - 1]);
    else
      work(t, pairs, std::integral_constant<int, ANY>(), 0.0f);
    if (more) {
      if (BUFS == 1) __syncthreads();
      kl.store(kt + ((t / KG + 1) % BUFS) * BN * TL::LD, tid);
      vl.store(vt + ((t / KG + 1) % BUFS) * BN * TL::LD, tid);
    }
  };
  if constexpr (KEYS > 0) {
#pragma unroll
    for (int round = 0; round < KEYS / NB / KG; ++round)
      if (round * KG < tiles) step(round * KG + kg, total + round * NB);
  } else {
    const int rounds = (tiles + KG - 1) / KG;
    __syncthreads();
    far_on = far_serves(eb, np);
    for (int round = 0; round < rounds; ++round) step(round * KG + kg, total);
  }
  if constexpr (KG > 1) {
    static_assert(KG == 2, "the second group's sums join the first's");
    float* joint = reinterpret_cast<float*>(smem) + wave * OB * 16 * 64 + lane;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (kg == 1) joint[(16 * i + r) * 64] = dq[i][r];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (kg == 0) dq[i][r] += joint[(16 * i + r) * 64];
  }
  if (kg == 0 && q < a.Lq) {
    T* drow = static_cast<T*>(g.dq) + b * g.dqs.b + h * g.dqs.h + q * g.dqs.t;
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = dq[i][4 * e4 + e] * a.scale;
        store4<T>(drow, 32 * i + 8 * e4 + 4 * hh, a.D, g.dqvec, w);
      }
  }
  }
  if (TABLE && KEYS > 0) {
    __syncthreads();
    for (int t = threadIdx.x; t < KG * NW * np; t += KG * NT) sums[t] = 0.0f;
    __syncthreads();
    const int at = a.pos.code(qc) - a.pos.lo + PAD;
    for (int turn = 0; turn < 2; ++turn) {  // the halves one after the other, as above
      if (hh == turn && q < a.Lq) {
#pragma unroll
        for (int i = 0; i < TOTALS; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = (i / NB * KG + kg) * BN + i % NB * 32 + 4 * hh + 8 * (r / 4) + r % 4;
            if (key < a.Lk) unsafeAtomicAdd(mine + at - codes[key], total[i][r]);
          }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  if (TABLE) {
    __syncthreads();  // (the zeros, where no tile of keys came between)
    // what the padding holds belongs to the ends
    far_lo += mine[lane];  // slots 0 .. PAD - 1
    far_hi += mine[a.pos.n + PAD + lane];
    far_lo = wave_sum(far_lo);
    far_hi = wave_sum(far_hi);
    if (lane == 0) {
      mine[PAD] += far_lo;
      mine[PAD + a.pos.n - 1] += far_hi;
    }
    __syncthreads();
    float* dst = g.parts + (static_cast<int64_t>(h) * chunks * q_tiles + chunk * q_tiles + tile) * a.pos.n;
    for (int t = threadIdx.x; t < a.pos.n; t += KG * NT) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < KG * NW; ++w) v += sums[w * np + PAD + t];
      dst[t] = v;
    }
  }
}

// ---------------------------------------------------------------------------
// dK and dV
// ---------------------------------------------------------------------------
// The query heads that share a key head may be split between workgroups, whose float32
// sums dkv_join_kernel adds in order.
template <typename T, int DP, int NW, int KG, bool WIDE>
__global__ __launch_bounds__(NW * 64 * KG, sizeof(T) == 2 ? (DP == 32 ? 3 : DP == 64 ? 2 : 1) : 1) void rel_attention_dkv_kernel(
    RelAttn a, Grads g, int k_tiles, int splits) {
  constexpr int NT = NW * 64;
  using M = Mat<T>;
  using TL = Tile<T, DP>;
  constexpr int BM = Shape<T, DP>::BN, NB = BM / 32, CH = DP / 16, OB = DP / 32;
  constexpr int BUFS = Shape<T, DP>::BUFS;
  extern __shared__ __align__(16) unsigned char smem[];
  static_assert(KG == 1 || BUFS == 2, "a second group");
  const int kg = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0;
  T* qt = reinterpret_cast<T*>(smem) + kg * 2 * BUFS * BM * TL::LD;
  T* gt = qt + BUFS * BM * TL::LD;
  float* eb = reinterpret_cast<float*>(reinterpret_cast<T*>(smem) + KG * 2 * BUFS * BM * TL::LD);
  const int np = a.pos.n + 2 * PAD;
  float* ls = eb + (np + 3) / 4 * 4 + kg * 4 * BM;  // [2][BM]: each query's shift
  float* dd = ls + 2 * BM;                          // [2][BM]: and D_i
  int* codes = reinterpret_cast<int*>(eb + (np + 3) / 4 * 4 + KG * 4 * BM);  // of a window's queries
  const int tid = threadIdx.x - kg * NT, lane = tid & 63, hh = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned wg = xcd_tile(blockIdx.x, gridDim.x);
  const int tile = int(wg % k_tiles), split = int(wg / k_tiles) % splits;
  const int hk = int(wg / k_tiles / splits) % a.Hk, b = int(wg / k_tiles / splits) / a.Hk;
  const int group = a.H / a.Hk, hg0 = split * group / splits, hg1 = (split + 1) * group / splits;
  const int kw = tile * (NW * 32) + wave * 32;  // the wave's first key
  const int key = kw + col, kc = min(key, a.Lk - 1), s0 = a.start(b), len = a.keys(b);
  const int ck = a.pos.code(kc);
  const float c = a.scale * LOG2E;
  const int k_first = tile * (NW * 32);
  if (a.pos.grid_w) load_codes(codes, a.pos, a.Lq, threadIdx.x, NT * KG);

  typename M::V8 kf[CH], vf[CH];
  load_row<T, WIDE>(kf, Rows<T>(static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h + k_first * a.ks.t, a.ks.t),
              key - k_first, 8 * hh, a.D, a.vec, key < len);
  load_row<T, WIDE>(vf, Rows<T>(static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h + k_first * a.vs.t, a.vs.t),
              key - k_first, 8 * hh, a.D, a.vec, key < len);
  f32x16 dk[OB], dv[OB];
#pragma unroll
  for (int i = 0; i < OB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[i][r] = dv[i][r] = 0.0f;

  // queries that see any key of the workgroup: from `first` on
  int first = 0;
  if (a.causal) {
    const int64_t f = static_cast<int64_t>(k_first) - s0;
    first = static_cast<int>(max<int64_t>(0, min<int64_t>(f, a.Lq)));
  }
  const int t0 = first / BM / KG * KG;  // (a tile's buffer goes by t / KG)
  const int tiles = k_first < len ? (a.Lq + BM - 1) / BM : 0;
  TileLoad<T, DP, BM, NT, WIDE> ql, gl;
  float lse_r = 0.0f, d_r = 0.0f;
  float row_lse[TileLoad<T, DP, BM, NT, WIDE>::N];  // of the rows that this thread brings

  for (int hg = hg0; hg < hg1; ++hg) {
    const int h = hk * group + hg;
    const uint8_t* mask = a.mask_of(b, h);
    const T* qb = static_cast<const T*>(a.q) + b * a.qs.b + h * a.qs.h;
    const T* gb = static_cast<const T*>(g.dout) + b * g.gs.b + h * g.gs.h;
    const int64_t row0 = (static_cast<int64_t>(b) * a.H + h) * a.Lq;
    auto load = [&](int t) {
      const int i0 = t * BM;
      ql.load(qb + i0 * a.qs.t, a.qs.t, a.Lq - i0, a.D, a.vec, tid);
      gl.load(gb + i0 * g.gs.t, g.gs.t, a.Lq - i0, a.D, a.vec, tid);
#pragma unroll
      for (int i = 0; i < ql.N; ++i) {
        const int r = t * BM + (tid + i * NT) / ql.PER_ROW;
        row_lse[i] = r < a.Lq ? g.lse[row0 + r] : INF;
      }
      if (tid < BM) {
        const int i = t * BM + tid;
        lse_r = i < a.Lq ? g.lse[row0 + i] : INF;
        d_r = i < a.Lq ? g.dsum[row0 + i] : 0.0f;
      }
    };
    auto store = [&](int t) {
      // a query that sees no key may hold anything, and 0 x anything has to be 0
#pragma unroll
      for (int i = 0; i < ql.N; ++i)
        if (row_lse[i] == INF)
#pragma unroll
          for (int e = 0; e < 8; ++e) ql.r[i][e] = gl.r[i][e] = T(0);
      ql.store(qt + (t / KG % BUFS) * BM * TL::LD, tid);
      gl.store(gt + (t / KG % BUFS) * BM * TL::LD, tid);
      bool factors = false;
#pragma unroll
      for (int i = 0; i < ql.N; ++i) factors |= has_factor(row_lse[i]);
      if (__ballot(factors)) {  // (as in dQ; each thread what it stored)
        T* tile = gt + (t / KG % BUFS) * BM * TL::LD;
#pragma unroll 1
        for (int piece = afresh(tid); piece < BM * ql.PER_ROW; piece += NT) {
          const int r = piece / ql.PER_ROW, i = t * BM + r;
          const float f = i < a.Lq ? factor_of(a, g, row0 + i, g.lse[row0 + i]) : 1.0f;
          T* p = tile + r * TL::LD + piece % ql.PER_ROW * 8;
#pragma unroll 1
          for (int e = 0; e < 8; ++e) p[e] = T(widen(p[e]) * f);
        }
      }
      if (tid < BM) {
        ls[(t / KG & 1) * BM + tid] = lse_r;
        dd[(t / KG & 1) * BM + tid] = d_r;
      }
    };
    __syncthreads();  // the head before is done with its tiles and bias
    load_bias<T>(eb, a, h, 1, threadIdx.x, NT * KG);
    if (t0 + kg < tiles) {
      load(t0 + kg);
      store(t0 + kg);
    }
    const int rounds = tiles > t0 ? (tiles - t0 + KG - 1) / KG : 0;
    for (int round = 0; round < rounds; ++round) {
      const int t = t0 + round * KG + kg;
      __syncthreads();
      if (KG > 1 && t >= tiles) continue;  // (in the last round)
      const T* qq = qt + (t / KG % BUFS) * BM * TL::LD;
      const T* gg = gt + (t / KG % BUFS) * BM * TL::LD;
      const float* lt = ls + (t / KG & 1) * BM;
      const float* dt = dd + (t / KG & 1) * BM;
      const bool more = t + KG < tiles;
      if (more) load(t + KG);
      auto work = [&](auto mode, float far) {
      constexpr int MODE = decltype(mode)::value;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int i0 = t * BM + nb * 32;  // the block's first query
        if (MODE == ANY && ((a.causal && s0 + i0 + 31 < kw) || kw >= len || i0 >= a.Lq)) continue;
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          s = M::mma(TL::straight(qq, nb * 32 + col, 16 * i + 8 * hh), kf[i], s);
          dp = M::mma(TL::straight(gg, nb * 32 + col, 16 * i + 8 * hh), vf[i], dp);
        }
        // (a query that sees no key, or stands past Lq, hides its pairs by one of these)
        const bool partial = MODE == ANY && (mask || kw + 32 > len || i0 + 32 > a.Lq ||
                                             (a.causal && kw + 31 > s0 + i0));
        int kind = NEAR;
        if (MODE == FAR) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = s[r] * c + far;
        } else if (MODE == ANY && a.pos.grid_w == 0) {
          kind = block_kind(a.pos, s0 + i0 - (kw + 31), s0 + i0 + 31 - kw);
          if (kind == NEAR) {
            const float* e = eb + (s0 + i0 + 4 * hh - key - a.pos.lo + PAD);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = s[r] * c + e[8 * (r / 4) + r % 4];
          } else {
            const float e = kind == ALL_BELOW ? eb[0] : eb[np - 1];
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = s[r] * c + e;
          }
        } else {
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const int4 cq = *reinterpret_cast<const int4*>(codes + i0 + 4 * hh + 8 * r4);
            const float* e = eb + PAD - ck - a.pos.lo;
            s[4 * r4] = s[4 * r4] * c + e[cq.x];
            s[4 * r4 + 1] = s[4 * r4 + 1] * c + e[cq.y];
            s[4 * r4 + 2] = s[4 * r4 + 2] * c + e[cq.z];
            s[4 * r4 + 3] = s[4 * r4 + 3] * c + e[cq.w];
          }
        }
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 l4 = *reinterpret_cast<const f32x4*>(lt + nb * 32 + 8 * r4 + 4 * hh);
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(dt + nb * 32 + 8 * r4 + 4 * hh);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * r4 + e;
            s[r] = __builtin_amdgcn_exp2f(s[r] - l4[e]);
            dp[r] = s[r] * (dp[r] - d4[e]);
          }
        }
        if (partial) {
          // queries from the key's position on, those before Lq
          const int i = i0 + 4 * hh, from = a.causal ? key - s0 - i : 0;
          uint32_t seen = key < len ? ~first_bits(from) & first_bits(a.Lq - i) : 0;
          if (mask && key < len) seen &= mask_bits(mask + i * a.mq + afresh(key) * a.mk, a.mq, a.Lq - i);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!(seen >> r & 1)) s[r] = dp[r] = 0.0f;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          typename M::V8 p, ds;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            p[i] = T(s[8 * half + i]);
            ds[i] = T(dp[8 * half + i]);
          }
#pragma unroll
          for (int i = 0; i < OB; ++i) {
            typename M::V8 gf = TL::transposed(gg, nb * 32 + 16 * half, 32 * i, lane);
            typename M::V8 qf = TL::transposed(qq, nb * 32 + 16 * half, 32 * i, lane);
            dv[i] = M::mma(gf, p, dv[i]);
            dk[i] = M::mma(qf, ds, dk[i]);
          }
        }
      }
      };
      const int q0 = t * BM, q1 = q0 + BM;  // the tile's queries
      const bool all = !mask && kw + 32 <= len && q1 <= a.Lq && (!a.causal || kw + 31 <= s0 + q0);
      const int kind = block_kind(a.pos, s0 + q0 - (kw + 31), s0 + q1 - 1 - kw);
      if (all && a.pos.grid_w)
        work(std::integral_constant<int, WINDOW>(), 0.0f);
      else if (const float far = far_bias(eb, np, kind); all && kind != NEAR && __builtin_fabsf(far) < FAR_MOST)
        work(std::integral_constant<int, FAR>(), far);
      else
        work(std::integral_constant<int, ANY>(), 0.0f);
      if (more) {
        if (BUFS == 1) __syncthreads();
        store(t + KG);
      }
    }
  }
  if constexpr (KG > 1) {
    static_assert(KG == 2, "the second group's sums join the first's");
    float* joint = reinterpret_cast<float*>(smem) + wave * OB * 32 * 64 + lane;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (kg == 1) {
          joint[(32 * i + r) * 64] = dk[i][r];
          joint[(32 * i + 16 + r) * 64] = dv[i][r];
        }
    __syncthreads();
    if (kg == 1) return;
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        dk[i][r] += joint[(32 * i + r) * 64];
        dv[i][r] += joint[(32 * i + 16 + r) * 64];
      }
  }
  if (key < a.Lk && splits > 1) {
    const int64_t each = static_cast<int64_t>(a.B) * a.Hk * a.Lk * a.D;
    float* krow = g.joint + 2 * split * each + ((static_cast<int64_t>(b) * a.Hk + hk) * a.Lk + key) * a.D;
    float* vrow = krow + each;
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = 32 * i + 8 * (r / 4) + 4 * hh + r % 4;
        if (d < a.D) {
          krow[d] = dk[i][r] * a.scale;
          vrow[d] = dv[i][r];
        }
      }
  } else if (key < a.Lk) {
    T* krow_o = static_cast<T*>(g.dk) + b * g.dks.b + hk * g.dks.h + key * g.dks.t;
    T* vrow_o = static_cast<T*>(g.dv) + b * g.dvs.b + hk * g.dvs.h + key * g.dvs.t;
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        float w[4], x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = dk[i][4 * e4 + e] * a.scale;
          x[e] = dv[i][4 * e4 + e];
        }
        store4<T>(krow_o, 32 * i + 8 * e4 + 4 * hh, a.D, g.dkvec, w);
        store4<T>(vrow_o, 32 * i + 8 * e4 + 4 * hh, a.D, g.dkvec, x);
      }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void dkv_join_kernel(RelAttn a, Grads g, int splits) {
  const int64_t each = static_cast<int64_t>(a.B) * a.Hk * a.Lk * a.D;
  for (int64_t t = blockIdx.x * static_cast<int64_t>(256) + threadIdx.x; t < 2 * each;
       t += static_cast<int64_t>(gridDim.x) * 256) {
    float v = 0.0f;
    for (int s = 0; s < splits; ++s) v += g.joint[2 * s * each + t];
    const bool second = t >= each;
    const int64_t e = second ? t - each : t, row = e / a.D;
    const int d = static_cast<int>(e - row * a.D), key = static_cast<int>(row % a.Lk);
    const int hk = static_cast<int>(row / a.Lk) % a.Hk, b = static_cast<int>(row / a.Lk / a.Hk);
    const View& st = second ? g.dvs : g.dks;
    static_cast<T*>(second ? g.dv : g.dk)[b * st.b + hk * st.h + key * st.t + d] = T(v);
  }
}

inline int tiles_of(int n, int nw) { return (n + nw * 32 - 1) / (nw * 32); }

// How a call is laid out over the card.  Four waves to a workgroup, two where four leave
// compute units without one (a causal line of 2048 in bfloat16, 256 workgroups of four: dQ
// 75 us against 103 of two, dK and dV 56 against 116; a line of 777 in float32, 112 and 28
// of four: dQ 132 against 83, dK and dV, the shared heads split, 137 against 84).
struct Plan {
  int nw_q, nw_k;  // waves of the workgroups that own queries, and keys
  int kg_q, kg_k;  // groups of them
  int chunks;      // batch entries in parallel for dQ: all, unless windows' sums stay in registers
  bool registers;
  int splits;      // of the query heads of a key head
};
inline Plan plan_of(int B, int H, int Hk, int Lq, int Lk, int D, int grid_w, bool table, int device) {
  Plan p;
  const int64_t enough = 2 * cu_count(device);
  p.registers = table && grid_w > 0 && Lq <= 256 && D <= 64;
  p.nw_q = p.registers || static_cast<int64_t>(B) * H * tiles_of(Lq, 4) >= cu_count(device) ? 4 : 2;
  p.nw_k = static_cast<int64_t>(B) * Hk * tiles_of(Lk, 4) >= cu_count(device) ? 4 : 2;
  p.kg_q = p.kg_k = 1;
  if (D <= 64) {
    // (windows: half of the sums by pair in each group leaves room for two waves on a SIMD)
    if (p.registers || (static_cast<int64_t>(B) * H * tiles_of(Lq, p.nw_q) < enough && Lk > 128)) p.kg_q = 2;
    if (static_cast<int64_t>(B) * Hk * tiles_of(Lk, p.nw_k) < enough && Lq > 128) p.kg_k = 2;
  }
  p.chunks = B;
  if (p.registers) {  // two workgroups for every compute unit
    const int64_t each = static_cast<int64_t>(H) * tiles_of(Lq, 4), want = (enough + each - 1) / each;
    p.chunks = static_cast<int>(want < B ? want : B);
  }
  const int64_t wgs = static_cast<int64_t>(B) * Hk * tiles_of(Lk, p.nw_k), most = H / Hk;
  const int64_t want = (enough + wgs - 1) / wgs;
  p.splits = static_cast<int>(want < most ? want : most);
  return p;
}

template <typename T, int DP, int NW, int KG, bool WIDE>
int launch_dq(const RelAttn& a, const Grads& g, const Plan& p, hipStream_t s) {
  const int qt = tiles_of(a.Lq, NW);
  const int64_t wgs = static_cast<int64_t>(p.chunks) * a.H * qt;
  if (wgs > 0x7fffffff) return FA_E_SHAPE;
  const size_t np = a.pos.n + 2 * PAD, tiles = KG * 2 * Shape<T, DP>::BUFS * Shape<T, DP>::TILE;
  const size_t lds = tiles + ((g.parts ? 1 + KG * NW : 1) * np + 3) / 4 * 16 +
                     (a.pos.grid_w ? codes_room(a.Lk) * sizeof(int) : 0);
  if constexpr (KG > 1)  // a table that leaves no room for the second group's sums
    if (lds > MOST_LDS) return launch_dq<T, DP, NW, 1, WIDE>(a, g, p, s);
  auto dq = g.parts ? rel_attention_dq_kernel<T, DP, NW, KG, true, WIDE, 0>
                    : rel_attention_dq_kernel<T, DP, NW, KG, false, WIDE, 0>;
  if constexpr (DP <= 64 && NW == 4)
    if (p.registers)
      dq = a.Lq <= 128 ? rel_attention_dq_kernel<T, DP, NW, KG, true, WIDE, 4>
                       : rel_attention_dq_kernel<T, DP, NW, KG, true, WIDE, 8>;
  if (const int e = launch_lds(dq, lds)) return e;
  dq<<<static_cast<unsigned>(wgs), NW * 64 * KG, lds, s>>>(a, g, qt, p.chunks);
  FA_LAUNCH_CHECK();
  return FA_OK;
}

template <typename T, int DP, int NW, int KG, bool WIDE>
int launch_dkv(const RelAttn& a, const Grads& g, const Plan& p, hipStream_t s) {
  const int kt = tiles_of(a.Lk, NW);
  const int64_t wgs = static_cast<int64_t>(a.B) * a.Hk * kt * p.splits;
  if (wgs > 0x7fffffff) return FA_E_SHAPE;
  const size_t np = a.pos.n + 2 * PAD, tiles = KG * 2 * Shape<T, DP>::BUFS * Shape<T, DP>::TILE;
  const size_t lds = tiles + ((np + 3) / 4 * 4 + KG * 4 * Shape<T, DP>::BN) * sizeof(float) +
                     (a.pos.grid_w ? codes_room(a.Lq) * sizeof(int) : 0);
  auto dkv = rel_attention_dkv_kernel<T, DP, NW, KG, WIDE>;
  if (const int e = launch_lds(dkv, lds)) return e;
  dkv<<<static_cast<unsigned>(wgs), NW * 64 * KG, lds, s>>>(a, g, kt, p.splits);
  FA_LAUNCH_CHECK();
  return FA_OK;
}

template <typename T, int DP, bool WIDE>
int launch_wide(const RelAttn& a, const Grads& g, const Plan& p, hipStream_t s) {
  int e;
  if constexpr (DP <= 64) {
    if (p.kg_q == 2)
      e = p.nw_q == 4 ? launch_dq<T, DP, 4, 2, WIDE>(a, g, p, s) : launch_dq<T, DP, 2, 2, WIDE>(a, g, p, s);
    else
      e = p.nw_q == 4 ? launch_dq<T, DP, 4, 1, WIDE>(a, g, p, s) : launch_dq<T, DP, 2, 1, WIDE>(a, g, p, s);
    if (e) return e;
    if (p.kg_k == 2)
      e = p.nw_k == 4 ? launch_dkv<T, DP, 4, 2, WIDE>(a, g, p, s) : launch_dkv<T, DP, 2, 2, WIDE>(a, g, p, s);
    else
      e = p.nw_k == 4 ? launch_dkv<T, DP, 4, 1, WIDE>(a, g, p, s) : launch_dkv<T, DP, 2, 1, WIDE>(a, g, p, s);
  } else {
    e = p.nw_q == 4 ? launch_dq<T, DP, 4, 1, WIDE>(a, g, p, s) : launch_dq<T, DP, 2, 1, WIDE>(a, g, p, s);
    if (e) return e;
    // (float32: a thread of two waves would hold 64 registers of tiles on their way beside
    // 256 of fragments and sums, which the compiler does not allocate)
    if constexpr (sizeof(T) == 4)
      e = launch_dkv<T, DP, 4, 1, WIDE>(a, g, p, s);
    else
      e = p.nw_k == 4 ? launch_dkv<T, DP, 4, 1, WIDE>(a, g, p, s) : launch_dkv<T, DP, 2, 1, WIDE>(a, g, p, s);
  }
  if (e || p.splits == 1) return e;
  const int64_t want = (2 * static_cast<int64_t>(a.B) * a.Hk * a.Lk * a.D + 255) / 256;
  dkv_join_kernel<T><<<static_cast<unsigned>(want < 4096 ? want : 4096), 256, 0, s>>>(a, g, p.splits);
  FA_LAUNCH_CHECK();
  return FA_OK;
}

template <typename T, int DP>
int launch_dim(const RelAttn& a, const Grads& g, const Plan& p, hipStream_t s) {
  return a.vec * sizeof(T) == 16 ? launch_wide<T, DP, true>(a, g, p, s) : launch_wide<T, DP, false>(a, g, p, s);
}

template <typename T>
int backward(RelAttn a, Grads g, int rows, void* dtable, const Plan& p, hipStream_t s) {
  const void* in[5] = {a.q, a.k, a.v, g.out, g.dout};
  const View iv[5] = {a.qs, a.ks, a.vs, g.os, g.gs};
  a.vec = widest_load<T>(in, iv, 5, a.D);
  const void* dqp[1] = {g.dq};
  g.dqvec = widest_load<T>(dqp, &g.dqs, 1, a.D);
  const void* dkp[2] = {g.dk, g.dv};
  const View dkv[2] = {g.dks, g.dvs};
  g.dkvec = widest_load<T>(dkp, dkv, 2, a.D);
  int e;
  if (a.D <= 32) e = launch_dim<T, 32>(a, g, p, s);
  else if (a.D <= 64) e = launch_dim<T, 64>(a, g, p, s);
  else e = launch_dim<T, 128>(a, g, p, s);
  if (e) return e;
  if (dtable) {
    launch_table_sum<T>(a, g.parts, p.chunks * tiles_of(a.Lq, p.nw_q), rows, dtable, s);
    FA_LAUNCH_CHECK();
  }
  return FA_OK;
}

inline int64_t align16(int64_t v) { return (v + 15) / 16 * 16; }

// The workspace: D_i, the table's sums, the split heads' sums.
struct Room {
  int64_t parts, joint, bytes;
};
inline Room bwd_room(int B, int H, int Hk, int Lq, int Lk, int D, int n, int grid_w, bool table, int device) {
  const Plan p = plan_of(B, H, Hk, Lq, Lk, D, grid_w, table, device);
  Room r;
  r.parts = align16(static_cast<int64_t>(B) * H * Lq * 4);
  // (a row for each workgroup of dQ, or of the windows' kernel: at most one for each
  // entry of the batch then)
  int64_t rows = static_cast<int64_t>(p.chunks) * tiles_of(Lq, p.nw_q);
  if (grid_w > 0 && Lq <= 64) rows = rows > window_parts(B, H, device) ? rows : window_parts(B, H, device);
  r.joint = r.parts + (table ? align16(H * rows * n * 4) : 0);
  r.bytes = r.joint + (p.splits > 1 ? 2 * p.splits * static_cast<int64_t>(B) * Hk * Lk * D * 4 : 0);
  return r;
}

}  // namespace
}  // namespace fa

extern "C" {

FA_API int fa_gpu_rel_attention_backward_workspace(int B, int H, int Hk, int Lq, int Lk, int D, int n,
                                                   int grid_w, int need_table, int device,
                                                   int64_t* out_bytes) {
  using namespace fa;
  if (!out_bytes) return FA_E_ARG;
  if (n < 1 || n > FA_REL_MAX || grid_w < 0) return FA_E_SHAPE;
  if (const int e = check_attention(B, H, Hk, Lq, Lk, D, nullptr, 1, nullptr)) return e;
  *out_bytes = bwd_room(B, H, Hk, Lq, Lk, D, n, grid_w, need_table != 0, device).bytes;
  return FA_OK;
}

FA_API int fa_gpu_rel_attention_backward(
    const void* q, const void* k, const void* v, const void* out, const void* dout,
    const float* lse, int dtype, int B, int H, int Hk, int Lq, int Lk, int D,
    const int64_t* strides, const void* table, int rows, const int* row_of, int lo, int n,
    int grid_w, int64_t q_start, const int* q_starts, const int* key_lengths, const uint8_t* mask,
    int mask_b, const int64_t* mask_strides, int causal, double scale, void* dq, void* dk,
    void* dv, void* dtable, void* workspace, int64_t workspace_bytes, int device, void* stream) {
  using namespace fa;
  if (!q || !k || !v || !out || !dout || !lse || !strides || !table || !dq || !dk || !dv ||
      !workspace)
    return FA_E_ARG;
  const bool table_f32 = dtype & FA_TABLE_F32;
  dtype &= ~FA_TABLE_F32;
  if (const int e = check_attention(B, H, Hk, Lq, Lk, D, mask, mask_b, mask_strides)) return e;
  if (const int e = check_relpos(row_of, rows, lo, n, grid_w, Lq, Lk, q_start, q_starts)) return e;
  if (const int e = check_strides(strides, 8, dtype)) return e;
  const Room room = bwd_room(B, H, Hk, Lq, Lk, D, n, grid_w, dtable != nullptr, device);
  if (workspace_bytes < room.bytes) return FA_E_ARG;
  DeviceScope scope(device);
  if (scope.status != hipSuccess) return -static_cast<int>(scope.status);
  const RelAttn a = rel_attn_args(q, k, v, B, H, Hk, Lq, Lk, D, strides, table, table_f32,
                                  RelPos{row_of, lo, n, grid_w}, q_start, q_starts, key_lengths,
                                  mask, mask_b, mask_strides, causal, scale);
  Grads g{};
  g.out = out;
  g.dout = dout;
  g.os = {strides[9], strides[10], strides[11]};
  g.gs = {strides[12], strides[13], strides[14]};
  g.dqs = {strides[15], strides[16], strides[17]};
  g.dks = {strides[18], strides[19], strides[20]};
  g.dvs = {strides[21], strides[22], strides[23]};
  g.lse = lse;
  g.dsum = static_cast<float*>(workspace);
  char* ws = static_cast<char*>(workspace);
  g.parts = dtable ? reinterpret_cast<float*>(ws + room.parts) : nullptr;
  g.joint = reinterpret_cast<float*>(ws + room.joint);
  g.dq = dq;
  g.dk = dk;
  g.dv = dv;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (window_serve(a)) {
    const WindowGrads w{dout, g.gs, dq, dk, dv, g.dqs, g.dks, g.dvs, g.parts};
    return window_backward(dtype, a, w, rows, dtable, device, s);
  }
  const Plan p = plan_of(B, H, Hk, Lq, Lk, D, grid_w, dtable != nullptr, device);
  switch (dtype) {
    case FA_F16: return backward<_Float16>(a, g, rows, dtable, p, s);
    case FA_BF16: return backward<__bf16>(a, g, rows, dtable, p, s);
    case FA_F32: return backward<float>(a, g, rows, dtable, p, s);
    default: return FA_E_DTYPE;
  }
}

}  // extern "C"
