// Attention in windows of up to 64 tokens with a relative position bias, forward and
// backward.
//
// Thousands of such windows make a layer, each a few kilobytes of queries, keys and
// values, so the memory's rate bounds it: every tensor is to be moved once.  A
// workgroup of two waves takes one head's share of the windows, one after the other, the
// next window on its way in registers.  A wave holds 32 queries and all keys: a row's
// softmax needs no running maximum, the bias stays in registers from window to window,
// and so do the sums of dS by pair, which reach the table's differences once at the end.
//
// Backward in one kernel, from q, k, v and dout alone: with P and dP of a whole row in
// registers D = sum P dP is exact to float32 (no rounded output enters), P and dS pass
// through LDS once, rounded, and the wave that owned queries then owns keys for dV =
// P^T dout and dK = dS^T Q.
#include "fa_rel_attention.h"

namespace fa {
namespace {

constexpr int NW = 2, NT = NW * 64, L = 64;

// How the tensors are read: one element, a pair or 16 bytes at once.
enum : int { ONE = 0, PAIR = 1, WIDE = 2 };
template <typename T, int DP, int ACCESS>
using Load = typename std::conditional<ACCESS == PAIR, PairLoad<T, DP, L, NT>,
                                       TileLoad<T, DP, L, NT, ACCESS == WIDE>>::type;

template <typename T, int DP> constexpr size_t tile_bytes() { return size_t(L) * Tile<T, DP>::LD * sizeof(T); }

// The pairs of one lane: query qw + l % 32 with keys 32 nb + 4 h + 8 (r / 4) + r % 4.
struct Pairs {
  int q, qc, hh;
  __device__ inline int key(int nb, int r) const { return 32 * nb + 4 * hh + 8 * (r / 4) + r % 4; }
};

// Bit 16 nb + r: whether the lane's pair counts, by its position alone ...
__device__ inline uint32_t reachable(const RelAttn& a, const Pairs& p, int len) {
  uint32_t bits = 0;
#pragma unroll 1
  for (int t = 0; t < 32; ++t) {
    const int k = p.key(t >> 4, t & 15);
    if (k < len && (!a.causal || k <= p.q)) bits |= 1u << t;
  }
  return bits;
}

// ... and by the mask.  Its bytes are 0 or 1.  Where its rows are 64 aligned bytes a lane
// reads half of its query's row, 32 bytes in two reads, and the halves of the wave exchange
// every other word: four bytes at a time, the bits that it needs, each read touches 32
// rows (24576 windows forward and backward 687 us so, and with scratch in the loops; 634 us
// without both).  The words of the next window are read
// with its tiles: memory answers in order, and a read made later would wait for them.
struct MaskWords {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  u32x4 row[2];
  __device__ inline void load(const RelAttn& a, const Pairs& p, int b, int h) {
    const __amdgpu_buffer_rsrc_t rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.mask_of(b, h)), 0, 0x7fffffff, 0x00020000);
    const int at = p.qc * static_cast<int>(a.mq) + 32 * p.hh;
    row[0] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0);
    row[1] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at + 16, 0, 0);
  }
  // word w of the row is keys 4 w ..; group t of a lane's bits is word 2 t + h.  A product
  // gathers a word's bytes into four bits.
  __device__ inline uint32_t bits() const {
    uint32_t r = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const auto w = __builtin_amdgcn_permlane32_swap(row[t >> 1][2 * (t & 1)], row[t >> 1][2 * (t & 1) + 1],
                                                      false, false);
      r |= (w[0] * 0x01020408u >> 24 & 15u) << (4 * t);
      r |= (w[1] * 0x01020408u >> 24 & 15u) << (16 + 4 * t);
    }
    return r;
  }
};
__device__ inline uint32_t allowed(const RelAttn& a, const Pairs& p, int b, int h) {
  const uint8_t* mask = a.mask_of(b, h);
  uint32_t bits = 0;
#pragma unroll 1
  for (int t = 0; t < 32; ++t) {
    const int k = p.key(t >> 4, t & 15);
    if (k < a.Lk && mask[p.qc * a.mq + k * a.mk]) bits |= 1u << t;
  }
  return bits;
}

// The wave's 32 rows of a block (C layout, transposed: lane l's row is l % 32) to memory by
// way of LDS of the wave's own, so that neighbouring lanes write neighbouring
// elements; rows from `valid` on and elements from D on are dropped.
template <typename T, int DP, int ACCESS>
__device__ inline void store_rows(T* own, const f32x16 (&acc)[DP / 32], float f, T* base, int64_t stride,
                                  int row0, int valid, int D, int lane) {
  constexpr int LD = Tile<T, DP>::LD;
  const int hh = lane >> 5, col = lane & 31;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      typename Mat<T>::V4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = T(acc[i][4 * g + e] * f);
      *reinterpret_cast<typename Mat<T>::V4*>(own + col * LD + 32 * i + 8 * g + 4 * hh) = w;
    }
  wave_sync();
  constexpr int W = ACCESS == WIDE ? 16 / int(sizeof(T)) : ACCESS == PAIR ? 2 : 1, PER_ROW = DP / W;
  constexpr int STEP = 64 / PER_ROW;  // rows between a lane's pieces
  static_assert(STEP > 0, "a row fits the wave");
  lane = afresh(lane);
  const int first = lane / PER_ROW, d = lane % PER_ROW * W;
  valid = d < D ? valid - row0 : 0;
#pragma unroll
  for (int i = 0; i < 32 / STEP; ++i) {
    const int row = first + i * STEP;
    const Rows<T> rows(base + (row0 + i * STEP) * stride, stride);
    const int at = row < valid ? first * rows.stride + d * int(sizeof(T)) : OUTSIDE;
    const T* from = own + row * LD + d;
    if constexpr (W * sizeof(T) == 16) {
      typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
      __builtin_amdgcn_raw_buffer_store_b128(*reinterpret_cast<const u32x4*>(from), rows.rsrc, at, 0, 0);
    } else if constexpr (W * sizeof(T) == 4) {
      __builtin_amdgcn_raw_buffer_store_b32(*reinterpret_cast<const unsigned*>(from), rows.rsrc, at, 0, 0);
    } else {
      __builtin_amdgcn_raw_buffer_store_b16(*reinterpret_cast<const unsigned short*>(from), rows.rsrc, at, 0, 0);
    }
  }
  wave_sync();
}

template <typename T>
__device__ inline void load_pair_bias(float (&bias)[2][16], const RelAttn& a, const Pairs& p, int h) {
  const int cq = a.pos.code(p.qc);
  with_table<T>(a, [&](auto* table) {
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = a.pos.row_of[a.pos.slot(cq - a.pos.code(min(p.key(nb, r), a.Lk - 1)))];
        bias[nb][r] = bias_log2(widen(table[static_cast<int64_t>(row) * a.H + h]));
      }
  });
}

// Scores of the wave's queries, hidden ones -inf; their maximum (0 where there is none).
template <typename T, int DP>
__device__ inline float scores(f32x16 (&s)[2], const T* kt, const typename Mat<T>::V8 (&qf)[DP / 16],
                               const float (&bias)[2][16], float c, bool all, uint32_t seen, int col,
                               int hh) {
  float top = -INF;
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[nb][r] = 0.0f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
      s[nb] = Mat<T>::mma(Tile<T, DP>::straight(kt, 32 * nb + col, 16 * i + 8 * hh), qf[i], s[nb]);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[nb][r] = s[nb][r] * c + bias[nb][r];
    if (!all) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[nb][r] = seen >> (16 * nb + r) & 1 ? s[nb][r] : -INF;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[nb][r]);
  }
  return both_max(top);
}

template <typename T, int DP, int ACCESS>
__global__ __launch_bounds__(NT, 2) void window_kernel(RelAttn a, T* out, View os, int chunks) {
  using M = Mat<T>;
  using TL = Tile<T, DP>;
  constexpr int CH = DP / 16, OB = DP / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  T* qt = reinterpret_cast<T*>(smem);
  T* kt = qt + L * TL::LD;
  T* vt = kt + L * TL::LD;
  T* ot = vt + L * TL::LD;
  __shared__ int wild[NW];  // whether a wave brought a value that is not finite
  const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned wg = xcd_tile(blockIdx.x, gridDim.x);
  const int h = int(wg % a.H), chunk = int(wg / a.H);
  const Pairs p{wave * 32 + col, min(wave * 32 + col, a.Lq - 1), hh};
  const float c = a.scale * LOG2E;
  float bias[2][16];
  load_pair_bias<T>(bias, a, p, h);
  const uint32_t reach = reachable(a, p, a.Lk);
  Load<T, DP, ACCESS> ql, kl, vl;
  MaskWords words;
  auto load = [&](int b) {
    const int len = a.keys(b);
    if (a.mask64) words.load(a, p, b, h);
    ql.load(static_cast<const T*>(a.q) + b * a.qs.b + h * a.qs.h, a.qs.t, a.Lq, a.D, a.vec, tid);
    kl.load(static_cast<const T*>(a.k) + b * a.ks.b + h * a.ks.h, a.ks.t, len, a.D, a.vec, tid);
    vl.load(static_cast<const T*>(a.v) + b * a.vs.b + h * a.vs.h, a.vs.t, len, a.D, a.vec, tid);
  };
  int len;
  uint32_t seen;
  auto store = [&](int b) {
    len = a.keys(b);
    seen = len == a.Lk ? reach : reachable(a, p, len);
    if (a.mask) seen &= a.mask64 ? words.bits() : allowed(a, p, b, h);
    ql.store(qt, tid);
    kl.store(kt, tid);
    vl.store(vt, tid);
    const bool bad = __ballot(vl.not_finite()) != 0;
    if (lane == 0) wild[wave] = bad;
  };
  load(chunk);
  store(chunk);
  for (int b = chunk; b < a.B; b += chunks) {
    __syncthreads();
    const bool tame = (wild[0] | wild[1]) == 0;
    const bool more = b + chunks < a.B;
    if (more) load(b + chunks);
    const bool all = __ballot(seen != ~0u) == 0;  // of the wave's queries
    typename M::V8 qf[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) qf[i] = TL::straight(qt, wave * 32 + col, 16 * i + 8 * hh);
    f32x16 s[2];
    const float m = scores<T, DP>(s, kt, qf, bias, c, all, seen, col, hh);
    const float sub = m == -INF ? 0.0f : m;
    float l = 0.0f;
    f32x16 o[OB];
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] = 0.0f;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[nb][r] = __builtin_amdgcn_exp2f(s[nb][r] - sub);
        l += s[nb][r];
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        typename M::V8 pf;
#pragma unroll
        for (int i = 0; i < 8; ++i) pf[i] = T(s[nb][8 * half + i]);
#pragma unroll
        for (int i = 0; i < OB; ++i) {
          const typename M::V8 vf = TL::transposed(vt, 32 * nb + 16 * half, 32 * i, lane);
          o[i] = all || tame ? M::mma(vf, pf, o[i])
                               : guarded<T>(vf, pf, o[i], seen >> (16 * nb + 8 * half));
        }
      }
    }
    l = both_sum(l);
    // the next window goes to LDS before this one's results go to memory: a wait for the
    // reads would wait for writes made before it
    __syncthreads();
    if (more) store(b + chunks);
    store_rows<T, DP, ACCESS>(ot + wave * 32 * TL::LD, o, l == 0.0f ? 0.0f : 1.0f / l, out + b * os.b + h * os.h, os.t, wave * 32,
                              a.Lq, a.D, lane);
  }
}

template <typename T, int DP, bool TABLE, int ACCESS>
__global__ __launch_bounds__(NT, 2) void window_backward_kernel(RelAttn a, const T* dout, View gs, T* dq,
                                                                View dqs, T* dk, View dks, T* dv, View dvs,
                                                                float* parts, int chunks) {
  using M = Mat<T>;
  using TL = Tile<T, DP>;
  using PL = Tile<T, L>;  // P and dS, [query][key]
  constexpr int CH = DP / 16, OB = DP / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  T* qt = reinterpret_cast<T*>(smem);
  T* gt = qt + L * TL::LD;
  T* kt = gt + L * TL::LD;
  T* vt = kt + L * TL::LD;
  T* pt = vt + L * TL::LD;
  T* dt = pt + L * PL::LD;
  float* sums = reinterpret_cast<float*>(smem);  // [NW][n], over the tiles at the end
  __shared__ int wild[NW];  // whether a wave brought a key that is not finite
  const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned wg = xcd_tile(blockIdx.x, gridDim.x);
  const int h = int(wg % a.H), chunk = int(wg / a.H);
  const Pairs p{wave * 32 + col, min(wave * 32 + col, a.Lq - 1), hh};
  const float c = a.scale * LOG2E;
  float bias[2][16], total[2][16];
  load_pair_bias<T>(bias, a, p, h);
  const uint32_t reach = reachable(a, p, a.Lk);
#pragma unroll
  for (int nb = 0; nb < 2; ++nb)
#pragma unroll
    for (int r = 0; r < 16; ++r) total[nb][r] = 0.0f;
  Load<T, DP, ACCESS> ql, gl, kl, vl;
  MaskWords words;
  auto load = [&](int b) {
    const int len = a.keys(b);
    if (a.mask64) words.load(a, p, b, h);
    ql.load(static_cast<const T*>(a.q) + b * a.qs.b + h * a.qs.h, a.qs.t, a.Lq, a.D, a.vec, tid);
    gl.load(dout + b * gs.b + h * gs.h, gs.t, a.Lq, a.D, a.vec, tid);
    kl.load(static_cast<const T*>(a.k) + b * a.ks.b + h * a.ks.h, a.ks.t, len, a.D, a.vec, tid);
    vl.load(static_cast<const T*>(a.v) + b * a.vs.b + h * a.vs.h, a.vs.t, len, a.D, a.vec, tid);
  };
  int len;
  uint32_t seen;
  auto store = [&](int b) {
    len = a.keys(b);
    seen = len == a.Lk ? reach : reachable(a, p, len);
    if (a.mask) seen &= a.mask64 ? words.bits() : allowed(a, p, b, h);
    ql.store(qt, tid);
    gl.store(gt, tid);
    kl.store(kt, tid);
    vl.store(vt, tid);
    const bool bad = __ballot(kl.not_finite()) != 0;
    if (lane == 0) wild[wave] = bad;
  };
  load(chunk);
  store(chunk);
  for (int b = chunk; b < a.B; b += chunks) {
    __syncthreads();
    const bool tame = (wild[0] | wild[1]) == 0;
    const bool more = b + chunks < a.B;
    if (more) load(b + chunks);
    const bool all = __ballot(seen != ~0u) == 0;  // of the wave's queries
    f32x16 s[2], dp[2];
    {
      typename M::V8 qf[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) qf[i] = TL::straight(qt, wave * 32 + col, 16 * i + 8 * hh);
      const float m = scores<T, DP>(s, kt, qf, bias, c, all, seen, col, hh);
      const float sub = m == -INF ? 0.0f : m;
      float l = 0.0f;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[nb][r] = __builtin_amdgcn_exp2f(s[nb][r] - sub);
          l += s[nb][r];
        }
      l = both_sum(l);
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int i = 0; i < CH; ++i) qf[i] = TL::straight(gt, wave * 32 + col, 16 * i + 8 * hh);
      float d = 0.0f;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[nb][r] = 0.0f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
          dp[nb] = M::mma(TL::straight(vt, 32 * nb + col, 16 * i + 8 * hh), qf[i], dp[nb]);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (!all && !(seen >> (16 * nb + r) & 1)) dp[nb][r] = 0.0f;
          s[nb][r] *= inv;
          d += s[nb][r] * dp[nb][r];
        }
      }
      d = both_sum(d);
      const bool none = l == 0.0f;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float x = s[nb][r] * (dp[nb][r] - d);
          if (!all && (none || !(seen >> (16 * nb + r) & 1))) x = 0.0f;
          dp[nb][r] = x;
          if (TABLE) total[nb][r] += x;
        }
      // a query that sees no key may hold anything, and 0 x anything has to be 0
      if (!all && __ballot(none)) {
        if (none)
          for (int e = hh; e < TL::LD; e += 2)
            qt[(wave * 32 + col) * TL::LD + e] = gt[(wave * 32 + col) * TL::LD + e] = T(0);
      }
    }
    f32x16 acc[OB];
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] = 0.0f;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        typename M::V8 pf, df;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pf[i] = T(s[nb][8 * half + i]);
          df[i] = T(dp[nb][8 * half + i]);
        }
        // keys 32 nb + 16 half + 4 h + {0 .. 3} and 8 further, of this lane's query
        const int at = (wave * 32 + col) * PL::LD + 32 * nb + 16 * half + 4 * hh;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          typename M::V4 x, y;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = pf[4 * e + i];
            y[i] = df[4 * e + i];
          }
          *reinterpret_cast<typename M::V4*>(pt + at + 8 * e) = x;
          *reinterpret_cast<typename M::V4*>(dt + at + 8 * e) = y;
        }
#pragma unroll
        for (int i = 0; i < OB; ++i) {
          typename M::V8 kf = TL::transposed(kt, 32 * nb + 16 * half, 32 * i, lane);
          if (!all && !tame) {
#pragma unroll
            for (int e = 0; e < 8; ++e) kf[e] = __builtin_fabsf(widen(kf[e])) < INF ? kf[e] : T(0);
          }
          acc[i] = M::mma(kf, df, acc[i]);
        }
      }
    __syncthreads();  // P and dS of all queries
    // the wave's keys: 32 wave + col
    f32x16 acc_v[OB], acc_k[OB];
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc_v[i][r] = acc_k[i][r] = 0.0f;
#pragma unroll
    for (int k = 0; k < L / 16; ++k) {
      const typename M::V8 pf = PL::transposed(pt, 16 * k, 32 * wave, lane);
      const typename M::V8 df = PL::transposed(dt, 16 * k, 32 * wave, lane);
#pragma unroll
      for (int i = 0; i < OB; ++i) {
        acc_v[i] = M::mma(TL::transposed(gt, 16 * k, 32 * i, lane), pf, acc_v[i]);
        acc_k[i] = M::mma(TL::transposed(qt, 16 * k, 32 * i, lane), df, acc_k[i]);
      }
    }
    // the next window goes to LDS before this one's results go to memory: a wait for the
    // reads would wait for writes made before it
    __syncthreads();
    if (more) store(b + chunks);
    T* own = pt + wave * 32 * PL::LD;
    store_rows<T, DP, ACCESS>(own, acc, a.scale, dq + b * dqs.b + h * dqs.h, dqs.t, wave * 32, a.Lq, a.D, lane);
    store_rows<T, DP, ACCESS>(own, acc_v, 1.0f, dv + b * dvs.b + h * dvs.h, dvs.t, wave * 32, a.Lk, a.D, lane);
    store_rows<T, DP, ACCESS>(own, acc_k, a.scale, dk + b * dks.b + h * dks.h, dks.t, wave * 32, a.Lk, a.D, lane);
  }
  if (TABLE) {
    const int n = a.pos.n;
    __syncthreads();
    for (int t = tid; t < NW * n; t += NT) sums[t] = 0.0f;
    __syncthreads();
    float* mine = sums + wave * n;
    const Pairs p2{p.q, afresh(p.qc), afresh(hh)};  // (its slots are not kept from the start)
    const int cq = a.pos.code(p2.qc);
    // within one half of the lanes one key meets 32 queries: 32 slots.  The halves add
    // one after the other, so the order of every slot's sum is fixed.
    for (int turn = 0; turn < 2; ++turn) {
      if (hh == turn && p.q < a.Lq) {
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (p2.key(nb, r) < a.Lk)
              unsafeAtomicAdd(mine + a.pos.slot(cq - a.pos.code(p2.key(nb, r))), total[nb][r]);
      }
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    for (int t = tid; t < n; t += NT)
      parts[(static_cast<int64_t>(h) * chunks + chunk) * n + t] = sums[t] + sums[n + t];
  }
}

// Workgroups that share a head's windows: `fit` for every compute unit over all heads.
inline int chunks_of(int B, int H, int device, int fit) {
  const int want = (fit * cu_count(device) + H - 1) / H;
  return want < B ? want : B;
}

template <typename T, int DP, int ACCESS>
int launch_forward(const RelAttn& a, T* out, const View& os, int chunks, hipStream_t s) {
  const size_t lds = 4 * tile_bytes<T, DP>();
  auto kernel = window_kernel<T, DP, ACCESS>;
  if (const int e = launch_lds(kernel, lds)) return e;
  kernel<<<static_cast<unsigned>(chunks * a.H), NT, lds, s>>>(a, out, os, chunks);
  FA_LAUNCH_CHECK();
  return FA_OK;
}

template <typename T, int DP, int ACCESS>
int launch_backward(const RelAttn& a, const WindowGrads& g, int chunks, hipStream_t s) {
  const size_t tiles = 4 * tile_bytes<T, DP>() + 2 * tile_bytes<T, L>();
  const size_t lds = tiles > NW * a.pos.n * sizeof(float) ? tiles : NW * a.pos.n * sizeof(float);
  auto kernel = g.parts ? window_backward_kernel<T, DP, true, ACCESS> : window_backward_kernel<T, DP, false, ACCESS>;
  if (const int e = launch_lds(kernel, lds)) return e;
  kernel<<<static_cast<unsigned>(chunks * a.H), NT, lds, s>>>(
      a, static_cast<const T*>(g.dout), g.gs, static_cast<T*>(g.dq), g.dqs, static_cast<T*>(g.dk),
      g.dks, static_cast<T*>(g.dv), g.dvs, g.parts, chunks);
  FA_LAUNCH_CHECK();
  return FA_OK;
}

template <typename T, typename Go> int with_access(int vec, const Go& go) {
  if (vec * sizeof(T) == 16) return go(std::integral_constant<int, WIDE>());
  if constexpr (sizeof(T) == 2)
    if (vec == 2) return go(std::integral_constant<int, PAIR>());
  return go(std::integral_constant<int, ONE>());
}

template <typename T>
int forward(RelAttn a, void* out, const View& os, int device, hipStream_t s) {
  const void* views[4] = {a.q, a.k, a.v, out};
  const View vs[4] = {a.qs, a.ks, a.vs, os};
  a.vec = widest_load<T>(views, vs, 4, a.D);
  const int chunks = chunks_of(a.B, a.H, device, 4);
  T* o = static_cast<T*>(out);
  auto go = [&](auto access) {
    constexpr int ACCESS = decltype(access)::value;
    return a.D <= 32 ? launch_forward<T, 32, ACCESS>(a, o, os, chunks, s)
                     : launch_forward<T, 64, ACCESS>(a, o, os, chunks, s);
  };
  return with_access<T>(a.vec, go);
}

template <typename T>
int backward(RelAttn a, const WindowGrads& g, int rows, void* dtable, int device, hipStream_t s) {
  const void* views[7] = {a.q, a.k, a.v, g.dout, g.dq, g.dk, g.dv};
  const View vs[7] = {a.qs, a.ks, a.vs, g.gs, g.dqs, g.dks, g.dvs};
  a.vec = widest_load<T>(views, vs, 7, a.D);
  const int chunks = chunks_of(a.B, a.H, device, 4);
  auto go = [&](auto access) {
    constexpr int ACCESS = decltype(access)::value;
    return a.D <= 32 ? launch_backward<T, 32, ACCESS>(a, g, chunks, s)
                     : launch_backward<T, 64, ACCESS>(a, g, chunks, s);
  };
  const int e = with_access<T>(a.vec, go);
  if (e) return e;
  if (dtable) {
    launch_table_sum<T>(a, g.parts, chunks, rows, dtable, s);
    FA_LAUNCH_CHECK();
  }
  return FA_OK;
}

}  // namespace

bool window_serve(const RelAttn& a) {
  return a.pos.grid_w > 0 && a.Lq <= L && a.H == a.Hk && a.D <= 64;
}

int window_parts(int B, int H, int device) { return chunks_of(B, H, device, 4); }

int window_forward(int dtype, const RelAttn& a, void* out, const View& os, int device, hipStream_t s) {
  switch (dtype) {
    case FA_F16: return forward<_Float16>(a, out, os, device, s);
    case FA_BF16: return forward<__bf16>(a, out, os, device, s);
    case FA_F32: return forward<float>(a, out, os, device, s);
    default: return FA_E_DTYPE;
  }
}

int window_backward(int dtype, const RelAttn& a, const WindowGrads& g, int rows, void* dtable, int device,
                    hipStream_t s) {
  switch (dtype) {
    case FA_F16: return backward<_Float16>(a, g, rows, dtable, device, s);
    case FA_BF16: return backward<__bf16>(a, g, rows, dtable, device, s);
    case FA_F32: return backward<float>(a, g, rows, dtable, device, s);
    default: return FA_E_DTYPE;
  }
}

}  // namespace fa
