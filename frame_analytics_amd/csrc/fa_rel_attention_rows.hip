// Attention with a relative position bias where few queries meet many keys: one new
// token (or a few) of each sequence against its cache.
//
// The memory's rate bounds it: every key and value is read once for all the query
// heads that share it.  The rows of one key head, its query heads times the queries,
// are the columns of one or two 16-wide blocks.  The keys are dealt out in runs to
// `splits` workgroups, in blocks of 32 to their waves; a wave works on its blocks by
// itself, the next block on its way in registers, so no wave waits for another: keys
// arrive as the fragments of S^T = K Q^T, values pass through LDS of the wave's own to
// be read transposed.  The waves' sums are joined in LDS, the workgroups' by
// rows_join_kernel.
//
// Blocks here are 16 x 16: with l the lane and g = l / 16 a C block holds rows 4 g + r
// of column l % 16 in registers r = 0 .. 3, and an A or B fragment row or column l % 16
// with eight of 32 k values, straight (8 g + i) or split (16 (i / 4) + 4 g + i % 4, the
// rows that two C blocks hold).
#include "fa_rel_attention.h"

namespace fa {

namespace {

constexpr int NW = 4, NT = NW * 64, BN = 32;
constexpr int MOST_BIAS = 6144;  // floats of LDS for the bias of the heads together

// Keys are dealt out in runs of `per` blocks for each wave of a workgroup: as few as keep
// two workgroups for every compute unit, so that entries of different lengths even out
// (the runs past an entry's end return at once).
inline int per_wave(int B, int Hk, int Lk, int device) {
  const int64_t blocks = static_cast<int64_t>(B) * Hk * ((Lk + BN - 1) / BN);
  const int64_t per = blocks / (static_cast<int64_t>(NW) * 2 * cu_count(device));
  return static_cast<int>(per < 1 ? 1 : per > 64 ? 64 : per);
}
inline int splits_of(int B, int Hk, int Lk, int device) {
  const int run = per_wave(B, Hk, Lk, device) * NW * BN;
  return (Lk + run - 1) / run;
}

template <typename T> __device__ inline f32x4 mma16(typename Mat<T>::V8 a, typename Mat<T>::V8 b, f32x4 c) {
  if constexpr (std::is_same<T, _Float16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  } else if constexpr (std::is_same<T, __bf16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
}

// Over the four lanes l % 16 + 16 g, in all of them.
__device__ inline float four_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  return both_max(fmaxf(__int_as_float(r[0]), __int_as_float(r[1])));
}
__device__ inline float four_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  return both_sum(__int_as_float(r[0]) + __int_as_float(r[1]));
}

// Column col0 + l % 16 of a tile's 32 rows, in split slots.
template <typename T, int DP>
__device__ inline typename Mat<T>::V8 transposed16(const T* t, int col0, int lane) {
  constexpr int LD = Tile<T, DP>::LD;
  typename Mat<T>::V8 r;
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((address_space(3))) s16x4 lds4;
    typedef typename Mat<T>::V4 V4;
    const T* p = t + (lane >> 2) * LD + col0 + 4 * (lane & 3);
    const V4 x = __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p));
    const V4 y = __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 16 * LD)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = x[i];
      r[4 + i] = y[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = t[(16 * (i / 4) + 4 * (lane >> 4) + i % 4) * LD + col0 + (lane & 15)];
  }
  return r;
}

// As guarded<T>, for 16 x 16 blocks.
template <typename T>
__device__ inline f32x4 guarded16(typename Mat<T>::V8 v, typename Mat<T>::V8 p, f32x4 acc, uint32_t seen) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) bad |= !(__builtin_fabsf(widen(v[i])) < INF);
  if (__ballot(bad) == 0) return mma16<T>(v, p, acc);
  typename Mat<T>::V8 fine;
#pragma unroll
  for (int i = 0; i < 8; ++i) fine[i] = __builtin_fabsf(widen(v[i])) < INF ? v[i] : T(0);
  acc = mma16<T>(fine, p, acc);
#pragma unroll 1
  for (float way = INF; way != 0.0f; way = way > 0.0f ? -INF : 0.0f) {
    typename Mat<T>::V8 bad_v, ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = widen(v[i]);
      bad_v[i] = x == way || x != x ? T(1) : T(0);
      ones[i] = seen >> i & 1 ? T(1) : T(0);
    }
    const f32x4 n = mma16<T>(bad_v, ones, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] += n[r] > 0.0f ? way : 0.0f;
  }
  return acc;
}

// A wave's LDS: its values, and later its O block of NC x 16 rows.
template <typename T, int DP, int NC> constexpr size_t region() {
  constexpr size_t tile = BN * Tile<T, DP>::LD * sizeof(T), o = size_t(DP) * 16 * NC * sizeof(float);
  return tile > o ? tile : o;
}

template <typename T, int DP, int NC, bool WIDE>
__global__ __launch_bounds__(NT, 2) void rows_kernel(RelAttn a, T* out, View os, float* lse, int splits,
                                                     int per, float* part_o, float* part_ml) {
  using M = Mat<T>;
  constexpr int CH = DP / 32, OB = DP / 16, ROWS = 16 * NC;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, gg = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  T* vt = reinterpret_cast<T*>(smem + wave * region<T, DP, NC>());
  float* ml = reinterpret_cast<float*>(smem + NW * region<T, DP, NC>());  // [NW][2][ROWS]
  float* eb = ml + NW * 2 * ROWS;                                         // [group][np]
  const int np = a.pos.n + 2 * PAD, group = a.H / a.Hk, rows = group * a.Lq;
  const int split = blockIdx.x % splits, bh = blockIdx.x / splits, hk = bh % a.Hk, b = bh / a.Hk;
  const int s0 = a.start(b), len = a.keys(b);
  const float c = a.scale * LOG2E;

  int end = len;
  if (a.causal)
    end = static_cast<int>(max<int64_t>(0, min<int64_t>(end, int64_t(s0) + a.Lq)));
  const int run = per * NW * BN, stride = NW * BN;
  if (splits > 1 && static_cast<int64_t>(split) * run >= end) {
    if (tid < rows) {
      float* none = part_ml + 2 * (static_cast<int64_t>(blockIdx.x) * rows + tid);
      none[0] = -INF;
      none[1] = 0.0f;
    }
    return;
  }
  end = static_cast<int>(min<int64_t>(end, (static_cast<int64_t>(split) + 1) * run));
  const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  TileLoad<T, DP, BN, 64, WIDE> vl;
  typename M::V8 kf[2][CH];
  auto load = [&](int k) {
    const Rows<T> kr(kb + k * a.ks.t, a.ks.t);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int row = 16 * n + col, d = 32 * i + 8 * gg;
        const bool on = k + row < len;
        if constexpr (WIDE) kf[n][i] = kr.wide(row, d, a.D, on);
        else if (a.vec == 2) kf[n][i] = kr.pairs(row, d, a.D, on);
        else kf[n][i] = kr.single(row, d, a.D, on);
      }
    vl.load(vb + k * a.vs.t, a.vs.t, len - k, a.D, a.vec, lane);
  };
  int k0 = split * run + wave * BN;
  if (k0 < end) load(k0);

  int qi[NC], gi[NC];
  const uint8_t* mask[NC];
  typename M::V8 qf[NC][CH];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int row = min(16 * n + col, rows - 1);
    gi[n] = row / a.Lq;
    qi[n] = row % a.Lq;
    mask[n] = a.mask_of(b, hk * group + gi[n]);
    // (the head's stride is per lane: its offset is part of the row's)
    Rows<T> qr(static_cast<const T*>(a.q) + b * a.qs.b + hk * group * a.qs.h, a.qs.t);
    qr.stride = 1;
    const int at = static_cast<int>((gi[n] * a.qs.h + qi[n] * a.qs.t) * static_cast<int64_t>(sizeof(T)));
    const bool on = 16 * n + col < rows;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int d = 32 * i + 8 * gg;
      if constexpr (WIDE) qf[n][i] = qr.wide(at, d, a.D, on);
      else if (a.vec == 2) qf[n][i] = qr.pairs(at, d, a.D, on);
      else qf[n][i] = qr.single(at, d, a.D, on);
    }
  }
  load_bias<T>(eb, a, hk * group, group, tid, NT);

  f32x4 o[NC][OB];
  float m[NC], l[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    m[n] = -INF;
    l[n] = 0.0f;
#pragma unroll
    for (int i = 0; i < OB; ++i) o[n][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  __syncthreads();  // the bias
  for (; k0 < end; k0 += stride) {
    vl.store(vt, lane);
    f32x4 s[NC][2];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        s[n][w] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < CH; ++i) s[n][w] = mma16<T>(kf[w][i], qf[n][i], s[n][w]);
      }
    wave_sync();
    if (k0 + stride < end) load(k0 + stride);
    const int kind = block_kind(a.pos, s0 - (k0 + 31), s0 + a.Lq - 1 - k0);
    const bool partial = a.mask || k0 + 32 > len || (a.causal && k0 + 31 > s0);
    typename M::V8 p[NC];
    uint32_t visible[NC];  // bit 4 w + r
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      visible[n] = 0;
      const float* e = eb + gi[n] * np + (s0 + qi[n] - k0 - 4 * gg - a.pos.lo + PAD);
      const float far = eb[gi[n] * np + (kind == ALL_BELOW ? 0 : np - 1)];
      float top = -INF;
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = s[n][w][r] * c + (kind == NEAR ? e[-(16 * w + r)] : far);
          if (partial) {
            const int key = k0 + 16 * w + 4 * gg + r;
            bool seen = key < len && (!a.causal || key <= s0 + qi[n]);
            if (a.mask && seen) seen = mask[n][qi[n] * a.mq + key * a.mk] != 0;
            if (!seen) x = -INF;
            visible[n] |= (seen ? 1u : 0u) << (4 * w + r);
          }
          s[n][w][r] = x;
          top = fmaxf(top, x);
        }
      top = four_max(top);
      const float mn = fmaxf(m[n], top);
      if (__ballot(mn > m[n])) {
        const float shrink = mn == -INF ? 1.0f : __builtin_amdgcn_exp2f(m[n] - mn);
        l[n] *= shrink;
#pragma unroll
        for (int i = 0; i < OB; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[n][i][r] *= shrink;
        m[n] = mn;
      }
      const float sub = m[n] == -INF ? 0.0f : m[n];
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = __builtin_amdgcn_exp2f(s[n][w][r] - sub);
          l[n] += x;
          p[n][4 * w + r] = T(x);
        }
    }
#pragma unroll
    for (int i = 0; i < OB; ++i) {
      const typename M::V8 vf = transposed16<T, DP>(vt, 16 * i, lane);
#pragma unroll
      for (int n = 0; n < NC; ++n)
        o[n][i] = partial ? guarded16<T>(vf, p[n], o[n][i], visible[n]) : mma16<T>(vf, p[n], o[n][i]);
    }
    wave_sync();
  }

  // join the waves: O^T in LDS as [d][row], each wave's in its own region
  float* ob = reinterpret_cast<float*>(smem + wave * region<T, DP, NC>());
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    l[n] = four_sum(l[n]);
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) ob[(16 * i + 4 * gg + r) * ROWS + 16 * n + col] = o[n][i][r];
    if (gg == 0) {
      ml[wave * 2 * ROWS + 16 * n + col] = m[n];
      ml[wave * 2 * ROWS + ROWS + 16 * n + col] = l[n];
    }
  }
  __syncthreads();
  for (int t = tid; t < rows * DP; t += NT) {
    const int row = t / DP, d = t % DP;
    if (d >= a.D) continue;
    float top = -INF;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, ml[w * 2 * ROWS + row]);
    float sum = 0.0f, total = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = ml[w * 2 * ROWS + row], f = mw == -INF ? 0.0f : __builtin_amdgcn_exp2f(mw - top);
      total += f * ml[w * 2 * ROWS + ROWS + row];
      const float x = reinterpret_cast<const float*>(smem + w * region<T, DP, NC>())[d * ROWS + row];
      if (mw != -INF) sum += f * x;
    }
    if (splits > 1) {
      const int64_t at = static_cast<int64_t>(blockIdx.x) * rows + row;
      part_o[at * a.D + d] = sum;
      if (d == 0) {
        part_ml[2 * at] = top;
        part_ml[2 * at + 1] = total;
      }
    } else {
      const int hr = hk * group + row / a.Lq, ir = row % a.Lq;
      const float x = total == 0.0f ? 0.0f : sum / total;
      out[b * os.b + hr * os.h + ir * os.t + d] = T(x);
      if (sizeof(T) == 2 && lse)
        low_of<T>(lse, static_cast<int64_t>(a.B) * a.H * a.Lq)[((static_cast<int64_t>(b) * a.H + hr) * a.Lq + ir) *
                                                                   a.D + d] = T(x - widen(T(x)));
      if (lse && d == 0)
        keep_row(lse, static_cast<int64_t>(a.B) * a.H * a.Lq, (static_cast<int64_t>(b) * a.H + hr) * a.Lq + ir, top,
                 total);
    }
  }
}

// One wave for each row: its sums of all splits, joined.
template <typename T>
__global__ __launch_bounds__(64) void rows_join_kernel(const float* part_o, const float* part_ml, int H,
                                                       int Hk, int Lq, int D, int splits, T* out,
                                                       View os, float* lse) {
  const int rows = H / Hk * Lq, row = blockIdx.x % rows, bh = blockIdx.x / rows, hk = bh % Hk, b = bh / Hk;
  const int h = hk * (H / Hk) + row / Lq, i = row % Lq;
  const int64_t first = static_cast<int64_t>(bh) * splits * rows + row;
  // the splits' maxima and sums, one lane each; then their values, eight reads at once
  const int lane = threadIdx.x, d0 = lane, d1 = lane + 64;
  float top = -INF;
  for (int s = lane; s < splits; s += 64)
    top = fmaxf(top, part_ml[2 * (first + static_cast<int64_t>(s) * rows)]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  float x0 = 0.0f, x1 = 0.0f, total = 0.0f;
  for (int s0 = 0; s0 < splits; s0 += 64) {
    float f = 0.0f;
    if (s0 + lane < splits) {
      const int64_t at = first + static_cast<int64_t>(s0 + lane) * rows;
      const float ms = part_ml[2 * at];
      // a split without a maximum saw no key, and its sum is 0, or NaN scores alone, which
      // no maximum takes, and its sum is NaN: the row's has to be
      f = ms != -INF ? __builtin_amdgcn_exp2f(ms - top) : 0.0f;
      total += ms != -INF ? f * part_ml[2 * at + 1] : part_ml[2 * at + 1];
    }
    const int here = min(64, splits - s0);
    for (int s1 = 0; s1 < here; s1 += 8) {
      float fs[8], y0[8], y1[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        fs[e] = s1 + e < here ? __shfl(f, (s1 + e) & 63, 64) : 0.0f;
        const float* p = part_o + (first + static_cast<int64_t>(s0 + s1 + e) * rows) * D;
        // (what a split that saw no key left in part_o is not read)
        y0[e] = fs[e] != 0.0f && d0 < D ? p[d0] : 0.0f;
        y1[e] = fs[e] != 0.0f && d1 < D ? p[d1] : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x0 += fs[e] * y0[e];
        x1 += fs[e] * y1[e];
      }
    }
  }
  total = wave_sum(total);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  T* o = out + b * os.b + h * os.h + i * os.t;
  x0 *= inv;
  x1 *= inv;
  if (d0 < D) o[d0] = T(x0);
  if (d1 < D) o[d1] = T(x1);
  if (!lse) return;
  const int64_t all = static_cast<int64_t>(gridDim.x / rows / Hk) * H * Lq;  // batch x heads x queries
  if (lane == 0) keep_row(lse, all, (static_cast<int64_t>(b) * H + h) * Lq + i, top, total);
  if (sizeof(T) == 2) {
    T* low = low_of<T>(lse, all) + ((static_cast<int64_t>(b) * H + h) * Lq + i) * D;
    if (d0 < D) low[d0] = T(x0 - widen(T(x0)));
    if (d1 < D) low[d1] = T(x1 - widen(T(x1)));
  }
}

template <typename T, int DP, int NC>
int launch_rows(const RelAttn& a, T* out, const View& os, float* lse, int splits, int per,
               float* part_o, float* part_ml, hipStream_t s) {
  const int group = a.H / a.Hk, rows = group * a.Lq;
  const int64_t wgs = static_cast<int64_t>(a.B) * a.Hk * splits;
  const int64_t joins = static_cast<int64_t>(a.B) * a.Hk * rows;
  if (wgs > 0x7fffffff || joins > 0x7fffffff) return FA_E_SHAPE;
  const size_t lds = NW * region<T, DP, NC>() + (NW * 32 * NC + group * (a.pos.n + 2 * PAD)) * sizeof(float);
  auto kernel = a.vec * sizeof(T) == 16 ? rows_kernel<T, DP, NC, true> : rows_kernel<T, DP, NC, false>;
  if (const int e = launch_lds(kernel, lds)) return e;
  kernel<<<static_cast<unsigned>(wgs), NT, lds, s>>>(a, out, os, lse, splits, per, part_o, part_ml);
  FA_LAUNCH_CHECK();
  if (splits > 1) {
    rows_join_kernel<T><<<static_cast<unsigned>(joins), 64, 0, s>>>(part_o, part_ml, a.H, a.Hk, a.Lq,
                                                                    a.D, splits, out, os, lse);
    FA_LAUNCH_CHECK();
  }
  return FA_OK;
}

template <typename T, int DP>
int launch_dim(const RelAttn& a, T* out, const View& os, float* lse, int splits, int per, float* part_o,
               float* part_ml, hipStream_t s) {
  return a.H / a.Hk * a.Lq <= 16 ? launch_rows<T, DP, 1>(a, out, os, lse, splits, per, part_o, part_ml, s)
                                 : launch_rows<T, DP, 2>(a, out, os, lse, splits, per, part_o, part_ml, s);
}

template <typename T>
int forward(RelAttn a, void* out, const View& os, float* lse, int splits, int per, float* part_o,
            float* part_ml, hipStream_t s) {
  const void* in[3] = {a.q, a.k, a.v};
  const View iv[3] = {a.qs, a.ks, a.vs};
  a.vec = widest_load<T>(in, iv, 3, a.D);
  T* o = static_cast<T*>(out);
  if (a.D <= 32) return launch_dim<T, 32>(a, o, os, lse, splits, per, part_o, part_ml, s);
  if (a.D <= 64) return launch_dim<T, 64>(a, o, os, lse, splits, per, part_o, part_ml, s);
  return launch_dim<T, 128>(a, o, os, lse, splits, per, part_o, part_ml, s);
}

}  // namespace

// A block's worth of rows for each key head, on a line.
bool rows_serve(const RelAttn& a) {
  const int group = a.H / a.Hk;
  return a.pos.grid_w == 0 && static_cast<int64_t>(group) * a.Lq <= 32 &&
         static_cast<int64_t>(group) * (a.pos.n + 2 * PAD) <= MOST_BIAS &&
         a.qs.h >= 0 && a.qs.h < (1 << 23);  // 32 heads' offsets in 32 bits
}

int rows_workspace(int B, int H, int Hk, int Lq, int Lk, int D, int device, int64_t* bytes) {
  *bytes = 0;
  if (static_cast<int64_t>(H / Hk) * Lq > 32) return FA_OK;
  const int splits = splits_of(B, Hk, Lk, device);
  if (splits > 1) *bytes = static_cast<int64_t>(B) * Hk * splits * (H / Hk) * Lq * (D + 2) * 4;
  return FA_OK;
}

int rows_forward(int dtype, const RelAttn& a, void* out, const View& os, float* lse, void* ws,
                 int64_t ws_bytes, int device, hipStream_t s) {
  int64_t need = 0;
  if (const int e = rows_workspace(a.B, a.H, a.Hk, a.Lq, a.Lk, a.D, device, &need)) return e;
  if (need > 0 && (!ws || ws_bytes < need)) return FA_E_ARG;
  const int splits = splits_of(a.B, a.Hk, a.Lk, device);
  const int per = per_wave(a.B, a.Hk, a.Lk, device);
  float* part_ml = static_cast<float*>(ws);
  float* part_o = part_ml ? part_ml + static_cast<int64_t>(a.B) * a.Hk * splits * (a.H / a.Hk) * a.Lq * 2
                          : nullptr;
  switch (dtype) {
    case FA_F16: return forward<_Float16>(a, out, os, lse, splits, per, part_o, part_ml, s);
    case FA_BF16: return forward<__bf16>(a, out, os, lse, splits, per, part_o, part_ml, s);
    case FA_F32: return forward<float>(a, out, os, lse, splits, per, part_o, part_ml, s);
    default: return FA_E_DTYPE;
  }
}

}  // namespace fa
