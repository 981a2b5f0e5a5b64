// Attention with a relative position bias where few queries meet many keys: one new
// token (or a few) of each sequence against its cache.
//
// The memory's rate bounds it: every key and value is read once for all the query
// heads that share it.  The rows of one key head, its query heads times the queries,
// are the columns of one 32-wide block.  The keys are dealt out in blocks of 32 to the
// waves of `splits` workgroups; a wave works on its blocks by itself, through LDS of
// its own, with the next block on its way in registers, so no wave waits for another.
// The waves' sums are joined in LDS, the workgroups' by rows_join_kernel.
#include "fa_rel_attention.h"

namespace fa {

int rows_workspace(int B, int H, int Hk, int Lq, int Lk, int D, int device, int64_t* bytes);

namespace {

constexpr int NW = 4, NT = NW * 64, BN = 32;
constexpr int MOST_BIAS = 6144;  // floats of LDS for the bias of the heads together

// Workgroups that share the keys of one key head: enough for eight waves on every
// compute unit, and at least two blocks of keys for each wave.
inline int splits_of(int B, int Hk, int Lk, int device) {
  const int64_t heads = static_cast<int64_t>(B) * Hk;
  const int64_t want = (2 * cu_count(device) + heads - 1) / heads;
  const int64_t most = (Lk + 2 * NW * BN - 1) / (2 * NW * BN);
  const int64_t s = want < most ? want : most;
  return static_cast<int>(s < 1 ? 1 : s);
}

// What a wave's LDS region has to hold: its tiles, and later its O block.
template <typename T, int DP> constexpr size_t region() {
  constexpr size_t tiles = 2 * BN * Tile<T, DP>::LD * sizeof(T), o = size_t(DP) * 32 * sizeof(float);
  return tiles > o ? tiles : o;
}

template <typename T, int DP, bool WIDE>
__global__ __launch_bounds__(NT, 2) void rows_kernel(RelAttn a, T* out, View os, float* lse, int splits,
                                                  float* part_o, float* part_ml) {
  using M = Mat<T>;
  using TL = Tile<T, DP>;
  constexpr int CH = DP / 16, OB = DP / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  T* kt = reinterpret_cast<T*>(smem + wave * region<T, DP>());
  T* vt = kt + BN * TL::LD;
  float* ml = reinterpret_cast<float*>(smem + NW * region<T, DP>());  // [NW][2][32]
  float* eb = ml + NW * 64;                                           // [group][np]
  const int np = a.pos.n + 2 * PAD, group = a.H / a.Hk, rows = group * a.Lq;
  const int split = blockIdx.x % splits, bh = blockIdx.x / splits, hk = bh % a.Hk, b = bh / a.Hk;
  const int s0 = a.start(b), len = a.keys(b);
  const int g = min(col, rows - 1) / a.Lq, i = min(col, rows - 1) % a.Lq, h = hk * group + g;
  const uint8_t* mask = a.mask_of(b, h);
  const float c = a.scale * LOG2E;

  int end = len;
  if (a.causal)
    end = static_cast<int>(max<int64_t>(0, min<int64_t>(end, int64_t(s0) + a.Lq)));
  const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  TileLoad<T, DP, BN, 64, WIDE> kl, vl;
  const int stride = splits * NW * BN;
  int k0 = (split * NW + wave) * BN;
  if (k0 < end) {
    kl.load(kb + k0 * a.ks.t, a.ks.t, len - k0, a.D, a.vec, lane);
    vl.load(vb + k0 * a.vs.t, a.vs.t, len - k0, a.D, a.vec, lane);
  }
  load_bias<T>(eb, static_cast<const T*>(a.table), a.H, hk * group, group, a.pos, tid, NT);

  typename M::V8 qf[CH];
  // (the head's stride is per lane: its offset is part of the row's)
  {
    const T* q0 = static_cast<const T*>(a.q) + b * a.qs.b + hk * group * a.qs.h;
    Rows<T> qr(q0, a.qs.t);
    qr.stride = 1;
    load_row<T, WIDE>(qf, qr, int((g * a.qs.h + i * a.qs.t) * int64_t(sizeof(T))), 8 * hh, a.D, a.vec, col < rows);
  }
  f32x16 o[OB];
#pragma unroll
  for (int n = 0; n < OB; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[n][r] = 0.0f;
  float m = -INF, l = 0.0f;
  __syncthreads();  // the bias
  for (; k0 < end; k0 += stride) {
    kl.store(kt, lane);
    vl.store(vt, lane);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (k0 + stride < end) {
      const int k1 = k0 + stride;
      kl.load(kb + k1 * a.ks.t, a.ks.t, len - k1, a.D, a.vec, lane);
      vl.load(vb + k1 * a.vs.t, a.vs.t, len - k1, a.D, a.vec, lane);
    }
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
    for (int n = 0; n < CH; ++n) s = M::mma(TL::straight(kt, col, 16 * n + 8 * hh), qf[n], s);
    const int kind = block_kind(a.pos, s0 - (k0 + 31), s0 + a.Lq - 1 - k0);
    if (kind == NEAR) {
      const float* e = eb + g * np + (s0 + i - k0 - 4 * hh - a.pos.lo + PAD);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = s[r] * c + e[-(8 * (r / 4) + r % 4)];
    } else {
      const float e = eb[g * np + (kind == ALL_BELOW ? 0 : np - 1)];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = s[r] * c + e;
    }
    const bool partial = mask || k0 + 32 > len || (a.causal && k0 + 31 > s0);
    if (partial) hide(s, a, mask, i, s0 + i, k0 + 4 * hh, len);
    float top = -INF;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
    top = both_max(top);
    const float mn = fmaxf(m, top);
    if (__ballot(mn > m)) {
      const float shrink = mn == -INF ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      l *= shrink;
#pragma unroll
      for (int n = 0; n < OB; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] *= shrink;
      m = mn;
    }
    const float sub = m == -INF ? 0.0f : m;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = __builtin_amdgcn_exp2f(s[r] - sub);
      l += s[r];
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      typename M::V8 p;
#pragma unroll
      for (int n = 0; n < 8; ++n) p[n] = T(s[8 * half + n]);
#pragma unroll
      for (int n = 0; n < OB; ++n) {
        const typename M::V8 vf = TL::transposed(vt, 16 * half, 32 * n, lane);
        o[n] = partial ? guarded<T>(vf, p, o[n]) : M::mma(vf, p, o[n]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  l = both_sum(l);

  // join the waves: O^T in LDS as [d][row], each wave's in its own region
  float* ob = reinterpret_cast<float*>(smem + wave * region<T, DP>());
#pragma unroll
  for (int n = 0; n < OB; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) ob[(32 * n + 8 * (r / 4) + 4 * hh + r % 4) * 32 + col] = o[n][r];
  if (hh == 0) {
    ml[wave * 64 + col] = m;
    ml[wave * 64 + 32 + col] = l;
  }
  __syncthreads();
  for (int t = tid; t < rows * DP; t += NT) {
    const int row = t / DP, d = t % DP;
    if (d >= a.D) continue;
    float top = -INF;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, ml[w * 64 + row]);
    float sum = 0.0f, total = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = ml[w * 64 + row], f = mw == -INF ? 0.0f : __builtin_amdgcn_exp2f(mw - top);
      total += f * ml[w * 64 + 32 + row];
      const float x = reinterpret_cast<const float*>(smem + w * region<T, DP>())[d * 32 + row];
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
      out[b * os.b + hr * os.h + ir * os.t + d] = T(total == 0.0f ? 0.0f : sum / total);
      if (lse && d == 0)
        lse[(static_cast<int64_t>(b) * a.H + hr) * a.Lq + ir] =
            total == 0.0f ? INF : top + __builtin_log2f(total);
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
  float top = -INF;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, part_ml[2 * (first + static_cast<int64_t>(s) * rows)]);
  float x0 = 0.0f, x1 = 0.0f, total = 0.0f;
  const int d0 = threadIdx.x, d1 = threadIdx.x + 64;
  for (int s = 0; s < splits; ++s) {
    const int64_t at = first + static_cast<int64_t>(s) * rows;
    const float ms = part_ml[2 * at];
    if (ms == -INF) continue;
    const float f = __builtin_amdgcn_exp2f(ms - top);
    total += f * part_ml[2 * at + 1];
    if (d0 < D) x0 += f * part_o[at * D + d0];
    if (d1 < D) x1 += f * part_o[at * D + d1];
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  T* o = out + b * os.b + h * os.h + i * os.t;
  if (d0 < D) o[d0] = T(x0 * inv);
  if (d1 < D) o[d1] = T(x1 * inv);
  if (lse && threadIdx.x == 0)
    lse[(static_cast<int64_t>(b) * H + h) * Lq + i] = total == 0.0f ? INF : top + __builtin_log2f(total);
}

template <typename T, int DP>
int launch_dim(const RelAttn& a, T* out, const View& os, float* lse, int splits, float* part_o,
               float* part_ml, hipStream_t s) {
  const int group = a.H / a.Hk, rows = group * a.Lq;
  const int64_t wgs = static_cast<int64_t>(a.B) * a.Hk * splits;
  const int64_t joins = static_cast<int64_t>(a.B) * a.Hk * rows;
  if (wgs > 0x7fffffff || joins > 0x7fffffff) return FA_E_SHAPE;
  const size_t lds = NW * region<T, DP>() + (NW * 64 + group * (a.pos.n + 2 * PAD)) * sizeof(float);
  auto kernel = a.vec * sizeof(T) == 16 ? rows_kernel<T, DP, true> : rows_kernel<T, DP, false>;
  if (const int e = launch_lds(kernel, lds)) return e;
  kernel<<<static_cast<unsigned>(wgs), NT, lds, s>>>(a, out, os, lse, splits, part_o, part_ml);
  FA_LAUNCH_CHECK();
  if (splits > 1) {
    rows_join_kernel<T><<<static_cast<unsigned>(joins), 64, 0, s>>>(part_o, part_ml, a.H, a.Hk, a.Lq,
                                                                    a.D, splits, out, os, lse);
    FA_LAUNCH_CHECK();
  }
  return FA_OK;
}

template <typename T>
int forward(RelAttn a, void* out, const View& os, float* lse, int splits, float* part_o, float* part_ml,
            hipStream_t s) {
  const void* in[3] = {a.q, a.k, a.v};
  const View iv[3] = {a.qs, a.ks, a.vs};
  a.vec = widest_load<T>(in, iv, 3, a.D);
  T* o = static_cast<T*>(out);
  if (a.D <= 32) return launch_dim<T, 32>(a, o, os, lse, splits, part_o, part_ml, s);
  if (a.D <= 64) return launch_dim<T, 64>(a, o, os, lse, splits, part_o, part_ml, s);
  return launch_dim<T, 128>(a, o, os, lse, splits, part_o, part_ml, s);
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
  float* part_ml = static_cast<float*>(ws);
  float* part_o = part_ml ? part_ml + static_cast<int64_t>(a.B) * a.Hk * splits * (a.H / a.Hk) * a.Lq * 2
                          : nullptr;
  switch (dtype) {
    case FA_F16: return forward<_Float16>(a, out, os, lse, splits, part_o, part_ml, s);
    case FA_BF16: return forward<__bf16>(a, out, os, lse, splits, part_o, part_ml, s);
    case FA_F32: return forward<float>(a, out, os, lse, splits, part_o, part_ml, s);
    default: return FA_E_DTYPE;
  }
}

}  // namespace fa
