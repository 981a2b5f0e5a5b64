// Attention with a relative position bias, forward.
//
// A wave owns 32 queries and walks over the keys, 64 at a time through LDS, with the
// running maximum and sum of its rows' softmax.  It forms S^T = K Q^T, so a lane
// holds one query's scores (a row's statistics are the lane's own, and one exchange
// with lane l ^ 32), and O^T = V^T P^T, whose B operand is the rounded scores as they
// stand in the registers.  The bias is added from one head's table in LDS: on a line a
// block of keys that is far from the wave's queries has one bias for all its pairs.
#include "fa_rel_attention.h"

namespace fa {

namespace {

template <typename T, int DP> struct Shape {
  static constexpr int BN = sizeof(T) == 2 || DP <= 64 ? 64 : 32;  // keys per tile
  static constexpr size_t TILE = size_t(BN) * Tile<T, DP>::LD * sizeof(T);
};

// KG groups of NW waves take every KG-th tile of keys for the same queries, and join their
// sums at the end: where there are few workgroups the longest row of tiles is the time.
template <typename T, int DP, int NW, int KG, bool WIDE>
__global__ __launch_bounds__(NW * 64 * KG) void rel_attention_kernel(RelAttn a, T* out, View os,
                                                                int ovec, float* lse,
                                                                int q_tiles) {
  using M = Mat<T>;
  using TL = Tile<T, DP>;
  constexpr int NT = NW * 64, BN = Shape<T, DP>::BN, NB = BN / 32, CH = DP / 16, OB = DP / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  const int kg = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0;
  T* kt = reinterpret_cast<T*>(smem) + kg * 4 * BN * TL::LD;  // [2][BN][LD] of each group
  T* vt = kt + 2 * BN * TL::LD;                               // [2][BN][LD]
  float* eb = reinterpret_cast<float*>(reinterpret_cast<T*>(smem) + KG * 4 * BN * TL::LD);
  const int tid = threadIdx.x - kg * NT, lane = tid & 63, hh = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned wg = xcd_tile(blockIdx.x, gridDim.x);
  const int tile = q_tiles - 1 - int(wg % q_tiles);  // the longest of a causal head first
  const int h = int(wg / q_tiles) % a.H, b = int(wg / q_tiles) / a.H, hk = h / (a.H / a.Hk);
  const int qw = tile * (NW * 32) + wave * 32;  // the wave's first query
  const int q = qw + col, qc = min(q, a.Lq - 1), s0 = a.start(b), len = a.keys(b);
  const int qpos = s0 + q, cq = s0 + a.pos.code(qc);
  const uint8_t* mask = a.mask_of(b, h);
  const float c = a.scale * LOG2E;

  int* codes = reinterpret_cast<int*>(eb + (a.pos.n + 2 * PAD + 3) / 4 * 4);  // of a window's keys
  load_bias<T>(eb, a, h, 1, threadIdx.x, NT * KG);
  if (a.pos.grid_w) load_codes(codes, a.pos, a.Lk, threadIdx.x, NT * KG);

  typename M::V8 qf[CH];
  const int q_first = tile * (NW * 32);
  load_row<T, WIDE>(qf, Rows<T>(static_cast<const T*>(a.q) + b * a.qs.b + h * a.qs.h + q_first * a.qs.t, a.qs.t),
              q - q_first, 8 * hh, a.D, a.vec, q < a.Lq);

  f32x16 o[OB];
#pragma unroll
  for (int i = 0; i < OB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.0f;
  float m = -INF, l = 0.0f;

  // keys that any query of the workgroup sees
  int end = len;
  if (a.causal) {
    const int64_t last = int64_t(s0) + min(tile * (NW * 32) + NW * 32, a.Lq);
    end = static_cast<int>(max<int64_t>(0, min<int64_t>(end, last)));
  }
  const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  TileLoad<T, DP, BN, NT, WIDE> kl, vl;
  const int tiles = (end + BN - 1) / BN;
  if (kg < tiles) {
    const int k1 = kg * BN;
    kl.load(kb + k1 * a.ks.t, a.ks.t, len - k1, a.D, a.vec, tid);
    vl.load(vb + k1 * a.vs.t, a.vs.t, len - k1, a.D, a.vec, tid);
    kl.store(kt, tid);
    vl.store(vt, tid);
  }
  // One tile of keys.  FAR: every pair of the wave is past one end of the bias table and
  // counts; WINDOW: a window's pairs, which all count; ANY: the rest.  The first two run
  // without a branch: with the tests of the third around each product (hidden pairs,
  // values that are not finite) no instruction of one could overlap the next.
  enum : int { ANY, FAR, WINDOW };
  auto work = [&](int t, auto mode, float far) {
    constexpr int MODE = decltype(mode)::value;
    const T* kk = kt + (t / KG & 1) * BN * TL::LD;
    const T* vv = vt + (t / KG & 1) * BN * TL::LD;
    f32x16 s[NB];
    bool partial[NB];
    uint32_t seen[NB];
    float top = -INF;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[nb][r] = 0.0f;
#pragma unroll
      for (int i = 0; i < CH; ++i)
        s[nb] = M::mma(TL::straight(kk, nb * 32 + col, 16 * i + 8 * hh), qf[i], s[nb]);
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int k0 = t * BN + nb * 32;
      partial[nb] = false;
      if (MODE == WINDOW || (MODE == ANY && a.pos.grid_w)) {
        const float* e = eb + afresh(cq - a.pos.lo + PAD);
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int4 ck = *reinterpret_cast<const int4*>(codes + k0 + 4 * hh + 8 * r4);
          s[nb][4 * r4] = s[nb][4 * r4] * c + e[-ck.x];
          s[nb][4 * r4 + 1] = s[nb][4 * r4 + 1] * c + e[-ck.y];
          s[nb][4 * r4 + 2] = s[nb][4 * r4 + 2] * c + e[-ck.z];
          s[nb][4 * r4 + 3] = s[nb][4 * r4 + 3] * c + e[-ck.w];
        }
      } else if (MODE == ANY) {
        // differences of the whole block: uniform over the wave
        const int dmax = s0 + qw + 31 - k0, dmin = s0 + qw - (k0 + 31);
        const int kind = block_kind(a.pos, dmin, dmax);
        if (kind == NEAR) {
          // rows past Lq stand at their own positions here: the block's reads stay
          // within PAD of the table
          const float* e = eb + (s0 + q - k0 - 4 * hh - a.pos.lo + PAD);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[nb][r] = s[nb][r] * c + e[-(8 * (r / 4) + r % 4)];
        } else {
          const float e = kind == ALL_BELOW ? eb[0] : eb[a.pos.n + 2 * PAD - 1];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[nb][r] = s[nb][r] * c + e;
        }
      }
      if (MODE == ANY) {
        partial[nb] = mask || k0 + 32 > len || (a.causal && k0 + 31 > s0 + qw);
        if (partial[nb]) hide(s[nb], seen[nb] = seen_keys(a, mask, qc, qpos, k0 + 4 * hh, len));
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[nb][r]);
    }
    if (MODE == FAR) top = top * c + far;  // (c > 0)
    top = both_max(top);
    const float mn = fmaxf(m, top);
    if (__ballot(mn > m)) {  // a row's maximum grew: what was summed shrinks by it
      const float shrink = mn == -INF ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      l *= shrink;
#pragma unroll
      for (int i = 0; i < OB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= shrink;
      m = mn;
    }
    const float sub = m == -INF ? 0.0f : m;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[nb][r] = __builtin_amdgcn_exp2f(MODE == FAR ? s[nb][r] * c + (far - sub) : s[nb][r] - sub);
        l += s[nb][r];
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // the weights are rounded to the element type for the product with V; their
        // sum is not
        typename M::V8 p;
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = T(s[nb][8 * half + i]);
#pragma unroll
        for (int i = 0; i < OB; ++i) {
          const typename M::V8 vf = TL::transposed(vv, nb * 32 + 16 * half, 32 * i, lane);
          o[i] = partial[nb] ? guarded<T>(vf, p, o[i], seen[nb] >> 8 * half) : M::mma(vf, p, o[i]);
        }
      }
    }
  };
  const int rounds = (tiles + KG - 1) / KG;
  __syncthreads();
  const bool far_on = c > 0.0f && far_serves(eb, a.pos.n + 2 * PAD);
  for (int round = 0; round < rounds; ++round) {
    const int t = round * KG + kg;
    __syncthreads();
    if (t >= tiles) continue;  // (in the last round)
    const bool more = t + KG < tiles;
    const int k0 = t * BN, k1 = k0 + KG * BN;
    if (more) {
      kl.load(kb + k1 * a.ks.t, a.ks.t, len - k1, a.D, a.vec, tid);
      vl.load(vb + k1 * a.vs.t, a.vs.t, len - k1, a.D, a.vec, tid);
    }
    const bool all = !mask && k0 + BN <= len && (!a.causal || k0 + BN - 1 <= s0 + qw);
    const int kind = block_kind(a.pos, s0 + qw - (k0 + BN - 1), s0 + qw + 31 - k0);
    if (all && a.pos.grid_w)
      work(t, std::integral_constant<int, WINDOW>(), 0.0f);
    else if (all && kind != NEAR && far_on)
      work(t, std::integral_constant<int, FAR>(), kind == ALL_BELOW ? eb[0] : eb[a.pos.n + 2 * PAD - 1]);
    else
      work(t, std::integral_constant<int, ANY>(), 0.0f);
    if (more) {
      kl.store(kt + ((t / KG + 1) & 1) * BN * TL::LD, tid);
      vl.store(vt + ((t / KG + 1) & 1) * BN * TL::LD, tid);
    }
  }
  if constexpr (KG > 1) {
    static_assert(KG == 2, "the second group's sums join the first's");
    float* sums = reinterpret_cast<float*>(smem) + wave * (OB * 16 + 2) * 64 + lane;
    __syncthreads();
    if (kg == 1) {
#pragma unroll
      for (int i = 0; i < OB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) sums[(16 * i + r) * 64] = o[i][r];
      sums[OB * 16 * 64] = m;
      sums[(OB * 16 + 1) * 64] = l;
    }
    __syncthreads();
    if (kg == 1) return;
    const float m1 = sums[OB * 16 * 64], mn = fmaxf(m, m1);
    const float f0 = m == -INF ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float f1 = m1 == -INF ? 0.0f : __builtin_amdgcn_exp2f(m1 - mn);
    l = l * f0 + sums[(OB * 16 + 1) * 64] * f1;
    m = mn;
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] = o[i][r] * f0 + sums[(16 * i + r) * 64] * f1;
  }
  l = both_sum(l);
  if (q < a.Lq) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* orow = out + b * os.b + h * os.h + q * os.t;
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = o[i][4 * g + e] * inv;
        store4<T>(orow, 32 * i + 8 * g + 4 * hh, a.D, ovec, w);
        if (sizeof(T) == 2 && lse && a.pos.grid_w == 0) {
          const int64_t all = static_cast<int64_t>(a.B) * a.H * a.Lq;
          T* low = low_of<T>(lse, all) + ((static_cast<int64_t>(b) * a.H + h) * a.Lq + q) * a.D;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] -= widen(T(w[e]));
          store4<T>(low, 32 * i + 8 * g + 4 * hh, a.D, a.D % 4 == 0 ? 8 : 1, w);
        }
      }
    if (lse && hh == 0)
      keep_row(lse, static_cast<int64_t>(a.B) * a.H * a.Lq, (static_cast<int64_t>(b) * a.H + h) * a.Lq + q, m, l);
  }
}

template <typename T, int DP, int NW, int KG, bool WIDE>
int launch_one(const RelAttn& a, T* out, const View& os, int ovec, float* lse, hipStream_t s) {
  const int q_tiles = (a.Lq + NW * 32 - 1) / (NW * 32);
  const int64_t wgs = static_cast<int64_t>(a.B) * a.H * q_tiles;
  if (wgs > 0x7fffffff) return FA_E_SHAPE;
  const size_t lds = KG * 4 * Shape<T, DP>::TILE + (a.pos.n + 2 * PAD + 3) / 4 * 16 +
                     (a.pos.grid_w ? codes_room(a.Lk) * sizeof(int) : 0);
  if constexpr (KG > 1)  // a table that leaves no room for the second group's tiles
    if (lds > MOST_LDS) return launch_one<T, DP, NW, 1, WIDE>(a, out, os, ovec, lse, s);
  auto kernel = rel_attention_kernel<T, DP, NW, KG, WIDE>;
  if (const int e = launch_lds(kernel, lds)) return e;
  kernel<<<static_cast<unsigned>(wgs), NW * 64 * KG, lds, s>>>(a, out, os, ovec, lse, q_tiles);
  FA_LAUNCH_CHECK();
  return FA_OK;
}

template <typename T, int DP, bool WIDE>
int launch_wide(const RelAttn& a, T* out, const View& os, int ovec, float* lse, int device, hipStream_t s) {
  // two waves to a workgroup where four leave compute units without one (a causal line of
  // 2048 in bfloat16: 256 workgroups of four 43 us, 512 of two 65; a line of 777 in float32:
  // 112 of four 70, 208 of two 49), and a second group of waves where there are less than two
  // workgroups for every compute unit
  const int cus = cu_count(device);
  const int64_t four = static_cast<int64_t>(a.B) * a.H * ((a.Lq + 127) / 128);
  const bool few = a.Lq <= 64 || four < cus;
  const int64_t wgs = few ? static_cast<int64_t>(a.B) * a.H * ((a.Lq + 63) / 64) : four;
  if constexpr (DP <= 64)
    if (wgs < 2 * cus && a.Lk > 2 * Shape<T, DP>::BN)
      return few ? launch_one<T, DP, 2, 2, WIDE>(a, out, os, ovec, lse, s)
                 : launch_one<T, DP, 4, 2, WIDE>(a, out, os, ovec, lse, s);
  return few ? launch_one<T, DP, 2, 1, WIDE>(a, out, os, ovec, lse, s)
             : launch_one<T, DP, 4, 1, WIDE>(a, out, os, ovec, lse, s);
}

template <typename T, int DP>
int launch_dim(const RelAttn& a, T* out, const View& os, int ovec, float* lse, int device, hipStream_t s) {
  return a.vec * sizeof(T) == 16 ? launch_wide<T, DP, true>(a, out, os, ovec, lse, device, s)
                                 : launch_wide<T, DP, false>(a, out, os, ovec, lse, device, s);
}

template <typename T>
int forward(RelAttn a, void* out, const View& os, float* lse, int device, hipStream_t s) {
  const void* in[3] = {a.q, a.k, a.v};
  const View iv[3] = {a.qs, a.ks, a.vs};
  a.vec = widest_load<T>(in, iv, 3, a.D);
  const void* op[1] = {out};
  const int ovec = widest_load<T>(op, &os, 1, a.D);
  T* o = static_cast<T*>(out);
  if (a.D <= 32) return launch_dim<T, 32>(a, o, os, ovec, lse, device, s);
  if (a.D <= 64) return launch_dim<T, 64>(a, o, os, ovec, lse, device, s);
  return launch_dim<T, 128>(a, o, os, ovec, lse, device, s);
}

}  // namespace
}  // namespace fa

extern "C" {

FA_API int fa_gpu_rel_attention_workspace(int B, int H, int Hk, int Lq, int Lk, int D, int n,
                                          int device,
                                          int64_t* out_bytes) {
  if (!out_bytes) return FA_E_ARG;
  if (n < 1 || n > FA_REL_MAX) return FA_E_SHAPE;
  if (const int e = fa::check_attention(B, H, Hk, Lq, Lk, D, nullptr, 1, nullptr)) return e;
  return fa::rows_workspace(B, H, Hk, Lq, Lk, D, device, out_bytes);
}

FA_API int fa_gpu_rel_attention(const void* q, const void* k, const void* v, int dtype, int B,
                                int H, int Hk, int Lq, int Lk, int D, const int64_t* strides,
                                const void* table, int rows, const int* row_of, int lo, int n,
                                int grid_w, int64_t q_start, const int* q_starts,
                                const int* key_lengths, const uint8_t* mask, int mask_b,
                                const int64_t* mask_strides, int causal, double scale, void* out,
                                float* lse, void* workspace, int64_t workspace_bytes, int device,
                                void* stream) {
  using namespace fa;
  if (!q || !k || !v || !strides || !table || !out) return FA_E_ARG;
  const bool table_f32 = dtype & FA_TABLE_F32;
  dtype &= ~FA_TABLE_F32;
  if (const int e = check_attention(B, H, Hk, Lq, Lk, D, mask, mask_b, mask_strides)) return e;
  if (const int e = check_relpos(row_of, rows, lo, n, grid_w, Lq, Lk, q_start, q_starts)) return e;
  if (const int e = check_strides(strides, 4, dtype)) return e;
  DeviceScope scope(device);
  if (scope.status != hipSuccess) return -static_cast<int>(scope.status);
  const RelAttn a = rel_attn_args(q, k, v, B, H, Hk, Lq, Lk, D, strides, table, table_f32,
                                  RelPos{row_of, lo, n, grid_w}, q_start, q_starts, key_lengths,
                                  mask, mask_b, mask_strides, causal, scale);
  const View os{strides[9], strides[10], strides[11]};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (window_serve(a)) return window_forward(dtype, a, out, os, device, s);
  if (rows_serve(a)) return rows_forward(dtype, a, out, os, lse, workspace, workspace_bytes, device, s);
  switch (dtype) {
    case FA_F16: return forward<_Float16>(a, out, os, lse, device, s);
    case FA_BF16: return forward<__bf16>(a, out, os, lse, device, s);
    case FA_F32: return forward<float>(a, out, os, lse, device, s);
    default: return FA_E_DTYPE;
  }
}

}  // extern "C"
