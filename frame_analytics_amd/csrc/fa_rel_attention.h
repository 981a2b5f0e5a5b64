// What the forward and the backward pass of the attention with a relative position
// bias share: the arguments, the bias of a block, and which of its pairs count.
#pragma once

#include "fa_matrix.h"
#include "fa_relpos.h"

namespace fa {

struct View {  // strides in elements
  int64_t b, h, t;
};

struct RelAttn {
  const void *q, *k, *v;
  View qs, ks, vs;
  int B, H, Hk, Lq, Lk, D;
  int vec;  // elements per load that q, k, v (and the backward's views) allow
  const void* table;
  int table_f32;  // the table is float32 whatever the type of q
  RelPos pos;
  int q0;               // position of query 0 where q_starts is null
  const int* q_starts;  // [B]
  const int* key_lengths;
  const uint8_t* mask;
  int mask_b;
  int64_t mb, mh, mq, mk;
  int mask64;  // the mask's rows are 64 bytes on 16-byte boundaries
  int causal;
  float scale;
  __device__ inline int start(int b) const {
    return q_starts ? min(max(q_starts[b], -POS_MOST), POS_MOST) : q0;
  }
  __device__ inline int keys(int b) const {
    return key_lengths ? min(max(key_lengths[b], 0), Lk) : Lk;
  }
  __device__ inline const uint8_t* mask_of(int b, int h) const {
    return mask ? mask + (b % mask_b) * mb + h * mh : nullptr;
  }
};

// go(table), once, with the table in its type: a test at each entry would hold up the reads
// (24576 windows of 8 x 8 with gradients 633 us, and 644 so).
template <typename T, typename Go> __device__ inline void with_table(const RelAttn& a, const Go& go) {
  if (sizeof(T) == 2 && a.table_f32) go(static_cast<const float*>(a.table));
  else go(static_cast<const T*>(a.table));
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr float INF = __builtin_inff();

// A bias times log2(e).  Past 2^126 that product would leave float32 (the lowest values of
// bfloat16 and float32 hide pairs in many a program): from there on it grows by 0.8, finite
// at the type's limit and in the same order.  A row of equal extremes has equal weights so.
__device__ inline float bias_log2(float v) {
  constexpr float T = 0x1p126f;
  const float m = __builtin_fabsf(v);
  return m > T ? __builtin_copysignf(T * LOG2E + (m - T) * 0.8f, v) : v * LOG2E;
}

// The largest bias (times log2(e)) that may be taken with a row's maximum at once, s + (far -
// maximum), and the largest maximum that may be kept with its sum in one number: larger ones
// round the scores, and have to round all of a row alike.
constexpr float FAR_MOST = 4096.0f;

// The bias of `heads` heads from h on, by slot in LDS, times log2(e), with PAD copies
// of either end's value: a 32 x 32 block that has one difference within (lo, lo + n -
// 1) has none further than 62 past it, so its reads need no clamp.  The two reads of a
// value depend on one another; four of each are under way at once.
constexpr int PAD = 64;
template <typename T>
__device__ inline void load_bias(float* eb, const RelAttn& a, int h, int heads, int tid, int nt) {
  const RelPos& pos = a.pos;
  const int np = pos.n + 2 * PAD, total = heads * np;
  with_table<T>(a, [&](auto* table) {
    for (int t0 = tid; t0 < total; t0 += 4 * nt) {
      int row[4], head[4];
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = min(t0 + e * nt, total - 1);
        head[e] = heads == 1 ? 0 : t / np;
        row[e] = pos.row_of[min(max(t - head[e] * np - PAD, 0), pos.n - 1)];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = widen(table[static_cast<int64_t>(row[e]) * a.H + h + head[e]]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (t0 + e * nt < total) eb[t0 + e * nt] = bias_log2(v[e]);
    }
  });
}

// Whether the biases past both ends of a head's table in LDS, np floats wide, are below
// FAR_MOST: asked once, behind a barrier before the loop over tiles (read from memory at the
// kernel's start, one load after the other, it took 1 us more of 43).
__device__ inline bool far_serves(const float* eb, int np) {
  return __builtin_amdgcn_readfirstlane(__builtin_fabsf(eb[0]) < FAR_MOST && __builtin_fabsf(eb[np - 1]) < FAR_MOST);
}

// The codes of a window's tokens in LDS, the last one's repeated to a whole tile (a
// division for each token here, in place of one for each pair).
inline __host__ __device__ int codes_room(int n) { return (n + 63) / 64 * 64; }
__device__ inline void load_codes(int* codes, const RelPos& pos, int n, int tid, int nt) {
  for (int t = tid; t < codes_room(n); t += nt) codes[t] = pos.code(min(t, n - 1));
}

// What a call with gradients keeps of each row's softmax: a shift, and for all rows behind
// them a factor, with which the weights are 2^(score - shift) times the factor.  The shift
// is the log of the sum and the factor 1, unless the largest score would round the sum away
// (a row whose biases are all the type's lowest): then that score and one over the sum.  A
// row that sees nothing has a shift of +inf.
__device__ inline void keep_row(float* rows, int64_t all, int64_t row, float top, float sum) {
  const bool plain = sum == 0.0f || __builtin_fabsf(top) < FAR_MOST;
  rows[row] = sum == 0.0f ? INF : plain ? top + __builtin_log2f(sum) : top;
  rows[all + row] = plain ? 1.0f : 1.0f / sum;
}
// Whether a row may have a factor other than 1.
__device__ inline bool has_factor(float shift) { return !(__builtin_fabsf(shift) < FAR_MOST) && shift != INF; }

// What the output's rounding left, kept behind the rows' for 16-bit types on a line:
// D_i = dout_i . out_i is subtracted from every dP of a row, and a row's far keys share one
// entry of the table, which takes D_i's error as many times.  Measured on a causal line of
// 2048 in bfloat16, three inputs: the largest relative error of a gradient 2.5e-3 without
// it and 2.4e-3 with, the largest difference from plain float32 0.084 .. 0.11 and 0.053 ..
// 0.068, 169 .. 172 us and 169 .. 171.  In a window an entry takes one pair of a row: 16 x
// 16 windows had 3.0e-4 with it and without, and 740 us without against 776 with, so that
// they keep none.
template <typename T> __device__ inline T* low_of(const float* lse, int64_t rows) {
  return reinterpret_cast<T*>(const_cast<float*>(lse) + (2 * rows + 3) / 4 * 4);
}

// How the pairs of a 32 x 32 block stand to the bias table.
enum : int { NEAR = 0, ALL_BELOW = 1, ALL_ABOVE = 2 };
__device__ inline int block_kind(const RelPos& pos, int dmin, int dmax) {
  return dmax <= pos.lo ? ALL_BELOW : dmin >= pos.lo + pos.n - 1 ? ALL_ABOVE : NEAR;
}

// The bias past an end of a head's table in LDS, np floats wide, in a scalar register (for
// dK and dV: there far_serves and the bias in a vector register spill 40 registers, 16-bit
// heads of 64).
__device__ inline float far_bias(const float* eb, int np, int kind) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(kind == ALL_BELOW ? eb[0] : eb[np - 1])));
}

// Bit r: whether pair r of a lane's 16 counts, steps 8 (r / 4) + r % 4 from its first
// along the keys (or the queries): the first `count` steps may, and where there is a mask
// its byte `step` bytes further on each step.
__device__ inline uint32_t mask_bits(const uint8_t* p, int64_t step, int count) {
  uint32_t bits = 0;
  if (count > 27) {  // the last step is 27
    uint8_t v[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) v[r] = p[(8 * (r / 4) + r % 4) * step];
#pragma unroll
    for (int r = 0; r < 16; ++r) bits |= (v[r] != 0 ? 1u : 0u) << r;
  } else {
#pragma unroll 1
    for (int r = 0; r < 16; ++r) {
      const int s = 8 * (r / 4) + r % 4;
      if (s < count && p[s * step]) bits |= 1u << r;
    }
  }
  return bits;
}
// Steps below `to`.
__device__ inline uint32_t first_bits(int to) {
  uint32_t bits = 0;
#pragma unroll
  for (int g = 0; g < 4; ++g) bits |= (15u >> (4 - min(max(to - 8 * g, 0), 4))) << (4 * g);
  return bits;
}
// The pairs of query q (position qpos) with the keys from k on.
__device__ inline uint32_t seen_keys(const RelAttn& a, const uint8_t* mask, int q, int qpos, int k, int len) {
  uint32_t bits = first_bits(min(len, a.causal ? max(qpos, -1) + 1 : len) - k);
  if (mask) bits &= mask_bits(mask + afresh(q) * a.mq + k * a.mk, a.mk, len - k);
  return bits;
}
// 16 scores of which some may be hidden: those are -inf.
__device__ inline void hide(f32x16& s, uint32_t seen) {
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = seen >> r & 1 ? s[r] : -INF;
}

// acc += V^T P^T over 16 keys of which some are hidden from some queries: a value
// that is not finite must not reach the queries that do not see it (0 x inf).  The
// finite values go through the product; the others are counted by two more, with 1 in
// the place of each value and of each visible pair (bit i of `seen`: a weight may be
// rounded to zero and its pair count all the same).
template <typename T>
__device__ inline f32x16 guarded(typename Mat<T>::V8 v, typename Mat<T>::V8 p, f32x16 acc, uint32_t seen) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) bad |= !(__builtin_fabsf(widen(v[i])) < INF);
  if (__ballot(bad) == 0) return Mat<T>::mma(v, p, acc);
  typename Mat<T>::V8 fine;
#pragma unroll
  for (int i = 0; i < 8; ++i) fine[i] = __builtin_fabsf(widen(v[i])) < INF ? v[i] : T(0);
  acc = Mat<T>::mma(fine, p, acc);
#pragma unroll 1
  for (float way = INF; way != 0.0f; way = way > 0.0f ? -INF : 0.0f) {
    typename Mat<T>::V8 bad_v, ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = widen(v[i]);
      bad_v[i] = x == way || x != x ? T(1) : T(0);  // NaN counts both ways
      ones[i] = seen >> i & 1 ? T(1) : T(0);
    }
    f32x16 n;
#pragma unroll
    for (int r = 0; r < 16; ++r) n[r] = 0.0f;
    n = Mat<T>::mma(bad_v, ones, n);
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] += n[r] > 0.0f ? way : 0.0f;
  }
  return acc;
}

template <typename T>
inline int widest_load(const void* const* ptr, const View* views, int count, int D) {
  for (int w : {16 / int(sizeof(T)), 4 / int(sizeof(T)), 1}) {
    if (w < 1 || D % w != 0) continue;
    bool ok = true;
    for (int i = 0; i < count; ++i)
      ok = ok && reinterpret_cast<uintptr_t>(ptr[i]) % (w * sizeof(T)) == 0 && views[i].b % w == 0 &&
           views[i].h % w == 0 && views[i].t % w == 0;
    if (ok) return w;
  }
  return 1;
}

inline int check_attention(int B, int H, int Hk, int Lq, int Lk, int D, const uint8_t* mask,
                           int mask_b, const int64_t* mask_strides) {
  if (B < 1 || H < 1 || Hk < 1 || H % Hk != 0 || Lq < 1 || Lk < 1 || D < 1 || D > 128)
    return FA_E_SHAPE;
  if (static_cast<int64_t>(B) * H > (1 << 30) || Lq > (1 << 29) || Lk > (1 << 29)) return FA_E_SHAPE;
  if (mask && !mask_strides) return FA_E_ARG;
  if (mask && (mask_b < 1 || B % mask_b != 0)) return FA_E_SHAPE;
  return FA_OK;
}

// `count` views' token strides (the third of each three): see Rows.
inline int check_strides(const int64_t* st, int count, int dtype) {
  const int64_t most = 0x7fffffff / (MAX_ROWS * (dtype == FA_F32 ? 4 : 2));
  for (int i = 0; i < count; ++i)
    if (st[3 * i + 2] < 0 || st[3 * i + 2] > most) return FA_E_SHAPE;
  return FA_OK;
}

inline RelAttn rel_attn_args(const void* q, const void* k, const void* v, int B, int H, int Hk,
                             int Lq, int Lk, int D, const int64_t* st, const void* table,
                             bool table_f32, const RelPos& pos, int64_t q_start, const int* q_starts,
                             const int* key_lengths, const uint8_t* mask, int mask_b,
                             const int64_t* ms, int causal, double scale) {
  RelAttn a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.qs = {st[0], st[1], st[2]};
  a.ks = {st[3], st[4], st[5]};
  a.vs = {st[6], st[7], st[8]};
  a.B = B;
  a.H = H;
  a.Hk = Hk;
  a.Lq = Lq;
  a.Lk = Lk;
  a.D = D;
  a.table = table;
  a.table_f32 = table_f32;
  a.pos = pos;
  a.q0 = clamp_pos(q_start);
  a.q_starts = q_starts;
  a.key_lengths = key_lengths;
  a.mask = mask;
  a.mask_b = mask ? mask_b : 1;
  if (mask) {
    a.mb = ms[0];
    a.mh = ms[1];
    a.mq = ms[2];
    a.mk = ms[3];
    a.mask64 = a.mk == 1 && Lk == 64 && a.mq >= 0 && a.mq < (1 << 22) && (a.mb | a.mh | a.mq) % 16 == 0 &&
               reinterpret_cast<uintptr_t>(mask) % 16 == 0;
  }
  a.causal = causal;
  a.scale = static_cast<float>(scale);
  return a;
}

constexpr size_t MOST_LDS = 160 * 1024;  // a workgroup's

// Raises a kernel's limit of LDS per workgroup where a launch asks for more than the
// default; the limit is the device's.
template <typename K> inline int launch_lds(K kernel, size_t bytes) {
  if (bytes > 64 * 1024)
    FA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                   hipFuncAttributeMaxDynamicSharedMemorySize,
                                   static_cast<int>(bytes)));
  return FA_OK;
}

// fa_rel_bias.hip: dtable from `parts` rows of n sums by slot for each head
template <typename T>
void launch_table_sum(const float* partial, int parts, int n, const int* row_of, int rows, int H,
                      T* dtable, hipStream_t s);

template <typename T>
void launch_table_sum(const RelAttn& a, const float* partial, int parts, int rows, void* dtable, hipStream_t s) {
  if (sizeof(T) == 2 && a.table_f32)
    launch_table_sum<float>(partial, parts, a.pos.n, a.pos.row_of, rows, a.H, static_cast<float*>(dtable), s);
  else
    launch_table_sum<T>(partial, parts, a.pos.n, a.pos.row_of, rows, a.H, static_cast<T*>(dtable), s);
}

// fa_rel_attention_rows.hip: few queries against many keys
int rows_workspace(int B, int H, int Hk, int Lq, int Lk, int D, int device, int64_t* bytes);
bool rows_serve(const RelAttn& a);
int rows_forward(int dtype, const RelAttn& a, void* out, const View& os, float* lse, void* ws,
                 int64_t ws_bytes, int device, hipStream_t s);

// fa_rel_attention_window.hip: windows of up to 64 tokens
struct WindowGrads {
  const void* dout;
  View gs;
  void *dq, *dk, *dv;
  View dqs, dks, dvs;
  float* parts;  // [H][window_parts][n], or null: the table needs no gradient
};
bool window_serve(const RelAttn& a);
int window_parts(int B, int H, int device);
int window_forward(int dtype, const RelAttn& a, void* out, const View& os, int device, hipStream_t s);
int window_backward(int dtype, const RelAttn& a, const WindowGrads& g, int rows, void* dtable, int device,
                    hipStream_t s);

}  // namespace fa
