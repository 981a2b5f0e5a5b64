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
  RelPos pos;
  int q0;               // position of query 0 where q_starts is null
  const int* q_starts;  // [B]
  const int* key_lengths;
  const uint8_t* mask;
  int mask_b;
  int64_t mb, mh, mq, mk;
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

constexpr float LOG2E = 1.4426950408889634f;
constexpr float INF = __builtin_inff();

// One head's bias by slot in LDS, times log2(e), with PAD copies of either end's
// value: a 32 x 32 block that has one difference within (lo, lo + n - 1) has none
// further than 62 past it, so its reads need no clamp.
constexpr int PAD = 64;
template <typename T>
__device__ inline void load_bias(float* eb, const T* table, int H, int h, const RelPos& pos,
                                 int tid, int nt) {
  for (int t = tid; t < pos.n + 2 * PAD; t += nt) {
    const int row = pos.row_of[min(max(t - PAD, 0), pos.n - 1)];
    eb[t] = widen(table[static_cast<int64_t>(row) * H + h]) * LOG2E;
  }
}

// How the pairs of a 32 x 32 block stand to the bias table.
enum : int { NEAR = 0, ALL_BELOW = 1, ALL_ABOVE = 2 };
__device__ inline int block_kind(const RelPos& pos, int dmin, int dmax) {
  return dmax <= pos.lo ? ALL_BELOW : dmin >= pos.lo + pos.n - 1 ? ALL_ABOVE : NEAR;
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

inline RelAttn rel_attn_args(const void* q, const void* k, const void* v, int B, int H, int Hk,
                             int Lq, int Lk, int D, const int64_t* st, const void* table,
                             const RelPos& pos, int64_t q_start, const int* q_starts,
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
  }
  a.causal = causal;
  a.scale = static_cast<float>(scale);
  return a;
}

// Raises a kernel's limit of LDS per workgroup where a launch asks for more than the
// default; the limit is the device's.
template <typename K> inline int launch_lds(K kernel, size_t bytes) {
  if (bytes > 64 * 1024)
    FA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                   hipFuncAttributeMaxDynamicSharedMemorySize,
                                   static_cast<int>(bytes)));
  return FA_OK;
}

}  // namespace fa
