// Element types, fragments and matrix instructions of the training operators.
//
// Every product here is made of 32 x 32 blocks: mma32 multiplies a 32 x 16 by a
// 16 x 32 fragment into a 32 x 32 float32 block.  With l the lane and h = l / 32:
//   A fragment: row l % 32, eight k values, slot (h, i);
//   B fragment: column l % 32, the same eight k values;
//   C block:    column l % 32, register r holds row 8 (r / 4) + 4 h + r % 4.
// A and B only have to agree on which k stands in slot (h, i).  "Straight" slots are
// k = 8 h + i (eight neighbours: one 16-byte read).  "Split" slots are k = 8 (i / 4)
// + 4 h + i % 4, the rows that registers 0-7 (or 8-15) of a C block hold: a C block
// rounded to the element type IS the B fragment of the next product over its rows,
// with no exchange between lanes.
#pragma once

#include "fa_common.h"

namespace fa {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Mat;
template <> struct Mat<_Float16> {
  typedef f16x8 V8;
  typedef f16x4 V4;
  typedef f16x2 V2;
  static __device__ inline f32x16 mma(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mat<__bf16> {
  typedef b16x8 V8;
  typedef b16x4 V4;
  typedef b16x2 V2;
  static __device__ inline f32x16 mma(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
// float32: eight products over two k each; slot i of both halves makes one of them
template <> struct Mat<float> {
  typedef f32x8 V8;
  typedef f32x4 V4;
  typedef f32x2 V2;
  static __device__ inline f32x16 mma(V8 a, V8 b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// Rows of a view, read with buffer instructions: what lies outside reads as zero, so
// edges cost a select and no branch.  `base` is the first row that the workgroup
// reads (rows further on are reached by 32-bit byte offsets, so a view's token
// stride times MAX_ROWS has to stay below 2^31 bytes; the base itself is 64-bit).
constexpr int MAX_ROWS = 256;
constexpr int OUTSIDE = static_cast<int>(0x80000000u);
template <typename T> struct Rows {
  __amdgpu_buffer_rsrc_t rsrc;
  int stride;  // bytes
  __device__ inline Rows(const T* base, int64_t stride_elements)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, 0x7fffffff, 0x00020000)),
        stride(static_cast<int>(stride_elements * sizeof(T))) {}

  // Elements d .. d + 7 of row `row`, zero from D on (all zero unless `on`).  `vec`
  // elements are read at once: the widest that the views' addresses, their strides and
  // D allow (16 bytes, 4 bytes or one element; uniform over the launch).
  __device__ inline typename Mat<T>::V8 wide(int row, int d, int D, bool on) const {
    const int at = row * stride + d * int(sizeof(T));
    if constexpr (sizeof(T) == 2) {
      return __builtin_bit_cast(typename Mat<T>::V8, __builtin_amdgcn_raw_buffer_load_b128(
                                                         rsrc, on && d < D ? at : OUTSIDE, 0, 0));
    } else {
      const f32x4 x = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                    rsrc, on && d < D ? at : OUTSIDE, 0, 0));
      const f32x4 y = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                    rsrc, on && d + 4 < D ? at + 16 : OUTSIDE, 0, 0));
      return f32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    }
  }
  __device__ inline typename Mat<T>::V8 pairs(int row, int d, int D, bool on) const {
    if constexpr (sizeof(T) == 2) {
      const int at = row * stride + d * int(sizeof(T));
      typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
      u32x4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[e] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, on && d + 2 * e < D ? at + 4 * e : OUTSIDE, 0, 0);
      return __builtin_bit_cast(typename Mat<T>::V8, r);
    } else {
      return single(row, d, D, on);  // (float32: a pair is one element)
    }
  }
  __device__ inline typename Mat<T>::V8 single(int row, int d, int D, bool on) const {
    const int at = row * stride + d * int(sizeof(T));
    typename Mat<T>::V8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int o = on && d + e < D ? at + e * int(sizeof(T)) : OUTSIDE;
      if constexpr (sizeof(T) == 2)
        r[e] = __builtin_bit_cast(T, static_cast<unsigned short>(
                                         __builtin_amdgcn_raw_buffer_load_b16(rsrc, o, 0, 0)));
      else
        r[e] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(rsrc, o, 0, 0));
    }
    return r;
  }
};

// Whether a launch's views are all read 16 bytes at a time is part of the kernel's type
// (WIDE): the narrow reads need up to eight registers for each element pair on its way
// and would set the register count of the wide ones.
// N fragments along a row, elements d0 + 16 i .., as Rows reads them.
template <typename T, bool WIDE, int N>
__device__ inline void load_row(typename Mat<T>::V8 (&f)[N], const Rows<T>& rows, int row, int d0, int D,
                                int vec, bool on) {
  if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = rows.wide(row, d0 + 16 * i, D, on);
  } else if (sizeof(T) == 2 && vec == 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = rows.pairs(row, d0 + 16 * i, D, on);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = rows.single(row, d0 + 16 * i, D, on);
  }
}

// Four elements d .. d + 3 of a row of D, those before D.
template <typename T>
__device__ inline void store4(T* row, int d, int D, int vec, const float* v) {
  typename Mat<T>::V4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = T(v[i]);
  if (vec * int(sizeof(T)) == 16) {  // 16-byte aligned rows, D a multiple of 4
    if (d < D) *reinterpret_cast<typename Mat<T>::V4*>(row + d) = r;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < D) row[d + i] = r[i];
  }
}

// The larger of a value in lanes l and l ^ 32, in both; and their sum.
__device__ inline float both_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}
__device__ inline float both_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  return __int_as_float(r[0]) + __int_as_float(r[1]);
}

// LDS that one wave wrote is read by its other lanes after this.
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A tile of ROWS rows of DP elements in LDS, rows LD apart: 16 bytes of padding put
// the rows that one instruction reads on different banks.
template <typename T, int DP> struct Tile {
  static constexpr int LD = DP + 16 / int(sizeof(T));
  typedef typename Mat<T>::V8 V8;

  // straight fragment: row `row` (l % 32 added by the caller), k = k0 + 8 h + i
  static __device__ inline V8 straight(const T* t, int row, int k) {
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const V8*>(t + row * LD + k);
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(t + row * LD + k);
      const f32x4 b = *reinterpret_cast<const f32x4*>(t + row * LD + k + 4);
      return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }

  // split fragment of the transpose: lane l holds column col0 + l % 32 of the rows
  // row0 + 8 (i / 4) + 4 h + i % 4.  16-bit: ds_read_b64_tr_b16, in which each 16
  // lanes read a 4 x 16 block (lane i: row i / 4, columns 4 (i % 4) ..) and lane i
  // receives column i.
  static __device__ inline V8 transposed(const T* t, int row0, int col0, int lane) {
    V8 r;
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const T* p = t + (row0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * LD + col0 +
                   16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 8 * LD));
      typedef typename Mat<T>::V4 V4;
      const V4 x = __builtin_bit_cast(V4, a), y = __builtin_bit_cast(V4, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r[i] = x[i];
        r[4 + i] = y[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        r[i] = t[(row0 + 8 * (i / 4) + 4 * (lane >> 5) + i % 4) * LD + col0 + (lane & 31)];
    }
    return r;
  }
};

// A value that the compiler takes as new each time: offsets made from it are computed
// where they are used, not kept in registers through a loop (there is one for each load).
__device__ inline int afresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Whether any element of a register of T is not finite: its exponent is all ones.
template <typename T> __device__ inline bool not_finite(unsigned x) {
  if constexpr (sizeof(T) == 4) return (x & 0x7f800000u) == 0x7f800000u;
  constexpr unsigned E = std::is_same<T, _Float16>::value ? 0x7c007c00u : 0x7f807f80u;
  constexpr unsigned ONE = E & (~E << 1);  // an exponent's lowest bit: all ones carry into the sign
  return (((x & E) + ONE) & 0x80008000u) != 0;
}

// A tile of ROWS rows on its way from memory to LDS: read into registers while the
// tile before is worked on, stored after.  The first `valid` rows are read, the rest
// and elements from D on are zeros.
template <typename T, int DP, int ROWS, int NT, bool WIDE> struct TileLoad {
  static constexpr int PER_ROW = DP / 8;
  static constexpr int N = (ROWS * PER_ROW + NT - 1) / NT;
  typename Mat<T>::V8 r[N];
  __device__ inline bool not_finite() const {
    constexpr int W = sizeof(T) * 2;
    typedef unsigned words __attribute__((ext_vector_type(W)));
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const words w = __builtin_bit_cast(words, r[i]);
#pragma unroll
      for (int e = 0; e < W; ++e) bad |= fa::not_finite<T>(w[e]);
    }
    return bad;
  }
  __device__ inline void load(const T* base, int64_t stride, int valid, int D, int vec, int tid) {
    static_assert(NT % PER_ROW == 0, "a thread keeps its columns");
    constexpr int STEP = NT / PER_ROW;  // rows between a thread's pieces
    valid = min(valid, ROWS);
    tid = afresh(tid);
    const int row = tid / PER_ROW, d = (tid % PER_ROW) * 8;
    auto each = [&](auto read) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        r[i] = read(Rows<T>(base + i * STEP * stride, stride), row + i * STEP < valid);
    };
    if constexpr (WIDE)
      each([&](const Rows<T>& rows, bool on) { return rows.wide(row, d, D, on); });
    else if (sizeof(T) == 2 && vec == 2)
      each([&](const Rows<T>& rows, bool on) { return rows.pairs(row, d, D, on); });
    else
      each([&](const Rows<T>& rows, bool on) { return rows.single(row, d, D, on); });
  }
  __device__ inline void store(T* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * NT, row = c / PER_ROW, d = (c % PER_ROW) * 8;
      if (ROWS * PER_ROW % NT != 0 && row >= ROWS) continue;
      T* p = lds + row * Tile<T, DP>::LD + d;
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<typename Mat<T>::V8*>(p) = r[i];
      } else {
        *reinterpret_cast<f32x4*>(p) = f32x4{r[i][0], r[i][1], r[i][2], r[i][3]};
        *reinterpret_cast<f32x4*>(p + 4) = f32x4{r[i][4], r[i][5], r[i][6], r[i][7]};
      }
    }
  }
};

// The same for 16-bit rows of an even number of elements on 4-byte boundaries: each
// thread takes pairs, neighbouring threads neighbouring pairs, so an instruction covers
// whole rows (TileLoad's 16-byte pieces, read 4 bytes at a time, cover each line four times).
template <typename T, int DP, int ROWS, int NT> struct PairLoad {
  static constexpr int PER_ROW = DP / 2;
  static constexpr int N = ROWS * PER_ROW / NT;
  static_assert(ROWS * PER_ROW % NT == 0, "whole rounds");
  unsigned r[N];
  __device__ inline bool not_finite() const {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N; ++i) bad |= fa::not_finite<T>(r[i]);
    return bad;
  }
  __device__ inline void load(const T* base, int64_t stride, int valid, int D, int, int tid) {
    static_assert(NT % PER_ROW == 0, "a thread keeps its columns");
    constexpr int STEP = NT / PER_ROW;
    tid = afresh(tid);
    const int row = tid / PER_ROW, d = (tid % PER_ROW) * 2;
    valid = d < D ? valid : 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Rows<T> rows(base + i * STEP * stride, stride);
      r[i] = __builtin_amdgcn_raw_buffer_load_b32(
          rows.rsrc, row + i * STEP < valid ? row * rows.stride + d * int(sizeof(T)) : OUTSIDE, 0, 0);
    }
  }
  __device__ inline void store(T* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * NT, row = c / PER_ROW, d = (c % PER_ROW) * 2;
      *reinterpret_cast<unsigned*>(lds + row * Tile<T, DP>::LD + d) = r[i];
    }
  }
};

}  // namespace fa
