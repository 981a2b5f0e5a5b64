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

// Eight elements d .. d + 7 of a row of D, zero from D on (all zero unless `on`).
// `vec` elements are read at once: the widest that the row's address, the strides
// and D allow (16 bytes, 4 bytes or one element; uniform over the launch).
template <typename T>
__device__ inline typename Mat<T>::V8 load8(const T* row, int d, int D, int vec, bool on) {
  typename Mat<T>::V8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = T(0);
  if (vec * int(sizeof(T)) == 16) {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int e = 0; e < 8; e += W) {
      if (on && d + e < D) {
        if constexpr (W == 8) {
          r = *reinterpret_cast<const typename Mat<T>::V8*>(row + d);
        } else {
          const typename Mat<T>::V4 t = *reinterpret_cast<const typename Mat<T>::V4*>(row + d + e);
#pragma unroll
          for (int i = 0; i < 4; ++i) r[e + i] = t[i];
        }
      }
    }
  } else if (sizeof(T) == 2 && vec == 2) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      if (on && d + e < D) {
        const typename Mat<T>::V2 t = *reinterpret_cast<const typename Mat<T>::V2*>(row + d + e);
        r[e] = t[0];
        r[e + 1] = t[1];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (on && d + e < D) r[e] = row[d + e];
  }
  return r;
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

// A tile's rows [row0, row0 + ROWS) on their way from memory to LDS: read into
// registers while the tile before is worked on, stored after.  Rows from row_end on
// and elements from D on are zeros.
template <typename T, int DP, int ROWS, int NT> struct TileLoad {
  static constexpr int PER_ROW = DP / 8;
  static constexpr int N = (ROWS * PER_ROW + NT - 1) / NT;
  typename Mat<T>::V8 r[N];
  __device__ inline void load(const T* base, int64_t stride, int row0, int row_end, int D, int vec,
                              int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * NT, row = c / PER_ROW, d = (c % PER_ROW) * 8;
      const bool on = row < ROWS && row0 + row < row_end;
      r[i] = load8<T>(base + (on ? (row0 + row) * stride : 0), d, D, vec, on);
    }
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

}  // namespace fa
