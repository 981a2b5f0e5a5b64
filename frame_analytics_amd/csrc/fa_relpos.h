// Relative positions: the one-number code of a token, and the table row of a pair.
#pragma once

#include "fa_common.h"
#include "fa_train_abi.h"

namespace fa {

// The table row of a pair is a function of c(i) - c(j), clamped to n values from lo:
// on a line the rows of far distances are one row each way, in a window every
// difference of coordinates has its own (c(t) = y (2 w - 1) + x, so no two share one).
// For one key, different queries have different c(i) - c(j), and the other way round.
struct RelPos {
  const int* row_of;
  int lo, n, grid_w;
  __device__ inline int code(int t) const { return grid_w ? t + (grid_w - 1) * (t / grid_w) : t; }
  __device__ inline int slot(int delta) const { return min(max(delta - lo, 0), n - 1); }
};

// Positions past +-2^30 are taken as there: no difference overflows.
constexpr int POS_MOST = 1 << 30;
__host__ __device__ inline int clamp_pos(int64_t s) {
  return static_cast<int>(s < -POS_MOST ? -POS_MOST : s > POS_MOST ? POS_MOST : s);
}

inline int check_relpos(const int* row_of, int rows, int lo, int n, int grid_w, int lq,
                        int lk, int64_t q_start, const int* q_starts) {
  if (!row_of) return FA_E_ARG;
  if (rows < 1 || n < 1 || n > FA_REL_MAX || grid_w < 0) return FA_E_SHAPE;
  if (grid_w > 0) {  // every pair's slot has to be its own: the whole window's table
    if (lq != lk || q_start != 0 || q_starts || lq % grid_w != 0) return FA_E_SHAPE;
    if (n != (2 * static_cast<int64_t>(lq / grid_w) - 1) * (2 * static_cast<int64_t>(grid_w) - 1) ||
        lo != -(n / 2))
      return FA_E_SHAPE;
  }
  return FA_OK;
}

template <typename T> __device__ inline float widen(T v) { return static_cast<float>(v); }

}  // namespace fa
