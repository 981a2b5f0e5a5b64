// The relative position bias as a tensor, and its gradient.
//
// out[h, i, j] = table[row(c(i) - c(j)), h] and its adjoint, the sum of up[h, i, j]
// over the pairs of a row.  Both move H Lq Lk elements once and do next to nothing
// else: the memory's rate bounds them, or the launches where they are small.
#include "fa_matrix.h"
#include "fa_relpos.h"

namespace fa {
namespace {

constexpr int NT = 256;

// ---------------------------------------------------------------------------
// forward
//
// A workgroup holds one head's n values in LDS and writes 16-byte pieces of the
// head's Lq x Lk plane, taken as one flat run (aligned pieces whatever Lk is; a piece
// may run over a row's end).
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(NT) void rel_bias_kernel(const T* table, int H, int Lq, int Lk,
                                                      RelPos pos, int q0, T* out) {
  constexpr int W = 16 / sizeof(T);
  extern __shared__ __align__(16) unsigned char smem[];
  T* val = reinterpret_cast<T*>(smem);
  const int h = blockIdx.y;
  for (int t = threadIdx.x; t < pos.n; t += NT)
    val[t] = table[static_cast<int64_t>(pos.row_of[t]) * H + h];
  __syncthreads();
  const int64_t plane = static_cast<int64_t>(Lq) * Lk;
  T* o = out + h * plane;
  // elements before the first 16-byte boundary of this head's plane
  const int64_t skip = ((16 - (reinterpret_cast<uintptr_t>(o) & 15)) & 15) / sizeof(T);
  const int64_t pieces = (plane - skip + W - 1) / W + 1;  // the first: the elements before it
  for (int64_t p = blockIdx.x * static_cast<int64_t>(NT) + threadIdx.x; p < pieces;
       p += static_cast<int64_t>(gridDim.x) * NT) {
    const int64_t e0 = p == 0 ? 0 : skip + (p - 1) * W;
    const int cnt = static_cast<int>(min<int64_t>(p == 0 ? skip : W, plane - e0));
    if (cnt <= 0) continue;
    int i = static_cast<int>(e0 / Lk), j = static_cast<int>(e0 - static_cast<int64_t>(i) * Lk);
    int ci = q0 + pos.code(i);
    T v[W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
      v[e] = val[pos.slot(ci - pos.code(j))];
      if (++j == Lk) {
        j = 0;
        i = min(i + 1, Lq - 1);
        ci = q0 + pos.code(i);
      }
    }
    if (cnt == W) {
      typedef typename std::conditional<W == 8, typename Mat<T>::V8, f32x4>::type V;
      V r;
#pragma unroll
      for (int e = 0; e < W; ++e) r[e] = v[e];
      *reinterpret_cast<V*>(o + e0) = r;
    } else {
      for (int e = 0; e < cnt; ++e) o[e0 + e] = v[e];
    }
  }
}

// ---------------------------------------------------------------------------
// backward
//
// A thread owns one difference delta = c(i) - c(j) of a band of query rows and adds
// its pairs in the order of the rows: no two threads write the same sum and the order
// is fixed.  For one row, neighbouring threads read neighbouring keys.  The sums of a
// band go to its own n slots (differences past either end into the end slots, through
// LDS); rel_bias_sum_kernel adds the bands and the differences of a table row.
// ---------------------------------------------------------------------------
constexpr int BAND = 32;

template <typename T>
__global__ __launch_bounds__(NT) void rel_bias_bwd_kernel(const T* up, int64_t sh, int64_t si,
                                                          int64_t sj, int Lq, int Lk, RelPos pos,
                                                          int q0, float* partial) {
  const int h = blockIdx.y, band = blockIdx.x;
  const int i0 = band * BAND, i1 = min(i0 + BAND, Lq);
  const T* u = up + h * sh;
  float* dst = partial + (static_cast<int64_t>(h) * gridDim.x + band) * pos.n;
  const int c0 = q0 + pos.code(i0), c1 = q0 + pos.code(i1 - 1);
  const int dmin = c0 - pos.code(Lk - 1), dmax = c1;
  float below = 0.0f, above = 0.0f;
  // slots that no pair of this band reaches
  for (int t = threadIdx.x; t < pos.n; t += NT)
    if (t + pos.lo < dmin || t + pos.lo > dmax) dst[t] = 0.0f;
  // the end slots gather what lies past them: written last, by thread 0
  for (int64_t d = static_cast<int64_t>(dmin) + threadIdx.x; d <= dmax; d += NT) {
    float acc = 0.0f;
    const int delta = static_cast<int>(d);
    if (pos.grid_w == 0) {
      const int a = max(i0, delta - q0), b = min(i1, delta - q0 + Lk);  // 0 <= j = q0+i-delta < Lk
      // (eight reads on their way at a time, added in order)
      const T* p = u + a * si + (static_cast<int64_t>(q0) + a - delta) * sj;
      int i = a;
      for (; i + 8 <= b; i += 8, p += 8 * (si + sj)) {
        T v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = p[e * (si + sj)];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc += widen(v[e]);
      }
      for (; i < b; ++i, p += si + sj) acc += widen(*p);
    } else {
      const int w = pos.grid_w, m = 2 * w - 1;
      const int s = delta - pos.lo;  // (dy + hgt - 1) m + dx + w - 1
      const int hgt = Lq / w, dy = s / m - (hgt - 1), dx = s % m - (w - 1);
      // the queries of the band whose key, dy rows and dx columns before, is in the window:
      // a run of columns in each row
      const int x0 = max(0, dx), x1 = min(w, w + dx);
      for (int y = max(i0 / w, dy); y <= min((i1 - 1) / w, hgt - 1 + dy); ++y) {
        const int a = max(y * w + x0, i0), b = min(y * w + x1, i1);
        const T* p = u + a * si + (a - dy * w - dx) * sj;
        for (int i = a; i < b; ++i, p += si + sj) acc += widen(*p);
      }
    }
    const int t = delta - pos.lo;
    if (t <= 0) below += acc;
    else if (t >= pos.n - 1) above += acc;
    else dst[t] = acc;
  }
  __shared__ float sums[2 * WAVES_PER_BLOCK];
  float lo, hi;
  block_sum2(below, above, sums, &lo, &hi);
  if (threadIdx.x == 0) {
    if (pos.n == 1) {
      dst[0] = lo + hi;
    } else {
      dst[0] = lo;
      dst[pos.n - 1] = hi;
    }
  }
}

}  // namespace

// dtable[r, h]: a workgroup adds, over `parts` partial rows of a head and over the
// slots of table row r, which stand next to one another.  Each thread takes its share
// in a fixed order, in float32 of at most parts * n / NT terms; the threads' sums are
// added by a fixed tree.  stride: floats from one partial row to the next.
template <typename T>
__global__ __launch_bounds__(NT) void rel_table_sum_kernel(const float* partial, int parts, int n,
                                                           const int* row_of, int H, T* dtable) {
  const int h = blockIdx.y, r = blockIdx.x;
  __shared__ int first, last;
  if (threadIdx.x == 0) {
    first = n;
    last = -1;
  }
  __syncthreads();
  for (int t = threadIdx.x; t < n; t += NT)
    if (row_of[t] == r) {
      atomicMin(&first, t);
      atomicMax(&last, t);
    }
  __syncthreads();
  const int f = first, w = last - first + 1;
  const float* p = partial + static_cast<int64_t>(h) * parts * n;
  float acc = 0.0f;
  if (w > 0) {
    const int64_t total = static_cast<int64_t>(parts) * w;
    for (int64_t k = threadIdx.x; k < total; k += NT) {
      const int64_t part = k / w;
      acc += p[part * n + f + (k - part * w)];
    }
  }
  __shared__ float sums[WAVES_PER_BLOCK];
  const float s = block_sum(acc, sums);
  if (threadIdx.x == 0) dtable[static_cast<int64_t>(r) * H + h] = T(s);
}

template <typename T>
void launch_table_sum(const float* partial, int parts, int n, const int* row_of, int rows, int H,
                      T* dtable, hipStream_t s) {
  rel_table_sum_kernel<T><<<dim3(rows, H), NT, 0, s>>>(partial, parts, n, row_of, H, dtable);
}
template void launch_table_sum<float>(const float*, int, int, const int*, int, int, float*, hipStream_t);
template void launch_table_sum<_Float16>(const float*, int, int, const int*, int, int, _Float16*, hipStream_t);
template void launch_table_sum<__bf16>(const float*, int, int, const int*, int, int, __bf16*, hipStream_t);

namespace {

inline int bands(int Lq) { return (Lq + BAND - 1) / BAND; }

template <typename T>
int bias_forward(const void* table, int H, int Lq, int Lk, const RelPos& pos, int q0, void* out,
                 int device, hipStream_t s) {
  constexpr int W = 16 / sizeof(T);
  const int64_t pieces = static_cast<int64_t>(Lq) * Lk / W + 2;
  const int64_t want = (pieces + NT - 1) / NT, most = (16 * cu_count(device) + H - 1) / H;
  const int gx = static_cast<int>(want < most ? want : most);
  rel_bias_kernel<T><<<dim3(gx, H), NT, pos.n * sizeof(T), s>>>(
      static_cast<const T*>(table), H, Lq, Lk, pos, q0, static_cast<T*>(out));
  FA_LAUNCH_CHECK();
  return FA_OK;
}

template <typename T>
int bias_backward(const void* up, const int64_t* st, int rows, int H, int Lq, int Lk,
                  const RelPos& pos, int q0, void* dtable, float* ws, hipStream_t s) {
  rel_bias_bwd_kernel<T><<<dim3(bands(Lq), H), NT, 0, s>>>(static_cast<const T*>(up), st[0], st[1],
                                                           st[2], Lq, Lk, pos, q0, ws);
  FA_LAUNCH_CHECK();
  launch_table_sum<T>(ws, bands(Lq), pos.n, pos.row_of, rows, H, static_cast<T*>(dtable), s);
  FA_LAUNCH_CHECK();
  return FA_OK;
}

}  // namespace
}  // namespace fa

extern "C" {

FA_API int fa_gpu_rel_bias(const void* table, int dtype, int rows, int H, int Lq, int Lk,
                           const int* row_of, int lo, int n, int grid_w, int64_t q_start,
                           void* out, int device, void* stream) {
  using namespace fa;
  if (!table || !out) return FA_E_ARG;
  if (H < 1 || H > 65535 || Lq < 1 || Lk < 1) return FA_E_SHAPE;
  if (const int e = check_relpos(row_of, rows, lo, n, grid_w, Lq, Lk, q_start, nullptr)) return e;
  DeviceScope scope(device);
  if (scope.status != hipSuccess) return -static_cast<int>(scope.status);
  const RelPos pos{row_of, lo, n, grid_w};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int q0 = clamp_pos(q_start);
  switch (dtype) {
    case FA_F16: return bias_forward<_Float16>(table, H, Lq, Lk, pos, q0, out, device, s);
    case FA_BF16: return bias_forward<__bf16>(table, H, Lq, Lk, pos, q0, out, device, s);
    case FA_F32: return bias_forward<float>(table, H, Lq, Lk, pos, q0, out, device, s);
    default: return FA_E_DTYPE;
  }
}

FA_API int fa_gpu_rel_bias_workspace(int H, int Lq, int Lk, int n, int64_t* out_bytes) {
  if (!out_bytes) return FA_E_ARG;
  if (H < 1 || H > 65535 || Lq < 1 || Lk < 1 || n < 1 || n > FA_REL_MAX) return FA_E_SHAPE;
  *out_bytes = static_cast<int64_t>(H) * fa::bands(Lq) * n * 4;
  return FA_OK;
}

FA_API int fa_gpu_rel_bias_backward(const void* up, const int64_t* up_strides, int dtype,
                                    int rows, int H, int Lq, int Lk, const int* row_of, int lo,
                                    int n, int grid_w, int64_t q_start, void* dtable,
                                    void* workspace, int64_t workspace_bytes, int device,
                                    void* stream) {
  using namespace fa;
  if (!up || !up_strides || !dtable || !workspace) return FA_E_ARG;
  int64_t need = 0;
  if (const int e = fa_gpu_rel_bias_workspace(H, Lq, Lk, n, &need)) return e;
  if (workspace_bytes < need) return FA_E_ARG;
  if (const int e = check_relpos(row_of, rows, lo, n, grid_w, Lq, Lk, q_start, nullptr)) return e;
  DeviceScope scope(device);
  if (scope.status != hipSuccess) return -static_cast<int>(scope.status);
  const RelPos pos{row_of, lo, n, grid_w};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int q0 = clamp_pos(q_start);
  float* ws = static_cast<float*>(workspace);
  switch (dtype) {
    case FA_F16: return bias_backward<_Float16>(up, up_strides, rows, H, Lq, Lk, pos, q0, dtable, ws, s);
    case FA_BF16: return bias_backward<__bf16>(up, up_strides, rows, H, Lq, Lk, pos, q0, dtable, ws, s);
    case FA_F32: return bias_backward<float>(up, up_strides, rows, H, Lq, Lk, pos, q0, dtable, ws, s);
    default: return FA_E_DTYPE;
  }
}

}  // extern "C"
