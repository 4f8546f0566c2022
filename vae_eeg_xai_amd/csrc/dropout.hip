// Inverted dropout without a stored mask:  y[r][c] = residual[r][c] + keep(r, c) * x[r][c] / (1 - rate).
// keep(r, c) comes from Philox-4x32-10 under (seed, row, column) (trunk_common.h), so the backward pass is the same call on
// dy: nothing is kept between the two.
//
// Bound: HBM (2 or 3 elements moved per element).  A thread owns blocks of 8 columns of one row -- one Philox call each, and
// 16 bytes per tensor of a 16-bit type.  16384x4096 bf16: 49 us (5.5 TB/s), with a residual 70 us (5.8 TB/s; a copy of 1 GB: 4.9).
// Stores that pass by the caches would take 4 % less, but the kernel that reads y next then waits for it: fp32 of 64 MB, a
// chain of dropouts, 20 us each as it is and 26 with them.
#include "trunk_common.h"
#include "../../include/veex.h"
#include <algorithm>

// VEC: the row length is a multiple of 8 and every tensor 16-byte aligned, so blocks are whole and load as 16-byte pieces
template <typename T, bool VEC, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y,
                                                      long long nblocks, int blocks_per_row, int cols, DropArgs d) {
  constexpr int V = 16 / sizeof(T);
  const unsigned long long base = drop_base(d);
  const long long step = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < nblocks; i += step) {
    // (most grids fit 32 bits: a 64-bit division costs about as much as the generator)
    const long long row = nblocks <= 0xFFFFFFFFll ? (long long)((unsigned)i / (unsigned)blocks_per_row) : i / blocks_per_row;
    const int block = (int)(i - row * blocks_per_row);
    const long long at = row * cols + 8 * block;
    if (VEC) {
      Piece<T, V> a[8 / V], b[8 / V];
#pragma unroll
      for (int q = 0; q < 8 / V; ++q) {
        a[q] = piece_load<T, V>(x + at + q * V);
        if (RES) b[q] = piece_load<T, V>(res + at + q * V);
      }
      unsigned w[4];
      drop_words(d, base + (unsigned long long)row, (unsigned)block, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = drop_u16(w, e) >= d.cut ? (float)a[e / V].v[e % V] * d.scale : 0.f;
        if (RES) v += (float)b[e / V].v[e % V];
        a[e / V].v[e % V] = (T)v;
      }
#pragma unroll
      for (int q = 0; q < 8 / V; ++q) piece_store<T, V>(y + at + q * V, a[q]);
    } else {
      const int n = min(8, cols - 8 * block);
      float a[8], b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a[e] = e < n ? (float)x[at + e] : 0.f;
        b[e] = RES && e < n ? (float)res[at + e] : 0.f;
      }
      unsigned w[4];
      drop_words(d, base + (unsigned long long)row, (unsigned)block, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = drop_u16(w, e) >= d.cut ? a[e] * d.scale : 0.f;
        if (e < n) y[at + e] = (T)(v + b[e]);
      }
    }
  }
}

template <typename T>
static int dropout_launch(const void* x, const void* res, void* y, long long rows, int cols, const DropArgs& d, hipStream_t st) {
  const int bpr = (cols + 7) / 8;
  const long long nblocks = rows * bpr;
  const unsigned grid = (unsigned)std::min<long long>((nblocks + 255) / 256, 1 << 16);
  const bool vec = cols % 8 == 0 && trunk_aligned16(x) && trunk_aligned16(y) && (res == nullptr || trunk_aligned16(res));
  const T* xs = static_cast<const T*>(x); const T* rs = static_cast<const T*>(res); T* ys = static_cast<T*>(y);
  if (vec && res) hipLaunchKernelGGL((dropout_kernel<T, true, true>), dim3(grid), dim3(256), 0, st, xs, rs, ys, nblocks, bpr, cols, d);
  else if (vec) hipLaunchKernelGGL((dropout_kernel<T, true, false>), dim3(grid), dim3(256), 0, st, xs, rs, ys, nblocks, bpr, cols, d);
  else if (res) hipLaunchKernelGGL((dropout_kernel<T, false, true>), dim3(grid), dim3(256), 0, st, xs, rs, ys, nblocks, bpr, cols, d);
  else hipLaunchKernelGGL((dropout_kernel<T, false, false>), dim3(grid), dim3(256), 0, st, xs, rs, ys, nblocks, bpr, cols, d);
  VEEX_CHECK_LAUNCH();
  return 0;
}

extern "C" int veex_dropout(const void* x, const void* residual, void* y, long long rows, int cols, int dtype, double rate,
                            unsigned long long seed, unsigned long long first_row, const unsigned long long* counter,
                            hipStream_t st) {
  DropArgs d;
  if (x == nullptr || y == nullptr || rows < 0 || cols < 1 || !trunk_dtype_ok(dtype)) {
    veex_set_error("dropout: x and y, rows >= 0, cols >= 1 and a dtype of VEEX_T_* are needed"); return VEEX_EINVAL;
  }
  if (cols > (1 << 30) || rows > (1ll << 46) / cols) { veex_set_error("dropout: at most 2^30 columns and 2^46 elements"); return VEEX_EINVAL; }
  if (!trunk_drop_args(rate, seed, first_row, counter, d)) {
    veex_set_error("dropout: rate %g is outside [0, 1 - 2^-17)", rate); return VEEX_EINVAL;
  }
  if (rows == 0) return 0;
  if (dtype == VEEX_T_F32) return dropout_launch<float>(x, residual, y, rows, cols, d, st);
  if (dtype == VEEX_T_BF16) return dropout_launch<bf16_t>(x, residual, y, rows, cols, d, st);
  return dropout_launch<f16_t>(x, residual, y, rows, cols, d, st);
}
