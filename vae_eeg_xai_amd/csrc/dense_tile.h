// Interface of dense_tile.hip: large products on the 16-bit matrix cores, and the packing their operands may need.
#ifndef VEEX_DENSE_TILE_H
#define VEEX_DENSE_TILE_H
#include "dense_common.h"

// a 16-bit operand: row-major, 16-byte aligned rows of ld_bytes; planes (the three terms of an fp32 tensor) plane_bytes apart
struct DtTensor { const void* p; long long ld_bytes, plane_bytes; };

struct DtGemm {
  DtTensor a, b;
  long long I;
  int J;
  long long K, k_per_split;
  unsigned splits, tiles_i, tiles_j;
  DenseEpi epi;
  float* slab;           // null: the epilogue runs here
  int vec_e;             // the epilogue's tensors move in 16-byte pieces
  float alpha;           // a gradient: grad_scale
};

// akc / bkc: that operand's k index is its contiguous one.  tile: 0 256x256 (16-bit types), 1 256x128, 2 128x128
int dense_tile_launch(int dtype, bool akc, bool bkc, int tile, const DtGemm& g, hipStream_t st);
// dx and dw together, both in tiles of 128x128
int dense_tile_grads_launch(int dtype, const DtGemm& dx, const DtGemm& dw, hipStream_t st);
// up to three packings in one launch
struct DtPack { const void* src; void* dst; long long ld, rows, plane_bytes; int cols; };
int dense_pack_launch(int dtype, const DtPack* jobs, int n, hipStream_t st);

// Eight fp32 values as their three bf16 terms: f = t1 + t2 + t3 to 2^-27 (each term rounds what the ones before left; the
// differences are exact).  A value that is not finite is its first term alone; one that would round to an infinity takes the largest bf16
// first.  Terms below 2^-126 may be lost: values under about 2^-110 keep fewer bits.
__device__ __forceinline__ void dt_store_planes(char* dst, long long plane_bytes, const float (&f)[8]) {
  Piece<bf16_t, 8> t[3];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool fin = __builtin_isfinite(f[e]);
    const bf16_t a = (bf16_t)(fin ? fminf(fmaxf(f[e], -0x1.FEp127f), 0x1.FEp127f) : f[e]);
    const float r1 = fin ? f[e] - (float)a : 0.f;
    const bf16_t b = (bf16_t)r1;
    const float r2 = r1 - (float)b;
    t[0].v[e] = a; t[1].v[e] = b; t[2].v[e] = (bf16_t)r2;
  }
#pragma unroll
  for (int pl = 0; pl < 3; ++pl) piece_store<bf16_t, 8>(reinterpret_cast<bf16_t*>(dst + pl * plane_bytes), t[pl]);
}

#endif
