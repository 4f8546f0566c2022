// Shared by the Dense kernels (dense.hip, dense_tile.hip): the epilogue  y = residual + D(act(acc + bias)), its derivative,
// and the parameters of one matrix product  C[i][j] = sum_k A(i, k) B(k, j).
#ifndef VEEX_DENSE_COMMON_H
#define VEEX_DENSE_COMMON_H
#include "trunk_common.h"
#include "../../include/veex.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));

struct DenseEpi {
  const void* bias;      // [J], optional
  const void* res;       // [I][J], optional
  void* y;               // [I][J]
  void* pre;             // [I][J], optional: acc + bias in the tensors' type
  int act;
  DropArgs drop;         // cut 0: none
};

// A relu unit passes a NaN on (a comparison with it is false), as the formula's where(z < 0, 0, z) does.
__device__ __forceinline__ float dense_act(float z, int act) {
  switch (act) {
    case VEEX_ACT_RELU: return z < 0.f ? 0.f : z;
    case VEEX_ACT_GELU: return z * (0.5f * (1.f + erff(z * 0.70710678118654752f)));
    case VEEX_ACT_SILU: return z * (1.f / (1.f + expf(-z)));
    case VEEX_ACT_SIGMOID: return 1.f / (1.f + expf(-z));
    default: return z;
  }
}
// d act / dz; for relu, s may be z or the kept output (both are <= 0 exactly where nothing passes)
__device__ __forceinline__ float dense_act_grad(float s, int act) {
  switch (act) {
    case VEEX_ACT_RELU: return s <= 0.f ? 0.f : 1.f;
    case VEEX_ACT_GELU: return 0.5f * (1.f + erff(s * 0.70710678118654752f)) + s * expf(-0.5f * s * s) * 0.39894228040143268f;
    case VEEX_ACT_SILU: { const float e = 1.f / (1.f + expf(-s)); return e * (1.f + s * (1.f - e)); }
    case VEEX_ACT_SIGMOID: { const float e = 1.f / (1.f + expf(-s)); return e * (1.f - e); }
    default: return 1.f;
  }
}

// Columns j .. j + W - 1 (W = 4 or 8, j a multiple of W) of row i.  half words: u16 of column j + e is words[(e0 + e) >> 1]'s
// half (e & 1), where e0 = j & 7 (the caller passes the Philox words of the block of 8 that holds them).
template <typename T, int W>
__device__ __forceinline__ void dense_epilogue(const DenseEpi& ep, float (&v)[W], long long i, int j, int J, bool vec,
                                               const unsigned* words) {
  const T* bias = static_cast<const T*>(ep.bias);
  const T* res = static_cast<const T*>(ep.res);
  T* y = static_cast<T*>(ep.y);
  T* pre = static_cast<T*>(ep.pre);
  const long long at = i * J + j;
  constexpr int V = W * (int)sizeof(T) <= 16 ? W : 16 / (int)sizeof(T);
  const int n = min(W, J - j);
  if (n <= 0) return;
  float r[W];
#pragma unroll
  for (int e = 0; e < W; ++e) r[e] = 0.f;
  if (vec) {
    if (bias != nullptr)
#pragma unroll
      for (int q = 0; q < W / V; ++q) {
        const Piece<T, V> b = piece_load<T, V>(bias + j + q * V);
#pragma unroll
        for (int e = 0; e < V; ++e) v[q * V + e] += (float)b.v[e];
      }
    if (res != nullptr)
#pragma unroll
      for (int q = 0; q < W / V; ++q) {
        const Piece<T, V> b = piece_load<T, V>(res + at + q * V);
#pragma unroll
        for (int e = 0; e < V; ++e) r[q * V + e] = (float)b.v[e];
      }
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (e < n) {
        if (bias != nullptr) v[e] += (float)bias[j + e];
        if (res != nullptr) r[e] = (float)res[at + e];
      }
  }
  float o[W];
#pragma unroll
  for (int e = 0; e < W; ++e) {
    o[e] = dense_act(v[e], ep.act);
    if (ep.drop.cut != 0u) {
      const unsigned u = (e & 1) ? words[e >> 1] >> 16 : words[e >> 1] & 0xFFFFu;
      o[e] = u >= ep.drop.cut ? o[e] * ep.drop.scale : 0.f;
    }
    o[e] += r[e];
  }
  auto put = [&](T* dst, const float (&s)[W]) {
    if (vec) {
#pragma unroll
      for (int q = 0; q < W / V; ++q) {
        Piece<T, V> p;
#pragma unroll
        for (int e = 0; e < V; ++e) p.v[e] = (T)s[q * V + e];
        piece_store<T, V>(dst + at + q * V, p);
      }
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (e < n) dst[at + e] = (T)s[e];
    }
  };
  if (pre != nullptr) put(pre, v);
  put(y, o);
}

// every tensor of the epilogue can be moved in pieces of W elements
inline bool dense_epi_vec(const DenseEpi& ep, int J, int W, int elem) {
  if (J % W != 0) return false;
  const uintptr_t mask = (uintptr_t)(W * elem < 16 ? W * elem : 16) - 1;
  for (const void* q : {ep.bias, ep.res, (const void*)ep.y, (const void*)ep.pre})
    if (reinterpret_cast<uintptr_t>(q) & mask) return false;
  return true;
}

// One operand: element (row, k) at p + row * row_stride + k * k_stride; exactly one of the strides is 1.
struct DenseOperand { const void* p; long long row_stride, k_stride; };

struct DenseGemm {
  DenseOperand a, b;     // rows i and j
  long long I;
  int J;
  long long K;
  DenseEpi epi;
  float* slab;           // [splits][I][J] when splits > 1
  int splits;
  long long k_per_split;
  int vec_a, vec_b, vec_e;
};

#endif
