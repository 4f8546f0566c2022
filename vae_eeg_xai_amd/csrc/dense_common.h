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

// The activations, W values at a time with the choice outside the loops: a small kernel's time is largely the fetch of its code, and
// an activation's code chosen per value, times the unrolled values, was most of it (512x28x4096 fp32: 22 us so, 8 us now).
//
// A 16-bit result keeps 11 bits at most, so there the hardware's exp2 and reciprocal (1 ulp) serve; fp32 takes the accurate expf
// and division.  gelu needs Phi(z) = erfc(-z / sqrt 2) / 2: with x = |z| / sqrt 2 and t = 1 / (1 + p x), erfc(x) = P(t) t exp(-x^2), P
// fitted here to exp(x^2) erfc(x) / t on 0 <= x <= 9.5 for the least largest relative error (7.3e-7 with 7 coefficients, 1.7e-8
// with 9).  In fp32 all of Phi(z) is off by up to 6e-7 for z > -4, and further down by what the rounding of z^2 does to exp(-z^2 / 2): 1.3e-6 to
// -8, 4e-6 at -12 (against Phi 1e-15 and 1e-33).  The derivative's exp(-z^2 / 2) is the same exponential.
template <typename T> __device__ __forceinline__ float act_exp(float x) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(x * 1.44269504f);
  else return expf(x);
}
template <typename T> __device__ __forceinline__ float act_rcp(float x) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(x);
  else return 1.f / x;
}
// Phi(z), and e = exp(-z^2 / 2); 16-bit types with every constant folded (8192x1024x4096 bf16: gelu was 16 us of 94)
template <typename T> __device__ __forceinline__ float act_phi(float z, float& e) {
  float q;
  if constexpr (sizeof(T) == 2) {
    const float t = act_rcp<T>(fmaf(0.261629509f, fabsf(z), 1.f));      // 0.37 / sqrt 2
    q = -0.0712758525f;                                                 // P / 2
    q = fmaf(q, t, 0.217830181f); q = fmaf(q, t, -0.093216069f); q = fmaf(q, t, 0.15870288f);
    q = fmaf(q, t, 0.0763279275f); q = fmaf(q, t, 0.107441359f); q = fmaf(q, t, 0.10418994f);
    e = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
    q *= t * e;
  } else {
    const float x = fabsf(z) * 0.70710678f, t = act_rcp<T>(fmaf(0.37f, x, 1.f));
    q = 0.0619231425f;
    q = fmaf(q, t, -0.303273201f); q = fmaf(q, t, 0.486842126f); q = fmaf(q, t, -0.285312116f); q = fmaf(q, t, 0.310802102f);
    q = fmaf(q, t, 0.106520303f); q = fmaf(q, t, 0.206254035f); q = fmaf(q, t, 0.207429841f); q = fmaf(q, t, 0.208813742f);
    e = act_exp<T>(-0.5f * z * z);
    q *= 0.5f * t * e;
  }
  return z > 0.f ? 1.f - q : q;
}

// A relu unit passes a NaN on (a comparison with it is false), as the formula's where(z < 0, 0, z) does.
template <typename T, int W>
__device__ __forceinline__ void dense_act(float (&v)[W], int act) {
  switch (act) {
    case VEEX_ACT_RELU:
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
      break;
    case VEEX_ACT_GELU:
#pragma unroll
      for (int e = 0; e < W; ++e) { float x; v[e] *= act_phi<T>(v[e], x); }
      break;
    case VEEX_ACT_SILU:
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] *= act_rcp<T>(1.f + act_exp<T>(-v[e]));
      break;
    case VEEX_ACT_SIGMOID:
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = act_rcp<T>(1.f + act_exp<T>(-v[e]));
      break;
    default: break;
  }
}
// d[e] *= d act / dz at s[e]; for relu, s may be z or the kept output (both are <= 0 exactly where nothing passes)
template <typename T, int W>
__device__ __forceinline__ void dense_act_grad(float (&d)[W], const float (&s)[W], int act) {
  switch (act) {
    case VEEX_ACT_RELU:
#pragma unroll
      for (int e = 0; e < W; ++e) d[e] = s[e] <= 0.f ? 0.f : d[e];
      break;
    case VEEX_ACT_GELU:
#pragma unroll
      for (int e = 0; e < W; ++e) { float x; const float phi = act_phi<T>(s[e], x); d[e] *= fmaf(s[e] * 0.39894228f, x, phi); }
      break;
    case VEEX_ACT_SILU:
#pragma unroll
      for (int e = 0; e < W; ++e) { const float x = act_rcp<T>(1.f + act_exp<T>(-s[e])); d[e] *= x * fmaf(s[e], 1.f - x, 1.f); }
      break;
    case VEEX_ACT_SIGMOID:
#pragma unroll
      for (int e = 0; e < W; ++e) { const float x = act_rcp<T>(1.f + act_exp<T>(-s[e])); d[e] *= x * (1.f - x); }
      break;
    default: break;
  }
}

// Eight elements at p (n of them inside the row), as they lie; vec: as 16-byte pieces (a row then ends with a piece: of fp32, which has
// two, the second may be missing and reads as zeros).  Kept apart from their conversion, so that
// several loads are on their way before the first is waited for.
template <typename T> struct Raw8 { T v[8]; };
template <typename T>
__device__ __forceinline__ void load_raw(Raw8<T>& r, const T* p, int n, bool vec) {
  constexpr int V = 16 / (int)sizeof(T);
  if (vec) {
#pragma unroll
    for (int q = 0; q < 8 / V; ++q) {
      const bool in = q * V < n;
      const Piece<T, V> b = piece_load<T, V>(in ? p + q * V : p);
#pragma unroll
      for (int e = 0; e < V; ++e) r.v[q * V + e] = in ? b.v[e] : (T)0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = p[e < n ? e : 0];
  }
}
template <typename T>
__device__ __forceinline__ void load8(float (&r)[8], const T* p, int n, bool vec) {
  Raw8<T> x;
  load_raw<T>(x, p, n, vec);
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = (float)x.v[e];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&s)[8], int n, bool vec) {
  constexpr int V = 16 / (int)sizeof(T);
  if (vec) {
#pragma unroll
    for (int q = 0; q < 8 / V; ++q) {
      Piece<T, V> b;
#pragma unroll
      for (int e = 0; e < V; ++e) b.v[e] = (T)s[q * V + e];
      if (q * V < n) piece_store<T, V>(p + q * V, b);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = (T)s[e];
  }
}

// A gradient on its way out: times alpha, which undoes the factor that fp16's dz was stored with (dense.hip; 1 for the other types)
template <typename T>
__device__ __forceinline__ void grad_scale(float (&v)[8], float alpha) {
  if constexpr (TrunkType<T>::code == VEEX_T_F16) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= alpha;
  }
}

// Columns j .. j + 7 (j a multiple of 8, n of them inside the row) of row i, `at` = i * J + j: v = acc, b = the bias there (zeros
// without one), words = the row's dropout words of that block.  A thread that walks down rows loads b once.
template <typename T>
__device__ __forceinline__ void dense_bias(const DenseEpi& ep, float (&b)[8], int j, int J, bool vec) {
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = 0.f;
  if (ep.bias != nullptr && j < J) load8<T>(b, static_cast<const T*>(ep.bias) + j, J - j, vec);
}
template <typename T>
__device__ __forceinline__ void dense_epilogue(const DenseEpi& ep, float (&v)[8], const float (&b)[8], long long at, int n, bool vec,
                                               const unsigned* words) {
  float r[8];
  if (ep.res != nullptr) load8<T>(r, static_cast<const T*>(ep.res) + at, n, vec);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += b[e];
  if (ep.pre != nullptr) {
    // z for the backward pass, rounded to the tensors' type like the activation that a user would keep.  A finite z that a 16-bit type
    // does not hold (fp16 ends at 65504, bf16 half a step below fp32) stays finite: the derivative there is its limit, and at an
    // infinity it would be NaN.  (One look at the largest of eight: each tested by itself, the forward pass of 8192x1024x4096 bf16 was 5 us longer.)
    float z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = v[e];
    if constexpr (sizeof(T) == 2) {
      constexpr float END = TrunkType<T>::code == VEEX_T_F16 ? 65504.f : 0x1.FEp127f;
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
      if (top > END)
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = __builtin_isfinite(v[e]) ? fminf(fmaxf(v[e], -END), END) : v[e];
    }
    store8<T>(static_cast<T*>(ep.pre) + at, z, n, vec);
  }
  dense_act<T, 8>(v, ep.act);
  if (ep.drop.cut != 0u)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = drop_u16(words, e) >= ep.drop.cut ? v[e] * ep.drop.scale : 0.f;
  if (ep.res != nullptr)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += r[e];
  store8<T>(static_cast<T*>(ep.y) + at, v, n, vec);
}

// every tensor of the epilogue can be moved in 16-byte pieces
inline bool dense_epi_vec(const DenseEpi& ep, int J, int elem) {
  if ((long long)J * elem % 16 != 0) return false;
  for (const void* q : {ep.bias, ep.res, (const void*)ep.y, (const void*)ep.pre})
    if (!trunk_aligned16(q)) return false;
  return true;
}

// floats between the rows of a split product's slab: rows of whole 16-byte pieces (what is behind column J is never used)
__host__ __device__ inline long long slab_ld(int J) { return (J + 3LL) / 4 * 4; }

// One operand: element (row, k) at p + row * row_stride + k * k_stride; exactly one of the strides is 1.
struct DenseOperand { const void* p; long long row_stride, k_stride; };

struct DenseGemm {
  DenseOperand a, b;     // rows i and j
  long long I;
  int J;
  long long K;
  DenseEpi epi;
  float* slab;           // [splits][I][slab_ld(J)] when splits > 1
  int splits;
  long long k_per_split;
  int vec_e;             // the epilogue's tensors move in 16-byte pieces
  float alpha;           // a gradient: grad_scale
};

#endif
