// The Dense layer of a trunk:  y = residual + D(act(x w + b))  and its gradients  dz = D'(dy) act'(z), dx = dz w^T,
// dw = x^T dz, db = column sums of dz.  x [M][K], w [K][N] (Keras layout), types fp32 / bf16 / fp16, sums in fp32.
//
// This file: the general product (any strides, alignment and size), the join of a split reduction, the dz / db pass, and
// the host side, which sends large products to the 16-bit matrix cores (dense_tile.hip).
#include "dense_tile.h"
#include <algorithm>

// ---------------------------------------------------------------------------------------------------------------
// The general product: 64 x 64 tiles, 4 waves of one 32 x 32 accumulator, fp32 MFMA (a product of two 16-bit numbers is exact
// there, so one kernel serves every type).  Operand tiles are staged through registers into [k][row] LDS; a tensor whose rows
// are whole aligned pieces loads 8 elements at a time, others element by element.  The MFMA takes B's rows as its first operand, so
// that a lane ends up with 4 consecutive columns of one row.
// Bound: the fp32 MFMA in long reductions (128x4096x4096 fp32 83 TFLOP/s, 64x4096x14336 76; a large library product 153), and in
// small layers the way in and out of a tile: 512x28x4096 fp32 6.6 us, 512x6400x100 16 us and 5 for the join of its 32 splits.
// ---------------------------------------------------------------------------------------------------------------
#define DG_LD 68     // floats per LDS row: 64 + one 16-byte piece

// One operand's 64 x 32 tiles, 8 elements a thread.  Whole pieces: 8 neighbours of the contiguous index (k: 4 threads a row, else 8
// threads a k).  Otherwise single elements with neighbouring threads on neighbouring addresses (32 threads along k, 8 rows apart,
// or 64 threads along the rows, 4 k's apart): eight at once from each thread's own place would touch eight times the lines.
template <typename T, bool KC, bool vec>
struct DgOperand {
  const T *at, *safe;           // this thread's first element of the next tile; what a thread outside the tensor reads
  long long rs, ks, rows_left, k_left;      // strides; rows and k's from this thread's first element on
  __device__ __forceinline__ void init(const DenseOperand& o, long long row0, long long rows, long long k0, long long k_end) {
    const int t = threadIdx.x;
    rs = o.row_stride; ks = o.k_stride;
    const int r = vec ? (KC ? t >> 2 : 8 * (t & 7)) : (KC ? t >> 5 : t & 63);
    const int k = vec ? (KC ? 8 * (t & 3) : t >> 3) : (KC ? t & 31 : t >> 6);
    rows_left = rows - row0 - r; k_left = k_end - k0 - k;
    safe = static_cast<const T*>(o.p);
    at = safe + (row0 + r) * rs + (k0 + k) * ks;
  }
  __device__ __forceinline__ void load(float (&r)[8]) {
    if (vec) {
      constexpr int V = 16 / sizeof(T);
#pragma unroll
      for (int c = 0; c < 8 / V; ++c) {
        const bool in = (KC ? rows_left > 0 && k_left > c * V : rows_left > c * V && k_left > 0);
        const Piece<T, V> x = piece_load<T, V>(in ? at + c * V : safe);
#pragma unroll
        for (int e = 0; e < V; ++e) r[c * V + e] = in ? (float)x.v[e] : 0.f;
      }
    } else {
      T x[8];
      bool in[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        in[e] = KC ? rows_left > 8 * e && k_left > 0 : rows_left > 0 && k_left > 4 * e;
        x[e] = *(in[e] ? at + e * (KC ? 8 * rs : 4 * ks) : safe);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = in[e] ? (float)x[e] : 0.f;
    }
    at += 32 * ks; k_left -= 32;
  }
  __device__ __forceinline__ void store(float* s, const float (&r)[8]) const {
    const int t = threadIdx.x;
    if (!vec) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[KC ? (t & 31) * DG_LD + (t >> 5) + 8 * e : ((t >> 6) + 4 * e) * DG_LD + (t & 63)] = r[e];
    } else if (KC) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[(8 * (t & 3) + e) * DG_LD + (t >> 2)] = r[e];
    } else {
      float4* d = reinterpret_cast<float4*>(s + (t >> 3) * DG_LD + 8 * (t & 7));
      d[0] = make_float4(r[0], r[1], r[2], r[3]);
      d[1] = make_float4(r[4], r[5], r[6], r[7]);
    }
  }
};

struct DgLds { float a[2][32 * DG_LD], b[2][32 * DG_LD]; };

// One tile of one split: part of C.  GRAD: a gradient, which has no epilogue.
template <typename T, bool AKC, bool BKC, bool GRAD, bool VEC>
__device__ __forceinline__ void dg_tile(const DenseGemm& g, unsigned tile, unsigned split, DgLds& lds) {
  float (&As)[2][32 * DG_LD] = lds.a;
  float (&Bs)[2][32 * DG_LD] = lds.b;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l31 = lane & 31, lh = lane >> 5, wi = wave & 1, wj = wave >> 1;
  const int tiles_j = (g.J + 63) / 64;
  const unsigned ti = tile / (unsigned)tiles_j;
  const long long i0 = ti * 64ll;
  const int j0 = (int)(tile - ti * tiles_j) * 64;
  const long long k_begin = (long long)split * g.k_per_split, k_end = min(g.K, k_begin + g.k_per_split);

  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  // Tiles two turns ahead are on their way in the forward product (64x4096x14336 fp32: one ahead 104 us, two 94; the gradients' shorter
  // reductions lose by it, 512x6400x100 27 us, 29).
  constexpr int AHEAD = GRAD ? 1 : 2;
  float ra[AHEAD][8], rb[AHEAD][8];
  DgOperand<T, AKC, VEC> a;
  DgOperand<T, BKC, VEC> b;
  a.init(g.a, i0, g.I, k_begin, k_end);
  b.init(g.b, j0, g.J, k_begin, k_end);
  const int turns = (int)((k_end - k_begin + 31) / 32);
#pragma unroll
  for (int q = 0; q < AHEAD; ++q)
    if (q < turns) { a.load(ra[q]); b.load(rb[q]); }
  auto turn = [&](int t, int cur, int q) {
    a.store(As[cur], ra[q]);
    b.store(Bs[cur], rb[q]);
    __syncthreads();      // (the other buffer's readers passed the barrier of the turn before)
    if (t + AHEAD < turns) { a.load(ra[q]); b.load(rb[q]); }
#pragma unroll
    for (int s = 0; s < 16; ++s)
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(Bs[cur][(2 * s + lh) * DG_LD + wj * 32 + l31],
                                                 As[cur][(2 * s + lh) * DG_LD + wi * 32 + l31], acc, 0, 0, 0);
  };
  if (AHEAD == 1) {
    for (int t = 0; t < turns; ++t) turn(t, t & 1, 0);
  } else {
    for (int t = 0; t < turns; t += 2) {
      turn(t, 0, 0);
      if (t + 1 < turns) turn(t + 1, 1, AHEAD - 1);
    }
  }
  // The way out, as in dense_tile.hip: each wave turns its 32 x 32 block round in LDS, so that a lane holds 8 columns of a row
  __syncthreads();
  float* strip = (wave < 2 ? As[wave] : Bs[wave - 2]);         // 32 rows of 36 floats
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<float4*>(strip + l31 * 36 + 8 * q + 4 * lh) = make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
  __syncthreads();
  const unsigned long long base = GRAD ? 0ull : drop_base(g.epi.drop);
  const int j = j0 + wj * 32 + 8 * (lane & 3);
  float bias[8];
  if (!GRAD && g.splits == 1) dense_bias<T>(g.epi, bias, j, g.J, g.vec_e);
#pragma unroll 1
  for (int r = lane >> 2; r < 32; r += 16) {
    const long long i = i0 + wi * 32 + r;
    if (i >= g.I || j >= g.J) continue;
    const float4 lo = *reinterpret_cast<const float4*>(strip + r * 36 + 8 * (lane & 3)), hi = *reinterpret_cast<const float4*>(strip + r * 36 + 8 * (lane & 3) + 4);
    float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (g.splits > 1) {
      float* s = g.slab + ((long long)split * g.I + i) * slab_ld(g.J) + j;
      *reinterpret_cast<float4*>(s) = lo;
      if (j + 4 < g.J) *reinterpret_cast<float4*>(s + 4) = hi;
    } else if (GRAD) {
      grad_scale<T>(v, g.alpha);
      store8<T>(static_cast<T*>(g.epi.y) + i * g.J + j, v, g.J - j, g.vec_e);
    } else {
      unsigned w[4] = {0u, 0u, 0u, 0u};
      if (g.epi.drop.cut != 0u) drop_words(g.epi.drop, base + (unsigned long long)i, (unsigned)j >> 3, w);
      dense_epilogue<T>(g.epi, v, bias, i * g.J + j, g.J - j, g.vec_e, w);
    }
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dense_general_kernel(DenseGemm g) {
  __shared__ DgLds lds;
  dg_tile<T, true, false, false, VEC>(g, blockIdx.x, blockIdx.y, lds);
}

// Both gradients in one launch (either may have no blocks): a small layer's products leave most of the chip idle one after the other,
// and a launch costs the host as much as such a product costs the GPU.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dense_general_grads_kernel(DenseGemm dx, DenseGemm dw, unsigned dx_tiles, unsigned dw_tiles, unsigned dx_from, unsigned dw_from) {
  __shared__ DgLds lds;
  const unsigned b = blockIdx.x;
  if (dx_from < dw_from ? b < dw_from : b >= dx_from) dg_tile<T, true, true, true, VEC>(dx, (b - dx_from) % dx_tiles, (b - dx_from) / dx_tiles, lds);
  else dg_tile<T, false, false, true, VEC>(dw, (b - dw_from) % dw_tiles, (b - dw_from) / dw_tiles, lds);
}

// Sum of the slabs [splits][I][slab_ld(J)], 8 columns of one row a thread.  Where the output alone is too small to fill the chip, SL
// threads share an output block, each adding every SL'th slab up; the SL sums are added in a fixed order.  out(v, i, j) gets the sums.
template <int SL, typename OUT>
__device__ __forceinline__ void dense_sum_slabs(const float* slab, long long I, int J, int splits, unsigned block, unsigned blocks, float* part, OUT out) {
  constexpr int OB = 256 / SL;                    // output blocks of a workgroup; a wave holds all of them (SL > 1), 64 / OB times
  static_assert(SL == 1 || OB <= 64, "");
  const int bpr = (J + 7) / 8;
  const long long nb = I * bpr, stride = I * slab_ld(J);
  const int ob = threadIdx.x % OB, sl = threadIdx.x / OB;
  for (long long b0 = (long long)block * OB; b0 < nb; b0 += (long long)blocks * OB) {
    const long long b = min(b0 + ob, nb - 1);     // (every thread meets the barriers)
    const long long i = nb <= 0xFFFFFFFFll ? (long long)((unsigned)b / (unsigned)bpr) : b / bpr;
    const int j = 8 * (int)(b - i * bpr);
    const float* s = slab + i * slab_ld(J) + j;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    const int second = j + 4 < J ? 4 : 0;
#pragma unroll 8
    for (int z = sl; z < splits; z += SL) {
      const float4 x = *reinterpret_cast<const float4*>(s + z * stride);
      const float4 t = *reinterpret_cast<const float4*>(s + z * stride + second);
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
      v[4] += t.x; v[5] += t.y; v[6] += t.z; v[7] += t.w;
    }
    if (SL > 1) {
#pragma unroll
      for (int o = OB; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += __shfl_xor(v[e], o);
      __syncthreads();
      if ((threadIdx.x & 63) < OB)
#pragma unroll
        for (int e = 0; e < 8; ++e) part[((threadIdx.x >> 6) * OB + ob) * 9 + e] = v[e];
      __syncthreads();
      if (sl == 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = part[ob * 9 + e] + part[(OB + ob) * 9 + e] + (part[(2 * OB + ob) * 9 + e] + part[(3 * OB + ob) * 9 + e]);
    }
    if (sl == 0 && b0 + ob < nb) out(v, i, j);
  }
}
#define DJ_PART (4 * 32 * 9)     // floats of `part` at SL = 8 (SL = 32 needs fewer)

// threads an output block: shared while there are fewer than two workgroups a CU (100 slabs of 100 columns: 34 us with 1, 5 with 32)
static int join_lanes(long long I, int J, int splits) {
  const long long nb = I * ((J + 7) / 8);
  return nb >= 512 * 256 || splits < 8 ? 1 : nb >= 512 * 32 || splits < 32 ? 8 : 32;
}
static unsigned join_blocks(long long I, int J, int lanes) {
  return (unsigned)std::min<long long>((I * ((J + 7) / 8) + 256 / lanes - 1) / (256 / lanes), 1 << 16);
}

// the forward product's join, with the epilogue
template <typename T, int SL>
__global__ __launch_bounds__(256) void dense_join_kernel(DenseGemm g) {
  __shared__ float part[SL > 1 ? DJ_PART : 1];
  dense_sum_slabs<SL>(g.slab, g.I, g.J, g.splits, blockIdx.x, gridDim.x, part, [&](float (&v)[8], long long i, int j) {
    unsigned w[4] = {0u, 0u, 0u, 0u};
    if (g.epi.drop.cut != 0u) drop_words(g.epi.drop, drop_base(g.epi.drop) + (unsigned long long)i, (unsigned)j >> 3, w);
    float bias[8];
    dense_bias<T>(g.epi, bias, j, g.J, g.vec_e);
    dense_epilogue<T>(g.epi, v, bias, i * g.J + j, g.J - j, g.vec_e, w);
  });
}

// What a backward pass has left to add up, in one launch: the slabs of dx and of dw, and db's partial rows (32 columns and 8 row lanes a
// block).  Jobs without blocks are skipped.
struct DenseFinish {
  struct Sum { const float* slab; void* out; long long I; int J, splits, lanes, vec; } sum[2];
  float alpha;
  const float* part; void* db; int chunks, n;
  unsigned first[4];             // a job's first block; the end
};

template <typename T>
__global__ __launch_bounds__(256) void dense_finish_kernel(DenseFinish f) {
  __shared__ float part[DJ_PART];
  const unsigned b = blockIdx.x;
  if (b < f.first[2]) {
    const int q = b < f.first[1] ? 0 : 1;
    const DenseFinish::Sum& s = f.sum[q];
    const unsigned block = b - f.first[q], blocks = f.first[q + 1] - f.first[q];
    auto out = [&](float (&v)[8], long long i, int j) { grad_scale<T>(v, f.alpha); store8<T>(static_cast<T*>(s.out) + i * s.J + j, v, s.J - j, s.vec); };
    if (s.lanes == 1) dense_sum_slabs<1>(s.slab, s.I, s.J, s.splits, block, blocks, part, out);
    else if (s.lanes == 8) dense_sum_slabs<8>(s.slab, s.I, s.J, s.splits, block, blocks, part, out);
    else dense_sum_slabs<32>(s.slab, s.I, s.J, s.splits, block, blocks, part, out);
    return;
  }
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, col = (b - f.first[2]) * 32 + tx;
  const float* p = f.part + min(col, f.n - 1);
  float a = 0.f;
#pragma unroll 8
  for (int c = ty; c < f.chunks; c += 8) a += p[(long long)c * f.n];
  part[ty * 33 + tx] = a;
  __syncthreads();
  if (ty == 0 && col < f.n) {
    a = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) a += part[q * 33 + tx];
    static_cast<T*>(f.db)[col] = (T)a;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Few rows (up to 8): the weights are read once and everything else is small, so the bound is their bandwidth (one row, bf16,
// weights from memory: 4096x14336 28 us, 4.2 TB/s; 4096x4096 13 us, from the cache behind the L2 10).  A thread owns V
// columns (16 bytes of a 16-byte aligned row of w, else one) and every KL'th k of the block's range, 8 loads in flight; KL threads a
// column meet in LDS.  Blocks split k until there are some thousand of them.  w [K][N] as it lies; x through LDS, as fp32.
// ---------------------------------------------------------------------------------------------------------------
#define DF_KB 256        // k's of x in LDS at a time
template <typename T, int R, bool VEC>
__global__ __launch_bounds__(256) void dense_few_rows_kernel(DenseGemm g) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  constexpr int CL = VEC ? 16 : 64, KL = 256 / CL;          // column threads, k threads: 256 bytes of a row, or 64 elements
  __shared__ float xs[R][DF_KB];
  __shared__ float part[KL][CL * V + 1];
  const int cl = threadIdx.x % CL, kl = threadIdx.x / CL;
  const int j = blockIdx.x * CL * V + cl * V;
  const bool ok = j < g.J;                                   // (VEC: J is a multiple of V)
  const T* x = static_cast<const T*>(g.a.p);
  const T* w = static_cast<const T*>(g.b.p) + (ok ? j : 0);
  const long long k_begin = blockIdx.y * g.k_per_split, k_end = min(g.K, k_begin + g.k_per_split);
  float acc[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < V; ++e) acc[r][e] = 0.f;
  for (long long k0 = k_begin; k0 < k_end; k0 += DF_KB) {
    const int n = (int)min((long long)DF_KB, k_end - k0);
    __syncthreads();
    for (int t = threadIdx.x; t < R * DF_KB; t += 256) {
      const int r = t / DF_KB, k = t % DF_KB;
      xs[r][k] = r < g.I && k < n ? (float)x[r * g.a.row_stride + k0 + k] : 0.f;
    }
    __syncthreads();
#pragma unroll 8
    for (int k = kl; k < n; k += KL) {
      const Piece<T, V> p = piece_load<T, V>(w + (k0 + k) * g.b.k_stride);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float a = xs[r][k];
#pragma unroll
        for (int e = 0; e < V; ++e) acc[r][e] = fmaf(a, (float)p.v[e], acc[r][e]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) part[kl][cl * V + e] = acc[r][e];
    __syncthreads();
    const int c = threadIdx.x;
    if (r < g.I && c < CL * V && blockIdx.x * CL * V + c < g.J) {
      float a = 0.f;
#pragma unroll
      for (int q = 0; q < KL; ++q) a += part[q][c];
      g.slab[((long long)blockIdx.y * g.I + r) * slab_ld(g.J) + blockIdx.x * CL * V + c] = a;
    }
  }
}

// The same for short columns (k up to 1024) of aligned weights: a block of 1024 threads owns 128 bytes of a row over all of k, each thread
// every 128th k, all its loads in flight at once; the threads of a column meet through lane rotations and LDS, and the epilogue runs
// here.  No second launch: one row of 1024x1024 bf16 6.0 us for 7.9, 100x6400 fp32 4.5 for 8.1; with longer columns the strips
// are too few (4096x1024 bf16 15 us, split 8.5).
#define DF_SHORT_K 1024
// sum over a wave's lanes of the same lane % 8
__device__ __forceinline__ float df_lanes_sum(float x) {
  x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x128, 0xF, 0xF, true));      // row_ror:8, of 16 lanes
  const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(h[0]) + __uint_as_float(h[1]);
  const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(w[0]) + __uint_as_float(w[1]);
}
template <typename T, int R>
__global__ __launch_bounds__(1024) void dense_few_short_kernel(DenseGemm g, unsigned strips) {
  constexpr int V = 16 / (int)sizeof(T), CL = 8, W = CL * V, KL = 1024 / CL, U = DF_SHORT_K / KL;
  __shared__ float xs[R][DF_SHORT_K];
  __shared__ float part[16][R][W + 4];
  const int cl = threadIdx.x % CL, kl = threadIdx.x / CL, K = (int)g.K;
  // (blocks go round the 8 XCDs in turn: neighbouring strips, which share lines where rows are not whole ones, to one of them)
  const unsigned per = strips / 8, extra = strips % 8, xcd = blockIdx.x % 8;
  const int j0 = (int)(xcd * per + min(xcd, extra) + blockIdx.x / 8) * W, j = j0 + cl * V;
  const T* x = static_cast<const T*>(g.a.p);
  const T* w = static_cast<const T*>(g.b.p) + (j < g.J ? j : 0);        // (J is a multiple of V)
  Piece<T, V> p[U];
#pragma unroll
  for (int u = 0; u < U; ++u) p[u] = piece_load<T, V>(w + min(kl + u * KL, K - 1) * g.b.k_stride);
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (threadIdx.x < K) xs[r][threadIdx.x] = r < g.I ? (float)x[r * g.a.row_stride + threadIdx.x] : 0.f;
  __syncthreads();
  float acc[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < V; ++e) acc[r][e] = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (kl + u * KL < K)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float a = xs[r][kl + u * KL];
#pragma unroll
        for (int e = 0; e < V; ++e) acc[r][e] = fmaf(a, (float)p[u].v[e], acc[r][e]);
      }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = df_lanes_sum(acc[r][e]);
      if (lane < CL) part[wave][r][lane * V + e] = a;
    }
  __syncthreads();
  const int t = threadIdx.x;
  if (t < R * W) {
    float a = 0.f;
#pragma unroll
    for (int q = 0; q < 16; ++q) a += part[q][t / W][t % W];
    part[0][t / W][t % W] = a;
  }
  __syncthreads();
  const int r = t / (W / 8), c = 8 * (t % (W / 8));
  if (r >= R || r >= g.I || j0 + c >= g.J) return;
  float v[8], bias[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = part[0][r][c + e];
  unsigned words[4] = {0u, 0u, 0u, 0u};
  if (g.epi.drop.cut != 0u) drop_words(g.epi.drop, drop_base(g.epi.drop) + (unsigned long long)r, (unsigned)(j0 + c) >> 3, words);
  dense_bias<T>(g.epi, bias, j0 + c, g.J, g.vec_e);
  dense_epilogue<T>(g.epi, v, bias, (long long)r * g.J + j0 + c, g.J - (j0 + c), g.vec_e, words);
}

// ---------------------------------------------------------------------------------------------------------------
// dz = D'(dy) act'(z) and the partial column sums of it (fp32, before dz is rounded): 256 columns a block as 32 threads of 8
// columns, 8 rows at a time; each block adds a run of rows up and writes one partial row.
// dz is rounded to the tensors' type, as the matrix cores take it and as a gradient handed on between layers would be: dx and dw of 16-bit
// types carry that half step beside their own (8192x1024x4096 bf16: 1.4 times the error of sums over an unrounded dz); db does not,
// and fp32 goes on as three planes.
// fp16's dz is stored without the dropout's scale and times 7/8 behind an activation whose slope passes 1 (gelu 1.129, silu 1.100): then
// it is no larger than dy, and a finite dy (of up to 65504) never becomes an infinity, which the products would spread over whole rows and columns;
// grad_scale undoes the factor on the fp32 sums.  At the low end dz has the steps of 2^-24 over the factor, 8/7 at most of those that D'(dy)
// has from dy's own.
// Bound: HBM.  8192x4096 bf16 gelu: 41 us with dy and z in the cache behind the L2, 54 without (201 MB, 4.9 and 3.7 TB/s).
// ---------------------------------------------------------------------------------------------------------------
struct DenseDz {
  const void *dy, *pre;
  void* dz;              // null: only the sums.  Rows of ld columns (the ones behind n as zeros), or fp32 as planes
  long long ld, plane_bytes;     // plane_bytes 0: dz in the tensors' type
  float* part;           // [chunks][N], null: none
  void* db;              // with one chunk: the sums themselves, instead of part
  long long rows, rows_per_chunk;
  int n, act, vec;
  float dz_scale;        // fp16: the factor that dz is stored with
  DropArgs drop;
};

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dense_dz_kernel(DenseDz p) {
  __shared__ float s[8][256];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int j = blockIdx.x * 256 + 8 * tx, n = min(8, p.n - j);
  const long long first = (long long)blockIdx.y * p.rows_per_chunk, last = min(p.rows, first + p.rows_per_chunk);
  const unsigned long long base = drop_base(p.drop);
  const T* const dy = static_cast<const T*>(p.dy) + j;
  const T* const pre = static_cast<const T*>(p.pre) + j;
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.f;
  if (n > 0) {
    constexpr int RB = 2;                 // rows in flight a thread
    for (long long i0 = first + ty; i0 < last; i0 += 8 * RB) {
      Raw8<T> d[RB], z[RB];
#pragma unroll
      for (int q = 0; q < RB; ++q) {
        const long long at = min(i0 + 8 * q, last - 1) * p.n;
        load_raw<T>(d[q], dy + at, n, VEC);
        if (p.act != VEEX_ACT_NONE) load_raw<T>(z[q], pre + at, n, VEC);
      }
#pragma unroll
      for (int q = 0; q < RB; ++q) {
        const long long i = i0 + 8 * q;
        if (i >= last) continue;
        float g[8], x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) { g[e] = VEC || e < n ? (float)d[q].v[e] : 0.f; x[e] = (float)z[q].v[e]; }
        if (p.drop.cut != 0u) {
          unsigned w[4];
          drop_words(p.drop, base + (unsigned long long)i, (unsigned)j >> 3, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = drop_u16(w, e) >= p.drop.cut ? g[e] * p.drop.scale : 0.f;
        }
        if (p.act != VEEX_ACT_NONE) {
          dense_act_grad<T, 8>(g, x, p.act);
          if (!VEC)
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = e < n ? g[e] : 0.f;       // (behind the last column z repeats another element)
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += g[e];
        if constexpr (TrunkType<T>::code == VEEX_T_F16) {
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] *= p.dz_scale;
        }
        if (p.dz != nullptr && p.plane_bytes != 0) dt_store_planes(static_cast<char*>(p.dz) + (i * p.ld + j) * 2, p.plane_bytes, g);
        else if (p.dz != nullptr) store8<T>(static_cast<T*>(p.dz) + i * p.ld + j, g, (int)(p.ld - j), VEC);
      }
    }
  }
  if (p.part == nullptr && p.db == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) s[ty][8 * tx + e] = sum[e];
  __syncthreads();
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col < p.n) {
    float a = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) a += s[q][threadIdx.x];
    if (p.db != nullptr) static_cast<T*>(p.db)[col] = (T)a;
    else p.part[(long long)blockIdx.y * p.n + col] = a;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
static const int kKindFwd = 0, kKindDx = 1, kKindDw = 2;     // which of A, B have k contiguous: A only; both; neither

// a tensor's 16-byte pieces along its contiguous index (length `len`) are whole and aligned
static bool operand_vec(const DenseOperand& o, long long len, int elem) {
  const long long other = o.k_stride == 1 ? o.row_stride : o.k_stride;
  return trunk_aligned16(o.p) && other * elem % 16 == 0 && len * elem % 16 == 0;
}

// The reduction is split where the tiles are fewer than two a CU: up to 512 blocks, at least 64 k each (1001x1003x1005 fp32 52 us
// with one a CU, 41 with two, 38 with three, where 640^3 goes from 17 to 19).
static void general_split(long long I, int J, long long K, int& splits, long long& per) {
  const long long tiles = (I + 63) / 64 * ((J + 63) / 64);
  long long s = tiles >= 512 ? 1 : std::min<long long>(512 / tiles, (K + 63) / 64);
  s = std::max<long long>(s, 1);
  per = ((K + s - 1) / s + 31) / 32 * 32;
  splits = (int)((K + per - 1) / per);
}

static long long align256(long long b) { return (b + 255) / 256 * 256; }

static long long general_bytes(long long I, int J, long long K) {
  int s; long long per;
  general_split(I, J, K, s, per);
  return s > 1 ? align256(s * I * slab_ld(J) * 4) : 0;
}

template <typename T>
static int join_launch(const DenseGemm& g, hipStream_t st) {
  const int lanes = join_lanes(g.I, g.J, g.splits);
  const dim3 grid(join_blocks(g.I, g.J, lanes));
  if (lanes == 1) hipLaunchKernelGGL((dense_join_kernel<T, 1>), grid, dim3(256), 0, st, g);
  else if (lanes == 8) hipLaunchKernelGGL((dense_join_kernel<T, 8>), grid, dim3(256), 0, st, g);
  else hipLaunchKernelGGL((dense_join_kernel<T, 32>), grid, dim3(256), 0, st, g);
  VEEX_CHECK_LAUNCH();
  return 0;
}
static int join_any(int dtype, const DenseGemm& g, hipStream_t st) {
  if (dtype == VEEX_T_F32) return join_launch<float>(g, st);
  if (dtype == VEEX_T_BF16) return join_launch<bf16_t>(g, st);
  return join_launch<f16_t>(g, st);
}

static bool general_vec(int kind, const DenseGemm& g, int elem) {
  return operand_vec(g.a, kind == kKindDw ? g.I : g.K, elem) && operand_vec(g.b, kind == kKindDx ? g.K : g.J, elem);
}
static long long general_tiles(const DenseGemm& g) { return (g.I + 63) / 64 * ((g.J + 63) / 64); }
static int too_many_tiles() { veex_set_error("dense: more tiles than a launch takes"); return VEEX_EINVAL; }

template <typename T>
static int general_launch(DenseGemm g, void* ws, hipStream_t st) {
  general_split(g.I, g.J, g.K, g.splits, g.k_per_split);
  g.slab = static_cast<float*>(ws);
  g.vec_e = dense_epi_vec(g.epi, g.J, sizeof(T));
  if (!trunk_grid_ok(general_tiles(g), 256)) return too_many_tiles();
  const dim3 grid((unsigned)general_tiles(g), (unsigned)g.splits);
  if (general_vec(kKindFwd, g, sizeof(T))) hipLaunchKernelGGL((dense_general_kernel<T, true>), grid, dim3(256), 0, st, g);
  else hipLaunchKernelGGL((dense_general_kernel<T, false>), grid, dim3(256), 0, st, g);
  VEEX_CHECK_LAUNCH();
  return g.splits > 1 ? join_launch<T>(g, st) : 0;
}

// g[0]: dx, g[1]: dw, as dense_product gives them with split and slab set; I = 0: not wanted
template <typename T>
static int general_grads_launch(const DenseGemm (&g)[2], hipStream_t st) {
  const long long t0 = general_tiles(g[0]), t1 = general_tiles(g[1]), n0 = t0 * g[0].splits, n1 = t1 * g[1].splits;
  if (!trunk_grid_ok(n0 + n1, 256)) return too_many_tiles();
  const bool vec = (n0 == 0 || general_vec(kKindDx, g[0], sizeof(T))) && (n1 == 0 || general_vec(kKindDw, g[1], sizeof(T)));
  const dim3 grid((unsigned)(n0 + n1));
  // dx's blocks come first, unless those of dw take over twice as long: started last they would run on alone (fp32 backward us, dx first and
  // dw first: dw's blocks three times as long, 3000x1500x150 60 and 54, 1024x4096x150 53 and 46; eight times, 2048x6400x100 104 and 82; twice,
  // 512x6400x100 30 and 33, 2048x2048x100 36 and 34; a tenth, 128x4096x4096 93 and 98, 64x4096x14336 179 and 206)
  const bool dw_first = n0 == 0 || (n1 > 0 && g[1].k_per_split > 2 * g[0].k_per_split);
  const unsigned dx_from = dw_first ? (unsigned)n1 : 0u, dw_from = dw_first ? 0u : (unsigned)n0;
  if (vec) hipLaunchKernelGGL((dense_general_grads_kernel<T, true>), grid, dim3(256), 0, st, g[0], g[1], (unsigned)t0, (unsigned)t1, dx_from, dw_from);
  else hipLaunchKernelGGL((dense_general_grads_kernel<T, false>), grid, dim3(256), 0, st, g[0], g[1], (unsigned)t0, (unsigned)t1, dx_from, dw_from);
  VEEX_CHECK_LAUNCH();
  return 0;
}

static int dense_check(const VeexDense* d, const char* who, DropArgs& drop) {
  if (d == nullptr || (d->struct_size != 0 && d->struct_size != (int)sizeof(VeexDense))) { veex_set_error("%s: struct_size is not this library's", who); return VEEX_EINVAL; }
  if (!trunk_dtype_ok(d->dtype) || d->activation < 0 || d->activation > VEEX_ACT_SIGMOID) { veex_set_error("%s: unknown dtype or activation", who); return VEEX_EINVAL; }
  if (d->rows < 0 || d->rows > (1ll << 31) || d->k < 1 || d->k > (1 << 30) || d->n < 1 || d->n > (1 << 30) || d->ldx < d->k) {
    veex_set_error("%s: 0 <= rows <= 2^31, 1 <= k, n <= 2^30 and ldx >= k are needed", who); return VEEX_EINVAL;
  }
  if (!trunk_drop_args(d->rate, d->seed, d->first_row, d->counter, drop)) { veex_set_error("%s: rate %g is outside [0, 1 - 2^-17)", who, d->rate); return VEEX_EINVAL; }
  return 0;
}

static bool lies_well(const VeexDense* d, const void* p, long long ld, long long cols);

// ---- few rows -------------------------------------------------------------------------------------------------------
// about 1024 blocks, at least 64 k's each
static void few_split(const DenseGemm& g, bool vec, int elem, int& splits, long long& per) {
  const long long strips = vec ? ((long long)g.J * elem + 255) / 256 : (g.J + 63) / 64;
  const long long s = std::max<long long>(std::min<long long>((1023 + strips) / strips, g.K / 64), 1);
  per = (g.K + s - 1) / s;
  splits = (int)((g.K + per - 1) / per);
}

static bool few_short(const DenseGemm& g, int elem) { return g.K <= DF_SHORT_K && operand_vec(g.b, g.J, elem); }

template <typename T>
static int few_launch(DenseGemm g, void* ws, hipStream_t st) {
  if (few_short(g, sizeof(T))) {
    g.splits = 1;
    g.vec_e = dense_epi_vec(g.epi, g.J, sizeof(T));
    const unsigned strips = (unsigned)(((long long)g.J * (int)sizeof(T) + 127) / 128);
    if (g.I == 1) hipLaunchKernelGGL((dense_few_short_kernel<T, 1>), dim3(strips), dim3(1024), 0, st, g, strips);
    else if (g.I == 2) hipLaunchKernelGGL((dense_few_short_kernel<T, 2>), dim3(strips), dim3(1024), 0, st, g, strips);
    else if (g.I <= 4) hipLaunchKernelGGL((dense_few_short_kernel<T, 4>), dim3(strips), dim3(1024), 0, st, g, strips);
    else hipLaunchKernelGGL((dense_few_short_kernel<T, 8>), dim3(strips), dim3(1024), 0, st, g, strips);
    VEEX_CHECK_LAUNCH();
    return 0;
  }
  const bool vec = operand_vec(g.b, g.J, sizeof(T));
  few_split(g, vec, sizeof(T), g.splits, g.k_per_split);
  g.slab = static_cast<float*>(ws);
  g.vec_e = dense_epi_vec(g.epi, g.J, sizeof(T));
  const long long strips = vec ? ((long long)g.J * (int)sizeof(T) + 255) / 256 : (g.J + 63) / 64;
  if (!trunk_grid_ok(strips, 256)) return too_many_tiles();
  const dim3 grid((unsigned)strips, (unsigned)g.splits);
#define DF_GO(R)                                                                                              \
  if (vec) hipLaunchKernelGGL((dense_few_rows_kernel<T, R, true>), grid, dim3(256), 0, st, g);                 \
  else hipLaunchKernelGGL((dense_few_rows_kernel<T, R, false>), grid, dim3(256), 0, st, g);
  if (g.I == 1) { DF_GO(1) }
  else if (g.I == 2) { DF_GO(2) }
  else if (g.I <= 4) { DF_GO(4) }
  else { DF_GO(8) }
#undef DF_GO
  VEEX_CHECK_LAUNCH();
  return join_launch<T>(g, st);
}

// Up to 8 rows; 2 where the tiles take the operands as they lie (4096x14336 bf16: 22.9 us for one row, 24.2 for two, 26.3 for three and
// 46 for eight, where the tiles take 25 for any of them; fp32 4096x14336: 38.4 to 49.6, the general product 90).  And the weights
// are worth a second launch to join: from 2^16 of them on (below, one tile of the general product is as quick).
static bool few_rows(const VeexDense* d) {
  const bool tiles = lies_well(d, d->x, d->ldx, d->k) && lies_well(d, d->w, d->n, d->n);
  return d->rows <= (tiles ? 2 : 8) && (long long)d->k * d->n >= (1 << 16) && d->n <= (1 << 24);
}

static long long few_bytes(const VeexDense* d, const DenseGemm& g) {
  const int elem = trunk_elem_bytes(d->dtype);
  if (few_short(g, elem)) return 0;
  int s; long long per;
  few_split(g, operand_vec(g.b, g.J, elem), elem, s, per);
  return align256(s * g.I * slab_ld(g.J) * 4);
}

// ---- large products -------------------------------------------------------------------------------------------------
// Which products go to dense_tile.hip.  16-bit types: all that need no packing (16x1024x1024 9.0 us on the general product, 8.5 on
// the tiles; 512^3 15.3, 8.4), packed ones from 2^26 multiplications on (257x255x259 10, 12.5; 385x383x387 13, 13.7).
// fp32, which is packed and multiplied six times: from 1.5e9 on (1000^3 34, 32; 2048x1024x1024 53, 43; 4096x1024x1024 90, 60), with 160
// rows and columns, or the packed copies are used too little (forward and training call of 128x4096x4096 52 and 154, 66 and 191;
// 176x4096x4096 92 and 232, 76 and 208; 4096x4096x128 52 and 169, 70 and 195; 8192x100x6400 196 and 614, 184 and 529).
static bool uses_tiles(const VeexDense* d) {
  // a tile addresses its operand by 32 bits from its first row on: 256 rows of up to 4 MB, 64 k's of up to 16 MB
  const long long widest = std::max<long long>(std::max<long long>(d->k, d->n), d->ldx);
  if (widest >= (1 << 21)) return false;
  const double work = (double)d->rows * d->k * d->n;
  if (d->dtype == VEEX_T_F32) return work >= 1.5e9 && d->rows >= 160 && d->n >= 160;
  return work >= (1 << 26) || (lies_well(d, d->x, d->ldx, d->k) && lies_well(d, d->w, d->n, d->n) && lies_well(d, d->dy, d->n, d->n));
}

static long long round8(long long v) { return (v + 7) / 8 * 8; }
static int planes_of(const VeexDense* d) { return d->dtype == VEEX_T_F32 ? 3 : 1; }
// a packed copy of a rows x cols tensor
static long long packed_plane(long long rows, long long cols) { return align256(rows * round8(cols) * 2); }
static long long packed_bytes(const VeexDense* d, long long rows, long long cols) { return planes_of(d) * packed_plane(rows, cols); }
// a 16-bit tensor that the tiles can load where it lies
static bool lies_well(const VeexDense* d, const void* p, long long ld, long long cols) {
  return d->dtype != VEEX_T_F32 && trunk_aligned16(p) && ld % 8 == 0 && cols % 8 == 0;
}

struct TilePlan { int tile, bm, bn; unsigned splits; long long per; };

// The tile and the split of the reduction: the fewest rounds of the chip's 256 tile slots, weighed by a tile's time: `step` is the measured
// time of 32 k's in microseconds with the chip full, 3 steps stand for the way in and out, and a split pays for its slabs at 4 TB/s
// and for the launch that joins them.
static TilePlan tile_plan(const VeexDense* d, long long I, long long J, long long K) {
  TilePlan best = {};
  double cost = 1e300;
  const bool f32 = d->dtype == VEEX_T_F32;
  const int bk = 32;
  struct Shape { int code, bm, bn, slots; double step; };
  static const Shape shapes16[] = {{0, 256, 256, 256, 0.93}, {1, 256, 128, 256, 0.53}, {2, 128, 128, 256, 0.33}};
  static const Shape shapes32[] = {{1, 256, 128, 256, 2.4}, {2, 128, 128, 256, 1.3}};
  for (int q = 0; q < (f32 ? 2 : 3); ++q) {
    const Shape& sh = f32 ? shapes32[q] : shapes16[q];
    const long long tiles = (I + sh.bm - 1) / sh.bm * ((J + sh.bn - 1) / sh.bn);
    for (long long s = 1; s <= 64; s *= 2) {
      const long long per = ((K + s - 1) / s + bk - 1) / bk * bk, splits = (K + per - 1) / per;
      if (s > 1 && per < 4 * bk) break;
      const double rounds = (double)((tiles * splits + sh.slots - 1) / sh.slots);
      const double join = splits > 1 ? (double)splits * I * J * 8.0 / 4.0e6 + 4.0 : 0.0;   // slabs out and in, one more launch
      const double c = rounds * sh.step * ((double)per / 32.0 + 3.0) + join;
      if (c < cost) { cost = c; best = {sh.code, sh.bm, sh.bn, (unsigned)splits, per}; }
    }
  }
  return best;
}

static DenseGemm dense_product(int kind, const VeexDense* d, const void* dz) {
  DenseGemm g = {};
  if (kind == kKindFwd) {
    g.I = d->rows; g.J = d->n; g.K = d->k;
    g.a = {d->x, d->ldx, 1}; g.b = {d->w, 1, d->n};
  } else if (kind == kKindDx) {          // dx[i][j] = sum_n dz(i, n) w(j, n)
    g.I = d->rows; g.J = d->k; g.K = d->n;
    g.a = {dz, d->n, 1}; g.b = {d->w, d->n, 1};
    g.epi.y = d->dx;
  } else {                               // dw[i][j] = sum_m x(m, i) dz(m, j)
    g.I = d->k; g.J = d->n; g.K = d->rows;
    g.a = {d->x, 1, d->ldx}; g.b = {dz, 1, d->n};
    g.epi.y = d->dw;
  }
  return g;
}

// bytes of one product's slabs
static long long product_bytes(int kind, const VeexDense* d) {
  const DenseGemm g = dense_product(kind, d, nullptr);
  if (kind == kKindFwd && few_rows(d)) return few_bytes(d, g);
  if (!uses_tiles(d)) return general_bytes(g.I, g.J, g.K);
  const TilePlan t = tile_plan(d, g.I, g.J, g.K);
  return t.splits > 1 ? align256(t.splits * g.I * slab_ld(g.J) * 4) : 0;
}

static int general_any(int dtype, const DenseGemm& g, void* ws, hipStream_t st) {
  if (dtype == VEEX_T_F32) return general_launch<float>(g, ws, st);
  if (dtype == VEEX_T_BF16) return general_launch<bf16_t>(g, ws, st);
  return general_launch<f16_t>(g, ws, st);
}

// a product on tiles, up to the launch; false: more tiles than one takes
static bool tile_gemm(int elem, const TilePlan& t, const DenseGemm& g, const DtTensor& a, const DtTensor& b, void* slab, DtGemm& q) {
  q = {};
  q.a = a; q.b = b; q.I = g.I; q.J = g.J; q.K = g.K; q.k_per_split = t.per; q.splits = t.splits;
  q.epi = g.epi;
  q.slab = t.splits > 1 ? static_cast<float*>(slab) : nullptr;
  q.vec_e = dense_epi_vec(g.epi, g.J, elem);
  q.alpha = g.alpha;
  return (double)((g.I + t.bm - 1) / t.bm) * ((g.J + t.bn - 1) / t.bn) * t.splits < (1 << 22);      // (512 threads each, two products a launch)
}

// x, w or dy as the tiles load it: where it lies, or packed into *at, which moves on (the job is added to the list)
static void tile_operand(const VeexDense* d, const void* p, long long ld, long long rows, int cols, char*& at, DtTensor& t, DtPack* jobs, int& n) {
  if (lies_well(d, p, ld, cols)) { t = {p, ld * 2, 0}; return; }
  const long long plane = packed_plane(rows, cols);
  t = {at, round8(cols) * 2, plane};
  jobs[n++] = {p, at, ld, rows, plane, cols};
  at += planes_of(d) * plane;
}
static long long tile_operand_bytes(const VeexDense* d, const void* p, long long ld, long long rows, int cols) {
  return lies_well(d, p, ld, cols) ? 0 : packed_bytes(d, rows, cols);
}

static long long fwd_bytes(const VeexDense* d) {
  long long b = product_bytes(kKindFwd, d);
  if (uses_tiles(d)) b += tile_operand_bytes(d, d->x, d->ldx, d->rows, d->k) + tile_operand_bytes(d, d->w, d->n, d->k, d->n);
  return b;
}

// the backward workspace: [dz: made here, or dy packed] [partial column sums] [x, w packed] [dx's slabs] [dw's slabs]
struct BwdLayout {
  bool dz_own, tiles;
  long long dz, part, packed, slab[2], rows_per_chunk;
  int chunks;
  long long total() const { return dz + part + packed + slab[0] + slab[1]; }
};

// what dz is stored with (dense_dz_kernel)
static float dz_factor(const VeexDense* d, const DropArgs& drop) {
  if (d->dtype != VEEX_T_F16) return 1.f;
  const bool steep = d->activation == VEEX_ACT_GELU || d->activation == VEEX_ACT_SILU;
  return (steep ? 0.875f : 1.f) * (drop.cut != 0u ? (float)(65536u - drop.cut) / 65536.f : 1.f);
}

static BwdLayout bwd_layout(const VeexDense* d, const DropArgs& drop) {
  BwdLayout l = {};
  l.dz_own = d->activation != VEEX_ACT_NONE || drop.cut != 0u;
  l.tiles = uses_tiles(d);
  const int strips = (d->n + 255) / 256;
  const long long want = std::max<long long>(1024 / strips, 1);
  // (up to 64 rows one chunk: eight turns, and no second launch to add partial rows)
  l.rows_per_chunk = d->rows <= 64 ? 64 : std::max<long long>(((d->rows + want - 1) / want + 7) / 8 * 8, 8);
  l.chunks = (int)((d->rows + l.rows_per_chunk - 1) / l.rows_per_chunk);
  if (l.tiles) {
    l.dz = l.dz_own ? packed_bytes(d, d->rows, d->n) : tile_operand_bytes(d, d->dy, d->n, d->rows, d->n);
    l.packed = (d->dw != nullptr ? tile_operand_bytes(d, d->x, d->ldx, d->rows, d->k) : 0) + (d->dx != nullptr ? tile_operand_bytes(d, d->w, d->n, d->k, d->n) : 0);
  } else {
    l.dz = l.dz_own ? align256(d->rows * d->n * trunk_elem_bytes(d->dtype)) : 0;
  }
  l.part = align256((long long)l.chunks * d->n * 4);
  l.slab[0] = d->dx != nullptr ? product_bytes(kKindDx, d) : 0;
  l.slab[1] = d->dw != nullptr ? product_bytes(kKindDw, d) : 0;
  return l;
}

extern "C" {

int veex_dense_plan(const VeexDense* d, int product) {
  DropArgs drop;
  if (dense_check(d, "dense", drop) != 0) return -1;
  if (product < kKindFwd || product > kKindDw || d->rows == 0) { veex_set_error("dense: product 0 (y), 1 (dx) or 2 (dw), and rows, are needed"); return -1; }
  const DenseGemm g = dense_product(product, d, nullptr);
  if (product == kKindFwd && few_rows(d)) {
    const int elem = trunk_elem_bytes(d->dtype);
    if (few_short(g, elem)) return VEEX_DENSE_FEW_SHORT | 1 << 8;
    int s; long long per;
    few_split(g, operand_vec(g.b, g.J, elem), elem, s, per);
    return VEEX_DENSE_FEW | s << 8;
  }
  if (!uses_tiles(d)) {
    int s; long long per;
    general_split(g.I, g.J, g.K, s, per);
    return VEEX_DENSE_GENERAL | s << 8;
  }
  const TilePlan t = tile_plan(d, g.I, g.J, g.K);
  return (t.tile == 0 ? VEEX_DENSE_TILE_256X256 : t.tile == 1 ? VEEX_DENSE_TILE_256X128 : VEEX_DENSE_TILE_128X128) | (int)t.splits << 8;
}

long long veex_dense_fwd_workspace_bytes(const VeexDense* d) {
  DropArgs drop;
  if (dense_check(d, "dense", drop) != 0) return -1;
  return d->rows == 0 ? 0 : fwd_bytes(d);
}

int veex_dense_fwd(const VeexDense* d, hipStream_t st) {
  DropArgs drop;
  if (int rc = dense_check(d, "dense", drop)) return rc;
  if (d->x == nullptr || d->w == nullptr || d->y == nullptr) { veex_set_error("dense: x, w and y are needed"); return VEEX_EINVAL; }
  if (d->rows == 0) return 0;
  const long long need = fwd_bytes(d);
  if (need > 0 && (!trunk_aligned16(d->workspace) || d->workspace == nullptr || d->workspace_bytes < need)) {
    veex_set_error("dense: a 16-byte aligned workspace of %lld bytes is needed", need); return VEEX_ENOMEM;
  }
  DenseGemm g = dense_product(kKindFwd, d, nullptr);
  g.epi = {d->bias, d->residual, d->y, d->pre, d->activation, drop};
  if (few_rows(d)) {
    if (d->dtype == VEEX_T_F32) return few_launch<float>(g, d->workspace, st);
    if (d->dtype == VEEX_T_BF16) return few_launch<bf16_t>(g, d->workspace, st);
    return few_launch<f16_t>(g, d->workspace, st);
  }
  if (!uses_tiles(d)) return general_any(d->dtype, g, d->workspace, st);
  char* at = static_cast<char*>(d->workspace);
  DtTensor x = {}, w = {};
  DtPack jobs[2];
  int n = 0;
  tile_operand(d, d->x, d->ldx, d->rows, d->k, at, x, jobs, n);
  tile_operand(d, d->w, d->n, d->k, d->n, at, w, jobs, n);
  if (int rc = dense_pack_launch(d->dtype, jobs, n, st)) return rc;
  const TilePlan t = tile_plan(d, g.I, g.J, g.K);
  DtGemm q;
  if (!tile_gemm(trunk_elem_bytes(d->dtype), t, g, x, w, at, q)) return too_many_tiles();
  if (int rc = dense_tile_launch(d->dtype, true, false, t.tile, q, st)) return rc;
  if (t.splits == 1) return 0;
  g.slab = q.slab; g.splits = (int)t.splits; g.vec_e = q.vec_e;
  return join_any(d->dtype, g, st);
}

long long veex_dense_bwd_workspace_bytes(const VeexDense* d) {
  DropArgs drop;
  if (dense_check(d, "dense backward", drop) != 0) return -1;
  return bwd_layout(d, drop).total();
}

int veex_dense_bwd(const VeexDense* d, hipStream_t st) {
  DropArgs drop;
  if (int rc = dense_check(d, "dense backward", drop)) return rc;
  if (d->dy == nullptr || (d->dw != nullptr && d->x == nullptr) || (d->dx != nullptr && d->w == nullptr) ||
      (d->activation != VEEX_ACT_NONE && d->pre == nullptr)) {
    veex_set_error("dense backward: dy, x for dw, w for dx and pre for an activation are needed"); return VEEX_EINVAL;
  }
  if (d->rows == 0) { veex_set_error("dense backward: no rows"); return VEEX_EINVAL; }
  const BwdLayout l = bwd_layout(d, drop);
  if (l.total() > 0 && (!trunk_aligned16(d->workspace) || d->workspace == nullptr || d->workspace_bytes < l.total())) {
    veex_set_error("dense backward: a 16-byte aligned workspace of %lld bytes is needed", l.total()); return VEEX_ENOMEM;
  }
  char* ws = static_cast<char*>(d->workspace);
  const bool products = d->dx != nullptr || d->dw != nullptr;
  const void* dz = l.dz_own ? ws : d->dy;                  // the general product's
  const float factor = l.dz_own ? dz_factor(d, drop) : 1.f;
  DtTensor dzt = {ws, round8(d->n) * 2, packed_plane(d->rows, d->n)};    // the tiles'
  if (l.dz_own || d->db != nullptr) {
    DenseDz p = {};
    p.dy = d->dy; p.pre = d->pre; p.dz = l.dz_own && products ? ws : nullptr;
    p.ld = l.tiles ? round8(d->n) : d->n;
    p.plane_bytes = l.tiles && d->dtype == VEEX_T_F32 ? dzt.plane_bytes : 0;
    p.db = l.chunks == 1 ? d->db : nullptr;
    p.part = d->db != nullptr && l.chunks > 1 ? reinterpret_cast<float*>(ws + l.dz) : nullptr;
    p.rows = d->rows; p.rows_per_chunk = l.rows_per_chunk; p.n = d->n; p.act = d->activation; p.drop = drop; p.dz_scale = factor;
    p.vec = (long long)d->n * trunk_elem_bytes(d->dtype) % 16 == 0 && trunk_aligned16(d->dy) && (d->activation == VEEX_ACT_NONE || trunk_aligned16(d->pre));
    if (p.dz != nullptr || d->db != nullptr) {
      const dim3 grid((d->n + 255) / 256, l.chunks);
#define DZ_GO(T)                                                                                              \
  if (p.vec) hipLaunchKernelGGL((dense_dz_kernel<T, true>), grid, dim3(256), 0, st, p);                        \
  else hipLaunchKernelGGL((dense_dz_kernel<T, false>), grid, dim3(256), 0, st, p);
      if (d->dtype == VEEX_T_F32) { DZ_GO(float) }
      else if (d->dtype == VEEX_T_BF16) { DZ_GO(bf16_t) }
      else { DZ_GO(f16_t) }
#undef DZ_GO
      VEEX_CHECK_LAUNCH();
    }
  }
  float* const part = d->db != nullptr && l.chunks > 1 ? reinterpret_cast<float*>(ws + l.dz) : nullptr;
  if (!products && part == nullptr) return 0;

  char* at = ws + l.dz + l.part;
  float* const slabs[2] = {reinterpret_cast<float*>(at + l.packed), reinterpret_cast<float*>(at + l.packed + l.slab[0])};
  DenseGemm g[2] = {};
  if (d->dx != nullptr) g[0] = dense_product(kKindDx, d, dz);
  if (d->dw != nullptr) g[1] = dense_product(kKindDw, d, dz);
  for (int q = 0; q < 2; ++q) { g[q].splits = 1; g[q].alpha = 1.f / factor; g[q].slab = slabs[q]; g[q].vec_e = dense_epi_vec(g[q].epi, g[q].J, trunk_elem_bytes(d->dtype)); }
  if (products && !l.tiles) {
    for (DenseGemm& q : g)
      if (q.I > 0) general_split(q.I, q.J, q.K, q.splits, q.k_per_split);
    const int rc = d->dtype == VEEX_T_F32 ? general_grads_launch<float>(g, st) : d->dtype == VEEX_T_BF16 ? general_grads_launch<bf16_t>(g, st) : general_grads_launch<f16_t>(g, st);
    if (rc != 0) return rc;
  } else if (products) {
    DtTensor x = {}, w = {};
    DtPack jobs[3];
    int n = 0;
    if (!l.dz_own) {
      char* p = ws;
      tile_operand(d, d->dy, d->n, d->rows, d->n, p, dzt, jobs, n);
    }
    if (d->dx != nullptr) tile_operand(d, d->w, d->n, d->k, d->n, at, w, jobs, n);
    if (d->dw != nullptr) tile_operand(d, d->x, d->ldx, d->rows, d->k, at, x, jobs, n);
    if (int rc = dense_pack_launch(d->dtype, jobs, n, st)) return rc;
    TilePlan t[2] = {};
    DtGemm q[2] = {};
    for (int k = 0; k < 2; ++k)
      if (g[k].I > 0) {
        t[k] = tile_plan(d, g[k].I, g[k].J, g[k].K);
        if (!tile_gemm(trunk_elem_bytes(d->dtype), t[k], g[k], k == 0 ? dzt : x, k == 0 ? w : dzt, slabs[k], q[k])) return too_many_tiles();
        g[k].splits = (int)t[k].splits;
      }
    if (g[0].I > 0 && g[1].I > 0 && t[0].tile == 2 && t[1].tile == 2) {
      if (int rc = dense_tile_grads_launch(d->dtype, q[0], q[1], st)) return rc;
    } else {
      for (int k = 0; k < 2; ++k)
        if (g[k].I > 0)
          if (int rc = dense_tile_launch(d->dtype, k == 0, k == 0, t[k].tile, q[k], st)) return rc;
    }
  }

  DenseFinish f = {};
  f.alpha = 1.f / factor;
  for (int q = 0; q < 2; ++q) {
    f.first[q + 1] = f.first[q];
    if (g[q].splits == 1) continue;
    const int lanes = join_lanes(g[q].I, g[q].J, g[q].splits);
    f.sum[q] = {slabs[q], g[q].epi.y, g[q].I, g[q].J, g[q].splits, lanes, g[q].vec_e};
    f.first[q + 1] += join_blocks(g[q].I, g[q].J, lanes);
  }
  f.first[3] = f.first[2];
  if (part != nullptr) {
    f.part = part; f.db = d->db; f.chunks = l.chunks; f.n = d->n;
    f.first[3] += (unsigned)((d->n + 31) / 32);
  }
  if (f.first[3] == 0) return 0;
  if (!trunk_grid_ok(f.first[3], 256)) return too_many_tiles();
  const dim3 grid(f.first[3]);
  if (d->dtype == VEEX_T_F32) hipLaunchKernelGGL((dense_finish_kernel<float>), grid, dim3(256), 0, st, f);
  else if (d->dtype == VEEX_T_BF16) hipLaunchKernelGGL((dense_finish_kernel<bf16_t>), grid, dim3(256), 0, st, f);
  else hipLaunchKernelGGL((dense_finish_kernel<f16_t>), grid, dim3(256), 0, st, f);
  VEEX_CHECK_LAUNCH();
  return 0;
}

}  // extern "C"
