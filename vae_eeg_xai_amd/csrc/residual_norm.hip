// The step between two blocks of a residual trunk, in one pass over the rows:
//   n = Norm_post(h),  x_out = x + scale * gate * n,  u = Norm_pre(x_out)
// Norm is LayerNorm (mean and variance over the row) or RMSNorm, each with an optional weight and bias; without h it is
// u = Norm_pre(x) alone (the trunk's entry).  gate has `groups` rows, each for rows/groups consecutive rows of x (rows: one
// gate per element; 1: one per column), scale one value per column.  Backward, with D the whole gradient at x_out:
//   t = du * pre_w;  D = dx_out + rstd2 (t - mean(t) - rhat mean(t rhat))        rhat = (x_out - mean2) rstd2
//   dn = D scale gate;  e = dn post_w;  dh = rstd1 (e - mean(e) - xhat mean(e xhat));  dx = D
//   dgate = sum over the group of D scale n;  dscale = sum D gate n;  dpost_w = sum dn xhat;  dpost_b = sum dn;
//   dpre_w = sum du rhat;  dpre_b = sum du          (RMSNorm: without the means of t and e)
//
// Bound: HBM.  A row lives in the registers of 8 lanes to 16 waves (8 or 16 elements a lane), so the forward pass reads x, h and
// gate once and writes x_out and u once; the backward pass recomputes x_out from x and h in fp32 instead of reading the
// rounded one (the same bytes, and the gradient is that of the unrounded chain).  8192x4096 bf16 with a gate of 8 groups: forward 58 us
// (4.6 TB/s), backward 104 us and 10 for its column sums (3.5 TB/s); fp32, the same call again and again, 98 and 174 us (5.5 and 4.6 TB/s); a copy
// of 1 GB runs at 4.9.  (Where a comment below gives two times of a backward pass, x and h stood for dx_out and du too: a third fewer
// bytes.)  All statistics and sums are fp32; the variance is the mean of squared deviations (two passes over registers), not a
// difference of moments.
// Column sums: each block adds up its own run of rows in registers, writes one partial row per sum, and a second kernel adds
// the partial rows in a fixed order: no atomics, the same bits every time.
#include "trunk_common.h"
#include "../../include/veex.h"
#include <algorithm>

struct RNormParams {
  const void *x, *h, *gate, *scale, *post_w, *post_b, *pre_w, *pre_b;
  void *x_out, *u;
  float* stats;              // [rows][4]: mean1, rstd1, mean2, rstd2
  const void *dx_out, *du;   // backward; either may be null (a zero gradient)
  void *dx, *dh, *dgate, *dscale, *dpost_w, *dpost_b, *dpre_w, *dpre_b;
  float* part;               // [chunks][5][cols]; walk: then [chunks][rows a block works on][cols], dscale's running sums
  long long rows;
  int cols, layer;
  float eps;
  long long groups, rows_per_group, rows_per_chunk, chunks_per_group;
  int walk;                  // a chunk is rows_per_chunk rows of whole groups (rnorm_plan)
};

// Sum over groups of G = 8 to 64 neighbouring lanes, in every lane: neighbours, pairs, quads and eights through DPP, rows of 16 through
// lane swaps.
// (A shuffle goes through LDS, some hundred cycles a step; six steps twice or more a row were a third of these kernels' time.)
template <int G> __device__ __forceinline__ float rn_lanes_sum(float x) {
#define RN_DPP(CTRL) x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xF, 0xF, true))
  RN_DPP(0xB1);       // quad_perm [1,0,3,2]
  RN_DPP(0x4E);       // quad_perm [2,3,0,1]
  RN_DPP(0x141);      // row_half_mirror
  if (G >= 16) RN_DPP(0x140);      // row_mirror
#undef RN_DPP
  if (G >= 32) {
    const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(h[0]) + __uint_as_float(h[1]);
  }
  if (G >= 64) {
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(w[0]) + __uint_as_float(w[1]);
  }
  return x;
}

// sum of a and b over the LANES lanes of a row; red: two buffers of 2 * 16 floats, taken in turn, so that one barrier a sum is enough
// (a wave can write a buffer again only after the barrier of the sum in between)
template <int LANES>
struct RowSum {
  static constexpr int WPR = LANES > 64 ? LANES / 64 : 1;        // waves a row
  float* red; int first, wave, turn;                             // first: the row's first wave
  __device__ __forceinline__ RowSum(float* r) : red(r), first(threadIdx.x / LANES * WPR), wave(threadIdx.x >> 6), turn(0) {}
  __device__ __forceinline__ float2 operator()(float a, float b) {
    a = rn_lanes_sum<LANES < 64 ? LANES : 64>(a); b = rn_lanes_sum<LANES < 64 ? LANES : 64>(b);
    if (WPR == 1) return make_float2(a, b);
    float* r = red + turn * 32;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) { r[wave * 2] = a; r[wave * 2 + 1] = b; }
    __syncthreads();
    a = 0.f; b = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) { a += r[(first + w) * 2]; b += r[(first + w) * 2 + 1]; }
    return make_float2(a, b);
  }
};

template <typename T, int V, int C> struct RowRaw { Piece<T, V> p[C]; };

template <typename T, int V, int C, int LANES>
__device__ __forceinline__ void row_load(RowRaw<T, V, C>& r, const void* base, long long at, int lane, int cols) {
  const T* p = static_cast<const T*>(base) + at;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * LANES + lane) * V;
    if (V == 1) {      // (whole pieces: a load of some piece and a choice; a branch around the load put fp32 rows into scratch memory,
                       // 16384x1024 65 us for 42)
      if (col < cols) r.p[c] = piece_load<T, V>(p + col);
      else r.p[c].v[0] = (T)0.f;
    } else {
      const Piece<T, V> q = piece_load<T, V>(p + (col < cols ? col : 0));
#pragma unroll
      for (int e = 0; e < V; ++e) r.p[c].v[e] = col < cols ? q.v[e] : (T)0.f;
    }
  }
}
template <typename T, int V, int C>
__device__ __forceinline__ void row_copy(RowRaw<T, V, C>& a, const RowRaw<T, V, C>& b) {
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) a.p[c].v[e] = b.p[c].v[e];
}
template <typename T, int V, int C, int LANES>
__device__ __forceinline__ void row_fill(RowRaw<T, V, C>& r, float v) {
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) r.p[c].v[e] = (T)v;
}
template <typename T, int V, int C, int LANES>
__device__ __forceinline__ void row_store(void* base, long long at, const float (&v)[V * C], int lane, int cols) {
  T* p = static_cast<T*>(base) + at;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * LANES + lane) * V;
    if (col < cols) {
      Piece<T, V> q;
#pragma unroll
      for (int e = 0; e < V; ++e) q.v[e] = (T)v[c * V + e];
      piece_store<T, V>(p + col, q);
    }
  }
}
template <typename T, int V, int C, int LANES>
__device__ __forceinline__ void row_param(RowRaw<T, V, C>& r, const void* p, float otherwise, int lane, int cols) {
  if (p != nullptr) row_load<T, V, C, LANES>(r, p, 0, lane, cols);
  else row_fill<T, V, C, LANES>(r, otherwise);
}

// LANES lanes a row (8 of a wave, 32 rows a block, up to 16 waves), EPL elements a lane; VEC: rows are whole 16-byte pieces
template <typename T, int LANES, int EPL, bool VEC>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void rnorm_fwd_kernel(RNormParams p) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1, C = EPL / V;
  constexpr int RG = LANES > 256 ? 1 : 256 / LANES;        // rows a block works on
  __shared__ float red[64];
  const int lane = threadIdx.x % LANES, rg = threadIdx.x / LANES;
  RowSum<LANES> row_sum(red);
  const float inv = 1.f / (float)p.cols;

  // (16 elements a lane of 16 waves, 128 registers each: the next row is not fetched ahead, and the vectors are read again each row)
  constexpr bool AHEAD = EPL == 8;
  RowRaw<T, V, C> scale, ow, ob, pw, pb;
  auto vectors_post = [&] {
    row_param<T, V, C, LANES>(scale, p.scale, 1.f, lane, p.cols);
    row_param<T, V, C, LANES>(ow, p.post_w, 1.f, lane, p.cols);
    row_param<T, V, C, LANES>(ob, p.post_b, 0.f, lane, p.cols);
  };
  auto vectors_pre = [&] {
    row_param<T, V, C, LANES>(pw, p.pre_w, 1.f, lane, p.cols);
    row_param<T, V, C, LANES>(pb, p.pre_b, 0.f, lane, p.cols);
  };
  if (AHEAD) { vectors_post(); vectors_pre(); }

  bool in[C];
#pragma unroll
  for (int c = 0; c < C; ++c) in[c] = (c * LANES + lane) * V < p.cols;
  // mean and 1/deviation of the row v (zero outside the row)
  auto moments = [&](const float (&v)[EPL], float& mean, float& rstd) {
    mean = 0.f;
    if (p.layer) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) s += v[e];
      mean = row_sum(s, 0.f).x * inv;
    }
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) { const float d = in[e / V] ? v[e] - mean : 0.f; q = fmaf(d, d, q); }
    rstd = 1.f / sqrtf(row_sum(q, 0.f).x * inv + p.eps);
  };

  // Every row group of a block takes the same number of turns (the sums hold barriers); a turn past the end repeats the last row.
  // The next turn's rows are on their way while this one's are worked on: a turn is a chain of load, two to four sums across the
  // waves and store, and the chip has too few rows in flight to hide it otherwise.
  struct In { RowRaw<T, V, C> x, h, g; };
  auto fetch = [&](In& r, long long row) {
    row = min(row, p.rows - 1);
    row_load<T, V, C, LANES>(r.x, p.x, row * p.cols, lane, p.cols);
    if (p.h != nullptr) row_load<T, V, C, LANES>(r.h, p.h, row * p.cols, lane, p.cols);
    if (p.gate != nullptr) row_load<T, V, C, LANES>(r.g, p.gate, (long long)((unsigned)row / (unsigned)p.rows_per_group) * p.cols, lane, p.cols);      // (rows <= 2^31)
    else row_fill<T, V, C, LANES>(r.g, 1.f);
  };
  const long long step = (long long)gridDim.x * RG;
  In in_now, in_next;
  if (AHEAD) fetch(in_now, (long long)blockIdx.x * RG + rg);
  for (long long r0 = (long long)blockIdx.x * RG; r0 < p.rows; r0 += step) {
    const bool live = r0 + rg < p.rows;
    const long long row = live ? r0 + rg : p.rows - 1, at = row * p.cols;
    if (!AHEAD) fetch(in_now, row);
    else if (r0 + step < p.rows) fetch(in_next, r0 + step + rg);
    float v[EPL], mean1 = 0.f, rstd1 = 0.f, mean2, rstd2;
    if (p.h != nullptr) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) v[e] = (float)in_now.h.p[e / V].v[e % V];
      moments(v, mean1, rstd1);
      if (!AHEAD) vectors_post();
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const int c = e / V, k = e % V;
        const float n = fmaf((v[e] - mean1) * rstd1, (float)ow.p[c].v[k], (float)ob.p[c].v[k]);
        v[e] = in[c] ? fmaf((float)scale.p[c].v[k] * (float)in_now.g.p[c].v[k], n, (float)in_now.x.p[c].v[k]) : 0.f;
      }
      if (live) row_store<T, V, C, LANES>(p.x_out, at, v, lane, p.cols);
    } else {
#pragma unroll
      for (int e = 0; e < EPL; ++e) v[e] = (float)in_now.x.p[e / V].v[e % V];
    }
    moments(v, mean2, rstd2);
    if (!AHEAD) vectors_pre();
#pragma unroll
    for (int e = 0; e < EPL; ++e) v[e] = fmaf((v[e] - mean2) * rstd2, (float)pw.p[e / V].v[e % V], (float)pb.p[e / V].v[e % V]);
    if (live) {
      row_store<T, V, C, LANES>(p.u, at, v, lane, p.cols);
      if (p.stats != nullptr && lane == 0) *reinterpret_cast<float4*>(p.stats + row * 4) = make_float4(mean1, rstd1, mean2, rstd2);
    }
    if (AHEAD) { row_copy(in_now.x, in_next.x); row_copy(in_now.h, in_next.h); row_copy(in_now.g, in_next.g); }
  }
}

// One block a chunk: rows_per_chunk consecutive rows of one gate group, or (WALK) of many whole groups.  BIAS: a bias learns too (two
// more sums a column).
template <typename T, int LANES, int EPL, bool VEC, bool BIAS, bool WALK>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void rnorm_bwd_kernel(RNormParams p) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1, C = EPL / V;
  constexpr int RG = LANES > 256 ? 1 : 256 / LANES;        // rows a block works on
  __shared__ float red[64];
  __shared__ float comb[RG > 1 ? RG * LANES * EPL : 1];
  const int lane = threadIdx.x % LANES, rg = threadIdx.x / LANES;
  RowSum<LANES> row_sum(red);
  const float inv = 1.f / (float)p.cols;
  const bool post = p.h != nullptr;

  // The vectors are kept as fp32 and scale times a grouped gate as one (unpacked for every row they were a fifth of the arithmetic, and
  // with two waves a SIMD that counts: 16384x1024 fp32 73 us, so 66; bf16 49, 47.5).  A block of 16 waves has 128 registers a lane: there they are read
  // again for each row (from the L2), the next row is not fetched ahead and the column sums stay in LDS, or registers would be
  // spilled (8192 columns, 4096 rows, bf16: 411 us, so 101).
  constexpr bool AHEAD = LANES < 1024;
  float sg[EPL], ow[EPL], ob[EPL], pw[EPL];
  auto vector = [&](float (&v)[EPL], const void* q, float otherwise) {
    RowRaw<T, V, C> r;
    row_param<T, V, C, LANES>(r, q, otherwise, lane, p.cols);
#pragma unroll
    for (int e = 0; e < EPL; ++e) v[e] = (float)r.p[e / V].v[e % V];
  };
  bool in[C];
#pragma unroll
  for (int c = 0; c < C; ++c) in[c] = (c * LANES + lane) * V < p.cols;

  const long long group = blockIdx.x / p.chunks_per_group, piece = blockIdx.x - group * p.chunks_per_group;
  const long long first = group * p.rows_per_group + piece * p.rows_per_chunk;
  const long long last = min(first + p.rows_per_chunk, (group + 1) * p.rows_per_group);     // one past
  const bool full_gate = p.gate != nullptr && p.rows_per_group == 1;
  const bool row_gate = full_gate || WALK;       // the gate is read with its row
  auto vectors_post = [&] {
    vector(sg, p.scale, 1.f); vector(ow, p.post_w, 1.f); vector(ob, p.post_b, 0.f);
    if (p.gate != nullptr && !row_gate) {
      float g[EPL];
      vector(g, static_cast<const T*>(p.gate) + group * p.cols, 1.f);
#pragma unroll
      for (int e = 0; e < EPL; ++e) sg[e] *= g[e];
    }
  };
  if (AHEAD) { vectors_post(); vector(pw, p.pre_w, 1.f); }

  // the column sums of the block's rows; a lane's own, the first HELD of them in LDS
  enum { GATE, POST_W, PRE_W, POST_B, PRE_B };
  constexpr int SUMS = BIAS ? 5 : 3, HELD = AHEAD ? 0 : EPL > 8 ? 2 : BIAS ? 4 : 3;
  __shared__ float held[HELD > 0 ? HELD * EPL * LANES : 1];
  float acc[SUMS][EPL];
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      if (k < HELD) held[(k * EPL + e) * LANES + lane] = 0.f;
      else acc[k][e] = 0.f;
    }
  auto add = [&](int k, int e, float x, float y) {
    float& a = k < HELD ? held[(k * EPL + e) * LANES + lane] : acc[k][e];
    a = fmaf(x, y, a);
  };

  // (a gate per element: the chunks of one row each would leave as many partial rows as there are rows, so there the host
  // hands out chunks of several "groups" and the gate is read with its row; where groups of few rows are many (walk), so too, and
  // each of the block's row lanes takes every RG'th group from its first row to its last: the group's gate gradient is then whole in its
  // registers, and is written there and then)
  const long long c_first = row_gate ? blockIdx.x * p.rows_per_chunk : first;
  const long long c_last = row_gate ? min(c_first + p.rows_per_chunk, p.rows) : last;
  const int t = (int)p.rows_per_group;             // (WALK: at most rows_per_chunk)
  // WALK: this lane's columns of dscale's sum over the groups behind it (its own words: no one else reads or writes them)
  float* const dscale_at = p.part + (long long)gridDim.x * 5 * p.cols + ((long long)blockIdx.x * RG + rg) * p.cols;
  const bool dscale_sum = WALK && p.dscale != nullptr;
  auto each_column = [&](auto f) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (in[c]) f(c * V + e, (c * LANES + lane) * V + e);
  };
  if (dscale_sum) each_column([&](int, int col) { dscale_at[col] = 0.f; });
  struct In { RowRaw<T, V, C> x, h, dout, du, g; float4 st; };
  auto fetch = [&](In& r, long long row) {
    row = min(row, c_last - 1);
    const long long at = row * p.cols;
    row_load<T, V, C, LANES>(r.x, p.x, at, lane, p.cols);
    if (post) row_load<T, V, C, LANES>(r.h, p.h, at, lane, p.cols);
    if (p.dx_out != nullptr) row_load<T, V, C, LANES>(r.dout, p.dx_out, at, lane, p.cols);
    else row_fill<T, V, C, LANES>(r.dout, 0.f);
    if (p.du != nullptr) row_load<T, V, C, LANES>(r.du, p.du, at, lane, p.cols);
    else row_fill<T, V, C, LANES>(r.du, 0.f);
    if (row_gate) row_load<T, V, C, LANES>(r.g, p.gate, full_gate ? at : (long long)((unsigned)row / (unsigned)t) * p.cols, lane, p.cols);      // (rows <= 2^31)
    r.st = *reinterpret_cast<const float4*>(p.stats + row * 4);
  };
  In in_now, in_next;
  // WALK: a turn's row of this row lane, and its place in its group.  Every row lane takes as many turns as the first, which has the most
  // rows: the sums hold barriers.
  constexpr int STEP = WALK ? 1 : RG;
  const long long from = WALK ? 0 : c_first, to = WALK ? ((c_last - c_first) / t + RG - 1) / RG * t : c_last;
  long long walk_row = c_first + (long long)rg * t;
  int in_group = 0;
  if (AHEAD && c_first < c_last) fetch(in_now, WALK ? walk_row : c_first + rg);
  for (long long r0 = from; r0 < to; r0 += STEP) {
    const long long own = WALK ? walk_row : r0 + rg;
    const bool live = own < c_last, group_ends = WALK && in_group == t - 1;
    const long long row = live ? own : c_last - 1, at = row * p.cols;
    if (WALK) { walk_row += group_ends ? 1 + (RG - 1ll) * t : 1; in_group = group_ends ? 0 : in_group + 1; }
    if (!AHEAD) { fetch(in_now, own); vectors_post(); vector(pw, p.pre_w, 1.f); }
    else if (r0 + STEP < to) fetch(in_next, WALK ? walk_row : r0 + RG + rg);          // (as in the forward kernel)
    const RowRaw<T, V, C>&xr = in_now.x, &hr = in_now.h, &dor = in_now.dout, &dur = in_now.du, &gr = in_now.g;
    const float4 st = in_now.st;
    // (behind the row's end x, h and the gradients are zeros: with a zero for 1 / deviation there, so is all that follows)
    float rstd1[C], rstd2[C];
#pragma unroll
    for (int c = 0; c < C; ++c) { rstd1[c] = in[c] ? st.y : 0.f; rstd2[c] = in[c] ? st.w : 0.f; }
    // scale times the gate of this row
    auto weight = [&](int e) { return row_gate ? sg[e] * (float)gr.p[e / V].v[e % V] : sg[e]; };
    float xh[EPL], rh[EPL], d[EPL];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const int c = e / V, k = e % V;
      float out = (float)xr.p[c].v[k];
      xh[e] = 0.f;
      if (post) {
        xh[e] = ((float)hr.p[c].v[k] - st.x) * rstd1[c];
        out = fmaf(weight(e), fmaf(xh[e], ow[e], ob[e]), out);
      }
      rh[e] = (out - st.z) * rstd2[c];
      const float du = (float)dur.p[c].v[k];
      if (live) {
        add(PRE_W, e, du, rh[e]);
        if (BIAS) add(PRE_B, e, du, 1.f);
      }
      d[e] = du * pw[e];
      s1 += d[e]; s2 = fmaf(d[e], rh[e], s2);
    }
    float2 m = row_sum(s1, s2);
    m.x = p.layer ? m.x * inv : 0.f; m.y *= inv;
    s1 = s2 = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) d[e] = fmaf(rstd2[e / V], d[e] - fmaf(rh[e], m.y, m.x), (float)dor.p[e / V].v[e % V]);      // D
    if (live && p.dx != nullptr) row_store<T, V, C, LANES>(p.dx, at, d, lane, p.cols);
    if (post) {
      if (!AHEAD) vectors_post();
      if (live && full_gate && p.dgate != nullptr) {
        float dg[EPL];
#pragma unroll
        for (int e = 0; e < EPL; ++e) dg[e] = d[e] * sg[e] * fmaf(xh[e], ow[e], ob[e]);
        row_store<T, V, C, LANES>(p.dgate, at, dg, lane, p.cols);
      }
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float n = fmaf(xh[e], ow[e], ob[e]), dn = d[e] * weight(e);
        if (live) {
          if (full_gate) add(GATE, e, d[e] * n, (float)gr.p[e / V].v[e % V]);
          else add(GATE, e, d[e], n);
          add(POST_W, e, dn, xh[e]);
          if (BIAS) add(POST_B, e, dn, 1.f);
        }
        d[e] = dn * ow[e];
        s1 += d[e]; s2 = fmaf(d[e], xh[e], s2);
      }
      if (live && group_ends) {       // the group is done: its dgate, and its part of dscale
        float sum[EPL], dg[EPL];
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          float& a = GATE < HELD ? held[(GATE * EPL + e) * LANES + lane] : acc[GATE][e];
          sum[e] = a; a = 0.f;
          dg[e] = sum[e] * sg[e];
        }
        if (p.dgate != nullptr) row_store<T, V, C, LANES>(p.dgate, (long long)((unsigned)row / (unsigned)t) * p.cols, dg, lane, p.cols);
        if (dscale_sum) each_column([&](int e, int col) { dscale_at[col] = fmaf(sum[e], (float)gr.p[e / V].v[e % V], dscale_at[col]); });
      }
      m = row_sum(s1, s2);
      m.x = p.layer ? m.x * inv : 0.f; m.y *= inv;
#pragma unroll
      for (int e = 0; e < EPL; ++e) d[e] = st.y * (d[e] - fmaf(xh[e], m.y, m.x));
      if (live && p.dh != nullptr) row_store<T, V, C, LANES>(p.dh, at, d, lane, p.cols);
    }
    if (AHEAD) {
      row_copy(in_now.x, in_next.x); row_copy(in_now.h, in_next.h); row_copy(in_now.dout, in_next.dout);
      row_copy(in_now.du, in_next.du); row_copy(in_now.g, in_next.g);
      in_now.st = in_next.st;
    }
  }

  float* part = p.part + (long long)blockIdx.x * 5 * p.cols;
  auto flush = [&](int sum, int k) {
    float a[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) a[e] = sum < HELD ? held[(sum * EPL + e) * LANES + lane] : acc[sum][e];
    if (WALK && sum == GATE) each_column([&](int e, int col) { a[e] = dscale_at[col]; });
    if (RG > 1) {                      // the block's row groups, added in order
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EPL; ++e) comb[(rg * LANES + lane) * EPL + e] = a[e];
      __syncthreads();
      if (rg != 0) return;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        a[e] = 0.f;
        for (int g = 0; g < RG; ++g) a[e] += comb[(g * LANES + lane) * EPL + e];
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * LANES + lane) * V;
      if (col < p.cols)
#pragma unroll
        for (int e = 0; e < V; ++e) part[(long long)k * p.cols + col + e] = a[c * V + e];
    }
  };
  if (p.dscale != nullptr || (p.dgate != nullptr && !row_gate)) flush(GATE, 0);
  if (p.dpost_w != nullptr) flush(POST_W, 1);
  if constexpr (BIAS) if (p.dpost_b != nullptr) flush(POST_B, 2);
  if (p.dpre_w != nullptr) flush(PRE_W, 3);
  if constexpr (BIAS) if (p.dpre_b != nullptr) flush(PRE_B, 4);
}

// Column sums of the partial rows, 64 columns and 16 row lanes a block.  blockIdx.y 0: dscale (each chunk's sum times its group's
// gate), 1 to 4: the vectors, 5 on: the gate rows of a grouped gate.
template <typename T>
__global__ __launch_bounds__(1024) void rnorm_sums_kernel(RNormParams p, long long chunks) {
  __shared__ float s[16][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const int col = blockIdx.x * 64 + tx, lc = min(col, p.cols - 1);
  const bool grouped = p.gate != nullptr && p.rows_per_group > 1 && !p.walk;
  const T* gate = static_cast<const T*>(p.gate);
  auto column = [&](int k, long long from, long long to, bool weigh) -> float {       // valid in row lane 0
    float a = 0.f;
    const float* part = p.part + (long long)k * p.cols + lc;
#pragma unroll 8
    for (long long c = from + ty; c < to; c += 16) {
      const float v = part[c * 5 * p.cols];
      a = weigh ? fmaf(v, (float)gate[c / p.chunks_per_group * p.cols + lc], a) : a + v;
    }
    __syncthreads();
    s[ty][tx] = a;
    __syncthreads();
    a = 0.f;
    if (ty == 0)
#pragma unroll
      for (int i = 0; i < 16; ++i) a += s[i][tx];
    return a;
  };
  if (blockIdx.y >= 5) {
    const float sc = p.scale != nullptr ? (float)static_cast<const T*>(p.scale)[lc] : 1.f;
    for (long long g = blockIdx.y - 5; g < p.groups; g += gridDim.y - 5) {
      const float a = column(0, g * p.chunks_per_group, (g + 1) * p.chunks_per_group, false);
      if (ty == 0 && col < p.cols) static_cast<T*>(p.dgate)[g * p.cols + col] = (T)(a * sc);
    }
    return;
  }
  void* const outs[5] = {p.dscale, p.dpost_w, p.dpost_b, p.dpre_w, p.dpre_b};
  T* out = static_cast<T*>(outs[blockIdx.y]);
  if (out == nullptr) return;
  const float a = column(blockIdx.y, 0, chunks, blockIdx.y == 0 && grouped);
  if (ty == 0 && col < p.cols) out[col] = (T)a;
}

// lanes a row: the fewest that hold it at 8 elements each, from 8 to 16 waves (65536 rows of 64 columns, fp32: 64 lanes a row 34 us
// forward and 63 backward, 8 lanes 12 and 37; of 128: 35 and 63, 16 lanes 21 and 38); wider rows take 16 elements a lane, and some
// spilled registers (16384 columns, 2048 rows, bf16: 117 and 437 us, 2.3 and 0.9 TB/s).  GO(lanes, elements)
#define RNORM_BY_WIDTH(GO)                                                                              \
  do {                                                                                                  \
    if (p.cols <= 64) { GO(8, 8); } else if (p.cols <= 128) { GO(16, 8); } else if (p.cols <= 256) { GO(32, 8); }     \
    else if (p.cols <= 512) { GO(64, 8); } else if (p.cols <= 1024) { GO(128, 8); } else if (p.cols <= 2048) { GO(256, 8); } \
    else if (p.cols <= 4096) { GO(512, 8); } else if (p.cols <= 8192) { GO(1024, 8); } else { GO(1024, 16); }           \
  } while (0)
static int rnorm_rows_per_block(int cols) { return cols <= 64 ? 32 : cols <= 128 ? 16 : cols <= 256 ? 8 : cols <= 512 ? 4 : cols <= 1024 ? 2 : 1; }

static bool rnorm_vec(const RNormParams& p, int dtype) {
  if (p.cols % (16 / trunk_elem_bytes(dtype)) != 0) return false;
  for (const void* q : {p.x, p.h, p.gate, p.scale, p.post_w, p.post_b, p.pre_w, p.pre_b, (const void*)p.x_out, (const void*)p.u,
                        p.dx_out, p.du, (const void*)p.dx, (const void*)p.dh, (const void*)p.dgate})
    if (!trunk_aligned16(q)) return false;
  return true;
}

template <typename T>
static int rnorm_fwd_launch(const RNormParams& p, bool vec, hipStream_t st) {
  // (as many blocks as the chip holds at a time: 8192x4096 64 us with 4096, 59 with 1024)
  const int rg = rnorm_rows_per_block(p.cols);
  const unsigned grid = (unsigned)std::min<long long>((p.rows + rg - 1) / rg, 1024);
#define RNORM_FWD_GO(L, E)                                                                                                        \
  if (vec) hipLaunchKernelGGL((rnorm_fwd_kernel<T, L, E, true>), dim3(grid), dim3((L) > 256 ? (L) : 256), 0, st, p);               \
  else hipLaunchKernelGGL((rnorm_fwd_kernel<T, L, E, false>), dim3(grid), dim3((L) > 256 ? (L) : 256), 0, st, p)
  RNORM_BY_WIDTH(RNORM_FWD_GO);
  VEEX_CHECK_LAUNCH();
  return 0;
}

template <typename T>
static int rnorm_bwd_launch(const RNormParams& p, bool vec, long long chunks, hipStream_t st) {
  const dim3 grid((unsigned)chunks);
  const bool bias = p.dpost_b != nullptr || p.dpre_b != nullptr;
#define RNORM_BWD_GO(L, E)                                                                                                        \
  if (p.walk && vec) hipLaunchKernelGGL((rnorm_bwd_kernel<T, L, E, true, true, true>), grid, dim3((L) > 256 ? (L) : 256), 0, st, p);  \
  else if (p.walk) hipLaunchKernelGGL((rnorm_bwd_kernel<T, L, E, false, true, true>), grid, dim3((L) > 256 ? (L) : 256), 0, st, p);   \
  else if (vec && bias) hipLaunchKernelGGL((rnorm_bwd_kernel<T, L, E, true, true, false>), grid, dim3((L) > 256 ? (L) : 256), 0, st, p);       \
  else if (vec) hipLaunchKernelGGL((rnorm_bwd_kernel<T, L, E, true, false, false>), grid, dim3((L) > 256 ? (L) : 256), 0, st, p);         \
  else if (bias) hipLaunchKernelGGL((rnorm_bwd_kernel<T, L, E, false, true, false>), grid, dim3((L) > 256 ? (L) : 256), 0, st, p);        \
  else hipLaunchKernelGGL((rnorm_bwd_kernel<T, L, E, false, false, false>), grid, dim3((L) > 256 ? (L) : 256), 0, st, p)
  RNORM_BY_WIDTH(RNORM_BWD_GO);
  VEEX_CHECK_LAUNCH();
  if (p.dgate != nullptr || p.dscale != nullptr || p.dpost_w != nullptr || p.dpost_b != nullptr || p.dpre_w != nullptr || p.dpre_b != nullptr) {
    const long long gate_rows = p.dgate != nullptr && p.rows_per_group > 1 && !p.walk ? std::min<long long>(p.groups, 1024) : 0;
    hipLaunchKernelGGL((rnorm_sums_kernel<T>), dim3((p.cols + 63) / 64, (unsigned)(5 + gate_rows)), dim3(1024), 0, st, p, chunks);
    VEEX_CHECK_LAUNCH();
  }
  return 0;
}

// How the backward pass hands its rows out: about as many chunks as the chip holds blocks, none across a group's end.  Groups that are
// many and small would leave a chunk each, and with it five partial rows to keep and to add (131072 rows of 1024 in 65536 groups: 1.3 GB
// and 3.2 ms): there (walk) a chunk is a run of whole groups, RG of them at a time, one for each of the block's row lanes.  That takes
// RG t rows a chunk, so it serves while they are not far more than a block's share (bf16 us, a chunk a group and walking: 131072x1024 in 65536
// groups 3181 and 422, in 8192 664 and 333, 2080x1024 in 1040 57 and 21, 16384x8192 in 4096 1538 and 535; at twice the share, 65536x128 in 4096,
// 142 and 40; at four times 65536x64 in 4096 146 and 36, 524288x64 in 4096 209 and 246, fp32 352 and 283; at eight times 524288x64 in 2048 152 and
// 465).  So there are at most 512 (RG / 4 + 1) partial rows, whatever the groups.
struct RNormPlan { long long chunks, rows_per_chunk, chunks_per_group; int walk; };

static RNormPlan rnorm_plan(long long rows, int cols, long long groups) {
  const long long t = rows / groups, blocks = cols > 2048 ? 256 : 512;       // (resident at once: 8 waves a CU)
  const int rg = rnorm_rows_per_block(cols);
  const long long want = std::max<long long>((rows + blocks - 1) / blocks, std::max(4, rg));
  if (groups == rows) return {(rows + want - 1) / want, want, 1, 0};          // (a gate per element, or one row)
  const long long per_group = (t + want - 1) / want, per_chunk = (t + per_group - 1) / per_group, of_group = (t + per_chunk - 1) / per_chunk;
  if (of_group * groups <= 2 * blocks || t * rg > 4 * want) return {of_group * groups, per_chunk, of_group, 0};
  const long long run = ((want + t - 1) / t + rg - 1) / rg * rg;              // groups of a chunk
  return {(groups + run - 1) / run, run * t, 1, 1};
}

static long long rnorm_workspace(const RNormPlan& q, int cols) { return q.chunks * (5 + (q.walk ? rnorm_rows_per_block(cols) : 0)) * cols; }

static bool rnorm_struct_ok(const VeexResidualNorm* d) {
  if (d != nullptr && (d->struct_size == 0 || d->struct_size == (int)sizeof(VeexResidualNorm))) return true;
  veex_set_error("residual_norm: struct_size is not this library's");
  return false;
}

static int rnorm_check(const char* who, long long rows, int cols, long long groups, int dtype, int kind, double eps, bool train) {
  if (!trunk_dtype_ok(dtype) || (kind != VEEX_NORM_LAYER && kind != VEEX_NORM_RMS)) { veex_set_error("%s: unknown dtype or kind", who); return VEEX_EINVAL; }
  if (rows < 0 || cols < 1 || cols > VEEX_NORM_MAX_COLS) { veex_set_error("%s: rows >= 0 and 1 <= cols <= %d are needed", who, VEEX_NORM_MAX_COLS); return VEEX_EINVAL; }
  if (rows > (1ll << 31)) { veex_set_error("%s: at most 2^31 rows", who); return VEEX_EINVAL; }
  if (groups < 1 || (rows > 0 && rows % groups != 0)) { veex_set_error("%s: the gate's groups have to divide the rows", who); return VEEX_EINVAL; }
  if (train && groups != rows && groups >= VEEX_NORM_MAX_GROUPS) { veex_set_error("%s: in training a gate has fewer than 2^22 groups, or one a row", who); return VEEX_EINVAL; }
  if (!(eps >= 0.0)) { veex_set_error("%s: eps has to be >= 0", who); return VEEX_EINVAL; }
  return 0;
}

static void rnorm_fill(RNormParams& p, const VeexResidualNorm* d) {
  p.x = d->x; p.h = d->h; p.gate = d->h != nullptr ? d->gate : nullptr; p.scale = d->scale;
  p.post_w = d->post_w; p.post_b = d->post_b; p.pre_w = d->pre_w; p.pre_b = d->pre_b;
  p.x_out = d->x_out; p.u = d->u; p.stats = d->stats;
  p.dx_out = d->dx_out; p.du = d->du; p.dx = d->dx;
  const bool post = d->h != nullptr;               // (without h nothing depends on the block's side)
  p.dh = post ? d->dh : nullptr; p.dgate = p.gate != nullptr ? d->dgate : nullptr; p.dscale = post ? d->dscale : nullptr;
  p.dpost_w = post ? d->dpost_w : nullptr; p.dpost_b = post ? d->dpost_b : nullptr; p.dpre_w = d->dpre_w; p.dpre_b = d->dpre_b;
  p.part = d->workspace;
  p.rows = d->rows; p.cols = d->cols; p.layer = d->kind == VEEX_NORM_LAYER; p.eps = d->eps;
  p.groups = p.gate != nullptr ? d->groups : 1;
  p.rows_per_group = std::max<long long>(d->rows / p.groups, 1);
  p.rows_per_chunk = p.chunks_per_group = 1; p.walk = 0;
}

extern "C" {

int veex_residual_norm_fwd(const VeexResidualNorm* d, hipStream_t st) {
  if (!rnorm_struct_ok(d)) return VEEX_EINVAL;
  if (d->x == nullptr || d->u == nullptr || (d->h != nullptr && d->x_out == nullptr)) {
    veex_set_error("residual_norm: x and u (with h also x_out) are needed"); return VEEX_EINVAL;
  }
  if (!trunk_aligned16(d->stats)) { veex_set_error("residual_norm: stats has to be 16-byte aligned"); return VEEX_EINVAL; }
  if (int rc = rnorm_check("residual_norm", d->rows, d->cols, d->gate != nullptr ? d->groups : 1, d->dtype, d->kind, d->eps, d->stats != nullptr)) return rc;
  if (d->rows == 0) return 0;
  RNormParams p;
  rnorm_fill(p, d);
  p.dx_out = p.du = nullptr; p.dx = p.dh = p.dgate = nullptr;
  const bool vec = rnorm_vec(p, d->dtype);
  if (d->dtype == VEEX_T_F32) return rnorm_fwd_launch<float>(p, vec, st);
  if (d->dtype == VEEX_T_BF16) return rnorm_fwd_launch<bf16_t>(p, vec, st);
  return rnorm_fwd_launch<f16_t>(p, vec, st);
}

long long veex_residual_norm_bwd_workspace_floats(long long rows, int cols, long long groups) {
  if (rows < 0 || cols < 1 || groups < 1 || (rows > 0 && rows % groups != 0)) return -1;
  if (rows == 0) return 0;
  return rnorm_workspace(rnorm_plan(rows, cols, groups), cols);
}

int veex_residual_norm_bwd(const VeexResidualNorm* d, hipStream_t st) {
  if (!rnorm_struct_ok(d)) return VEEX_EINVAL;
  if (d->x == nullptr || d->stats == nullptr || !trunk_aligned16(d->stats) || d->workspace == nullptr) {
    veex_set_error("residual_norm backward: x, 16-byte aligned stats and workspace are needed"); return VEEX_EINVAL;
  }
  if (int rc = rnorm_check("residual_norm backward", d->rows, d->cols, d->gate != nullptr ? d->groups : 1, d->dtype, d->kind, d->eps, true)) return rc;
  if (d->rows == 0) { veex_set_error("residual_norm backward: no rows"); return VEEX_EINVAL; }
  RNormParams p;
  rnorm_fill(p, d);
  p.x_out = p.u = nullptr;
  const RNormPlan plan = rnorm_plan(p.rows, p.cols, p.groups);
  const long long chunks = plan.chunks, need = rnorm_workspace(plan, p.cols);
  p.rows_per_chunk = plan.rows_per_chunk; p.chunks_per_group = plan.chunks_per_group; p.walk = plan.walk;
  if (d->workspace_floats < need) { veex_set_error("residual_norm backward: workspace of %lld floats is needed", need); return VEEX_ENOMEM; }
  const bool vec = rnorm_vec(p, d->dtype);
  if (d->dtype == VEEX_T_F32) return rnorm_bwd_launch<float>(p, vec, chunks, st);
  if (d->dtype == VEEX_T_BF16) return rnorm_bwd_launch<bf16_t>(p, vec, chunks, st);
  return rnorm_bwd_launch<f16_t>(p, vec, chunks, st);
}

}  // extern "C"
