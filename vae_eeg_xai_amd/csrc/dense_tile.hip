// Large Dense products on the bf16 / fp16 matrix cores:  C[i][j] = sum_k A(i, k) B(k, j), fp32 accumulate, the epilogue of
// dense_common.h on the way out.  PL = 1: 16-bit tensors.  PL = 3: fp32 tensors, split beforehand into three bf16 terms
// (a = a1 + a2 + a3 to 2^-27, dense_pack_kernel); a product is the six partial products a1b1, a1b2, a2b1, a1b3, a2b2, a3b1, smallest
// first; what is left out is below 2^-25 of |a b|.
//
// A tile of BM x BN is computed by WM x WN waves, BK of the reduction at a time.  Operands go from memory straight into LDS
// (16 bytes a lane, no registers in between) into the buffer that the step before has finished with, while the MFMAs of
// this step read the other one: one barrier a step.  An operand whose k index is contiguous lies in LDS as [row][BK] and is
// read as the MFMA wants it, 8 consecutive k a lane; one whose row index is contiguous lies as [k][128 rows] and is
// read through the transposing LDS read.  The load writes LDS in lane order, so the bank swizzle is applied to the address
// that a lane loads from: 16-byte piece q of an LDS row holds the tensor's piece q ^ s(row).
//   [row][64]: s = (row >> 1) & 7;  [row][32]: s = (row >> 2) & 3;  [k][128]: s = (k & 3) << 2
// (16 lanes read at a time, 256 bytes: 16 consecutive rows of one piece have to fall on 16 different ones)
//
// Bound: matrix cores and the chip's power: 4096^3 bf16 runs at 1 120 TFLOP/s, 8192x4096x4096 at 1 190, with the matrix cores busy 55 %
// of the cycles and the clock down to 1.9 GHz (library: 1 116 at 8192^3, 1 340 at 8192x4096x4096); fp32 at 190 to 200 (library 153).
// Short reductions pay for the epilogue, which nothing overlaps (one tile a CU): 8192x1024x4096 bf16 77 us, with gelu 92, with z
// kept as well 96 to 105; 8192x4096x1024 70.  Two tiles a CU of half the size overlap it but gather twice the operands: 88 to 130 us.
// 256x256 by 4 waves of 128x128, with a third fewer LDS reads: 107 us for 92, one wave a SIMD hides nothing.
//
// Needs: 16-byte aligned operands and rows; a k-contiguous operand's K a multiple of 8.  Pieces past a tensor's end
// are sent out of the buffer's range and arrive as zeros.
#include "dense_tile.h"
#include <algorithm>

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float dt_f4 __attribute__((ext_vector_type(4)));
typedef unsigned dt_u4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
#define DT_LDS __attribute__((address_space(3)))
#define DT_OOB 0xFFFFFFF0u      // past every buffer's end

__device__ __forceinline__ f32x16 dt_mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 dt_mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
template <typename T> struct DtVec;
template <> struct DtVec<bf16_t> { typedef bf16x8 x8; };
template <> struct DtVec<f16_t> { typedef f16x8 x8; };

// One operand's ROWS x BK tiles (ROWS a multiple of 128 where the row index is contiguous)
template <int ROWS, int BK, bool KC, int PL, int WAVES>
struct DtOperand {
  static constexpr int BYTES = ROWS * BK * 2;                  // of a plane's tile
  static constexpr int LOADS = BYTES / 1024 / WAVES;           // 1024-byte loads of a wave, per plane
  static_assert(BYTES % (1024 * WAVES) == 0, "whole loads for every wave");
  static_assert(KC ? (BK == 64 || BK == 32) : ROWS % 128 == 0, "layouts with a swizzle");
  static constexpr int COUNT = PL * LOADS;                     // loads of a wave, a stage
  static constexpr int ROWB = BK * 2;

  const char* base;                // (row0, k = 0) of plane 0
  long long ld, plane;             // bytes between rows (KC) or k's (not KC); between planes
  long long K, rows_left;          // rows_left: rows from row0 on
  unsigned voff[LOADS], piece_k[LOADS];
  int wave, lane;

  __device__ __forceinline__ static int swz(int row) { return BK == 64 ? (row >> 1) & 7 : (row >> 2) & 3; }

  __device__ __forceinline__ void init(const DtTensor& t, long long row0, long long rows, long long K_, int wave_, int lane_) {
    wave = wave_; lane = lane_; ld = t.ld_bytes; plane = t.plane_bytes; K = K_; rows_left = rows - row0;
    base = static_cast<const char*>(t.p) + (KC ? row0 * ld : row0 * 2);
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int at = (u * WAVES + wave) * 1024 + lane * 16;    // byte of the LDS tile that this lane fills
      if (KC) {
        const int row = at / ROWB, q = (at % ROWB) / 16, piece = q ^ swz(row);
        piece_k[u] = piece * 8;
        voff[u] = row < rows_left ? (unsigned)(row * ld) + piece * 16 : DT_OOB;
      } else {
        const int sub = at / (BK * 256), in = at % (BK * 256), k = in / 256, q = (in % 256) / 16, piece = q ^ ((k & 3) << 2);
        const int row = sub * 128 + piece * 8;
        piece_k[u] = k;
        voff[u] = row < rows_left ? (unsigned)(k * ld) + row * 2 : DT_OOB;
      }
    }
  }

  // load c (of COUNT) of the tile that holds the BK reduction indices from k0 on (those at or past k_end arrive as zeros)
  __device__ __forceinline__ void load(int c, DT_LDS char* lds, long long k0, long long k_end) const {
    const int pl = c / LOADS, u = c % LOADS;
    const uint64_t at = reinterpret_cast<uint64_t>(base + pl * plane + (KC ? k0 * 2 : k0 * ld));
    const dt_u4 r = {(unsigned)at, (unsigned)(at >> 32) & 0xFFFFu, 0xFFFFFFE0u, 0x00020000u};
    const unsigned v = k0 + piece_k[u] < k_end ? voff[u] : DT_OOB;
    // (asm: the compiler's own load into LDS makes it wait for that load before the next LDS read of whatever buffer, which
    // leaves nothing in flight.  No register is written, and m0 only here; the wait is the one before the barrier.)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 : : "s"((unsigned)(uintptr_t)(lds + pl * BYTES + (u * WAVES + wave) * 1024)), "v"(v), "s"(r) : "memory");
  }

  // the 8 k's of lane half lh at k step ks (16 k's), of the 32 rows from `row` on (a multiple of 32)
  template <typename V8>
  __device__ __forceinline__ V8 frag(const DT_LDS char* lds, int pl, int row, int ks) const {
    const int l31 = lane & 31, lh = lane >> 5;
    if (KC) {
      const int r = row + l31, q = (2 * ks + lh) ^ swz(r);
      return *reinterpret_cast<const DT_LDS V8*>(lds + pl * BYTES + r * ROWB + q * 16);
    } else {
      const int g = lane >> 4, tq = (lane & 15) >> 2, tp = lane & 3;
      const int k = ks * 16 + 8 * (g >> 1) + tq, piece = (row & 127) / 8 + 2 * (g & 1) + (tp >> 1);
      const DT_LDS char* a = lds + pl * BYTES + (row >> 7) * (BK * 256) + k * 256 + 16 * (piece ^ ((k & 3) << 2)) + 8 * (tp & 1);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DT_LDS s16x4*)a);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DT_LDS s16x4*)(a + 4 * 256));     // four k's on: the same swizzle
      return __builtin_bit_cast(V8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// block -> (tile row, tile column, split): blocks go round the 8 XCDs in turn, so each XCD takes a contiguous run of tiles,
// walked in bands of 8 tile rows: the tiles that one L2 holds at a time share 8 strips of A and a few of B
__device__ __forceinline__ void dt_tile_of(unsigned b, unsigned ti, unsigned tj, unsigned splits, unsigned& i, unsigned& j, unsigned& z) {
  const unsigned total = ti * tj * splits, per = total / 8, extra = total % 8;
  const unsigned x = b % 8, s = b / 8;
  unsigned t = x * per + min(x, extra) + s;
  z = t / (ti * tj); t -= z * (ti * tj);
  const unsigned band = t / (8 * tj), in = t - band * 8 * tj, h = min(8u, ti - band * 8);
  j = in / h; i = band * 8 + in - j * h;
}

// LDS written and read by different lanes of one wave: the wave's LDS accesses complete in order, so only the compiler has to keep them so
__device__ __forceinline__ void dt_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// the 32 rows from `row` on that a tensor of `rows` has, as bits
__device__ __forceinline__ unsigned dt_rows_in(long long row, long long rows) {
  return rows - row >= 32 ? ~0u : rows <= row ? 0u : (1u << (rows - row)) - 1u;
}

// Which of the 32 rows of a packed operand from `row` on hold a NaN among the k's of [k_begin, k_end): a bit each, the same in every lane.
// (The first plane says it: a value that is not finite is its first term alone.  Rows and k's lie in pieces of 8, padded with zeros.)
template <bool KC>
__device__ __forceinline__ unsigned dt_nan_rows(const DtTensor& t, long long row, long long rows, long long k_begin, long long k_end, int lane) {
  const long long own = KC ? row + (lane & 31) : row + 8 * (lane & 3);
  const int step = 16, k0 = KC ? 8 * (lane >> 5) : lane >> 2;       // 16 k's a turn
  const char* p = static_cast<const char*>(t.p) + (KC ? own * t.ld_bytes : own * 2);
  const unsigned all = dt_rows_in(row, rows);
  unsigned found = 0u;
  for (long long k = k_begin; k < k_end && (found & all) != all; k += 4 * step) {
    unsigned mine = 0u;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const long long at = k + q * step + k0;
      if (own < rows && at < k_end) {
        const Piece<bf16_t, 8> x = piece_load<bf16_t, 8>(reinterpret_cast<const bf16_t*>(p + (KC ? at * 2 : at * t.ld_bytes)));
#pragma unroll
        for (int e = 0; e < 8; ++e) mine |= (float)x.v[e] != (float)x.v[e] ? 1u << (KC ? 0 : e) : 0u;
      }
    }
    if (KC) {
      const unsigned long long b = __ballot(mine != 0u);
      found |= (unsigned)b | (unsigned)(b >> 32);
    } else {
#pragma unroll
      for (int o = 4; o < 64; o <<= 1) mine |= __shfl_xor(mine, o);
#pragma unroll
      for (int q = 0; q < 4; ++q) found |= __shfl(mine, q) << (8 * q);
    }
  }
  return found;
}

// Split operands and infinities: an infinite operand times the other's lower terms gives NaN where fp32 gives an infinity.  A 32 x 32
// block that holds such a NaN is computed again with the fp32 MFMA from the terms' sums (which are the operands to 2^-27, and exactly them
// where they are not finite), and its NaN elements take those values.  A NaN that its row of A or its column of B explains stays: a run that
// has diverged to NaN looks for them and computes nothing again (4096x1024x1024 forward: x all NaN 59 us for 62 without, w all NaN 94; an infinity
// in each row of x, where all of it is computed again, 418).  Finite data come here only where partial products overflow to opposite
// infinities.
template <bool AKC, bool BKC, int MT, int NT>
__device__ __forceinline__ void dt_mend(const DtGemm& g, f32x16 (&acc)[MT][NT], long long i0, int j0, long long k_begin, long long k_end, int lane) {
  const int l31 = lane & 31, lh = lane >> 5;
  // the terms' sums of the 8 k's from k on, of one row (elements outside read the tensor's first one, so that all loads are on their way at once)
  auto values = [&](const DtTensor& t, bool kc, long long row, bool in, long long k, float (&v)[8]) {
    const bf16_t* const safe = static_cast<const bf16_t*>(t.p);
    const long long ld = t.ld_bytes / 2, plane = t.plane_bytes / 2;
    bf16_t x[3][8];
#pragma unroll
    for (int pl = 0; pl < 3; ++pl) {
      if (kc) {
        const Piece<bf16_t, 8> y = piece_load<bf16_t, 8>(in && k < k_end ? safe + row * ld + k + pl * plane : safe);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[pl][e] = y.v[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[pl][e] = *(in && k + e < k_end ? safe + (k + e) * ld + row + pl * plane : safe);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = in && (kc ? k : k + e) < k_end ? (float)x[0][e] + (float)x[1][e] + (float)x[2][e] : 0.f;
  };
#pragma unroll
  for (int mi = 0; mi < MT; ++mi)
#pragma unroll
    for (int nj = 0; nj < NT; ++nj) {
      // this lane's elements of the block are row i0 + 32 mi + l31, columns j0 + 32 nj + 8 (r / 4) + 4 lh + r % 4
      unsigned nan = 0u;
#pragma unroll
      for (int r = 0; r < 16; ++r) nan |= acc[mi][nj][r] != acc[mi][nj][r] ? 1u << r : 0u;
      if (!__any(nan != 0u)) continue;
      const long long row = i0 + mi * 32, i = row + l31;
      const int col = j0 + nj * 32, j = col + l31;
      const unsigned rows = ~dt_rows_in(row, g.I) | dt_nan_rows<AKC>(g.a, row, g.I, k_begin, k_end, lane);
      if ((rows >> l31 & 1u) != 0u) nan = 0u;
      if (!__any(nan != 0u)) continue;
      const unsigned cols = ~dt_rows_in(col, g.J) | dt_nan_rows<BKC>(g.b, col, g.J, k_begin, k_end, lane);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if ((cols >> (8 * (r / 4) + 4 * lh + r % 4) & 1u) != 0u) nan &= ~(1u << r);
      if (!__any(nan != 0u)) continue;
      f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll 1
      for (long long k = k_begin; k < k_end; k += 16) {      // lane half lh holds the k's k + 8 lh .. + 7
        float av[8], bv[8];
        values(g.a, AKC, i, i < g.I, k + 8 * lh, av);
        values(g.b, BKC, j, j < g.J, k + 8 * lh, bv);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(bv[e], av[e], s, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[mi][nj][r] = (nan >> r & 1u) != 0u ? s[r] : acc[mi][nj][r];
    }
}

// One tile (or one split of it): block number -> its part of C.  GRAD: a gradient, which has no epilogue.
template <typename T, typename M, int PL, bool AKC, bool BKC, bool GRAD, int BM, int BN, int BK, int ST, int WM, int WN>
__device__ __forceinline__ void dt_tile(const DtGemm& g, unsigned block, char* smem_raw) {
  constexpr int WAVES = WM * WN, MT = BM / WM / 32, NT = BN / WN / 32;
  typedef DtOperand<BM, BK, AKC, PL, WAVES> OpA;
  typedef DtOperand<BN, BK, BKC, PL, WAVES> OpB;
  typedef typename DtVec<M>::x8 V8;
  constexpr int STAGE = PL * (OpA::BYTES + OpB::BYTES);
  DT_LDS char* smem = (DT_LDS char*)smem_raw;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / WN, wj = wave % WN;
  unsigned ti, tj, z;
  dt_tile_of(block, g.tiles_i, g.tiles_j, g.splits, ti, tj, z);
  const long long i0 = (long long)ti * BM;
  const int j0 = tj * BN;
  const long long k_begin = z * g.k_per_split, k_end = min(g.K, k_begin + g.k_per_split);

  OpA a; OpB b;
  a.init(g.a, i0, g.I, g.K, wave, lane);
  b.init(g.b, j0, g.J, g.K, wave, lane);
  f32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  // ST stages in a ring: while step t is computed, the loads of the ST - 1 steps behind it are on their way (past the end they
  // fetch nothing, so that the count of loads in flight stays the same)
  constexpr int COUNT = OpA::COUNT + OpB::COUNT, KS = BK / 16, PER = (COUNT + KS - 1) / KS, MF = MT * NT * (PL == 1 ? 1 : 6);
  static_assert(ST >= 2 && KS % 2 == 0, "");
  auto load = [&](int c, int stage, long long k0) {
    if (c < OpA::COUNT) a.load(c, smem + stage * STAGE, k0, k_end);
    else if (c < COUNT) b.load(c - OpA::COUNT, smem + stage * STAGE + PL * OpA::BYTES, k0, k_end);
  };
  V8 av[2][PL][MT], bv[2][PL][NT];
  auto read = [&](int buf, const DT_LDS char* st, int ks) {
#pragma unroll
    for (int pl = 0; pl < PL; ++pl) {
#pragma unroll
      for (int j = 0; j < NT; ++j) bv[buf][pl][j] = b.template frag<V8>(st + PL * OpA::BYTES, pl, (wj * NT + j) * 32, ks);
#pragma unroll
      for (int i = 0; i < MT; ++i) av[buf][pl][i] = a.template frag<V8>(st, pl, (wi * MT + i) * 32, ks);
    }
  };
#pragma unroll
  for (int t = 0; t < ST - 1; ++t)
#pragma unroll
    for (int c = 0; c < COUNT; ++c) load(c, t, k_begin + t * BK);
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"((ST - 2) * COUNT) : "memory");
  read(0, smem, 0);
#pragma unroll
  for (int c = 0; c < PER; ++c) load(c, ST - 1, k_begin + (ST - 1) * BK);
  int cur = 0;
  for (long long k0 = k_begin; k0 < k_end; k0 += BK) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      // the operands of the k step after this one are read before this one's MFMAs are issued; before the first of the next
      // stage: that stage has landed, and every wave has read what it needs of this one, which is loaded again from here on
      int stage; long long at; int c0;
      if (ks < KS - 1) {
        read((ks + 1) & 1, smem + cur * STAGE, ks + 1);
        stage = cur == 0 ? ST - 1 : cur - 1; at = k0 + (ST - 1) * BK; c0 = (ks + 1) * PER;
      } else {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((ST - 2) * COUNT) : "memory");
        stage = cur; at = k0 + ST * BK; c0 = 0;
        cur = cur == ST - 1 ? 0 : cur + 1;
        read(0, smem + cur * STAGE, 0);          // (behind the last step: what is read is not used)
      }
      __builtin_amdgcn_sched_barrier(0);
      // the loads go out one by one between the MFMAs: a wave's instructions issue in order, and a burst of loads holds up
      // everything behind it until the memory path has taken them
#pragma unroll
      for (int m = 0; m < MF; ++m) {
        const int t = m / (MT * NT), i = m % (MT * NT) / NT, j = m % NT;
        constexpr int PA[6] = {2, 1, 0, 1, 0, 0}, PB[6] = {0, 1, 2, 0, 1, 0};       // smallest terms first
        const int pa = PL == 1 ? 0 : PA[t], pb = PL == 1 ? 0 : PB[t];
        acc[i][j] = dt_mfma(bv[ks & 1][pb % PL][j], av[ks & 1][pa % PL][i], acc[i][j]);
#pragma unroll
        for (int c = 0; c < PER; ++c)
          if (m == (c + 1) * MF / (PER + 1)) {
            __builtin_amdgcn_sched_barrier(0);
            load(c0 + c, stage, at);
            __builtin_amdgcn_sched_barrier(0);
          }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  if (PL == 3) dt_mend<AKC, BKC, MT, NT>(g, acc, i0 + wi * MT * 32, j0 + wj * NT * 32, k_begin, k_end, lane);

  // The way out: each wave turns 64 rows at a time round through a corner of LDS of its own (fp32, 16-byte pieces swizzled by the
  // row), so that a lane holds 8 consecutive columns of a row and eight lanes (four for 32 columns) write a whole line.  Straight
  // from the accumulators' layout a store would touch 32 lines.
  constexpr int CW = NT * 32, OCT = CW / 8, RPP = 64 / OCT;      // columns, their blocks of 8, rows a pass
  constexpr int SM = MT < 2 || WAVES * 64 * CW * 4 > ST * STAGE ? 1 : 2;                            // 32-row blocks a strip holds
  static_assert(WAVES * SM * 32 * CW * 4 <= ST * STAGE && MT % SM == 0, "the strips fit the stages");
  // every wave is done with the operand tiles, and no load is on its way into them
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");
  DT_LDS char* strip = smem + wave * SM * 32 * CW * 4;
  const int l31 = lane & 31, lh = lane >> 5;
  const unsigned long long base = GRAD ? 0ull : drop_base(g.epi.drop);
  const int o = lane % OCT, j = j0 + wj * CW + 8 * o;
  float bias[8];
  if (!GRAD && g.slab == nullptr) dense_bias<T>(g.epi, bias, j, g.J, g.vec_e);
#pragma unroll
  for (int m0 = 0; m0 < MT; m0 += SM) {
#pragma unroll
    for (int mi = m0; mi < m0 + SM; ++mi)
#pragma unroll
      for (int nj = 0; nj < NT; ++nj)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<DT_LDS dt_f4*>(strip + ((mi - m0) * 32 + l31) * CW * 4 + (((nj * 8 + 2 * q + lh) ^ (l31 & 7)) * 16)) =
              dt_f4{acc[mi][nj][4 * q], acc[mi][nj][4 * q + 1], acc[mi][nj][4 * q + 2], acc[mi][nj][4 * q + 3]};
    dt_wave_sync();
    const long long ld = g.slab != nullptr ? slab_ld(g.J) : g.J;
    long long i = i0 + (wi * MT + m0) * 32 + lane / OCT, at = i * ld + j;
#pragma unroll 2
    for (int r = lane / OCT; r < 32 * SM; r += RPP, i += RPP, at += RPP * ld) {
      const dt_f4 lo = *reinterpret_cast<DT_LDS dt_f4*>(strip + r * CW * 4 + (((2 * o) ^ (r & 7)) * 16));
      const dt_f4 hi = *reinterpret_cast<DT_LDS dt_f4*>(strip + r * CW * 4 + (((2 * o + 1) ^ (r & 7)) * 16));
      if (i >= g.I || j >= g.J) continue;
      if (g.slab != nullptr) {
        float* s = g.slab + z * g.I * ld + at;
        *reinterpret_cast<dt_f4*>(s) = lo;
        if (j + 4 < g.J) *reinterpret_cast<dt_f4*>(s + 4) = hi;
      } else {
        float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        if (GRAD) {
          grad_scale<T>(v, g.alpha);
          store8<T>(static_cast<T*>(g.epi.y) + at, v, g.J - j, g.vec_e);
        } else {
          unsigned w[4] = {0u, 0u, 0u, 0u};
          if (g.epi.drop.cut != 0u) drop_words(g.epi.drop, base + (unsigned long long)i, (unsigned)j >> 3, w);
          dense_epilogue<T>(g.epi, v, bias, at, g.J - j, g.vec_e, w);
        }
      }
    }
    dt_wave_sync();
  }
}

template <typename T, typename M, int PL, bool AKC, bool BKC, int BM, int BN, int BK, int ST, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void dense_tile_kernel(DtGemm g) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  dt_tile<T, M, PL, AKC, BKC, !(AKC && !BKC), BM, BN, BK, ST, WM, WN>(g, blockIdx.x, smem);
}

// Both gradients in one launch: dx = dz w^T (k contiguous in both), dw = x^T dz (in neither).  A small layer's products leave most of
// the chip idle one after the other.
template <typename T, typename M, int PL, int BM, int BN, int BK, int ST, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void dense_tile_grads_kernel(DtGemm dx, DtGemm dw, unsigned dx_blocks) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  if (blockIdx.x < dx_blocks) dt_tile<T, M, PL, true, true, true, BM, BN, BK, ST, WM, WN>(dx, blockIdx.x, smem);
  else dt_tile<T, M, PL, false, false, true, BM, BN, BK, ST, WM, WN>(dw, blockIdx.x - dx_blocks, smem);
}

// ---------------------------------------------------------------------------------------------------------------
// Packing: rows of a tensor (any row stride and alignment) as 16-byte aligned rows of `cols8` = cols rounded up to 8, zeros behind
// the last column; an fp32 tensor as its three bf16 terms in three planes.  8 columns a thread.
// ---------------------------------------------------------------------------------------------------------------
struct DtPackJobs { DtPack job[3]; unsigned first[4]; int vec[3]; };     // first: a job's first workgroup; the last one's end

template <typename T>
__global__ __launch_bounds__(256) void dense_pack_kernel(DtPackJobs jobs) {
  const int q = blockIdx.x < jobs.first[1] ? 0 : blockIdx.x < jobs.first[2] ? 1 : 2;
  const DtPack& o = jobs.job[q];
  const T* __restrict__ src = static_cast<const T*>(o.src);
  char* __restrict__ dst = static_cast<char*>(o.dst);
  const long long ld = o.ld, plane_bytes = o.plane_bytes;
  const int cols = o.cols, cols8 = (cols + 7) / 8 * 8, bpr = cols8 / 8;
  const bool vec = jobs.vec[q];
  const long long nb = o.rows * bpr, step = (long long)(jobs.first[q + 1] - jobs.first[q]) * 256;
  for (long long t = (long long)(blockIdx.x - jobs.first[q]) * 256 + threadIdx.x; t < nb; t += step) {
    const long long r = nb <= 0xFFFFFFFFll ? (long long)((unsigned)t / (unsigned)bpr) : t / bpr;
    const int c = 8 * (int)(t - r * bpr);
    const T* p = src + r * ld + c;
    constexpr int V = 16 / sizeof(T);
    T x[8];
    if (vec) {
#pragma unroll
      for (int q = 0; q < 8 / V; ++q) {
        const Piece<T, V> y = piece_load<T, V>(p + q * V);
#pragma unroll
        for (int e = 0; e < V; ++e) x[q * V + e] = y.v[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = p[c + e < cols ? e : 0];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = c + e < cols ? x[e] : (T)0.f;
    }
    char* d = dst + (r * cols8 + c) * 2;
    if constexpr (sizeof(T) == 2) {
      Piece<T, 8> y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y.v[e] = x[e];
      piece_store<T, 8>(reinterpret_cast<T*>(d), y);
    } else {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = x[e];
      dt_store_planes(d, plane_bytes, f);
    }
  }
}

int dense_pack_launch(int dtype, const DtPack* jobs, int n, hipStream_t st) {
  if (n == 0) return 0;
  DtPackJobs j = {};
  for (int q = 0; q < 3; ++q) {
    j.first[q + 1] = j.first[q];
    if (q >= n) continue;
    j.job[q] = jobs[q];
    j.vec[q] = jobs[q].cols % 8 == 0 && trunk_aligned16(jobs[q].src) && jobs[q].ld * trunk_elem_bytes(dtype) % 16 == 0;
    j.first[q + 1] += (unsigned)std::min<long long>((jobs[q].rows * ((jobs[q].cols + 7) / 8) + 255) / 256, 1 << 16);
  }
  const dim3 grid(j.first[3]);
  if (dtype == VEEX_T_F32) hipLaunchKernelGGL((dense_pack_kernel<float>), grid, dim3(256), 0, st, j);
  else if (dtype == VEEX_T_BF16) hipLaunchKernelGGL((dense_pack_kernel<bf16_t>), grid, dim3(256), 0, st, j);
  else hipLaunchKernelGGL((dense_pack_kernel<f16_t>), grid, dim3(256), 0, st, j);
  VEEX_CHECK_LAUNCH();
  return 0;
}

// ---------------------------------------------------------------------------------------------------------------
template <typename T, typename M, int PL, bool AKC, bool BKC, int BM, int BN, int BK, int ST, int WM, int WN>
static int dt_go(const DtGemm& gin, hipStream_t st) {
  DtGemm g = gin;
  g.tiles_i = (unsigned)((g.I + BM - 1) / BM); g.tiles_j = (unsigned)((g.J + BN - 1) / BN);
  constexpr int lds = ST * PL * (BM + BN) * BK * 2;
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  const void* fn = reinterpret_cast<const void*>(dense_tile_kernel<T, M, PL, AKC, BKC, BM, BN, BK, ST, WM, WN>);
  // (a function's attribute belongs to the current device: set before each launch, a host-side call of well under a microsecond)
  if (lds > 64 * 1024 && hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
    veex_set_error("dense: cannot raise the dynamic LDS limit"); return VEEX_ELAUNCH;
  }
  hipLaunchKernelGGL((dense_tile_kernel<T, M, PL, AKC, BKC, BM, BN, BK, ST, WM, WN>), dim3(g.tiles_i * g.tiles_j * g.splits), dim3(64 * WM * WN), lds, st, g);
  VEEX_CHECK_LAUNCH();
  return 0;
}

template <typename T, typename M, bool AKC, bool BKC>
static int dt_pick(int tile, const DtGemm& g, hipStream_t st) {
  if constexpr (sizeof(T) == 4) {
    if (tile == 1) return dt_go<T, M, 3, AKC, BKC, 256, 128, 32, 2, 4, 2>(g, st);
    return dt_go<T, M, 3, AKC, BKC, 128, 128, 32, 3, 2, 4>(g, st);
  } else {
    if (tile == 0) return dt_go<T, M, 1, AKC, BKC, 256, 256, 32, 4, 2, 4>(g, st);
    if (tile == 1) return dt_go<T, M, 1, AKC, BKC, 256, 128, 64, 3, 4, 2>(g, st);
    return dt_go<T, M, 1, AKC, BKC, 128, 128, 64, 4, 2, 4>(g, st);
  }
}

template <typename T, typename M, int PL, int BM, int BN, int BK, int ST, int WM, int WN>
static int dt_grads_go(const DtGemm& dx_in, const DtGemm& dw_in, hipStream_t st) {
  DtGemm g[2] = {dx_in, dw_in};
  for (DtGemm& q : g) { q.tiles_i = (unsigned)((q.I + BM - 1) / BM); q.tiles_j = (unsigned)((q.J + BN - 1) / BN); }
  constexpr int lds = ST * PL * (BM + BN) * BK * 2;
  const void* fn = reinterpret_cast<const void*>(dense_tile_grads_kernel<T, M, PL, BM, BN, BK, ST, WM, WN>);
  if (lds > 64 * 1024 && hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
    veex_set_error("dense: cannot raise the dynamic LDS limit"); return VEEX_ELAUNCH;
  }
  const unsigned n0 = g[0].tiles_i * g[0].tiles_j * g[0].splits, n1 = g[1].tiles_i * g[1].tiles_j * g[1].splits;
  hipLaunchKernelGGL((dense_tile_grads_kernel<T, M, PL, BM, BN, BK, ST, WM, WN>), dim3(n0 + n1), dim3(64 * WM * WN), lds, st, g[0], g[1], n0);
  VEEX_CHECK_LAUNCH();
  return 0;
}

int dense_tile_grads_launch(int dtype, const DtGemm& dx, const DtGemm& dw, hipStream_t st) {
  if (dtype == VEEX_T_F32) return dt_grads_go<float, bf16_t, 3, 128, 128, 32, 3, 2, 4>(dx, dw, st);
  if (dtype == VEEX_T_BF16) return dt_grads_go<bf16_t, bf16_t, 1, 128, 128, 64, 4, 2, 4>(dx, dw, st);
  return dt_grads_go<f16_t, f16_t, 1, 128, 128, 64, 4, 2, 4>(dx, dw, st);
}

template <typename T, typename M>
static int dt_kind(bool akc, bool bkc, int tile, const DtGemm& g, hipStream_t st) {
  if (akc && bkc) return dt_pick<T, M, true, true>(tile, g, st);
  if (akc) return dt_pick<T, M, true, false>(tile, g, st);
  return dt_pick<T, M, false, false>(tile, g, st);
}

int dense_tile_launch(int dtype, bool akc, bool bkc, int tile, const DtGemm& g, hipStream_t st) {
  if (dtype == VEEX_T_F32) return dt_kind<float, bf16_t>(akc, bkc, tile, g, st);
  if (dtype == VEEX_T_BF16) return dt_kind<bf16_t, bf16_t>(akc, bkc, tile, g, st);
  return dt_kind<f16_t, f16_t>(akc, bkc, tile, g, st);
}
