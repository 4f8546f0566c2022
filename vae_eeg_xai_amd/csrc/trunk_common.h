// Device helpers shared by the dense-trunk operators (dense.hip, dense_tile.hip, dropout.hip, residual_norm.hip):
// element types, 16-byte row pieces, and the dropout decision.
#ifndef VEEX_TRUNK_COMMON_H
#define VEEX_TRUNK_COMMON_H
#include "veex_internal.h"
#include "philox.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> struct TrunkType;
template <> struct TrunkType<float> { static constexpr int code = 0; };
template <> struct TrunkType<bf16_t> { static constexpr int code = 1; };
template <> struct TrunkType<f16_t> { static constexpr int code = 2; };

inline int trunk_elem_bytes(int dtype) { return dtype == 0 ? 4 : 2; }
inline bool trunk_dtype_ok(int dtype) { return dtype >= 0 && dtype <= 2; }
inline bool trunk_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// V consecutive elements as they lie in memory: one load / store of up to 16 bytes (address aligned to its size)
template <typename T, int V> struct alignas(sizeof(T) * V) Piece { T v[V]; };

template <typename T, int V>
__device__ __forceinline__ Piece<T, V> piece_load(const T* p) { return *reinterpret_cast<const Piece<T, V>*>(p); }
template <typename T, int V>
__device__ __forceinline__ void piece_store(T* p, const Piece<T, V>& x) { *reinterpret_cast<Piece<T, V>*>(p) = x; }

// Inverted dropout on 16-bit uniform numbers: an element is dropped with probability cut / 65536 and scaled by
// 65536 / (65536 - cut) otherwise.  Philox gives four 32-bit words per call; 16 bits an element instead of 32 halve the
// generator's work (32-bit multiplies run at a quarter of the vector rate) and leave the rate exact to 2^-17.
struct DropArgs {
  unsigned cut;                       // 0: no dropout
  float scale;                        // 65536 / (65536 - cut)
  unsigned k0, k1;                    // key: the seed's two words
  unsigned long long first_row;       // row of the grid that row 0 of this call is (a shard's or a step's offset)
  const unsigned long long* counter;  // optional device word added to first_row when the kernel runs
};

__device__ __forceinline__ unsigned long long drop_base(const DropArgs& d) {
  return d.first_row + (d.counter != nullptr ? d.counter[0] : 0ull);
}

// the four words that decide columns 8 * block .. + 7 of a row: column c takes half word c & 1 of word (c & 7) >> 1.
// The second counter word is a tag: the sampler's epsilon under the same seed (special.hip) uses counters with a small
// number there.  A block never straddles rows, so the decisions depend on (seed, row, column) alone: not on the width's divisibility,
// on vectorisation, or on how a batch is split over calls and ranks.
__device__ __forceinline__ void drop_words(const DropArgs& d, unsigned long long row, unsigned block, unsigned w[4]) {
  w[0] = block; w[1] = 0x44524F50u; w[2] = (unsigned)row; w[3] = (unsigned)(row >> 32);
  philox4x32_10(w, d.k0, d.k1);
}
__device__ __forceinline__ unsigned drop_u16(const unsigned w[4], int e) { return (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu; }

// host: cut and scale of a rate in [0, 1); false where the rate is none or rounds to dropping everything
inline bool trunk_drop_args(double rate, unsigned long long seed, unsigned long long first_row,
                            const unsigned long long* counter, DropArgs& d) {
  if (!(rate >= 0.0 && rate < 1.0)) return false;
  d.cut = (unsigned)(long long)__builtin_rint(rate * 65536.0);
  if (d.cut >= 65536u) return false;
  d.scale = (float)(65536.0 / (double)(65536u - d.cut));
  d.k0 = (unsigned)(seed & 0xFFFFFFFFull); d.k1 = (unsigned)(seed >> 32);
  d.first_row = first_row; d.counter = counter;
  return true;
}

// host: a launch counts its threads along x in 32 bits
inline bool trunk_grid_ok(long long blocks, int threads) { return blocks > 0 && blocks <= 0xFFFFFFFFll / threads; }

#endif
