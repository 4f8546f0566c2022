// Philox-4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): ten rounds over a
// 128-bit counter c[0..3] under a 64-bit key; the counter is replaced by four random words.
#ifndef VEEX_PHILOX_H
#define VEEX_PHILOX_H
#include <hip/hip_runtime.h>

__device__ __forceinline__ void philox4x32_10(unsigned c[4], unsigned k0, unsigned k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p0 = (unsigned long long)c[0] * 0xD2511F53u, p1 = (unsigned long long)c[2] * 0xCD9E8D57u;
    c[0] = (unsigned)(p1 >> 32) ^ c[1] ^ k0; c[1] = (unsigned)p1;
    c[2] = (unsigned)(p0 >> 32) ^ c[3] ^ k1; c[3] = (unsigned)p0;
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
}

#endif
