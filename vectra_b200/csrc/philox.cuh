// philox.cuh: the random numbers of dropout (vectra_drop in
// include/vectra_block.h), made from an element's index wherever they are
// needed, so that no mask is stored.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011): ten rounds of two 32 x 32 -> 64 bit products on a
// counter of four words. One counter gives eight 16-bit numbers, so eight
// consecutive elements share the rounds: about 9 instructions an element,
// where one 32-bit word an element would take 18 and set the pace of 16-bit
// tensors (at 6.5 TB/s an SM has some 20 issue slots for each element that it
// reads and writes). The price is that p comes in steps of 2^-16; the scale
// is that of the share that is kept, so the expectation is exact.
#pragma once

#include <stdint.h>

#include "vectra_block.h"

// The formulation for CPU tensors (decoder_ext.cpp) makes the same numbers.
#ifdef __CUDACC__
#define VECTRA_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define VECTRA_HOST_DEVICE inline
#endif

namespace vectra {

struct Drop {
  const int64_t* rng = nullptr;
  uint32_t stream = 0;
  uint32_t cut = 0;    // keep a number of at least this; 0: no dropout
  float scale = 1.f;   // of what is kept
};

// p in [0, 1].
inline Drop make_drop(const vectra_drop& d) {
  Drop r;
  r.rng = d.rng;
  r.stream = d.stream;
  r.cut = uint32_t(d.p * 65536.0 + 0.5);
  r.scale = r.cut < 65536 ? float(65536.0 / double(65536 - r.cut)) : 0.f;
  return r;
}

struct PhiloxKey {
  uint32_t k0, k1, step, stream;
};

#ifdef __CUDACC__
__device__ __forceinline__ PhiloxKey load_key(const Drop& d) {
  PhiloxKey k{};
  if (d.cut) {
    const uint64_t seed = uint64_t(__ldg(
        reinterpret_cast<const long long*>(d.rng)));
    k.k0 = uint32_t(seed);
    k.k1 = uint32_t(seed >> 32);
    k.step = uint32_t(uint64_t(
        __ldg(reinterpret_cast<const long long*>(d.rng) + 1)));
    k.stream = d.stream;
  }
  return k;
}
#endif

// Bit i: element 8 group + i is kept.
VECTRA_HOST_DEVICE uint32_t keep_bits(const PhiloxKey& key,
                                      uint64_t group, uint32_t cut) {
  uint32_t c0 = uint32_t(group), c1 = uint32_t(group >> 32);
  uint32_t c2 = key.step, c3 = key.stream;
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = uint64_t(c0) * 0xD2511F53u;
    const uint64_t p1 = uint64_t(c2) * 0xCD9E8D57u;
    c0 = uint32_t(p1 >> 32) ^ c1 ^ k0;
    c1 = uint32_t(p1);
    c2 = uint32_t(p0 >> 32) ^ c3 ^ k1;
    c3 = uint32_t(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const uint32_t w[4] = {c0, c1, c2, c3};
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bits |= uint32_t((w[i] & 0xffffu) >= cut) << (2 * i);
    bits |= uint32_t((w[i] >> 16) >= cut) << (2 * i + 1);
  }
  return bits;
}

}  // namespace vectra
