// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", SC'11): four 32-bit words as a pure function of a 128-bit
// counter and a 64-bit key.
//
// Two users share it: the input generator (gen_kernels.cu, counter word 3 = 0)
// and dropout (counter word 3 = 1, so a model that draws its inputs and its
// masks from one seed never meets the same block twice).
#pragma once

#include <stdint.h>

#include "kernels.h"

namespace askb {

struct Philox {
  uint32_t c[4];
};

__device__ __forceinline__ Philox philox4x32_10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0,
                                               uint32_t k1) {
  constexpr uint32_t kM0 = 0xD2511F53u, kM1 = 0xCD9E8D57u, kW0 = 0x9E3779B9u, kW1 = 0xBB67AE85u;
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    // one widening product gives both halves
    const uint64_t p0 = uint64_t(kM0) * c0, p1 = uint64_t(kM1) * c2;
    const uint32_t n0 = uint32_t(p1 >> 32) ^ c1 ^ k0, n2 = uint32_t(p0 >> 32) ^ c3 ^ k1;
    c0 = n0; c1 = uint32_t(p1); c2 = n2; c3 = uint32_t(p0);
    k0 += kW0; k1 += kW1;
  }
  return Philox{{c0, c1, c2, c3}};
}

// Dropout at one site of a model.  Element i of the site's tensor (row-major)
// takes word i % 4 of the block with counter (lo(b), hi(b), stream, 1),
// b = offset + i / 4 (mod 2^64), under key (lo(seed), hi(seed)); it is kept
// when that word is at least `threshold` = floor(p * 2^32), and then scaled by
// 1 / (1 - p).  seed and offset are read from device memory, so a captured
// graph replays with new masks.  A dropped element is replaced by zero and not
// multiplied, so a NaN or an infinity in it is gone too.
struct DropRun {
  uint64_t offset;
  uint32_t k0, k1, stream, threshold;
  float scale;
};

__device__ __forceinline__ DropRun drop_run(const DropSite& d, const int64_t* seed) {
  DropRun r{};
  if (d.on) {
    const uint64_t key = uint64_t(__ldg(reinterpret_cast<const unsigned long long*>(seed)));
    r.offset = uint64_t(__ldg(reinterpret_cast<const unsigned long long*>(seed) + 1));
    r.k0 = uint32_t(key);
    r.k1 = uint32_t(key >> 32);
    r.stream = d.stream;
    r.threshold = d.threshold;
    r.scale = d.scale;
  }
  return r;
}

// The words of the four elements starting at element `i` (a multiple of 4).
__device__ __forceinline__ Philox drop_words(const DropRun& r, uint64_t i) {
  const uint64_t b = r.offset + (i >> 2);
  return philox4x32_10(uint32_t(b), uint32_t(b >> 32), r.stream, 1u, r.k0, r.k1);
}
__device__ __forceinline__ float drop_apply(const DropRun& r, uint32_t word, float v) {
  return word >= r.threshold ? __fmul_rn(v, r.scale) : 0.0f;
}
// N elements starting at element i: whole blocks when N is a multiple of 4
// (then i is one too), else one element.
template <int N>
__device__ __forceinline__ void drop_unit(const DropRun& r, uint64_t i, float* v) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int g = 0; g < N / 4; ++g) {
      const Philox w = drop_words(r, i + uint64_t(4 * g));
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * g + j] = drop_apply(r, w.c[j], v[4 * g + j]);
    }
  } else {
    static_assert(N == 1, "whole blocks or one element");
    const Philox w = drop_words(r, i);
    const uint32_t k = uint32_t(i) & 3u;
    v[0] = drop_apply(r, k < 2 ? (k == 0 ? w.c[0] : w.c[1]) : (k == 2 ? w.c[2] : w.c[3]), v[0]);
  }
}

}  // namespace askb
