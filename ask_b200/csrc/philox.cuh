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

// The same, out of line: what is rarely taken costs its callers no registers.
static __device__ __noinline__ Philox philox4x32_10_call(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0,
                                                  uint32_t k1) {
  return philox4x32_10(c0, c1, c2, c3, k0, k1);
}

// Dropout at one site of a model.  Element i of the site's tensor (row-major)
// takes word i % 4 of the block with counter (lo(b), hi(b), stream, 1),
// b = offset + i / 4 (mod 2^64), under key (lo(seed), hi(seed)); it is kept
// when that word is at least `threshold` = floor(p * 2^32), and then scaled by
// 1 / (1 - p).  seed and offset are read from device memory, so a captured
// graph replays with new masks.  A dropped element is replaced by zero and not
// multiplied, so a NaN or an infinity in it is gone too.
//
// The generator is the cost of dropout.  On a B200 a widening product takes a
// scheduler 4 clocks a warp and a three-way xor 2 (measured, 512 threads on an
// SM), so ten rounds of two products are 80 clocks for four elements a lane: 75 us
// for 2^27 elements, as long as HBM needs for their 2-byte reads and writes.
// The rounds that see only the counter's constant words are therefore taken out
// of the loop (DropRun): counter word 2 is the site's, word 1 changes once in
// 2^34 elements, so of the first round only lo(b)'s product is left, and of
// the second one product; and block b + 1 adds the multiplier to block b's first
// product.  That leaves 17 or 18 products of 20; the tensor takes 120 us with
// its memory traffic (dropout_kernels.cu).  Products by f64 multiply-adds
// (88-91 us for the generator alone against 76) and a comparison by a widening
// multiply-add (157 against 134 us for the whole kernel then) were slower.  A
// block whose high word is not the run's takes all rounds.
struct DropRun {
  uint64_t offset;
  uint32_t high;                // hi(b) that the constants below belong to
  uint32_t k0, k1;              // the key
  uint32_t n2, n0_2, n2_2, n2_3;  // what the first three rounds xor onto their products
  uint32_t stream, threshold;
  float scale;
};

constexpr uint32_t kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u, kPhiloxW0 = 0x9E3779B9u, kPhiloxW1 = 0xBB67AE85u;

__device__ __forceinline__ DropRun drop_run(const DropSite& d, const int64_t* seed) {
  DropRun r{};
  if (d.on) {
    const uint64_t key = uint64_t(__ldg(reinterpret_cast<const unsigned long long*>(seed)));
    r.offset = uint64_t(__ldg(reinterpret_cast<const unsigned long long*>(seed) + 1));
    r.high = uint32_t(r.offset >> 32);
    r.k0 = uint32_t(key);
    r.k1 = uint32_t(key >> 32);
    r.stream = d.stream;
    const uint64_t p1 = uint64_t(kPhiloxM1) * d.stream;                    // round 1, words 2 and 3
    const uint64_t p0 = uint64_t(kPhiloxM0) * (uint32_t(p1 >> 32) ^ r.high ^ r.k0);  // round 2, word 0
    r.n2 = 1u ^ r.k1;
    r.n0_2 = uint32_t(p1) ^ (r.k0 + kPhiloxW0);
    r.n2_2 = uint32_t(p0 >> 32) ^ (r.k1 + kPhiloxW1);
    r.n2_3 = uint32_t(p0) ^ (r.k1 + 2 * kPhiloxW1);
    r.threshold = d.threshold;
    r.scale = d.scale;
  }
  return r;
}

// The rounds that are left of kBlocks blocks whose first products (round 1,
// lo(b)) are known, side by side: the key schedule is stepped once for all.
template <int kBlocks>
__device__ __forceinline__ void drop_rounds(const DropRun& r, const uint64_t (&first)[kBlocks], Philox (&w)[kBlocks]) {
  uint32_t k0 = r.k0 + 2 * kPhiloxW0, k1 = r.k1 + 2 * kPhiloxW1;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    // round 2: only word 2's product is not the run's
    const uint64_t q = uint64_t(kPhiloxM1) * (uint32_t(first[b] >> 32) ^ r.n2);
    const uint32_t c0 = uint32_t(q >> 32) ^ r.n0_2, c2 = uint32_t(first[b]) ^ r.n2_2;
    // round 3
    const uint64_t p0 = uint64_t(kPhiloxM0) * c0, p1 = uint64_t(kPhiloxM1) * c2;
    w[b].c[0] = uint32_t(p1 >> 32) ^ uint32_t(q) ^ k0;
    w[b].c[1] = uint32_t(p1);
    w[b].c[2] = uint32_t(p0 >> 32) ^ r.n2_3;
    w[b].c[3] = uint32_t(p0);
  }
#pragma unroll
  for (int round = 3; round < 10; ++round) {
    k0 += kPhiloxW0;
    k1 += kPhiloxW1;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      uint32_t(&c)[4] = w[b].c;
      const uint64_t p0 = uint64_t(kPhiloxM0) * c[0], p1 = uint64_t(kPhiloxM1) * c[2];
      c[0] = uint32_t(p1 >> 32) ^ c[1] ^ k0;
      c[2] = uint32_t(p0 >> 32) ^ c[3] ^ k1;
      c[1] = uint32_t(p1);
      c[3] = uint32_t(p0);
    }
  }
}

// The words of kRuns runs of kBlocks blocks; run u starts at the block of
// element i[u].
template <int kRuns, int kBlocks>
__device__ __forceinline__ void drop_words(const DropRun& r, const uint64_t (&i)[kRuns], Philox (&w)[kRuns * kBlocks]) {
  uint64_t first[kRuns * kBlocks];
  bool plain = true;  // every block's high word is the run's
#pragma unroll
  for (int u = 0; u < kRuns; ++u) {
    const uint64_t b = r.offset + (i[u] >> 2);
    plain = plain && uint32_t(b >> 32) == r.high && uint32_t(b) <= 0xffffffffu - uint32_t(kBlocks - 1);
    first[u * kBlocks] = uint64_t(kPhiloxM0) * uint32_t(b);
#pragma unroll
    for (int k = 1; k < kBlocks; ++k) first[u * kBlocks + k] = first[u * kBlocks + k - 1] + kPhiloxM0;
  }
  if (plain) {
    drop_rounds<kRuns * kBlocks>(r, first, w);
  } else {
#pragma unroll
    for (int k = 0; k < kRuns * kBlocks; ++k) {
      const uint64_t at = r.offset + (i[k / kBlocks] >> 2) + uint64_t(k % kBlocks);
      w[k] = philox4x32_10_call(uint32_t(at), uint32_t(at >> 32), r.stream, 1u, r.k0, r.k1);
    }
  }
}
// Which elements are kept of kRuns runs of N (a multiple of 4), run u starting
// at element i[u].  kAnywhere: i[u] may be any element, then a block more is
// drawn and its words are moved down by i[u] % 4.
template <int kRuns, int N, bool kAnywhere = false>
__device__ __forceinline__ void drop_keep(const DropRun& r, const uint64_t (&i)[kRuns], bool (&keep)[kRuns * N]) {
  static_assert(N % 4 == 0, "whole blocks");
  if (!kAnywhere || (i[0] & 3) == 0) {  // the runs of a row start at whole units from one another
    Philox w[kRuns * (N / 4)];
    drop_words<kRuns, N / 4>(r, i, w);
#pragma unroll
    for (int j = 0; j < kRuns * N; ++j) keep[j] = w[j / 4].c[j % 4] >= r.threshold;
  } else {
    constexpr int B = N / 4 + 1;
    Philox w[kRuns * B];
    drop_words<kRuns, B>(r, i, w);
#pragma unroll
    for (int u = 0; u < kRuns; ++u) {
      uint32_t v[4 * B];
#pragma unroll
      for (int j = 0; j < 4 * B; ++j) v[j] = w[u * B + j / 4].c[j % 4];
#pragma unroll
      for (int j = 0; j < 4 * B - 1; ++j) v[j] = (i[0] & 1) ? v[j + 1] : v[j];
#pragma unroll
      for (int j = 0; j < 4 * B - 3; ++j) v[j] = (i[0] & 2) ? v[j + 2] : v[j];
#pragma unroll
      for (int j = 0; j < N; ++j) keep[u * N + j] = v[j] >= r.threshold;
    }
  }
}
// The same of single elements: a block for each.
template <int kRuns>
__device__ __forceinline__ void drop_keep_words(const DropRun& r, const uint64_t (&i)[kRuns], bool* keep) {
  Philox w[kRuns];
  drop_words<kRuns, 1>(r, i, w);
#pragma unroll
  for (int u = 0; u < kRuns; ++u) {
    const bool upper = i[u] & 2;
    const uint32_t a = upper ? w[u].c[2] : w[u].c[0], b = upper ? w[u].c[3] : w[u].c[1];
    keep[u] = ((i[u] & 1) ? b : a) >= r.threshold;
  }
}
// N elements dropped and scaled.
template <int N>
__device__ __forceinline__ void drop_unit(const DropRun& r, uint64_t i, float* v) {
  bool keep[N];
  const uint64_t at[1] = {i};
  drop_keep<1, N>(r, at, keep);
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = keep[j] ? __fmul_rn(v[j], r.scale) : 0.0f;
}

}  // namespace askb
