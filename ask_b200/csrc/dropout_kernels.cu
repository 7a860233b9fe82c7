// Dropout: y = D(x) (+ residual), with the mask drawn from a counter and never
// stored; the backward pass is the same map of dy (philox.cuh has the rule).
//
// Bound: HBM, 2 (3 with a residual) elements moved for each one computed; the
// generator's products (philox.cuh) take about as long as HBM needs for 2-byte
// elements and half as long as for 4-byte ones, so the next units' loads are
// issued before this one's integer work.  2^27 bf16 elements take 120 us
// (4.5 TB/s; the copy alone 82, the generator alone 76).  Nothing is full then:
// issue slots 54%, the busiest pipe (widening products) 64%, DRAM below that; four
// warps a scheduler, which is what the registers leave, wait for the generator's
// fixed latencies.  2^26 f32 elements take 84.7 us (6.3 TB/s), 17,000,051 of them
// with a residual 32.7 us (6.2 TB/s).
#include <cuda_runtime.h>

#include <algorithm>

#include "act_io.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "philox.cuh"

namespace askb {

namespace {

// 16-byte units a thread has in flight, and CTAs an SM the registers are held
// to.  The generator's work is what 2-byte elements wait for, so they take
// four units (eight blocks side by side) and all the registers that takes; the
// others wait for memory.
template <int T, bool kRes>
constexpr int units_in_flight() { return act_vec<T>() == 8 && !kRes ? 4 : 2; }
template <int T, bool kRes>
constexpr int ctas_per_sm() { return act_vec<T>() == 8 ? (kRes ? 3 : 2) : 4; }

template <int T>
__device__ __forceinline__ void load_elems(const void* p, uint64_t i, int n, float* v) {
#pragma unroll
  for (int j = 0; j < act_vec<T>(); ++j) v[j] = j < n ? act_load<T>(p, i + j) : 0.0f;
}

template <int T, bool kRes, bool kAligned>
__global__ void __launch_bounds__(kDropThreads, ctas_per_sm<T, kRes>()) dropout_kernel(const DropoutArgs a) {
  constexpr int V = act_vec<T>();
  pdl_enter();
  const DropRun run = drop_run(a.drop, a.seed);
  const uint64_t units = a.count / V, stride = uint64_t(gridDim.x) * kDropThreads;
  uint64_t u = uint64_t(blockIdx.x) * kDropThreads + threadIdx.x;
  auto finish = [&](uint64_t at, int n, float* v, const float* r) {
    if (a.drop.on) drop_unit<V>(run, at, v);
    if constexpr (kRes) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = __fadd_rn(v[j], r[j]);
    }
    if (kAligned && n == V) {
      act_put<T, V>(a.y, at, v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) act_store<T>(a.y, at + j, v[j]);
    }
  };
  if constexpr (kAligned) {
    // U units a step, the next step's loads issued before this one's math
    constexpr int U = units_in_flight<T, kRes>();
    ActRaw<T, V> x[U], r[U];
    auto fetch = [&](uint64_t from) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        x[k].load(a.x, (from + k * stride) * V);
        if constexpr (kRes) r[k].load(a.residual, (from + k * stride) * V);
      }
    };
    bool more = u + (U - 1) * stride < units;
    if (more) fetch(u);
    while (more) {
      float v[U][V], w[U][V];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        x[k].widen(v[k]);
        if constexpr (kRes) r[k].widen(w[k]);
      }
      const uint64_t now = u;
      u += U * stride;
      more = u + (U - 1) * stride < units;
      if (more) fetch(u);
#pragma unroll
      for (int k = 0; k < U; ++k) finish((now + k * stride) * V, V, v[k], w[k]);
    }
  }
  // the rest, the last unit possibly cut short
  for (; u * V < a.count; u += stride) {
    const uint64_t at = u * V;
    const int n = int(a.count - at < uint64_t(V) ? a.count - at : uint64_t(V));
    float v[V], w[V];
    if (kAligned && n == V) {
      ActRaw<T, V> x, r;
      x.load(a.x, at);
      if constexpr (kRes) r.load(a.residual, at);
      x.widen(v);
      if constexpr (kRes) r.widen(w);
    } else {
      load_elems<T>(a.x, at, n, v);
      if constexpr (kRes) load_elems<T>(a.residual, at, n, w);
    }
    finish(at, n, v, w);
  }
}

using Kernel = void (*)(const DropoutArgs);
template <int T>
Kernel pick(bool res, bool aligned) {
  return res ? (aligned ? dropout_kernel<T, true, true> : dropout_kernel<T, true, false>)
             : (aligned ? dropout_kernel<T, false, true> : dropout_kernel<T, false, false>);
}
Kernel kernel_for(int type, bool res, bool aligned) {
  return type == kF32 ? pick<kF32>(res, aligned) : type == kF16 ? pick<kF16>(res, aligned) : pick<kBF16>(res, aligned);
}

}  // namespace

cudaError_t dropout_occupancy(int type, bool residual, int* blocks_per_sm) {
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(blocks_per_sm, kernel_for(type, residual, true), kDropThreads, 0);
}

cudaError_t dropout_launch(const DropoutArgs& a, int grid, cudaStream_t stream) {
  if (a.count == 0) return cudaSuccess;
  const auto at16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const bool aligned = at16(a.x) && at16(a.y) && (!a.residual || at16(a.residual));
  (void)launch_pdl(kernel_for(a.type, a.residual != nullptr, aligned), dim3(unsigned(grid)), dim3(kDropThreads), stream, a);
  return cudaGetLastError();
}

}  // namespace askb
