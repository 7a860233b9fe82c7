// The threads that share a row, and their reductions.
//
// A row is held by part of a warp or a warp (short rows: several independent
// teams in a CTA, no barrier), by some warps or all of a CTA (a named barrier
// for each team), or by a cluster of up to eight CTAs (rows longer than a CTA's
// registers hold, or so few rows that most SMs would idle).  A reduction
// folds each warp by shuffles, then every warp writes its record into the
// shared memory of every CTA of the team (distributed shared memory within a
// cluster), one barrier follows, and every thread folds the records in warp
// order: one barrier a reduction whatever the team, and every thread gets the
// same bits.
//
// Records are kept in two sets by the row's parity: a thread writes a row's
// records only after the barrier of the row before, which no thread passes
// until all have read the records of the row before that.  Reductions of one
// row use slots of their own.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <map>
#include <mutex>
#include <utility>

#include "kernels.h"

namespace askb {

constexpr int kTeamThreads = 512;                   // threads of a CTA at most
constexpr int kTeamCluster = 8;                     // CTAs of a team at most (the portable cluster size)
constexpr int kTeamRecords = kTeamThreads / 32 * kTeamCluster;

struct Team {
  uint32_t tid;      // thread within this CTA's part of the team
  uint32_t threads;  // threads of that part
  uint32_t lanes;    // lanes of a warp that belong to one team
  uint32_t lane, warp, warps;
  uint32_t ctas, rank;  // CTAs of the team (the cluster) and this one's place among them
  uint32_t count, index;  // teams of this CTA, and which this is
};

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_address(const void* mine, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
  return r;
}

__device__ __forceinline__ Team team_of(const TeamShape& s) {
  Team t;
  t.lane = threadIdx.x & 31u;
  if (s.warp_teams) {
    t.lanes = uint32_t(s.warp_teams);
    t.tid = t.lane & (t.lanes - 1);
    t.threads = t.lanes;
    t.warp = 0;
    t.warps = 1;
    t.ctas = 1;
    t.rank = 0;
    t.count = blockDim.x / t.lanes;
    t.index = threadIdx.x / t.lanes;
  } else {
    t.lanes = 32;
    t.threads = uint32_t(s.team_threads);
    t.count = blockDim.x / t.threads;
    t.index = t.count == 1 ? 0 : threadIdx.x / t.threads;
    t.tid = threadIdx.x - t.index * t.threads;
    t.warp = t.tid >> 5;
    t.warps = t.threads >> 5;
    t.ctas = cluster_size();
    t.rank = cluster_rank();
  }
  return t;
}

// Before the first reduction: a CTA's shared memory may be written by a peer
// only once that CTA runs.
__device__ __forceinline__ void team_start(const Team& t) {
  if (t.ctas > 1) cluster_barrier();
}

template <int N>
struct alignas(16) TeamRecords {
  float v[2][kTeamRecords][N];
};

// Where a team's records begin: teams that share a CTA have theirs side by side.
__device__ __forceinline__ uint32_t team_base(const Team& t) { return t.index * t.warps; }

// Write this warp's record (v, the same in all lanes) to the team; then barrier.
// kShared: several teams of whole warps may share the CTA, each with its named
// barrier.  Such a kernel reserves all 16 barriers of a CTA, and an SM then
// holds 4 CTAs at most (65536 norm rows of 1024 took 175 us so, and 124 without), so
// only a kernel whose CTAs fill the SM asks for it.
template <int N, bool kShared = false>
__device__ __forceinline__ void team_exchange(const Team& t, TeamRecords<N>& sh, int parity, const float (&v)[N]) {
  if (t.ctas == 1) {
    if (t.lane == 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) sh.v[parity][team_base(t) + t.warp][n] = v[n];
    }
    if (!kShared || t.count == 1) __syncthreads();
    else asm volatile("barrier.sync %0, %1;" ::"r"(t.index + 1u), "r"(t.threads) : "memory");
    return;
  }
  if (t.lane < t.ctas) {
    const uint32_t at = peer_address(&sh.v[parity][t.rank * t.warps + t.warp][0], t.lane);
#pragma unroll
    for (int n = 0; n < N; ++n)
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 4u * n), "f"(v[n]) : "memory");
  }
  cluster_barrier();
}

// Sum of N values over the team, the same bits in every thread.
template <int N, bool kShared = false>
__device__ __forceinline__ void team_sum(const Team& t, TeamRecords<N>& sh, int parity, float (&v)[N]) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    if (uint32_t(d) >= t.lanes) continue;
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], d);
  }
  const uint32_t records = t.warps * t.ctas;
  if (records == 1) return;
  team_exchange<N, kShared>(t, sh, parity, v);
  const float(*const rec)[N] = sh.v[parity] + team_base(t);
  // Eight warps (norm rows of 2049 to 4096 columns) are added without a loop: bf16
  // [32768, 4096] norms with dropout 231 us, 243 by the loop, gradient 314 and 342, layer
  // norms with biases of half the rows 171 and 196.  Without dropout it costs some
  // (188 and 180), and in f32 (8192 rows 99 and 97).
  if (records == 8) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float r[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = rec[k][n];
      v[n] = ((r[0] + r[1]) + (r[2] + r[3])) + ((r[4] + r[5]) + (r[6] + r[7]));
    }
  } else if (records < 8) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = rec[0][n];
    for (uint32_t k = 1; k < records; ++k) {
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += rec[k][n];
    }
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = 0.0f;
      for (uint32_t k = t.lane; k < records; k += 32) v[n] += rec[k][n];
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], d);
    }
  }
}

// Readies a row kernel on the current device, once: all of an SM's memory that
// can be shared memory is to be that (by itself the driver kept back so much
// that 4 CTAs ran where 10 fit), and a CTA may use `shared_bytes` of it.
inline cudaError_t prepare_rows(const void* kernel, unsigned shared_bytes) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, unsigned> ready;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  unsigned& allowed = ready[{kernel, device}];
  if (allowed > shared_bytes) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(shared_bytes));
  if (e == cudaSuccess) allowed = shared_bytes + 1;
  return e;
}

// Launch of a row kernel: CTAs of the shape's threads in clusters of its size,
// as a programmatic dependent (pdl.cuh).
inline cudaError_t launch_rows(const void* kernel, const TeamShape& s, unsigned grid, unsigned shared_bytes, void** args,
                               cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(unsigned(s.threads));
  cfg.dynamicSmemBytes = shared_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(s.ctas);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = s.ctas > 1 ? 2 : 1;
  (void)cudaLaunchKernelExC(&cfg, kernel, args);
  return cudaGetLastError();
}

}  // namespace askb
