// Block norms: the row work between two blocks of a transformer in one pass,
//   h = alpha x + D(g * N_post(y)),   u = N_pre(h),
// and its gradient in one pass plus a join of the column sums.
//
//   N(v) = vhat * w (+ b),  vhat = (v - mean) r,  r = 1 / sqrt(var + eps);
//   the rms norm has mean = 0.  D is dropout, g a gate shared by a group of
//   consecutive rows.  mean and r are the row's saved statistics.
//
// Gradient, with dh and du the gradients to h and u:
//   a = w_pre du;  G = dh + r (a - [mean a] - hhat mean(a hhat));  dx = alpha G
//   B = D(G);  c = w_post g B;  dy = r (c - [mean c] - yhat mean(c yhat))
//   T = sum B yhat, S = sum B over a group's rows; P = sum du hhat, Q = sum du
//   dgate = w_post T + b_post S;  dw_post = sum over groups g T;  db_post = sum g S
//   dw_pre = P;  db_pre = Q
// ([..]: layer norm only; without a post norm yhat is y and dy = g B.)  One
// sum over a group's rows thus serves both the gate's gradient and the
// weight's.
//
// Statistics come from 32-bit values: var of a layer norm is the mean square
// of v - mean, taken in registers in a second step, and u is computed from h
// before h is rounded to its storage type.
#include <cuda_runtime.h>

#include <algorithm>

#include "act_io.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "philox.cuh"
#include "row_team.cuh"

namespace askb {

namespace {

constexpr int kWarpTeamThreads = 256;
constexpr int kElems = 16;  // row elements a thread holds

// A row array in flight: every thread copies the 16-byte words of its own
// units into its own places of a ring in shared memory (cp.async) and reads
// them back, so no barrier is needed, rows are fetched kStages - 1 ahead, and no
// register holds what is on its way.  Where rows start anywhere (kAnywhere) a
// unit spans two words.
template <int T, bool kAnywhere>
struct Ring {
  static constexpr int V = act_vec<T>(), Q = kElems / V, W = kAnywhere ? 2 : 1;
  static constexpr int kWords = Q * W;  // 16-byte words of one thread, array and stage
};

// The team's columns of a row, as the thread holds them: units of 16 bytes, as
// f32 pairs.  A row is named by the byte offset of this thread's first column.
template <int T, bool kAnywhere>
struct Columns {
  static constexpr int E = kElems, V = act_vec<T>(), Q = E / V, P = E / 2, B = dtype_bytes(T);
  uint32_t first, step;  // column of unit q: first + q * step
  uint32_t cols, pitch;  // pitch: between a thread's words in shared memory
  __device__ __forceinline__ Columns(const Team& t, const NormArgs& a)
      : first((t.rank * uint32_t(Q) * t.threads + t.tid) * uint32_t(V)), step(t.threads * uint32_t(V)), cols(a.cols),
        pitch(blockDim.x * 16) {}
  __device__ __forceinline__ uint32_t at(int q) const { return first + uint32_t(q) * step; }
  __device__ __forceinline__ bool in(int q) const { return at(q) < cols; }
  __device__ __forceinline__ int count(int q) const { return in(q) ? int(min(cols - at(q), uint32_t(V))) : 0; }
  __device__ __forceinline__ uint64_t offset(uint64_t row) const { return (row * cols + first) * uint64_t(B); }
  __device__ __forceinline__ const char* unit(const void* p, uint64_t off, int q) const {
    return static_cast<const char*>(p) + off + uint64_t(uint32_t(q) * step * uint32_t(B));
  }

  // `slot`: this thread's words of the array in a stage.  What no column fills
  // is zeroed once, by clear().
  __device__ __forceinline__ void fetch(const void* p, uint64_t off, uint64_t bytes, uint32_t slot) const {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (!in(q)) continue;
      const char* from = unit(p, off, q);
      if constexpr (!kAnywhere) {
        copy_to_shared(slot + uint32_t(q) * pitch, from);
      } else {
        const char* word = from - (reinterpret_cast<uintptr_t>(from) & 15u);
        const char* begin = static_cast<const char*>(p);
        const char* last = from + count(q) * B;  // the unit's elements end here
#pragma unroll
        for (int k = 0; k < 2; ++k, word += 16) {
          const uint32_t to = slot + uint32_t(q * 2 + k) * pitch;
          if (word >= last) continue;  // nothing of the unit in it
          if (word >= begin && word + 16 <= begin + bytes) copy_to_shared(to, word);
          else st_shared(to, load_part<T>(word, begin, begin + bytes));
        }
      }
    }
  }
  __device__ __forceinline__ void clear(uint32_t slot) const {
    if constexpr (!kAnywhere) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (!in(q)) st_shared(slot + uint32_t(q) * pitch, make_uint4(0u, 0u, 0u, 0u));
    }
  }
  __device__ __forceinline__ void read(uint32_t slot, const void* p, uint64_t off, uint64_t (&v)[P]) const {
    float f[E];
    const uint32_t shift = (uint32_t(reinterpret_cast<uintptr_t>(p)) + uint32_t(off)) & 15u;  // of all units: they are words apart
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if constexpr (!kAnywhere) {
        act_widen<T>(ld_shared(slot + uint32_t(q) * pitch), f + q * V);
      } else {
        act_widen<T>(unit_at<T>(ld_shared(slot + uint32_t(2 * q) * pitch), ld_shared(slot + uint32_t(2 * q + 1) * pitch), shift),
                     f + q * V);
        const int n = count(q);
        if (n < V) {
#pragma unroll
          for (int j = 0; j < V; ++j) f[q * V + j] = j < n ? f[q * V + j] : 0.0f;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = pack2(f[2 * k], f[2 * k + 1]);
  }
  __device__ __forceinline__ void put(const Team& t, void* p, uint64_t off, bool on, const uint64_t (&v)[P]) const {
    float f[E];
    unpack(v, f);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      char* to = const_cast<char*>(unit(p, off, q));
      if constexpr (kAnywhere) {
        const uint32_t place = t.lane & (t.lanes - 1);
        store_anywhere<T>(to, act_narrow<T>(f + q * V), on ? count(q) : 0, place == 0, place == t.lanes - 1);
      } else if (on && in(q)) {
        st_stream_v4(to, act_narrow<T>(f + q * V));
      }
    }
  }
  __device__ __forceinline__ static void unpack(const uint64_t (&v)[P], float* f) {
#pragma unroll
    for (int k = 0; k < P; ++k) unpack2(v[k], f[2 * k], f[2 * k + 1]);
  }
  // parameters of these columns, `fill` where the step has none; 0 past the row
  __device__ __forceinline__ void params(const void* p, int type, uint64_t offset, float fill, float* f) const {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int n = count(q);
#pragma unroll
      for (int j = 0; j < V; ++j) f[q * V + j] = j < n ? fill : 0.0f;
      if (!p) continue;
      if (!kAnywhere && n) {
        param_load<V>(p, type, offset + at(q), f + q * V);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < n) param_load<1>(p, type, offset + at(q) + j, f + q * V + j);
      }
    }
  }
  // v - mean where there is a column; the rest stays 0
  __device__ __forceinline__ void center(float mean, uint64_t (&v)[P]) const {
    float f[E];
    unpack(v, f);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int n = count(q);
#pragma unroll
      for (int j = 0; j < V; ++j) f[q * V + j] -= (kAnywhere ? j < n : n != 0) ? mean : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = pack2(f[2 * k], f[2 * k + 1]);
  }
  // zero where dropped; the scale is folded into what the values meet next.
  // Units past the row hold zeros, whatever is drawn for them.
  __device__ __forceinline__ void drop(const DropRun& run, uint64_t off, uint64_t (&v)[P]) const {
    float f[E];
    unpack(v, f);
    uint64_t i[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) i[q] = off / B + uint32_t(q) * step;
    bool keep[E];
    drop_keep<Q, V, kAnywhere>(run, i, keep);
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = pack2(keep[2 * k] ? f[2 * k] : 0.0f, keep[2 * k + 1] ? f[2 * k + 1] : 0.0f);
  }
};

// A thread's parameters, in its own words of shared memory.
struct ParamSlot {
  uint32_t at, pitch;
  __device__ __forceinline__ void write(const float (&f)[kElems]) const {
#pragma unroll
    for (int k = 0; k < kElems / 4; ++k)
      st_shared(at + uint32_t(k) * pitch, make_uint4(__float_as_uint(f[4 * k]), __float_as_uint(f[4 * k + 1]),
                                                     __float_as_uint(f[4 * k + 2]), __float_as_uint(f[4 * k + 3])));
  }
  __device__ __forceinline__ void pair(int k, uint64_t& lo, uint64_t& hi) const {  // elements 4k .. 4k + 3
    asm volatile("ld.shared.v2.u64 {%0,%1}, [%2];" : "=l"(lo), "=l"(hi) : "r"(at + uint32_t(k) * pitch) : "memory");
  }
};

template <int N>
__device__ __forceinline__ float dot(const uint64_t (&a)[N], const uint64_t (&b)[N]) {
  uint64_t s = mul2(a[0], b[0]), t = N > 1 ? mul2(a[1], b[1]) : 0;
#pragma unroll
  for (int k = 2; k < N; k += 2) {
    s = fma2(a[k], b[k], s);
    if (k + 1 < N) t = fma2(a[k + 1], b[k + 1], t);
  }
  return sum2(N > 1 ? add2(s, t) : s);
}
template <int N>
__device__ __forceinline__ float total(const uint64_t (&a)[N]) {
  uint64_t s = a[0];
#pragma unroll
  for (int k = 1; k < N; ++k) s = add2(s, a[k]);
  return sum2(s);
}

// Centres the row (layer norm) and gives its mean and 1 / sqrt(variance + eps).
template <int T, bool kAnywhere>
__device__ __forceinline__ void row_stats(const Team& t, const Columns<T, kAnywhere>& c, TeamRecords<1>& sh_mean,
                                          TeamRecords<1>& sh_sq, int parity, bool layer, float inv_cols, float eps,
                                          uint64_t (&v)[kElems / 2], float& mean, float& rstd) {
  mean = 0.0f;
  if (layer) {
    float s[1] = {total(v)};
    team_sum<1>(t, sh_mean, parity, s);
    mean = s[0] * inv_cols;
    c.center(mean, v);
  }
  float s[1] = {dot(v, v)};
  team_sum<1>(t, sh_sq, parity, s);
  rstd = rsqrtf(__fmaf_rn(s[0], inv_cols, eps));
}

// v <- v * f (+ b)
template <bool kAdd>
__device__ __forceinline__ void scale_by(uint64_t (&v)[kElems / 2], const ParamSlot& f, const ParamSlot& b) {
#pragma unroll
  for (int k = 0; k < kElems / 4; ++k) {
    uint64_t f0, f1;
    f.pair(k, f0, f1);
    if constexpr (kAdd) {
      uint64_t b0, b1;
      b.pair(k, b0, b1);
      v[2 * k] = fma2(v[2 * k], f0, b0);
      v[2 * k + 1] = fma2(v[2 * k + 1], f1, b1);
    } else {
      v[2 * k] = mul2(v[2 * k], f0);
      v[2 * k + 1] = mul2(v[2 * k + 1], f1);
    }
  }
}

#ifndef KSMEM
#define KSMEM 440
#endif
// Stages of the ring: up to three while 512 threads an SM (what the registers
// allow) still fit its shared memory.
constexpr int kParamBytes = kElems * 4, kThreadBytes = KSMEM;
constexpr int ring_stages(int stage_bytes, int param_bytes) {
  return 3 * stage_bytes + param_bytes <= kThreadBytes ? 3 : 2 * stage_bytes + param_bytes <= kThreadBytes ? 2 : 1;
}
template <int T, bool kAnywhere, bool kFull>
struct Forward {
  static constexpr int kStage = 2 * Ring<T, kAnywhere>::kWords * 16, kParams = (kFull ? 4 : 2) * kParamBytes;
  static constexpr int kStages = ring_stages(kStage, kParams), kBytes = kStages * kStage + kParams;
};
template <int T, bool kAnywhere>
struct Grad {
  static constexpr int kStage = 4 * Ring<T, kAnywhere>::kWords * 16, kParams = 2 * kParamBytes;
  static constexpr int kStages = ring_stages(kStage, kParams), kBytes = kStages * kStage + kParams;
};
// f32 rows that start anywhere need more than 512 threads' share: 256 threads.
constexpr int norm_threads(int type) { return type == kF32 ? 256 : kTeamThreads; }

// kFull: layer norms or biases too; a plain rms norm drops that code.
template <int T, bool kAnywhere, bool kFull, bool kDrop>
__global__ void __launch_bounds__(norm_threads(T)) norm_rows_kernel(const __grid_constant__ NormArgs a) {
  constexpr int P = kElems / 2, S = Forward<T, kAnywhere, kFull>::kStages, kWords = Ring<T, kAnywhere>::kWords;
  extern __shared__ uint4 dynamic[];
  __shared__ TeamRecords<1> sh[4];
  const Team t = team_of(a.shape.warp_teams);
  const Columns<T, kAnywhere> col(t, a);
  const uint32_t teams = blockDim.x / t.threads;
  // rows of a warp's teams follow one another: a warp goes on while its first has a row
  const uint32_t team = a.shape.warp_teams ? threadIdx.x / t.threads : 0;
  const uint64_t step = a.shape.warp_teams ? uint64_t(gridDim.x) * teams : gridDim.x / t.ctas;
  uint64_t row = a.shape.warp_teams ? uint64_t(blockIdx.x) * teams + team : blockIdx.x / t.ctas;
  const uint32_t ahead = a.shape.warp_teams ? t.lane / t.lanes : 0;  // rows this team is ahead of its warp's first
  const float inv_cols = 1.0f / float(a.cols);
  const bool factor_on = a.post || a.gated || kDrop;
  const uint32_t pitch = col.pitch, ring = shared_address(dynamic) + threadIdx.x * 16;
  const uint32_t array = uint32_t(kWords) * pitch, stage_bytes = 2 * array, params = ring + S * stage_bytes;
  const ParamSlot pre{params, pitch}, fac{params + kElems / 4 * pitch, pitch}, pre_b{params + 2 * (kElems / 4) * pitch, pitch},
      fac_b{params + 3 * (kElems / 4) * pitch, pitch};
  const uint64_t bytes = a.rows * a.cols * uint64_t(dtype_bytes(T)), advance = step * a.cols * uint64_t(dtype_bytes(T));
  pdl_enter();
  team_start(t);
  DropRun run{};
  if constexpr (kDrop) run = drop_run(a.drop, a.seed);
  uint64_t next_row = row, next = col.offset(row);  // to be fetched
  auto fetch = [&](uint32_t slot) {
    if (next_row < a.rows) {
      col.fetch(a.x, next, bytes, slot);
      if (a.branch) col.fetch(a.y, next, bytes, slot + array);
    }
    copy_async_commit();
    next_row += step;
    next += advance;
  };
#pragma unroll
  for (int s = 0; s < S; ++s) {
    col.clear(ring + s * stage_bytes);
    col.clear(ring + s * stage_bytes + array);
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(ring + s * stage_bytes);
  {
    float f[kElems];
    col.params(a.w_pre, a.ptype, 0, 1.0f, f);
    pre.write(f);
    if constexpr (kFull) {
      col.params(a.b_pre, a.ptype, 0, 0.0f, f);
      pre_b.write(f);
    }
  }
  uint64_t group_end = 0;  // the factors in shared memory are those of the rows before it
  uint32_t slot = ring, free_slot = ring + (S - 1) * stage_bytes;
  uint64_t off = col.offset(row);
  for (int parity = 0; row - ahead < a.rows; row += step, off += advance, parity ^= 1) {
    const bool on = row < a.rows;
    fetch(free_slot);
    if (a.branch && on && row >= group_end) {
      // post weight, gate and the dropout's scale as one factor
      const uint64_t group = row / a.rows_per_group;
      group_end = (group + 1) * a.rows_per_group;
      float g[kElems], f[kElems];
      col.params(a.gate, a.ptype, group * a.cols, 1.0f, g);
      col.params(a.w_post, a.ptype, 0, 1.0f, f);
      const float scale = kDrop ? run.scale : 1.0f;
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        g[e] *= scale;
        f[e] *= g[e];
      }
      fac.write(f);
      if constexpr (kFull) {
        col.params(a.b_post, a.ptype, 0, 0.0f, f);
#pragma unroll
        for (int e = 0; e < kElems; ++e) f[e] *= g[e];
        fac_b.write(f);
      }
    }
    copy_async_wait<S - 1>();
    uint64_t h[P];
    const bool writer = on && t.tid == 0 && t.rank == 0;
    if (a.branch) {
      uint64_t n[P];
      col.read(slot + array, a.y, off, n);
      if (a.post) {
        float mean, rstd;
        row_stats(t, col, sh[0], sh[1], parity, kFull && a.layer, inv_cols, a.eps, n, mean, rstd);
        if (writer) {
          if (kFull && a.layer) a.stats_post[2 * row] = mean;
          a.stats_post[kFull && a.layer ? 2 * row + 1 : row] = rstd;
        }
        const uint64_t r2 = both(rstd);
#pragma unroll
        for (int k = 0; k < P; ++k) n[k] = mul2(n[k], r2);
      }
      if (factor_on) scale_by<kFull>(n, fac, fac_b);
      if constexpr (kDrop) col.drop(run, off, n);
      const uint64_t alpha = both(a.alpha);
      col.read(slot, a.x, off, h);
#pragma unroll
      for (int k = 0; k < P; ++k) h[k] = fma2(alpha, h[k], n[k]);
      col.put(t, a.h, off, on, h);
    } else {
      col.read(slot, a.x, off, h);
    }
    if (a.pre) {
      float mean, rstd;
      row_stats(t, col, sh[2], sh[3], parity, kFull && a.layer, inv_cols, a.eps, h, mean, rstd);
      if (writer) {
        if (kFull && a.layer) a.stats_pre[2 * row] = mean;
        a.stats_pre[kFull && a.layer ? 2 * row + 1 : row] = rstd;
      }
      const uint64_t r2 = both(rstd);
#pragma unroll
      for (int k = 0; k < P; ++k) h[k] = mul2(h[k], r2);
      scale_by<kFull>(h, pre, pre_b);
      col.put(t, a.u, off, on, h);
    }
    free_slot = slot;  // read by its own thread alone, and that is done
    slot = slot == ring + (S - 1) * stage_bytes ? ring : slot + stage_bytes;
  }
}

// A team takes a chunk of one group's rows and leaves its column sums in
// a.partial, [kind][group * chunks + chunk][cols].
template <int T, bool kAnywhere, bool kFull, bool kDrop>
__global__ void __launch_bounds__(norm_threads(T)) norm_grad_kernel(const __grid_constant__ NormArgs a, const NormSums kinds) {
  constexpr int E = kElems, P = E / 2, V = act_vec<T>(), Q = E / V, S = Grad<T, kAnywhere>::kStages,
                kWords = Ring<T, kAnywhere>::kWords, N = kFull ? 2 : 1;
  extern __shared__ uint4 dynamic[];
  __shared__ TeamRecords<N> sh[2];
  const Team t = team_of(a.shape.warp_teams);
  const Columns<T, kAnywhere> col(t, a);
  const uint32_t teams = a.shape.warp_teams ? blockDim.x / t.threads : 1, team = a.shape.warp_teams ? threadIdx.x / t.threads : 0;
  const uint32_t ahead = a.shape.warp_teams ? t.lane / t.lanes : 0;
  const uint32_t place = blockIdx.x / t.ctas;  // this CTA's (or cluster's) chunk among all
  const uint32_t group = place / a.chunks, chunk = place % a.chunks;
  const uint64_t begin = uint64_t(group) * a.rows_per_group + a.rows_per_group * chunk / a.chunks;
  const uint64_t end = uint64_t(group) * a.rows_per_group + a.rows_per_group * (chunk + 1) / a.chunks;
  const float inv_cols = 1.0f / float(a.cols);
  const bool need_y = a.branch && (a.post || a.gated);
  const uint32_t pitch = col.pitch, ring = shared_address(dynamic) + threadIdx.x * 16;
  const uint32_t array = uint32_t(kWords) * pitch, stage_bytes = 4 * array, params = ring + S * stage_bytes;
  const ParamSlot pre{params, pitch}, fac{params + E / 4 * pitch, pitch};
  const uint64_t bytes = a.rows * a.cols * uint64_t(dtype_bytes(T)), advance = teams * uint64_t(a.cols) * dtype_bytes(T);
  pdl_enter();
  team_start(t);
  DropRun run{};
  if constexpr (kDrop) run = drop_run(a.drop, a.seed);
  uint64_t row = begin + team, next_row = row, next = col.offset(row), off = next;
  auto fetch = [&](uint32_t slot) {
    if (next_row < end) {
      if (a.branch) col.fetch(a.dh, next, bytes, slot);
      if (a.pre) {
        col.fetch(a.du, next, bytes, slot + array);
        col.fetch(a.h_in, next, bytes, slot + 2 * array);
      }
      if (need_y) col.fetch(a.y, next, bytes, slot + 3 * array);
    }
    copy_async_commit();
    next_row += teams;
    next += advance;
  };
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int k = 0; k < 4; ++k) col.clear(ring + s * stage_bytes + k * array);
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(ring + s * stage_bytes);
  // post weight, gate and dropout scale as one factor; the scale of the sums
  // over dropped gradients is applied once, to the sums
  const float scale = kDrop ? run.scale : 1.0f;
  {
    float f[E], g[E];
    col.params(a.w_pre, a.ptype, 0, 1.0f, f);
    pre.write(f);
    col.params(a.w_post, a.ptype, 0, 1.0f, f);
    col.params(a.gate, a.ptype, uint64_t(group) * a.cols, 1.0f, g);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] *= g[e] * scale;
    fac.write(f);
  }
  uint64_t acc_t[P] = {}, acc_p[P] = {}, acc_s[kFull ? P : 1] = {}, acc_q[kFull ? P : 1] = {};
  uint32_t slot = ring, free_slot = ring + (S - 1) * stage_bytes;
  for (int parity = 0; row - ahead < end; row += teams, off += advance, parity ^= 1) {
    const bool on = row < end;  // a row that is not there counts as zeros
    float mean_h = 0.0f, rstd_h = 0.0f, mean_y = 0.0f, rstd_y = 0.0f;
    if (a.pre && on) {
      if (kFull && a.layer) mean_h = __ldg(a.stats_pre_in + 2 * row);
      rstd_h = __ldg(a.stats_pre_in + (kFull && a.layer ? 2 * row + 1 : row));
    }
    if (a.post && on) {
      if (kFull && a.layer) mean_y = __ldg(a.stats_post_in + 2 * row);
      rstd_y = __ldg(a.stats_post_in + (kFull && a.layer ? 2 * row + 1 : row));
    }
    fetch(free_slot);
    copy_async_wait<S - 1>();
    uint64_t g[P] = {};
    if (a.pre) {
      uint64_t du[P], hh[P];
      col.read(slot + array, a.du, off, du);
      col.read(slot + 2 * array, a.h_in, off, hh);
      if (!on) {
#pragma unroll
        for (int k = 0; k < P; ++k) du[k] = hh[k] = 0;
      }
      if (kFull && a.layer) col.center(mean_h, hh);
      const uint64_t r2 = both(rstd_h);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        hh[k] = mul2(hh[k], r2);
        acc_p[k] = fma2(du[k], hh[k], acc_p[k]);
        if constexpr (kFull) acc_q[k] = add2(acc_q[k], du[k]);
      }
      scale_by<false>(du, pre, pre);
      float s[N];
      s[0] = dot(du, hh);
      if constexpr (kFull) s[1] = a.layer ? total(du) : 0.0f;
      team_sum<N>(t, sh[0], parity, s);
      const uint64_t k2 = both(-s[0] * inv_cols);
      if (a.branch) col.read(slot, a.dh, off, g);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        uint64_t v = fma2(hh[k], k2, du[k]);
        if constexpr (kFull) v = add2(v, both(-s[1] * inv_cols));
        g[k] = fma2(r2, v, g[k]);
      }
    } else if (a.branch) {
      col.read(slot, a.dh, off, g);
    }
    if (!on) {
#pragma unroll
      for (int k = 0; k < P; ++k) g[k] = 0;
    }
    {
      const uint64_t alpha = both(a.alpha);
      uint64_t o[P];
#pragma unroll
      for (int k = 0; k < P; ++k) o[k] = mul2(alpha, g[k]);
      col.put(t, a.dx, off, on, o);
    }
    if (a.branch) {
      if constexpr (kDrop) col.drop(run, off, g);
      uint64_t yy[P] = {};
      if (need_y) {
        col.read(slot + 3 * array, a.y, off, yy);
        if (!on) {
#pragma unroll
          for (int k = 0; k < P; ++k) yy[k] = 0;
        }
        if (a.post) {
          if (kFull && a.layer) col.center(mean_y, yy);
          const uint64_t r2 = both(rstd_y);
#pragma unroll
          for (int k = 0; k < P; ++k) yy[k] = mul2(yy[k], r2);
        }
#pragma unroll
        for (int k = 0; k < P; ++k) {
          acc_t[k] = fma2(g[k], yy[k], acc_t[k]);
          if constexpr (kFull) acc_s[k] = add2(acc_s[k], g[k]);
        }
      }
      scale_by<false>(g, fac, fac);
      if (a.post) {
        float s[N];
        s[0] = dot(g, yy);
        if constexpr (kFull) s[1] = a.layer ? total(g) : 0.0f;
        team_sum<N>(t, sh[1], parity, s);
        const uint64_t r2 = both(rstd_y), k2 = both(-s[0] * inv_cols);
#pragma unroll
        for (int k = 0; k < P; ++k) {
          uint64_t v = fma2(yy[k], k2, g[k]);
          if constexpr (kFull) v = add2(v, both(-s[1] * inv_cols));
          g[k] = mul2(r2, v);
        }
      }
      col.put(t, a.dy, off, on, g);
    }
    free_slot = slot;
    slot = slot == ring + (S - 1) * stage_bytes ? ring : slot + stage_bytes;
  }
  // the team's column sums; teams that share a CTA are added in their order,
  // through shared memory (the ring is done with)
  const uint64_t places = uint64_t(a.groups) * a.chunks;
  float* const joined = reinterpret_cast<float*>(dynamic);
  copy_async_wait<0>();
  __syncthreads();
  auto put = [&](const uint64_t (&pairs)[P], float by, int kind) {
    float v[E];
#pragma unroll
    for (int k = 0; k < P; ++k) {
      unpack2(pairs[k], v[2 * k], v[2 * k + 1]);
      v[2 * k] *= by;
      v[2 * k + 1] *= by;
    }
    float* out = a.partial + (uint64_t(kind) * places + place) * a.cols;
    if (!a.shape.warp_teams) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < col.count(q)) out[col.at(q) + j] = v[q * V + j];
      return;
    }
    for (uint32_t w = 0; w < teams; ++w) {
      if (team == w) {
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j < col.count(q)) {
              float* at = joined + col.at(q) + j;
              *at = w ? *at + v[q * V + j] : v[q * V + j];
            }
      }
      __syncthreads();
    }
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) out[c] = joined[c];
    __syncthreads();
  };
  int kind = 0;
  if (kinds.t) put(acc_t, scale, kind++);
  if constexpr (kFull) {
    if (kinds.s) put(acc_s, scale, kind++);
  }
  if (kinds.p) put(acc_p, 1.0f, kind++);
  if constexpr (kFull) {
    if (kinds.q) put(acc_q, 1.0f, kind++);
  }
}

// Join of the partial column sums in place order: 32 columns a CTA, 32 warps
// sharing the places of a group (few groups) or the groups (many).
constexpr int kJoinWarps = 32;
constexpr uint32_t kJoinFewGroups = 32;

__global__ void __launch_bounds__(32 * kJoinWarps) norm_grad_join_kernel(const NormArgs a, const NormSums kinds) {
  __shared__ float red[2][kJoinWarps][33];
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const uint64_t c = uint64_t(blockIdx.x) * 32 + lane;
  const bool in = c < a.cols;
  const uint64_t places = uint64_t(a.groups) * a.chunks;
  pdl_enter();
  const float* sum_t = a.partial;
  const float* sum_s = a.partial + uint64_t(kinds.t) * places * a.cols;
  const float* sum_p = a.partial + uint64_t(int(kinds.t) + int(kinds.s)) * places * a.cols;
  const float* sum_q = sum_p + uint64_t(kinds.p) * places * a.cols;
  // sum over `n` places from `first`, every `by`-th
  auto gather = [&](const float* s, uint64_t first, uint64_t n, uint64_t begin, uint64_t by) {
    float v = 0.0f;
    if (in) {
#pragma unroll 4
      for (uint64_t k = begin; k < n; k += by) v += s[(first + k) * a.cols + c];
    }
    return v;
  };
  // over the warps, in order; the total in every warp's lane
  auto across = [&](float x, float y, float& sx, float& sy) {
    red[0][warp][lane] = x;
    red[1][warp][lane] = y;
    __syncthreads();
    sx = sy = 0.0f;
    for (int w = 0; w < kJoinWarps; ++w) {
      sx += red[0][w][lane];
      sy += red[1][w][lane];
    }
    __syncthreads();
  };
  auto param = [&](const void* p, uint64_t i) {
    float v[1] = {0.0f};
    if (in && p) param_load<1>(p, a.ptype, i, v);
    return v[0];
  };
  if (kinds.t) {
    const float w = a.post ? param(a.w_post, c) : 1.0f;
    const float b = a.post && a.bias && a.gated ? param(a.b_post, c) : 0.0f;
    float dw = 0.0f, db = 0.0f;
    auto group_out = [&](uint64_t g, float st, float ss) {
      const float gate = a.gated ? param(a.gate, g * a.cols + c) : 1.0f;
      dw = __fmaf_rn(gate, st, dw);
      db = __fmaf_rn(gate, ss, db);
      return __fmaf_rn(w, st, b * ss);
    };
    if (a.groups <= kJoinFewGroups) {
      for (uint64_t g = 0; g < a.groups; ++g) {
        float st, ss;
        across(gather(sum_t, g * a.chunks, a.chunks, warp, kJoinWarps),
               kinds.s ? gather(sum_s, g * a.chunks, a.chunks, warp, kJoinWarps) : 0.0f, st, ss);
        const float dg = group_out(g, st, ss);
        if (a.gated && in && warp == 0) a.dgate[g * a.cols + c] = dg;
      }
    } else {
      for (uint64_t g = warp; g < a.groups; g += kJoinWarps) {
        const float st = gather(sum_t, g * a.chunks, a.chunks, 0, 1);
        const float ss = kinds.s ? gather(sum_s, g * a.chunks, a.chunks, 0, 1) : 0.0f;
        const float dg = group_out(g, st, ss);
        if (a.gated && in) a.dgate[g * a.cols + c] = dg;
      }
      across(dw, db, dw, db);
    }
    if (a.post && in && warp == 0) {
      a.dw_post[c] = dw;
      if (a.bias) a.db_post[c] = db;
    }
  }
  if (kinds.p) {
    float sp, sq;
    across(gather(sum_p, 0, places, warp, kJoinWarps), kinds.q ? gather(sum_q, 0, places, warp, kJoinWarps) : 0.0f, sp,
           sq);
    if (in && warp == 0) {
      a.dw_pre[c] = sp;
      if (a.bias) a.db_pre[c] = sq;
    }
  }
}

struct Chosen {
  const void* kernel;
  unsigned shared_bytes;
};
template <int T, bool kAnywhere, bool kFull, bool kDrop>
Chosen choice(const NormArgs& a, bool grad) {
  const unsigned threads = unsigned(a.shape.threads);
  if (grad) return {(const void*)norm_grad_kernel<T, kAnywhere, kFull, kDrop>, threads * unsigned(Grad<T, kAnywhere>::kBytes)};
  return {(const void*)norm_rows_kernel<T, kAnywhere, kFull, kDrop>, threads * unsigned(Forward<T, kAnywhere, kFull>::kBytes)};
}
template <int T, bool kAnywhere>
Chosen choice_of_switches(const NormArgs& a, bool grad) {
  if (a.layer || a.bias)
    return a.drop.on ? choice<T, kAnywhere, true, true>(a, grad) : choice<T, kAnywhere, true, false>(a, grad);
  return a.drop.on ? choice<T, kAnywhere, false, true>(a, grad) : choice<T, kAnywhere, false, false>(a, grad);
}
template <int T>
Chosen choice_of_type(const NormArgs& a, bool grad, bool aligned) {
  return aligned ? choice_of_switches<T, false>(a, grad) : choice_of_switches<T, true>(a, grad);
}
// The kernel of a step, its shared memory allowed (above 48 KB that has to be asked for).
cudaError_t choose(const NormArgs& a, bool grad, bool aligned, Chosen* c) {
  *c = a.type == kF32   ? choice_of_type<kF32>(a, grad, aligned)
       : a.type == kF16 ? choice_of_type<kF16>(a, grad, aligned) : choice_of_type<kBF16>(a, grad, aligned);
  return c->shared_bytes <= 32 * 1024
             ? cudaSuccess
             : cudaFuncSetAttribute(c->kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(c->shared_bytes));
}

}  // namespace

TeamShape norm_shape(uint64_t cols, int type) {
  TeamShape s{0, kWarpTeamThreads, 1, kElems};
  if (cols <= 32 * kElems) {
    s.warp_teams = 4;
    while (cols > uint64_t(s.warp_teams) * kElems) s.warp_teams *= 2;
    return s;
  }
  while (cols > uint64_t(norm_threads(type)) * kElems * s.ctas) s.ctas *= 2;
  const uint64_t per = uint64_t(kElems) * s.ctas;
  s.threads = int((((cols + per - 1) / per) + 31) / 32 * 32);
  return s;
}

NormSums norm_sums(const NormArgs& a) {
  return NormSums{a.branch && (a.post || a.gated), a.post && a.bias, bool(a.pre), a.pre && a.bias};
}

cudaError_t norm_occupancy(const NormArgs& a, bool grad, int* blocks_per_sm) {
  Chosen c;
  const cudaError_t e = choose(a, grad, a.cols % (a.type == kF32 ? 4 : 8) == 0, &c);
  if (e != cudaSuccess) return e;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(blocks_per_sm, c.kernel, a.shape.threads, c.shared_bytes);
}

cudaError_t norm_launch(const NormArgs& a, bool aligned, int grid, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  Chosen c;
  const cudaError_t e = choose(a, false, aligned, &c);
  if (e != cudaSuccess) return e;
  NormArgs args = a;
  void* params[] = {&args};
  return launch_rows(c.kernel, a.shape, unsigned(grid), c.shared_bytes, params, stream);
}

cudaError_t norm_grad_launch(const NormArgs& a, bool aligned, cudaStream_t stream) {
  NormArgs args = a;
  NormSums kinds = norm_sums(a);
  if (a.rows) {
    Chosen c;
    cudaError_t e = choose(a, true, aligned, &c);
    if (e != cudaSuccess) return e;
    void* params[] = {&args, &kinds};
    e = launch_rows(c.kernel, a.shape, a.groups * a.chunks * unsigned(a.shape.ctas), c.shared_bytes, params, stream);
    if (e != cudaSuccess) return e;
  } else {
    args.chunks = 0;  // the column sums of no rows are zero
  }
  if (kinds.count() == 0) return cudaSuccess;
  (void)launch_pdl(&norm_grad_join_kernel, dim3((a.cols + 31) / 32), dim3(32 * kJoinWarps), stream, args, kinds);
  return cudaGetLastError();
}

}  // namespace askb
