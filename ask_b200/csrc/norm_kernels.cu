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

// Mean and 1 / sqrt(variance + eps) of the team's row; v is zero past cols.
template <int E, int V, class Valid>
__device__ __forceinline__ void row_stats(const Team& t, TeamRecords<1>& sh_mean, TeamRecords<1>& sh_sq, int parity,
                                          bool layer, float inv_cols, float eps, const float (&v)[E], Valid valid,
                                          float& mean, float& rstd) {
  mean = 0.0f;
  if (layer) {
    float s[1] = {0.0f};
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] += v[e];
    team_sum<1>(t, sh_mean, parity, s);
    mean = s[0] * inv_cols;
  }
  float s[1] = {0.0f};
#pragma unroll
  for (int q = 0; q < E / V; ++q) {
    const float m = valid(q) ? mean : 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = v[q * V + j] - m;
      s[0] = __fmaf_rn(d, d, s[0]);
    }
  }
  team_sum<1>(t, sh_sq, parity, s);
  rstd = __frsqrt_rn(__fmaf_rn(s[0], inv_cols, eps));
}

template <int T, int V, int E>
__global__ void __launch_bounds__(kTeamThreads) norm_rows_kernel(const NormArgs a) {
  constexpr int Q = E / V;
  __shared__ TeamRecords<1> sh[4];
  const bool warp_teams = a.shape.warp_teams;
  const Team t = team_of(warp_teams);
  const uint32_t teams = warp_teams ? blockDim.x >> 5 : 1;
  uint64_t row = warp_teams ? uint64_t(blockIdx.x) * teams + (threadIdx.x >> 5) : blockIdx.x / t.ctas;
  const uint64_t step = warp_teams ? uint64_t(gridDim.x) * teams : gridDim.x / t.ctas;
  auto column = [&](int q) { return ((t.rank * Q + q) * t.threads + t.tid) * uint32_t(V); };
  auto valid = [&](int q) { return column(q) < a.cols; };
  const float inv_cols = 1.0f / float(a.cols);
  pdl_enter();
  team_start(t);
  const DropRun run = drop_run(a.drop, a.seed);
  ActRaw<T, V> rx[Q], ry[Q];
  auto fetch = [&](uint64_t r) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      rx[q].zero();
      ry[q].zero();
      if (valid(q)) {
        rx[q].load(a.x, r * a.cols + column(q));
        if (a.branch) ry[q].load(a.y, r * a.cols + column(q));
      }
    }
  };
  if (row < a.rows) fetch(row);
  for (int parity = 0; row < a.rows; row += step, parity ^= 1) {
    float h[E], n[E];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      rx[q].widen(h + q * V);
      ry[q].widen(n + q * V);
    }
    if (row + step < a.rows) fetch(row + step);
    const bool writer = t.tid == 0 && t.rank == 0;
    if (a.branch) {
      if (a.post) {
        float mean, rstd;
        row_stats<E, V>(t, sh[0], sh[1], parity, a.layer, inv_cols, a.eps, n, valid, mean, rstd);
        if (writer) {
          if (a.layer) a.stats_post[2 * row] = mean;
          a.stats_post[a.layer ? 2 * row + 1 : row] = rstd;
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          if (!valid(q)) continue;
          float w[V];
          param_load<V>(a.w_post, a.ptype, column(q), w);
#pragma unroll
          for (int j = 0; j < V; ++j) n[q * V + j] = (n[q * V + j] - mean) * rstd * w[j];
          if (a.bias) {
            param_load<V>(a.b_post, a.ptype, column(q), w);
#pragma unroll
            for (int j = 0; j < V; ++j) n[q * V + j] += w[j];
          }
        }
      }
      const uint64_t group = a.groups > 1 ? row / a.rows_per_group : 0;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        if (!valid(q)) continue;
        if (a.gated) {
          float g[V];
          param_load<V>(a.gate, a.ptype, group * a.cols + column(q), g);
#pragma unroll
          for (int j = 0; j < V; ++j) n[q * V + j] *= g[j];
        }
        if (a.drop.on) drop_unit<V>(run, row * a.cols + column(q), n + q * V);
#pragma unroll
        for (int j = 0; j < V; ++j) h[q * V + j] = __fmaf_rn(a.alpha, h[q * V + j], n[q * V + j]);
        act_put<T, V>(a.h, row * a.cols + column(q), h + q * V);
      }
    }
    if (a.pre) {
      float mean, rstd;
      row_stats<E, V>(t, sh[2], sh[3], parity, a.layer, inv_cols, a.eps, h, valid, mean, rstd);
      if (writer) {
        if (a.layer) a.stats_pre[2 * row] = mean;
        a.stats_pre[a.layer ? 2 * row + 1 : row] = rstd;
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        if (!valid(q)) continue;
        float w[V], u[V];
        param_load<V>(a.w_pre, a.ptype, column(q), w);
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] = (h[q * V + j] - mean) * rstd * w[j];
        if (a.bias) {
          param_load<V>(a.b_pre, a.ptype, column(q), w);
#pragma unroll
          for (int j = 0; j < V; ++j) u[j] += w[j];
        }
        act_put<T, V>(a.u, row * a.cols + column(q), u);
      }
    }
  }
}

// A team takes a chunk of one group's rows and leaves its column sums in
// a.partial, [kind][group * chunks + chunk][cols].
template <int T, int V, int E, bool kBias>
__global__ void __launch_bounds__(kTeamThreads) norm_grad_kernel(const NormArgs a, const NormSums kinds) {
  constexpr int Q = E / V;
  __shared__ TeamRecords<2> sh[2];
  __shared__ float joined[32 * E];
  const bool warp_teams = a.shape.warp_teams;
  const Team t = team_of(warp_teams);
  const uint32_t teams = warp_teams ? blockDim.x >> 5 : 1, team = warp_teams ? threadIdx.x >> 5 : 0;
  const uint32_t place = blockIdx.x / t.ctas;  // this CTA's (or cluster's) chunk among all
  const uint32_t group = place / a.chunks, chunk = place % a.chunks;
  const uint64_t begin = uint64_t(group) * a.rows_per_group + a.rows_per_group * chunk / a.chunks;
  const uint64_t end = uint64_t(group) * a.rows_per_group + a.rows_per_group * (chunk + 1) / a.chunks;
  auto column = [&](int q) { return ((t.rank * Q + q) * t.threads + t.tid) * uint32_t(V); };
  auto valid = [&](int q) { return column(q) < a.cols; };
  const float inv_cols = 1.0f / float(a.cols);
  const bool need_y = a.branch && (a.post || a.gated);
  pdl_enter();
  team_start(t);
  const DropRun run = drop_run(a.drop, a.seed);
  float acc_t[E] = {}, acc_p[E] = {}, acc_s[kBias ? E : 1] = {}, acc_q[kBias ? E : 1] = {};
  ActRaw<T, V> rdh[Q], rdu[Q], rh[Q], ry[Q];
  float mean_h = 0.0f, rstd_h = 0.0f, mean_y = 0.0f, rstd_y = 1.0f;
  auto fetch = [&](uint64_t r) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      rdh[q].zero(); rdu[q].zero(); rh[q].zero(); ry[q].zero();
      if (!valid(q)) continue;
      const uint64_t at = r * a.cols + column(q);
      if (a.branch) rdh[q].load(a.dh, at);
      if (a.pre) {
        rdu[q].load(a.du, at);
        rh[q].load(a.h_in, at);
      }
      if (need_y) ry[q].load(a.y, at);
    }
    if (a.pre) {
      if (a.layer) mean_h = __ldg(a.stats_pre_in + 2 * r);
      rstd_h = __ldg(a.stats_pre_in + (a.layer ? 2 * r + 1 : r));
    }
    if (a.post) {
      if (a.layer) mean_y = __ldg(a.stats_post_in + 2 * r);
      rstd_y = __ldg(a.stats_post_in + (a.layer ? 2 * r + 1 : r));
    }
  };
  uint64_t row = begin + team;
  if (row < end) fetch(row);
  for (int parity = 0; row < end; row += teams, parity ^= 1) {
    float g[E], du[E], hh[E], yy[E];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      rdh[q].widen(g + q * V);
      rdu[q].widen(du + q * V);
      rh[q].widen(hh + q * V);
      ry[q].widen(yy + q * V);
    }
    const float mh = mean_h, sh_ = rstd_h, my = mean_y, sy = rstd_y;
    if (row + teams < end) fetch(row + teams);
    if (a.pre) {
      float s[2] = {0.0f, 0.0f};
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        if (!valid(q)) continue;
        float w[V];
        param_load<V>(a.w_pre, a.ptype, column(q), w);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int e = q * V + j;
          hh[e] = (hh[e] - mh) * sh_;
          acc_p[e] = __fmaf_rn(du[e], hh[e], acc_p[e]);
          if constexpr (kBias) acc_q[e] += du[e];
          du[e] *= w[j];
          s[0] = __fmaf_rn(du[e], hh[e], s[0]);
          s[1] += du[e];
        }
      }
      team_sum<2>(t, sh[0], parity, s);
      const float k = s[0] * inv_cols, m = a.layer ? s[1] * inv_cols : 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) g[e] = __fmaf_rn(sh_, du[e] - m - hh[e] * k, g[e]);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (!valid(q)) continue;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = a.alpha * g[q * V + j];
      act_put<T, V>(a.dx, row * a.cols + column(q), o);
    }
    if (a.branch) {
      float s[2] = {0.0f, 0.0f};
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        if (!valid(q)) continue;
        if (a.drop.on) drop_unit<V>(run, row * a.cols + column(q), g + q * V);
        float gate[V], w[V];
        if (a.gated) param_load<V>(a.gate, a.ptype, uint64_t(group) * a.cols + column(q), gate);
        if (a.post) param_load<V>(a.w_post, a.ptype, column(q), w);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int e = q * V + j;
          if (a.post) yy[e] = (yy[e] - my) * sy;
          acc_t[e] = __fmaf_rn(g[e], yy[e], acc_t[e]);
          if constexpr (kBias) acc_s[e] += g[e];
          if (a.gated) g[e] *= gate[j];
          if (a.post) {
            g[e] *= w[j];
            s[0] = __fmaf_rn(g[e], yy[e], s[0]);
            s[1] += g[e];
          }
        }
      }
      if (a.post) {
        team_sum<2>(t, sh[1], parity, s);
        const float k = s[0] * inv_cols, m = a.layer ? s[1] * inv_cols : 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) g[e] = sy * (g[e] - m - yy[e] * k);
      }
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (valid(q)) act_put<T, V>(a.dy, row * a.cols + column(q), g + q * V);
    }
  }
  // the team's column sums; warps of a CTA that were teams of their own are
  // added in warp order
  const uint64_t places = uint64_t(a.groups) * a.chunks;
  auto put = [&](const float* v, int kind) {
    float* out = a.partial + (uint64_t(kind) * places + place) * a.cols;
    if (!warp_teams) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (valid(q)) {
#pragma unroll
          for (int j = 0; j < V; ++j) out[column(q) + j] = v[q * V + j];
        }
      return;
    }
    for (uint32_t w = 0; w < teams; ++w) {
      if (team == w) {
#pragma unroll
        for (int q = 0; q < Q; ++q)
          if (valid(q)) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              float* at = joined + column(q) + j;
              *at = w ? *at + v[q * V + j] : v[q * V + j];
            }
          }
      }
      __syncthreads();
    }
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) out[c] = joined[c];
    __syncthreads();
  };
  int kind = 0;
  if (kinds.t) put(acc_t, kind++);
  if constexpr (kBias) {
    if (kinds.s) put(acc_s, kind++);
  }
  if (kinds.p) put(acc_p, kind++);
  if constexpr (kBias) {
    if (kinds.q) put(acc_q, kind++);
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

template <int T, int V>
const void* forward_kernel(int elems) {
  return elems == 8 ? (const void*)norm_rows_kernel<T, V, 8> : (const void*)norm_rows_kernel<T, V, 16>;
}
template <int T, int V>
const void* grad_kernel(bool bias) {
  return bias ? (const void*)norm_grad_kernel<T, V, 8, true> : (const void*)norm_grad_kernel<T, V, 8, false>;
}
template <int T>
const void* kernel_of_type(const NormArgs& a, bool grad, bool vec) {
  constexpr int V = act_vec<T>();
  if (grad) return vec ? grad_kernel<T, V>(a.bias) : grad_kernel<T, 1>(a.bias);
  return vec ? forward_kernel<T, V>(a.shape.elems) : forward_kernel<T, 1>(a.shape.elems);
}
const void* kernel_for(const NormArgs& a, bool grad, bool vec) {
  return a.type == kF32 ? kernel_of_type<kF32>(a, grad, vec)
         : a.type == kF16 ? kernel_of_type<kF16>(a, grad, vec) : kernel_of_type<kBF16>(a, grad, vec);
}

}  // namespace

TeamShape norm_shape(uint64_t cols, bool grad) {
  // The gradient keeps column sums beside four rows: 8 elements a thread, and
  // a cluster for rows beyond 4096 columns (16 elements spilled).
  TeamShape s{0, kWarpTeamThreads, 1, 8};
  if (!grad && cols > 32 * 8) s.elems = cols <= 32 * 16 ? 16 : cols <= 8 * kTeamThreads ? 8 : 16;
  if (cols <= uint64_t(32) * s.elems) {
    s.warp_teams = 1;
    return s;
  }
  while (cols > uint64_t(kTeamThreads) * s.elems * s.ctas) s.ctas *= 2;
  const uint64_t per = uint64_t(s.elems) * s.ctas;
  s.threads = int((((cols + per - 1) / per) + 31) / 32 * 32);
  return s;
}

NormSums norm_sums(const NormArgs& a) {
  return NormSums{a.branch && (a.post || a.gated), a.post && a.bias, bool(a.pre), a.pre && a.bias};
}

cudaError_t norm_occupancy(const NormArgs& a, bool grad, int* blocks_per_sm) {
  const uint64_t vec = a.type == kF32 ? 4 : 8;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(blocks_per_sm, kernel_for(a, grad, a.cols % vec == 0),
                                                       a.shape.threads, 0);
}

cudaError_t norm_launch(const NormArgs& a, bool vec, int grid, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  NormArgs args = a;
  void* params[] = {&args};
  return launch_rows(kernel_for(a, false, vec), a.shape, unsigned(grid), 0, params, stream);
}

cudaError_t norm_grad_launch(const NormArgs& a, bool vec, cudaStream_t stream) {
  NormArgs args = a;
  NormSums kinds = norm_sums(a);
  if (a.rows) {
    void* params[] = {&args, &kinds};
    const cudaError_t e = launch_rows(kernel_for(a, true, vec), a.shape,
                                      a.groups * a.chunks * unsigned(a.shape.ctas), 0, params, stream);
    if (e != cudaSuccess) return e;
  } else {
    args.chunks = 0;  // the column sums of no rows are zero
  }
  if (kinds.count() == 0) return cudaSuccess;
  (void)launch_pdl(&norm_grad_join_kernel, dim3((a.cols + 31) / 32), dim3(32 * kJoinWarps), stream, args, kinds);
  return cudaGetLastError();
}

}  // namespace askb
