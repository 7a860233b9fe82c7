// Block norms, gradient (norm_rows.cuh has the forward map).  With dh and du the
// gradients to h and u:
//   a = w_pre du;  G = dh + r (a - [mean a] - hhat mean(a hhat));  dx = alpha G
//   B = D(G);  c = w_post g B;  dy = r (c - [mean c] - yhat mean(c yhat))
//   T = sum B yhat, S = sum B over a group's rows; P = sum du hhat, Q = sum du
//   dgate = w_post T + b_post S;  dw_post = sum over groups g T;  db_post = sum g S
//   dw_pre = P;  db_pre = Q
// ([..]: layer norm only; without a post norm yhat is y and dy = g B.)  One
// sum over a group's rows thus serves both the gate's gradient and the
// weight's.  A CTA keeps the sums of its rows' columns in registers, leaves them
// once in scratch, and a second kernel joins the CTAs' sums in order.
#include "norm_rows.cuh"

namespace askb {

namespace {

template <int T, int F>
struct Layout {
  static constexpr int kStage = 4 * Columns<T, F>::kArrayBytes, kParams = 2 * kParamBytes;
  static constexpr int kStages = ring_stages(kStage, kParams), kBytes = kStages * kStage + kParams;
};

// A CTA (or cluster) takes a chunk of one group's rows and leaves its column
// sums in a.partial, [kind][group * chunks + chunk][cols].
template <int T, int F, int kForm, bool kFull, bool kDrop>
__global__ void __launch_bounds__(kTeamThreads) norm_grad_kernel(const __grid_constant__ NormArgs a, const NormSums kinds) {
  using Cols = Columns<T, F>;
  using Shape = Layout<T, F>;
  constexpr int E = kElems, P = kPairs, V = Cols::V, Q = Cols::Q, S = Shape::kStages, N = kFull ? 2 : 1;
  const bool branch = kForm == FORM_ANY ? a.branch : kForm != FORM_NORM;
  const bool post = kForm == FORM_ANY ? a.post : kForm == FORM_BOTH;
  const bool pre = kForm == FORM_ANY ? a.pre : true;
  const bool need_y = kForm == FORM_ANY ? a.branch && (a.post || a.gated) : kForm == FORM_BOTH;
  const bool factors = kForm == FORM_ANY || kForm == FORM_BOTH;
  extern __shared__ uint4 dynamic[];
  __shared__ TeamRecords<N> sh[2];
  const Team t = team_of(a.shape);
  const Cols col(t, a);
  const uint32_t place = blockIdx.x / t.ctas, group = place / a.chunks, chunk = place % a.chunks;
  const uint64_t begin = uint64_t(group) * a.rows_per_group + a.rows_per_group * chunk / a.chunks;
  const uint64_t end = uint64_t(group) * a.rows_per_group + a.rows_per_group * (chunk + 1) / a.chunks;
  uint64_t row = begin + t.index;
  const uint32_t mine = row < end ? uint32_t((end - row + t.count - 1) / t.count) : 0;
  const uint32_t turns = __shfl_sync(0xffffffffu, mine, 0);  // of the warp: its first team has the most rows
  const float inv_cols = 1.0f / float(a.cols);
  const uint32_t ring = Cols::ring(dynamic), array = blockDim.x * uint32_t(Cols::kArrayBytes), stage_bytes = 4 * array;
  const uint32_t pitch = blockDim.x * 16, params = shared_address(dynamic) + S * stage_bytes + threadIdx.x * 16;
  const ParamSlot pre_w{params, pitch}, fac{params + E / 4 * pitch, pitch};
  const uint64_t bytes = a.rows * a.cols * uint64_t(Cols::B), advance = t.count * uint64_t(a.cols) * Cols::B;
  pdl_enter();
  team_start(t);
  DropRun run{};
  if constexpr (kDrop) run = drop_run(a.drop, a.seed);
  uint64_t off = col.offset(row);
  auto fetch = [&](uint32_t turn, uint64_t at, uint32_t slot) {
    if (turn < mine) {
      if (branch) col.fetch(a.dh, at, bytes, slot);
      if (pre) {
        col.fetch(a.du, at, bytes, slot + array);
        col.fetch(a.h_in, at, bytes, slot + 2 * array);
      }
      if (need_y) col.fetch(a.y, at, bytes, slot + 3 * array);
    }
    copy_async_commit();
  };
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int k = 0; k < 4; ++k) col.clear(ring + s * stage_bytes + k * array);
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s, off + s * advance, ring + s * stage_bytes);
  // post weight, gate and dropout scale as one factor; the scale of the sums
  // over dropped gradients is applied once, to the sums
  const float scale = kDrop ? run.scale : 1.0f;
  {
    float f[E], g[E];
    if (pre) {
      col.params(a.w_pre, a.ptype, 0, 1.0f, f);
      pre_w.write(f);
    }
    if (factors) {
      col.params(a.w_post, a.ptype, 0, 1.0f, f);
      col.params(a.gate, a.ptype, uint64_t(group) * a.cols, 1.0f, g);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] *= g[e] * scale;
      fac.write(f);
    }
  }
  uint64_t acc_t[P] = {}, acc_p[P] = {}, acc_s[kFull ? P : 1] = {}, acc_q[kFull ? P : 1] = {};
  uint32_t slot = ring, free_slot = ring + (S - 1) * stage_bytes;
  for (uint32_t turn = 0; turn < turns; ++turn, row += t.count, off += advance) {
    const int parity = int(turn & 1u);
    const bool on = turn < mine;  // a row that is not there counts as zeros
    float mean_h = 0.0f, rstd_h = 0.0f, mean_y = 0.0f, rstd_y = 0.0f;
    if (pre && on) {
      if (kFull && a.layer) mean_h = __ldg(a.stats_pre_in + 2 * row);
      rstd_h = __ldg(a.stats_pre_in + (kFull && a.layer ? 2 * row + 1 : row));
    }
    if (post && on) {
      if (kFull && a.layer) mean_y = __ldg(a.stats_post_in + 2 * row);
      rstd_y = __ldg(a.stats_post_in + (kFull && a.layer ? 2 * row + 1 : row));
    }
    fetch(turn + S - 1, off + (S - 1) * advance, free_slot);
    copy_async_wait<S - 1>();
    uint64_t g[P];
    if (pre) {
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
      scale_by<false>(du, pre_w, pre_w);
      float s[N];
      s[0] = dot(du, hh);
      if constexpr (kFull) s[1] = a.layer ? total(du) : 0.0f;
      team_sum<N>(t, sh[0], parity, s);
      const uint64_t k2 = both(-s[0] * inv_cols);
      if (branch) {
        col.read(slot, a.dh, off, g);
      } else {
#pragma unroll
        for (int k = 0; k < P; ++k) g[k] = 0;
      }
#pragma unroll
      for (int k = 0; k < P; ++k) {
        uint64_t v = fma2(hh[k], k2, du[k]);
        if constexpr (kFull) v = add2(v, both(-s[1] * inv_cols));
        g[k] = fma2(r2, v, g[k]);
      }
    } else {
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
    if (branch) {
      if constexpr (kDrop) col.drop(run, off, g);
      if (need_y) {
        uint64_t yy[P];
        col.read(slot + 3 * array, a.y, off, yy);
        if (!on) {
#pragma unroll
          for (int k = 0; k < P; ++k) yy[k] = 0;
        }
        if (post) {
          if (kFull && a.layer) col.center(mean_y, yy);
          scale_all(yy, rstd_y);
        }
#pragma unroll
        for (int k = 0; k < P; ++k) {
          acc_t[k] = fma2(g[k], yy[k], acc_t[k]);
          if constexpr (kFull) acc_s[k] = add2(acc_s[k], g[k]);
        }
        scale_by<false>(g, fac, fac);
        if (post) {
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
      } else if (factors) {
        scale_by<false>(g, fac, fac);
      } else if (kDrop) {
        scale_all(g, scale);
      }
      col.put(t, a.dy, off, on, g);
    }
    free_slot = slot;
    slot = slot == ring + (S - 1) * stage_bytes ? ring : slot + stage_bytes;
  }
  // The column sums: teams of one warp are added by shuffles, the warps or teams
  // of a CTA one after the other in shared memory (the ring is done with).
  const uint64_t places = uint64_t(a.groups) * a.chunks;
  float* const joined = reinterpret_cast<float*>(dynamic);
  const uint32_t order = a.shape.warp_teams ? threadIdx.x >> 5 : t.index;
  const uint32_t holders = a.shape.warp_teams ? blockDim.x >> 5 : t.count;
  copy_async_wait<0>();
  __syncthreads();
  auto put = [&](const uint64_t (&pairs)[P], float by, int kind) {
    float v[E];
    Cols::unpack(pairs, v);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= by;
    float* out = a.partial + (uint64_t(kind) * places + place) * a.cols;
    if (a.shape.warp_teams) {
#pragma unroll
      for (int d = 16; d >= 4; d >>= 1) {
        if (uint32_t(d) < t.lanes) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += __shfl_xor_sync(0xffffffffu, v[e], d);
      }
    } else if (holders == 1) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < col.count(q)) out[col.at(q) + j] = v[q * V + j];
      return;
    }
    for (uint32_t w = 0; w < holders; ++w) {
      if (order == w && t.lane < t.lanes) {
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

template <int T, int F, int kForm, bool kFull, bool kDrop>
struct Pick {
  static Chosen get(unsigned threads) {
    return {(const void*)norm_grad_kernel<T, F, kForm, kFull, kDrop>, threads * unsigned(Layout<T, F>::kBytes)};
  }
};

}  // namespace

NormSums norm_sums(const NormArgs& a) {
  return NormSums{a.branch && (a.post || a.gated), a.post && a.bias, bool(a.pre), a.pre && a.bias};
}

cudaError_t norm_grad_occupancy(const NormArgs& a, NormFit fit, int* blocks_per_sm) {
  const Chosen c = choose<Pick>(a, fit);
  const cudaError_t e = allow(c);
  if (e != cudaSuccess) return e;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(blocks_per_sm, c.kernel, a.shape.threads, c.shared_bytes);
}

cudaError_t norm_grad_launch(const NormArgs& a, NormFit fit, cudaStream_t stream) {
  NormArgs args = a;
  NormSums kinds = norm_sums(a);
  if (a.rows) {
    const Chosen c = choose<Pick>(a, fit);
    cudaError_t e = allow(c);
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
