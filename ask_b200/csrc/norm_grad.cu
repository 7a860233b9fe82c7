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
// once in scratch, and a second kernel joins the CTAs' sums in order: results do
// not depend on the order of execution.  What hhat and yhat hold where there is no
// column meets du = 0 and c = 0.  bf16 [32768, 4096] takes 338 us with
// dropout (4.8 TB/s) and 268 without; f16 [4099, 1000] layer norms 29.6 us: the
// latency of two dependent kernels, the join of 148 places 9 us of it.  Forms for
// layer norms or biases spill up to 340 bytes a thread at 128 registers, f32 by words most.
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
  const uint32_t place = blockIdx.x / t.ctas, group = place / a.chunks, chunk = place % a.chunks;
  const uint32_t stretch = chunk / a.spread, stretches = a.chunks / a.spread, stride = t.count * a.spread;
  const uint64_t begin = uint64_t(group) * a.rows_per_group + a.rows_per_group * stretch / stretches;
  const uint64_t end = uint64_t(group) * a.rows_per_group + a.rows_per_group * (stretch + 1) / stretches;
  // the teams of a warp add their column sums, so their rows begin at the same place of a unit
  const uint32_t warp = threadIdx.x >> 5, of_warp = 32u / t.lanes;
  const uint32_t order_in = a.shape.warp_teams
                                ? warp % a.classes + a.classes * (warp / a.classes * of_warp + t.index % of_warp)
                                : t.index;
  uint64_t row = begin + chunk % a.spread * t.count + order_in;
  const Cols col(t, a, row);
  const uint32_t mine = row < end ? uint32_t((end - row + stride - 1) / stride) : 0;
  const uint32_t turns = __shfl_sync(0xffffffffu, mine, 0);  // of the warp: its first team has the most rows
  const float inv_cols = 1.0f / float(a.cols);
  const uint32_t ring = Cols::ring(dynamic), array = blockDim.x * uint32_t(Cols::kArrayBytes), stage_bytes = 4 * array;
  const uint32_t pitch = blockDim.x * 16, params = shared_address(dynamic) + S * stage_bytes + threadIdx.x * 16;
  const ParamSlot pre_w{params, pitch}, fac{params + E / 4 * pitch, pitch};
  const uint64_t bytes = a.rows * a.cols * uint64_t(Cols::B), advance = stride * uint64_t(a.cols) * Cols::B;
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
  // a row's statistics, loaded one row ahead
  struct {
    float mean_h, rstd_h, mean_y, rstd_y;
  } stats;
  auto load_stats = [&](uint32_t turn, uint64_t r) {
    stats = {0.0f, 0.0f, 0.0f, 0.0f};
    if (turn >= mine) return;
    if (pre) {
      if (kFull && a.layer) stats.mean_h = __ldg(a.stats_pre_in + 2 * r);
      stats.rstd_h = __ldg(a.stats_pre_in + (kFull && a.layer ? 2 * r + 1 : r));
    }
    if (post) {
      if (kFull && a.layer) stats.mean_y = __ldg(a.stats_post_in + 2 * r);
      stats.rstd_y = __ldg(a.stats_post_in + (kFull && a.layer ? 2 * r + 1 : r));
    }
  };
  load_stats(0, row);
  uint64_t acc_t[P] = {}, acc_p[P] = {}, acc_s[kFull ? P : 1] = {}, acc_q[kFull ? P : 1] = {};
  uint32_t slot = ring, free_slot = ring + (S - 1) * stage_bytes;
  for (uint32_t turn = 0; turn < turns; ++turn, row += stride, off += advance) {
    const int parity = int(turn & 1u);
    const bool on = turn < mine;  // a row that is not there counts as zeros
    const float mean_h = stats.mean_h, rstd_h = stats.rstd_h, mean_y = stats.mean_y, rstd_y = stats.rstd_y;
    load_stats(turn + 1, row + stride);
    fetch(turn + S - 1, off + (S - 1) * advance, free_slot);
    copy_async_wait<S - 1>();
    col.trim(slot, 4, array);
    uint64_t g[P];
    if (pre) {
      uint64_t du[P], hh[P];
      col.template read<false>(slot + array, a.du, off, du);
      col.template read<false>(slot + 2 * array, a.h_in, off, hh);
      if (!on) {
#pragma unroll
        for (int k = 0; k < P; ++k) du[k] = hh[k] = 0;
      }
      if (kFull && a.layer) col.template center<false>(mean_h, hh);
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
      team_sum<N, true>(t, sh[0], parity, s);
      const uint64_t k2 = both(-s[0] * inv_cols);
      if (branch) {
        col.template read<false>(slot, a.dh, off, g);
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
      col.template read<false>(slot, a.dh, off, g);
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
        col.template read<false>(slot + 3 * array, a.y, off, yy);
        if (!on) {
#pragma unroll
          for (int k = 0; k < P; ++k) yy[k] = 0;
        }
        if (post) {
          if (kFull && a.layer) col.template center<false>(mean_y, yy);
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
          team_sum<N, true>(t, sh[1], parity, s);
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
  // The column sums: teams of one warp are added by shuffles; the warps or teams
  // of a CTA lay theirs side by side in shared memory (the ring is done with: it
  // held more), and the CTA adds them in order.
  const uint64_t places = uint64_t(a.groups) * a.chunks;
  float* const laid = reinterpret_cast<float*>(dynamic);
  const uint32_t order = a.shape.warp_teams ? threadIdx.x >> 5 : t.index;
  const uint32_t holders = a.shape.warp_teams ? blockDim.x >> 5 : t.count;
  const bool direct = !a.shape.warp_teams && holders == 1;
  const uint32_t lane_cols = direct ? 0 : (a.cols + 3u) & ~3u;
  copy_async_wait<0>();
  __syncthreads();
  auto put = [&](const uint64_t (&pairs)[P], float by, int kind) {
    float v[E];
    Cols::unpack(pairs, v);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= by;
    if (a.shape.warp_teams) {
#pragma unroll
      for (int d = 16; d >= 4; d >>= 1) {
        if (uint32_t(d) < t.lanes) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += __shfl_xor_sync(0xffffffffu, v[e], d);
      }
      if (t.lane >= t.lanes) return;
    }
    float* const to = direct ? a.partial + (uint64_t(kind) * places + place) * a.cols
                             : laid + (uint32_t(kind) * holders + order) * lane_cols;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (V % 4 == 0 && F == NORM_UNITS && (!direct || a.cols % 4 == 0)) {
        if (!col.in(q)) continue;
#pragma unroll
        for (int j = 0; j < V; j += 4)
          *reinterpret_cast<float4*>(to + col.at(q) + j) =
              make_float4(v[q * V + j], v[q * V + j + 1], v[q * V + j + 2], v[q * V + j + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (col.has(q, j)) to[col.at(q) + j] = v[q * V + j];
      }
    }
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
  if (direct) return;
  __syncthreads();
  for (int k = 0; k < kind; ++k)
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float* from = laid + uint32_t(k) * holders * lane_cols + c;
      float v = from[0];
      for (uint32_t w = 1; w < holders; ++w) v += from[w * lane_cols];
      a.partial[(uint64_t(k) * places + place) * a.cols + c] = v;
    }
}

// Join of the places' column sums, 32 columns a CTA, its warps sharing the places
// and adding what they found in warp order.  A CTA row (blockIdx.y) has one task:
// a group's gate gradient, the post norm's parameters (gate times the groups'
// sums), or the pre norm's.
constexpr int kJoinWarps = kNormJoinThreads;

__global__ void __launch_bounds__(32 * kJoinWarps) norm_grad_join_kernel(const __grid_constant__ NormArgs a,
                                                                         const NormSums kinds, const uint32_t gate_rows) {
  __shared__ float red[2][kJoinWarps][32];
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const uint64_t c = uint64_t(blockIdx.x) * 32 + lane;
  const bool in = c < a.cols;
  const uint64_t places = uint64_t(a.groups) * a.chunks;
  pdl_enter();
  const float* const sum_t = a.partial + c;
  const float* const sum_s = sum_t + uint64_t(kinds.t) * places * a.cols;
  const float* const sum_p = sum_s + uint64_t(kinds.s) * places * a.cols;
  const float* const sum_q = sum_p + uint64_t(kinds.p) * places * a.cols;
  auto param = [&](const void* p, uint64_t i, float fill) {
    float v[1] = {fill};
    if (in && p) param_load<1>(p, a.ptype, i, v);
    return v[0];
  };
  // x, y: sums over the places [first, first + n), each times its group's gate if `gated`
  auto gather = [&](const float* s, const float* s2, uint64_t first, uint64_t n, bool gated, float& x, float& y) {
    float u = 0.0f, v = 0.0f;
    if (in) {
#pragma unroll 4
      for (uint64_t k = first + warp; k < first + n; k += kJoinWarps) {
        const float g = gated ? param(a.gate, k / a.chunks * a.cols + c, 1.0f) : 1.0f;
        u = __fmaf_rn(g, s[k * a.cols], u);
        if (s2) v = __fmaf_rn(g, s2[k * a.cols], v);
      }
    }
    red[0][warp][lane] = u;
    red[1][warp][lane] = v;
    __syncthreads();
    x = y = 0.0f;
    if (warp == 0) {
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) {
        x += red[0][w][lane];
        y += red[1][w][lane];
      }
    }
    __syncthreads();
  };
  float x, y;
  if (blockIdx.y < gate_rows) {
    const float w = a.post ? param(a.w_post, c, 1.0f) : 1.0f, b = kinds.s ? param(a.b_post, c, 0.0f) : 0.0f;
    for (uint64_t g = blockIdx.y; g < a.groups; g += gate_rows) {
      gather(sum_t, kinds.s ? sum_s : nullptr, g * a.chunks, a.chunks, false, x, y);
      if (in && warp == 0) a.dgate[g * a.cols + c] = __fmaf_rn(w, x, b * y);
    }
  } else if (blockIdx.y == gate_rows && a.post) {
    gather(sum_t, kinds.s ? sum_s : nullptr, 0, places, a.gated, x, y);
    if (in && warp == 0) {
      a.dw_post[c] = x;
      if (a.bias) a.db_post[c] = y;
    }
  } else {
    gather(sum_p, kinds.q ? sum_q : nullptr, 0, places, false, x, y);
    if (in && warp == 0) {
      a.dw_pre[c] = x;
      if (a.bias) a.db_pre[c] = y;
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

cudaError_t norm_grad_occupancy(const NormArgs& a, NormFit fit, int* blocks_per_sm, unsigned* shared_bytes) {
  const Chosen c = choose<Pick>(a, fit);
  *shared_bytes = c.shared_bytes;
  const cudaError_t e = prepare_rows(c.kernel, c.shared_bytes);
  if (e != cudaSuccess) return e;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(blocks_per_sm, c.kernel, a.shape.threads, c.shared_bytes);
}

cudaError_t norm_grad_launch(const NormArgs& a, NormFit fit, cudaStream_t stream) {
  NormArgs args = a;
  NormSums kinds = norm_sums(a);
  if (a.rows) {
    const Chosen c = choose<Pick>(a, fit);
    cudaError_t e = prepare_rows(c.kernel, c.shared_bytes);
    if (e != cudaSuccess) return e;
    void* params[] = {&args, &kinds};
    e = launch_rows(c.kernel, a.shape, a.groups * a.chunks * unsigned(a.shape.ctas), c.shared_bytes, params, stream);
    if (e != cudaSuccess) return e;
  } else {
    args.chunks = 0;  // the column sums of no rows are zero
  }
  if (kinds.count() == 0) return cudaSuccess;
  const uint32_t gate_rows = a.gated ? std::min<uint32_t>(a.groups, 1024) : 0;
  (void)launch_pdl(&norm_grad_join_kernel, dim3((a.cols + 31) / 32, gate_rows + (a.post ? 1u : 0u) + (a.pre ? 1u : 0u)),
                   dim3(32 * kJoinWarps), stream, args, kinds, gate_rows);
  return cudaGetLastError();
}

}  // namespace askb
