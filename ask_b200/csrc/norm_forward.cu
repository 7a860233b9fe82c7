// Block norms, forward: see norm_rows.cuh.
//
// A stretch of consecutive rows a CTA, all resident at once, so a group's factors
// are put together once and the ring never drains.  The switches of the usual
// steps are template arguments: read at run time they cost a fifth (bf16 [32768,
// 4096] 283 against 248 us).
#include "norm_rows.cuh"

#include <numeric>

namespace askb {

namespace {

// Threads that an SM is to hold, and the ring's rows that they leave room for.  A
// plain norm of 16-bit rows takes 80 registers and two rows: 800 threads, which
// is three teams for 4096 columns and two up to 6400 (bf16 [32768, 4096] 243 us
// with 128 registers and three rows, 231 so; [16384, 5120] 241 and 175).  The
// others need more of both: 576 threads, two teams up to 4608 columns, and f32
// rows with four parameters a ring of one row.
template <int T, int F, bool kFull>
struct Layout {
  static constexpr int kThreads = T != kF32 && !kFull ? 800 : 576;
  static constexpr int kStage = 2 * Columns<T, F>::kArrayBytes, kParams = (kFull ? 4 : 2) * kParamBytes;
  static constexpr int kStages = ring_stages(kStage, kParams);
  static constexpr int kBytes = kStages * kStage + kParams;
};

// Centres the row (layer norm) and gives its mean and 1 / sqrt(variance + eps).
template <int T, int F>
__device__ __forceinline__ void row_stats(const Team& t, const Columns<T, F>& c, TeamRecords<1>& sh_mean,
                                          TeamRecords<1>& sh_sq, int parity, bool layer, float inv_cols, float eps,
                                          uint64_t (&v)[kPairs], float& mean, float& rstd) {
  mean = 0.0f;
  if (layer) {
    float s[1] = {total(v)};
    team_sum<1>(t, sh_mean, parity, s);
    mean = s[0] * inv_cols;
    c.template center<true>(mean, v);
  }
  float s[1] = {dot(v, v)};
  team_sum<1>(t, sh_sq, parity, s);
  rstd = rsqrtf(__fmaf_rn(s[0], inv_cols, eps));
}

// kFull: layer norms or biases too; a plain rms norm drops that code.
template <int T, int F, int kForm, bool kFull, bool kDrop>
__global__ void __launch_bounds__(Layout<T, F, kFull>::kThreads) norm_rows_kernel(const __grid_constant__ NormArgs a) {
  using Cols = Columns<T, F>;
  using Shape = Layout<T, F, kFull>;
  constexpr int S = Shape::kStages, P = kPairs;
  const bool branch = kForm == FORM_ANY ? a.branch : kForm != FORM_NORM;
  const bool post = kForm == FORM_ANY ? a.post : kForm == FORM_BOTH;
  const bool pre = kForm == FORM_ANY ? a.pre : true;
  const bool factors = kForm == FORM_ANY || kForm == FORM_BOTH;
  extern __shared__ uint4 dynamic[];
  __shared__ TeamRecords<1> sh[kFull ? 4 : 2];
  const Team t = team_of(a.shape);
  // CTAs (or clusters; `spread` of them) have a stretch of rows, and their teams take them in turn
  const uint32_t places = gridDim.x / (t.ctas * a.spread), place = blockIdx.x / t.ctas;
  const uint64_t begin = a.rows * (place / a.spread) / places, end = a.rows * (place / a.spread + 1) / places;
  const uint32_t stride = t.count * a.spread;
  uint64_t row = begin + place % a.spread * t.count + t.index;
  const Cols col(t, a, row);
  const uint32_t mine = row < end ? uint32_t((end - row + stride - 1) / stride) : 0;
  const uint32_t turns = __shfl_sync(0xffffffffu, mine, 0);  // of the warp: its first team has the most rows
  const float inv_cols = 1.0f / float(a.cols);
  const uint32_t ring = Cols::ring(dynamic), array = blockDim.x * uint32_t(Cols::kArrayBytes), stage_bytes = 2 * array;
  const uint32_t pitch = blockDim.x * 16, params = shared_address(dynamic) + S * stage_bytes + threadIdx.x * 16;
  const ParamSlot pre_w{params, pitch}, fac{params + kElems / 4 * pitch, pitch},
      pre_b{params + 2 * (kElems / 4) * pitch, pitch}, fac_b{params + 3 * (kElems / 4) * pitch, pitch};
  const uint64_t bytes = a.rows * a.cols * uint64_t(Cols::B), advance = stride * uint64_t(a.cols) * Cols::B;
  pdl_enter();
  team_start(t);
  DropRun run{};
  if constexpr (kDrop) run = drop_run(a.drop, a.seed);
  const float scale = kDrop ? run.scale : 1.0f;
  uint64_t off = col.offset(row);
  auto fetch = [&](uint32_t turn, uint64_t at, uint32_t slot) {
    if (turn < mine) {
      col.fetch(a.x, at, bytes, slot);
      if (branch) col.fetch(a.y, at, bytes, slot + array);
    }
    copy_async_commit();
  };
#pragma unroll
  for (int s = 0; s < S; ++s) {
    col.clear(ring + s * stage_bytes);
    col.clear(ring + s * stage_bytes + array);
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s, off + s * advance, ring + s * stage_bytes);
  if (pre) {
    float f[kElems];
    col.params(a.w_pre, a.ptype, 0, 1.0f, f);
    pre_w.write(f);
    if constexpr (kFull) {
      col.params(a.b_pre, a.ptype, 0, 0.0f, f);
      pre_b.write(f);
    }
  }
  uint64_t group_end = 0;  // the factors in shared memory are those of the rows before it
  uint32_t slot = ring, free_slot = ring + (S - 1) * stage_bytes;
  for (uint32_t turn = 0; turn < turns; ++turn, row += stride, off += advance) {
    const int parity = int(turn & 1u);
    const bool on = turn < mine;
    fetch(turn + S - 1, off + (S - 1) * advance, free_slot);
    if (factors && branch && on && row >= group_end) {
      // post weight, gate and the dropout's scale as one factor
      const uint64_t group = row / a.rows_per_group;
      group_end = (group + 1) * a.rows_per_group;
      float g[kElems], f[kElems];
      col.params(a.gate, a.ptype, group * a.cols, 1.0f, g);
      col.params(a.w_post, a.ptype, 0, 1.0f, f);
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
    if (branch) {
      uint64_t n[P];
      col.template read<true>(slot + array, a.y, off, n);
      if (post) {
        float mean, rstd;
        row_stats(t, col, sh[kFull ? 2 : 0], sh[0], parity, kFull && a.layer, inv_cols, a.eps, n, mean, rstd);
        if (writer) {
          if (kFull && a.layer) a.stats_post[2 * row] = mean;
          a.stats_post[kFull && a.layer ? 2 * row + 1 : row] = rstd;
        }
        scale_all(n, rstd);
      }
      if (factors) scale_by<kFull>(n, fac, fac_b);
      else if (kDrop) scale_all(n, scale);
      if constexpr (kDrop) col.drop(run, off, n);
      const uint64_t alpha = both(a.alpha);
      col.template read<true>(slot, a.x, off, h);
#pragma unroll
      for (int k = 0; k < P; ++k) h[k] = fma2(alpha, h[k], n[k]);
      col.put(t, a.h, off, on, h);
    } else {
      col.template read<true>(slot, a.x, off, h);
    }
    if (pre) {
      float mean, rstd;
      row_stats(t, col, sh[kFull ? 3 : 1], sh[1], parity, kFull && a.layer, inv_cols, a.eps, h, mean, rstd);
      if (writer) {
        if (kFull && a.layer) a.stats_pre[2 * row] = mean;
        a.stats_pre[kFull && a.layer ? 2 * row + 1 : row] = rstd;
      }
      scale_all(h, rstd);
      scale_by<kFull>(h, pre_w, pre_b);
      col.put(t, a.u, off, on, h);
    }
    free_slot = slot;  // read by its own thread alone, and that is done
    slot = slot == ring + (S - 1) * stage_bytes ? ring : slot + stage_bytes;
  }
}

template <int T, int F, int kForm, bool kFull, bool kDrop>
struct Pick {
  static Chosen get(unsigned threads) {
    return {(const void*)norm_rows_kernel<T, F, kForm, kFull, kDrop>, threads * unsigned(Layout<T, F, kFull>::kBytes)};
  }
};

}  // namespace

static TeamShape shape_of(uint64_t span, bool grad) {
  TeamShape s{0, 256, 256, 1, kElems};
  if (span <= 32 * kElems) {
    s.warp_teams = 4;
    while (span > uint64_t(s.warp_teams) * kElems) s.warp_teams *= 2;
  } else {
    while (span > uint64_t(kTeamThreads) * kElems * s.ctas) s.ctas *= 2;
    const uint64_t per = uint64_t(kElems) * s.ctas;
    s.threads = s.team_threads = int((((span + per - 1) / per) + 31) / 32 * 32);
  }
  // The gradient's teams share a CTA as large as the registers allow: one set
  // of column sums leaves it.
  if (grad && s.ctas == 1) s.threads = s.warp_teams ? kTeamThreads : kTeamThreads / s.team_threads * s.team_threads;
  return s;
}

void norm_layout(NormArgs* a, bool grad) {
  const uint32_t v = 16u / uint32_t(dtype_bytes(a->type));
  a->classes = 1;
  a->shape = shape_of(a->cols, grad);
  if (a->cols % v == 0) return;
  // Rows off the units go by cut units (bf16 [33520, 1001] 87 us, and 146 shifted out
  // of neighbouring words; f32 107, and 207 word by word), unless the unit more that a
  // row may spread over needs threads that halve the teams an SM holds (gradient
  // of bf16 [8191, 4095] 222 us, and 190 shifted; of 511 columns 235 and 187; with
  // two thirds of the teams cut units are ahead: 1023 columns 185 and 202) or,
  // in f32 with four parameters, any (1023 columns 374 us, and 301 by words).
  const TeamShape cut = shape_of(a->cols + v - 1, grad);
  const auto team = [](const TeamShape& s) { return s.warp_teams ? s.warp_teams : s.team_threads * s.ctas; };
  if (team(cut) > team(a->shape)) {
    const bool full = a->layer || a->bias;
    if (a->type == kF32 && full) return;
    const int held = grad ? kTeamThreads : a->type != kF32 && !full ? Layout<kBF16, NORM_CUT, false>::kThreads
                                                                    : Layout<kF32, NORM_CUT, true>::kThreads;
    if (held / team(cut) * 2 <= held / team(a->shape)) return;
  }
  a->shape = cut;
  a->classes = v / std::gcd(v, a->cols);
}

cudaError_t norm_occupancy(const NormArgs& a, NormFit fit, int* blocks_per_sm, unsigned* shared_bytes) {
  const Chosen c = choose<Pick>(a, fit);
  *shared_bytes = c.shared_bytes;
  const cudaError_t e = prepare_rows(c.kernel, c.shared_bytes);
  if (e != cudaSuccess) return e;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(blocks_per_sm, c.kernel, a.shape.threads, c.shared_bytes);
}

cudaError_t norm_launch(const NormArgs& a, NormFit fit, int grid, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  const Chosen c = choose<Pick>(a, fit);
  const cudaError_t e = prepare_rows(c.kernel, c.shared_bytes);
  if (e != cudaSuccess) return e;
  NormArgs args = a;
  void* params[] = {&args};
  return launch_rows(c.kernel, a.shape, unsigned(grid), c.shared_bytes, params, stream);
}

}  // namespace askb
