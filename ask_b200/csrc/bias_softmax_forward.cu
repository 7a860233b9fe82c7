// Softmax of biased scores, forward: see bias_softmax.cuh.
#include "bias_softmax.cuh"

namespace askb {

namespace {

// kSmall: CTAs of 128 threads at most, five an SM (102 registers): single tokens
// against 4096 keys took 10.7 us so and 11.6 with what the compiler takes by
// itself (six: 11.4, and rows of 1024 keys 183 for 177); 40 elements a thread
// take four (1021 keys: 262 us, and 282 with three).
template <int T, int E, bool kDrop, bool kEven, bool kSmall>
__global__ void __launch_bounds__(kSmall ? kWarpTeamThreads : kTeamThreads, kSmall ? (E <= 32 ? 5 : 4) : 1)
    bias_softmax_kernel(const __grid_constant__ BiasSoftmaxArgs a) {
  constexpr int V = act_vec<T>(), U = E / V, H = V / 2;
  extern __shared__ uint4 dynamic[];
  __shared__ TeamRecords<2> sh;
  const Team t = team_of(a.shape);
  const Window<V> win(a);
  const uint32_t pitch = blockDim.x * 16, ring = shared_address(dynamic) + threadIdx.x * 16;
  float* const copies = reinterpret_cast<float*>(dynamic + a.ring_rows * row_words<T, E>() * blockDim.x);
  float* const window = copies + (a.window_copies ? Lut<V>::words(win) : 0);
  const Units<T, kEven> units(a, t);
  pdl_enter();
  team_start(t);
  Rows<T, kEven> rows(a, t, U);
  RowView row{};
  uint64_t index = 0;
  auto fetch = [&](uint32_t slot) {
#pragma unroll
    for (int u = 0; u < U; ++u) units.fetch(a.s, row, rows.index < a.whole_rows, u, slot + uint32_t(u) * pitch);
  };
  bool on = rows.left > 0;
  if (on) {
    row = units.view(a, rows);
    index = rows.index;
    fetch(ring);
  }
  copy_async_commit();
  DropRun run{};
  if constexpr (kDrop) run = drop_run(a.drop, a.seed);
  const Lut<V> lut = fill_window(a, win, rows.head, window, copies);
  const uint64_t scale = both(a.scale);
  const bool two = a.ring_rows == 2;  // a row ahead; else the next one is fetched when this one is read
  // the teams of a warp go on together while one of them has a row
  for (uint32_t turn = 0; __any_sync(0xffffffffu, on); ++turn) {
    const uint32_t slot = ring + (two ? turn & 1u : 0u) * (uint32_t(U) * pitch);
    const int parity = int(turn & 1u);
    const RowView r = row;
    const uint64_t this_index = index;
    const bool here = on;
    if (on) {
      rows.next(a);
      on = rows.left > 0;
      if (on) {
        row = units.view(a, rows);
        index = rows.index;
        if (two) fetch(ring + ((turn & 1u) ^ 1u) * (uint32_t(U) * pitch));
      }
    }
    copy_async_commit();
    if (two) copy_async_wait<1>();
    else copy_async_wait<0>();
    uint64_t e[U][H];
    float m = kNegInf;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      act_widen2<T>(ld_shared(slot + uint32_t(u) * pitch), e[u]);
      units.logits(r, win, lut, scale, u, e[u]);
      if (!units.all_whole(r, u)) units.mask(r, u, kNegInf, e[u]);
#pragma unroll
      for (int j = 0; j < H; ++j) {
        float lo, hi;
        unpack2(e[u][j], lo, hi);
        m = max3(m, lo, hi);
      }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1)
      if (uint32_t(d) < t.lanes) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float base = m == kNegInf ? 0.0f : m;  // nothing visible: every 2^x below is 0
    uint64_t s2 = 0, s3 = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      exp_minus<H>(e[u], both(-base));
#pragma unroll
      for (int j = 0; j < H; j += 2) {
        s2 = add2(s2, e[u][j]);
        s3 = add2(s3, e[u][j + 1]);
      }
    }
    float s = sum2(add2(s2, s3));
#pragma unroll
    for (int d = 16; d; d >>= 1)
      if (uint32_t(d) < t.lanes) s += __shfl_xor_sync(0xffffffffu, s, d);
    // the team's maximum and sum from the warps' own
    float top = base, sum = s, factor = 1.0f;
    const uint32_t records = t.warps * t.ctas;
    if (records > 1) {
      const float rec[2] = {m, s};
      team_exchange<2>(t, sh, parity, rec);
      top = kNegInf;
      for (uint32_t k = 0; k < records; ++k) top = fmaxf(top, sh.v[parity][k][0]);
      if (top == kNegInf) top = 0.0f;
      sum = 0.0f;
      for (uint32_t k = 0; k < records; ++k)
        sum = __fmaf_rn(sh.v[parity][k][1], ex2_approx((sh.v[parity][k][0] - top) * kLog2e), sum);
      factor = ex2_approx((m - top) * kLog2e);
    }
    factor = sum == 0.0f ? 0.0f : factor * rcp_approx(sum);
    // masked keys hold 0 already, unless a NaN in the row makes the factor one
    const bool odd = __any_sync(0xffffffffu, here && !(factor >= 0.0f));
    if (!two && on) fetch(ring);
    if (here && t.tid == 0 && t.rank == 0) a.lse[this_index] = sum == 0.0f ? kNegInf : __fmaf_rn(lg2_approx(sum), kLn2, top);
    const uint64_t by = both(kDrop ? factor * run.scale : factor);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint4 o = make_uint4(0u, 0u, 0u, 0u);
      if (units.any_seen(r, u)) {
        uint64_t* x = e[u];
#pragma unroll
        for (int j = 0; j < H; ++j) x[j] = mul2(x[j], by);
        if constexpr (kDrop) {
          const uint64_t i[1] = {units.offset(r, u) / dtype_bytes(T)};
          bool keep[V];
          drop_keep<1, V>(run, i, keep);
#pragma unroll
          for (int j = 0; j < H; ++j) {
            float lo, hi;
            unpack2(x[j], lo, hi);
            x[j] = pack2(keep[2 * j] ? lo : 0.0f, keep[2 * j + 1] ? hi : 0.0f);
          }
        }
        if (odd) units.mask(r, u, 0.0f, x);
        o = act_narrow2<T>(x);
      }
      if (here) units.store(a, r, u, o);
    }
  }
}

template <int T, int E, bool kDrop, bool kEven>
struct Pick {
  static const void* get(const BiasSoftmaxArgs& a) {
    return a.shape.threads <= kWarpTeamThreads ? (const void*)bias_softmax_kernel<T, E, kDrop, kEven, true>
                                               : (const void*)bias_softmax_kernel<T, E, kDrop, kEven, false>;
  }
};

constexpr uint32_t kSharedBytes = 216 * 1024;  // dynamic shared memory of a CTA at most

}  // namespace

TeamShape bias_softmax_shape(uint64_t keys, uint64_t rows, int type, bool grad, int sms) {
  const uint64_t v = type == kF32 ? 4 : 8;
  // a row that starts inside a unit spreads over one more
  const uint64_t span = keys % v ? keys + v - 1 : keys;
  TeamShape s{0, kWarpTeamThreads, kWarpTeamThreads, 1, 32};
  // The threads a row takes and the elements of each: the least threads *
  // (elements + 8), a row's own work being worth about 8 elements of a thread.
  // More elements cost registers (40: 5 units of 16 bits, for rows a little over
  // a warp's 1024), fewer leave a row's work to more threads.
  uint64_t least = UINT64_MAX;
  if (rows >= uint64_t(sms) * 8 && span <= 32 * 40) {
    for (int e : {40, 32, 24, 16}) {
      if (grad && e == 40) continue;  // two rows of 40 elements a thread spill
      uint64_t lanes = grad ? 8 : 4;  // each team of a gradient has a window of its own
      while (span > lanes * uint64_t(e)) lanes *= 2;
      if (lanes <= 32 && lanes * uint64_t(e + 8) < least) {
        least = lanes * uint64_t(e + 8);
        s.elems = e;
        s.warp_teams = int(lanes);
      }
    }
    if (s.warp_teams) return s;
  }
  // few rows take more threads for each
  for (int e : {40, 32, 24, 16, 8}) {
    if (grad && e == 40) continue;
    const uint64_t threads = ((span + uint64_t(e) - 1) / uint64_t(e) + 31) / 32 * 32;
    if (threads > uint64_t(kTeamThreads)) continue;
    const uint64_t cost = rows < uint64_t(sms) * 2 ? uint64_t(e) : threads * uint64_t(e + 8);
    if (cost < least) {
      least = cost;
      s.elems = e;
    }
  }
  // few rows: spread each over a cluster while SMs idle and every CTA keeps 256 threads' worth of a row
  while (s.ctas < kTeamCluster &&
         (span > uint64_t(kTeamThreads) * s.elems * s.ctas ||
          (rows * s.ctas * 2 <= uint64_t(sms) && span >= uint64_t(512) * s.elems * s.ctas)))
    s.ctas *= 2;
  const uint64_t per = uint64_t(s.elems) * s.ctas;
  s.threads = s.team_threads = int(std::max<uint64_t>(32, ((span + per - 1) / per + 31) / 32 * 32));
  return s;
}

void bias_softmax_shared(BiasSoftmaxArgs* a, bool grad) {
  const uint32_t window = uint32_t(a->type == kF32 ? Window<4>(*a).words() : Window<8>(*a).words()) * 4;
  const uint32_t row = (grad ? 2u : 1u) * uint32_t(a->shape.elems) * (a->type == kF32 ? 4u : 2u);  // bytes of a thread
  const uint32_t copies = uint32_t(a->type == kF32 ? Lut<4>::words(Window<4>(*a)) : Lut<8>::words(Window<8>(*a))) * 4;
  a->ring_rows = 2;
  a->window_copies = 0;
  auto total = [&] {
    return a->ring_rows * row * uint32_t(a->shape.threads) + a->window_copies * copies +
           (1 + (grad ? uint32_t(team_count(a->shape)) : 0u)) * window;
  };
  // wide windows leave room for fewer teams, the longest f32 rows for one row at a time
  while (a->shape.warp_teams && total() > kSharedBytes / 2) {
    if (a->shape.threads > 32) a->shape.threads -= 32;
    else if (a->shape.warp_teams < 32) a->shape.warp_teams *= 2;
    else break;
  }
  if (total() > kSharedBytes) a->ring_rows = 1;
  // The window's copies where a warp's rows are many and they take little of the SM:
  // bf16 [8, 16, 1024, 1024] to distance 128 95 us with them and 100 without, gradient 145
  // and 150; 200 (9 KB) 96 and 102, 150 and 155.  Past 12 KB (the last threshold some
  // 180) fewer gradient CTAs fit: to distance 512 they would win the forward kernel
  // 7 us of 109 and cost the gradient 19 of 169.
  a->window_copies = a->shape.warp_teams && copies <= 12 * 1024 && total() + copies <= kSharedBytes ? 1 : 0;
  a->shared_bytes = total();
}

cudaError_t bias_softmax_occupancy(const BiasSoftmaxArgs& a, int* blocks_per_sm) {
  return rows_occupancy(choose<Pick>(a), a, blocks_per_sm);
}

cudaError_t bias_softmax_launch(const BiasSoftmaxArgs& a, cudaStream_t stream) {
  if (a.batch == 0 || a.heads == 0 || a.queries == 0) return cudaSuccess;
  return rows_launch(choose<Pick>(a), a, stream);
}

}  // namespace askb
