// Softmax of biased scores, gradient: see bias_softmax.cuh.
//
// One pass: P is recomputed from s and lse, so besides s and dp nothing of the
// forward pass is read.  Each team has a window of its own for the table's
// gradient; adds of a row go to distinct places, and rows follow each other
// behind the team's reduction, so sums have one order and no atomics.
#include "bias_softmax.cuh"

#include <type_traits>

namespace askb {

namespace {

// lse in 32 bits carries a row's sum only so well: its rounding moves P by half a unit
// in lse's last place, 2^-18 below this magnitude, 0.2% at -65504, and where a whole row
// is at the lowest f32, as masks of that value leave it, every key had P = 1.  From
// here on P is divided by its sum over the row.  The loop's body is there twice for
// it: dividing every row took 268 us (the registers that add P beside P d spill), a
// branch within the body 236, this 234, and no division 233 (bf16 [8, 16, 1024, 1024],
// ragged, with dropout).
constexpr float kCoarseLse = 128.0f;

template <int T, int E, bool kDrop, bool kEven>
__global__ void __launch_bounds__(kTeamThreads) bias_softmax_grad_kernel(const __grid_constant__ BiasSoftmaxArgs a) {
  constexpr int V = act_vec<T>(), U = E / V, H = V / 2;
  extern __shared__ uint4 dynamic[];
  __shared__ TeamRecords<1> sh, sh_total;
  __shared__ float ends[2][kTeamThreads / 32];
  const Team t = team_of(a.shape);
  const Window<V> win(a);
  const int teams = int(t.count);
  const uint32_t pitch = blockDim.x * 16, ring = shared_address(dynamic) + threadIdx.x * 16;
  float* const copies = reinterpret_cast<float*>(dynamic + a.ring_rows * 2 * row_words<T, E>() * blockDim.x);
  float* const window = copies + (a.window_copies ? Lut<V>::words(win) : 0);
  float* const sums = window + win.words();  // the teams' windows
  const uint32_t mine = shared_address(sums + int(t.index) * win.words());
  const Units<T, kEven> units(a, t);
  pdl_enter();
  team_start(t);
  Rows<T, kEven> rows(a, t, U);
  RowView row{};
  float row_lse = 0.0f;
  auto fetch = [&](uint32_t slot) {
    const bool whole = rows.index < a.whole_rows;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      units.fetch(a.s, row, whole, u, slot + uint32_t(2 * u) * pitch);
      units.fetch(a.dp, row, whole, u, slot + uint32_t(2 * u + 1) * pitch);
    }
  };
  bool on = rows.left > 0;
  if (on) {
    row = units.view(a, rows);
    row_lse = __ldg(a.lse_in + rows.index);
    fetch(ring);
  }
  copy_async_commit();
  DropRun run{};
  if constexpr (kDrop) run = drop_run(a.drop, a.seed);
  for (int i = int(threadIdx.x); i < teams * win.words(); i += int(blockDim.x)) sums[i] = 0.0f;
  const Lut<V> lut = fill_window(a, win, rows.head, window, copies);
  const uint64_t scale = both(a.scale);
  const float drop_scale = kDrop ? run.scale : 1.0f;
  float left = 0.0f, right = 0.0f;  // dl of units wholly at rel <= -W, or at rel >= hi
  const bool two = a.ring_rows == 2;
  for (uint32_t turn = 0; __any_sync(0xffffffffu, on); ++turn) {
    const uint32_t slot = ring + (two ? turn & 1u : 0u) * (uint32_t(2 * U) * pitch);
    const RowView r = row;
    const bool here = on;
    const float base = row_lse == kNegInf ? 0.0f : row_lse;  // all logits are -inf then, and every P is 0
    if (on) {
      rows.next(a);
      on = rows.left > 0;
      if (on) {
        row = units.view(a, rows);
        row_lse = __ldg(a.lse_in + rows.index);
        if (two) fetch(ring + ((turn & 1u) ^ 1u) * (uint32_t(2 * U) * pitch));
      }
    }
    copy_async_commit();
    if (two) copy_async_wait<1>();
    else copy_async_wait<0>();
    const bool coarse = here && fabsf(base) >= kCoarseLse;  // the warps of a team agree: they hold the same row
    auto work = [&](auto coarse_rows) {
      uint64_t p[U][H], d[U][H], s2 = 0, s3 = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        act_widen2<T>(ld_shared(slot + uint32_t(2 * u) * pitch), p[u]);
        act_widen2<T>(ld_shared(slot + uint32_t(2 * u + 1) * pitch), d[u]);
        units.logits(r, win, lut, scale, u, p[u]);
        if (!units.all_whole(r, u)) {
          units.mask(r, u, kNegInf, p[u]);
          units.mask(r, u, 0.0f, d[u]);
        }
        if (kDrop && units.any_seen(r, u)) {
          const uint64_t i[1] = {units.offset(r, u) / dtype_bytes(T)};
          bool keep[V];
          drop_keep<1, V>(run, i, keep);
#pragma unroll
          for (int j = 0; j < H; ++j) {
            float lo, hi;
            unpack2(d[u][j], lo, hi);
            d[u][j] = pack2(keep[2 * j] ? lo : 0.0f, keep[2 * j + 1] ? hi : 0.0f);
          }
        }
        exp_minus<H>(p[u], both(-base));
#pragma unroll
        for (int j = 0; j < H; j += 2) {
          s2 = fma2(p[u][j], d[u][j], s2);
          s3 = fma2(p[u][j + 1], d[u][j + 1], s3);
        }
      }
      float dot[1] = {sum2(add2(s2, s3))};
      team_sum<1>(t, sh, int(turn & 1u), dot);
      if constexpr (decltype(coarse_rows)::value) {
        s2 = s3 = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < H; j += 2) {
            s2 = add2(s2, p[u][j]);
            s3 = add2(s3, p[u][j + 1]);
          }
        float total[1] = {sum2(add2(s2, s3))};
        team_sum<1>(t, sh_total, int(turn & 1u), total);
        const float over = !coarse ? 1.0f : total[0] == 0.0f ? 0.0f : __frcp_rn(total[0]);
        dot[0] *= over;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < H; ++j) p[u][j] = mul2(p[u][j], both(over));
      }
      // The lanes' adds of the row before are done: a team of several warps has met at
      // its barrier, shuffles alone order no memory.
      __syncwarp();
      // dl = P (D(dp) - sum): the dropout's scale enters here
      const float minus_sum = -dot[0] * drop_scale;
      // masked keys hold P = 0 already, unless what it meets is a NaN or infinite
      const bool odd = __any_sync(0xffffffffu, here && !(fabsf(minus_sum) <= 3.4e38f));
      if (!two && on) fetch(ring);
      const uint64_t by = both(drop_scale), minus = both(minus_sum);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint4 o = make_uint4(0u, 0u, 0u, 0u);
        if (units.any_seen(r, u)) {
          uint64_t* x = p[u];
#pragma unroll
          for (int j = 0; j < H; ++j) x[j] = mul2(x[j], fma2(d[u][j], by, minus));
          if (odd) units.mask(r, u, 0.0f, x);
          const int rel = units.key(r, u) - r.pos;
          const bool near = units.any_near(r, win, u);
          if (!near || rel >= win.hi || rel + V - 1 <= -win.w) {
            uint64_t v = x[0];
#pragma unroll
            for (int j = 1; j < H; ++j) v = add2(v, x[j]);
            const float f = here ? sum2(v) : 0.0f;
            left += rel >= win.hi ? 0.0f : f;
            right += rel >= win.hi ? f : 0.0f;
          } else if (here) {
            const Places<V> at(mine, win.place(rel));
#pragma unroll
            for (int j = 0; j < H; ++j) {
              float lo, hi;
              unpack2(x[j], lo, hi);
              st_shared_f32(at(2 * j), ld_shared_f32(at(2 * j)) + lo);
              st_shared_f32(at(2 * j + 1), ld_shared_f32(at(2 * j + 1)) + hi);
            }
          }
#pragma unroll
          for (int j = 0; j < H; ++j) x[j] = mul2(x[j], scale);
          o = act_narrow2<T>(x);
        }
        if (here) units.store(a, r, u, o);
      }
    };
    if (__any_sync(0xffffffffu, coarse)) work(std::true_type{});
    else work(std::false_type{});
  }
  // fold the windows by bucket
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    left += __shfl_xor_sync(0xffffffffu, left, d);
    right += __shfl_xor_sync(0xffffffffu, right, d);
  }
  const int warp = int(threadIdx.x >> 5), lane = int(threadIdx.x & 31u), warps = int(blockDim.x >> 5);
  if (lane == 0) {
    ends[0][warp] = left;
    ends[1][warp] = right;
  }
  __syncthreads();
  const int side = a.n_thresholds + 1;
  for (int b = warp; b < int(a.buckets); b += warps) {
    const bool ahead = b >= side;  // rel > 0
    const int j = ahead ? b - side : b;
    const bool is_left = !ahead && j == a.n_thresholds, is_right = a.bidirectional ? ahead && j == a.n_thresholds : j == 0;
    // the bucket's distances [n0, n1): from the last threshold on the V - 1 places
    // beyond the window too, as have the keys ahead where only distances behind count
    const int n0 = max(j ? a.thresholds[j - 1] : 0, ahead ? 1 : 0);
    const int n1 = j < a.n_thresholds ? a.thresholds[j] : win.w + V;
    float v = 0.0f;
    for (int k = 0; k < teams; ++k) {
      const float* at = sums + k * win.words();
      for (int n = n0 + lane; n < n1; n += 32) v += at[win.word(win.place(ahead ? n : -n))];
      if (!a.bidirectional && j == 0 && lane > 0 && lane < V) v += at[win.word(win.place(lane))];
    }
    if (lane < warps) v += (is_left ? ends[0][lane] : 0.0f) + (is_right ? ends[1][lane] : 0.0f);
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if (lane == 0) a.partial[uint64_t(blockIdx.x) * a.buckets + b] = v;
  }
}

// dtable[b, head]: a warp (kBiasJoinThreads) adds the head's CTAs in order of their chunks.
__global__ void __launch_bounds__(256) bias_table_join_kernel(const float* __restrict__ partial, float* __restrict__ dtable,
                                                              uint32_t heads, uint32_t buckets, uint32_t chunks,
                                                              uint32_t ctas) {
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t out = uint64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (out >= uint64_t(heads) * buckets) return;
  const uint32_t b = uint32_t(out / heads), head = uint32_t(out % heads);
  double v = 0.0;
  for (uint32_t k = lane; k < chunks * ctas; k += 32) {
    const uint64_t cta = (uint64_t(k / ctas) * heads + head) * ctas + k % ctas;
    v += double(partial[cta * buckets + b]);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (lane == 0) dtable[out] = float(v);
}

template <int T, int E, bool kDrop, bool kEven>
struct Pick {
  static const void* get(const BiasSoftmaxArgs&) {
    // bias_softmax_shape gives a gradient 32 elements a thread at most
    return (const void*)bias_softmax_grad_kernel<T, E <= 32 ? E : 32, kDrop, kEven>;
  }
};

}  // namespace

cudaError_t bias_softmax_grad_occupancy(const BiasSoftmaxArgs& a, int* blocks_per_sm) {
  return rows_occupancy(choose<Pick>(a), a, blocks_per_sm);
}

cudaError_t bias_softmax_grad_launch(const BiasSoftmaxArgs& a, cudaStream_t stream) {
  const bool rows = a.batch && a.heads && a.queries;
  if (rows) {
    const cudaError_t e = rows_launch(choose<Pick>(a), a, stream);
    if (e != cudaSuccess) return e;
  }
  const uint64_t entries = uint64_t(a.heads) * a.buckets;
  if (!entries) return cudaSuccess;
  (void)launch_pdl(&bias_table_join_kernel, dim3(unsigned((entries + 7) / 8)), dim3(256), stream,
                   static_cast<const float*>(a.partial), a.dtable, a.heads, a.buckets, rows ? a.chunks : 0u,
                   uint32_t(a.shape.ctas));
  return cudaGetLastError();
}

}  // namespace askb
