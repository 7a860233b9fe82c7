// Softmax of scores with a learned relative-position bias, and its gradient.
//
//   l = scale s + table[bucket(k - pos), head],  pos = query + offset[batch]
//   over the keys k < length[batch] (and k <= pos when causal);
//   p = D(exp(l - lse)),  lse = log sum exp l,  D dropout; a row without keys
//   gives zeros and lse = -inf.
//   Gradient: P = exp(l - lse), d = D(dp), dl = P (d - sum P d), ds = scale dl,
//   dtable[b, head] = sum of dl where the bucket is b.
//
// bucket(rel): the number of thresholds that are at most the distance |rel|
// (bidirectional; the buckets of rel > 0 follow those of rel <= 0) or
// max(-rel, 0).  From the last threshold W on the bucket stays the same, so a
// row meets a window of less than 2W distances and two constants outside it.
// A CTA works on one head: it looks the table up once, into a shared array of
// the window by distance.  In the gradient a row holds each distance of the
// window once, so its owner adds dl to the window's sum without atomics, in row
// order; what lies outside is summed in registers.  Buckets are ranges of
// the window: they are folded once at the end, into a partial sum for each
// CTA that a second kernel adds in CTA order.
//
// Rows start anywhere (any number of keys): a row is read and written in the
// tensor's own aligned 16-byte units, whose first and last may hold elements of
// the neighbouring rows; those are masked, and only such cut units are stored
// element by element.  Units without a visible key are not read.  The next row's
// units are on their way (cp.async into words that only their own thread reads)
// while this row is worked on.
//
// exp(l - m) is 2^(l L - RN(m L)) with L = log2 e: an element costs a fused
// multiply-add for its logit, one for the exponent (both on f32 pairs) and
// ex2.approx (relative error 2^-22).  The rounding of m L is one factor for all
// that share m.  Where m L could overflow (|m| > 2^100: rows at the type's
// lowest value) the difference is taken first.  Each warp takes its own
// maximum, and its sum is rescaled when the team's records meet: one exchange a
// row.
#include <cuda_runtime.h>

#include <algorithm>

#include "act_io.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "philox.cuh"
#include "row_team.cuh"

namespace askb {

namespace {

#ifndef KWT
#define KWT 128
#endif
constexpr int kWarpTeamThreads = KWT;
constexpr float kNegInf = -__builtin_huge_valf();

// The window's geometry: distances rel in [-W, hi], and V - 1 places beyond
// either end, so that a unit that reaches into the window has a place for each
// of its elements.  Place i lies at word i + i / V: the lanes of a warp, whose
// units are V places apart, then fall on different banks.
template <int V>
struct Window {
  int w, hi;
  __host__ __device__ explicit Window(const BiasSoftmaxArgs& a)
      : w(a.n_thresholds ? a.thresholds[a.n_thresholds - 1] : 0), hi(a.bidirectional ? w : 0) {}
  __host__ __device__ int places() const { return w + hi + 1 + 2 * (V - 1); }
  __host__ __device__ static int word(int place) { return place + place / V; }
  __host__ __device__ int words() const { return word(places() - 1) + 1; }
  __host__ __device__ int place(int rel) const { return rel + w + (V - 1); }
  __host__ __device__ int rel(int place) const { return place - w - (V - 1); }
};
// The words of V places from `place` on: word(place) + j, and one more from the
// next multiple of V on.
template <int V>
struct Places {
  uint32_t at;  // shared address of the first
  int wrap;     // j from which one word is skipped
  __device__ __forceinline__ Places(uint32_t base, int place)
      : at(base + 4u * uint32_t(place + place / V)), wrap(V - place % V) {}
  __device__ __forceinline__ uint32_t operator()(int j) const { return at + (j >= wrap ? 4u * j + 4u : 4u * j); }
};
__device__ __forceinline__ float ld_shared_f32(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_f32(uint32_t at, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}

__device__ __forceinline__ int bucket_of(const BiasSoftmaxArgs& a, int rel) {
  const int n = a.bidirectional ? abs(rel) : max(-rel, 0);
  int lo = 0, hi = a.n_thresholds;  // thresholds[0, lo) <= n < thresholds[hi, ..)
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.thresholds[mid] <= n) lo = mid + 1; else hi = mid;
  }
  return a.bidirectional && rel > 0 ? lo + a.n_thresholds + 1 : lo;
}

// The head's bias by distance.
template <int V>
__device__ __forceinline__ void fill_window(const BiasSoftmaxArgs& a, const Window<V>& win, uint32_t head, float* lut) {
  for (int i = int(threadIdx.x); i < win.places(); i += int(blockDim.x)) {
    float v[1];
    param_load<1>(a.table, a.table_type, uint64_t(bucket_of(a, win.rel(i))) * a.heads + head, v);
    lut[win.word(i)] = v[0];
  }
}

// The rows of a team, one after the other: pairs (batch, query) of one head.
template <int T>
struct Rows {
  static constexpr int V = act_vec<T>(), B = dtype_bytes(T);
  const BiasSoftmaxArgs& a;
  uint32_t head, step, b, q;
  uint64_t left;          // rows from this one on, in steps
  int length, place;      // of the sequence: keys in use, position of its query 0
  // of the row
  uint64_t index, first;  // byte offset of its first unit
  int shift;              // elements of that unit before the row
  int pos, visible;       // query position; keys [0, visible) are seen

  __device__ __forceinline__ Rows(const BiasSoftmaxArgs& args, const Team& t) : a(args) {
    const uint32_t cta = blockIdx.x / t.ctas, chunk = cta / a.heads;
    const uint64_t n = a.batch * a.queries, begin = n * chunk / a.chunks, end = n * (chunk + 1) / a.chunks;
    const uint32_t team = a.shape.warp_teams ? threadIdx.x / t.threads : 0;
    head = cta % a.heads;
    step = a.shape.warp_teams ? blockDim.x / t.threads : 1;
    left = begin + team < end ? (end - begin - team + step - 1) / step : 0;
    b = uint32_t((begin + team) / a.queries);
    q = uint32_t((begin + team) % a.queries);
  }
  __device__ __forceinline__ void sequence() {
    length = int(a.keys);
    place = 0;
    if (a.lengths) length = max(min(__ldg(a.lengths + b), length), 0);
    if (a.offsets) place = __ldg(a.offsets + b);
  }
  __device__ __forceinline__ void locate() {
    index = (uint64_t(b) * a.heads + head) * a.queries + q;
    const uint64_t e = index * a.keys;
    shift = int(uint32_t(e) & uint32_t(V - 1));
    first = (e - uint64_t(shift)) * B;
    const int64_t at = int64_t(place) + int64_t(q);
    visible = length;
    if (a.causal) visible = int(max(min(int64_t(length), at + 1), int64_t(0)));
    // far positions meet only the window's ends, whatever their distance
    pos = int(max(min(at, int64_t(1) << 30), -(int64_t(1) << 30)));
  }
  // to be called once before the first row, then to go on
  __device__ __forceinline__ void start() {
    if (left) {
      sequence();
      locate();
    }
  }
  __device__ __forceinline__ void next() {
    if (--left == 0) return;
    q += step;
    if (q >= a.queries) {
      const uint32_t n = q / uint32_t(a.queries);
      b += n;
      q -= n * uint32_t(a.queries);
      sequence();
    }
    locate();
  }
};

// One row of a team in flight or at work: which units the thread has, and what
// it may read of them.
template <int T>
struct RowView {
  static constexpr int V = act_vec<T>(), B = dtype_bytes(T);
  uint64_t index, first;
  int k, step;  // first key of unit 0, keys between this thread's units
  int pos, visible;
  RowView() = default;
  __device__ __forceinline__ RowView(const Rows<T>& r, const Team& t, int vpt)
      : index(r.index), first(r.first + uint64_t((t.rank * uint32_t(vpt) * t.threads + t.tid) * 16u)),
        k(int((t.rank * uint32_t(vpt) * t.threads + t.tid) * uint32_t(V)) - r.shift), step(int(t.threads) * V), pos(r.pos),
        visible(r.visible) {}
  __device__ __forceinline__ int key(int u) const { return k + u * step; }
  __device__ __forceinline__ uint64_t offset(int u) const { return first + uint64_t(uint32_t(u * step * B)); }
  __device__ __forceinline__ bool seen(int u) const { return key(u) < visible && key(u) + V > 0; }
  __device__ __forceinline__ bool whole(int u) const { return key(u) >= 0 && key(u) + V <= visible; }

  __device__ __forceinline__ void fetch(const BiasSoftmaxArgs& a, const void* p, uint64_t bytes, int u, uint32_t slot) const {
    if (!seen(u)) return;
    const char* from = static_cast<const char*>(p) + offset(u);
    if (a.aligned && offset(u) + 16 <= bytes) {
      copy_to_shared(slot, from);
    } else {  // a tensor's last unit, or a tensor that starts inside 16 bytes: by elements
      uint32_t w[4] = {};
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (key(u) + j < 0 || key(u) + j >= visible) continue;
        const uint32_t bits = B == 4 ? __ldg(reinterpret_cast<const uint32_t*>(from) + j)
                                     : uint32_t(__ldg(reinterpret_cast<const unsigned short*>(from) + j));
        w[j * B / 4] |= bits << (8 * (j * B % 4));
      }
      st_shared(slot, make_uint4(w[0], w[1], w[2], w[3]));
    }
  }
  // the unit's elements that belong to the row
  __device__ __forceinline__ void store(const BiasSoftmaxArgs& a, int u, const uint64_t* v) const {
    const int k0 = key(u), n = int(a.keys);
    if (k0 >= n) return;
    char* to = static_cast<char*>(a.out) + offset(u);
    const uint4 o = act_narrow2<T>(v);
    if (a.aligned && k0 >= 0 && k0 + V <= n) {
      st_stream_v4(to, o);
    } else {
      const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (k0 + j < 0 || k0 + j >= n) continue;
        if constexpr (B == 4) reinterpret_cast<uint32_t*>(to)[j] = w[j];
        else reinterpret_cast<uint16_t*>(to)[j] = uint16_t(w[j / 2] >> (16 * (j % 2)));
      }
    }
  }
  // v <- v where the key is visible, else `other`
  __device__ __forceinline__ void mask(int u, float other, uint64_t* v) const {
    if (whole(u)) return;
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      float lo, hi;
      unpack2(v[j / 2], lo, hi);
      const int at = key(u) + j;
      v[j / 2] = pack2(at >= 0 && at < visible ? lo : other, at + 1 >= 0 && at + 1 < visible ? hi : other);
    }
  }
  // x <- scale x + bias
  __device__ __forceinline__ void logits(const Window<V>& win, uint32_t lut, float left, float right, uint64_t scale, int u,
                                         uint64_t* x) const {
    const int rel = key(u) - pos;
    if (rel >= win.hi || rel + V - 1 <= -win.w) {
      const uint64_t bias = both(rel >= win.hi ? right : left);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) x[j] = fma2(x[j], scale, bias);
    } else {
      const Places<V> at(lut, win.place(rel));
#pragma unroll
      for (int j = 0; j < V; j += 2)
        x[j / 2] = fma2(x[j / 2], scale, pack2(ld_shared_f32(at(j)), ld_shared_f32(at(j + 1))));
    }
  }
};

// v <- exp(v - m); v may be -inf, m is not.
template <int N>
__device__ __forceinline__ void exp_minus(uint64_t (&v)[N], float m) {
  const bool direct = fabsf(m) <= 0x1p100f;
  const uint64_t l = both(kLog2e), nm = both(direct ? -m * kLog2e : 0.0f);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint64_t t;
    if (direct) t = fma2(v[i], l, nm);
    else t = mul2(add2(v[i], both(-m)), l);
    float lo, hi;
    unpack2(t, lo, hi);
    v[i] = pack2(ex2_approx(lo), ex2_approx(hi));
  }
}

// 16-byte words of a thread for one row of one array.
template <int T, int kElems>
constexpr int row_words() { return kElems / act_vec<T>(); }

template <int T, int E, bool kDrop>
__global__ void __launch_bounds__(kTeamThreads) bias_softmax_kernel(const __grid_constant__ BiasSoftmaxArgs a) {
  constexpr int V = act_vec<T>(), U = E / V, P = E / 2, H = V / 2;
  extern __shared__ uint4 dynamic[];
  __shared__ TeamRecords<2> sh;
  const Team t = team_of(a.shape.warp_teams);
  const Window<V> win(a);
  Rows<T> rows(a, t);
  const uint32_t pitch = blockDim.x * 16, ring = shared_address(dynamic) + threadIdx.x * 16;
  float* const lut = reinterpret_cast<float*>(dynamic + a.ring_rows * row_words<T, E>() * blockDim.x);
  const uint32_t lut_at = shared_address(lut);
  const uint64_t bytes = a.batch * a.heads * a.queries * a.keys * uint64_t(dtype_bytes(T));
  pdl_enter();
  team_start(t);
  RowView<T> row;
  auto fetch = [&](uint32_t slot) {
#pragma unroll
    for (int u = 0; u < U; ++u) row.fetch(a, a.s, bytes, u, slot + uint32_t(u) * pitch);
  };
  rows.start();
  if (rows.left) {
    row = RowView<T>(rows, t, U);
    fetch(ring);
  }
  copy_async_commit();
  DropRun run{};
  if constexpr (kDrop) run = drop_run(a.drop, a.seed);
  fill_window(a, win, rows.head, lut);
  __syncthreads();
  const float left = lut[0], right = lut[win.word(win.places() - 1)];
  const uint64_t scale = both(a.scale);
  // the teams of a warp go on together: one without a row works on its last
  // again, without writing
  bool on = rows.left > 0;
  const bool two = a.ring_rows == 2;  // a row ahead; else the next one is fetched when this one is read
  for (uint32_t turn = 0; __any_sync(0xffffffffu, on); ++turn) {
    const uint32_t slot = ring + (two ? turn & 1u : 0u) * (uint32_t(U) * pitch);
    const int parity = int(turn & 1u);
    const RowView<T> r = row;
    const bool here = on;
    if (on) {
      rows.next();
      on = rows.left > 0;
      if (on) {
        row = RowView<T>(rows, t, U);
        if (two) fetch(ring + ((turn & 1u) ^ 1u) * (uint32_t(U) * pitch));
      }
    }
    copy_async_commit();
    if (two) copy_async_wait<1>();
    else copy_async_wait<0>();
    uint64_t e[P];
    float m = kNegInf;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint64_t* x = e + u * H;
      if (here && r.seen(u)) {
        act_widen2<T>(ld_shared(slot + uint32_t(u) * pitch), x);
        r.logits(win, lut_at, left, right, scale, u, x);
        r.mask(u, kNegInf, x);
#pragma unroll
        for (int j = 0; j < H; ++j) {
          float lo, hi;
          unpack2(x[j], lo, hi);
          m = fmaxf(m, fmaxf(lo, hi));
        }
      } else {
#pragma unroll
        for (int j = 0; j < H; ++j) x[j] = both(kNegInf);
      }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1)
      if (uint32_t(d) < t.lanes) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float base = m == kNegInf ? 0.0f : m;  // nothing visible: every 2^x below is 0
    exp_minus(e, base);
    uint64_t s2 = e[0], s3 = e[1];
#pragma unroll
    for (int i = 2; i < P; i += 2) {
      s2 = add2(s2, e[i]);
      s3 = add2(s3, e[i + 1]);
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
    factor = sum == 0.0f ? 0.0f : factor * __frcp_rn(sum);
    if (!two && on) fetch(ring);
    if (!here) continue;
    if (t.tid == 0 && t.rank == 0) a.lse[r.index] = sum == 0.0f ? kNegInf : top + logf(sum);
    const uint64_t by = both(kDrop ? factor * run.scale : factor);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint64_t* x = e + u * H;
      if (r.seen(u)) {
#pragma unroll
        for (int j = 0; j < H; ++j) x[j] = mul2(x[j], by);
        if constexpr (kDrop) {
          const uint64_t i[1] = {r.offset(u) / dtype_bytes(T)};
          bool keep[V];
          drop_keep<1, V>(run, i, keep);
#pragma unroll
          for (int j = 0; j < H; ++j) {
            float lo, hi;
            unpack2(x[j], lo, hi);
            x[j] = pack2(keep[2 * j] ? lo : 0.0f, keep[2 * j + 1] ? hi : 0.0f);
          }
        }
        r.mask(u, 0.0f, x);  // a row with a NaN has a NaN factor
      } else {
#pragma unroll
        for (int j = 0; j < H; ++j) x[j] = 0;
      }
      r.store(a, u, x);
    }
  }
}

template <int T, int E, bool kDrop>
__global__ void __launch_bounds__(kTeamThreads) bias_softmax_grad_kernel(const __grid_constant__ BiasSoftmaxArgs a) {
  constexpr int V = act_vec<T>(), U = E / V, P = E / 2, H = V / 2;
  extern __shared__ uint4 dynamic[];
  __shared__ TeamRecords<1> sh;
  __shared__ float ends[2][kTeamThreads / 32];
  const Team t = team_of(a.shape.warp_teams);
  const Window<V> win(a);
  Rows<T> rows(a, t);
  const int teams = a.shape.warp_teams ? int(blockDim.x / t.threads) : 1;
  const uint32_t pitch = blockDim.x * 16, ring = shared_address(dynamic) + threadIdx.x * 16;
  float* const lut = reinterpret_cast<float*>(dynamic + a.ring_rows * 2 * row_words<T, E>() * blockDim.x);
  float* const sums = lut + win.words();  // the teams' windows
  const uint32_t lut_at = shared_address(lut),
                 mine = shared_address(sums + (a.shape.warp_teams ? int(threadIdx.x / t.threads) : 0) * win.words());
  const uint64_t bytes = a.batch * a.heads * a.queries * a.keys * uint64_t(dtype_bytes(T));
  pdl_enter();
  team_start(t);
  RowView<T> row;
  float row_lse = 0.0f;
  auto fetch = [&](uint32_t slot) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      row.fetch(a, a.s, bytes, u, slot + uint32_t(2 * u) * pitch);
      row.fetch(a, a.dp, bytes, u, slot + uint32_t(2 * u + 1) * pitch);
    }
    row_lse = __ldg(a.lse_in + row.index);
  };
  rows.start();
  if (rows.left) {
    row = RowView<T>(rows, t, U);
    fetch(ring);
  }
  copy_async_commit();
  DropRun run{};
  if constexpr (kDrop) run = drop_run(a.drop, a.seed);
  fill_window(a, win, rows.head, lut);
  for (int i = int(threadIdx.x); i < teams * win.words(); i += int(blockDim.x)) sums[i] = 0.0f;
  __syncthreads();
  const float bias_left = lut[0], bias_right = lut[win.word(win.places() - 1)];
  const uint64_t scale = both(a.scale);
  const float drop_scale = kDrop ? run.scale : 1.0f;
  float left = 0.0f, right = 0.0f;  // dl of units wholly at rel <= -W, or at rel >= hi
  bool on = rows.left > 0;
  const bool two = a.ring_rows == 2;
  for (uint32_t turn = 0; __any_sync(0xffffffffu, on); ++turn) {
    const uint32_t slot = ring + (two ? turn & 1u : 0u) * (uint32_t(2 * U) * pitch);
    const RowView<T> r = row;
    const bool here = on;
    const float lse = row_lse, base = lse == kNegInf ? 0.0f : lse;  // all logits are -inf then, and every P is 0
    if (on) {
      rows.next();
      on = rows.left > 0;
      if (on) {
        row = RowView<T>(rows, t, U);
        if (two) fetch(ring + ((turn & 1u) ^ 1u) * (uint32_t(2 * U) * pitch));
      }
    }
    copy_async_commit();
    if (two) copy_async_wait<1>();
    else copy_async_wait<0>();
    uint64_t p[P], d[P];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint64_t *x = p + u * H, *y = d + u * H;
      if (here && r.seen(u)) {
        act_widen2<T>(ld_shared(slot + uint32_t(2 * u) * pitch), x);
        act_widen2<T>(ld_shared(slot + uint32_t(2 * u + 1) * pitch), y);
        r.logits(win, lut_at, bias_left, bias_right, scale, u, x);
        r.mask(u, kNegInf, x);
        r.mask(u, 0.0f, y);
        if constexpr (kDrop) {
          const uint64_t i[1] = {r.offset(u) / dtype_bytes(T)};
          bool keep[V];
          drop_keep<1, V>(run, i, keep);
#pragma unroll
          for (int j = 0; j < H; ++j) {
            float lo, hi;
            unpack2(y[j], lo, hi);
            y[j] = pack2(keep[2 * j] ? lo : 0.0f, keep[2 * j + 1] ? hi : 0.0f);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < H; ++j) {
          x[j] = both(kNegInf);
          y[j] = 0;
        }
      }
    }
    exp_minus(p, base);
    uint64_t s2 = mul2(p[0], d[0]), s3 = mul2(p[1], d[1]);
#pragma unroll
    for (int i = 2; i < P; i += 2) {
      s2 = fma2(p[i], d[i], s2);
      s3 = fma2(p[i + 1], d[i + 1], s3);
    }
    float dot[1] = {sum2(add2(s2, s3))};
    team_sum<1>(t, sh, int(turn & 1u), dot);
    if (a.shape.warp_teams) __syncwarp();  // the lanes' adds of the row before are done
    if (!two && on) fetch(ring);
    if (!here) continue;
    // dl = P (D(dp) - sum): the dropout's scale enters here
    const uint64_t by = both(drop_scale), minus = both(-dot[0] * drop_scale);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint64_t *x = p + u * H, o[H];
      if (r.seen(u)) {
#pragma unroll
        for (int j = 0; j < H; ++j) x[j] = mul2(x[j], fma2(d[u * H + j], by, minus));
        r.mask(u, 0.0f, x);  // a NaN sum stays with the keys that are seen
        const int rel = r.key(u) - r.pos;
        if (rel >= win.hi || rel + V - 1 <= -win.w) {
          uint64_t v = x[0];
#pragma unroll
          for (int j = 1; j < H; ++j) v = add2(v, x[j]);
          const float f = sum2(v);
          left += rel >= win.hi ? 0.0f : f;
          right += rel >= win.hi ? f : 0.0f;
        } else {
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
        for (int j = 0; j < H; ++j) o[j] = mul2(x[j], scale);
      } else {
#pragma unroll
        for (int j = 0; j < H; ++j) o[j] = 0;
      }
      r.store(a, u, o);
    }
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

// dtable[b, head]: a warp adds the head's CTAs in order of their chunks.
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

template <int T, bool kDrop>
const void* kernel_of_type(int elems, bool grad) {
  if (grad)
    return elems == 8    ? (const void*)bias_softmax_grad_kernel<T, 8, kDrop>
           : elems == 16 ? (const void*)bias_softmax_grad_kernel<T, 16, kDrop>
                         : (const void*)bias_softmax_grad_kernel<T, 32, kDrop>;
  return elems == 8    ? (const void*)bias_softmax_kernel<T, 8, kDrop>
         : elems == 16 ? (const void*)bias_softmax_kernel<T, 16, kDrop>
                       : (const void*)bias_softmax_kernel<T, 32, kDrop>;
}
template <bool kDrop>
const void* kernel_of(const BiasSoftmaxArgs& a, bool grad) {
  return a.type == kF32   ? kernel_of_type<kF32, kDrop>(a.shape.elems, grad)
         : a.type == kF16 ? kernel_of_type<kF16, kDrop>(a.shape.elems, grad)
                          : kernel_of_type<kBF16, kDrop>(a.shape.elems, grad);
}
const void* kernel_for(const BiasSoftmaxArgs& a, bool grad) {
  return a.drop.on ? kernel_of<true>(a, grad) : kernel_of<false>(a, grad);
}

// Shared memory above the default 48 KB (static arrays included) needs the kernel's limit raised.
cudaError_t allow_shared(const void* kernel, uint32_t bytes) {
  return bytes <= 32 * 1024 ? cudaSuccess
                            : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
}

constexpr uint32_t kSharedBytes = 216 * 1024;  // dynamic shared memory of a CTA at most

}  // namespace

TeamShape bias_softmax_shape(uint64_t keys, uint64_t rows, int type, bool grad, int sms) {
  (void)grad;
  const uint64_t v = type == kF32 ? 4 : 8;
  // a row that starts inside a unit spreads over one more
  const uint64_t span = keys % v ? keys + v - 1 : keys;
  TeamShape s{0, kWarpTeamThreads, 1, 32};
  if (rows >= uint64_t(sms) * 8 && span <= 32 * 32) {
    s.elems = span <= 32 * 16 ? 16 : 32;
    s.warp_teams = 4;
    while (span > uint64_t(s.warp_teams) * uint64_t(s.elems)) s.warp_teams *= 2;
    return s;
  }
  if (rows < uint64_t(sms) * 2) s.elems = 8;  // few rows: more threads for each
  while (s.elems < 32 && span > uint64_t(kTeamThreads) * s.elems) s.elems *= 2;
  // few rows: spread each over a cluster while SMs idle and every CTA keeps 256 threads' worth of a row
  while (s.ctas < kTeamCluster &&
         (span > uint64_t(kTeamThreads) * s.elems * s.ctas ||
          (rows * s.ctas * 2 <= uint64_t(sms) && span >= uint64_t(512) * s.elems * s.ctas)))
    s.ctas *= 2;
  const uint64_t per = uint64_t(s.elems) * s.ctas;
  s.threads = int(std::max<uint64_t>(32, ((span + per - 1) / per + 31) / 32 * 32));
  return s;
}

void bias_softmax_shared(BiasSoftmaxArgs* a, bool grad) {
  const uint32_t window = uint32_t(a->type == kF32 ? Window<4>(*a).words() : Window<8>(*a).words()) * 4;
  const uint32_t row = (grad ? 2u : 1u) * uint32_t(a->shape.elems) * (a->type == kF32 ? 4u : 2u);  // bytes of a thread
  a->ring_rows = 2;
  auto total = [&] {
    return a->ring_rows * row * uint32_t(a->shape.threads) +
           (1 + (grad ? uint32_t(team_count(a->shape)) : 0u)) * window;
  };
  // wide windows leave room for fewer teams, the longest f32 rows for one row at a time
  while (a->shape.warp_teams && total() > kSharedBytes / 2) {
    if (a->shape.threads > 32) a->shape.threads -= 32;
    else if (a->shape.warp_teams < 32) a->shape.warp_teams *= 2;
    else break;
  }
  if (total() > kSharedBytes) a->ring_rows = 1;
  a->shared_bytes = total();
}

cudaError_t bias_softmax_occupancy(const BiasSoftmaxArgs& a, bool grad, int* blocks_per_sm) {
  const void* kernel = kernel_for(a, grad);
  const cudaError_t e = allow_shared(kernel, a.shared_bytes);
  if (e != cudaSuccess) return e;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(blocks_per_sm, kernel, a.shape.threads, a.shared_bytes);
}

cudaError_t bias_softmax_launch(const BiasSoftmaxArgs& a, bool grad, cudaStream_t stream) {
  const uint64_t pairs = a.batch * a.queries;
  if (pairs && a.heads) {
    const void* kernel = kernel_for(a, grad);
    cudaError_t e = allow_shared(kernel, a.shared_bytes);
    if (e != cudaSuccess) return e;
    BiasSoftmaxArgs args = a;
    void* params[] = {&args};
    e = launch_rows(kernel, a.shape, a.heads * a.chunks * unsigned(a.shape.ctas), a.shared_bytes, params, stream);
    if (e != cudaSuccess) return e;
  }
  const uint64_t entries = uint64_t(a.heads) * a.buckets;
  if (!grad || !entries) return cudaSuccess;
  (void)launch_pdl(&bias_table_join_kernel, dim3(unsigned((entries + 7) / 8)), dim3(256), stream,
                   static_cast<const float*>(a.partial), a.dtable, a.heads, a.buckets, pairs ? a.chunks : 0u,
                   uint32_t(a.shape.ctas));
  return cudaGetLastError();
}

}  // namespace askb
