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
// exp(l - m) is 2^((l - m) log2 e) by ex2.approx (relative error 2^-22); the
// difference is taken first, as m log2 e overflows for rows at the type's
// lowest value (and a branch for them cost more than the second operation).
// Each warp takes its own maximum, and its sum is rescaled when the team's
// records meet: one exchange a row.
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

// The window as units meet it: V copies, the r-th shifted by r places, so that a
// unit's V biases are V neighbouring words on a 16-byte boundary (2 loads in place
// of V, and no place to work out for each).  Column c of copy r holds distances
// V (c + low) + r and up; columns at either end hold the constants.  They pay
// where teams have many rows and the window is not too wide.
template <int V>
struct Lut {
  uint32_t at;        // shared address of the window
  uint32_t copies;    // of the copies
  int columns;        // of a copy; 0: there are none
  int low, high;      // first and last column
  float left, right;  // biases at rel <= -W and at rel >= hi
  __host__ __device__ static int first_column(int w) { return -((w + 2 * V - 2 + V - 1) / V); }
  __host__ __device__ static int last_column(int hi) { return (hi + V - 1) / V; }
  __host__ __device__ static int words(const Window<V>& win) {
    return (last_column(win.hi) - first_column(win.w) + 1) * V * V;
  }
  __device__ __forceinline__ uint32_t shifted(int rel) const {
    const int c = max(min(rel >> (V == 8 ? 3 : 2), high), low) - low;
    return copies + uint32_t(((rel & (V - 1)) * columns + c) * (V * 4));
  }
};

// The head's bias by distance into `window` (and the copies behind it).
template <int V>
__device__ __forceinline__ Lut<V> fill_window(const BiasSoftmaxArgs& a, const Window<V>& win, uint32_t head, float* window,
                                              float* copies) {
  for (int i = int(threadIdx.x); i < win.places(); i += int(blockDim.x)) {
    float v[1];
    param_load<1>(a.table, a.table_type, uint64_t(bucket_of(a, win.rel(i))) * a.heads + head, v);
    window[win.word(i)] = v[0];
  }
  __syncthreads();
  Lut<V> lut;
  lut.at = shared_address(window);
  lut.copies = shared_address(copies);
  lut.low = Lut<V>::first_column(win.w);
  lut.high = Lut<V>::last_column(win.hi);
  lut.columns = a.window_copies ? lut.high - lut.low + 1 : 0;
  lut.left = window[0];
  lut.right = window[win.word(win.places() - 1)];
  if (lut.columns) {
    for (int i = int(threadIdx.x); i < lut.columns * V; i += int(blockDim.x))
#pragma unroll
      for (int r = 0; r < V; ++r) {
        const int rel = V * lut.low + i + r;  // column i / V of copy r, word i % V
        copies[r * lut.columns * V + i] = window[win.word(win.place(max(min(rel, win.hi), -win.w)))];
      }
    __syncthreads();
  }
  return lut;
}

// The rows of a team, one after the other: pairs (batch, query) of one head.
// kEven: rows are whole 16-byte units (keys a multiple of V, aligned tensors).
template <int T, bool kEven>
struct Rows {
  static constexpr int V = act_vec<T>();
  uint32_t head, step, b, q;
  uint32_t left;       // rows from this one on
  int length, place;   // of the sequence: keys in use, position of its query 0
  uint64_t index;      // of the row
  uint32_t mine;       // this thread's first unit, in elements of a row

  __device__ __forceinline__ Rows(const BiasSoftmaxArgs& a, const Team& t, int units) {
    const uint32_t cta = blockIdx.x / t.ctas, chunk = cta / a.heads;
    // rows of one head go round its teams, so short sequences and the short rows
    // of a causal head fall to all of them alike
    const uint64_t n = a.batch * a.queries, begin = uint64_t(chunk) * t.count + t.index;
    head = cta % a.heads;
    step = a.chunks * t.count;
    left = begin < n ? uint32_t((n - begin + step - 1) / step) : 0;
    b = uint32_t(begin / a.queries);
    q = uint32_t(begin % a.queries);
    mine = (t.rank * uint32_t(units) * t.threads + t.tid) * uint32_t(V);
    if (left) sequence(a);
  }
  __device__ __forceinline__ void sequence(const BiasSoftmaxArgs& a) {
    length = int(a.keys);
    place = 0;
    if (a.lengths) length = max(min(__ldg(a.lengths + b), length), 0);
    // far positions meet only the window's ends, whatever their distance
    if (a.offsets) place = max(min(__ldg(a.offsets + b), (1 << 30) - 1), -(1 << 30));
    index = (uint64_t(b) * a.heads + head) * a.queries + q;
  }
  __device__ __forceinline__ void next(const BiasSoftmaxArgs& a) {
    if (--left == 0) return;
    q += step;
    index += step;
    if (q >= uint32_t(a.queries)) {
      const uint32_t n = q / uint32_t(a.queries);
      b += n;
      q -= n * uint32_t(a.queries);
      sequence(a);
    }
  }
};

// One row, in flight or at work, as a thread sees it: unit u begins at key
// k + u * (keys between units) and at byte offset off + u * (bytes between units).
struct RowView {
  uint64_t off;
  int k, visible, pos;  // keys [0, visible) are seen; position of the query
};
// What a unit of a warp's lanes is (seen by some, whole and seen in all, reaching
// into the window in some) is decided for the warp by votes, so that no unit
// costs a divergent branch.  Units without a visible key are worked on all the
// same, on what their words last held, and masked: leaving them out cost more
// (a branch around a unit's registers took 4.6 instructions an element, its
// arithmetic takes 9); only their random words are not drawn.
template <int T, bool kEven>
struct Units {
  static constexpr int V = act_vec<T>(), B = dtype_bytes(T);
  int keys;
  int key_step;        // keys between a thread's units
  __device__ __forceinline__ Units(const BiasSoftmaxArgs& a, const Team& t) : keys(int(a.keys)), key_step(int(t.threads) * V) {}

  __device__ __forceinline__ RowView view(const BiasSoftmaxArgs& a, const Rows<T, kEven>& rows) const {
    RowView r;
    uint64_t e = rows.index * a.keys + rows.mine;
    r.k = int(rows.mine);
    if constexpr (!kEven) {  // the tensor's own units: the first begins before the row
      const uint32_t shift = uint32_t(e) & uint32_t(V - 1);
      e -= shift;
      r.k -= int(shift);
    }
    r.off = e * B;
    r.pos = rows.place + int(rows.q);  // q is below 2^30
    r.visible = rows.length;
    if (a.causal) r.visible = max(min(r.visible, r.pos + 1), 0);
    return r;
  }
  __device__ __forceinline__ int key(const RowView& r, int u) const { return r.k + u * key_step; }
  __device__ __forceinline__ uint64_t offset(const RowView& r, int u) const { return r.off + uint32_t(u * key_step * B); }
  __device__ __forceinline__ bool seen(const RowView& r, int u) const {
    return key(r, u) < r.visible && (kEven || key(r, u) > -V);
  }

  // `units` lie in the tensor whole: all rows but its last one's, of an aligned tensor
  __device__ __forceinline__ void fetch(const void* p, const RowView& r, bool units, int u, uint32_t slot) const {
    if (!seen(r, u)) return;
    const char* from = static_cast<const char*>(p) + offset(r, u);
    if (kEven || units) {
      copy_to_shared(slot, from);
    } else {  // by elements
      uint32_t w[4] = {};
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int at = key(r, u) + j;
        if (at < 0 || at >= r.visible) continue;
        const uint32_t bits = B == 4 ? __ldg(reinterpret_cast<const uint32_t*>(from) + j)
                                     : uint32_t(__ldg(reinterpret_cast<const unsigned short*>(from) + j));
        w[j * B / 4] |= bits << (8 * (j * B % 4));
      }
      st_shared(slot, make_uint4(w[0], w[1], w[2], w[3]));
    }
  }
  __device__ __forceinline__ bool any_seen(const RowView& r, int u) const { return __any_sync(0xffffffffu, seen(r, u)); }
  __device__ __forceinline__ bool all_whole(const RowView& r, int u) const {
    const int k0 = key(r, u);
    return __all_sync(0xffffffffu, (kEven || k0 >= 0) && k0 + V <= r.visible);
  }
  __device__ __forceinline__ bool any_near(const RowView& r, const Window<V>& win, int u) const {
    const int rel = key(r, u) - r.pos;
    return __any_sync(0xffffffffu, rel < win.hi && rel + V - 1 > -win.w);
  }
  // the unit's elements that belong to the row
  __device__ __forceinline__ void store(const BiasSoftmaxArgs& a, const RowView& r, int u, const uint4& o) const {
    const int k0 = key(r, u);
    if (k0 >= keys) return;
    char* to = static_cast<char*>(a.out) + offset(r, u);
    if (kEven || (a.aligned && k0 >= 0 && k0 + V <= keys)) {
      st_stream_v4(to, o);
      return;
    }
    const uint32_t w[4] = {o.x, o.y, o.z, o.w};
    const int first = max(-k0, 0), end = min(keys - k0, V);
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // by words, and by halves of them
      if constexpr (B == 4) {
        if (k >= first && k < end) reinterpret_cast<uint32_t*>(to)[k] = w[k];
      } else {
        const bool lo = 2 * k >= first && 2 * k < end, hi = 2 * k + 1 >= first && 2 * k + 1 < end;
        if (lo && hi && a.aligned) reinterpret_cast<uint32_t*>(to)[k] = w[k];
        else {
          if (lo) reinterpret_cast<uint16_t*>(to)[2 * k] = uint16_t(w[k]);
          if (hi) reinterpret_cast<uint16_t*>(to)[2 * k + 1] = uint16_t(w[k] >> 16);
        }
      }
    }
  }
  // v <- v where the key is visible, else `other`
  __device__ __forceinline__ void mask(const RowView& r, int u, float other, uint64_t* v) const {
    // key k0 + j is visible when j - first is below n, without a sign
    const int k0 = key(r, u), first = kEven ? 0 : max(-k0, 0);
    const uint32_t n = uint32_t(max(r.visible - k0 - first, 0));
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      float lo, hi;
      unpack2(v[j / 2], lo, hi);
      v[j / 2] = pack2(uint32_t(j - first) < n ? lo : other, uint32_t(j + 1 - first) < n ? hi : other);
    }
  }
  // x <- scale x + bias
  __device__ __forceinline__ void logits(const RowView& r, const Window<V>& win, const Lut<V>& lut, uint64_t scale, int u,
                                         uint64_t* x) const {
    const int rel = key(r, u) - r.pos;
    if (!any_near(r, win, u)) {
      const uint64_t bias = both(rel >= win.hi ? lut.right : lut.left);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) x[j] = fma2(x[j], scale, bias);
    } else if (lut.columns) {
      const uint32_t at = lut.shifted(rel);
#pragma unroll
      for (int j = 0; j < V / 2; j += 2) {
        uint64_t b0, b1;
        asm volatile("ld.shared.v2.u64 {%0,%1}, [%2];" : "=l"(b0), "=l"(b1) : "r"(at + 8u * j) : "memory");
        x[j] = fma2(x[j], scale, b0);
        x[j + 1] = fma2(x[j + 1], scale, b1);
      }
    } else {
      // the places from hi on, and those up to -W, hold the constants
      const Places<V> at(lut.at, win.place(max(min(rel, win.hi), -win.w - (V - 1))));
#pragma unroll
      for (int j = 0; j < V; j += 2)
        x[j / 2] = fma2(x[j / 2], scale, pack2(ld_shared_f32(at(j)), ld_shared_f32(at(j + 1))));
    }
  }
};

__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float lg2_approx(float v) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// v <- exp(v - m); v may be -inf, m is not.
template <int N>
__device__ __forceinline__ void exp_minus(uint64_t* v, uint64_t minus_m) {
  const uint64_t l = both(kLog2e);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float lo, hi;
    unpack2(mul2(add2(v[i], minus_m), l), lo, hi);
    v[i] = pack2(ex2_approx(lo), ex2_approx(hi));
  }
}
// The largest of three.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 16-byte words of a thread for one row of one array.
template <int T, int kElems>
constexpr int row_words() { return kElems / act_vec<T>(); }

template <int T, int E, bool kDrop, bool kEven>
__global__ void __launch_bounds__(kTeamThreads) bias_softmax_kernel(const __grid_constant__ BiasSoftmaxArgs a) {
  constexpr int V = act_vec<T>(), U = E / V, H = V / 2;
  extern __shared__ uint4 dynamic[];
  __shared__ TeamRecords<2> sh;
  const Team t = team_of(a.shape);
  const Window<V> win(a);
  const uint32_t pitch = blockDim.x * 16, ring = shared_address(dynamic) + threadIdx.x * 16;
  float* const copies = reinterpret_cast<float*>(dynamic + a.ring_rows * row_words<T, E>() * blockDim.x);
  float* const window = copies + (a.window_copies ? Lut<V>::words(win) : 0);
  const uint64_t last_row = a.batch * a.heads * a.queries - 1;
  const Units<T, kEven> units(a, t);
  pdl_enter();
  team_start(t);
  Rows<T, kEven> rows(a, t, U);
  RowView row{};
  uint64_t index = 0;
  auto fetch = [&](uint32_t slot) {
#pragma unroll
    for (int u = 0; u < U; ++u) units.fetch(a.s, row, a.aligned && rows.index != last_row, u, slot + uint32_t(u) * pitch);
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
__global__ void __launch_bounds__(kTeamThreads) bias_softmax_grad_kernel(const __grid_constant__ BiasSoftmaxArgs a) {
  constexpr int V = act_vec<T>(), U = E / V, H = V / 2;
  extern __shared__ uint4 dynamic[];
  __shared__ TeamRecords<1> sh;
  __shared__ float ends[2][kTeamThreads / 32];
  const Team t = team_of(a.shape);
  const Window<V> win(a);
  const int teams = int(t.count);
  const uint32_t pitch = blockDim.x * 16, ring = shared_address(dynamic) + threadIdx.x * 16;
  float* const copies = reinterpret_cast<float*>(dynamic + a.ring_rows * 2 * row_words<T, E>() * blockDim.x);
  float* const window = copies + (a.window_copies ? Lut<V>::words(win) : 0);
  float* const sums = window + win.words();  // the teams' windows
  const uint32_t mine = shared_address(sums + int(t.index) * win.words());
  const uint64_t last_row = a.batch * a.heads * a.queries - 1;
  const Units<T, kEven> units(a, t);
  pdl_enter();
  team_start(t);
  Rows<T, kEven> rows(a, t, U);
  RowView row{};
  float row_lse = 0.0f;
  auto fetch = [&](uint32_t slot) {
    const bool whole = a.aligned && rows.index != last_row;
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
    if (a.shape.warp_teams) __syncwarp();  // the lanes' adds of the row before are done
    // masked keys hold P = 0 already, unless the sum is a NaN or infinite
    const bool odd = __any_sync(0xffffffffu, here && !(fabsf(dot[0]) <= 3.4e38f));
    if (!two && on) fetch(ring);
    // dl = P (D(dp) - sum): the dropout's scale enters here
    const uint64_t by = both(drop_scale), minus = both(-dot[0] * drop_scale);
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

template <int T, int E, bool kDrop>
const void* kernel_of_fit(bool grad, bool even) {
  if (grad)
    return even ? (const void*)bias_softmax_grad_kernel<T, E, kDrop, true> : (const void*)bias_softmax_grad_kernel<T, E, kDrop, false>;
  return even ? (const void*)bias_softmax_kernel<T, E, kDrop, true> : (const void*)bias_softmax_kernel<T, E, kDrop, false>;
}
template <int T, bool kDrop>
const void* kernel_of_type(const BiasSoftmaxArgs& a, bool grad) {
  const bool even = a.aligned && a.keys % uint32_t(act_vec<T>()) == 0;
  return a.shape.elems == 8    ? kernel_of_fit<T, 8, kDrop>(grad, even)
         : a.shape.elems == 16 ? kernel_of_fit<T, 16, kDrop>(grad, even)
         : a.shape.elems == 24 ? kernel_of_fit<T, 24, kDrop>(grad, even)
         : a.shape.elems == 32 ? kernel_of_fit<T, 32, kDrop>(grad, even)
         : even                ? (const void*)bias_softmax_kernel<T, 40, kDrop, true>
                               : (const void*)bias_softmax_kernel<T, 40, kDrop, false>;
}
template <bool kDrop>
const void* kernel_of(const BiasSoftmaxArgs& a, bool grad) {
  return a.type == kF32   ? kernel_of_type<kF32, kDrop>(a, grad)
         : a.type == kF16 ? kernel_of_type<kF16, kDrop>(a, grad) : kernel_of_type<kBF16, kDrop>(a, grad);
}
const void* kernel_for(const BiasSoftmaxArgs& a, bool grad) {
  return a.drop.on ? kernel_of<true>(a, grad) : kernel_of<false>(a, grad);
}

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
  // the window's copies where a warp's rows are many and they take little
  a->window_copies = a->shape.warp_teams && copies <= 12 * 1024 && total() + copies <= kSharedBytes ? 1 : 0;
  a->shared_bytes = total();
}

cudaError_t bias_softmax_occupancy(const BiasSoftmaxArgs& a, bool grad, int* blocks_per_sm) {
  const void* kernel = kernel_for(a, grad);
  const cudaError_t e = prepare_rows(kernel, a.shared_bytes);
  if (e != cudaSuccess) return e;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(blocks_per_sm, kernel, a.shape.threads, a.shared_bytes);
}

cudaError_t bias_softmax_launch(const BiasSoftmaxArgs& a, bool grad, cudaStream_t stream) {
  const uint64_t pairs = a.batch * a.queries;
  if (pairs && a.heads) {
    const void* kernel = kernel_for(a, grad);
    cudaError_t e = prepare_rows(kernel, a.shared_bytes);
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
