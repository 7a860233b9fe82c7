// Softmax of scores with a learned relative-position bias (bias_softmax_forward.cu),
// and its gradient (bias_softmax_grad.cu).
//
//   l = scale s + table[bucket(k - pos), head],  pos = query + offset[batch]
//   over the keys k < length[batch] (and k <= pos when causal);
//   p = D(exp(l - lse)),  lse = log sum exp l,  D dropout; a row without keys
//   gives zeros and lse = -inf.
//   Gradient: P = exp(l - lse), divided by its sum where lse is too coarse to carry
//   that, d = D(dp), dl = P (d - sum P d), ds = scale dl, dtable[b, head] = sum of dl
//   where the bucket is b.
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
// the neighbouring rows; those are masked, and only such cut units are stored in
// parts (by words, and halves at either end).  Units without a visible key are not read.  The next row's
// units are on their way (cp.async into words that only their own thread reads)
// while this row is worked on.
//
// exp(l - m) is 2^((l - m) log2 e) by ex2.approx (relative error 2^-22); the
// difference is taken first, as m log2 e overflows for rows at the type's
// lowest value (and a branch for them cost more than the second operation).
// Each warp takes its own maximum, and its sum is rescaled when the team's
// records meet: one exchange a row.
//
// Bound: instruction issue.  A warp's 32 bf16 elements move 128 bytes, 22 clocks
// of a scheduler's share of HBM; they take about 20 instructions, 8 clocks of ex2
// among them, and with dropout the generator's 21 clocks more.  bf16 [8, 16, 1024, 1024]: 95 us full
// and without dropout (5.6 TB/s), 177 us with dropout and ragged lengths;
// gradient 145 and 234 us.  Rows that are not whole units add masks, cut
// stores and a unit more a row (1021 keys: 264 us).
#pragma once

#include <cuda_runtime.h>

#include <algorithm>

#include "act_io.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "philox.cuh"
#include "row_team.cuh"

namespace askb {

namespace {

constexpr int kWarpTeamThreads = 128;
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
    // far positions meet only the window's ends, whatever their distance; the upper bound
    // leaves a unit that begins before its row within 32 bits of the last query
    if (a.offsets) place = max(min(__ldg(a.offsets + b), (1 << 30) - 16), -(1 << 30));
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

  // `units`: the row's units lie in the tensor whole
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
    const int first = max(-k0, 0), end = min(keys - k0, V);
    if (B == 4 || a.aligned) {
      store_cut<T>(to, o, first, end);
    } else {  // a 16-bit tensor may begin inside a word
      const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j >= first && j < end) reinterpret_cast<uint16_t*>(to)[j] = uint16_t(w[j / 2] >> (16 * (j % 2)));
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

// The kernel of a step: Pick<T, elements a thread, drop, even>::get(args).
template <template <int, int, bool, bool> class Pick, int T, int E, bool kDrop>
const void* choose_fit(const BiasSoftmaxArgs& a) {
  const bool even = a.aligned && a.keys % uint32_t(act_vec<T>()) == 0;
  return even ? Pick<T, E, kDrop, true>::get(a) : Pick<T, E, kDrop, false>::get(a);
}
template <template <int, int, bool, bool> class Pick, int T, bool kDrop>
const void* choose_elems(const BiasSoftmaxArgs& a) {
  switch (a.shape.elems) {
    case 8: return choose_fit<Pick, T, 8, kDrop>(a);
    case 16: return choose_fit<Pick, T, 16, kDrop>(a);
    case 24: return choose_fit<Pick, T, 24, kDrop>(a);
    case 32: return choose_fit<Pick, T, 32, kDrop>(a);
    default: return choose_fit<Pick, T, 40, kDrop>(a);
  }
}
template <template <int, int, bool, bool> class Pick, bool kDrop>
const void* choose_type(const BiasSoftmaxArgs& a) {
  return a.type == kF32   ? choose_elems<Pick, kF32, kDrop>(a)
         : a.type == kF16 ? choose_elems<Pick, kF16, kDrop>(a) : choose_elems<Pick, kBF16, kDrop>(a);
}
template <template <int, int, bool, bool> class Pick>
const void* choose(const BiasSoftmaxArgs& a) {
  return a.drop.on ? choose_type<Pick, true>(a) : choose_type<Pick, false>(a);
}

inline cudaError_t rows_occupancy(const void* kernel, const BiasSoftmaxArgs& a, int* blocks_per_sm) {
  const cudaError_t e = prepare_rows(kernel, a.shared_bytes);
  if (e != cudaSuccess) return e;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(blocks_per_sm, kernel, a.shape.threads, a.shared_bytes);
}
inline cudaError_t rows_launch(const void* kernel, const BiasSoftmaxArgs& a, cudaStream_t stream) {
  const cudaError_t e = prepare_rows(kernel, a.shared_bytes);
  if (e != cudaSuccess) return e;
  BiasSoftmaxArgs args = a;
  void* params[] = {&args};
  return launch_rows(kernel, a.shape, a.heads * a.chunks * unsigned(a.shape.ctas), a.shared_bytes, params, stream);
}

}  // namespace

}  // namespace askb
