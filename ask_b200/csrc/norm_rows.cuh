// Block norms: the row work between two blocks of a transformer in one pass,
//   h = alpha x + D(g * N_post(y)),   u = N_pre(h),
// (norm_forward.cu) and its gradient in one pass plus a join of the column sums
// (norm_grad.cu).
//
//   N(v) = vhat * w (+ b),  vhat = (v - mean) r,  r = 1 / sqrt(var + eps);
//   the rms norm has mean = 0.  D is dropout, g a gate shared by a group of
//   consecutive rows.  mean and r are the row's saved statistics.
//
// Statistics come from 32-bit values: var of a layer norm is the mean square
// of v - mean, taken in registers in a second step, and u is computed from h
// before h is rounded to its storage type.
//
// A row is held by a team of threads, 16 elements each.  Every thread copies
// its own words of the rows to come into its own places of a ring in shared
// memory (cp.async) and reads them back, so no barrier is needed and no register
// holds what is on its way.  Its parameters lie beside them in shared memory for
// all of its rows.  Arithmetic runs on f32 pairs.  (Rows prefetched into
// registers and parameters reloaded for each row took 446 us where this takes
// 243, the gradient 831 where it takes 338.)
//
// Bound: HBM, four tensors forward and six for the gradient, up to 6400
// columns without dropout (bf16 [32768, 4096]: 188 us = 5.7 TB/s, gradient 268 us =
// 6.0 TB/s); with dropout the generator's latencies add to it (243 and 338 us; 231
// and 314 where the same kernel runs back to back, as both sides did in the
// comparisons below and in the kernels' files).  Wider rows have one team an SM, whose loads wait while it reduces
// (8192 columns: 161 us for half the elements, gradient 206), and those over a
// cluster wait for its barriers (16384: 238 and 284).
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

constexpr int kElems = 16;  // row elements a thread holds
constexpr int kPairs = kElems / 2;

// Which of the step's switches the kernel has folded in; FORM_ANY reads them.
enum NormForm { FORM_ANY = 0, FORM_BOTH = 1 /* branch, post and pre norm */, FORM_ADD = 2 /* branch as it is, pre norm */,
                FORM_NORM = 3 /* pre norm alone */ };

// The team's columns of a row, as the thread holds them: kElems / V units of V
// elements.  A unit is 16 bytes of the row (NORM_UNITS); an aligned unit of the
// tensor, of which the row's first and last may hold neighbours' elements that
// count as zeros and are not written (NORM_CUT: all rows of a team begin at the
// same place of a unit, so its columns and parameters stay as they are); an f32
// (NORM_WORDS, lane after lane); or 16 bytes that begin anywhere (NORM_ANYWHERE,
// 16-bit types: it spans two aligned words, from which it is shifted out, and
// stores are put together across lanes).  A row is named by the byte offset of
// this thread's first column.
template <int T, int F>
struct Columns {
  static constexpr int E = kElems, P = kPairs, B = dtype_bytes(T);
  static constexpr int kUnitBytes = F == NORM_WORDS ? 4 : 16, V = kUnitBytes / B, Q = E / V;
  static constexpr int kCopies = F == NORM_ANYWHERE ? 2 : 1;     // words of a unit in the ring
  static constexpr int kArrayBytes = Q * kCopies * kUnitBytes;   // of a thread, for one row of one array
  int first, step;  // column of unit q: first + q * step
  int cols;
  uint32_t pitch;  // between a thread's words in shared memory
  uint32_t cuts;   // bit q: the warp's units q are not all whole (NORM_CUT)
  __device__ __forceinline__ Columns(const Team& t, const NormArgs& a, uint64_t row)
      : first(int((t.rank * uint32_t(Q) * t.threads + t.tid) * uint32_t(V))), step(int(t.threads) * V), cols(int(a.cols)),
        pitch(blockDim.x * uint32_t(kUnitBytes)), cuts(0) {
    if constexpr (F == NORM_CUT) {
      first -= int(uint32_t(row * a.cols) & uint32_t(V - 1));
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (__any_sync(0xffffffffu, in(q) && count(q) < V)) cuts |= 1u << q;
    }
  }
  __device__ __forceinline__ int at(int q) const { return first + q * step; }
  __device__ __forceinline__ bool in(int q) const { return at(q) < cols; }
  // unit q's elements [low(q), high(q)) are columns of the row
  __device__ __forceinline__ int low(int q) const { return F == NORM_CUT ? max(-at(q), 0) : 0; }
  __device__ __forceinline__ int high(int q) const { return max(min(cols - at(q), V), 0); }
  __device__ __forceinline__ int count(int q) const { return high(q) - (in(q) ? low(q) : 0); }
  __device__ __forceinline__ bool has(int q, int j) const { return j >= low(q) && j < high(q); }
  __device__ __forceinline__ uint64_t offset(uint64_t row) const {
    return (row * uint32_t(cols) + uint64_t(int64_t(first))) * uint64_t(B);
  }
  __device__ __forceinline__ uint64_t unit(uint64_t off, int q) const { return off + uint32_t(q * step * B); }
  __device__ __forceinline__ static uint32_t ring(const void* shared) {
    return shared_address(shared) + threadIdx.x * uint32_t(kUnitBytes);
  }

  // `slot`: this thread's words of the array in a stage.  What no column fills
  // is zeroed once, by clear().
  __device__ __forceinline__ void fetch(const void* p, uint64_t off, uint64_t bytes, uint32_t slot) const {
    const char* begin = static_cast<const char*>(p);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (!in(q)) continue;
      const uint64_t o = unit(off, q);
      if constexpr (F == NORM_UNITS) {
        copy_to_shared(slot + uint32_t(q) * pitch, begin + o);
      } else if constexpr (F == NORM_CUT) {
        if (o + 16 <= bytes) copy_to_shared(slot + uint32_t(q) * pitch, begin + o);
        else st_shared(slot + uint32_t(q) * pitch, load_part<T>(begin + o, begin, begin + bytes));
      } else if constexpr (F == NORM_WORDS) {
        copy_word_to_shared(slot + uint32_t(q) * pitch, begin + o);
      } else {
        const char* word = begin + o - (uint32_t(reinterpret_cast<uintptr_t>(begin + o)) & 15u);
        const uint32_t to = slot + uint32_t(2 * q) * pitch;
        if (o >= 16 && o + 32 <= bytes) {  // both words lie in the tensor
          copy_to_shared(to, word);
          copy_to_shared(to + pitch, word + 16);
        } else {  // its ends: only what belongs to it is read
          st_shared(to, load_part<T>(word, begin, begin + bytes));
          st_shared(to + pitch, load_part<T>(word + 16, begin, begin + bytes));
        }
      }
    }
  }
  __device__ __forceinline__ void clear(uint32_t slot) const {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (in(q)) continue;
      if constexpr (F == NORM_UNITS || F == NORM_CUT) st_shared(slot + uint32_t(q) * pitch, make_uint4(0u, 0u, 0u, 0u));
      if constexpr (F == NORM_WORDS) st_shared_word(slot + uint32_t(q) * pitch, 0u);
    }
  }
  // Cut units' elements of neighbouring rows count as zeros.  The forward kernel masks
  // what it reads (kMask); the gradient has no registers for that, and zeroes
  // them where they lie, in `arrays` arrays of a stage (f32 [33520, 1001]
  // gradients 216 us masked, 173 so; forward 107 masked, 112 so).
  __device__ __forceinline__ void trim(uint32_t slot, int arrays, uint32_t array) const {
    if constexpr (F == NORM_CUT) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        if (!(cuts & 1u << q) || !in(q)) continue;
        const uint32_t to = slot + uint32_t(q) * pitch;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (has(q, j)) continue;
          for (int k = 0; k < arrays; ++k) {
            if constexpr (B == 4) st_shared_word(to + uint32_t(k) * array + 4u * j, 0u);
            else st_shared_half(to + uint32_t(k) * array + 2u * j, 0);
          }
        }
      }
    }
  }
  __device__ __forceinline__ void clear_outside(int q, uint64_t* v) const {
    const uint32_t from = uint32_t(low(q)), n = uint32_t(count(q));
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      float lo, hi;
      unpack2(v[j / 2], lo, hi);
      v[j / 2] = pack2(uint32_t(j) - from < n ? lo : 0.0f, uint32_t(j + 1) - from < n ? hi : 0.0f);
    }
  }
  template <bool kMask>
  __device__ __forceinline__ void read(uint32_t slot, const void* p, uint64_t off, uint64_t (&v)[P]) const {
    if constexpr (F == NORM_UNITS || F == NORM_CUT) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        act_widen2<T>(ld_shared(slot + uint32_t(q) * pitch), v + q * V / 2);
        if (kMask && F == NORM_CUT && (cuts & 1u << q)) clear_outside(q, v + q * V / 2);
      }
    } else if constexpr (F == NORM_WORDS) {
#pragma unroll
      for (int k = 0; k < P; ++k)
        v[k] = pack2(__uint_as_float(ld_shared_word(slot + uint32_t(2 * k) * pitch)),
                     __uint_as_float(ld_shared_word(slot + uint32_t(2 * k + 1) * pitch)));
    } else {
      // of all units: they are whole words apart
      const uint32_t shift = (uint32_t(reinterpret_cast<uintptr_t>(p)) + uint32_t(off)) & 15u;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        float f[V];
        act_widen<T>(unit_at<T>(ld_shared(slot + uint32_t(2 * q) * pitch), ld_shared(slot + uint32_t(2 * q + 1) * pitch), shift), f);
        const int n = count(q);
        if (n < V) {
#pragma unroll
          for (int j = 0; j < V; ++j) f[j] = j < n ? f[j] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < V; j += 2) v[(q * V + j) / 2] = pack2(f[j], f[j + 1]);
      }
    }
  }
  __device__ __forceinline__ void put(const Team& t, void* p, uint64_t off, bool on, const uint64_t (&v)[P]) const {
    char* to = static_cast<char*>(p);
    if constexpr (F == NORM_UNITS) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (on && in(q)) st_stream_v4(to + unit(off, q), act_narrow2<T>(v + q * V / 2));
    } else if constexpr (F == NORM_CUT) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        if (!on || !in(q)) continue;
        const uint4 o = act_narrow2<T>(v + q * V / 2);
        if (count(q) == V) st_stream_v4(to + unit(off, q), o);
        else store_cut<T>(to + unit(off, q), o, low(q), high(q));
      }
    } else if constexpr (F == NORM_WORDS) {
#pragma unroll
      for (int k = 0; k < P; ++k) {
        float lo, hi;
        unpack2(v[k], lo, hi);
        if (on && in(2 * k)) st_stream_u32(to + unit(off, 2 * k), __float_as_uint(lo));
        if (on && in(2 * k + 1)) st_stream_u32(to + unit(off, 2 * k + 1), __float_as_uint(hi));
      }
    } else {
      const uint32_t place = t.lane & (t.lanes - 1);
#pragma unroll
      for (int q = 0; q < Q; ++q)
        store_anywhere<T>(to + unit(off, q), act_narrow2<T>(v + q * V / 2), on ? count(q) : 0, place == 0,
                          place == t.lanes - 1);
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
#pragma unroll
      for (int j = 0; j < V; ++j) f[q * V + j] = has(q, j) ? fill : 0.0f;
      if (!p) continue;
      if constexpr (F == NORM_UNITS) {
        if (in(q)) param_load<V>(p, type, offset + uint32_t(at(q)), f + q * V);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (has(q, j)) param_load<1>(p, type, offset + uint32_t(at(q) + j), f + q * V + j);
      }
    }
  }
  // v - mean; where there is no column, 0 if kExact
  template <bool kExact>
  __device__ __forceinline__ void center(float mean, uint64_t (&v)[P]) const {
    if constexpr (!kExact) {
      const uint64_t m = both(-mean);
#pragma unroll
      for (int k = 0; k < P; ++k) v[k] = add2(v[k], m);
    } else if constexpr (F == NORM_UNITS || F == NORM_CUT) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const uint64_t m = both(in(q) ? -mean : 0.0f);
#pragma unroll
        for (int k = 0; k < V / 2; ++k) v[q * V / 2 + k] = add2(v[q * V / 2 + k], m);
        if (F == NORM_CUT && (cuts & 1u << q)) clear_outside(q, v + q * V / 2);
      }
    } else {
      float f[E];
      unpack(v, f);
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int n = count(q);
#pragma unroll
        for (int j = 0; j < V; ++j) f[q * V + j] -= j < n ? mean : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < P; ++k) v[k] = pack2(f[2 * k], f[2 * k + 1]);
    }
  }
  // zero where dropped; the scale is folded into what the values meet next.
  // Units past the row hold zeros, whatever is drawn for them.
  __device__ __forceinline__ void drop(const DropRun& run, uint64_t off, uint64_t (&v)[P]) const {
    float f[E];
    unpack(v, f);
    bool keep[E];
    const uint64_t e = off / B;
    if constexpr (F == NORM_WORDS) {
#pragma unroll
      for (int q = 0; q < Q; q += 4) {  // four blocks side by side
        const uint64_t i[4] = {e + uint32_t(q * step), e + uint32_t((q + 1) * step), e + uint32_t((q + 2) * step),
                               e + uint32_t((q + 3) * step)};
        drop_keep_words<4>(run, i, keep + q);
      }
    } else {
      uint64_t i[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) i[q] = e + uint32_t(q * step);
      drop_keep<Q, V, F == NORM_ANYWHERE>(run, i, keep);
    }
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

__device__ __forceinline__ float dot(const uint64_t (&a)[kPairs], const uint64_t (&b)[kPairs]) {
  uint64_t s = mul2(a[0], b[0]), t = mul2(a[1], b[1]);
#pragma unroll
  for (int k = 2; k < kPairs; k += 2) {
    s = fma2(a[k], b[k], s);
    t = fma2(a[k + 1], b[k + 1], t);
  }
  return sum2(add2(s, t));
}
__device__ __forceinline__ float total(const uint64_t (&a)[kPairs]) {
  uint64_t s = a[0], t = a[1];
#pragma unroll
  for (int k = 2; k < kPairs; k += 2) {
    s = add2(s, a[k]);
    t = add2(t, a[k + 1]);
  }
  return sum2(add2(s, t));
}
__device__ __forceinline__ void scale_all(uint64_t (&v)[kPairs], float by) {
  const uint64_t b = both(by);
#pragma unroll
  for (int k = 0; k < kPairs; ++k) v[k] = mul2(v[k], b);
}
// v <- v * f (+ b)
template <bool kAdd>
__device__ __forceinline__ void scale_by(uint64_t (&v)[kPairs], const ParamSlot& f, const ParamSlot& b) {
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

// Stages of the ring: two where 512 threads still fit an SM's shared memory.
constexpr int kParamBytes = kElems * 4, kThreadBytes = 440;
constexpr int ring_stages(int stage_bytes, int param_bytes) {
  return 2 * stage_bytes + param_bytes <= kThreadBytes ? 2 : 1;
}

struct Chosen {
  const void* kernel;
  unsigned shared_bytes;
};
inline int norm_form(const NormArgs& a) {
  if (!a.branch) return FORM_NORM;
  if (a.post && a.pre) return FORM_BOTH;
  return !a.post && a.pre && !a.gated ? FORM_ADD : FORM_ANY;
}
// The kernel of a step: Pick<T, F, form, full, drop>::get().  The folded forms
// are for whole units and 16-bit cut ones (bf16 [33520, 1001] layer norms 114 us, and 131
// with the switches read; gradient 167 and 185); cut f32 units are faster without
// (107 us, and 131 folded; layer norms' gradient 306 and 363).
template <template <int, int, int, bool, bool> class Pick, int T, int F, int kForm>
Chosen choose_switches(const NormArgs& a) {
  const unsigned threads = unsigned(a.shape.threads);
  if constexpr (kForm == FORM_NORM)  // nothing to drop
    return a.layer || a.bias ? Pick<T, F, kForm, true, false>::get(threads) : Pick<T, F, kForm, false, false>::get(threads);
  else if (a.layer || a.bias)
    return a.drop.on ? Pick<T, F, kForm, true, true>::get(threads) : Pick<T, F, kForm, true, false>::get(threads);
  else
    return a.drop.on ? Pick<T, F, kForm, false, true>::get(threads) : Pick<T, F, kForm, false, false>::get(threads);
}
template <template <int, int, int, bool, bool> class Pick, int T, int F>
Chosen choose_form(const NormArgs& a) {
  switch (norm_form(a)) {
    case FORM_BOTH: return choose_switches<Pick, T, F, FORM_BOTH>(a);
    case FORM_ADD: return choose_switches<Pick, T, F, FORM_ADD>(a);
    case FORM_NORM: return choose_switches<Pick, T, F, FORM_NORM>(a);
    default: return choose_switches<Pick, T, F, FORM_ANY>(a);
  }
}
template <template <int, int, int, bool, bool> class Pick, int T>
Chosen choose_type(const NormArgs& a, NormFit fit) {
  if (fit == NORM_UNITS) return choose_form<Pick, T, NORM_UNITS>(a);
  if (fit == NORM_CUT) {
    if constexpr (T == kF32) return choose_switches<Pick, T, NORM_CUT, FORM_ANY>(a);
    else return choose_form<Pick, T, NORM_CUT>(a);
  }
  return choose_switches<Pick, T, T == kF32 ? NORM_WORDS : NORM_ANYWHERE, FORM_ANY>(a);
}
template <template <int, int, int, bool, bool> class Pick>
Chosen choose(const NormArgs& a, NormFit fit) {
  return a.type == kF32   ? choose_type<Pick, kF32>(a, fit)
         : a.type == kF16 ? choose_type<Pick, kF16>(a, fit) : choose_type<Pick, kBF16>(a, fit);
}

}  // namespace

}  // namespace askb
