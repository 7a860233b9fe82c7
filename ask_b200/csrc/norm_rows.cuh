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
// 243, the gradient 831 where it takes 321.)
//
// Bound: HBM, four tensors forward and six for the gradient, up to 4096
// columns without dropout (bf16 [32768, 4096]: 180 us = 6.0 TB/s, gradient 270 us =
// 6.0 TB/s); with dropout the generator's products share the issue slots (243 and
// 321 us).  Rows of 8192 columns have one team an SM, whose loads wait
// while it reduces (156 us for half the elements, gradient 221), and those over a
// cluster wait for its barriers (16384: 236 and 282).  Rows off whole units
// spend three to four times the address arithmetic (NORM_ANYWHERE: bf16 [8191, 4095]
// 136 us; a quarter of [32768, 4096] is 61).
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
// elements.  A unit is 16 bytes (NORM_UNITS), a 4-byte word (NORM_WORDS: single
// f32 columns or pairs of 16-bit ones, lane after lane), or 16 bytes that begin
// anywhere (NORM_ANYWHERE: it spans two aligned words, from which it is shifted
// out, and stores are put together across lanes).  A row is named by the byte
// offset of this thread's first column.
template <int T, int F>
struct Columns {
  static constexpr int E = kElems, P = kPairs, B = dtype_bytes(T);
  static constexpr int kUnitBytes = F == NORM_WORDS ? 4 : 16, V = kUnitBytes / B, Q = E / V;
  static constexpr int kCopies = F == NORM_ANYWHERE ? 2 : 1;     // words of a unit in the ring
  static constexpr int kArrayBytes = Q * kCopies * kUnitBytes;   // of a thread, for one row of one array
  uint32_t first, step;  // column of unit q: first + q * step
  uint32_t cols, pitch;  // pitch: between a thread's words in shared memory
  __device__ __forceinline__ Columns(const Team& t, const NormArgs& a)
      : first((t.rank * uint32_t(Q) * t.threads + t.tid) * uint32_t(V)), step(t.threads * uint32_t(V)), cols(a.cols),
        pitch(blockDim.x * uint32_t(kUnitBytes)) {}
  __device__ __forceinline__ uint32_t at(int q) const { return first + uint32_t(q) * step; }
  __device__ __forceinline__ bool in(int q) const { return at(q) < cols; }
  __device__ __forceinline__ int count(int q) const { return in(q) ? int(min(cols - at(q), uint32_t(V))) : 0; }
  __device__ __forceinline__ uint64_t offset(uint64_t row) const { return (row * cols + first) * uint64_t(B); }
  __device__ __forceinline__ uint64_t unit(uint64_t off, int q) const { return off + uint32_t(q) * step * uint32_t(B); }
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
      if constexpr (F == NORM_UNITS) st_shared(slot + uint32_t(q) * pitch, make_uint4(0u, 0u, 0u, 0u));
      if constexpr (F == NORM_WORDS) st_shared_word(slot + uint32_t(q) * pitch, 0u);
    }
  }
  __device__ __forceinline__ void read(uint32_t slot, const void* p, uint64_t off, uint64_t (&v)[P]) const {
    if constexpr (F == NORM_UNITS) {
#pragma unroll
      for (int q = 0; q < Q; ++q) act_widen2<T>(ld_shared(slot + uint32_t(q) * pitch), v + q * V / 2);
    } else if constexpr (F == NORM_WORDS) {
      if constexpr (T == kF32) {
#pragma unroll
        for (int k = 0; k < P; ++k)
          v[k] = pack2(__uint_as_float(ld_shared_word(slot + uint32_t(2 * k) * pitch)),
                       __uint_as_float(ld_shared_word(slot + uint32_t(2 * k + 1) * pitch)));
      } else {
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const uint32_t w = ld_shared_word(slot + uint32_t(k) * pitch);
          v[k] = pack2(widen_lo<T>(w), widen_hi<T>(w));
        }
      }
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
    } else if constexpr (F == NORM_WORDS) {
#pragma unroll
      for (int k = 0; k < P; ++k) {
        float lo, hi;
        unpack2(v[k], lo, hi);
        if constexpr (T == kF32) {
          if (on && in(2 * k)) st_stream_u32(to + unit(off, 2 * k), __float_as_uint(lo));
          if (on && in(2 * k + 1)) st_stream_u32(to + unit(off, 2 * k + 1), __float_as_uint(hi));
        } else {
          if (on && in(k)) st_stream_u32(to + unit(off, k), narrow_two<T>(lo, hi));
        }
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
      const int n = count(q);
#pragma unroll
      for (int j = 0; j < V; ++j) f[q * V + j] = j < n ? fill : 0.0f;
      if (!p) continue;
      if (F == NORM_UNITS) {
        if constexpr (F == NORM_UNITS) {
          if (n) param_load<V>(p, type, offset + at(q), f + q * V);
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < n) param_load<1>(p, type, offset + at(q) + j, f + q * V + j);
      }
    }
  }
  // v - mean where there is a column; the rest stays 0
  __device__ __forceinline__ void center(float mean, uint64_t (&v)[P]) const {
    if constexpr (F == NORM_UNITS) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const uint64_t m = both(in(q) ? -mean : 0.0f);
#pragma unroll
        for (int k = 0; k < V / 2; ++k) v[q * V / 2 + k] = add2(v[q * V / 2 + k], m);
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
        const uint64_t i[4] = {e + uint32_t(q) * step, e + uint32_t(q + 1) * step, e + uint32_t(q + 2) * step,
                               e + uint32_t(q + 3) * step};
        drop_keep_words<4, V>(run, i, keep + q * V);
      }
    } else {
      uint64_t i[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) i[q] = e + uint32_t(q) * step;
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

// Stages of the ring: up to three while 512 threads an SM (what the registers
// allow) still fit its shared memory.
constexpr int kParamBytes = kElems * 4, kThreadBytes = 440;
constexpr int ring_stages(int stage_bytes, int param_bytes) {
  return 3 * stage_bytes + param_bytes <= kThreadBytes ? 3 : 2 * stage_bytes + param_bytes <= kThreadBytes ? 2 : 1;
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
// are for whole units; other rows read the switches.
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
template <template <int, int, int, bool, bool> class Pick, int T>
Chosen choose_type(const NormArgs& a, NormFit fit) {
  if (fit == NORM_WORDS) return choose_switches<Pick, T, NORM_WORDS, FORM_ANY>(a);
  if constexpr (T != kF32) {
    if (fit == NORM_ANYWHERE) return choose_switches<Pick, T, NORM_ANYWHERE, FORM_ANY>(a);
  }
  switch (norm_form(a)) {
    case FORM_BOTH: return choose_switches<Pick, T, NORM_UNITS, FORM_BOTH>(a);
    case FORM_ADD: return choose_switches<Pick, T, NORM_UNITS, FORM_ADD>(a);
    case FORM_NORM: return choose_switches<Pick, T, NORM_UNITS, FORM_NORM>(a);
    default: return choose_switches<Pick, T, NORM_UNITS, FORM_ANY>(a);
  }
}
template <template <int, int, int, bool, bool> class Pick>
Chosen choose(const NormArgs& a, NormFit fit) {
  return a.type == kF32   ? choose_type<Pick, kF32>(a, fit)
         : a.type == kF16 ? choose_type<Pick, kF16>(a, fit) : choose_type<Pick, kBF16>(a, fit);
}

}  // namespace

}  // namespace askb
