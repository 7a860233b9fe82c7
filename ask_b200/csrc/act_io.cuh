// Activations as f32 values: units of 16 bytes or of single elements of an
// f32, f16 or bf16 tensor, shared by the dropout, block-norm and bias-softmax
// kernels.
#pragma once

#include "ask_numerics.cuh"
#include "kernels.h"
#include "pair_f32.cuh"
#include "vec_io.cuh"

namespace askb {

template <int T>
__host__ __device__ constexpr int act_vec() { return T == kF32 ? 4 : 8; }  // elements in 16 bytes

template <int T>
__device__ __forceinline__ float act_load(const void* p, uint64_t i) {
  if constexpr (T == kF32) return __ldg(static_cast<const float*>(p) + i);
  else {
    const uint16_t h = __ldg(static_cast<const unsigned short*>(p) + i);
    if constexpr (T == kF16) return __half2float(__ushort_as_half(h));
    else return bf16_bits_to_f32(h);
  }
}
template <int T>
__device__ __forceinline__ void act_store(void* p, uint64_t i, float f) {
  if constexpr (T == kF32) static_cast<float*>(p)[i] = f;
  else static_cast<uint16_t*>(p)[i] = uint16_t(narrow_one<T>(f));
}

template <int T>
__device__ __forceinline__ void act_widen(const uint4& r, float* v) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (T == kF32) v[j] = __uint_as_float(w[j]);
    else {
      v[2 * j] = widen_lo<T>(w[j]);
      v[2 * j + 1] = widen_hi<T>(w[j]);
    }
  }
}
template <int T>
__device__ __forceinline__ uint4 act_narrow(const float* v) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (T == kF32) w[j] = __float_as_uint(v[j]);
    else w[j] = narrow_two<T>(v[2 * j], v[2 * j + 1]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The 16 bytes at byte `shift` (0 to 15, a multiple of the element size) of
// two neighbouring 16-byte words.
template <int T>
__device__ __forceinline__ uint4 unit_at(const uint4& a, const uint4& b, uint32_t shift) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int k = 0; k < 6; ++k) w[k] = (shift & 8u) ? w[k + 2] : w[k];
#pragma unroll
  for (int k = 0; k < 5; ++k) w[k] = (shift & 4u) ? w[k + 1] : w[k];
  if constexpr (T != kF32) {
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], (shift & 2u) * 8u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The aligned 16 bytes at `at`, of which only those in [begin, end) may be read;
// the others are 0.
template <int T>
__device__ __forceinline__ uint4 load_part(const char* at, const char* begin, const char* end) {
  constexpr int kBytes = dtype_bytes(T), kPerWord = 4 / kBytes;
  uint32_t w[4] = {};
#pragma unroll
  for (int k = 0; k < 16 / kBytes; ++k) {
    const char* e = at + k * kBytes;
    if (e < begin || e >= end) continue;
    const uint32_t bits = kBytes == 4 ? __ldg(reinterpret_cast<const uint32_t*>(e))
                                      : uint32_t(__ldg(reinterpret_cast<const unsigned short*>(e)));
    w[k / kPerWord] |= bits << (8 * kBytes * (k % kPerWord));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Stores a warp's units (16 bytes a lane, lane after lane) to rows that start
// anywhere: lane k puts together the aligned word that its unit begins in from
// lane k - 1's unit and its own, so only the ends of a run of lanes are stored
// element by element.  `p`: where this lane's unit belongs; `n` of its elements
// exist (0: none); `first`, `last`: the run begins or ends with this lane.  All
// lanes of the warp call it.
template <int T>
__device__ __forceinline__ void store_anywhere(char* p, const uint4& own, int n, bool first, bool last) {
  constexpr int kBytes = dtype_bytes(T);
  const uint32_t shift = uint32_t(reinterpret_cast<uintptr_t>(p)) & 15u;
  uint4 prev;
  prev.x = __shfl_up_sync(0xffffffffu, own.x, 1);
  prev.y = __shfl_up_sync(0xffffffffu, own.y, 1);
  prev.z = __shfl_up_sync(0xffffffffu, own.z, 1);
  prev.w = __shfl_up_sync(0xffffffffu, own.w, 1);
  const int head = int(16u - shift) / kBytes;  // own elements in the word that the unit begins in
  // a unit with elements follows whole units of its run
  const bool whole = shift == 0 ? n == 16 / kBytes : !first && n >= head;
  const bool next_whole = __shfl_down_sync(0xffffffffu, int(whole), 1) && !last;
  if (whole) st_stream_v4(p - shift, shift == 0 ? own : unit_at<T>(prev, own, 16u - shift));
  if (n > 0 && (!whole || (shift != 0 && !next_whole))) {
    const uint32_t w[4] = {own.x, own.y, own.z, own.w};
#pragma unroll
    for (int k = 0; k < 16 / kBytes; ++k) {
      if (k >= n || (k < head ? whole : next_whole)) continue;
      if constexpr (kBytes == 4) reinterpret_cast<uint32_t*>(p)[k] = w[k];
      else reinterpret_cast<uint16_t*>(p)[k] = uint16_t(w[k / 2] >> (16 * (k % 2)));
    }
  }
}

// Elements [first, end) of a 16-byte unit at `to`, by words and the halves at either end.
template <int T>
__device__ __forceinline__ void store_cut(char* to, const uint4& own, int first, int end) {
  const uint32_t w[4] = {own.x, own.y, own.z, own.w};
  if constexpr (T == kF32) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k >= first && k < end) reinterpret_cast<uint32_t*>(to)[k] = w[k];
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (2 * k >= first && 2 * k + 1 < end) reinterpret_cast<uint32_t*>(to)[k] = w[k];
    const auto word = [&](int e) { return e < 4 ? (e < 2 ? w[0] : w[1]) : (e < 6 ? w[2] : w[3]); };
    if ((first & 1) && end > first) reinterpret_cast<uint16_t*>(to)[first] = uint16_t(word(first) >> 16);
    if ((end & 1) && end > first) reinterpret_cast<uint16_t*>(to)[end - 1] = uint16_t(word(end - 1));
  }
}

// What a thread holds of a row before it is widened: 16 bytes.
template <int T, int V>
struct ActRaw {
  static_assert(V == act_vec<T>(), "16 bytes");
  uint4 r;
  __device__ __forceinline__ void load(const void* p, uint64_t i) {
    r = ld_stream_v4(static_cast<const char*>(p) + i * dtype_bytes(T));
  }
  __device__ __forceinline__ void widen(float* v) const { act_widen<T>(r, v); }
};
template <int T, int V>
__device__ __forceinline__ void act_put(void* p, uint64_t i, const float* v) {
  st_stream_v4(static_cast<char*>(p) + i * dtype_bytes(T), act_narrow<T>(v));
}

// Shared memory by its 32-bit address, and asynchronous 16-byte copies into it.
__device__ __forceinline__ uint32_t shared_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
  return r;
}
__device__ __forceinline__ void st_shared(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint32_t ld_shared_word(uint32_t at) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(at) : "memory");
  return r;
}
__device__ __forceinline__ void st_shared_word(uint32_t at, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void st_shared_half(uint32_t at, uint16_t v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(v) : "memory");
}
__device__ __forceinline__ void copy_word_to_shared(uint32_t at, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_to_shared(uint32_t at, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
}

// f32 pairs.
__device__ __forceinline__ uint64_t both(float v) { return pack2(v, v); }
__device__ __forceinline__ float sum2(uint64_t v) {
  float lo, hi;
  unpack2(v, lo, hi);
  return lo + hi;
}
template <int T>
__device__ __forceinline__ void act_widen2(const uint4& r, uint64_t* v) {
  float f[act_vec<T>()];
  act_widen<T>(r, f);
#pragma unroll
  for (int k = 0; k < act_vec<T>() / 2; ++k) v[k] = pack2(f[2 * k], f[2 * k + 1]);
}
template <int T>
__device__ __forceinline__ uint4 act_narrow2(const uint64_t* v) {
  float f[act_vec<T>()];
#pragma unroll
  for (int k = 0; k < act_vec<T>() / 2; ++k) unpack2(v[k], f[2 * k], f[2 * k + 1]);
  return act_narrow<T>(f);
}

// V parameters (weights, gates, a bias table's entries) of run-time type starting
// at column c: read once for many rows and kept in shared memory by the callers.
template <int V>
__device__ __forceinline__ void param_load(const void* p, int type, uint64_t c, float* v) {
  if constexpr (V == 1) {
    v[0] = type == kF32 ? act_load<kF32>(p, c) : type == kF16 ? act_load<kF16>(p, c) : act_load<kBF16>(p, c);
  } else if (type == kF32) {
#pragma unroll
    for (int k = 0; k < V / 4; ++k)
      act_widen<kF32>(__ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(p) + c) + k), v + 4 * k);
  } else {
    // V 16-bit values: one 16-byte load, or 8 bytes for the four of an f32 unit
    uint32_t w[V / 2];
    const char* at = static_cast<const char*>(p) + 2 * c;
    if constexpr (V == 8) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(at));
      w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(at));
      w[0] = q.x; w[1] = q.y;
    }
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      v[2 * j] = type == kF16 ? widen_lo<kF16>(w[j]) : widen_lo<kBF16>(w[j]);
      v[2 * j + 1] = type == kF16 ? widen_hi<kF16>(w[j]) : widen_hi<kBF16>(w[j]);
    }
  }
}

}  // namespace askb
