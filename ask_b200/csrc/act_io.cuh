// Activations as f32 values: units of 16 bytes or of single elements of an
// f32, f16 or bf16 tensor, shared by the dropout, block-norm and bias-softmax
// kernels.
#pragma once

#include "ask_numerics.cuh"
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

// What a thread holds of a row before it is widened: V elements, 16 bytes or one.
template <int T, int V>
struct ActRaw {
  uint4 r;
  __device__ __forceinline__ void load(const void* p, uint64_t i) {
    r = ld_stream_v4(static_cast<const char*>(p) + i * dtype_bytes(T));
  }
  __device__ __forceinline__ void zero() { r = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void widen(float* v) const { act_widen<T>(r, v); }
};
template <int T>
struct ActRaw<T, 1> {
  float f;
  __device__ __forceinline__ void load(const void* p, uint64_t i) { f = act_load<T>(p, i); }
  __device__ __forceinline__ void zero() { f = 0.0f; }
  __device__ __forceinline__ void widen(float* v) const { v[0] = f; }
};
template <int T, int V>
__device__ __forceinline__ void act_put(void* p, uint64_t i, const float* v) {
  if constexpr (V == 1) act_store<T>(p, i, v[0]);
  else st_stream_v4(static_cast<char*>(p) + i * dtype_bytes(T), act_narrow<T>(v));
}

// V parameters (weights, gates) of run-time type starting at column c: read
// again for every row, so they stay in L1 or L2.
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
