// Element types of the operators that take fp32, bf16 and fp16 tensors alike (csrc/diff_attention.hip, rms_norm.hip, dropout.hip).
#pragma once
#include "common.hpp"

// exactly n waves per SIMD: the scheduler uses the registers that leaves instead of saving some for more waves
#ifdef HITADV_EMULATED
#define HITADV_WAVES_PER_SIMD(n)
#else
#define HITADV_WAVES_PER_SIMD(n) __attribute__((amdgpu_waves_per_eu(n, n)))
#endif

namespace hitadv {

// the lane, counted anew: what an epilogue computes from it is not kept in registers throughout the loop in front
__device__ __forceinline__ int lane_counted() {
#ifdef HITADV_EMULATED
  return threadIdx.x & 63;
#else
  return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
#endif
}

// two floats -> two bf16, to nearest even
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
#ifdef HITADV_EMULATED
  const float v[2] = {a, b};
  uint32_t w[2];
  for (int i = 0; i < 2; ++i) {
    const uint32_t u = __float_as_uint(v[i]);
    w[i] = v[i] != v[i] ? 0x7fc0u : (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
  }
  return w[0] | (w[1] << 16);
#else
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  bf16x2 r;
  r.x = (__bf16)a;
  r.y = (__bf16)b;
  return __builtin_bit_cast(uint32_t, r);
#endif
}
__device__ __forceinline__ uint32_t f16_pair(float a, float b) {
  return __builtin_bit_cast(uint16_t, (_Float16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16);
}
__device__ __forceinline__ float f16_bits_to_float(uint32_t h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)h); }

// dtype codes of the C ABI (include/hitadv.h HITADV_DTYPE_*)
constexpr int ELEM_F32 = 0, ELEM_BF16 = 1, ELEM_F16 = 2;
template <int T> constexpr int ELEM_BYTES = T == ELEM_F32 ? 4 : 2;
template <int T> constexpr int ELEM_VEC = 16 / ELEM_BYTES<T>;  // elements of a 16-byte access

template <int T> __device__ __forceinline__ float elem_load(const void *p, int64_t i) {
  if constexpr (T == ELEM_F32) return ((const float *)p)[i];
  else if constexpr (T == ELEM_F16) return (float)((const _Float16 *)p)[i];
  else return __uint_as_float((uint32_t)((const uint16_t *)p)[i] << 16);
}
template <int T> __device__ __forceinline__ void elem_store(void *p, int64_t i, float v) {
  if constexpr (T == ELEM_F32) ((float *)p)[i] = v;
  else if constexpr (T == ELEM_F16) ((_Float16 *)p)[i] = (_Float16)v;
  else ((uint16_t *)p)[i] = (uint16_t)bf16_pair(v, 0.f);
}
// what the type keeps of v
template <int T> __device__ __forceinline__ float elem_round(float v) {
  if constexpr (T == ELEM_F32) return v;
  else if constexpr (T == ELEM_F16) return (float)(_Float16)v;
  else return __uint_as_float(bf16_pair(v, 0.f) << 16);
}

// elements i .. i + V - 1, of which `n` exist (n >= V: one 16-byte access at whatever alignment the element type has, which gfx950's
// global accesses take; n < V: one by one; the rest is 0)
template <int T> __device__ __forceinline__ void elem_load_vec(const void *p, int64_t i, int n, float (&f)[ELEM_VEC<T>]) {
  constexpr int V = ELEM_VEC<T>;
  if (n >= V) {
    uint32_t w[4];
    __builtin_memcpy(w, (const char *)p + i * ELEM_BYTES<T>, 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (T == ELEM_F32) {
        f[k] = __uint_as_float(w[k]);
      } else if constexpr (T == ELEM_F16) {
        f[2 * k] = f16_bits_to_float(w[k] & 0xffffu);
        f[2 * k + 1] = f16_bits_to_float(w[k] >> 16);
      } else {
        f[2 * k] = __uint_as_float(w[k] << 16);
        f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = k < n ? elem_load<T>(p, i + k) : 0.f;
  }
}
template <int T> __device__ __forceinline__ void elem_store_vec(void *p, int64_t i, int n, const float (&f)[ELEM_VEC<T>]) {
  constexpr int V = ELEM_VEC<T>;
  if (n >= V) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (T == ELEM_F32) w[k] = __float_as_uint(f[k]);
      else if constexpr (T == ELEM_F16) w[k] = f16_pair(f[2 * k], f[2 * k + 1]);
      else w[k] = bf16_pair(f[2 * k], f[2 * k + 1]);
    }
    __builtin_memcpy((char *)p + i * ELEM_BYTES<T>, w, 16);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < n) elem_store<T>(p, i + k, f[k]);
  }
}

}  // namespace hitadv
