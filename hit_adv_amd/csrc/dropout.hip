// Dropout from a counter-based generator, with an optional residual: the mask is a function of the element's index and (seed, offset), so
// it is never stored -- the backward pass computes it again.
//
//     y[i] = residual[i] + keep(i) x[i] / (1 - p),   keep(i) = word i mod 4 of Philox4x32-10(counter (i / 4, offset), key seed) >= p 2^32
//
// Philox4x32-10 is the generator of Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3" (SC 2011): ten rounds
// of two 32 x 32 -> 64 bit products.  Bound by bytes and by those products (quarter rate: 20 per four elements) about alike: 16384 x 4096
// bfloat16 74 us with a residual = 5.4 TB/s, 50 us without = 5.4 TB/s (a copy of 2 GiB: 4.9 TB/s).
#include "elements.hpp"
#include "hitadv.h"

namespace hitadv {

struct Philox4 {
  uint32_t w[4];
};
__device__ __forceinline__ Philox4 philox4x32_10(uint64_t block, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// eight elements a thread (two generator blocks); `rng` = (seed, offset) in device memory, read here, so that a captured call follows it
template <int T, bool RES>
__global__ __launch_bounds__(256) void dropout_k(const void *__restrict__ x, const void *__restrict__ residual, void *__restrict__ y, int64_t n,
                                                 const int64_t *__restrict__ rng, uint64_t threshold, float scale) {
  constexpr int V = ELEM_VEC<T>;
  const uint64_t seed = (uint64_t)rng[0], offset = (uint64_t)rng[1];
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 2048) {
    uint32_t w[8];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const Philox4 r = philox4x32_10((uint64_t)(i >> 2) + b, offset, seed);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[4 * b + k] = r.w[k];
    }
#pragma unroll
    for (int j = 0; j < 8; j += V) {
      const int64_t left = n - (i + j);
      if (left <= 0) break;
      const int m = left < V ? (int)left : V;
      float f[V], g[V];
      elem_load_vec<T>(x, i + j, m, f);
      if (RES) elem_load_vec<T>(residual, i + j, m, g);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        f[k] = (uint64_t)w[j + k] >= threshold ? f[k] * scale : 0.f;  // a select: a dropped infinity or NaN is 0
        if (RES) f[k] += g[k];
      }
      elem_store_vec<T>(y, i + j, m, f);
    }
  }
}

template <int T> static int dropout_launch(const void *x, const void *residual, void *y, int64_t n, const int64_t *rng, uint64_t threshold,
                                           float scale, hipStream_t s) {
  const int64_t blocks = (n + 2047) / 2048;
  const unsigned grid = (unsigned)(blocks < 16384 ? blocks : 16384);
  if (residual) dropout_k<T, true><<<grid, 256, 0, s>>>(x, residual, y, n, rng, threshold, scale);
  else dropout_k<T, false><<<grid, 256, 0, s>>>(x, residual, y, n, rng, threshold, scale);
  HITADV_LAUNCH_CHECK();
  return 0;
}

}  // namespace hitadv

using namespace hitadv;

extern "C" int hitadv_dropout(int dtype, const void *x, const void *residual, void *y, int64_t n, const int64_t *rng, uint64_t threshold,
                              float scale, void *stream) {
  if (!x || !y || !rng || n <= 0 || n > (1ll << 40) || threshold > (1ull << 32) || dtype < 0 || dtype > 2) return HITADV_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == ELEM_F32) return dropout_launch<ELEM_F32>(x, residual, y, n, rng, threshold, scale, s);
  if (dtype == ELEM_BF16) return dropout_launch<ELEM_BF16>(x, residual, y, n, rng, threshold, scale, s);
  return dropout_launch<ELEM_F16>(x, residual, y, n, rng, threshold, scale, s);
}
