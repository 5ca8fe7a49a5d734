// Root-mean-square norm of rows, with the residual's addition in front and an 8-bit output with a scale per row behind.
//
//     s = x + residual (rounded to the element type: it is an output)      r = 1 / sqrt(mean(s^2) + eps)      y = s r w
//     8 bits: scale = max |y| / 448 (1 where that is 0; NaN, infinite as the maximum is), q = e4m3(y / scale)
//     backward, g = dy w:  ds = dsum + r (g - s r^2 mean(g s)),   dw = sum over rows of dy s r
//
// All of it is bound by bytes: a row is read once, held in registers as fp32 and written once.  A row belongs to a team of lanes as wide
// as the row needs -- 16 lanes (four rows a wave: the per-head norms of an attention), a wave, a workgroup -- with KI 16-byte accesses in
// flight per lane.  The backward kernel's teams walk over many rows and keep their share of dw in registers; the shares of a workgroup
// meet in LDS, those of the grid in a second small kernel, both in a fixed order (no atomics).  Sums are fp32.
//
// Measured, 16384 rows of 4096 bfloat16: forward with residual 94 us = 5.7 TB/s, 8-bit output with residual 98 - 107 us = 4.4 - 4.8 TB/s, backward
// 115 us = 4.7 TB/s and its second kernel 12 us (a copy of 2 GiB: 4.9 TB/s).  8192 rows of 256 fp32: forward 5.1, backward 6.6 + 4.5 us.
#include "elements.hpp"
#include "hitadv.h"

namespace hitadv {

constexpr float E4M3_MAX = 448.f;

struct RnP {
  const void *x, *residual, *w, *dy, *dsum;
  void *y, *sum, *dx;
  float *rstd, *scale, *dw_part;
  int64_t rows;
  int cols, w32;  // w32: fp32 weights
  float eps, inv_cols;
};

// the larger of two values >= +0, NaN if one is (compared as integers, where NaN lies above infinity)
__device__ __forceinline__ float max_or_nan(float a, float b) {
  const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
  return __uint_as_float(x > y ? x : y);
}

// sum / maximum (of values >= +0, NaN kept) over a team of lanes; `red`: LDS of one float per wave (teams wider than a wave)
template <int TEAM, bool MAX> __device__ __forceinline__ float team_reduce(float v, float *red) {
  constexpr int W = TEAM < 64 ? TEAM : 64;
#pragma unroll
  for (int m = W / 2; m >= 1; m >>= 1) {
    const float o = __shfl_xor(v, m, HITADV_WAVE);
    v = MAX ? max_or_nan(v, o) : v + o;
  }
  if constexpr (TEAM > 64) {
    __syncthreads();  // the last reduction's readers are done
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < TEAM / 64; ++i) v = MAX ? max_or_nan(v, red[i]) : v + red[i];
  }
  return v;
}

// four fp32 -> four e4m3 (to nearest even; the values are at most 448 in magnitude, or NaN)
__device__ __forceinline__ uint32_t e4m3_quad(float a, float b, float c, float d) {
#ifdef HITADV_EMULATED
  const float v[4] = {a, b, c, d};
  uint32_t out = 0;
  for (int i = 0; i < 4; ++i) {
    const uint32_t sign = (__float_as_uint(v[i]) >> 24) & 0x80u;
    const float m = fabsf(v[i]);
    uint32_t code;
    if (m != m) {
      code = 0x7fu;
    } else if (m < 0.015625f) {  // below 2^-6: steps of 2^-9
      code = (uint32_t)rintf(m * 512.f);
    } else {
      const uint32_t u = __float_as_uint(m), r = (u + 0x7ffffu + ((u >> 20) & 1u)) >> 20;
      code = r - ((127u - 7u) << 3);
    }
    out |= (sign | code) << (8 * i);
  }
  return out;
#else
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
#endif
}

// the weight's columns c .. c + V - 1: of the element type, or fp32 (`w32`, the same for every lane)
template <int T> __device__ __forceinline__ void load_weight(const RnP &p, int c, float (&w)[ELEM_VEC<T>]) {
  const int n = p.cols - c;
  if (T == ELEM_F32 || !p.w32) {
    elem_load_vec<T>(p.w, c, n, w);
  } else {
#pragma unroll
    for (int h = 0; h < ELEM_VEC<T>; h += 4) {
      float w4[4];
      elem_load_vec<ELEM_F32>(p.w, c + h, n - h, w4);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[h + j] = w4[j];
    }
  }
}

// T element type; MODE 0: y (and rstd for a backward pass), 1: e4m3 with scales
template <int T, int TEAM, int KI, int MODE, bool RES>
__global__ __launch_bounds__(TEAM > 256 ? TEAM : 256) void rms_norm_k(RnP p) {
  constexpr int V = ELEM_VEC<T>, NT = TEAM > 256 ? TEAM : 256, PER = NT / TEAM;
  __shared__ float red[TEAM > 64 ? TEAM / 64 : 1];
  const int lane = threadIdx.x % TEAM;
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * PER + threadIdx.x / TEAM;
  if (row >= p.rows) return;  // (a team of several waves is the whole workgroup)
  const int64_t at = row * p.cols;
  float f[KI][V];
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < KI; ++k) {
    const int c = (k * TEAM + lane) * V, n = p.cols - c;
    elem_load_vec<T>(p.x, at + c, n, f[k]);
    if (RES) {
      float g[V];
      elem_load_vec<T>(p.residual, at + c, n, g);
#pragma unroll
      for (int j = 0; j < V; ++j) f[k][j] = elem_round<T>(f[k][j] + g[j]);
      elem_store_vec<T>(p.sum, at + c, n, f[k]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) ss += f[k][j] * f[k][j];
  }
  ss = team_reduce<TEAM, false>(ss, red);
  const float r = 1.0f / sqrtf(ss * p.inv_cols + p.eps);
  if (MODE == 0 && p.rstd && lane == 0) p.rstd[row] = r;
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < KI; ++k) {
    const int c = (k * TEAM + lane) * V, n = p.cols - c;
    float w[V];
    load_weight<T>(p, c, w);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      f[k][j] = (f[k][j] * r) * w[j];
      if (MODE == 1) top = max_or_nan(top, fabsf(f[k][j]));
    }
    if (MODE == 0) elem_store_vec<T>(p.y, at + c, n, f[k]);
  }
  if constexpr (MODE == 1) {
    top = team_reduce<TEAM, true>(top, red);
    const float share = top / E4M3_MAX, scale = share == 0.f ? 1.f : share;  // (0 also where max |y| is below 448 2^-150)
    if (lane == 0) p.scale[row] = scale;
#pragma unroll
    for (int k = 0; k < KI; ++k) {
      const int c = (k * TEAM + lane) * V, n = p.cols - c;
      uint32_t q[V / 4];
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float t = f[k][j + u] / scale;
          v[u] = t != t ? t : fmaxf(-E4M3_MAX, fminf(E4M3_MAX, t));
        }
        q[j / 4] = e4m3_quad(v[0], v[1], v[2], v[3]);
      }
      char *o = (char *)p.y + at + c;
      if (n >= V) {
        __builtin_memcpy(o, q, V);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < n) o[j] = (char)(q[j / 4] >> (8 * (j & 3)));
      }
    }
  }
}

// p.x holds s; DW: also this workgroup's share of dw into dw_part[blockIdx.x][cols]
template <int T, int TEAM, int KI, bool RES, bool DW>
__global__ __launch_bounds__(TEAM > 256 ? TEAM : 256) void rms_norm_bwd_k(RnP p) {
  constexpr int V = ELEM_VEC<T>, NT = TEAM > 256 ? TEAM : 256, PER = NT / TEAM, NWAVE = NT / 64;
  constexpr int SPAN = KI * TEAM * V;  // columns a team covers
  __shared__ float red[TEAM > 64 ? TEAM / 64 : 1];
  __shared__ float share[DW && TEAM <= 64 ? NWAVE * SPAN : 1];
  const int lane = threadIdx.x % TEAM;
  float w[KI][V], acc[KI][V];
#pragma unroll
  for (int k = 0; k < KI; ++k) {
    load_weight<T>(p, (k * TEAM + lane) * V, w[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) acc[k][j] = 0.f;
  }
  for (int64_t row0 = (int64_t)blockIdx.x * PER; row0 < p.rows; row0 += (int64_t)gridDim.x * PER) {  // the same trips for every team
    const int64_t row = row0 + threadIdx.x / TEAM, at = row * p.cols;
    const int cols = row < p.rows ? p.cols : 0;
    const float r = cols ? p.rstd[row] : 0.f;
    float s[KI][V], g[KI][V];
    float dot = 0.f;
#pragma unroll
    for (int k = 0; k < KI; ++k) {
      const int c = (k * TEAM + lane) * V, n = cols - c;
      elem_load_vec<T>(p.x, at + c, n, s[k]);
      elem_load_vec<T>(p.dy, at + c, n, g[k]);
    }
#pragma unroll
    for (int k = 0; k < KI; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[k][j] *= r;  // the normalised value
        if (DW) acc[k][j] += g[k][j] * s[k][j];
        g[k][j] *= w[k][j];
        dot += g[k][j] * s[k][j];
      }
    dot = team_reduce<TEAM, false>(dot, red) * p.inv_cols;
#pragma unroll
    for (int k = 0; k < KI; ++k) {
      const int c = (k * TEAM + lane) * V, n = cols - c;
      float o[V];
      if (RES) elem_load_vec<T>(p.dsum, at + c, n, o);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = r * (g[k][j] - s[k][j] * dot);
        o[j] = RES ? o[j] + d : d;
      }
      elem_store_vec<T>(p.dx, at + c, n, o);
    }
  }
  if constexpr (DW) {
    float *out = p.dw_part + (int64_t)blockIdx.x * p.cols;
    if constexpr (TEAM <= 64) {
#pragma unroll
      for (int k = 0; k < KI; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
#pragma unroll
          for (int m = TEAM; m < 64; m <<= 1) acc[k][j] += __shfl_xor(acc[k][j], m, HITADV_WAVE);  // the teams of a wave
          if ((threadIdx.x & 63) < TEAM) share[(threadIdx.x >> 6) * SPAN + (k * TEAM + lane) * V + j] = acc[k][j];
        }
      __syncthreads();
#pragma clang loop vectorize(disable)
      for (int c = threadIdx.x; c < p.cols; c += NT) {
        float t = share[c];
#pragma unroll
        for (int u = 1; u < NWAVE; ++u) t += share[u * SPAN + c];
        out[c] = t;
      }
    } else {
#pragma unroll
      for (int k = 0; k < KI; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = (k * TEAM + lane) * V + j;
          if (c < p.cols) out[c] = acc[k][j];
        }
    }
  }
}

// dw[c] = sum of the workgroups' shares: 8 columns x 32 slices a workgroup, eight shares of a slice in flight
template <int TW>
__global__ __launch_bounds__(256) void rms_norm_dw_k(const float *__restrict__ part, int n, int cols, void *__restrict__ dw) {
  __shared__ float s[32][9];
  const int cl = threadIdx.x & 7, sl = threadIdx.x >> 3, c = blockIdx.x * 8 + cl;
  float t = 0.f;
  for (int i = sl; i < n; i += 256) {
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = c < cols && i + 32 * u < n ? part[(int64_t)(i + 32 * u) * cols + c] : 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) t += x[u];
  }
  s[sl][cl] = t;
  __syncthreads();
  if (sl == 0 && c < cols) {
    for (int i = 1; i < 32; ++i) t += s[i][cl];
    elem_store<TW>(dw, c, t);
  }
}

constexpr int RN_MAX_COLS = 16384;
// workgroups in a grid's first dimension: 2^31 threads at most.  A dimension takes 2^32 - 1; a launch with more came back without an
// error and with wrong rows (2^28 + 5 rows of 8 columns).
constexpr int64_t RN_GRID_X = 1 << 21;

// workgroups of the backward kernel: enough to fill the chip, few enough that the shares of dw stay a small part of the bytes (16384 x 4096
// bfloat16, with the second kernel: 512 at most 126 us, 1024 96, 2048 112)
static int rn_bwd_blocks(int64_t rows, int cols) {
  const int per = cols <= 128 ? 16 : cols <= 1024 ? 4 : 1;
  const int64_t b = (rows + per - 1) / per;
  return (int)(b < 1024 ? b : 1024);
}

template <int T, int TEAM, int KI> static int rn_launch(const RnP &p, int mode, hipStream_t s) {
  constexpr int PER = (TEAM > 256 ? TEAM : 256) / TEAM, NT = TEAM > 256 ? TEAM : 256;
  const int64_t blocks = (p.rows + PER - 1) / PER;
  const dim3 grid((unsigned)(blocks < RN_GRID_X ? blocks : RN_GRID_X), (unsigned)((blocks + RN_GRID_X - 1) / RN_GRID_X));
  if (mode == 0) {
    if (p.residual) rms_norm_k<T, TEAM, KI, 0, true><<<grid, NT, 0, s>>>(p);
    else rms_norm_k<T, TEAM, KI, 0, false><<<grid, NT, 0, s>>>(p);
  } else if (mode == 1) {
    if (p.residual) rms_norm_k<T, TEAM, KI, 1, true><<<grid, NT, 0, s>>>(p);
    else rms_norm_k<T, TEAM, KI, 1, false><<<grid, NT, 0, s>>>(p);
  } else {
    const unsigned g = (unsigned)rn_bwd_blocks(p.rows, p.cols);
    if (p.dw_part) {
      if (p.dsum) rms_norm_bwd_k<T, TEAM, KI, true, true><<<g, NT, 0, s>>>(p);
      else rms_norm_bwd_k<T, TEAM, KI, false, true><<<g, NT, 0, s>>>(p);
    } else {
      if (p.dsum) rms_norm_bwd_k<T, TEAM, KI, true, false><<<g, NT, 0, s>>>(p);
      else rms_norm_bwd_k<T, TEAM, KI, false, false><<<g, NT, 0, s>>>(p);
    }
  }
  HITADV_LAUNCH_CHECK();
  return 0;
}

// the narrowest team whose registers hold the row (forward + backward, bfloat16: 262144 x 64 with 16 lanes 55 us, with 64 175; 65536 x 256 with
// 64 lanes 55 us, with 256 170; 16384 x 1024 with 64 37 us, with 256 50; 16384 x 4096 with 256 150, with 1024 235)
template <int T> static int rn_dispatch(const RnP &p, int mode, hipStream_t s) {
  constexpr int U = T == ELEM_F32 ? 2 : 1;  // fp32: half as many elements in an access, twice the accesses
  if (p.cols <= 128) return rn_launch<T, 16, U>(p, mode, s);
  if (p.cols <= 512) return rn_launch<T, 64, U>(p, mode, s);
  if (p.cols <= 1024) return rn_launch<T, 64, 2 * U>(p, mode, s);
  if (p.cols <= 2048) return rn_launch<T, 256, U>(p, mode, s);
  if (p.cols <= 4096) return rn_launch<T, 256, 2 * U>(p, mode, s);
  if (p.cols <= 8192) return rn_launch<T, 256, 4 * U>(p, mode, s);
  return rn_launch<T, 1024, 2 * U>(p, mode, s);
}
static int rn_run(const RnP &p, int dtype, int mode, hipStream_t s) {
  if (dtype == ELEM_F32) return rn_dispatch<ELEM_F32>(p, mode, s);
  if (dtype == ELEM_BF16) return rn_dispatch<ELEM_BF16>(p, mode, s);
  return rn_dispatch<ELEM_F16>(p, mode, s);
}
static bool rn_ok(int dtype, int wtype, int64_t rows, int cols) {
  return dtype >= 0 && dtype <= 2 && (wtype == dtype || wtype == ELEM_F32) && rows > 0 && rows < (1ll << 31) && cols > 0 && cols <= RN_MAX_COLS;
}

}  // namespace hitadv

using namespace hitadv;

extern "C" int hitadv_rms_norm_fwd(int dtype, int wtype, const void *x, const void *residual, const void *w, int64_t rows, int cols, float eps,
                                   void *y, void *sum, float *rstd, void *stream) {
  if (!x || !w || !y || (residual && !sum) || !rn_ok(dtype, wtype, rows, cols)) return HITADV_E_ARG;
  RnP p = {};
  p.x = x; p.residual = residual; p.w = w; p.y = y; p.sum = sum; p.rstd = rstd; p.rows = rows; p.cols = cols; p.eps = eps;
  p.w32 = wtype == ELEM_F32;
  p.inv_cols = 1.0f / (float)cols;
  return rn_run(p, dtype, 0, (hipStream_t)stream);
}

extern "C" int hitadv_rms_norm_e4m3(int dtype, int wtype, const void *x, const void *residual, const void *w, int64_t rows, int cols, float eps,
                                    void *q, float *scale, void *sum, void *stream) {
  if (!x || !w || !q || !scale || (residual && !sum) || !rn_ok(dtype, wtype, rows, cols)) return HITADV_E_ARG;
  RnP p = {};
  p.x = x; p.residual = residual; p.w = w; p.y = q; p.scale = scale; p.sum = sum; p.rows = rows; p.cols = cols; p.eps = eps;
  p.w32 = wtype == ELEM_F32;
  p.inv_cols = 1.0f / (float)cols;
  return rn_run(p, dtype, 1, (hipStream_t)stream);
}

extern "C" int64_t hitadv_rms_norm_bwd_scratch_floats(int64_t rows, int cols) {
  return rn_ok(0, 0, rows, cols) ? (int64_t)rn_bwd_blocks(rows, cols) * cols : 0;
}

extern "C" int hitadv_rms_norm_bwd(int dtype, int wtype, const void *s, const void *w, const float *rstd, const void *dy, const void *dsum,
                                   int64_t rows, int cols, void *dx, float *scratch, void *dw, void *stream) {
  if (!s || !w || !rstd || !dy || !dx || (dw && !scratch) || !rn_ok(dtype, wtype, rows, cols)) return HITADV_E_ARG;
  RnP p = {};
  p.x = s; p.w = w; p.rstd = const_cast<float *>(rstd); p.dy = dy; p.dsum = dsum; p.dx = dx; p.dw_part = dw ? scratch : nullptr;
  p.rows = rows; p.cols = cols;
  p.w32 = wtype == ELEM_F32;
  p.inv_cols = 1.0f / (float)cols;
  hipStream_t st = (hipStream_t)stream;
  const int rc = rn_run(p, dtype, 2, st);
  if (rc != 0 || !dw) return rc;
  const unsigned g = (unsigned)((cols + 7) / 8);
  const int n = rn_bwd_blocks(rows, cols);
  if (wtype == ELEM_F32) rms_norm_dw_k<ELEM_F32><<<g, 256, 0, st>>>(scratch, n, cols, dw);
  else if (wtype == ELEM_BF16) rms_norm_dw_k<ELEM_BF16><<<g, 256, 0, st>>>(scratch, n, cols, dw);
  else rms_norm_dw_k<ELEM_F16><<<g, 256, 0, st>>>(scratch, n, cols, dw);
  HITADV_LAUNCH_CHECK();
  return 0;
}
