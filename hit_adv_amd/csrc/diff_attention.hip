// Differential attention: the difference of two softmax maps over shared values, with a learned weight per head.
//
//     P_m[i,j] = softmax over the visible j of  scale q[i,m] . k[j,m]   (m = 1, 2)
//     out[i]   = sum_j (P_1[i,j] - lam P_2[i,j]) v[j]
//
// q [B,Nq,H,2,D], k [B,Nk,Hkv,2,D], v [B,Nk,Hkv,2D], out [B,Nq,H,2D]; H / Hkv = G query heads share one key / value head.  A key is
// visible below its cloud's length and, if causal, at j <= i + Nk - Nq.  A row that sees nothing gives 0 and has no gradient.
//
// Arithmetic.  Everything runs on the 16-bit matrix cores with fp32 accumulators.  The products of two inputs (the scores, dO V^T) take
// bf16 and fp16 inputs as they are: every product is exact.  fp32 inputs enter as three bf16 pieces whose sum is the value (each the
// truncation of what is left) and six piece products.  The products with a map on one side are bf16 pieces, in the backward pass also where
// the inputs are fp16 (two pieces, exact): a bf16 piece has fp32's exponent, so no gradient leaves the range.  (P V of fp16 inputs: see the
// forward kernel.)  The map itself is two pieces (three in fp32) also where the inputs are bf16:
// rounding P_1 and P_2 to one bf16 each before their difference is taken puts back the noise that the difference is there to cancel,
// and one-piece dS and A = P_1 - lam P_2 put the gradients at 1.5x the error of their own last rounding (two: 1.0x).  Maxima, sums
// and accumulators are fp32.  A row is empty if its limit says so, not if its sum is 0: where every visible score is -inf (an infinite query or
// key, a product beyond fp32) softmax is 0 / 0 and the row NaN.  One score of -inf is a probability of 0 in 16-bit types; the pieces of an
// infinity in fp32 are NaN.  Any other visible value that is not finite makes the row not finite.
//
// Layout.  All products are computed transposed so that no map ever leaves the registers: S^T = K Q^T has the query in the lane (column
// lane & 31) and 16 keys in its registers, which is -- with the keys of a 16-chunk in the order 4h..4h+3, 8+4h..8+4h+3 for lane half h --
// exactly the B operand of O^T = V^T P^T.  The transposed tiles (V^T here, K^T, Q^T and dO^T in the backward pass) are written to LDS in
// that key order, so that an A operand is one 16-byte read.  Rows of one key / value head's G query heads are packed (row r = query r / G,
// head r % G): a tile of 32 rows then shares every key and value it stages, for a single new token too.
#include "elements.hpp"
#include "hitadv.h"

#include <type_traits>

namespace hitadv {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int DA_T = 32;          // rows (keys) of a tile = the matrix instruction's width
constexpr float DA_LOG2E = 1.4426950408889634f;
constexpr float DA_SLACK = 8.0f;  // the running maximum is raised only when it would rise by 2^8: a probability stays below 2^8
#define DA_INF __builtin_inff()

struct DaP {
  const void *q, *k, *v, *dout;
  const float *lam;
  const int *lengths;
  void *out;             // forward: out; backward: unused
  void *dq, *dk, *dv;
  float *stats;          // [4][B*H*Nq]: running maximum and log2 of the sum, map 1 then map 2
  float *r;              // [2][B*H*Nq]: sum_j P_m dP
  float *part_o, *part_ml;
  int64_t q_b, q_n, q_h, q_m, k_b, k_n, k_h, k_m, v_b, v_n, v_h;
  int B, Nq, Nk, H, Hkv, D, G, lam_n, causal, rows, chunk, splits;
  uint32_t g_magic;      // ceil(2^32 / G), G > 1
  float scale, scale2;   // scale, |scale| log2(e) (1 if scale is 0)
  uint32_t s_and, s_xor; // what makes one operand of the scores carry the scale's sign (or its zero): its elements' words and, xor these
};

// The row (key) tile of a workgroup, causal: the heaviest first -- the last rows, or (`rising` false: tiles of keys) the first keys.
__device__ __forceinline__ int da_tile(bool causal, bool rising) {
  return causal && rising ? (int)(gridDim.y - 1 - blockIdx.y) : (int)blockIdx.y;
}
__device__ __forceinline__ int da_div_g(const DaP &p, int r) { return p.G == 1 ? r : (int)(((uint64_t)(uint32_t)r * p.g_magic) >> 32); }
__device__ __forceinline__ float da_lam(const DaP &p, int h) { return p.lam[p.lam_n == 1 ? 0 : h]; }
__device__ __forceinline__ int da_len(const DaP &p, int b) {
  return p.lengths ? max(0, min(p.lengths[b], p.Nk)) : p.Nk;
}
// the first key that query i does not see
__device__ __forceinline__ int da_limit(const DaP &p, int i, int len) {
  return p.causal ? max(0, min(len, i + p.Nk - p.Nq + 1)) : len;
}

// ---------------------------------------------------------------------------------------------------------------- elements and pieces

template <int NP> struct Raw8 { uint4 a; };
template <> struct Raw8<3> { float4 a, b; };
template <int NP> struct Raw4 { uint2 a; };
template <> struct Raw4<3> { float4 a; };

template <class R> __device__ __forceinline__ R da_zero() { return R{}; }
template <int NP> __device__ __forceinline__ Raw8<NP> da_load8(const char *at) {
  Raw8<NP> r;
  if constexpr (NP == 3) {
    r.a = ((const float4 *)at)[0];
    r.b = ((const float4 *)at)[1];
  } else {
    r.a = *(const uint4 *)at;
  }
  return r;
}
template <int NP> __device__ __forceinline__ Raw4<NP> da_load4(const char *at) {
  Raw4<NP> r;
  if constexpr (NP == 3) r.a = *(const float4 *)at;
  else r.a = *(const uint2 *)at;
  return r;
}
// eight elements, or zeros
template <int NP> __device__ __forceinline__ Raw8<NP> da_load8_if(const void *base, int64_t at, bool ok) {
  return ok ? da_load8<NP>((const char *)base + at * (NP == 3 ? 4 : 2)) : da_zero<Raw8<NP>>();
}

// the pieces of a value, each a bf16 in the upper half of a word
template <int NP> __device__ __forceinline__ void da_pieces(float f, uint32_t (&p)[NP]) {
  p[0] = __float_as_uint(f) & 0xffff0000u;
  if constexpr (NP >= 2) {
    const float r1 = f - __uint_as_float(p[0]);
    p[1] = __float_as_uint(r1) & 0xffff0000u;
    if constexpr (NP == 3) p[2] = __float_as_uint(r1 - __uint_as_float(p[1]));
  }
}

// eight values of a row -> the operand(s) of a product of two inputs: 16-bit elements as they are, fp32 as three pieces
template <int NP> constexpr int DA_NR = NP == 3 ? 3 : 1;
template <int NP> __device__ __forceinline__ void da_pieces8(const Raw8<NP> &r, uint4 (&out)[DA_NR<NP>]) {
  if constexpr (NP != 3) {
    out[0] = r.a;
  } else {
    const float f[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    uint32_t p[8][3];
#pragma unroll
    for (int i = 0; i < 8; ++i) da_pieces<3>(f[i], p[i]);
#pragma unroll
    for (int k = 0; k < 3; ++k)
      out[k] = make_uint4(pack_hi(p[0][k], p[1][k]), pack_hi(p[2][k], p[3][k]), pack_hi(p[4][k], p[5][k]), pack_hi(p[6][k], p[7][k]));
  }
}
// a score's operand with the scale's sign (pieces are 16-bit values of either format: two to a word)
template <int N> __device__ __forceinline__ void da_sign(uint4 (&w)[N], const DaP &p) {
#pragma unroll
  for (int k = 0; k < N; ++k)
    w[k] = make_uint4((w[k].x & p.s_and) ^ p.s_xor, (w[k].y & p.s_and) ^ p.s_xor, (w[k].z & p.s_and) ^ p.s_xor, (w[k].w & p.s_and) ^ p.s_xor);
}
// dP's operand, its sign turned in every other tile of keys
template <int N> __device__ __forceinline__ void da_turn(uint4 (&w)[N], bool neg) {
  const uint32_t x = neg ? 0x80008000u : 0u;
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = make_uint4(w[k].x ^ x, w[k].y ^ x, w[k].z ^ x, w[k].w ^ x);
}
// the pieces of four rows of four values, [row][column][piece]
template <int NP> __device__ __forceinline__ void da_pieces4x4(const Raw4<NP> (&r)[4], uint32_t (&p)[4][4][NP]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (NP == 3) {
      da_pieces<NP>(r[i].a.x, p[i][0]);
      da_pieces<NP>(r[i].a.y, p[i][1]);
      da_pieces<NP>(r[i].a.z, p[i][2]);
      da_pieces<NP>(r[i].a.w, p[i][3]);
    } else if constexpr (NP == 2) {
      da_pieces<NP>(f16_bits_to_float(r[i].a.x & 0xffffu), p[i][0]);
      da_pieces<NP>(f16_bits_to_float(r[i].a.x >> 16), p[i][1]);
      da_pieces<NP>(f16_bits_to_float(r[i].a.y & 0xffffu), p[i][2]);
      da_pieces<NP>(f16_bits_to_float(r[i].a.y >> 16), p[i][3]);
    } else {
      p[i][0][0] = r[i].a.x << 16;
      p[i][1][0] = r[i].a.x & 0xffff0000u;
      p[i][2][0] = r[i].a.y << 16;
      p[i][3][0] = r[i].a.y & 0xffff0000u;
    }
  }
}

// eight probabilities -> NPP pieces, each the B operand of a matrix instruction
template <int NPP> __device__ __forceinline__ void da_operand(const float *x, bf16x8 (&out)[NPP]) {
  if constexpr (NPP == 3) {
    uint32_t p[8][3];
#pragma unroll
    for (int i = 0; i < 8; ++i) da_pieces<3>(x[i], p[i]);
#pragma unroll
    for (int k = 0; k < 3; ++k)
      out[k] = as_bf16x8(make_uint4(pack_hi(p[0][k], p[1][k]), pack_hi(p[2][k], p[3][k]), pack_hi(p[4][k], p[5][k]), pack_hi(p[6][k], p[7][k])));
  } else {
    uint32_t w[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = bf16_pair(x[2 * i], x[2 * i + 1]);
      if constexpr (NPP == 2)
        l[i] = bf16_pair(x[2 * i] - __uint_as_float(w[i] << 16), x[2 * i + 1] - __uint_as_float(w[i] & 0xffff0000u));
    }
    out[0] = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
    if constexpr (NPP == 2) out[1] = as_bf16x8(make_uint4(l[0], l[1], l[2], l[3]));
  }
}

// the same as two fp16 pieces (22 bits)
__device__ __forceinline__ void da_operand_f16(const float *x, bf16x8 (&out)[2]) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  uint32_t w[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f16x2 h, r;
    h.x = (_Float16)x[2 * i];
    h.y = (_Float16)x[2 * i + 1];
    r.x = (_Float16)(x[2 * i] - (float)h.x);
    r.y = (_Float16)(x[2 * i + 1] - (float)h.y);
    w[i] = __builtin_bit_cast(uint32_t, h);
    l[i] = __builtin_bit_cast(uint32_t, r);
  }
  out[0] = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
  out[1] = as_bf16x8(make_uint4(l[0], l[1], l[2], l[3]));
}

// c += a b over the pieces that count: weights 2^-8(i + j) with i + j < max(NA, NB)
template <int NA, int NB> __device__ __forceinline__ f32x16 da_mfma(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x16 c) {
  constexpr int CUT = NA > NB ? NA : NB;
#pragma unroll
  for (int s = CUT - 1; s >= 0; --s)  // the small products first
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (i + j == s) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], c, 0, 0, 0);
  return c;
}

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
// c += a b for two inputs' operands.  QUERY_A: the query's operand is a (else b); the piece products are taken in the same order either
// way, so that every kernel computes a score and a dP to the same bits (a row with one key: dP - r = 0).
template <int NP, bool QUERY_A> __device__ __forceinline__ f32x16 da_mfma_in(const bf16x8 (&a)[DA_NR<NP>], const bf16x8 (&b)[DA_NR<NP>], f32x16 c) {
  if constexpr (NP == 2)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a[0]), __builtin_bit_cast(f16x8, b[0]), c, 0, 0, 0);
#pragma unroll
  for (int s = DA_NR<NP> - 1; s >= 0; --s)  // the small products first
#pragma unroll
    for (int i = 0; i <= s; ++i) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[QUERY_A ? s - i : i], b[QUERY_A ? i : s - i], c, 0, 0, 0);
  return c;
}
// The same with fp32's small products in a sum of their own: the instruction truncates what it aligns to a larger accumulator, always
// downwards, and r = sum P dP adds such an offset of dP up over every row (dlam of 32 x 256 rows: 5.6e-6 off with one sum)
template <int NP, bool QUERY_A>
__device__ __forceinline__ void da_mfma_in2(const bf16x8 (&a)[DA_NR<NP>], const bf16x8 (&b)[DA_NR<NP>], f32x16 &c, f32x16 &small) {
  if constexpr (NP == 3) {
#pragma unroll
    for (int s = 2; s >= 1; --s)
#pragma unroll
      for (int i = 0; i <= s; ++i)
        small = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[QUERY_A ? s - i : i], b[QUERY_A ? i : s - i], small, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], c, 0, 0, 0);
  } else {
    c = da_mfma_in<NP, QUERY_A>(a, b, c);
  }
}

// ---------------------------------------------------------------------------------------------------------------- LDS tiles
// A tile of 32 rows: [DA_NR][32][2 DP]; its transpose: [NP][2 DP][32] with the rows in operand order.  No padding (two workgroups of the
// backward kernels share a CU's LDS); instead the 16-byte pieces are permuted so that the lanes of an access lie on different banks:
// a row's pieces by xor with the row; a transposed row goes to place `place(c)` (the two low pairs of bits of its column swapped: lanes that
// write have columns four apart, lanes that read neighbouring ones) and its four pieces by xor with the column's low bits.
template <int NP, int DP> struct DaTile {
  static constexpr int W = 2 * DP, NR = DA_NR<NP>, M = W / 8 < 16 ? W / 8 - 1 : 15;
  static constexpr int ROWS = NR * DA_T * W, COLS = NP * W * DA_T;  // 16-bit elements
  static __device__ __forceinline__ int row_at(int row, int col) { return row * W + (((col >> 3) ^ (row & M)) << 3) + (col & 7); }
  static __device__ __forceinline__ int col_at(int c, int row) {
    return ((c & ~15) | ((c & 3) << 2) | ((c >> 2) & 3)) * DA_T + (((row >> 3) ^ (c & 3)) << 3) + (row & 7);
  }
  static __device__ __forceinline__ void frag_row(const uint16_t *t, int row, int col, bf16x8 (&f)[NR]) {
#pragma unroll
    for (int k = 0; k < NR; ++k) f[k] = as_bf16x8(*(const uint4 *)(t + k * DA_T * W + row_at(row, col)));
  }
  static __device__ __forceinline__ void frag_col(const uint16_t *t, int col, int chunk, int half, bf16x8 (&f)[NP]) {
#pragma unroll
    for (int k = 0; k < NP; ++k) f[k] = as_bf16x8(*(const uint4 *)(t + k * W * DA_T + col_at(col, 16 * chunk + 8 * half)));
  }
  static __device__ __forceinline__ void put_row(uint16_t *t, int row, int col, const Raw8<NP> &r) {
    uint4 p[NR];
    da_pieces8<NP>(r, p);
#pragma unroll
    for (int k = 0; k < NR; ++k) *(uint4 *)(t + k * DA_T * W + row_at(row, col)) = p[k];
  }
  // rows 4 rg .. 4 rg + 3, columns col .. col + 3, as rows and / or transposed: there row 16 c + 8 y + 4 x + j sits at 16 c + 8 x + 4 y + j
  template <bool AS_ROWS, bool AS_COLS> static __device__ __forceinline__ void put_block(uint16_t *rows, uint16_t *cols, int rg, int col, const Raw4<NP> (&r)[4]) {
    if constexpr (AS_ROWS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint16_t *to = rows + row_at(4 * rg + i, col);
        if constexpr (NP == 3) {
          uint32_t p[4][3];
          da_pieces<3>(r[i].a.x, p[0]);
          da_pieces<3>(r[i].a.y, p[1]);
          da_pieces<3>(r[i].a.z, p[2]);
          da_pieces<3>(r[i].a.w, p[3]);
#pragma unroll
          for (int k = 0; k < 3; ++k) *(uint2 *)(to + k * DA_T * W) = make_uint2(pack_hi(p[0][k], p[1][k]), pack_hi(p[2][k], p[3][k]));
        } else {
          *(uint2 *)to = r[i].a;
        }
      }
    }
    if constexpr (AS_COLS) {
      uint32_t p[4][4][NP];
      da_pieces4x4<NP>(r, p);
      const int at = 16 * (rg >> 2) + 8 * (rg & 1) + 4 * ((rg >> 1) & 1);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int k = 0; k < NP; ++k)
          *(uint2 *)(cols + k * W * DA_T + col_at(col + c, at)) = make_uint2(pack_hi(p[0][c][k], p[1][c][k]), pack_hi(p[2][c][k], p[3][c][k]));
    }
  }
};

template <int NP> constexpr int DA_ES = NP == 3 ? 4 : 2;  // bytes of an element
// byte offset of a column of the padded [2][DP] (maps) or [2 DP] columns; false: padding
template <int NP, int DP> __device__ __forceinline__ bool da_bind(int col, int64_t m, int D, bool maps, uint32_t &off) {
  const int map = maps && col >= DP ? 1 : 0, d = col - map * DP;
  off = (uint32_t)(map * (int)m + d) * DA_ES<NP>;
  return d < (maps ? D : 2 * D);
}
// Rows that do not exist are fetched as the last one that does and zeroed when they are stored: a load behind a branch, its register zeroed
// first, has the compiler wait for every load in flight (with that the backward kernels took 1.5x as long).
template <int NP, int DP, int NT> struct DaFetchRows {  // 16-byte (32-byte) pieces of 32 rows of k, v
  static constexpr int CH = 2 * DP / 8, STEP = NT / CH, C = STEP >= DA_T ? 1 : DA_T / STEP, ES = DA_ES<NP>;
  Raw8<NP> x[C];
  int row, col, left;
  uint32_t off;  // of the column
  bool there;
  __device__ __forceinline__ void bind(int64_t m, int D, bool maps, int tid) {
    row = tid / CH;
    col = 8 * (tid % CH);
    there = da_bind<NP, DP>(col, m, D, maps, off) && row < DA_T;
  }
  // rows t .. t + 31 of the rows at `base` (elements, wave-uniform); `end` > 0: the first row that does not exist
  __device__ __forceinline__ void load(const void *src, int64_t base, int64_t n, int t, int end) {
    left = end - t;
    if (!there) return;
    const int first = min(t, end - 1);
    const char *at = (const char *)src + (base + first * n) * ES;
#pragma unroll
    for (int c = 0; c < C; ++c) x[c] = da_load8<NP>(at + (uint32_t)(min(row + c * STEP, end - 1 - first) * (int)n) * ES + off);
  }
  __device__ __forceinline__ void put(uint16_t *rows) {
    if (!there) return;
    if (left < DA_T) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (row + c * STEP >= left) x[c] = da_zero<Raw8<NP>>();
    }
#pragma unroll
    for (int c = 0; c < C; ++c) DaTile<NP, DP>::put_row(rows, row + c * STEP, col, x[c]);
  }
  __device__ __forceinline__ void zero_padding(uint16_t *rows) const {
    if (there || row >= DA_T) return;
#pragma unroll
    for (int c = 0; c < C; ++c) DaTile<NP, DP>::put_row(rows, row + c * STEP, col, da_zero<Raw8<NP>>());
  }
};
// 4 x 4 blocks, for a transposed tile, or both.  Lanes: four row groups, then sixteen column groups: sixteen lanes write on different
// banks, and a wave still fetches 128 (256) bytes of every row (eight row groups: 64, and the backward kernels 10 % slower).
template <int NP, int DP, int NT> struct DaFetchBlocks {
  static constexpr int CH = 2 * DP / 4, STEP = NT / 8, C = STEP >= CH ? 1 : CH / STEP, ES = DA_ES<NP>;
  Raw4<NP> x[C][4];
  int row, col, left;
  uint32_t off[C];
  bool there[C];
  __device__ __forceinline__ void bind(int64_t m, int D, bool maps, int tid) {
    row = 4 * ((tid & 3) | ((tid >> 4) & 4));
    col = 4 * (((tid >> 2) & 15) | ((tid >> 7) << 4));
#pragma unroll
    for (int c = 0; c < C; ++c) there[c] = da_bind<NP, DP>(col + 4 * c * STEP, m, D, maps, off[c]) && col < 2 * DP;
  }
  __device__ __forceinline__ void load(const void *src, int64_t base, int64_t n, int t, int end) {
    left = end - t;
    const int first = min(t, end - 1);
    const char *at = (const char *)src + (base + first * n) * ES;
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (uint32_t)(min(row + i, end - 1 - first) * (int)n) * ES;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!there[c]) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[c][i] = da_load4<NP>(at + (o[i] + off[c]));
    }
  }
  // packed query rows: row r is query r / G, head r % G.  Two ways to a row's address meet before the loads, so none is behind a branch:
  // a column that does not exist is fetched as the row's first and dropped.
  __device__ __forceinline__ void load_packed(const void *src, int64_t base, int64_t n, int64_t h, const DaP &p, int t) {
    left = p.rows - t;
    const char *at = (const char *)src + base * ES;
    int64_t o[4];
    if (p.G == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = min(t + row + i, p.rows - 1) * n;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = min(t + row + i, p.rows - 1), q = da_div_g(p, r);
        o[i] = q * n + (r - q * p.G) * h;
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const uint32_t oc = there[c] ? off[c] : 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[c][i] = da_load4<NP>(at + (o[i] * ES + oc));
    }
  }
  // `none` > 0: so many rows of the tile see no key, and what they hold is dropped
  template <bool ROWS, bool COLS> __device__ __forceinline__ void put(uint16_t *rows, uint16_t *cols, int none = 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!there[c]) continue;
      if (none > 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (row + i < none) x[c][i] = da_zero<Raw4<NP>>();
      }
      if (left < DA_T) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (row + i >= left) x[c][i] = da_zero<Raw4<NP>>();
      }
      DaTile<NP, DP>::template put_block<ROWS, COLS>(rows, cols, row / 4, col + 4 * c * STEP, x[c]);
    }
  }
  template <bool ROWS, bool COLS> __device__ __forceinline__ void zero_padding(uint16_t *rows, uint16_t *cols) const {
    const Raw4<NP> z[4] = {da_zero<Raw4<NP>>(), da_zero<Raw4<NP>>(), da_zero<Raw4<NP>>(), da_zero<Raw4<NP>>()};
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (!there[c] && col < 2 * DP) DaTile<NP, DP>::template put_block<ROWS, COLS>(rows, cols, row / 4, col + 4 * c * STEP, z);
  }
};

// four consecutive outputs
template <int NP> __device__ __forceinline__ void da_store4(void *base, int64_t at, float a, float b, float c, float d) {
  if constexpr (NP == 3) {
    *(float4 *)((float *)base + at) = make_float4(a, b, c, d);
  } else if constexpr (NP == 2) {
    *(uint2 *)((uint16_t *)base + at) = make_uint2(f16_pair(a, b), f16_pair(c, d));
  } else {
    *(uint2 *)((uint16_t *)base + at) = make_uint2(bf16_pair(a, b), bf16_pair(c, d));
  }
}

__device__ __forceinline__ f32x16 da_zero16() {
  f32x16 z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}
__device__ __forceinline__ int da_wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// ---------------------------------------------------------------------------------------------------------------- forward
// One workgroup: PAIRS pairs of waves over the keys [split chunk, ...) of one (cloud, key / value head); a pair has 32 packed rows, one of
// its waves the first map, the other the second: half the accumulators each (two or three waves per SIMD, where one wave with both
// maps fills the registers), and the difference is taken once, at the end, through LDS.  The next tile's elements are on their way in
// registers while this one's are multiplied; two buffers, one barrier a tile.  LDS operands are read a phase ahead of their products.
// Bound by the matrix instructions, most of which are V times either map in two pieces: a pair of keys costs 4 D flop for the scores and
// 2 maps x 2 pieces x 4 D for the values = 20 D (fp32: six products for one, 72 D) where the formula has 8 D, the difference taken first.  Taking
// it first needs both maps in one wave, whose accumulators then fill the registers.  Two exponentials, splits and a maximum come on top: a
// SIMD's matrix and vector instructions do not overlap here.  Measured: 2 clouds x 8 heads x 4096 x 4096, D 64, bfloat16: 351 - 371 us (137 GFLOP
// of the formula: 370 - 391 TFLOP/s; 926 - 979 executed, where a large library product reaches 1094), causal 196 - 205; 8 clouds x 8 heads (2
// shared) x 1000, D 48, fp16: 96 us with three fifths of the keys; 32 x 4 x 256 x 256, D 32, fp32: 23 - 25 us; 16 tokens x 16 heads over 8192 keys
// of 4 heads, in 16 parts: 43 us = 6.2 TB/s of cache, and 4.8 us for the join.
template <int NP> constexpr float DA_LIFT = NP == 2 ? 7.f : 0.f;
// the stored statistics: without the lift, so that the logarithm keeps its bits
template <int NP> __device__ __forceinline__ void da_store_stats(float *at, int64_t n, float mx, float sum, bool empty) {
  at[0] = empty ? 0.f : mx + DA_LIFT<NP>;
  at[n] = empty ? DA_INF : log2f(NP == 2 ? sum * 0.0078125f : sum);  // an empty row: every probability 2^-inf = 0
}
template <int NP, int DP, int PAIRS> constexpr int DA_FWD_WAVES = NP == 3 && DP == 64 && PAIRS == 1 ? 1 : 2;  // waves per SIMD
template <int NP, int DP, int PAIRS, bool SPLIT>
__global__ __launch_bounds__(128 * PAIRS) HITADV_WAVES_PER_SIMD((DA_FWD_WAVES<NP, DP, PAIRS>)) void diff_attn_fwd_k(DaP p) {
  using Tile = DaTile<NP, DP>;
  constexpr int NR = DA_NR<NP>, NT = 128 * PAIRS;
  constexpr int NPP = NP == 3 ? 3 : 2;  // pieces of a probability
  constexpr int KC = DP / 16, VB = 2 * DP / 32;
  constexpr bool AHEAD = NP != 3;
  // fp16 values stay as they are, and so a probability is two fp16 pieces: carried 2^7 times as large (the maximum that is kept, and the sum,
  // follow), it lies below 2^15 and is off by at most 2^-22 of itself or 2^-32 of the running maximum
  constexpr int NV = NP == 2 ? 1 : NP;
  constexpr float LIFT = DA_LIFT<NP>;
  using VTile = DaTile<NV, DP>;
  constexpr int BUF = Tile::ROWS + VTile::COLS;
  extern __shared__ __attribute__((aligned(16))) uint16_t da_lds[];
  uint16_t *Ks = da_lds, *Vt = da_lds + Tile::ROWS;
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, wave = da_wave_id(), m = wave & 1, tid = threadIdx.x;
  const int b = blockIdx.x / p.Hkv, hk = blockIdx.x % p.Hkv, split = blockIdx.z;
  const int tile = da_tile(p.causal, true);
  const int row0 = (tile * PAIRS + (wave >> 1)) * DA_T;
  const int len = da_len(p, b);
  const int lim_lo = da_limit(p, da_div_g(p, row0), len), lim_hi = da_limit(p, da_div_g(p, row0 + DA_T - 1), len);
  const int last = da_limit(p, da_div_g(p, min(p.rows, (tile + 1) * PAIRS * DA_T) - 1), len);
  const int k0 = split * p.chunk, k1 = min(last, k0 + p.chunk);
  int lim;
  bf16x8 qf[KC][NR];
  {
    const int r = row0 + col, i = da_div_g(p, r), h = hk * p.G + r - i * p.G;
    lim = da_limit(p, i, len);
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int d = 16 * c + 8 * half;
      uint4 w[NR];
      da_pieces8<NP>(da_load8_if<NP>(p.q, b * p.q_b + i * p.q_n + h * p.q_h + m * p.q_m + d, r < p.rows && d < p.D), w);
      da_sign(w, p);
#pragma unroll
      for (int k = 0; k < NR; ++k) qf[c][k] = as_bf16x8(w[k]);
    }
  }

  f32x16 o[VB];
#pragma unroll
  for (int v = 0; v < VB; ++v) o[v] = da_zero16();
  float mx = -DA_INF, sum = 0.f;

  DaFetchRows<NP, DP, NT> fk;
  DaFetchBlocks<NV, DP, NT> fv;
  const int64_t k_at = b * p.k_b + hk * p.k_h, v_at = b * p.v_b + hk * p.v_h;
  fk.bind(p.k_m, p.D, true, tid);
  fv.bind(0, p.D, false, tid);
  fk.zero_padding(Ks);
  fv.template zero_padding<false, true>(nullptr, Vt);
  fk.zero_padding(Ks + BUF);
  fv.template zero_padding<false, true>(nullptr, Vt + BUF);
  if (k0 < k1) {
    fk.load(p.k, k_at, p.k_n, k0, len);
    fv.load(p.v, v_at, p.v_n, k0, len);
    fk.put(Ks);
    fv.template put<false, true>(nullptr, Vt);
  }
  __syncthreads();
#pragma unroll 1
  for (int t = k0; t < k1; t += DA_T) {
    const bool more = t + DA_T < k1;
    if (more) {
      fk.load(p.k, k_at, p.k_n, t + DA_T, len);
      fv.load(p.v, v_at, p.v_n, t + DA_T, len);
    }
    if (t < lim_hi) {
      f32x16 s = da_zero16();
      bf16x8 kf[KC][NR], vf[2][VB][NV];
      auto read_v = [&](int c) {
#pragma unroll
        for (int v = 0; v < VB; ++v) VTile::frag_col(Vt, 32 * v + col, c, half, vf[c][v]);
      };
#pragma unroll
      for (int c = 0; c < KC; ++c) Tile::frag_row(Ks, col, m * DP + 16 * c + 8 * half, kf[c]);
      if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < KC; ++c) s = da_mfma_in<NP, false>(kf[c], qf[c], s);
      if (AHEAD) {
        read_v(0);
        __builtin_amdgcn_sched_barrier(0);
      }
      float pr[16];
      if (t + DA_T > lim_lo) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (t + 8 * (e >> 2) + 4 * half + (e & 3) >= lim) s[e] = -DA_INF;
      }
      float top = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
      top = __builtin_fmaf(fmaxf(top, __shfl_xor(top, 32, HITADV_WAVE)), p.scale2, -LIFT);
      if (__ballot(top > mx + DA_SLACK) != 0ull) {  // (-inf + slack = -inf: the first visible key raises it)
        const float nm = fmaxf(mx, top);
        const float f = nm == -DA_INF ? 1.f : exp2_flush(mx - nm);
        sum *= f;
        mx = nm;
#pragma unroll
        for (int v = 0; v < VB; ++v)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[v][e] *= f;
      }
      const float base = mx == -DA_INF ? 0.f : mx;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        pr[e] = exp2_flush(__builtin_fmaf(s[e], p.scale2, -base));
        sum += pr[e];
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        bf16x8 bo[NPP];
        if (!AHEAD) read_v(c);
        if (AHEAD && c == 0) {
          read_v(1);
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (NP == 2) da_operand_f16(&pr[8 * c], bo);
        else da_operand<NPP>(&pr[8 * c], bo);
#pragma unroll
        for (int v = 0; v < VB; ++v) {
          if constexpr (NP == 2) o[v] = da_mfma_in<NP, false>(vf[c][v], {bo[0]}, da_mfma_in<NP, false>(vf[c][v], {bo[1]}, o[v]));
          else o[v] = da_mfma<NP, NPP>(vf[c][v], bo, o[v]);
        }
      }
    }
    Ks = Ks == da_lds ? da_lds + BUF : da_lds;  // the other buffer's readers met the barrier that ended the tile before this one
    Vt = Ks + Tile::ROWS;
    if (more) {
      fk.put(Ks);
      fv.template put<false, true>(nullptr, Vt);
    }
    __syncthreads();
  }

  sum += __shfl_xor(sum, 32, HITADV_WAVE);
  const int r = row0 + col, i = da_div_g(p, r), h = hk * p.G + r - i * p.G;
  const bool valid = r < p.rows;
  if (SPLIT) {
    if (!valid) return;
    const int64_t row = ((int64_t)split * p.B * p.Hkv + blockIdx.x) * p.rows + r;
    if (half == 0) *(float2 *)(p.part_ml + 4 * row + 2 * m) = make_float2(mx, sum);
    float *po = p.part_o + (2 * row + m) * 2 * p.D;
#pragma unroll
    for (int v = 0; v < VB; ++v)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = 32 * v + 2 * e + 4 * half;
        if (d < 2 * p.D) *(float4 *)(po + d) = make_float4(o[v][e], o[v][e + 1], o[v][e + 2], o[v][e + 3]);
      }
    return;
  }
  if (p.stats && valid && half == 0) {
    const int64_t n = (int64_t)p.B * p.H * p.Nq, row = ((int64_t)b * p.H + h) * p.Nq + i;
    da_store_stats<NP>(p.stats + (2 * m) * n + row, n, mx, sum, lim == 0);
  }
  const float w = lim == 0 ? 0.f : (m && valid ? -da_lam(p, h) : 1.f) / sum;
  // the second map's part of a value block of 32 columns at a time, in the tiles' place (the last barrier is behind their readers)
  float4 *part = (float4 *)da_lds + (wave >> 1) * 256 + lane;
  const int64_t at = (((int64_t)b * p.Nq + i) * p.H + h) * 2 * p.D;
#pragma unroll
  for (int v = 0; v < VB; ++v) {
    if (m) {
#pragma unroll
      for (int e = 0; e < 4; ++e) part[64 * e] = make_float4(o[v][4 * e] * w, o[v][4 * e + 1] * w, o[v][4 * e + 2] * w, o[v][4 * e + 3] * w);
    }
    __syncthreads();
    if (!m && valid) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 y = part[64 * e];
        const int d = 32 * v + 8 * e + 4 * half;
        if (d < 2 * p.D)
          da_store4<NP>(p.out, at + d, o[v][4 * e] * w + y.x, o[v][4 * e + 1] * w + y.y, o[v][4 * e + 2] * w + y.z, o[v][4 * e + 3] * w + y.w);
      }
    }
    __syncthreads();
  }
}

// joins the splits of a row: waves 0 and 1 weigh a map's splits each, then a thread has a (map, value column), eight splits in flight (one at
// a time: 18.8 us against 6.0 for 256 rows of 32 splits, 2 x 128 columns)
constexpr int DA_MAX_SPLITS = 1024;
template <int NP>
__global__ __launch_bounds__(256) void diff_attn_join_k(DaP p) {
  __shared__ float weight[2][DA_MAX_SPLITS], total[2], other[128];
  const int r = blockIdx.x, bh = blockIdx.y, lane = threadIdx.x & 63, wave = da_wave_id();
  const int b = bh / p.Hkv, hk = bh % p.Hkv, i = da_div_g(p, r), h = hk * p.G + r - i * p.G;
  const int64_t step = (int64_t)p.B * p.Hkv * p.rows, row = (int64_t)bh * p.rows + r;
  if (wave < 2) {
    float mx = -DA_INF, sum = 0.f;
    for (int s = lane; s < p.splits; s += 64) mx = fmaxf(mx, p.part_ml[4 * (row + s * step) + 2 * wave]);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d, HITADV_WAVE));
    const float base = mx == -DA_INF ? 0.f : mx;
    for (int s = lane; s < p.splits; s += 64) {
      const float2 ml = *(const float2 *)(p.part_ml + 4 * (row + s * step) + 2 * wave);
      const float w = exp2_flush(ml.x - base);  // a split that saw nothing: 2^-inf = 0
      weight[wave][s] = w;
      sum += ml.y * w;
    }
    sum = wave_sum(sum);
    if (lane == 0) {
      const bool empty = da_limit(p, i, da_len(p, b)) == 0;
      total[wave] = empty ? 0.f : (wave ? -da_lam(p, h) : 1.f) / sum;
      if (p.stats) {
        const int64_t n = (int64_t)p.B * p.H * p.Nq, srow = ((int64_t)b * p.H + h) * p.Nq + i;
        da_store_stats<NP>(p.stats + (2 * wave) * n + srow, n, mx, sum, empty);
      }
    }
  }
  __syncthreads();
  const int m = threadIdx.x >> 7, d = threadIdx.x & 127;
  float o = 0.f;
  if (d < 2 * p.D) {
    const float *po = p.part_o + (2 * row + m) * 2 * p.D + d;
    const int64_t st = step * 4 * p.D;
    for (int s = 0; s < p.splits; s += 8) {
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = s + u < p.splits ? po[(s + u) * st] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) o += s + u < p.splits ? x[u] * weight[m][s + u] : 0.f;
    }
    o *= total[m];
  }
  if (m) other[d] = o;
  __syncthreads();
  if (!m && d < 2 * p.D) {
    const float x = o + other[d];
    const int64_t at = (((int64_t)b * p.Nq + i) * p.H + h) * 2 * p.D + d;
    if constexpr (NP == 3) ((float *)p.out)[at] = x;
    else if constexpr (NP == 2) ((_Float16 *)p.out)[at] = (_Float16)x;
    else ((uint16_t *)p.out)[at] = (uint16_t)(bf16_pair(x, 0.f) & 0xffffu);
  }
}

// The same for few splits of many rows, where a workgroup a row is mostly its own launch: a thread has four columns of a row and both maps, four
// splits in flight, and weighs the splits for itself.  16384 rows of 3 splits 10.6 us against 27.7 with a workgroup each; 256 rows of 16 splits
// 12.6 us against 5.4, so up to 8.
constexpr int DA_FEW_SPLITS = 8;
template <int NP>
__global__ __launch_bounds__(256) void diff_attn_join_few_k(DaP p) {
  const int w = p.D / 2, at4 = blockIdx.x * 256 + threadIdx.x, r = at4 / w, c = 4 * (at4 - r * w), bh = blockIdx.y;
  if (r >= p.rows) return;
  const int b = bh / p.Hkv, hk = bh % p.Hkv, i = da_div_g(p, r), h = hk * p.G + r - i * p.G;
  const int64_t step = (int64_t)p.B * p.Hkv * p.rows, row = (int64_t)bh * p.rows + r;
  const float4 *ml = (const float4 *)p.part_ml + row;  // maximum and sum of map 1, of map 2
  const float *po = p.part_o + 4 * row * p.D + c;
  float mx[2] = {-DA_INF, -DA_INF}, sum[2] = {0.f, 0.f}, o[2][4] = {};
  for (int s = 0; s < p.splits; ++s) {
    const float4 x = ml[s * step];
    mx[0] = fmaxf(mx[0], x.x);
    mx[1] = fmaxf(mx[1], x.z);
  }
  const float base0 = mx[0] == -DA_INF ? 0.f : mx[0], base1 = mx[1] == -DA_INF ? 0.f : mx[1];
  for (int s0 = 0; s0 < p.splits; s0 += 4) {
    float4 x[4], y[4][2];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = min(s0 + u, p.splits - 1);
      x[u] = ml[s * step];
      y[u][0] = *(const float4 *)(po + s * step * 4 * p.D);
      y[u][1] = *(const float4 *)(po + s * step * 4 * p.D + 2 * p.D);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (s0 + u >= p.splits) break;
      const float f[2] = {exp2_flush(x[u].x - base0), exp2_flush(x[u].z - base1)};  // a split that saw nothing: 2^-inf = 0
      sum[0] += x[u].y * f[0];
      sum[1] += x[u].w * f[1];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        o[m][0] += y[u][m].x * f[m];
        o[m][1] += y[u][m].y * f[m];
        o[m][2] += y[u][m].z * f[m];
        o[m][3] += y[u][m].w * f[m];
      }
    }
  }
  const bool empty = da_limit(p, i, da_len(p, b)) == 0;
  const float t0 = empty ? 0.f : 1.f / sum[0], t1 = empty ? 0.f : -da_lam(p, h) / sum[1];
  da_store4<NP>(p.out, (((int64_t)b * p.Nq + i) * p.H + h) * 2 * p.D + c, o[0][0] * t0 + o[1][0] * t1, o[0][1] * t0 + o[1][1] * t1,
                o[0][2] * t0 + o[1][2] * t1, o[0][3] * t0 + o[1][3] * t1);
  if (p.stats && c == 0) {
    const int64_t n = (int64_t)p.B * p.H * p.Nq, srow = ((int64_t)b * p.H + h) * p.Nq + i;
    da_store_stats<NP>(p.stats + srow, n, mx[0], sum[0], empty);
    da_store_stats<NP>(p.stats + 2 * n + srow, n, mx[1], sum[1], empty);
  }
}

// ---------------------------------------------------------------------------------------------------------------- backward
// dP = dO V^T;  r_m = sum_j P_m dP;  dS_1 = P_1 (dP - r_1), dS_2 = -lam P_2 (dP - r_2).  The r are sums over the very P and dP that the
// second pass multiplies (not dO . out: out is rounded, and where a row sees one key dS has to vanish exactly).
//
// dQ: the forward kernel's layout, two passes over the keys: first r, then dQ_m^T = K_m^T dS_m^T.
// A pair of waves shares 32 packed rows and takes the even and the odd tiles of 32 keys; the two meet in LDS (r behind the first pass, dQ at
// the end): half the longest row's way through the keys, and twice the waves where clouds are few or short.  Bound by instruction issue:
// 24 D matrix flop a pair of keys where the formula has 12 (the scores and dP twice, dS as two pieces).  2 x 8 x 4096 x 4096, D 64, bfloat16:
// 526 - 567 us, causal 298 - 311 (660 - 690 TFLOP/s executed); 32 x 4 x 256, D 32, fp32: 44 us.  A one-pass form (a third of the products less)
// needs r before the sweep, as dO . O_m of the unrounded sums O_m of either map: 4 D fp32 values a row written and read once more.
template <int NP, int DP> constexpr int DA_DQ_WAVES = NP == 3 && DP == 64 ? 1 : 2;  // waves per SIMD
template <int NP, int DP, int PAIRS>
__global__ __launch_bounds__(128 * PAIRS) HITADV_WAVES_PER_SIMD((DA_DQ_WAVES<NP, DP>)) void diff_attn_dq_k(DaP p) {
  using Tile = DaTile<NP, DP>;
  constexpr int NR = DA_NR<NP>;
  constexpr int NS = NP == 3 ? 3 : 2;  // pieces of dS
  constexpr int KC = DP / 16, VC = 2 * DP / 16, DB = DP / 32;
  constexpr int SET = 2 * Tile::ROWS + Tile::COLS, NT = 64 * PAIRS;
  extern __shared__ __attribute__((aligned(16))) uint16_t da_lds[];
  float *red = (float *)(da_lds + 2 * SET);  // [2 parities][PAIRS][3][32]: either map's r, key 0's dP
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, wave = da_wave_id(), tid = threadIdx.x;
  const int pair = wave >> 1, odd = wave & 1;
  const int b = blockIdx.x / p.Hkv, hk = blockIdx.x % p.Hkv;
  const int tile = da_tile(p.causal, true);
  const int row0 = (tile * PAIRS + pair) * DA_T;
  const int len = da_len(p, b);
  const int lim_lo = da_limit(p, da_div_g(p, row0), len), lim_hi = da_limit(p, da_div_g(p, row0 + DA_T - 1), len);
  const int last = da_limit(p, da_div_g(p, min(p.rows, (tile + 1) * PAIRS * DA_T) - 1), len);
  const int64_t n = (int64_t)p.B * p.H * p.Nq;
  const uint16_t *Ks = da_lds + odd * SET, *Vs = Ks + Tile::ROWS, *Kt = Vs + Tile::ROWS;  // the wave's tiles
  const int ph = wave / PAIRS;  // the parity that the wave stages
  uint16_t *Kp = da_lds + ph * SET, *Vp = Kp + Tile::ROWS, *Tp = Vp + Tile::ROWS;

  // every other tile of keys takes dP with its sign turned: the matrix instruction truncates downwards, and the offsets cancel in r (with one
  // sign dlam of 7 x 2 heads x 1987 rows in bf16 is 1.8e-6 off)
  const bool neg = odd != 0;
  const float sgn = neg ? -1.f : 1.f;
  bf16x8 qf[2][KC][NR], gf[VC][NR];
  float mx[2], ll[2], rs[2] = {0.f, 0.f}, back[2] = {1.f, 1.f};
  int lim;
  {
    const int r = row0 + col, i = da_div_g(p, r), h = hk * p.G + r - i * p.G;
    const bool valid = r < p.rows;
    const int64_t srow = ((int64_t)b * p.H + h) * p.Nq + i;
    lim = da_limit(p, i, len);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int d = 16 * c + 8 * half;
        uint4 w[NR];
        da_pieces8<NP>(da_load8_if<NP>(p.q, b * p.q_b + i * p.q_n + h * p.q_h + m * p.q_m + d, valid && d < p.D), w);
        da_sign(w, p);
#pragma unroll
        for (int k = 0; k < NR; ++k) qf[m][c][k] = as_bf16x8(w[k]);
      }
#pragma unroll
    for (int c = 0; c < VC; ++c) {
      const int d = 16 * c + 8 * half;
      uint4 w[NR];
      da_pieces8<NP>(da_load8_if<NP>(p.dout, (((int64_t)b * p.Nq + i) * p.H + h) * 2 * p.D + d, valid && lim > 0 && d < 2 * p.D), w);
      da_turn(w, neg);
#pragma unroll
      for (int k = 0; k < NR; ++k) gf[c][k] = as_bf16x8(w[k]);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      mx[m] = valid ? p.stats[(2 * m) * n + srow] : 0.f;
      ll[m] = valid ? p.stats[(2 * m + 1) * n + srow] : DA_INF;
      if (NP != 3) {
        // one subtraction less (fp32 keeps the two apart).  What the sum rounds off is the row's factor 2^-off, which r gets back: dlam adds r over
        // all rows
        const float c = mx[m] + ll[m], y = c - mx[m], off = (mx[m] - (c - y)) + (ll[m] - y);
        back[m] = ll[m] == DA_INF ? 1.f : 1.f - 0.69314718f * off;
        mx[m] = c;
      }
    }
  }
  f32x16 acc[2][DB];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int v = 0; v < DB; ++v) acc[m][v] = da_zero16();

  DaFetchBlocks<NP, DP, NT> fk;
  DaFetchRows<NP, DP, NT> fv;
  const int64_t k_at = b * p.k_b + hk * p.k_h, v_at = b * p.v_b + hk * p.v_h;
  fk.bind(p.k_m, p.D, true, tid % NT);
  fv.bind(0, p.D, false, tid % NT);
  fk.template zero_padding<true, true>(Kp, Tp);
  fv.zero_padding(Vp);
  if (last > 0) {
    fk.load(p.k, k_at, p.k_n, ph * DA_T, len);
    fv.load(p.v, v_at, p.v_n, ph * DA_T, len);
  }
  // Matrix and vector instructions of a SIMD do not overlap here, so a wave's time is its instructions and its waits; left to itself the
  // compiler reads an LDS operand, waits, multiplies and reads the next.  Scheduling fences hold the reads ahead (three pieces have six
  // products to an operand and no registers for more than one).
  constexpr int AHEAD = NP == 3 ? 1 : 4;
  auto sweep = [&](auto second) {
    constexpr bool SECOND = decltype(second)::value;
#pragma unroll 1
    for (int t0 = 0; t0 < last; t0 += 2 * DA_T) {
      __syncthreads();
      fv.put(Vp);
      fk.template put<true, SECOND>(Kp, Tp);
      __syncthreads();
      const int next = (t0 + 2 * DA_T < last ? t0 + 2 * DA_T : 0) + ph * DA_T;  // (behind the second pass: the first tiles once more, not used)
      fk.load(p.k, k_at, p.k_n, next, len);
      fv.load(p.v, v_at, p.v_n, next, len);
      const int t = t0 + odd * DA_T;
      if (t >= lim_hi) continue;
      // V's operands, then the first map's K's: a stream read AHEAD operands before the products that take them
      bf16x8 fr[VC + KC][NR], kt[2][DB][NP];
      auto read = [&](int c) {
        if (c < VC) Tile::frag_row(Vs, col, 16 * c + 8 * half, fr[c]);
        else Tile::frag_row(Ks, col, 16 * (c - VC) + 8 * half, fr[c]);
      };
      auto read_kt = [&](int m) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int v = 0; v < DB; ++v) Tile::frag_col(Kt, m * DP + 32 * v + col, c, half, kt[c][v]);
      };
      f32x16 dp = da_zero16(), small = da_zero16(), s = da_zero16();
#pragma unroll
      for (int c = 0; c < AHEAD; ++c) read(c);
      if (AHEAD > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < VC + KC; ++c) {
        if (c + AHEAD < VC + KC) read(c + AHEAD);
        if (AHEAD > 1) __builtin_amdgcn_sched_barrier(0);
        if (c < VC) da_mfma_in2<NP, false>(fr[c], gf[c < VC ? c : 0], dp, small);
        else s = da_mfma_in<NP, false>(fr[c], qf[0][c < VC ? 0 : c - VC], s);
      }
      if (NP == 3) {
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] += small[e];
      }
      if (!SECOND && t == 0 && half == 0) red[(pair * 3 + 2) * 32 + col] = sgn * dp[0];  // key 0
      const bool edge = t + DA_T > lim_lo;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (SECOND && NP == 1) read_kt(m);
        __builtin_amdgcn_sched_barrier(0);  // (three pieces: without it four registers too many)
        float pr[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = __builtin_fmaf(s[e], p.scale2, -mx[m]);
          pr[e] = exp2_flush(NP == 3 ? x - ll[m] : x);
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (t + 8 * (e >> 2) + 4 * half + (e & 3) >= lim) pr[e] = 0.f;
        }
        bf16x8 kn[KC][NR];
        if (m == 0 && AHEAD > 1) {
#pragma unroll
          for (int c = 0; c < KC; ++c) Tile::frag_row(Ks, col, DP + 16 * c + 8 * half, kn[c]);
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!SECOND) {
#pragma unroll
          for (int e = 0; e < 16; ++e) rs[m] = __builtin_fmaf(pr[e], dp[e], rs[m]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) pr[e] *= dp[e] - rs[m];
          if (NP != 1) read_kt(m);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            bf16x8 bo[NS];
            da_operand<NS>(&pr[8 * c], bo);
#pragma unroll
            for (int v = 0; v < DB; ++v) acc[m][v] = da_mfma<NP, NS>(kt[c][v], bo, acc[m][v]);
          }
        }
        if (m == 0) {
          s = da_zero16();
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            if (AHEAD == 1) Tile::frag_row(Ks, col, DP + 16 * c + 8 * half, kn[c]);
            s = da_mfma_in<NP, false>(kn[c], qf[1][c], s);
          }
        }
      }
    }
  };
  sweep(std::false_type());
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    rs[m] += __shfl_xor(rs[m], 32, HITADV_WAVE);
    if (half == 0) red[((odd * PAIRS + pair) * 3 + m) * 32 + col] = sgn * rs[m];
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    rs[m] = (red[(pair * 3 + m) * 32 + col] + red[((PAIRS + pair) * 3 + m) * 32 + col]) * back[m];
    if (lim == 1) rs[m] = red[(pair * 3 + 2) * 32 + col];  // a row with one key: its probability is 1, dP - r exactly 0
    rs[m] *= sgn;
  }
  sweep(std::true_type());
  // the odd wave's dQ, a block of 32 columns at a time, in the tiles' place
  float4 *part = (float4 *)da_lds + pair * 256 + lane;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int v = 0; v < DB; ++v) {
      __syncthreads();
      if (odd) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          part[64 * e] = make_float4(acc[m][v][4 * e], acc[m][v][4 * e + 1], acc[m][v][4 * e + 2], acc[m][v][4 * e + 3]);
      }
      __syncthreads();
      if (!odd) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 y = part[64 * e];
          acc[m][v][4 * e] -= y.x, acc[m][v][4 * e + 1] -= y.y, acc[m][v][4 * e + 2] -= y.z, acc[m][v][4 * e + 3] -= y.w;  // (turned)
        }
      }
    }
  if (odd) return;
  const int ln = lane_counted(), r = row0 + (ln & 31), i = da_div_g(p, r), h = hk * p.G + r - i * p.G;
  if (r >= p.rows) return;
  if (ln < 32) {
    const int64_t srow = ((int64_t)b * p.H + h) * p.Nq + i;
    p.r[srow] = sgn * rs[0];
    p.r[n + srow] = sgn * rs[1];
  }
  const int64_t at = (((int64_t)b * p.Nq + i) * p.H + h) * 2 * p.D;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const float w = sgn * (m == 0 ? p.scale : -da_lam(p, h) * p.scale);
#pragma unroll
    for (int v = 0; v < DB; ++v)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = 32 * v + 2 * e + 4 * (ln >> 5);
        if (d < p.D) da_store4<NP>(p.dq, at + m * p.D + d, acc[m][v][e] * w, acc[m][v][e + 1] * w, acc[m][v][e + 2] * w, acc[m][v][e + 3] * w);
      }
  }
}

// dK and dV: a wave owns 32 keys (the lane's column) and walks over the packed rows of all G heads, so that the sum over the heads that
// share a key needs no atomics: dV^T += dO^T A, dK_m^T += Q_m^T dS_m, A = P_1 - lam P_2.  One launch for both, except for fp32 at DP = 64,
// where three pieces of K and V and both accumulators are more than 512 registers: dV and dK in a launch each (the scores twice, a quarter
// more products).  Bound by instruction issue and, with one wave a SIMD (the accumulators: 192 registers at DP = 64), by what of a barrier
// and of LDS latency a wave sees alone.  2 x 8 x 4096 x 4096, D 64, bfloat16: 687 - 742 us, causal 390 - 406 (508 - 529 TFLOP/s executed);
// 32 x 4 x 256, D 32, fp32: 48 us.
template <int NP, int DP> constexpr int DA_DKV_WAVES = NP != 3 && DP == 32 ? 2 : 1;  // waves per SIMD
template <int NP, int DP, int NW, bool DV, bool DK>
__global__ __launch_bounds__(64 * NW) HITADV_WAVES_PER_SIMD((DA_DKV_WAVES<NP, DP>)) void diff_attn_dkv_k(DaP p) {
  using Tile = DaTile<NP, DP>;
  constexpr int NR = DA_NR<NP>;
  constexpr int NS = NP == 3 ? 3 : 2;
  constexpr int KC = DP / 16, VC = 2 * DP / 16, DB = DP / 32, VB = 2 * DP / 32;
  extern __shared__ __attribute__((aligned(16))) uint16_t da_lds[];
  uint16_t *Qs = da_lds, *Gs = Qs + Tile::ROWS, *Qt = Gs + (DK ? Tile::ROWS : 0), *Gt = Qt + (DK ? Tile::COLS : 0);
  float *st = (float *)(Gt + (DV ? Tile::COLS : 0));  // [7][32]: max 1, log2 sum 1, max 2, log2 sum 2, r 1, r 2, -lam
  int *lims = (int *)(st + 7 * DA_T);
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, wave = da_wave_id(), tid = threadIdx.x;
  const int b = blockIdx.x / p.Hkv, hk = blockIdx.x % p.Hkv;
  const int first = da_tile(p.causal, false) * NW * DA_T, key0 = first + wave * DA_T, key = key0 + col;
  const int len = da_len(p, b);
  const int64_t n = (int64_t)p.B * p.H * p.Nq;

  const bool neg = (key0 / DA_T & 1) != 0;  // (as in diff_attn_dq_k)
  const float sgn = neg ? -1.f : 1.f;
  bf16x8 kf[2][KC][NR], vf[VC][NR];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int d = 16 * c + 8 * half;
      uint4 w[NR];
      da_pieces8<NP>(da_load8_if<NP>(p.k, b * p.k_b + key * p.k_n + hk * p.k_h + m * p.k_m + d, key < len && d < p.D), w);
      da_sign(w, p);
#pragma unroll
      for (int k = 0; k < NR; ++k) kf[m][c][k] = as_bf16x8(w[k]);
    }
#pragma unroll
  for (int c = 0; c < (DK ? VC : 0); ++c) {
    const int d = 16 * c + 8 * half;
    uint4 w[NR];
    da_pieces8<NP>(da_load8_if<NP>(p.v, b * p.v_b + key * p.v_n + hk * p.v_h + d, key < len && d < 2 * p.D), w);
    da_turn(w, neg);
#pragma unroll
    for (int k = 0; k < NR; ++k) vf[c][k] = as_bf16x8(w[k]);
  }
  f32x16 av[VB], ak[2][DB];
#pragma unroll
  for (int v = 0; v < VB; ++v) av[v] = da_zero16();
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int v = 0; v < DB; ++v) ak[m][v] = da_zero16();

  // causal: query i sees key j when i >= j - (Nk - Nq): rows before that of the workgroup's first key have nothing here
  int begin = p.causal ? max(0, first - (p.Nk - p.Nq)) : 0;
  begin = first >= len ? p.rows : (int)min((int64_t)p.rows, (int64_t)begin * p.G) / DA_T * DA_T;
  // rows that see no key at all share a tile with the first that do: 0 times what they hold need not be 0
  const int none = p.causal ? max(0, p.Nq - p.Nk) * p.G : 0;
  DaFetchBlocks<NP, DP, 64 * NW> fq, fg;
  const int64_t g_n = (int64_t)p.H * 2 * p.D;
  const int64_t q_at = b * p.q_b + hk * p.G * p.q_h, g_at = ((int64_t)b * p.Nq * p.H + hk * p.G) * 2 * p.D;
  fq.bind(p.q_m, p.D, true, tid);
  fg.bind(0, p.D, false, tid);
  fq.template zero_padding<true, DK>(Qs, Qt);
  fg.template zero_padding<DK, DV>(Gs, Gt);
  // the rows' own values, fetched ahead like the tiles: thread (w = tid / 32, row): w = 0, 1 a map's maximum and log2 sum, 2 both r, 3 lam
  float ahead[2] = {0.f, 0.f};
  auto load_row = [&](int t) {
    if (tid >= 4 * DA_T) return;
    const int w = tid >> 5, r = min(t + (tid & 31), p.rows - 1), i = da_div_g(p, r), h = hk * p.G + r - i * p.G;
    const int64_t srow = ((int64_t)b * p.H + h) * p.Nq + i;
    const float *one = w < 2 ? p.stats + 2 * w * n + srow : w == 2 ? p.r + srow : p.lam + (p.lam_n == 1 ? 0 : h);
    const float *two = w < 3 ? one + n : one;
    ahead[0] = *one;
    ahead[1] = *two;
  };
  auto put_row = [&](int t) {
    if (tid >= 4 * DA_T) return;
    const int w = tid >> 5, at = tid & 31;
    if (w < 2) {
      const float ll = t + at < p.rows ? ahead[1] : DA_INF;  // a row that does not exist: probability 2^-inf
      st[2 * w * DA_T + at] = NP == 3 ? ahead[0] : ahead[0] + ll;  // (as in diff_attn_dq_k)
      st[(2 * w + 1) * DA_T + at] = ll;
    } else if (w == 2) {
      st[4 * DA_T + at] = ahead[0];
      st[5 * DA_T + at] = ahead[1];
    } else {
      st[6 * DA_T + at] = -ahead[0];
      lims[at] = da_limit(p, da_div_g(p, t + at), len);  // the first key that the row does not see
    }
  };
  if (begin < p.rows) {
    load_row(begin);
    fq.load_packed(p.q, q_at, p.q_n, p.q_h, p, begin);
    fg.load_packed(p.dout, g_at, g_n, 2 * p.D, p, begin);
  }
#pragma unroll 1
  for (int t = begin; t < p.rows; t += DA_T) {
    __syncthreads();
    fq.template put<true, DK>(Qs, Qt, none - t);
    fg.template put<DK, DV>(Gs, Gt, none - t);
    put_row(t);
    __syncthreads();
    load_row(t + DA_T);  // (behind the last tile: its last row once more, not used)
    fq.load_packed(p.q, q_at, p.q_n, p.q_h, p, t + DA_T);
    fg.load_packed(p.dout, g_at, g_n, 2 * p.D, p, t + DA_T);
    constexpr bool FENCED = NP != 3 && DP == 64;      // (as in diff_attn_dq_k)
    constexpr bool SPOT = (NP == 3) == (DP == 64);    // read where they are used: no registers left, or two waves to a SIMD
    bf16x8 ga[VC][NR], qa[2][KC][NR];
    auto read_q = [&](int m) {
#pragma unroll
      for (int c = 0; c < KC; ++c) Tile::frag_row(Qs, col, m * DP + 16 * c + 8 * half, qa[m][c]);
      if (FENCED) __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int c = 0; c < (DK && !SPOT ? VC : 0); ++c) Tile::frag_row(Gs, col, 16 * c + 8 * half, ga[c]);
    if (!SPOT) read_q(0);
    f32x16 dp = da_zero16(), small = da_zero16(), s[2] = {da_zero16(), da_zero16()};
#pragma unroll
    for (int c = 0; c < (DK ? VC : 0); ++c) {
      if (SPOT) Tile::frag_row(Gs, col, 16 * c + 8 * half, ga[c]);
      da_mfma_in2<NP, true>(ga[c], vf[c], dp, small);
    }
    if (FENCED) __builtin_amdgcn_sched_barrier(0);
    if (!SPOT) read_q(1);
    auto scores = [&](int m) {
      if (SPOT) read_q(m);
#pragma unroll
      for (int c = 0; c < KC; ++c) s[m] = da_mfma_in<NP, true>(qa[m][c], kf[m][c], s[m]);
    };
    if (!SPOT) {
      scores(0);
      scores(1);
    }
    if (FENCED) __builtin_amdgcn_sched_barrier(0);
    if (NP == 3) {
#pragma unroll
      for (int e = 0; e < 16; ++e) dp[e] += small[e];
    }
    const bool edge = key0 + DA_T > da_limit(p, da_div_g(p, t), len);  // (limits grow with the row; rows that do not exist: 2^-inf = 0)
    bf16x8 gt[2][VB][NP];
    float A[16];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      if (SPOT) scores(m);
      // rows 8 q + 4 half .. + 3 in registers 4 q .. 4 q + 3
      float4 mx[4], ll[4], rr[4], nl[4];
      bf16x8 qt[2][DB][NP];
      auto read_softmax = [&](int q) {
        mx[q] = *(const float4 *)(st + (2 * m) * DA_T + 8 * q + 4 * half);
        if (NP == 3) ll[q] = *(const float4 *)(st + (2 * m + 1) * DA_T + 8 * q + 4 * half);
      };
      auto read_r = [&](int q) {
        if (DK) rr[q] = *(const float4 *)(st + (4 + m) * DA_T + 8 * q + 4 * half);
        if (m) nl[q] = *(const float4 *)(st + 6 * DA_T + 8 * q + 4 * half);
      };
      if (!SPOT) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          read_softmax(q);
          read_r(q);
        }
#pragma unroll
        for (int c = 0; c < (DK ? 2 : 0); ++c)
#pragma unroll
          for (int v = 0; v < DB; ++v) Tile::frag_col(Qt, m * DP + 32 * v + col, c, half, qt[c][v]);
        if (DV && m) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int v = 0; v < VB; ++v) Tile::frag_col(Gt, 32 * v + col, c, half, gt[c][v]);
        }
      }
      if (FENCED) __builtin_amdgcn_sched_barrier(0);
      float pr[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (SPOT) read_softmax(q);
        const float mxs[4] = {mx[q].x, mx[q].y, mx[q].z, mx[q].w};
        float lls[4] = {0.f, 0.f, 0.f, 0.f};
        if (NP == 3) lls[0] = ll[q].x, lls[1] = ll[q].y, lls[2] = ll[q].z, lls[3] = ll[q].w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = __builtin_fmaf(s[m][4 * q + j], p.scale2, -mxs[j]);
          pr[4 * q + j] = exp2_flush(NP == 3 ? x - lls[j] : x);
        }
      }
      if (edge) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int4 li = *(const int4 *)(lims + 8 * q + 4 * half);
          const int lis[4] = {li.x, li.y, li.z, li.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (key >= lis[j]) pr[4 * q + j] = 0.f;
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (SPOT) read_r(q);
        float *x = &pr[4 * q];
        if (m) x[0] *= nl[q].x, x[1] *= nl[q].y, x[2] *= nl[q].z, x[3] *= nl[q].w;  // -lam P_2
#pragma unroll
        for (int j = 0; j < 4; ++j) A[4 * q + j] = m ? A[4 * q + j] + x[j] : x[j];
        if (DK) {
          const f32x16 &d = dp;
          x[0] *= __builtin_fmaf(sgn, d[4 * q], -rr[q].x), x[1] *= __builtin_fmaf(sgn, d[4 * q + 1], -rr[q].y);
          x[2] *= __builtin_fmaf(sgn, d[4 * q + 2], -rr[q].z), x[3] *= __builtin_fmaf(sgn, d[4 * q + 3], -rr[q].w);
        }
      }
#pragma unroll
      for (int c = 0; c < (DK ? 2 : 0); ++c) {
        bf16x8 bo[NS];
        da_operand<NS>(&pr[8 * c], bo);
#pragma unroll
        for (int v = 0; v < DB; ++v) {
          if (SPOT) Tile::frag_col(Qt, m * DP + 32 * v + col, c, half, qt[c][v]);
          ak[m][v] = da_mfma<NP, NS>(qt[c][v], bo, ak[m][v]);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < (DV ? 2 : 0); ++c) {
      bf16x8 bo[NS];
      da_operand<NS>(&A[8 * c], bo);
#pragma unroll
      for (int v = 0; v < VB; ++v) {
        if (SPOT) Tile::frag_col(Gt, 32 * v + col, c, half, gt[c][v]);
        av[v] = da_mfma<NP, NS>(gt[c][v], bo, av[v]);
      }
    }
  }
  if (key >= p.Nk) return;
  const int64_t at = (((int64_t)b * p.Nk + key) * p.Hkv + hk) * 2 * p.D;
#pragma unroll
  for (int v = 0; v < (DV ? VB : 0); ++v)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int d = 32 * v + 2 * e + 4 * half;
      if (d < 2 * p.D) da_store4<NP>(p.dv, at + d, av[v][e], av[v][e + 1], av[v][e + 2], av[v][e + 3]);
    }
#pragma unroll
  for (int m = 0; m < (DK ? 2 : 0); ++m)
#pragma unroll
    for (int v = 0; v < DB; ++v)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = 32 * v + 2 * e + 4 * half;
        if (d < p.D)
          da_store4<NP>(p.dk, at + m * p.D + d, ak[m][v][e] * p.scale, ak[m][v][e + 1] * p.scale, ak[m][v][e + 2] * p.scale,
                        ak[m][v][e + 3] * p.scale);
      }
}

// dlam[h] = -sum over clouds and queries of r_2 (one value for all heads: over the heads too); one workgroup per output, fixed order,
// sums in double (a long sum of values of both signs); latency of one pass: 5 us for 32 x 256 rows
__global__ __launch_bounds__(1024) void diff_attn_dlam_k(const float *__restrict__ r2, int B, int H, int Nq, int lam_n, float *__restrict__ dlam) {
  __shared__ double part[16];
  double s = 0.0;
  const int heads = lam_n == 1 ? H : 1;
  const int64_t n = (int64_t)B * heads * Nq;
  for (int64_t at = threadIdx.x; at < n; at += 8192) {  // eight in flight
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t k = at + 1024 * u, bh = k < n ? k / Nq : 0;
      x[u] = k < n ? r2[lam_n == 1 ? k : (bh * H + blockIdx.x) * Nq + (k - bh * Nq)] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) s += (double)x[u];
  }
  for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, HITADV_WAVE);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int u = 1; u < 16; ++u) s += part[u];
    dlam[blockIdx.x] = (float)-s;
  }
}

// ---------------------------------------------------------------------------------------------------------------- host
constexpr int64_t DA_STRIDE = 1 << 24;
struct DaPlan {
  int pairs, tiles, splits, chunk;
};
// Up to 32 rows: one pair of waves (16 tokens x 16 heads over 8192 keys of 4: one pair 44 us, two 70, four 117).  Else four pairs share the keys'
// tiles (2 x 8 x 4096 causal: one 305 us, two 227, four 196; 32 x 4 x 256 in fp32: 42, 25, 23), but two where few short rows leave the chip
// empty (16 x 4 x 128: two 11.2 us, four 12.5; 2 x 4 x 100 rows over 1000 keys with the join: 18.6, 29.4).
// Below 2048 waves the keys are split so that the chip fills (the tokens over 8192 keys with the join: one part 297 us, 16 parts 49, 32 parts
// 62; 4 x 4096 rows causal: one 152, three 68 + 11 for the join), parts of 256 keys at least (5 tokens over 3000 keys: 256 keys a part 18.6 us,
// 512 28.8), of 512 with four pairs, where the join of many rows costs what the parts save (8 x 4 x 512 rows over 512 keys: one part 26 us, two 25
// and 8 for the join).
static DaPlan da_plan(int B, int Nq, int Nk, int H, int Hkv) {
  DaPlan pl;
  const int64_t rows = (int64_t)Nq * (H / Hkv), bh = (int64_t)B * Hkv;
  pl.pairs = rows <= DA_T ? 1 : rows <= 8 * DA_T && bh * ((rows + 4 * DA_T - 1) / (4 * DA_T)) < 256 ? 2 : 4;
  pl.tiles = (int)((rows + DA_T * pl.pairs - 1) / (DA_T * pl.pairs));
  const int64_t waves = bh * pl.tiles * pl.pairs * 2, want = ((pl.pairs == 1 ? 2048 : 3000) + waves - 1) / waves;
  const int64_t most = pl.pairs == 4 ? (Nk + 511) / 512 : (Nk + 255) / 256;
  int64_t s = waves >= 2048 ? 1 : want < most ? want : most;
  if (s < 1) s = 1;
  if (s > DA_MAX_SPLITS) s = DA_MAX_SPLITS;
  int64_t chunk = ((Nk + s - 1) / s + DA_T - 1) / DA_T * DA_T;
  if (chunk < DA_T) chunk = DA_T;
  pl.chunk = (int)chunk;
  pl.splits = (int)((Nk + chunk - 1) / chunk);
  if (pl.splits < 1) pl.splits = 1;
  return pl;
}

template <int NP, int DP, int PAIRS> static int da_launch_fwd_pairs(const DaP &p, const DaPlan &pl, hipStream_t s) {
  const int tiles = 4 * (DaTile<NP, DP>::ROWS + DaTile<NP == 2 ? 1 : NP, DP>::COLS), parts = PAIRS * 4096;  // bytes
  const int lds = tiles > parts ? tiles : parts;
  const dim3 grid(p.B * p.Hkv, pl.tiles, pl.splits);
  if (pl.splits > 1) {
    HITADV_RAISE_LDS((diff_attn_fwd_k<NP, DP, PAIRS, true>), lds);
    diff_attn_fwd_k<NP, DP, PAIRS, true><<<grid, 128 * PAIRS, lds, s>>>(p);
    HITADV_LAUNCH_CHECK();
    if (pl.splits <= DA_FEW_SPLITS) diff_attn_join_few_k<NP><<<dim3((p.rows * (p.D / 2) + 255) / 256, p.B * p.Hkv), 256, 0, s>>>(p);
    else diff_attn_join_k<NP><<<dim3(p.rows, p.B * p.Hkv), 256, 0, s>>>(p);
  } else {
    HITADV_RAISE_LDS((diff_attn_fwd_k<NP, DP, PAIRS, false>), lds);
    diff_attn_fwd_k<NP, DP, PAIRS, false><<<grid, 128 * PAIRS, lds, s>>>(p);
  }
  HITADV_LAUNCH_CHECK();
  return 0;
}
template <int NP, int DP> static int da_launch_fwd(const DaP &p, const DaPlan &pl, hipStream_t s) {
  return pl.pairs == 1 ? da_launch_fwd_pairs<NP, DP, 1>(p, pl, s)
       : pl.pairs == 2 ? da_launch_fwd_pairs<NP, DP, 2>(p, pl, s) : da_launch_fwd_pairs<NP, DP, 4>(p, pl, s);
}
template <int NP, int DP, int PAIRS> static int da_launch_dq(const DaP &p, hipStream_t s) {
  const int lds = 4 * (2 * DaTile<NP, DP>::ROWS + DaTile<NP, DP>::COLS) + 2 * PAIRS * 3 * 32 * 4;  // bytes
  const int tiles = (p.rows + PAIRS * DA_T - 1) / (PAIRS * DA_T);
  HITADV_RAISE_LDS((diff_attn_dq_k<NP, DP, PAIRS>), lds);
  diff_attn_dq_k<NP, DP, PAIRS><<<dim3(p.B * p.Hkv, tiles), 128 * PAIRS, lds, s>>>(p);
  HITADV_LAUNCH_CHECK();
  return 0;
}
template <int NP, int DP> static int da_launch_bwd(const DaP &p, float *dlam, hipStream_t s) {
  const int tk = (p.Nk + 4 * DA_T - 1) / (4 * DA_T);
  const int rc = da_launch_dq<NP, DP, NP == 3 && DP == 64 ? 2 : 4>(p, s);
  if (rc != 0) return rc;
  if (p.dk) {
    const dim3 grid(p.B * p.Hkv, tk);
    constexpr int R = 2 * DaTile<NP, DP>::ROWS, C = 2 * DaTile<NP, DP>::COLS, ST = 8 * DA_T * 4;  // bytes
    if constexpr (NP == 3 && DP == 64) {
      HITADV_RAISE_LDS((diff_attn_dkv_k<NP, DP, 4, true, false>), R + C + ST);
      diff_attn_dkv_k<NP, DP, 4, true, false><<<grid, 256, R + C + ST, s>>>(p);
      HITADV_LAUNCH_CHECK();
      HITADV_RAISE_LDS((diff_attn_dkv_k<NP, DP, 4, false, true>), 2 * R + C + ST);
      diff_attn_dkv_k<NP, DP, 4, false, true><<<grid, 256, 2 * R + C + ST, s>>>(p);
    } else {
      HITADV_RAISE_LDS((diff_attn_dkv_k<NP, DP, 4, true, true>), 2 * (R + C) + ST);
      diff_attn_dkv_k<NP, DP, 4, true, true><<<grid, 256, 2 * (R + C) + ST, s>>>(p);
    }
    HITADV_LAUNCH_CHECK();
  }
  if (dlam) {
    diff_attn_dlam_k<<<p.lam_n, 1024, 0, s>>>(p.r + (int64_t)p.B * p.H * p.Nq, p.B, p.H, p.Nq, p.lam_n, dlam);
    HITADV_LAUNCH_CHECK();
  }
  return 0;
}

static bool da_shape_ok(int dtype, int64_t B, int64_t Nq, int64_t Nk, int64_t H, int64_t Hkv, int64_t D) {
  if (dtype < 0 || dtype > 2 || B < 1 || Nq < 1 || Nk < 1 || H < 1 || Hkv < 1 || H % Hkv || D < 8 || D > 64 || D % 8) return false;
  const int64_t G = H / Hkv, rows = Nq * G;
  // rows and keys are 32-bit indexes (with room for a tile beyond the end), the division by G is exact below 2^32 / G, and the grid's
  // second and third extents are 16-bit; dlam's kernel has a workgroup of 1024 a head (2^32 threads are too many for a dimension)
  return rows <= 2000000 && (rows + 256) * G < (1ll << 32) && Nk <= 2000000 && B * Hkv < (1ll << 31) && B * Hkv <= 65535 && H < (1 << 22) &&
         B * H * Nq < (1ll << 40);
}
static void da_fill(DaP &p, int B, int Nq, int Nk, int H, int Hkv, int D, int lam_n, int causal, float scale, const int64_t *st) {
  p.B = B; p.Nq = Nq; p.Nk = Nk; p.H = H; p.Hkv = Hkv; p.D = D; p.G = H / Hkv; p.lam_n = lam_n; p.causal = causal;
  p.rows = Nq * p.G;
  p.g_magic = p.G > 1 ? (uint32_t)(((1ull << 32) + p.G - 1) / p.G) : 0u;
  p.scale = scale;
  // a positive factor: the maximum of the scaled scores is the scaled maximum
  p.scale2 = scale == 0.f ? 1.f : (scale < 0.f ? -scale : scale) * DA_LOG2E;
  p.s_and = scale == 0.f ? 0u : ~0u;
  p.s_xor = scale < 0.f ? 0x80008000u : 0u;
  p.q_b = st[0]; p.q_n = st[1]; p.q_h = st[2]; p.q_m = st[3];
  p.k_b = st[4]; p.k_n = st[5]; p.k_h = st[6]; p.k_m = st[7];
  p.v_b = st[8]; p.v_n = st[9]; p.v_h = st[10];
}
static bool da_strides_ok(int dtype, const void *q, const void *k, const void *v, const int64_t *st) {
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) return false;
  for (int i = 0; i < 11; ++i)
    if (st[i] < 0 || st[i] % (dtype == 0 ? 4 : 8)) return false;
  // a tile's 32 rows and its two maps are addressed with 32 bits
  return st[1] < DA_STRIDE && st[3] < DA_STRIDE && st[5] < DA_STRIDE && st[7] < DA_STRIDE && st[9] < DA_STRIDE;
}

}  // namespace hitadv

using namespace hitadv;

extern "C" int hitadv_diff_attention_supported(int dtype, int64_t B, int64_t Nq, int64_t Nk, int64_t H, int64_t Hkv, int64_t D) {
  return da_shape_ok(dtype, B, Nq, Nk, H, Hkv, D) ? 1 : 0;
}

extern "C" int64_t hitadv_diff_attention_scratch_floats(int B, int Nq, int Nk, int H, int Hkv, int D) {
  if (!da_shape_ok(0, B, Nq, Nk, H, Hkv, D)) return 0;
  const DaPlan pl = da_plan(B, Nq, Nk, H, Hkv);
  return pl.splits > 1 ? (int64_t)pl.splits * B * H * Nq * (4 * D + 4) : 0;
}

extern "C" int hitadv_diff_attention_fwd(int dtype, const void *q, const void *k, const void *v, const float *lam, int lam_n, const int32_t *lengths,
                                         const int64_t *strides, int B, int Nq, int Nk, int H, int Hkv, int D, int causal, float scale, void *out,
                                         float *stats, float *scratch, void *stream) {
  if (!q || !k || !v || !lam || !strides || !out || !da_shape_ok(dtype, B, Nq, Nk, H, Hkv, D) || (lam_n != 1 && lam_n != H) ||
      !da_strides_ok(dtype, q, k, v, strides) || ((uintptr_t)out & 15))
    return HITADV_E_ARG;
  DaP p = {};
  da_fill(p, B, Nq, Nk, H, Hkv, D, lam_n, causal != 0, scale, strides);
  const DaPlan pl = da_plan(B, Nq, Nk, H, Hkv);
  if (pl.splits > 1 && (!scratch || ((uintptr_t)scratch & 15))) return HITADV_E_ARG;
  p.q = q; p.k = k; p.v = v; p.lam = lam; p.lengths = lengths; p.out = out; p.stats = stats;
  p.chunk = pl.chunk;
  p.splits = pl.splits;
  p.part_ml = scratch;
  p.part_o = scratch ? scratch + (int64_t)pl.splits * B * H * Nq * 4 : nullptr;
  hipStream_t s = (hipStream_t)stream;
  if (D <= 32) return dtype == 0 ? da_launch_fwd<3, 32>(p, pl, s) : dtype == 1 ? da_launch_fwd<1, 32>(p, pl, s) : da_launch_fwd<2, 32>(p, pl, s);
  return dtype == 0 ? da_launch_fwd<3, 64>(p, pl, s) : dtype == 1 ? da_launch_fwd<1, 64>(p, pl, s) : da_launch_fwd<2, 64>(p, pl, s);
}

extern "C" int hitadv_diff_attention_bwd(int dtype, const void *q, const void *k, const void *v, const float *lam, int lam_n, const int32_t *lengths,
                                         const int64_t *strides, const void *dout, const float *stats, int B, int Nq, int Nk, int H, int Hkv, int D,
                                         int causal, float scale, float *r, void *dq, void *dk, void *dv, float *dlam, void *stream) {
  if (!q || !k || !v || !lam || !strides || !dout || !stats || !r || !dq || !dk != !dv || !da_shape_ok(dtype, B, Nq, Nk, H, Hkv, D) ||
      (lam_n != 1 && lam_n != H) || !da_strides_ok(dtype, q, k, v, strides) ||
      (((uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15))
    return HITADV_E_ARG;
  DaP p = {};
  da_fill(p, B, Nq, Nk, H, Hkv, D, lam_n, causal != 0, scale, strides);
  p.q = q; p.k = k; p.v = v; p.lam = lam; p.lengths = lengths; p.dout = dout; p.stats = const_cast<float *>(stats); p.r = r;
  p.dq = dq; p.dk = dk; p.dv = dv;
  hipStream_t s = (hipStream_t)stream;
  if (D <= 32) return dtype == 0 ? da_launch_bwd<3, 32>(p, dlam, s) : dtype == 1 ? da_launch_bwd<1, 32>(p, dlam, s) : da_launch_bwd<2, 32>(p, dlam, s);
  return dtype == 0 ? da_launch_bwd<3, 64>(p, dlam, s) : dtype == 1 ? da_launch_bwd<1, 64>(p, dlam, s) : da_launch_bwd<2, 64>(p, dlam, s);
}
