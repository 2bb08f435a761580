// Shared parts of the gated delta rule's kernels (ssm_delta.hip, ssm_delta_bwd.hip).
//
// Per batch row and value head, with the state S (Dk, Dv):
//   S' = e^{g_t} S_{t-1},  u_t = beta_t (v_t - S'^T k_t),  S_t = S' + k_t u_t^T,  o_t = scale S_t^T q_t.
// Over a chunk of kC tokens with G = cumsum(g) and the entering state S0 this is
//   X = V - e^G K S0,  R = beta X,  U = T R,  T = (I + strictly lower(beta_i e^{G_i - G_j} k_i.k_j))^-1
//   O = scale e^G Q S0 + P U,  P_ij = scale e^{G_i - G_j} q_i.k_j (j <= i),  S1 = e^{G_C} S0 + K^T (e^{G_C - G} U)
// so that everything but the factors is products of 64-row tiles, which run on the matrix cores.
// Every exponent is a difference of later minus earlier cumulative decays, taken in float64.
//
// Products take bf16 operands and accumulate in float32.  A float32 operand is held as the sum of NS
// bf16 parts (x = p0 + p1 + ..., each the rounding of what the earlier ones leave), and a product of
// parts i and j is formed where i + j < the larger count: bf16 inputs are one part and exact, fp16
// inputs two and exact.  With two parts an operand is off by 2^-18 of itself at most, with three by
// 2^-26; one part alone (2^-9) would show in the float32 state and in dg.
#pragma once

#include "ssm_device.hpp"
#include "ssm_internal.hpp"
#include "ssm_wave.hpp"

namespace ssm {

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr int kC = kDeltaChunk;   // tokens per chunk
constexpr int kCP = kC + 8;       // LDS row of kC bf16, padded by 16 bytes: rows on distinct bank groups
constexpr int kDT = 256;          // threads of a workgroup: wavefront w owns token rows 16 w .. 16 w + 15
constexpr int kFrag = kC * kC;    // elements of one part of a 64 x 64 matrix stored as operand fragments

// Parts of an input of type IT, and of float32 intermediates beside it.
template <typename IT> struct DParts;
template <> struct DParts<bf16_t> { static constexpr int in = 1, mid = 2; };
template <> struct DParts<f16_t> { static constexpr int in = 2, mid = 2; };
template <> struct DParts<float> { static constexpr int in = 3, mid = 3; };

template <int N, typename F, typename V>
__device__ __forceinline__ void split_parts(F x, V (&p)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    p[n] = __builtin_convertvector(x, V);
    if (n + 1 < N) x -= __builtin_convertvector(p[n], F);
  }
}

// acc += a b over one step of 32: lane l holds row (a) or column (b) l % 16, elements 8 (l / 16) + j
// of the step; of the 16 x 16 result it holds column l % 16, rows 4 (l / 16) + i.
template <int NA, int NB>
__device__ __forceinline__ f4 mma(const bf8 (&a)[NA], const bf8 (&b)[NB], f4 acc) {
  constexpr int M = NA > NB ? NA : NB;
#pragma unroll
  for (int s = M - 1; s >= 0; --s)  // the smallest products first
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], acc, 0, 0, 0);
  return acc;
}

// Operand fragment of one step from an LDS matrix whose rows are the operand's rows / columns.
template <int N, int PITCH>
__device__ __forceinline__ void lds_frag(const __bf16 *m, int part, int row, int col, bf8 (&f)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) f[n] = *(const bf8 *)(m + n * part + row * PITCH + col);
}
// The same from a matrix stored the other way round (rows are the contraction index): the transposing
// LDS read gives lane l of 16 the column l of the 4 rows whose 8-byte pieces the 16 lanes address.
template <int N, int PITCH>
__device__ __forceinline__ void lds_frag_t(const __bf16 *m, int part, int k0, int col0, int lane, bf8 (&f)[N]) {
  const int r = k0 + (lane / 16) * 8 + (lane % 16) / 4, c = col0 + (lane % 4) * 4;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    typedef __attribute__((address_space(3))) s4 *P;
    const __bf16 *p = m + n * part + r * PITCH + c;
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)p);
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p + 4 * PITCH));
    f[n] = __builtin_bit_cast(bf8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// Eight consecutive elements of a row as floats, 0 from `have` on; vec: the row is 16-byte aligned
// and `have` is a multiple of 8.
template <typename IT>
__device__ __forceinline__ f8 row8(const IT *p, int have, bool vec) {
  f8 x = 0;
  if (vec) {
    if (have > 0) {
      if constexpr (sizeof(IT) == 4) {
        const f4 a = *(const f4 *)p, b = *(const f4 *)(p + 4);
        x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
      } else {
        struct alignas(16) Pack { IT e[8]; };
        const Pack k = *(const Pack *)p;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = Conv<IT>::load(&k.e[j]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < have) x[j] = Conv<IT>::load(p + j);
  }
  return x;
}
// The same as operand parts; bf16 rows need no conversion.
template <typename IT, int N>
__device__ __forceinline__ void row_frag(const IT *p, int have, bool vec, bf8 (&f)[N]) {
  if constexpr (sizeof(IT) == 2 && N == 1) {
    if (vec) {
      f[0] = have > 0 ? *(const bf8 *)p : (bf8)(__bf16)0.0f;
      return;
    }
  }
  split_parts<N>(row8<IT>(p, have, vec), f);
}

// Element `at` of a tensor that is float32 or of type IT.
template <typename IT>
__device__ __forceinline__ float load_either(const void *t, bool f32, int64_t at) {
  return f32 ? ((const float *)t)[at] : Conv<IT>::load((const IT *)t + at);
}
template <typename IT>
__device__ __forceinline__ void store_either(void *t, bool f32, int64_t at, float v) {
  if (f32) ((float *)t)[at] = v;
  else Conv<IT>::store((IT *)t + at, v);
}

__device__ __forceinline__ float fexp(float x) { return fast_exp2(x * LOG2E); }

// Head, chunk-independent addressing.  Workgroup l runs on XCD l % 8: the NV column tiles of a head
// read the same keys, queries and factors, so they are placed 8 apart where the heads divide evenly.
__device__ __forceinline__ void delta_tile(int nv, int heads, int &bh, int &vt) {
  const int x = blockIdx.x;
  if (heads % 8 == 0) {
    bh = x % 8 + 8 * (x / 8 / nv);
    vt = x / 8 % nv;
  } else {
    bh = x / nv;
    vt = x % nv;
  }
}

// Row factors of a chunk, kDeltaRows floats: [0] a = |k|^-1 e^G, [1] beta, [2] c = |k|^-1 e^{G_C - G},
// [3] d = scale |q|^-1 e^G, [4] |k|^-1, [5] scale |q|^-1 (the norms are 1 without qk_norm), [6..7] G as float64.
__device__ __forceinline__ const float *delta_rows(const DeltaParams &p, int64_t ch) { return p.rows + ch * kDeltaRows; }
__device__ __forceinline__ f4 row4(const float *rows, int which, int r) { return *(const f4 *)(rows + which * kC + r); }
__device__ __forceinline__ float chunk_decay(const float *rows) { return fexp((float)((const double *)(rows + 6 * kC))[kC - 1]); }

}  // namespace ssm
