// Shared parts of the gated delta rule's kernels (ssm_delta.hip, ssm_delta_bwd.hip).
//
// Per batch row and value head, with the state S (Dk, Dv):
//   S' = e^{g_t} S_{t-1},  u_t = beta_t (v_t - S'^T k_t),  S_t = S' + k_t u_t^T,  o_t = scale S_t^T q_t.
// Over a chunk of kC tokens with G = cumsum(g) and the entering state S0 this is
//   X = V - e^G K S0,  Y = T X,  U = beta Y,  T = (I + strictly lower(e^{G_i - G_j} k_i.k_j beta_j))^-1
//   O = scale e^G Q S0 + P U,  P_ij = scale e^{G_i - G_j} q_i.k_j (j <= i),  S1 = e^{G_C} S0 + K^T (e^{G_C - G} U)
// so that everything but the factors is products of 64-row tiles, which run on the matrix cores.
// Every exponent is a difference of later minus earlier cumulative decays, which are summed in float64 and
// kept as two floats, so that the difference is off by its own rounding only.
//
// Products take bf16 operands and accumulate in float32.  A float32 operand is held as the sum of
// bf16 parts (x = p0 + p1 + ..., each the rounding of what the earlier ones leave: 8 significant bits
// each, so one part is off by 2^-8 of the operand at most, two by 2^-16, three by 2^-24), and a product
// of parts i and j is formed where i + j is below the count of parts kept.  bf16 inputs are one part and
// exact, fp16 inputs two and exact, float32 inputs three.  Every intermediate has three, whatever the inputs'
// type: the state, its gradient and dg are float32 outputs, and where the terms of an output of 16 bits
// cancel, two parts would leave more than its rounding.
//
// Where the contraction index is stored.  A lane's 8 elements of a fragment of 32 are, in this order,
// 4 kg + 0..3 and 16 + 4 kg + 0..3 (kg = lane / 16): the order in which lanes hold the rows of two
// 16 x 16 results, so that results and transposing LDS reads become operands without a permutation.
#pragma once

#include <type_traits>

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
constexpr int kDT = 256;          // four wavefronts: wavefront w owns tokens 16 w .. 16 w + 15
// The walks and the gradient kernel have one workgroup's two wavefronts on a SIMD: the scheduler may use the
// registers that more would need.
#define SSM_TWO_WAVES __attribute__((amdgpu_waves_per_eu(2, 2)))
constexpr int kFrag = kC * kC;    // elements of one part of a 64 x 64 matrix stored as operand fragments

// Parts of an input of type IT and of the float32 intermediates beside it.
template <typename IT> struct DParts;
template <> struct DParts<bf16_t> { static constexpr int in = 1, mid = 3; };
template <> struct DParts<f16_t> { static constexpr int in = 2, mid = 3; };
template <> struct DParts<float> { static constexpr int in = 3, mid = 3; };

template <int N, typename F, typename V>
__device__ __forceinline__ void split_parts(F x, V (&p)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    p[n] = __builtin_convertvector(x, V);
    if (n + 1 < N) x -= __builtin_convertvector(p[n], F);
  }
}

// acc += a b over one step of 32: lane l holds row (a) or column (b) l % 16, of the 16 x 16 result
// column l % 16, rows 4 (l / 16) + i.  The first M parts are kept, the smallest products come first.
template <int M, int NA, int NB>
__device__ __forceinline__ f4 mma(const bf8 (&a)[NA], const bf8 (&b)[NB], f4 acc) {
#pragma unroll
  for (int s = M - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], acc, 0, 0, 0);
  return acc;
}

// The transposing LDS read: lane l of 16 gets column l of the 4 rows whose 8-byte pieces the 16 lanes address.
__device__ __forceinline__ bf8 read_tr(const __bf16 *lo, const __bf16 *hi) {
  typedef __attribute__((address_space(3))) s4 *P;
  const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)lo), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)hi);
  return __builtin_bit_cast(bf8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// An intermediate of R rows (keys or tokens, the next product's contraction index) by 16 columns of v in
// LDS, N parts.  A row is four 8-byte pieces; rows 8..15 of every 16 swap its halves, so that neither the
// writes (16 rows by two pieces in 32 lanes) nor the reads (8 rows by four) meet twice in a bank.
template <int N, int R> struct VTile {
  __bf16 e[N][R * 16];
  // x: row `row`, columns 4 kg + i
  __device__ __forceinline__ void put(int row, int kg, f4 x) {
    bf4 p[N];
    split_parts<N>(x, p);
    put_parts(row, kg, p);
  }
  __device__ __forceinline__ void put_parts(int row, int kg, const bf4 (&p)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) *(bf4 *)&e[n][row * 16 + ((kg ^ ((row >> 2) & 2)) * 4)] = p[n];
  }
  // the value of (row, columns 4 kg + i): the parts' sum, exact with three
  __device__ __forceinline__ f4 whole(int row, int kg) const {
    f4 x = 0;
#pragma unroll
    for (int n = N - 1; n >= 0; --n) x += __builtin_convertvector(*(const bf4 *)&e[n][row * 16 + ((kg ^ ((row >> 2) & 2)) * 4)], f4);
    return x;
  }
  // whole(), but infinite where the value is (its other parts are inf - inf)
  __device__ __forceinline__ f4 value(int row, int kg) const {
    f4 x = whole(row, kg);
    const f4 first = __builtin_convertvector(*(const bf4 *)&e[0][row * 16 + ((kg ^ ((row >> 2) & 2)) * 4)], f4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fabsf(first[i]) < INFINITY ? x[i] : first[i];
    return x;
  }
  // operand of rows 32 s .. 32 s + 31: lane = column of v
  template <int M>
  __device__ __forceinline__ void get(int s, int lane, bf8 (&f)[M]) const {  // the first M parts
    const int row = 32 * s + 4 * (lane / 16) + (lane % 16) / 4, at = row * 16 + ((lane % 4) ^ ((row >> 2) & 2)) * 4;
#pragma unroll
    for (int n = 0; n < M; ++n) f[n] = read_tr(&e[n][at], &e[n][at + 256]);
  }
};

// Products formed of NA by NB parts when the first M are kept.
constexpr int products(int m, int na, int nb) {
  int n = 0;
  for (int i = 0; i < na; ++i)
    for (int j = 0; j < nb; ++j) n += i + j < m;
  return n;
}
// Orders a block of READS LDS reads and MMAS products: AHEAD reads first, then products and reads in turn, so that
// a product's operands are read AHEAD reads before it.
template <int READS, int MMAS, int AHEAD>
__device__ __forceinline__ void read_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < MMAS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, (READS + MMAS - 1) / MMAS, 0);
  }
}

// Fragment `at` (of 64 lanes x 8) of an array of N parts, `part` elements each.
template <int N>
__device__ __forceinline__ void load_frag(const __bf16 *m, int64_t part, int at, int lane, bf8 (&f)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) f[n] = *(const bf8 *)(m + n * part + at * 512 + (unsigned)(lane * 8));
}

// The products of a chunk's triangular matrices run over steps of 32 tokens, with the zeros beyond the diagonal,
// and a zero times an infinity or NaN is NaN: it would reach tokens that the recurrence keeps free of it.  It
// shows in the wavefront's own results, so these are looked at, and only where one is not finite that was before
// the product (with the state infinite or NaN, all are, from chunk to chunk) are they formed again from the tokens
// that belong to them.
template <int N> __device__ __forceinline__ bool not_finite(const f4 (&x)[N]) {
  float s = 0;
#pragma unroll
  for (int n = 0; n < N; ++n) s += (fabsf(x[n][0]) + fabsf(x[n][1])) + (fabsf(x[n][2]) + fabsf(x[n][3]));
  return __builtin_amdgcn_ballot_w64(!(s < INFINITY)) != 0;
}
template <int N> __device__ __forceinline__ bool not_finite_of(const f4 (&x)[N], const f4 (&before)[N]) {
  bool b = false;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) b |= fabsf(before[n][i]) < INFINITY && !(fabsf(x[n][i]) < INFINITY);
  return __builtin_amdgcn_ballot_w64(b) != 0;
}
// acc + sum over the tokens j, lo <= j < hi, of m[tok][j] x_j (columns 4 kg + i): m as fragments of token rows.
template <int N, typename TILE>
__device__ __forceinline__ f4 row_times(const __bf16 *m, int tok, int lo, int hi, const TILE &x, int kg, f4 acc) {
#pragma unroll 1
  for (int j = lo; j < hi; ++j) {
    const __bf16 *e = m + (2 * (tok / 16) + j / 32) * 512 + (j % 16 / 4 * 16 + tok % 16) * 8 + j % 32 / 16 * 4 + j % 4;
    float c = 0;
#pragma unroll
    for (int n = N - 1; n >= 0; --n) c += (float)e[n * kFrag];
    acc += c * x.value(j, kg);
  }
  return acc;
}

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x / 64); }

// Four consecutive elements of a row as words.  vec: rows are whole words of 4 elements; the words are then
// read whether `have` > 0 or not (from `safe`, any readable element), so that nothing waits for them before
// their use, which takes 0 in their place.  Otherwise the elements from `have` on are 0.
template <typename IT> using Raw4 = unsigned __attribute__((ext_vector_type(sizeof(IT))));
template <typename IT> struct alignas(4 * sizeof(IT)) Four { IT e[4]; };
template <typename IT>
__device__ __forceinline__ Raw4<IT> load4(const IT *p, const IT *safe, int have, bool vec) {
  if (vec) return *(const Raw4<IT> *)(have > 0 ? p : safe);
  Four<IT> x{};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < have) x.e[j] = p[j];
  return __builtin_bit_cast(Raw4<IT>, x);
}
template <typename IT>
__device__ __forceinline__ f4 to_f4(Raw4<IT> w, bool live) {
  const Four<IT> x = __builtin_bit_cast(Four<IT>, live ? w : (Raw4<IT>)0u);
  f4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = Conv<IT>::load(&x.e[j]);
  return r;
}
// The same as operand parts.
template <typename IT, int N>
__device__ __forceinline__ void to_parts(Raw4<IT> x, bool live, bf4 (&p)[N]) {
  if constexpr (std::is_same_v<IT, bf16_t> && N == 1) p[0] = __builtin_bit_cast(bf4, live ? x : (Raw4<IT>)0u);
  else split_parts<N>(to_f4<IT>(x, live), p);
}
template <typename IT>
__device__ __forceinline__ void store4(IT *p, f4 x, int have, bool vec) {
  Four<IT> r;
  if constexpr (std::is_same_v<IT, bf16_t>) {
    r = __builtin_bit_cast(Four<IT>, __builtin_convertvector(x, bf4));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) Conv<IT>::store(&r.e[j], x[j]);
  }
  if (vec) {
    if (have > 0) *(Raw4<IT> *)p = __builtin_bit_cast(Raw4<IT>, r);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < have) p[j] = r.e[j];
  }
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

// Sum over the four lanes of a column (l % 16).
__device__ __forceinline__ float kg_sum(float v) {
  const unsigned a = __builtin_bit_cast(unsigned, v);
  const auto x = __builtin_amdgcn_permlane16_swap(a, a, false, false);  // even rows, odd rows
  const unsigned x0 = x[0], x1 = x[1];
  const unsigned b = __builtin_bit_cast(unsigned, __builtin_bit_cast(float, x0) + __builtin_bit_cast(float, x1));
  const auto y = __builtin_amdgcn_permlane32_swap(b, b, false, false);  // lower half, upper half
  const unsigned y0 = y[0], y1 = y[1];
  return __builtin_bit_cast(float, y0) + __builtin_bit_cast(float, y1);
}
// Inclusive sums over the wavefront's lanes.
template <int CTRL, int ROWS>
__device__ __forceinline__ double scan_part(double v) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)u, CTRL, ROWS, 0xF, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(u >> 32), CTRL, ROWS, 0xF, false);
  return v + __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double wave_scan_f64(double v) {
  v = scan_part<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
  v = scan_part<0x112, 0xF>(v);
  v = scan_part<0x114, 0xF>(v);
  v = scan_part<0x118, 0xF>(v);
  v = scan_part<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  return scan_part<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}

__device__ __forceinline__ float fexp(float x) { return fast_exp2(x * LOG2E); }

// Head and first column tile of a walk's workgroup, which takes `per` of them.  Workgroup l runs on XCD l % 8: the
// workgroups of a head read the same keys, queries and factors, so they are placed 8 apart where the heads
// divide evenly.
__device__ __forceinline__ void delta_tile(const DeltaParams &p, int per, int &bh, int &vt) {
  const int x = (int)p.first + (int)blockIdx.x, heads = (int)p.B * p.H, nv = (p.VT + per - 1) / per;
  if (heads % 8 == 0) {
    bh = x % 8 + 8 * (x / 8 / nv);
    vt = x / 8 % nv * per;
  } else {
    bh = x / nv;
    vt = x % nv * per;
  }
}

// Row factors of a chunk, kDeltaRows floats: per token a = |k|^-1 e^G, beta, c = |k|^-1 e^{G_C - G} and
// e^{G_C}, which the chain takes in one read; then [4] |k|^-1, [5] scale |q|^-1 (the norms are 1 without
// qk_norm), [6] + [7] G as the sum of two floats, [8] d = scale |q|^-1 e^G; for the backward [9] |q|^-1.
__device__ __forceinline__ const float *delta_rows(const DeltaParams &p, int64_t ch) { return p.rows + ch * kDeltaRows; }
__device__ __forceinline__ f4 token_row(const float *rows, int tok) { return *(const f4 *)(rows + (unsigned)(4 * tok)); }

// Arrays of operand fragments.  Per chunk and key head, in DParts::in parts of 64 DK: the rows of K and Q
// (token tile w, step s of keys: fragment w DK/32 + s) and their columns (key tile t, step s of tokens:
// fragment 2 t + s).  Per chunk and head, of kFrag each: T and P or their transposes (token tile w, step s:
// fragment 2 w + s).
template <int DK, int N>
__device__ __forceinline__ const __bf16 *key_frags(const void *f, int64_t kch) { return (const __bf16 *)f + kch * N * kC * DK; }

// The states and the values by chunk, head and 16 columns of v: element (row, column)
// (rows are added as 32-bit lane offsets).
__device__ __forceinline__ float *state_of(float *m, const DeltaParams &p, int64_t ch, int vt) {
  return m + (ch * p.VT + vt) * p.Dkp * 16;
}
__device__ __forceinline__ float *value_of(float *m, const DeltaParams &p, int64_t ch, int vt) {
  return m + (ch * p.VT + vt) * kC * 16;
}

// Whether a wavefront of the walks takes two tiles of 16 columns of v.  Every read of memory takes a compute
// unit's address unit 16 cycles, whatever its width, and the fragments' reads are the most of them; two
// tiles share them.  While every tile can have a compute unit of its own, the pair only leaves some without
// work.  Forward + backward of H16 L1024 with values of 64 columns, us, single tiles and pairs at 256 and at 384
// tiles: bf16 keys of 64 131 153, 214 196; of 128 190 213, 312 292; fp16 143 172, 245 229; 255 285, 450 400;
// float32 189 212, 331 299; 356 381, 612 534.  Either direction alone decides alike.  With one tile a head the
// pair is half empty and 0 to 4 % longer.
inline bool delta_pairs(const DeltaParams &p) { return p.B * p.H * p.VT > 256; }
// launch(p, grid) over a walk's workgroups of `per` column tiles each, as many at once as a grid row takes.
template <typename F>
static void delta_walk(const DeltaParams &p, int per, F launch) {
  const int64_t all = p.B * p.H * ((p.VT + per - 1) / per), most = kGridThreads / (2 * kDT);
  DeltaParams part = p;
  for (; part.first < all; part.first += most) launch(part, dim3((unsigned)(all - part.first < most ? all - part.first : most)));
}

}  // namespace ssm
