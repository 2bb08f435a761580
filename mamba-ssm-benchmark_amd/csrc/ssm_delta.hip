// Gated delta rule, chunked forward (the mathematics and the operand layouts: ssm_delta.hpp).
//
//   k_delta_prep  one workgroup per (batch row, value head, chunk): decays, norms, T, P and the keys' and
//                 queries' operand fragments
//   k_delta_fwd   one workgroup per (batch row, value head, 16 columns of v): the columns of S do not
//                 mix, so each walks the chunks with its own columns in registers
#include "ssm_delta.hpp"

namespace ssm {

// c(16 x 16) += a b from float32 LDS matrices: a's rows and b's columns of 16.
template <int PA, int PB>
__device__ __forceinline__ f4 mma_f32(const float *a, const float *b, int lane, f4 c) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[(lane % 16) * PA + 4 * k + lane / 16],
                                             b[(4 * k + lane / 16) * PB + lane % 16], c, 0, 0, 0);
  return c;
}
// The same where a (la) or b (lb) is a lower triangular block: where a result is not finite, all are formed again
// without the zeros above the diagonals (not_finite(), ssm_delta.hpp).
template <int PA, int PB>
__device__ __forceinline__ f4 mma_lower(const float *a, bool la, const float *b, bool lb, int lane, f4 c) {
  const f4 r[1] = {mma_f32<PA, PB>(a, b, lane, c)};
  if (__builtin_expect(!not_finite(r), 1)) return r[0];
  const int col = lane % 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 4 * (lane / 16) + i;
#pragma unroll 1
    for (int k = lb ? col : 0; k <= (la ? row : 15); ++k) c[i] = fmaf(a[row * PA + k], b[k * PB + col], c[i]);
  }
  return c;
}
template <int PITCH>
__device__ __forceinline__ void put16(float *m, int lane, f4 c, float sign) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m[(4 * (lane / 16) + i) * PITCH + lane % 16] = sign * c[i];
}

// Whether any of 8 elements is infinite or NaN: an exponent of all ones carries into the sign's place.
typedef unsigned u4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ bool odd_halves(bf8 x) {
  const u4 t = (__builtin_bit_cast(u4, x) & 0x7f807f80u) + 0x00800080u;
  return ((t[0] | t[1]) | (t[2] | t[3])) & 0x80008000u;
}
__device__ __forceinline__ bf8 without_odd(bf8 x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fabsf((float)x[i]) < INFINITY ? x[i] : (__bf16)0.0f;
  return x;
}

// Writes T - I and P as operand fragments, the row factors, and, for the first of the value heads that
// share a key head, the fragments of K and Q.  BWD: the transposes of T = (I + strictly lower(beta_i
// e^{G_i - G_j} k_i.k_j))^-1, which the gradient takes, and of P.
// The backward's columns of K and Q have 0 in the place of an infinity or NaN: J K, J^T Q, H K and H^T K take them
// with zeros beyond the diagonals, and what the tokens concerned get of them is infinite or NaN without it, through
// U, dR and J's diagonal.
// T is inverted in float32: the four 16 x 16 diagonal blocks by substitution, one wavefront each, the
// rest by T10 = -T11 (L10 T00) for blocks of 16, then of 32 rows.
// Chunks are independent, so everything that does not hang on the state is done here, once for all columns
// of v.  Latency bounds a workgroup (two waits for memory, a chain of five barriers: 9 us alone), hence three
// to a compute unit for bf16 rows.  B4 L4096 H16 Hk8 128 x 128 bf16: 89 us for 261 MB written; 512 threads of
// the first version's occupancy (two workgroups, all 16 tiles of L and P computed) took 113.
template <typename IT, int DK, bool BWD>
__global__ void __launch_bounds__(kDT, 4 - DParts<IT>::in) k_delta_prep(const DeltaParams p) {
  constexpr int NK = DParts<IT>::in, NM = DParts<IT>::mid, KS = DK / 32, FP = kC + 4, YP = 32 + 4;
  constexpr int kRowsOf = 4 * KS * 64 * 8;  // elements of one part of K or Q
  __shared__ __align__(16) __bf16 Kf[NK][kRowsOf], Qf[BWD ? NK : 1][BWD ? kRowsOf : 8];  // as in memory
  __shared__ __align__(16) float Lm[kC][FP];
  __shared__ float Gh[kC], Gl[kC], fk[kC], fq[kC], fu[BWD ? kC : 1], bs[kC];  // G as the sum of two floats
  static_assert(sizeof(Kf) >= sizeof(float) * 32 * YP, "the inversion's scratch");
  float *const Yr = (float *)&Kf[0][0];                     // ... lies where the keys were
  const int tid = threadIdx.x, lane = tid % 64, w = wave_id(), r16 = lane % 16, kg = lane / 16, own = 16 * w + r16;
  const int64_t ch = blockIdx.x;
  const int heads = (int)p.B * p.H, group = p.H / p.Hk, bh = (int)(ch % heads), c = (int)(ch / heads), b = bh / p.H, h = bh % p.H, hk = h / group;
  const int64_t t0 = (int64_t)c * kC, t = t0 + own, kch = ((int64_t)c * p.B + b) * p.Hk + hk;
  const IT *kp = (const IT *)p.k.p + b * p.k.s0 + t * p.k.s1 + hk * p.k.s2;
  const IT *qp = (const IT *)p.q.p + b * p.q.s0 + t * p.q.s1 + hk * p.q.s2;
  const int have = t < p.L ? p.Dk : 0;
  const bool first = h % group == 0;
  float head_in = 0;  // wavefront 0: g, 1: beta, of token `lane`
  if (w < 2 && t0 + lane < p.L)
    head_in = w ? load_either<IT>(p.beta.p, p.beta32, b * p.beta.s0 + (t0 + lane) * p.beta.s1 + h * p.beta.s2)
                : ((const float *)p.g.p)[b * p.g.s0 + (t0 + lane) * p.g.s1 + h * p.g.s2];
  bf8 K[KS][NK], Q[KS][NK];
  Raw4<IT> x[KS][4];
  const IT *const ks = (const IT *)p.k.p, *const qs = (const IT *)p.q.p;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int e = 32 * s + 4 * kg;
    x[s][0] = load4(kp + e, ks, have - e, p.vk);
    x[s][1] = load4(kp + e + 16, ks, have - e - 16, p.vk);
    x[s][2] = load4(qp + e, qs, have - e, p.vq);
    x[s][3] = load4(qp + e + 16, qs, have - e - 16, p.vq);
  }
  if (w == 0) {
    double G = (double)head_in;
    if (G < -1e4) G = -1e4;  // e^-1e4 is 0 in either width, and -inf would make inf - inf of the differences
    G = wave_scan_f64(G);
    Gh[lane] = (float)G;
    Gl[lane] = (float)(G - (double)(float)G);
  } else if (w == 1) {
    bs[lane] = head_in;
  }
  float kk = 0, qq = 0;  // sums of squares
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int e = 32 * s + 4 * kg;
    bf4 a[4][NK];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool live = have - e - 16 * (i % 2) > 0;
      to_parts<IT, NK>(x[s][i], live, a[i]);
      const f4 f = to_f4<IT>(x[s][i], live);
#pragma unroll
      for (int j = 0; j < 4; ++j) (i < 2 ? kk : qq) = fmaf(f[j], f[j], i < 2 ? kk : qq);
    }
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      K[s][n] = __builtin_shufflevector(a[0][n], a[1][n], 0, 1, 2, 3, 4, 5, 6, 7);
      Q[s][n] = __builtin_shufflevector(a[2][n], a[3][n], 0, 1, 2, 3, 4, 5, 6, 7);
      *(bf8 *)&Kf[n][((w * KS + s) * 64 + lane) * 8] = K[s][n];
      if (BWD) *(bf8 *)&Qf[n][((w * KS + s) * 64 + lane) * 8] = Q[s][n];
    }
  }
  float nk = 1.0f, nq = p.scale, uq = 1.0f;
  if (p.qk_norm) {
    const float len = sqrtf(kg_sum(qq) + 1e-6f);
    nk = 1.0f / sqrtf(kg_sum(kk) + 1e-6f);
    nq = p.scale / len;
    uq = 1.0f / len;
  }
  if (kg == 0) {
    fk[own] = nk;
    fq[own] = nq;
    if (BWD) fu[own] = uq;
  }
  lds_barrier();
  if (first) {
    __bf16 *const gK = (__bf16 *)p.fK + kch * NK * kC * DK, *const gQ = (__bf16 *)p.fQ + kch * NK * kC * DK;
    __bf16 *const gKt = (__bf16 *)p.fKt + kch * NK * kC * DK, *const gQt = BWD ? (__bf16 *)p.fQt + kch * NK * kC * DK : nullptr;
#pragma unroll
    for (int n = 0; n < NK; ++n) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        *(bf8 *)(gK + n * kC * DK + (w * KS + s) * 512 + (unsigned)(lane * 8)) = K[s][n];
        *(bf8 *)(gQ + n * kC * DK + (w * KS + s) * 512 + (unsigned)(lane * 8)) = Q[s][n];
      }
#pragma unroll
      for (int y = 0; y < DK / 32; ++y) {  // key tile kt, step s of tokens
        const int kt = w + 4 * (y / 2), s = y % 2, row = 4 * kg + r16 / 4;
        const int lo = ((2 * s * KS + kt / 2) * 64 + (lane % 4) * 16 + row) * 8 + 4 * (kt % 2), hi = lo + KS * 64 * 8;
        bf8 k = read_tr(&Kf[n][lo], &Kf[n][hi]);
        if (BWD) {
          bf8 q = read_tr(&Qf[BWD ? n : 0][lo], &Qf[BWD ? n : 0][hi]);
          if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd_halves(k) | odd_halves(q)) != 0, 0)) {
            k = without_odd(k);
            q = without_odd(q);
          }
          *(bf8 *)(gQt + n * kC * DK + (2 * kt + s) * 512 + (unsigned)(lane * 8)) = q;
        }
        *(bf8 *)(gKt + n * kC * DK + (2 * kt + s) * 512 + (unsigned)(lane * 8)) = k;
      }
    }
  }
  {
    const float gh = Gh[own], gl = Gl[own], be = bs[own];
    f4 P[4];  // P_ij, token tile w as i, j = 16 x + 4 kg + r; BWD: tile w as j, i = 16 x + 4 kg + r
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      f4 l = 0, ln = 0, qk = 0;
      const int at = 16 * x + 4 * kg;
      const f4 xh = *(const f4 *)&Gh[at], xl = *(const f4 *)&Gl[at], xk = *(const f4 *)&fk[at];
      if (x <= w) {  // L, and P but in BWD
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          bf8 A[NK];
          load_frag<NK>(&Kf[0][0], kRowsOf, x * KS + s, lane, A);
          l = mma<NM>(A, K[s], l);
          if (!BWD) qk = mma<NM>(A, Q[s], qk);
        }
        const f4 xb = *(const f4 *)&bs[at];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = fexp((gh - xh[r]) + (gl - xl[r])) * xk[r];
          ln[r] = at + r < own ? nk * e * (BWD ? be : xb[r]) * l[r] : 0.0f;
          if (!BWD) qk[r] = at + r <= own ? nq * e * qk[r] : 0.0f;
        }
      }
      if (BWD && x >= w) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          bf8 A[NK];
          load_frag<NK>(&Qf[0][0], kRowsOf, x * KS + s, lane, A);
          qk = mma<NM>(A, K[s], qk);
        }
        const f4 xq = *(const f4 *)&fq[at];
#pragma unroll
        for (int r = 0; r < 4; ++r) qk[r] = own <= at + r ? fexp((xh[r] - gh) + (xl[r] - gl)) * xq[r] * nk * qk[r] : 0.0f;
      }
      P[x] = qk;
      *(f4 *)&Lm[own][at] = ln;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (BWD ? s >= w / 2 : s <= w / 2) {  // the walks read no other
        bf8 q[NM];
        split_parts<NM>((f8)__builtin_shufflevector(P[2 * s], P[2 * s + 1], 0, 1, 2, 3, 4, 5, 6, 7), q);
#pragma unroll
        for (int n = 0; n < NM; ++n) *(bf8 *)((__bf16 *)p.fP + (ch * NM + n) * kFrag + (2 * w + s) * 512 + (unsigned)(lane * 8)) = q[n];
      }
  }
  if (tid < kC) {
    float *rows = p.rows + ch * kDeltaRows;
    const float gh = Gh[tid], gl = Gl[tid], eG = fexp(gh);
    *(f4 *)(rows + 4 * tid) = f4{fk[tid] * eG, bs[tid], fk[tid] * fexp((Gh[kC - 1] - gh) + (Gl[kC - 1] - gl)), fexp(Gh[kC - 1])};
    rows[4 * kC + tid] = fk[tid];
    rows[5 * kC + tid] = fq[tid];
    rows[6 * kC + tid] = gh;
    rows[7 * kC + tid] = gl;
    rows[8 * kC + tid] = fq[tid] * eG;
    if (BWD) rows[9 * kC + tid] = fu[tid];
  }
  wave_lds_sync();  // the diagonal block is this wavefront's own
  {
    const float *D = &Lm[16 * w][16 * w];
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == r16 ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; ++j) s = fmaf(-D[i * FP + j], x[j], s);
      x[i] = s;
    }
    float sum = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += fabsf(x[i]);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(sum < INFINITY)) != 0, 0)) {  // a column's zeros above the diagonal left out
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = i == r16 ? 1.0f : 0.0f;
#pragma unroll
        for (int j = 0; j < i; ++j) s = j < r16 ? s : fmaf(-D[i * FP + j], x[j], s);
        x[i] = s;
      }
    }
    wave_lds_sync();
    if (kg == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) Lm[16 * w + i][own] = x[i];
    }
  }
  lds_barrier();
  if (w < 2) {
    float *Y = Yr + 16 * w * YP;
    put16<YP>(Y, lane, mma_lower<FP, FP>(&Lm[32 * w + 16][32 * w], false, &Lm[32 * w][32 * w], true, lane, (f4)0.0f), 1.0f);
    wave_lds_sync();
    const f4 t10 = mma_lower<FP, YP>(&Lm[32 * w + 16][32 * w + 16], true, Y, false, lane, (f4)0.0f);
    wave_lds_sync();
    put16<FP>(&Lm[32 * w + 16][32 * w], lane, t10, -1.0f);
  }
  lds_barrier();
  const int r = w / 2, cc = w % 2;
  {
    f4 y = 0;
    for (int k = cc; k < 2; ++k) y = mma_lower<FP, FP>(&Lm[32 + 16 * r][16 * k], false, &Lm[16 * k][16 * cc], k == cc, lane, y);
    put16<YP>(Yr + 16 * r * YP + 16 * cc, lane, y, 1.0f);
  }
  lds_barrier();
  {
    f4 y = 0;
    for (int k = 0; k <= r; ++k) y = mma_lower<FP, YP>(&Lm[32 + 16 * r][32 + 16 * k], k == r, Yr + 16 * k * YP + 16 * cc, false, lane, y);
    put16<FP>(&Lm[32 + 16 * r][16 * cc], lane, y, -1.0f);
  }
  lds_barrier();
#pragma unroll
  for (int s = 0; s < 2; ++s)
    if (BWD ? s >= w / 2 : s <= w / 2) {
      f8 x;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int e = 32 * s + 16 * (j / 4) + 4 * kg + j % 4;
        x[j] = e == own ? 0.0f : BWD ? Lm[e][own] : Lm[own][e];
      }
      bf8 a[NM];
      split_parts<NM>(x, a);
#pragma unroll
      for (int n = 0; n < NM; ++n) *(bf8 *)((__bf16 *)p.fT + (ch * NM + n) * kFrag + (2 * w + s) * 512 + (unsigned)(lane * 8)) = a[n];
    }
}

// The chain from state to state is what bounds the walk (per chunk three products, each split into parts and
// handed on through LDS), so four wavefronts do nothing else and four more take the outputs (Q S, P U and
// the stores) from what the chain leaves in LDS, while it goes on.
// One stream of 16384 tokens, H8 128 x 128 bf16: 350 us, 1.37 us a chunk (320 with two parts of the outputs'
// operands and no search for results that are not finite; 18 more where the outputs' LDS reads do not run ahead of
// their products; four wavefronts for everything, nothing read ahead: 1214).  B4 L4096 H16: 202 us, 283 with the
// states saved: 435 MB of stores, which all workgroups, walking in step, send at the same time.
// Everything that does not hang on the state is read a chunk ahead, into the registers that the chunk has
// just used.  All products are of transposes: rows are 16 columns of v, so a lane holds 4 columns of
// one token or key, and moves them as one word.  A workgroup walks NV tiles of 16 columns.
template <typename IT, int DK, int NV>
__global__ void __launch_bounds__(2 * kDT) SSM_TWO_WAVES k_delta_fwd(const DeltaParams p) {
  constexpr int NK = DParts<IT>::in, NM = DParts<IT>::mid, KS = DK / 32, RT = DK / 64;
  __shared__ __align__(16) VTile<NM, DK> St[NV];
  __shared__ __align__(16) VTile<NM, kC> Xt[NV], Wt[NV], Ut[NV];  // X, c U, U
  const int lane = threadIdx.x % 64, w = wave_id() % 4, r16 = lane % 16, kg = lane / 16;
  int bh, vt;
  delta_tile(p, NV, bh, vt);
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk), v0 = 16 * vt + 4 * kg, have = p.Dv - v0;
  const int tok = 16 * w + r16;
  auto at = [&](int c) { return (int64_t)c * p.B * p.H + bh; };
  auto kat = [&](int c) { return ((int64_t)c * p.B + b) * p.Hk + hk; };

  if (wave_id() < 4) {
    const IT *vp = (const IT *)p.v.p + b * p.v.s0 + h * p.v.s2 + v0;
    f4 S[NV][RT];  // S[key][v0 + 16 n + i] of key 16 (RT w + r) + r16
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int key = 16 * (RT * w + r) + r16;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          S[n][r][i] = p.h0 && key < p.Dk && 16 * n + i < have ? p.h0[((int64_t)bh * p.Dk + key) * p.Dv + v0 + 16 * n + i] : 0.0f;
      }
    bf8 K[KS][NK], T[2][NM], Kt[RT][2][NK];
    Raw4<IT> v[NV];
    f4 row;  // a, beta, c of the token, e^{G_C}
    auto load_v = [&](int c) {
      const int64_t t = (int64_t)c * kC + tok;
#pragma unroll
      for (int n = 0; n < NV; ++n) v[n] = load4(vp + t * p.v.s1 + 16 * n, (const IT *)p.v.p, t < p.L ? have - 16 * n : 0, p.vv);
      row = token_row(delta_rows(p, at(c)), tok);
    };
    auto load_k = [&](int c) {
#pragma unroll
      for (int s = 0; s < KS; ++s) load_frag<NK>(key_frags<DK, NK>(p.fK, kat(c)), kC * DK, w * KS + s, lane, K[s]);
    };
    auto load_t = [&](int c) {  // T is lower triangular
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= w / 2) load_frag<NM>((const __bf16 *)p.fT + at(c) * NM * kFrag, kFrag, 2 * w + s, lane, T[s]);
    };
    auto load_kt = [&](int c) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int r = 0; r < RT; ++r) load_frag<NK>(key_frags<DK, NK>(p.fKt, kat(c)), kC * DK, 2 * (RT * w + r) + s, lane, Kt[r][s]);
    };
    load_k(0);
    load_v(0);
    load_t(0);
    load_kt(0);
    for (int c = 0; c < p.NC; ++c) {
      const int64_t t = (int64_t)c * kC + tok;
      const int next = c + 1 < p.NC ? c + 1 : c;
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int r = 0; r < RT; ++r) St[n].put(16 * (RT * w + r) + r16, kg, S[n][r]);
      lds_barrier();
      f4 x[NV], y[NV];
#pragma unroll
      for (int n = 0; n < NV; ++n) x[n] = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          bf8 A[NM];
          St[n].get(s, lane, A);
          x[n] = mma<NM>(A, K[s], x[n]);
        }
      read_ahead<KS * NM * 2 * NV, KS * products(NM, NM, NK) * NV, 12>();
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        y[n] = to_f4<IT>(v[n], t < p.L && have - 16 * n > 0) - row[0] * x[n];
        Xt[n].put(tok, kg, y[n]);
      }
      const float bu = row[1], bc = row[1] * row[2], decay = row[3];
      load_k(next);
      load_v(next);
      lds_barrier();
      bf8 X[NV][2][NM];
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        Xt[n].get(0, lane, X[n][0]);
        Xt[n].get(1, lane, X[n][1]);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)  // Y = X + (T - I) X
        if (s <= w / 2) {
#pragma unroll
          for (int n = 0; n < NV; ++n) y[n] = mma<NM>(X[n][s], T[s], y[n]);
        }
      auto put_u = [&] {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          Wt[n].put(tok, kg, bc * y[n]);
          Ut[n].put(tok, kg, bu * y[n]);
        }
      };
      put_u();
      load_t(next);
      if (__builtin_expect(not_finite(y), 0)) {  // after the writes, which need not wait for it
#pragma unroll
        for (int n = 0; n < NV; ++n) x[n] = Xt[n].value(tok, kg);
        if (not_finite_of(y, x)) {
#pragma unroll
          for (int n = 0; n < NV; ++n)
            y[n] = row_times<NM>((const __bf16 *)p.fT + at(c) * NM * kFrag, tok, 0, tok, Xt[n], kg, x[n]);
          put_u();
        }
      }
      lds_barrier();
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int r = 0; r < RT; ++r) S[n][r] *= decay;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          bf8 A[NM];
          Wt[n].get(s, lane, A);
#pragma unroll
          for (int r = 0; r < RT; ++r) S[n][r] = mma<NM>(A, Kt[r][s], S[n][r]);
        }
      read_ahead<2 * NM * 2 * NV, 2 * products(NM, NM, NK) * RT * NV, 12>();
      load_kt(next);
      if (p.y) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
          if (vt + n < p.VT) *(f4 *)(value_of(p.y, p, at(c), vt + n) + (unsigned)(16 * tok + 4 * kg)) = y[n];
      }
    }
    if (p.last) {
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int key = 16 * (RT * w + r) + r16;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key < p.Dk && 16 * n + i < have) p.last[((int64_t)bh * p.Dk + key) * p.Dv + v0 + 16 * n + i] = S[n][r][i];
        }
    }
  } else {
    IT *op = (IT *)p.o.p + b * p.o.s0 + h * p.o.s2 + v0;
    bf8 Q[KS][NK], P[2][NM];
    float fd;
    auto load_q = [&](int c) {
#pragma unroll
      for (int s = 0; s < KS; ++s) load_frag<NK>(key_frags<DK, NK>(p.fQ, kat(c)), kC * DK, w * KS + s, lane, Q[s]);
      fd = delta_rows(p, at(c))[8 * kC + (unsigned)tok];
    };
    auto load_p = [&](int c) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= w / 2) load_frag<NM>((const __bf16 *)p.fP + at(c) * NM * kFrag, kFrag, 2 * w + s, lane, P[s]);
    };
    load_q(0);
    load_p(0);
    for (int c = 0; c < p.NC; ++c) {
      const int64_t t = (int64_t)c * kC + tok;
      const int next = c + 1 < p.NC ? c + 1 : c;
      lds_barrier();
      f4 o[NV];
#pragma unroll
      for (int n = 0; n < NV; ++n) o[n] = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          bf8 A[NM];
          St[n].get(s, lane, A);
          o[n] = mma<NM>(A, Q[s], o[n]);
        }
      read_ahead<KS * NM * 2 * NV, KS * products(NM, NM, NK) * NV, 12>();
#pragma unroll
      for (int n = 0; n < NV; ++n) o[n] *= fd;
      if (p.states) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const int key = 16 * (RT * w + r) + r16;
            if (key < p.Dkp && vt + n < p.VT)
              *(f4 *)(state_of(p.states, p, at(c), vt + n) + (unsigned)(16 * key + 4 * kg)) = St[n].whole(key, kg);
          }
      }
      load_q(next);
      lds_barrier();
      lds_barrier();
      f4 qs[NV];
#pragma unroll
      for (int n = 0; n < NV; ++n) qs[n] = o[n];
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= w / 2) {
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            bf8 A[NM];
            Ut[n].get(s, lane, A);
            o[n] = mma<NM>(A, P[s], o[n]);
          }
        }
      if (__builtin_expect(not_finite(o), 0) && not_finite_of(o, qs)) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
          o[n] = row_times<NM>((const __bf16 *)p.fP + at(c) * NM * kFrag, tok, 0, tok + 1, Ut[n], kg, qs[n]);
      }
      load_p(next);
#pragma unroll
      for (int n = 0; n < NV; ++n) store4(op + t * p.o.s1 + 16 * n, o[n], t < p.L ? have - 16 * n : 0, p.vo);
    }
  }
}

template <typename IT, int DK>
static hipError_t delta_fwd(const DeltaParams &p, hipStream_t s) {
  const unsigned heads = (unsigned)(p.B * p.H);
  hipLaunchKernelGGL((k_delta_prep<IT, DK, false>), dim3(heads * (unsigned)p.NC), dim3(kDT), 0, s, p);
  if (delta_pairs(p))
    delta_walk(p, 2, [&](const DeltaParams &part, dim3 grid) { hipLaunchKernelGGL((k_delta_fwd<IT, DK, 2>), grid, dim3(2 * kDT), 0, s, part); });
  else
    delta_walk(p, 1, [&](const DeltaParams &part, dim3 grid) { hipLaunchKernelGGL((k_delta_fwd<IT, DK, 1>), grid, dim3(2 * kDT), 0, s, part); });
  return hipGetLastError();
}
template <typename IT>
static hipError_t delta_fwd_k(const DeltaParams &p, hipStream_t s) {
  return p.Dk <= 64 ? delta_fwd<IT, 64>(p, s) : delta_fwd<IT, 128>(p, s);
}
hipError_t launch_delta_fwd(const DeltaParams &p, int dtype, hipStream_t s) {
  return dtype == 0 ? delta_fwd_k<float>(p, s) : dtype == 1 ? delta_fwd_k<bf16_t>(p, s) : delta_fwd_k<f16_t>(p, s);
}

// The backward's preparation.
template <typename IT>
static hipError_t delta_prep_t(const DeltaParams &p, hipStream_t s) {
  const dim3 grid((unsigned)(p.B * p.H) * (unsigned)p.NC);
  if (p.Dk <= 64) hipLaunchKernelGGL((k_delta_prep<IT, 64, true>), grid, dim3(kDT), 0, s, p);
  else hipLaunchKernelGGL((k_delta_prep<IT, 128, true>), grid, dim3(kDT), 0, s, p);
  return hipGetLastError();
}
hipError_t launch_delta_prep_t(const DeltaParams &p, int dtype, hipStream_t s) {
  return dtype == 0 ? delta_prep_t<float>(p, s) : dtype == 1 ? delta_prep_t<bf16_t>(p, s) : delta_prep_t<f16_t>(p, s);
}

}  // namespace ssm
