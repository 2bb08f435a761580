// Gated delta rule, chunked forward (the mathematics and the operand layouts: ssm_delta.hpp).
//
//   k_delta_prep  one workgroup per (batch row, value head, chunk): decays, norms, T and P
//   k_delta_fwd   one workgroup per (batch row, value head, 16 NV columns of v): the columns of S do
//                 not mix, so each walks the chunks with its own columns in registers
#include "ssm_delta.hpp"

namespace ssm {

// c(16 x 16) += a b from float32 LDS matrices: a's rows and b's columns of 16.
template <int PITCH>
__device__ __forceinline__ f4 mma_f32(const float *a, const float *b, int lane, f4 c) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[(lane % 16) * PITCH + 4 * k + lane / 16],
                                             b[(4 * k + lane / 16) * PITCH + lane % 16], c, 0, 0, 0);
  return c;
}
template <int PITCH>
__device__ __forceinline__ void put16(float *m, int lane, f4 c, float sign) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m[(4 * (lane / 16) + i) * PITCH + lane % 16] = sign * c[i];
}

// Writes T - I and P (TR: their transposes) as operand fragments, and the row factors.
// T is inverted in float32: the four 16 x 16 diagonal blocks by substitution, one wavefront each, the
// rest by T10 = -T11 (L10 T00) for blocks of 16, then of 32 rows.
template <typename IT, int DK, bool TR>
__global__ void __launch_bounds__(kDT) k_delta_prep(const DeltaParams p) {
  constexpr int NK = DParts<IT>::in, NM = DParts<IT>::mid, KS = DK / 32, KP = DK + 8, FP = kC + 4;
  __shared__ __align__(16) __bf16 Kr[NK][kC][KP];
  __shared__ __align__(16) float Lm[kC][FP], Pm[kC][FP];
  __shared__ double Gs[kC];
  __shared__ float fk[kC], fq[kC], bs[kC];
  const int tid = threadIdx.x, lane = tid % 64, w = tid / 64, r16 = lane % 16, kg = lane / 16;
  const int64_t ch = blockIdx.x;
  const int bh = (int)(ch / p.NC), c = (int)(ch % p.NC), b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk);
  const int64_t t0 = (int64_t)c * kC, t = t0 + 16 * w + r16;
  const IT *kp = (const IT *)p.k.p + b * p.k.s0 + t * p.k.s1 + hk * p.k.s2;
  const IT *qp = (const IT *)p.q.p + b * p.q.s0 + t * p.q.s1 + hk * p.q.s2;
  const int have = t < p.L ? p.Dk : 0;
  bf8 K[KS][NK], Q[KS][NK];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int e = 32 * s + 8 * kg;
    row_frag<IT, NK>(kp + e, have - e, p.vk, K[s]);
    row_frag<IT, NK>(qp + e, have - e, p.vq, Q[s]);
#pragma unroll
    for (int n = 0; n < NK; ++n) *(bf8 *)&Kr[n][16 * w + r16][e] = K[s][n];
  }
  if (w == 0) {
    const int64_t tt = t0 + lane;
    double g = 0;
    if (tt < p.L) g = (double)((const float *)p.g.p)[b * p.g.s0 + tt * p.g.s1 + h * p.g.s2];
    if (g < -1e4) g = -1e4;  // e^-1e4 is 0 in either width, and -inf would make inf - inf of the differences
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double up = __shfl_up(g, d);
      if (lane >= d) g += up;
    }
    Gs[lane] = g;
  } else if (w == 1) {
    const int64_t tt = t0 + lane;
    bs[lane] = tt < p.L ? load_either<IT>(p.beta.p, p.beta32, b * p.beta.s0 + tt * p.beta.s1 + h * p.beta.s2) : 0.0f;
  }
  {  // the norms are the diagonals of K K^T and Q Q^T
    f4 kk = 0, qq = 0;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      kk = mma(K[s], K[s], kk);
      qq = mma(Q[s], Q[s], qq);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * kg + i == r16) {
        fk[16 * w + r16] = p.qk_norm ? 1.0f / sqrtf(kk[i] + 1e-6f) : 1.0f;
        fq[16 * w + r16] = p.qk_norm ? p.scale / sqrtf(qq[i] + 1e-6f) : p.scale;
      }
  }
  __syncthreads();
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) {
    f4 kk = 0, qk = 0;
    const int col = 16 * jt + r16;
    if (jt <= w) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        bf8 B[NK];
        lds_frag<NK, KP>(&Kr[0][0][0], kC * KP, col, 32 * s + 8 * kg, B);
        kk = mma(K[s], B, kk);
        qk = mma(Q[s], B, qk);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * w + 4 * kg + i;
      float l = 0, pr = 0;
      if (col <= row) {
        const float e = fexp((float)(Gs[row] - Gs[col])) * fk[col];
        pr = e * fq[row] * qk[i];
        if (col < row) l = bs[row] * fk[row] * e * kk[i];
      }
      Lm[row][col] = l;
      Pm[row][col] = pr;
    }
  }
  __syncthreads();
  float *Yr = (float *)&Kr[0][0][0];  // the keys are no longer read: scratch of 32 x FP floats
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
    wave_lds_sync();
    if (kg == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) Lm[16 * w + i][16 * w + r16] = x[i];
    }
  }
  __syncthreads();
  if (w < 2) {
    float *Y = Yr + 16 * w * FP;
    put16<FP>(Y, lane, mma_f32<FP>(&Lm[32 * w + 16][32 * w], &Lm[32 * w][32 * w], lane, (f4)0.0f), 1.0f);
    wave_lds_sync();
    const f4 t10 = mma_f32<FP>(&Lm[32 * w + 16][32 * w + 16], Y, lane, (f4)0.0f);
    wave_lds_sync();
    put16<FP>(&Lm[32 * w + 16][32 * w], lane, t10, -1.0f);
  }
  __syncthreads();
  const int r = w / 2, cc = w % 2;
  {
    f4 y = 0;
    for (int k = cc; k < 2; ++k) y = mma_f32<FP>(&Lm[32 + 16 * r][16 * k], &Lm[16 * k][16 * cc], lane, y);
    put16<FP>(Yr + 16 * r * FP + 16 * cc, lane, y, 1.0f);
  }
  __syncthreads();
  {
    f4 y = 0;
    for (int k = 0; k <= r; ++k) y = mma_f32<FP>(&Lm[32 + 16 * r][32 + 16 * k], Yr + 16 * k * FP + 16 * cc, lane, y);
    put16<FP>(&Lm[32 + 16 * r][16 * cc], lane, y, -1.0f);
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int row = 16 * w + r16, e = 32 * s + 8 * kg;
    f8 x, y;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = TR ? Lm[e + j][row] : Lm[row][e + j];
      if (e + j == row) x[j] = 0;  // T - I
      y[j] = TR ? Pm[e + j][row] : Pm[row][e + j];
    }
    bf8 a[NM];
    const int64_t at = ch * NM * kFrag + ((2 * w + s) * 64 + lane) * 8;
    split_parts<NM>(x, a);
#pragma unroll
    for (int n = 0; n < NM; ++n) *(bf8 *)((__bf16 *)p.fT + at + n * kFrag) = a[n];
    split_parts<NM>(y, a);
#pragma unroll
    for (int n = 0; n < NM; ++n) *(bf8 *)((__bf16 *)p.fP + at + n * kFrag) = a[n];
  }
  if (tid < kC) {
    float *rows = p.rows + ch * kDeltaRows;
    const double G = Gs[tid];
    const float eG = fexp((float)G);
    rows[tid] = fk[tid] * eG;
    rows[kC + tid] = bs[tid];
    rows[2 * kC + tid] = fk[tid] * fexp((float)(Gs[kC - 1] - G));
    rows[3 * kC + tid] = fq[tid] * eG;
    rows[4 * kC + tid] = fk[tid];
    rows[5 * kC + tid] = fq[tid];
    ((double *)(rows + 6 * kC))[tid] = G;
  }
}

template <typename IT, int DK, int NV>
__global__ void __launch_bounds__(kDT) k_delta_fwd(const DeltaParams p) {
  constexpr int NK = DParts<IT>::in, NM = DParts<IT>::mid, KS = DK / 32, KP = DK + 8, BV = 16 * NV, RT = DK / 64;
  __shared__ __align__(16) __bf16 Kr[NK][kC][KP];                       // keys, row per token
  __shared__ __align__(16) __bf16 St[NM][BV][KP];                       // state, row per column of v
  __shared__ __align__(16) __bf16 Rt[NM][BV][kCP], Ut[NM][BV][kCP], Wt[NM][BV][kCP];  // R, U, c U, row per column
  const int tid = threadIdx.x, lane = tid % 64, w = tid / 64, r16 = lane % 16, kg = lane / 16;
  int bh, vt;
  delta_tile((p.Dv + BV - 1) / BV, (int)p.B * p.H, bh, vt);
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk), v0 = vt * BV;
  const int tr = 16 * w + 4 * kg;  // the lane's token rows of a result tile: tr + i
  const IT *kb = (const IT *)p.k.p + b * p.k.s0 + hk * p.k.s2, *qb = (const IT *)p.q.p + b * p.q.s0 + hk * p.q.s2;
  const IT *vb = (const IT *)p.v.p + b * p.v.s0 + h * p.v.s2;
  IT *ob = (IT *)p.o.p + b * p.o.s0 + h * p.o.s2;

  f4 S[RT][NV];  // rows 16 (RT w + r) + 4 kg + i, columns v0 + 16 n + r16
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int kr = 16 * (RT * w + r) + 4 * kg + i, vc = v0 + 16 * n + r16;
        S[r][n][i] = p.h0 && kr < p.Dk && vc < p.Dv ? p.h0[((int64_t)bh * p.Dk + kr) * p.Dv + vc] : 0.0f;
      }

  for (int c = 0; c < p.NC; ++c) {
    const int64_t t0 = (int64_t)c * kC, ch = (int64_t)bh * p.NC + c;
    const float *rows = delta_rows(p, ch);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        bf4 parts[NM];
        split_parts<NM>(S[r][n], parts);
#pragma unroll
        for (int m = 0; m < NM; ++m) *(bf4 *)&St[m][16 * n + r16][16 * (RT * w + r) + 4 * kg] = parts[m];
        if (p.states) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kr = 16 * (RT * w + r) + 4 * kg + i, vc = v0 + 16 * n + r16;
            if (kr < p.Dk && vc < p.Dv) p.states[(ch * p.Dk + kr) * p.Dv + vc] = S[r][n][i];
          }
        }
      }
    const int64_t t = t0 + 16 * w + r16;
    const int have = t < p.L ? p.Dk : 0;
    bf8 K[KS][NK], Q[KS][NK];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int e = 32 * s + 8 * kg;
      row_frag<IT, NK>(kb + t * p.k.s1 + e, have - e, p.vk, K[s]);
      row_frag<IT, NK>(qb + t * p.q.s1 + e, have - e, p.vq, Q[s]);
#pragma unroll
      for (int n = 0; n < NK; ++n) *(bf8 *)&Kr[n][16 * w + r16][e] = K[s][n];
    }
    const f4 fa = row4(rows, 0, tr), be = row4(rows, 1, tr), fc = row4(rows, 2, tr), fd = row4(rows, 3, tr);
    const float eC = chunk_decay(rows);
    lds_barrier();
    f4 U[NV], O[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      f4 x = 0, o = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        bf8 B[NM];
        lds_frag<NM, KP>(&St[0][0][0], BV * KP, 16 * n + r16, 32 * s + 8 * kg, B);
        x = mma(K[s], B, x);
        o = mma(Q[s], B, o);
      }
      const int vc = v0 + 16 * n + r16;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = t0 + tr + i < p.L && vc < p.Dv ? Conv<IT>::load(vb + (t0 + tr + i) * p.v.s1 + vc) : 0.0f;
        U[n][i] = be[i] * fmaf(-fa[i], x[i], v);
      }
      O[n] = fd * o;
      bf4 parts[NM];
      split_parts<NM>(U[n], parts);
#pragma unroll
      for (int m = 0; m < NM; ++m) *(bf4 *)&Rt[m][16 * n + r16][tr] = parts[m];
    }
    lds_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {  // U = R + (T - I) R; T is lower triangular
      if (s <= w / 2) {
        bf8 A[NM];
#pragma unroll
        for (int m = 0; m < NM; ++m) A[m] = *(const bf8 *)((const __bf16 *)p.fT + (ch * NM + m) * kFrag + ((2 * w + s) * 64 + lane) * 8);
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          bf8 B[NM];
          lds_frag<NM, kCP>(&Rt[0][0][0], BV * kCP, 16 * n + r16, 32 * s + 8 * kg, B);
          U[n] = mma(A, B, U[n]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      bf4 parts[NM];
      split_parts<NM>(U[n], parts);
#pragma unroll
      for (int m = 0; m < NM; ++m) *(bf4 *)&Ut[m][16 * n + r16][tr] = parts[m];
      split_parts<NM>((f4)(fc * U[n]), parts);
#pragma unroll
      for (int m = 0; m < NM; ++m) *(bf4 *)&Wt[m][16 * n + r16][tr] = parts[m];
      if (p.u) {
        const int vc = v0 + 16 * n + r16;
        if (vc < p.Dv) {
#pragma unroll
          for (int i = 0; i < 4; ++i) p.u[(ch * kC + tr + i) * p.Dv + vc] = U[n][i];
        }
      }
    }
    lds_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s <= w / 2) {
        bf8 A[NM];
#pragma unroll
        for (int m = 0; m < NM; ++m) A[m] = *(const bf8 *)((const __bf16 *)p.fP + (ch * NM + m) * kFrag + ((2 * w + s) * 64 + lane) * 8);
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          bf8 B[NM];
          lds_frag<NM, kCP>(&Ut[0][0][0], BV * kCP, 16 * n + r16, 32 * s + 8 * kg, B);
          O[n] = mma(A, B, O[n]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int vc = v0 + 16 * n + r16;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t0 + tr + i < p.L && vc < p.Dv) Conv<IT>::store(ob + (t0 + tr + i) * p.o.s1 + vc, O[n][i]);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int n = 0; n < NV; ++n) S[r][n] *= eC;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf8 A[RT][NK];
#pragma unroll
      for (int r = 0; r < RT; ++r) lds_frag_t<NK, KP>(&Kr[0][0][0], kC * KP, 32 * s, 16 * (RT * w + r), lane, A[r]);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        bf8 B[NM];
        lds_frag<NM, kCP>(&Wt[0][0][0], BV * kCP, 16 * n + r16, 32 * s + 8 * kg, B);
#pragma unroll
        for (int r = 0; r < RT; ++r) S[r][n] = mma(A[r], B, S[r][n]);
      }
    }
    lds_barrier();  // the keys and Wt are read, the next chunk may write
  }
  if (p.last) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kr = 16 * (RT * w + r) + 4 * kg + i, vc = v0 + 16 * n + r16;
          if (kr < p.Dk && vc < p.Dv) p.last[((int64_t)bh * p.Dk + kr) * p.Dv + vc] = S[r][n][i];
        }
  }
}

template <typename IT, int DK>
static hipError_t delta_fwd(const DeltaParams &p, hipStream_t s) {
  const unsigned heads = (unsigned)(p.B * p.H);
  hipLaunchKernelGGL((k_delta_prep<IT, DK, false>), dim3(heads * (unsigned)p.NC), dim3(kDT), 0, s, p);
  constexpr int NV = 1;
  hipLaunchKernelGGL((k_delta_fwd<IT, DK, NV>), dim3(heads * (unsigned)((p.Dv + 16 * NV - 1) / (16 * NV))), dim3(kDT), 0, s, p);
  return hipGetLastError();
}
template <typename IT>
static hipError_t delta_fwd_k(const DeltaParams &p, hipStream_t s) {
  return p.Dk <= 64 ? delta_fwd<IT, 64>(p, s) : delta_fwd<IT, 128>(p, s);
}
hipError_t launch_delta_fwd(const DeltaParams &p, int dtype, hipStream_t s) {
  return dtype == 0 ? delta_fwd_k<float>(p, s) : dtype == 1 ? delta_fwd_k<bf16_t>(p, s) : delta_fwd_k<f16_t>(p, s);
}

// The transposed prep of the backward.
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
