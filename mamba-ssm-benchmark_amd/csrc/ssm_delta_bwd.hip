// Gated delta rule, backward of the chunked form (notation: ssm_delta.hpp).  With D = dS1, the gradient of
// the state leaving a chunk, a = |k|^-1 e^G, c = |k|^-1 e^{G_C - G}, d = scale |q|^-1 e^G:
//   dU = P^T dO + c K D,  dR = T^T dU,  dV = beta dR
//   dS0 = e^{G_C} D + Q^T (d dO) - K^T (beta a dR)
// k_delta_bwd walks the chunks backward, one workgroup per 16 NV columns of v like the forward, and
// leaves D and dR of every chunk; k_delta_grad then treats every chunk by itself, one workgroup per
// (batch row, key head, chunk), adding the value heads that share the key head in registers.  With
// A = dO U^T and N = dR U^T, k^ and q^ the normalised rows and e_ij = e^{G_i - G_j}:
//   dq^ = scale (e^G dO S0^T + (A e)_{j <= i} K^)
//   dk^ = e^{G_C - G} U D^T + (scale A e)^T_{j <= i} Q^ - (beta N e and its transpose)_{j < i} K^ - beta e^G dR S0^T
//   dbeta_i = dR_i.v_i - e^{G_i} k^_i.(dR S0^T)_i - sum_{j < i} N_ij e_ij k^_i.k^_j
//   dG_i, G's gradient: every factor e^x times its derivative, x's terms of G with their signs; dg is its
//   sum from i to the chunk's end.  Each product enters a row and a column sum with the same value, so
//   that what does not straddle a token cancels to rounding.
#include "ssm_delta.hpp"
#include "ssm_dpp.hpp"

namespace ssm {

hipError_t launch_delta_prep_t(const DeltaParams &p, int dtype, hipStream_t s);

template <typename IT, int DK, int NV>
__global__ void __launch_bounds__(kDT) k_delta_bwd(const DeltaParams p) {
  constexpr int NK = DParts<IT>::in, NM = DParts<IT>::mid, KS = DK / 32, KP = DK + 8, BV = 16 * NV, RT = DK / 64;
  __shared__ __align__(16) __bf16 Kr[NK][kC][KP], Qr[NK][kC][KP];  // keys and queries, row per token
  __shared__ __align__(16) __bf16 Dt[NM][BV][KP];                  // D, row per column of v
  __shared__ __align__(16) __bf16 Ot[NK][BV][kCP];                 // dO, row per column of v; below d dO, dU, -beta a dR
  __shared__ __align__(16) __bf16 Et[NM][BV][kCP], Xt[NM][BV][kCP], Yt[NM][BV][kCP];
  const int tid = threadIdx.x, lane = tid % 64, w = tid / 64, r16 = lane % 16, kg = lane / 16;
  int bh, vt;
  delta_tile((p.Dv + BV - 1) / BV, (int)p.B * p.H, bh, vt);
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk), v0 = vt * BV;
  const int tr = 16 * w + 4 * kg;
  const IT *kb = (const IT *)p.k.p + b * p.k.s0 + hk * p.k.s2, *qb = (const IT *)p.q.p + b * p.q.s0 + hk * p.q.s2;
  const IT *ob = (const IT *)p.dout.p + b * p.dout.s0 + h * p.dout.s2;
  IT *vb = (IT *)p.dv.p + b * p.dv.s0 + h * p.dv.s2;

  f4 D[RT][NV];  // rows 16 (RT w + r) + 4 kg + i, columns v0 + 16 n + r16
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int kr = 16 * (RT * w + r) + 4 * kg + i, vc = v0 + 16 * n + r16;
        D[r][n][i] = p.dlast && kr < p.Dk && vc < p.Dv ? p.dlast[((int64_t)bh * p.Dk + kr) * p.Dv + vc] : 0.0f;
      }

  for (int c = p.NC - 1; c >= 0; --c) {
    const int64_t t0 = (int64_t)c * kC, ch = (int64_t)bh * p.NC + c;
    const float *rows = delta_rows(p, ch);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        bf4 parts[NM];
        split_parts<NM>(D[r][n], parts);
#pragma unroll
        for (int m = 0; m < NM; ++m) *(bf4 *)&Dt[m][16 * n + r16][16 * (RT * w + r) + 4 * kg] = parts[m];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kr = 16 * (RT * w + r) + 4 * kg + i, vc = v0 + 16 * n + r16;
          if (kr < p.Dk && vc < p.Dv) p.dstates[(ch * p.Dk + kr) * p.Dv + vc] = D[r][n][i];
        }
      }
    const int64_t t = t0 + 16 * w + r16;
    const int have = t < p.L ? p.Dk : 0;
    bf8 K[KS][NK];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int e = 32 * s + 8 * kg;
      bf8 Q[NK];
      row_frag<IT, NK>(kb + t * p.k.s1 + e, have - e, p.vk, K[s]);
      row_frag<IT, NK>(qb + t * p.q.s1 + e, have - e, p.vq, Q);
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        *(bf8 *)&Kr[n][16 * w + r16][e] = K[s][n];
        *(bf8 *)&Qr[n][16 * w + r16][e] = Q[n];
      }
    }
    const f4 fa = row4(rows, 0, tr), be = row4(rows, 1, tr), fc = row4(rows, 2, tr), fd = row4(rows, 3, tr);
    const float eC = chunk_decay(rows);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int vc = v0 + 16 * n + r16;
      f4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[i] = t0 + tr + i < p.L && vc < p.Dv ? Conv<IT>::load(ob + (t0 + tr + i) * p.dout.s1 + vc) : 0.0f;
      bf4 in[NK], mid[NM];
      split_parts<NK>(x, in);
#pragma unroll
      for (int m = 0; m < NK; ++m) *(bf4 *)&Ot[m][16 * n + r16][tr] = in[m];
      split_parts<NM>((f4)(fd * x), mid);
#pragma unroll
      for (int m = 0; m < NM; ++m) *(bf4 *)&Et[m][16 * n + r16][tr] = mid[m];
    }
    lds_barrier();
    f4 X[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      f4 x = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        bf8 B[NM];
        lds_frag<NM, KP>(&Dt[0][0][0], BV * KP, 16 * n + r16, 32 * s + 8 * kg, B);
        x = mma(K[s], B, x);
      }
      X[n] = fc * x;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {  // P^T is upper triangular
      if (s >= w / 2) {
        bf8 A[NM];
#pragma unroll
        for (int m = 0; m < NM; ++m) A[m] = *(const bf8 *)((const __bf16 *)p.fP + (ch * NM + m) * kFrag + ((2 * w + s) * 64 + lane) * 8);
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          bf8 B[NK];
          lds_frag<NK, kCP>(&Ot[0][0][0], BV * kCP, 16 * n + r16, 32 * s + 8 * kg, B);
          X[n] = mma(A, B, X[n]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      bf4 parts[NM];
      split_parts<NM>(X[n], parts);
#pragma unroll
      for (int m = 0; m < NM; ++m) *(bf4 *)&Xt[m][16 * n + r16][tr] = parts[m];
    }
    lds_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s >= w / 2) {
        bf8 A[NM];
#pragma unroll
        for (int m = 0; m < NM; ++m) A[m] = *(const bf8 *)((const __bf16 *)p.fT + (ch * NM + m) * kFrag + ((2 * w + s) * 64 + lane) * 8);
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          bf8 B[NM];
          lds_frag<NM, kCP>(&Xt[0][0][0], BV * kCP, 16 * n + r16, 32 * s + 8 * kg, B);
          X[n] = mma(A, B, X[n]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      bf4 parts[NM];
      split_parts<NM>((f4)(-be * fa * X[n]), parts);
#pragma unroll
      for (int m = 0; m < NM; ++m) *(bf4 *)&Yt[m][16 * n + r16][tr] = parts[m];
      const int vc = v0 + 16 * n + r16;
      if (vc < p.Dv) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p.dr[(ch * kC + tr + i) * p.Dv + vc] = X[n][i];
          if (t0 + tr + i < p.L) Conv<IT>::store(vb + (t0 + tr + i) * p.dv.s1 + vc, be[i] * X[n][i]);
        }
      }
    }
    lds_barrier();
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int n = 0; n < NV; ++n) D[r][n] *= eC;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf8 A[RT][NK], Q[RT][NK];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        lds_frag_t<NK, KP>(&Kr[0][0][0], kC * KP, 32 * s, 16 * (RT * w + r), lane, A[r]);
        lds_frag_t<NK, KP>(&Qr[0][0][0], kC * KP, 32 * s, 16 * (RT * w + r), lane, Q[r]);
      }
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        bf8 E[NM], Y[NM];
        lds_frag<NM, kCP>(&Et[0][0][0], BV * kCP, 16 * n + r16, 32 * s + 8 * kg, E);
        lds_frag<NM, kCP>(&Yt[0][0][0], BV * kCP, 16 * n + r16, 32 * s + 8 * kg, Y);
#pragma unroll
        for (int r = 0; r < RT; ++r) D[r][n] = mma(A[r], Y, mma(Q[r], E, D[r][n]));
      }
    }
    lds_barrier();
  }
  if (p.dh0) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kr = 16 * (RT * w + r) + 4 * kg + i, vc = v0 + 16 * n + r16;
          if (kr < p.Dk && vc < p.Dv) p.dh0[((int64_t)bh * p.Dk + kr) * p.Dv + vc] = D[r][n][i];
        }
  }
}

// Element (row, col) of an LDS matrix of N parts.
template <int N, int PITCH>
__device__ __forceinline__ float lds_elem(const __bf16 *m, int part, int row, int col) {
  float s = 0;
#pragma unroll
  for (int n = N - 1; n >= 0; --n) s += (float)m[n * part + row * PITCH + col];
  return s;
}

template <typename IT, int DK>
__global__ void __launch_bounds__(kDT) k_delta_grad(const DeltaParams p) {
  constexpr int NK = DParts<IT>::in, NM = DParts<IT>::mid, KS = DK / 32, KP = DK + 8, CT = DK / 64;
  constexpr int SV = 32, SP = SV + 8;  // columns of v staged at a time
  constexpr int kSlab = (NK + 2 * NM) * kC * SP, kE = NM * kC * kCP;
  __shared__ __align__(16) __bf16 Kr[NK][kC][KP], Qr[NK][kC][KP];
  __shared__ __align__(16) __bf16 buf[kSlab > kE ? kSlab : kE];  // slabs of dO, dR, U; then a 64 x 64 operand
  __shared__ double Gs[kC];
  __shared__ float red[4][4][kC], colsum[4][kC], rowg[kC], rowb[kC], bt[kC], sdot[4];
  __bf16 *const Os = buf, *const Rs = Os + NK * kC * SP, *const Us = Rs + NM * kC * SP, *const Es = buf;
  const int tid = threadIdx.x, lane = tid % 64, w = tid / 64, r16 = lane % 16, kg = lane / 16;
  const int c = blockIdx.x % p.NC, bk = blockIdx.x / p.NC, b = bk / p.Hk, hk = bk % p.Hk, group = p.H / p.Hk;
  const int64_t t0 = (int64_t)c * kC;
  const bool vec32 = p.Dv % 8 == 0;
  {
    const int64_t t = t0 + 16 * w + r16;
    const int have = t < p.L ? p.Dk : 0;
    const IT *kp = (const IT *)p.k.p + b * p.k.s0 + t * p.k.s1 + hk * p.k.s2;
    const IT *qp = (const IT *)p.q.p + b * p.q.s0 + t * p.q.s1 + hk * p.q.s2;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int e = 32 * s + 8 * kg;
      bf8 f[NK];
      row_frag<IT, NK>(kp + e, have - e, p.vk, f);
#pragma unroll
      for (int n = 0; n < NK; ++n) *(bf8 *)&Kr[n][16 * w + r16][e] = f[n];
      row_frag<IT, NK>(qp + e, have - e, p.vq, f);
#pragma unroll
      for (int n = 0; n < NK; ++n) *(bf8 *)&Qr[n][16 * w + r16][e] = f[n];
    }
  }
  f4 Yq[4][CT], Zk[4][CT];  // token rows 16 it + 4 kg + i, key columns 16 (CT w + ct) + r16
#pragma unroll
  for (int it = 0; it < 4; ++it)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) Yq[it][ct] = Zk[it][ct] = 0;
  const float *rows = nullptr;

  for (int hg = 0; hg < group; ++hg) {
    const int h = hk * group + hg;
    const int64_t ch = ((int64_t)b * p.H + h) * p.NC + c;
    rows = delta_rows(p, ch);
    const IT *ob = (const IT *)p.dout.p + b * p.dout.s0 + h * p.dout.s2, *vb = (const IT *)p.v.p + b * p.v.s0 + h * p.v.s2;
    f4 F1[4][CT], F2[4][CT], F3[4][CT], A[4], N[4];  // dO S0^T, U D^T, dR S0^T; row tile w of dO U^T, dR U^T
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      A[it] = N[it] = 0;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) F1[it][ct] = F2[it][ct] = F3[it][ct] = 0;
    }
    float sd = 0, rv = 0;  // <S0, D>, dR.v of row tid / 4
    if (tid < kC) Gs[tid] = ((const double *)(rows + 6 * kC))[tid];
    for (int d0 = 0; d0 < p.Dv; d0 += SV) {
      if (d0) lds_barrier();
      {
        const int row = tid / 4, e = 8 * (tid % 4), have = p.Dv - d0 - e;
        const int64_t t = t0 + row, at = (ch * kC + row) * p.Dv + d0 + e;
        bf8 in[NK], mid[NM];
        row_frag<IT, NK>(ob + t * p.dout.s1 + d0 + e, t < p.L ? have : 0, p.vdo, in);
#pragma unroll
        for (int n = 0; n < NK; ++n) *(bf8 *)(Os + (n * kC + row) * SP + e) = in[n];
        const f8 x = row8<float>(p.dr + at, have, vec32), v = row8<IT>(vb + t * p.v.s1 + d0 + e, t < p.L ? have : 0, p.vv);
#pragma unroll
        for (int j = 0; j < 8; ++j) rv = fmaf(x[j], v[j], rv);
        split_parts<NM>(x, mid);
#pragma unroll
        for (int n = 0; n < NM; ++n) *(bf8 *)(Rs + (n * kC + row) * SP + e) = mid[n];
        split_parts<NM>(row8<float>(p.u + at, have, vec32), mid);
#pragma unroll
        for (int n = 0; n < NM; ++n) *(bf8 *)(Us + (n * kC + row) * SP + e) = mid[n];
      }
      bf8 SB[CT][NM], DB[CT][NM];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const int kr = 16 * (CT * w + ct) + r16, have = kr < p.Dk ? p.Dv - d0 - 8 * kg : 0;
        const int64_t at = (ch * p.Dk + kr) * p.Dv + d0 + 8 * kg;
        const f8 s = row8<float>(p.states + at, have, vec32), d = row8<float>(p.dstates + at, have, vec32);
#pragma unroll
        for (int j = 0; j < 8; ++j) sd = fmaf(s[j], d[j], sd);
        split_parts<NM>(s, SB[ct]);
        split_parts<NM>(d, DB[ct]);
      }
      lds_barrier();
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        bf8 O[NK], R[NM], U[NM];
        lds_frag<NK, SP>(Os, kC * SP, 16 * it + r16, 8 * kg, O);
        lds_frag<NM, SP>(Rs, kC * SP, 16 * it + r16, 8 * kg, R);
        lds_frag<NM, SP>(Us, kC * SP, 16 * it + r16, 8 * kg, U);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          F1[it][ct] = mma(O, SB[ct], F1[it][ct]);
          F3[it][ct] = mma(R, SB[ct], F3[it][ct]);
          F2[it][ct] = mma(U, DB[ct], F2[it][ct]);
        }
        if (it <= w) {
          bf8 Ow[NK], Rw[NM];
          lds_frag<NK, SP>(Os, kC * SP, 16 * w + r16, 8 * kg, Ow);
          lds_frag<NM, SP>(Rs, kC * SP, 16 * w + r16, 8 * kg, Rw);
          A[it] = mma(Ow, U, A[it]);
          N[it] = mma(Rw, U, N[it]);
        }
      }
    }
    rv += __shfl_xor(rv, 1);
    rv += __shfl_xor(rv, 2);
    if (tid % 4 == 0) bt[tid / 4] = rv;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) sd += __shfl_xor(sd, m);
    if (lane == 0) sdot[w] = sd;

    // row dots with the rows of Q and K, and the state terms of dq, dk
    const double GC = Gs[kC - 1];
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int r0 = 16 * it + 4 * kg;
      const f4 fa = row4(rows, 0, r0), be = row4(rows, 1, r0), fc = row4(rows, 2, r0), fd = row4(rows, 3, r0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float eG = fexp((float)Gs[r0 + i]), cG = fexp((float)(GC - Gs[r0 + i]));
        float v1 = 0, v2 = 0, v3 = 0;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const int col = 16 * (CT * w + ct) + r16;
          const float q = lds_elem<NK, KP>(&Qr[0][0][0], kC * KP, r0 + i, col), k = lds_elem<NK, KP>(&Kr[0][0][0], kC * KP, r0 + i, col);
          v1 = fmaf(q, F1[it][ct][i], v1);
          v2 = fmaf(k, F2[it][ct][i], v2);
          v3 = fmaf(k, F3[it][ct][i], v3);
          Yq[it][ct][i] = fmaf(eG, F1[it][ct][i], Yq[it][ct][i]);
          Zk[it][ct][i] += cG * F2[it][ct][i] - be[i] * eG * F3[it][ct][i];
        }
        v1 = row_sum(v1);
        v2 = row_sum(v2);
        v3 = row_sum(v3);
        if (r16 == 0) {
          red[w][0][r0 + i] = fd[i] * v1 - be[i] * fa[i] * v3;
          red[w][1][r0 + i] = fc[i] * v2;
          red[w][2][r0 + i] = -fa[i] * v3;
        }
      }
    }
    // the masked products within the chunk, row tile w
    f4 E2[4], E3[4];
    f4 fqr = row4(rows, 5, 16 * w + 4 * kg), fkr = row4(rows, 4, 16 * w + 4 * kg), ber = row4(rows, 1, 16 * w + 4 * kg);
    f4 rg = 0, rb = 0;
    lds_barrier();  // the slabs are read
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
      const int col = 16 * jt + r16;
      f4 kk = 0, qk = 0;
      if (jt <= w) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          bf8 B[NK], Kw[NK], Qw[NK];
          lds_frag<NK, KP>(&Kr[0][0][0], kC * KP, col, 32 * s + 8 * kg, B);
          lds_frag<NK, KP>(&Kr[0][0][0], kC * KP, 16 * w + r16, 32 * s + 8 * kg, Kw);
          lds_frag<NK, KP>(&Qr[0][0][0], kC * KP, 16 * w + r16, 32 * s + 8 * kg, Qw);
          kk = mma(Kw, B, kk);
          qk = mma(Qw, B, qk);
        }
      }
      const float fkc = rows[4 * kC + col];
      float cs = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * w + 4 * kg + i;
        float e1 = 0, e2 = 0, e3 = 0;
        if (col <= row) {
          const float e = fexp((float)(Gs[row] - Gs[col]));
          e1 = A[jt][i] * e;
          e2 = e1 * fqr[i];
          if (col < row) {
            const float nm = N[jt][i] * e * fkr[i] * fkc * kk[i];
            e3 = N[jt][i] * e * ber[i];
            rb[i] += nm;
            const float z = e2 * fkc * qk[i] - ber[i] * nm;
            rg[i] += z;
            cs += z;
          }
          e1 *= fkc;
        }
        E2[jt][i] = e2;
        E3[jt][i] = e3;
        float x = e1;
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          const __bf16 q = (__bf16)x;
          Es[(m * kC + row) * kCP + col] = q;
          x -= (float)q;
        }
      }
      cs += __shfl_xor(cs, 16);
      cs += __shfl_xor(cs, 32);
      if (kg == 0) colsum[w][col] = cs;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      rg[i] = row_sum(rg[i]);
      rb[i] = row_sum(rb[i]);
      if (r16 == 0) {
        rowg[16 * w + 4 * kg + i] = rg[i];
        rowb[16 * w + 4 * kg + i] = rb[i];
      }
    }
    lds_barrier();
    if (w == 0) {  // dbeta and dg of the head
      float g = rowg[lane], cv = 0, db = bt[lane] - rowb[lane];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        g += red[k][0][lane] - colsum[k][lane];
        cv += red[k][1][lane];
        db += red[k][2][lane];
      }
      double s = (double)g - cv, all = cv;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const double up = __shfl_down(s, d);
        if (lane + d < 64) s += up;
        all += __shfl_xor(all, d);
      }
      s += all + (double)chunk_decay(rows) * ((double)sdot[0] + sdot[1] + sdot[2] + sdot[3]);
      const int64_t t = t0 + lane;
      if (t < p.L) {
        ((float *)p.dg.p)[b * p.dg.s0 + t * p.dg.s1 + h * p.dg.s2] = (float)s;
        store_either<IT>((void *)p.dbeta.p, p.beta32, b * p.dbeta.s0 + t * p.dbeta.s1 + h * p.dbeta.s2, db);
      }
    }
    // dq^ += (A e) K
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf8 B[CT][NK];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) lds_frag_t<NK, KP>(&Kr[0][0][0], kC * KP, 32 * s, 16 * (CT * w + ct), lane, B[ct]);
#pragma unroll
      for (int it = 2 * s; it < 4; ++it) {
        bf8 E[NM];
        lds_frag<NM, kCP>(Es, kC * kCP, 16 * it + r16, 32 * s + 8 * kg, E);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) Yq[it][ct] = mma(E, B[ct], Yq[it][ct]);
      }
    }
    lds_barrier();
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
      bf4 parts[NM];
      split_parts<NM>(E2[jt], parts);
#pragma unroll
      for (int m = 0; m < NM; ++m) *(bf4 *)(Es + (m * kC + 16 * jt + r16) * kCP + 16 * w + 4 * kg) = parts[m];
    }
    lds_barrier();
    // dk^ += (scale A e)^T Q
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf8 B[CT][NK];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) lds_frag_t<NK, KP>(&Qr[0][0][0], kC * KP, 32 * s, 16 * (CT * w + ct), lane, B[ct]);
#pragma unroll
      for (int it = 0; it < 2 + 2 * s; ++it) {
        bf8 E[NM];
        lds_frag<NM, kCP>(Es, kC * kCP, 16 * it + r16, 32 * s + 8 * kg, E);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) Zk[it][ct] = mma(E, B[ct], Zk[it][ct]);
      }
    }
    lds_barrier();
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
      if (jt > w) continue;
      const int col = 16 * jt + r16;
      const float fkc = rows[4 * kC + col];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * w + 4 * kg + i;
        if (col > row) continue;
        float x = -E3[jt][i] * fkc, y = -E3[jt][i] * fkr[i];
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          const __bf16 xq = (__bf16)x, yq = (__bf16)y;
          Es[(m * kC + row) * kCP + col] = xq;
          if (col < row) Es[(m * kC + col) * kCP + row] = yq;
          x -= (float)xq;
          y -= (float)yq;
        }
      }
    }
    lds_barrier();
    // dk^ -= (beta N e and its transpose) K
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf8 B[CT][NK];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) lds_frag_t<NK, KP>(&Kr[0][0][0], kC * KP, 32 * s, 16 * (CT * w + ct), lane, B[ct]);
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        bf8 E[NM];
        lds_frag<NM, kCP>(Es, kC * kCP, 16 * it + r16, 32 * s + 8 * kg, E);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) Zk[it][ct] = mma(E, B[ct], Zk[it][ct]);
      }
    }
    lds_barrier();
  }

  // through the norms: dq = |q|^-1 (dq^ - q^ (q^.dq^)), likewise dk
  if (p.qk_norm) {
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * it + 4 * kg + i;
        float sq = 0, sk = 0;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const int col = 16 * (CT * w + ct) + r16;
          sq = fmaf(lds_elem<NK, KP>(&Qr[0][0][0], kC * KP, row, col), Yq[it][ct][i], sq);
          sk = fmaf(lds_elem<NK, KP>(&Kr[0][0][0], kC * KP, row, col), Zk[it][ct][i], sk);
        }
        sq = row_sum(sq);
        sk = row_sum(sk);
        if (r16 == 0) {
          red[w][0][row] = sq;
          red[w][1][row] = sk;
        }
      }
    lds_barrier();
  }
  IT *dqb = (IT *)p.dq.p + b * p.dq.s0 + hk * p.dq.s2, *dkb = (IT *)p.dk.p + b * p.dk.s0 + hk * p.dk.s2;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int r0 = 16 * it + 4 * kg;
    const f4 fk = row4(rows, 4, r0), fq = row4(rows, 5, r0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = r0 + i;
      float sq = 0, sk = 0;
      if (p.qk_norm) {
        const float nq = fq[i] / p.scale;
        sq = nq * nq * (red[0][0][row] + red[1][0][row] + red[2][0][row] + red[3][0][row]);
        sk = fk[i] * fk[i] * (red[0][1][row] + red[1][1][row] + red[2][1][row] + red[3][1][row]);
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const int col = 16 * (CT * w + ct) + r16;
        if (t0 + row < p.L && col < p.Dk) {
          float y = Yq[it][ct][i], z = Zk[it][ct][i];
          if (p.qk_norm) {
            y = fmaf(-sq, lds_elem<NK, KP>(&Qr[0][0][0], kC * KP, row, col), y);
            z = fmaf(-sk, lds_elem<NK, KP>(&Kr[0][0][0], kC * KP, row, col), z);
          }
          Conv<IT>::store(dqb + (t0 + row) * p.dq.s1 + col, fq[i] * y);
          Conv<IT>::store(dkb + (t0 + row) * p.dk.s1 + col, fk[i] * z);
        }
      }
    }
  }
}

template <typename IT, int DK>
static hipError_t delta_bwd(const DeltaParams &p, hipStream_t s) {
  constexpr int NV = 1;
  hipLaunchKernelGGL((k_delta_bwd<IT, DK, NV>), dim3((unsigned)(p.B * p.H) * (unsigned)((p.Dv + 16 * NV - 1) / (16 * NV))),
                     dim3(kDT), 0, s, p);
  hipLaunchKernelGGL((k_delta_grad<IT, DK>), dim3((unsigned)(p.B * p.Hk) * (unsigned)p.NC), dim3(kDT), 0, s, p);
  return hipGetLastError();
}
template <typename IT>
static hipError_t delta_bwd_k(const DeltaParams &p, hipStream_t s) {
  return p.Dk <= 64 ? delta_bwd<IT, 64>(p, s) : delta_bwd<IT, 128>(p, s);
}
hipError_t launch_delta_bwd(const DeltaParams &p, int dtype, hipStream_t s) {
  const hipError_t e = launch_delta_prep_t(p, dtype, s);
  if (e != hipSuccess) return e;
  return dtype == 0 ? delta_bwd_k<float>(p, s) : dtype == 1 ? delta_bwd_k<bf16_t>(p, s) : delta_bwd_k<f16_t>(p, s);
}

}  // namespace ssm
