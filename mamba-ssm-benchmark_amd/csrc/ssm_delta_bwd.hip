// Gated delta rule, backward of the chunked form (notation: ssm_delta.hpp).  With D the gradient of the state
// leaving a chunk, a = |k|^-1 e^G, c = |k|^-1 e^{G_C - G}, d = scale |q|^-1 e^G, e_ij = e^{G_i - G_j}, and here
// T = (I + strictly lower(beta_i e_ij k_i.k_j))^-1:
//   dU = P^T dO + c K D,  dR = T^T dU,  dV = beta dR,  dbeta = dR.Y (row dots)
//   dS0 = e^{G_C} D + Q^T (d dO) - K^T (beta a dR)
// k_delta_bwd walks the chunks backward, one workgroup per 16 columns of v like the forward, and leaves D and
// dR of every chunk; k_delta_grad then treats every chunk by itself, one workgroup per (batch row, key head,
// chunk), adding the value heads that share the key head in registers.  With U = beta Y and the lower
// triangular J_ij = scale |q_i|^-1 |k_j|^-1 e_ij dO_i.U_j, H_ij = beta_i |k_i|^-1 |k_j|^-1 e_ij dR_i.U_j (i > j):
//   dq' = d dO S0^T + J K,   dk' = c U D^T - beta a dR S0^T + J^T Q - (H + H^T) K
// of which dq, dk are what the norms leave: dq = dq' - q (q.dq') / (|q|^2), likewise dk.
// G enters O_i by a factor e^{G_i}, and every path from v_i by e^{-G_i}, whence G's gradient is dO_i.O_i -
// dV_i.v_i, with dO_i.O_i = q_i.dq'_i since O is linear in q.  The state that leaves has the factor e^{G_C}:
//   dg_t = <D, S1> + sum over i >= t of (q_i.dq'_i - dV_i.v_i),  <D, S1> = e^{G_C} <D, S0> + sum_j k_j.(c U D^T)_j
// Every chunk starts from its own <D, S1>, so that at most 64 terms are added to it.
#include "ssm_delta.hpp"
#include "ssm_dpp.hpp"

namespace ssm {

hipError_t launch_delta_prep_t(const DeltaParams &p, int dtype, hipStream_t s);

template <typename IT, int DK, int NV>
__global__ void __launch_bounds__(kDT, DK * sizeof(IT) * NV <= 256 ? 2 : 1) k_delta_bwd(const DeltaParams p) {
  constexpr int NK = DParts<IT>::in, NM = DParts<IT>::mid, KS = DK / 32, RT = DK / 64;
  __shared__ __align__(16) VTile<NM, DK> Dt[NV];
  __shared__ __align__(16) VTile<NK, kC> Ot[NV];              // dO
  __shared__ __align__(16) VTile<NM, kC> Et[NV], Xt[NV], Yt[NV];  // d dO, dU, -beta a dR
  const int lane = threadIdx.x % 64, w = wave_id(), r16 = lane % 16, kg = lane / 16;
  int bh, vt;
  delta_tile((p.VT + NV - 1) / NV, (int)p.B * p.H, bh, vt);
  vt *= NV;
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk), v0 = 16 * vt + 4 * kg, have = p.Dv - v0;
  const int tok = 16 * w + r16;
  const IT *dop = (const IT *)p.dout.p + b * p.dout.s0 + h * p.dout.s2 + v0;
  IT *dvp = (IT *)p.dv.p + b * p.dv.s0 + h * p.dv.s2 + v0;
  const int64_t ch0 = (int64_t)bh * p.NC, kch0 = ((int64_t)b * p.Hk + hk) * p.NC;

  f4 D[NV][RT];  // D[key][v0 + 16 n + i] of key 16 (RT w + r) + r16
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int key = 16 * (RT * w + r) + r16;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        D[n][r][i] = p.dlast && key < p.Dk && 16 * n + i < have ? p.dlast[((int64_t)bh * p.Dk + key) * p.Dv + v0 + 16 * n + i] : 0.0f;
    }
  bf8 K[KS][NK], T[2][NM], P[2][NM], Kt[RT][2][NK], Qt[RT][2][NK];
  Raw4<IT> go[NV];
  f4 row;  // a, beta, c, d of the token
  float eC;
  auto load_rows = [&](int c) {
    row = token_row(delta_rows(p, ch0 + c), tok);
    eC = chunk_decay(delta_rows(p, ch0 + c));
  };
  auto load_o = [&](int c) {
    const int64_t t = (int64_t)c * kC + tok;
#pragma unroll
    for (int n = 0; n < NV; ++n)
      go[n] = load4(dop + t * p.dout.s1 + 16 * n, (const IT *)p.dout.p, t < p.L ? have - 16 * n : 0, p.vdo);
  };
  auto load_kp = [&](int c) {  // the transposes of T and P are upper triangular
    const __bf16 *k = key_frags<DK, NK>(p.fK, kch0 + c);
#pragma unroll
    for (int s = 0; s < KS; ++s) load_frag<NK>(k, kC * DK, w * KS + s, lane, K[s]);
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (s >= w / 2) load_frag<NM>((const __bf16 *)p.fP + (ch0 + c) * NM * kFrag, kFrag, 2 * w + s, lane, P[s]);
  };
  auto load_t = [&](int c) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (s >= w / 2) load_frag<NM>((const __bf16 *)p.fT + (ch0 + c) * NM * kFrag, kFrag, 2 * w + s, lane, T[s]);
  };
  auto load_cols = [&](const void *m, int c, bf8 (&f)[RT][2][NK]) {
    const __bf16 *kt = key_frags<DK, NK>(m, kch0 + c);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < RT; ++r) load_frag<NK>(kt, kC * DK, 2 * (RT * w + r) + s, lane, f[r][s]);
  };
  load_rows(p.NC - 1);
  load_o(p.NC - 1);
  load_kp(p.NC - 1);
  load_t(p.NC - 1);
  load_cols(p.fQt, p.NC - 1, Qt);
  load_cols(p.fKt, p.NC - 1, Kt);
  for (int c = p.NC - 1; c >= 0; --c) {
    const int64_t t = (int64_t)c * kC + tok, ch = ch0 + c;
    const int next = c ? c - 1 : 0;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int key = 16 * (RT * w + r) + r16;
        Dt[n].put(key, kg, D[n][r]);
        if (key < p.Dkp && vt + n < p.VT)
          *(f4 *)(state_of(p.dstates, p, ch, vt + n) + (unsigned)(16 * key + 4 * kg)) = D[n][r];
      }
      bf4 o[NK];
      const bool live = t < p.L && have - 16 * n > 0;
      to_parts<IT, NK>(go[n], live, o);
      Ot[n].put_parts(tok, kg, o);
      Et[n].put(tok, kg, row[3] * to_f4<IT>(go[n], live));
    }
    const float cc = row[2], bu = row[1], by = -row[1] * row[0], decay = eC;
    load_rows(next);
    load_o(next);
    lds_barrier();
    f4 x[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) x[n] = 0;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        bf8 A[NM];
        Dt[n].get(s, lane, A);
        x[n] = mma<NM>(A, K[s], x[n]);
      }
#pragma unroll
    for (int n = 0; n < NV; ++n) x[n] *= cc;
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (s >= w / 2) {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          bf8 A[NK];
          Ot[n].get(s, lane, A);
          x[n] = mma<NM>(A, P[s], x[n]);
        }
      }
#pragma unroll
    for (int n = 0; n < NV; ++n) Xt[n].put(tok, kg, x[n]);
    load_kp(next);
    lds_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s)  // dR = dU + (T^T - I) dU
      if (s >= w / 2) {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          bf8 A[NM];
          Xt[n].get(s, lane, A);
          x[n] = mma<NM>(A, T[s], x[n]);
        }
      }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      Yt[n].put(tok, kg, by * x[n]);
      if (vt + n < p.VT) *(f4 *)(value_of(p.dr, p, ch, vt + n) + (unsigned)(16 * tok + 4 * kg)) = x[n];
      store4(dvp + t * p.dv.s1 + 16 * n, (f4)(bu * x[n]), t < p.L ? have - 16 * n : 0, p.vdv);
#pragma unroll
      for (int r = 0; r < RT; ++r) D[n][r] *= decay;
    }
    load_t(next);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        bf8 A[NM];
        Et[n].get(s, lane, A);
#pragma unroll
        for (int r = 0; r < RT; ++r) D[n][r] = mma<NM>(A, Qt[r][s], D[n][r]);
      }
    load_cols(p.fQt, next, Qt);
    lds_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        bf8 A[NM];
        Yt[n].get(s, lane, A);
#pragma unroll
        for (int r = 0; r < RT; ++r) D[n][r] = mma<NM>(A, Kt[r][s], D[n][r]);
      }
    load_cols(p.fKt, next, Kt);
  }
  if (p.dh0) {
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int key = 16 * (RT * w + r) + r16;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (key < p.Dk && 16 * n + i < have) p.dh0[((int64_t)bh * p.Dk + key) * p.Dv + v0 + 16 * n + i] = D[n][r][i];
      }
  }
}

__device__ __forceinline__ float kg_sum(float v) {  // over the four lanes of a column
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Wavefront w owns keys 16 w .. 16 w + 15 (DK / 16 wavefronts).  Results are transposed, so that a lane
// holds 4 keys of one token.  The values are staged 32 columns at a time, as fragments in two buffers, the
// states go from memory to registers, both one slab ahead.
template <typename IT, int DK>
__global__ void __launch_bounds__(4 * DK) k_delta_grad(const DeltaParams p) {
  constexpr int NK = DParts<IT>::in, NM = DParts<IT>::mid, NP = DParts<IT>::out, NT = 4 * DK, NW = DK / 16;
  constexpr int NJ = 16 / NW;                    // tiles of J and H per wavefront
  constexpr int SF = 4 * 64 * 8;                 // staged elements of one part: 64 tokens x 32 columns
  constexpr int kStage = (NK + NM + NP) * SF, JP = kC + 8, kE = (NM + NP) * kC * JP, PT = 512 / NT;
  __shared__ __align__(16) __bf16 buf[2 * kStage > kE ? 2 * kStage : kE];  // dO, U, dR; then J and H
  __shared__ double Gs[kC];
  __shared__ float red[NW][2][kC], rowb[kC], rowv[kC], sdot[NW];
  const int tid = threadIdx.x, lane = tid % 64, w = wave_id(), r16 = lane % 16, kg = lane / 16;
  const int c = blockIdx.x % p.NC, bk = blockIdx.x / p.NC, b = bk / p.Hk, hk = bk % p.Hk, group = p.H / p.Hk;
  const int64_t t0 = (int64_t)c * kC, kch = (int64_t)bk * p.NC + c;
  const int wi = w * NJ / 4, wj = w * NJ % 4;    // J's tiles (wi, wj .. wj + NJ - 1)
  const bool keys = 16 * w < p.Dkp;
  const __bf16 *fK = key_frags<DK, NK>(p.fK, kch), *fQ = key_frags<DK, NK>(p.fQ, kch);
  const __bf16 *fKt = key_frags<DK, NK>(p.fKt, kch), *fQt = key_frags<DK, NK>(p.fQt, kch);
  // Makes the compiler read K and Q anew where they are used: kept over the slabs, they would spill.
  auto reread = [&] { asm volatile("" : "+s"(fK), "+s"(fQ), "+s"(fKt), "+s"(fQt)); };
  const int slabs = (p.VT + 1) / 2;
  const int64_t ao = r16 * p.dout.s1 + 4 * kg, av = r16 * p.v.s1 + 4 * kg;
  __bf16 *const Jm = buf, *const Hm = buf + NM * kC * JP;

  // K or Q of token 16 it + r16, keys 16 w + 4 kg + i
  auto elems = [&](const __bf16 *f, int it) {
    f4 x = 0;
#pragma unroll
    for (int n = NK - 1; n >= 0; --n)
      x += __builtin_convertvector(*(const bf4 *)(f + n * kC * DK + (it * (DK / 32) + w / 2) * 512 + 4 * (w % 2) + (unsigned)(lane * 8)), f4);
    return x;
  };

  f4 Yq[4], Zk[4];  // dq', dk' of token 16 it + r16, keys 16 w + 4 kg + i
#pragma unroll
  for (int it = 0; it < 4; ++it) Yq[it] = Zk[it] = 0;
  const float *rows = nullptr;

  for (int hg = 0; hg < group; ++hg) {
    const int h = hk * group + hg;
    const int64_t ch = ((int64_t)b * p.H + h) * p.NC + c;
    rows = delta_rows(p, ch);
    const IT *dop = (const IT *)p.dout.p + b * p.dout.s0 + h * p.dout.s2, *vp = (const IT *)p.v.p + b * p.v.s0 + h * p.v.s2;
    f4 F1[4], F2[4], F3[4], A[NJ], N[NJ];  // S0 dO^T, D U^T, S0 dR^T; tiles of dO U^T, dR U^T, transposed
#pragma unroll
    for (int it = 0; it < 4; ++it) F1[it] = F2[it] = F3[it] = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) A[j] = N[j] = 0;
    float sd = 0, rv[PT], rb[PT];  // <S0, D>; dR.v and dR.Y of the staged tokens
    f4 sv[2], dv[2], yv[PT], xv[PT];
    Raw4<IT> go[PT], vv[PT];
    // staged piece x of this thread: half sh of the slab, token st, columns 4 kg + i
    auto stage_of = [&](int x, int &sh, int &it) {
      sh = (w + x * NW) / 4;
      it = (w + x * NW) % 4;
    };
    auto load = [&](int s) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int vt = 2 * s + x;
        const bool in = keys && vt < p.VT;
        sv[x] = in ? *(const f4 *)(state_of(p.states, p, ch, vt) + 256 * w + (unsigned)(16 * r16 + 4 * kg)) : (f4)0.0f;
        dv[x] = in ? *(const f4 *)(state_of(p.dstates, p, ch, vt) + 256 * w + (unsigned)(16 * r16 + 4 * kg)) : (f4)0.0f;
      }
#pragma unroll
      for (int x = 0; x < PT; ++x) {
        int sh, it;
        stage_of(x, sh, it);
        const int vt = 2 * s + sh, have = t0 + 16 * it + r16 < p.L ? p.Dv - 16 * vt - 4 * kg : 0;
        yv[x] = vt < p.VT ? *(const f4 *)(value_of(p.y, p, ch, vt) + 256 * it + (unsigned)(16 * r16 + 4 * kg)) : (f4)0.0f;
        xv[x] = vt < p.VT ? *(const f4 *)(value_of(p.dr, p, ch, vt) + 256 * it + (unsigned)(16 * r16 + 4 * kg)) : (f4)0.0f;
        go[x] = load4(dop + (t0 + 16 * it) * p.dout.s1 + 16 * vt + ao, (const IT *)p.dout.p, have, p.vdo);
        vv[x] = load4(vp + (t0 + 16 * it) * p.v.s1 + 16 * vt + av, (const IT *)p.v.p, have, p.vv);
      }
    };
    load(0);
    if (tid < kC) Gs[tid] = ((const double *)(rows + 6 * kC))[tid];
#pragma unroll
    for (int x = 0; x < PT; ++x) rv[x] = rb[x] = 0;
    for (int s = 0; s < slabs; ++s) {
      __bf16 *const Os = buf + (s & 1) * kStage, *const Us = Os + NK * SF, *const Rs = Us + NM * SF;
#pragma unroll
      for (int x = 0; x < PT; ++x) {
        int sh, it;
        stage_of(x, sh, it);
        const int at = (it * 64 + lane) * 8 + 4 * sh;
        const float be = rows[4 * (16 * it + r16) + 1];
        bf4 o[NK], u[NM], r[NP];
        const bool live = t0 + 16 * it + r16 < p.L && p.Dv - 32 * s - 16 * sh - 4 * kg > 0;
        to_parts<IT, NK>(go[x], live, o);
        split_parts<NM>((f4)(be * yv[x]), u);
        split_parts<NP>(xv[x], r);
        const f4 v = to_f4<IT>(vv[x], live);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          rv[x] = fmaf(xv[x][i], v[i], rv[x]);
          rb[x] = fmaf(xv[x][i], yv[x][i], rb[x]);
        }
#pragma unroll
        for (int n = 0; n < NK; ++n) *(bf4 *)(Os + n * SF + at) = o[n];
#pragma unroll
        for (int n = 0; n < NM; ++n) *(bf4 *)(Us + n * SF + at) = u[n];
#pragma unroll
        for (int n = 0; n < NP; ++n) *(bf4 *)(Rs + n * SF + at) = r[n];
      }
      bf8 SA[NM], DA[NM];
      {
        const f8 x = __builtin_shufflevector(sv[0], sv[1], 0, 1, 2, 3, 4, 5, 6, 7);
        const f8 y = __builtin_shufflevector(dv[0], dv[1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int j = 0; j < 8; ++j) sd = fmaf(x[j], y[j], sd);
        split_parts<NM>(x, SA);
        split_parts<NM>(y, DA);
      }
      if (s + 1 < slabs) load(s + 1);
      lds_barrier();  // the other buffer's readers are a barrier behind
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        bf8 O[NK], U[NM], R[NP];
        load_frag<NK>(Os, SF, it, lane, O);
        load_frag<NM>(Us, SF, it, lane, U);
        load_frag<NP>(Rs, SF, it, lane, R);
        F1[it] = mma<NM>(SA, O, F1[it]);
        F3[it] = mma<NP>(SA, R, F3[it]);
        F2[it] = mma<NM>(DA, U, F2[it]);
        if (it == wi) {
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            if (wj + j <= wi) {
              bf8 Uj[NM];
              load_frag<NM>(Us, SF, wj + j, lane, Uj);
              A[j] = mma<NM>(Uj, O, A[j]);
              N[j] = mma<NP>(Uj, R, N[j]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // one token tile's operands in registers at a time
      }
    }
    sd = group_sum<64>(sd);
    if (lane == 0) sdot[w] = sd;
#pragma unroll
    for (int x = 0; x < PT; ++x) {
      rv[x] = kg_sum(rv[x]);
      rb[x] = kg_sum(rb[x]);
    }
    lds_barrier();  // the slabs are read; red, rowv and rowb of the head before are too
    // the two halves of the slabs are wavefronts 0..3 and 4..7, or one wavefront's two pieces
    if constexpr (PT == 2) {
      if (kg == 0) {
        rowv[16 * w + r16] = rv[0] + rv[PT - 1];
        rowb[16 * w + r16] = rb[0] + rb[PT - 1];
      }
    } else if (w >= 4 && kg == 0) {
      rowv[16 * (w - 4) + r16] = rv[0];
      rowb[16 * (w - 4) + r16] = rb[0];
    }
    {  // J and H
      const int i = 16 * wi + r16;
      const float fqi = rows[5 * kC + i], fki = rows[4 * kC + i] * rows[4 * i + 1];
      const double Gi = Gs[i];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        f4 jv, hv;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int jj = 16 * (wj + j) + 4 * kg + x;
          const float e = jj <= i ? fexp((float)(Gi - Gs[jj])) * rows[4 * kC + jj] : 0.0f;
          jv[x] = jj <= i ? fqi * e * A[j][x] : 0.0f;
          hv[x] = jj < i ? -fki * e * N[j][x] : 0.0f;
        }
        bf4 jp[NM], hp[NP];
        split_parts<NM>(jv, jp);
        split_parts<NP>(hv, hp);
#pragma unroll
        for (int n = 0; n < NM; ++n) *(bf4 *)(Jm + (n * kC + i) * JP + 16 * (wj + j) + 4 * kg) = jp[n];
#pragma unroll
        for (int n = 0; n < NP; ++n) *(bf4 *)(Hm + (n * kC + i) * JP + 16 * (wj + j) + 4 * kg) = hp[n];
      }
    }
    reread();
    bf8 Kt[2][NK], Qt[2][NK];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      load_frag<NK>(fKt, kC * DK, 2 * w + s, lane, Kt[s]);
      load_frag<NK>(fQt, kC * DK, 2 * w + s, lane, Qt[s]);
    }
    float cd = 0;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int tok = 16 * it + r16;
      const f4 row = token_row(rows, tok), ke = elems(fK, it), f2 = row[2] * F2[it];
#pragma unroll
      for (int i = 0; i < 4; ++i) cd = fmaf(ke[i], f2[i], cd);
      F1[it] *= row[3];
      Zk[it] += f2 - (row[1] * row[0]) * F3[it];
    }
    cd = group_sum<64>(cd);
    if (lane == 0) red[w][1][0] = cd;
    lds_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const int at = (16 * it + r16) * JP + 32 * s + 4 * kg;                                   // row it, columns of step s
        const int tr = (32 * s + 4 * kg + r16 / 4) * JP + 16 * it + 4 * (r16 % 4);               // rows of step s, column it
        if (s <= it / 2) {
          bf8 B[NM], C[NP];
#pragma unroll
          for (int n = 0; n < NM; ++n) {
            const __bf16 *m = Jm + n * kC * JP + at;
            B[n] = __builtin_shufflevector(*(const bf4 *)m, *(const bf4 *)(m + 16), 0, 1, 2, 3, 4, 5, 6, 7);
          }
#pragma unroll
          for (int n = 0; n < NP; ++n) {
            const __bf16 *m = Hm + n * kC * JP + at;
            C[n] = __builtin_shufflevector(*(const bf4 *)m, *(const bf4 *)(m + 16), 0, 1, 2, 3, 4, 5, 6, 7);
          }
          F1[it] = mma<NM>(Kt[s], B, F1[it]);
          Zk[it] = mma<NP>(Kt[s], C, Zk[it]);
        }
        if (s >= it / 2) {
          bf8 B[NP], C[NP];
#pragma unroll
          for (int n = 0; n < NP; ++n) {
            B[n] = read_tr(Jm + n * kC * JP + tr, Jm + (n * kC + 16) * JP + tr);
            C[n] = read_tr(Hm + n * kC * JP + tr, Hm + (n * kC + 16) * JP + tr);
          }
          Zk[it] = mma<NP>(Qt[s], B, Zk[it]);
          Zk[it] = mma<NP>(Kt[s], C, Zk[it]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const f4 q = elems(fQ, it) * F1[it];
      const float x = kg_sum((q[0] + q[1]) + (q[2] + q[3]));
      if (kg == 0) red[w][0][16 * it + r16] = x;
      Yq[it] += F1[it];
    }
    if constexpr (PT == 1) {
      if (w < 4 && kg == 0) {
        rowv[16 * w + r16] += rv[0];
        rowb[16 * w + r16] += rb[0];
      }
    }
    lds_barrier();
    if (w == 0) {  // dbeta and dg of the head
      const float db = rowb[lane];
      double s = -(double)rows[4 * lane + 1] * rowv[lane], all = 0, ss = 0;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        s += red[k][0][lane];
        all += red[k][1][0];
        ss += sdot[k];
      }
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const double up = __shfl_down(s, d);
        if (lane + d < 64) s += up;
      }
      s += all + (double)chunk_decay(rows) * ss;
      const int64_t t = t0 + lane;
      if (t < p.L) {
        ((float *)p.dg.p)[b * p.dg.s0 + t * p.dg.s1 + h * p.dg.s2] = (float)s;
        store_either<IT>((void *)p.dbeta.p, p.beta32, b * p.dbeta.s0 + t * p.dbeta.s1 + h * p.dbeta.s2, db);
      }
    }
    lds_barrier();  // J, H, Gs and sdot are read
  }

  // through the norms
  reread();
  if (p.qk_norm) {
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const f4 q = elems(fQ, it) * Yq[it], k = elems(fK, it) * Zk[it];
      const float sq = kg_sum((q[0] + q[1]) + (q[2] + q[3])), sk = kg_sum((k[0] + k[1]) + (k[2] + k[3]));
      if (kg == 0) {
        red[w][0][16 * it + r16] = sq;
        red[w][1][16 * it + r16] = sk;
      }
    }
    lds_barrier();
  }
  IT *dqb = (IT *)p.dq.p + b * p.dq.s0 + hk * p.dq.s2, *dkb = (IT *)p.dk.p + b * p.dk.s0 + hk * p.dk.s2;
  const int e = 16 * w + 4 * kg;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int tok = 16 * it + r16, have = t0 + tok < p.L ? p.Dk - e : 0;
    f4 y = Yq[it], z = Zk[it];
    if (p.qk_norm) {
      float sq = 0, sk = 0;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        sq += red[k][0][tok];
        sk += red[k][1][tok];
      }
      const float fk = rows[4 * kC + tok], nq = rows[5 * kC + tok] / p.scale;
      y -= (nq * nq * sq) * elems(fQ, it);
      z -= (fk * fk * sk) * elems(fK, it);
    }
    store4(dqb + (t0 + tok) * p.dq.s1 + e, y, have, p.vdq);
    store4(dkb + (t0 + tok) * p.dk.s1 + e, z, have, p.vdk);
  }
}

template <typename IT, int DK>
static hipError_t delta_bwd(const DeltaParams &p, hipStream_t s) {
  if (delta_pairs(p))
    hipLaunchKernelGGL((k_delta_bwd<IT, DK, 2>), dim3((unsigned)(p.B * p.H) * (unsigned)((p.VT + 1) / 2)), dim3(kDT), 0, s, p);
  else
    hipLaunchKernelGGL((k_delta_bwd<IT, DK, 1>), dim3((unsigned)(p.B * p.H) * (unsigned)p.VT), dim3(kDT), 0, s, p);
  hipLaunchKernelGGL((k_delta_grad<IT, DK>), dim3((unsigned)(p.B * p.Hk) * (unsigned)p.NC), dim3(4 * DK), 0, s, p);
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
