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
// of which dq, dk are what the norms leave: dq = dq' - q (q.dq') / |q|^2, likewise dk.
// G's gradient dG_i: every product of a pair i > j, J_ij q_i.k_j of the outputs and H_ij k_i.k_j of the system,
// has a factor e^{G_i - G_j} and enters row i and, with the other sign, column j, so that in the sum from t on a
// pair that does not straddle t cancels to its rounding; J's diagonal has no factor and is kept apart.  The
// state that enters has e^{G_i} in row i; what goes into the leaving state has e^{G_C - G_j}:
//   dG_i = q_i.(d dO S0^T + J K)_i + k_i.(H K - J^T Q - H^T K - beta a dR S0^T)_i   (J, H below the diagonal; H with its sign)
//   dg_t = sum over i >= t of dG_i + sum over j < t of k_j.(c U D^T)_j + e^{G_C} <D, S0>
#include "ssm_delta.hpp"

namespace ssm {

hipError_t launch_delta_prep_t(const DeltaParams &p, int dtype, hipStream_t s);

// As in the forward, four wavefronts walk the chain and four more prepare what it takes: P^T dO of the chunk
// to come, d dO and Q^T (d dO), and they store D, dR and dV.  Same bounds as the forward: B4 L4096 H16 Hk8
// 128 x 128 bf16 274 us (576 in the first version).
template <typename IT, int DK, int NV>
__global__ void __launch_bounds__(2 * kDT) SSM_TWO_WAVES k_delta_bwd(const DeltaParams p) {
  constexpr int NK = DParts<IT>::in, NM = DParts<IT>::mid, KS = DK / 32, RT = DK / 64;
  __shared__ __align__(16) VTile<NM, DK> Dt[NV];
  __shared__ __align__(16) VTile<NK, kC> Ot[NV];                  // dO
  __shared__ __align__(16) VTile<NM, kC> Et[NV], Xt[NV], Yt[NV];  // d dO, dU, -beta a dR
  __shared__ __align__(16) f4 Gt[NV][kDT], Rt[NV][RT][kDT], Zt[NV][kDT];  // P^T dO, Q^T (d dO), dR, by lane
  const int lane = threadIdx.x % 64, w = wave_id() % 4, r16 = lane % 16, kg = lane / 16, me = threadIdx.x % kDT;
  int bh, vt;
  delta_tile(p, NV, bh, vt);
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk), v0 = 16 * vt + 4 * kg, have = p.Dv - v0;
  const int tok = 16 * w + r16;
  auto at = [&](int c) { return (int64_t)c * p.B * p.H + bh; };
  auto kat = [&](int c) { return ((int64_t)c * p.B + b) * p.Hk + hk; };
  auto load_cols = [&](const void *m, int c, bf8 (&f)[RT][2][NK]) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < RT; ++r) load_frag<NK>(key_frags<DK, NK>(m, kat(c)), kC * DK, 2 * (RT * w + r) + s, lane, f[r][s]);
  };

  if (wave_id() < 4) {
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
    bf8 K[KS][NK], T[2][NM], Kt[RT][2][NK];
    f4 row;  // a, beta, c of the token, e^{G_C}
    auto load_k = [&](int c) {
#pragma unroll
      for (int s = 0; s < KS; ++s) load_frag<NK>(key_frags<DK, NK>(p.fK, kat(c)), kC * DK, w * KS + s, lane, K[s]);
      row = token_row(delta_rows(p, at(c)), tok);
    };
    auto load_t = [&](int c) {  // the transpose of T is upper triangular
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s >= w / 2) load_frag<NM>((const __bf16 *)p.fT + at(c) * NM * kFrag, kFrag, 2 * w + s, lane, T[s]);
    };
    load_k(p.NC - 1);
    load_t(p.NC - 1);
    load_cols(p.fKt, p.NC - 1, Kt);
    lds_barrier();  // the first chunk's dO
    for (int c = p.NC - 1; c >= 0; --c) {
      const int next = c ? c - 1 : 0;
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int r = 0; r < RT; ++r) Dt[n].put(16 * (RT * w + r) + r16, kg, D[n][r]);
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
      read_ahead<KS * NM * 2 * NV, KS * products(NM, NM, NK) * NV, 12>();
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        x[n] = row[2] * x[n] + Gt[n][me];
        Xt[n].put(tok, kg, x[n]);
      }
      const float by = -row[1] * row[0], decay = row[3];
      load_k(next);
      lds_barrier();
      bf8 X[NV][2][NM];
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        Xt[n].get(1, lane, X[n][1]);
        Xt[n].get(0, lane, X[n][0]);
      }
#pragma unroll
      for (int s = 1; s >= 0; --s)  // dR = dU + (T^T - I) dU
        if (s >= w / 2) {
#pragma unroll
          for (int n = 0; n < NV; ++n) x[n] = mma<NM>(X[n][s], T[s], x[n]);
        }
      auto put_r = [&] {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          Yt[n].put(tok, kg, by * x[n]);
          Zt[n][me] = x[n];
        }
      };
      put_r();
      load_t(next);
      if (__builtin_expect(not_finite(x), 0)) {
        f4 before[NV];
#pragma unroll
        for (int n = 0; n < NV; ++n) before[n] = Xt[n].value(tok, kg);
        if (not_finite_of(x, before)) {
#pragma unroll
          for (int n = 0; n < NV; ++n)
            x[n] = row_times<NM>((const __bf16 *)p.fT + at(c) * NM * kFrag, tok, tok + 1, kC, Xt[n], kg, before[n]);
          put_r();
        }
      }
      lds_barrier();
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int r = 0; r < RT; ++r) D[n][r] = decay * D[n][r] + Rt[n][r][me];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          bf8 A[NM];
          Yt[n].get(s, lane, A);
#pragma unroll
          for (int r = 0; r < RT; ++r) D[n][r] = mma<NM>(A, Kt[r][s], D[n][r]);
        }
      read_ahead<2 * NM * 2 * NV, 2 * products(NM, NM, NK) * RT * NV, 12>();
      load_cols(p.fKt, next, Kt);
    }
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int key = 16 * (RT * w + r) + r16;
        if (key < p.Dkp && vt + n < p.VT)  // behind the chunks' own
          *(f4 *)(state_of(p.dstates, p, at(p.NC), vt + n) + (unsigned)(16 * key + 4 * kg)) = D[n][r];
        if (p.dh0) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key < p.Dk && 16 * n + i < have) p.dh0[((int64_t)bh * p.Dk + key) * p.Dv + v0 + 16 * n + i] = D[n][r][i];
        }
      }
  } else {
    const IT *dop = (const IT *)p.dout.p + b * p.dout.s0 + h * p.dout.s2 + v0;
    IT *dvp = (IT *)p.dv.p + b * p.dv.s0 + h * p.dv.s2 + v0;
    bf8 P[2][NM], Qt[RT][2][NK];
    Raw4<IT> go[NV], next_go[NV];  // dO of this chunk and of the one to come
    auto load_o = [&](int c, Raw4<IT> (&g)[NV]) {
      const int64_t t = (int64_t)c * kC + tok;
#pragma unroll
      for (int n = 0; n < NV; ++n)
        g[n] = load4(dop + t * p.dout.s1 + 16 * n, (const IT *)p.dout.p, t < p.L ? have - 16 * n : 0, p.vdo);
    };
    auto load_p = [&](int c) {  // so is that of P
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s >= w / 2) load_frag<NM>((const __bf16 *)p.fP + at(c) * NM * kFrag, kFrag, 2 * w + s, lane, P[s]);
    };
    auto put_o = [&](int c, Raw4<IT> (&g)[NV]) {
      const int64_t t = (int64_t)c * kC + tok;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        bf4 o[NK];
        to_parts<IT, NK>(g[n], t < p.L && have - 16 * n > 0, o);
        Ot[n].put_parts(tok, kg, o);
      }
    };
    auto make_g = [&](int c) {
      f4 g[NV];
#pragma unroll
      for (int n = 0; n < NV; ++n) g[n] = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s >= w / 2) {
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            bf8 A[NK];
            Ot[n].get(s, lane, A);
            g[n] = mma<NM>(A, P[s], g[n]);
          }
        }
      if (__builtin_expect(not_finite(g), 0)) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
          g[n] = row_times<NM>((const __bf16 *)p.fP + at(c) * NM * kFrag, tok, tok, kC, Ot[n], kg, (f4)0.0f);
      }
#pragma unroll
      for (int n = 0; n < NV; ++n) Gt[n][me] = g[n];
    };
    load_o(p.NC - 1, go);
    load_p(p.NC - 1);
    load_cols(p.fQt, p.NC - 1, Qt);
    float beta = delta_rows(p, at(p.NC - 1))[(unsigned)(4 * tok + 1)], d = delta_rows(p, at(p.NC - 1))[8 * kC + (unsigned)tok];
    put_o(p.NC - 1, go);
    load_o(p.NC > 1 ? p.NC - 2 : 0, next_go);
    lds_barrier();
    make_g(p.NC - 1);
    load_p(p.NC > 1 ? p.NC - 2 : 0);
    for (int c = p.NC - 1; c >= 0; --c) {
      const int64_t t = (int64_t)c * kC + tok;
      const int next = c ? c - 1 : 0, after = c > 1 ? c - 2 : 0;
      const float be = beta, fd = d;
      lds_barrier();
#pragma unroll
      for (int n = 0; n < NV; ++n) Et[n].put(tok, kg, fd * to_f4<IT>(go[n], t < p.L && have - 16 * n > 0));
      put_o(next, next_go);
#pragma unroll
      for (int n = 0; n < NV; ++n) go[n] = next_go[n];
      load_o(after, next_go);
      beta = delta_rows(p, at(next))[(unsigned)(4 * tok + 1)];
      d = delta_rows(p, at(next))[8 * kC + (unsigned)tok];
      f4 D[NV][RT];
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int r = 0; r < RT; ++r) D[n][r] = Dt[n].whole(16 * (RT * w + r) + r16, kg);
      lds_barrier();
      f4 R[NV][RT];
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int r = 0; r < RT; ++r) R[n][r] = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          bf8 A[NM];
          Et[n].get(s, lane, A);
#pragma unroll
          for (int r = 0; r < RT; ++r) R[n][r] = mma<NM>(A, Qt[r][s], R[n][r]);
        }
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int r = 0; r < RT; ++r) Rt[n][r][me] = R[n][r];
      make_g(next);
      load_cols(p.fQt, next, Qt);
      load_p(after);
      lds_barrier();
      // no store stands before a barrier that the chain has to wait at
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const f4 x = Zt[n][me];
        if (vt + n < p.VT) {
          *(f4 *)(value_of(p.dr, p, at(c), vt + n) + (unsigned)(16 * tok + 4 * kg)) = x;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const int key = 16 * (RT * w + r) + r16;
            if (key < p.Dkp) *(f4 *)(state_of(p.dstates, p, at(c), vt + n) + (unsigned)(16 * key + 4 * kg)) = D[n][r];
          }
        }
        store4(dvp + t * p.dv.s1 + 16 * n, (f4)(be * x), t < p.L ? have - 16 * n : 0, p.vdv);
      }
    }
  }
}

// Wavefront w owns keys 16 w .. 16 w + 15 (DK / 16 wavefronts).  Results are transposed, so that a lane
// holds 4 keys of one token.  The values are staged 32 columns (a slab) at a time, as fragments in two buffers,
// the states go from memory to registers, both one slab ahead; what the products of the chunk's end want is
// read during the last slab.  One workgroup of eight wavefronts fills a compute unit's registers at DK = 128 (F1,
// F2, F3 alone are 48 of them), so a slab's phases add up: 1.5 us of products, 0.7 of splitting, the rest
// barriers.  B4 L4096 H16 Hk8 128 x 128 bf16: 365 us for 0.7 GB (779 with 16 keys by two tiles a wavefront of
// four, which spilled); B16 L512 H8 64 x 64 float32: 58 us.  SHARED: several value heads add to dq', dk', which wait in LDS meanwhile.
template <typename IT, int DK, bool SHARED>
__global__ void __launch_bounds__(4 * DK) SSM_TWO_WAVES k_delta_grad(const DeltaParams p) {
  constexpr int NK = DParts<IT>::in, NM = DParts<IT>::mid, NT = 4 * DK, NW = DK / 16;
  constexpr int NJ = 16 / NW;                    // tiles of J and H per wavefront
  constexpr int SF = 4 * 64 * 8;                 // staged elements of one part: 64 tokens x 32 columns
  constexpr int kStage = (NK + 2 * NM) * SF, JP = kC + 8, kE = 2 * NM * kC * JP, PT = 512 / NT;
  __shared__ __align__(16) __bf16 buf[2 * kStage > kE ? 2 * kStage : kE];  // dO, U, dR; then J and H
  __shared__ __align__(16) f4 sum[SHARED ? 8 : 1][SHARED ? NT : 1];
  __shared__ __align__(16) float rows[kDeltaRows];
  __shared__ float red[NW][2][kC], norm[NW][2][kC], rowb[kC], diag[kC], sdot[NW];
  const int tid = threadIdx.x, lane = tid % 64, w = wave_id(), r16 = lane % 16, kg = lane / 16;
  const int keyed = (int)p.B * p.Hk, c = blockIdx.x / keyed, bk = blockIdx.x % keyed, b = bk / p.Hk, hk = bk % p.Hk, group = SHARED ? p.H / p.Hk : 1;
  const int64_t t0 = (int64_t)c * kC, kch = blockIdx.x;
  const int wi = w * NJ / 4, wj = w * NJ % 4;    // J's tiles (wi, wj .. wj + NJ - 1)
  const bool keys = 16 * w < p.Dkp;
  const int slabs = (p.VT + 1) / 2;
  const int64_t ao = r16 * p.dout.s1 + 4 * kg;
  const unsigned at16 = 16 * r16 + 4 * kg;
  __bf16 *const Jm = buf, *const Hm = buf + NM * kC * JP;

  bf8 Kt[2][NK], Qt[2][NK];  // K and Q by columns: keys 16 w + r16
  bf4 Ke[4][NK], Qe[4][NK];  // K and Q of token 16 it + r16, keys 16 w + 4 kg + i
  const __bf16 *kt = key_frags<DK, NK>(p.fKt, kch), *qt = key_frags<DK, NK>(p.fQt, kch);
  const __bf16 *kr = key_frags<DK, NK>(p.fK, kch), *qr = key_frags<DK, NK>(p.fQ, kch);
  auto load_keys = [&](int it) {
    asm volatile("" : "+s"(kt), "+s"(qt), "+s"(kr), "+s"(qr));  // read for every head anew: kept over its slabs, they would spill
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const int at = n * kC * DK + (it * (DK / 32) + w / 2) * 512 + 4 * (w % 2);
      Ke[it][n] = *(const bf4 *)(kr + at + (unsigned)(lane * 8));
      Qe[it][n] = *(const bf4 *)(qr + at + (unsigned)(lane * 8));
    }
    load_frag<NK>(it < 2 ? kt : qt, kC * DK, 2 * w + it % 2, lane, it < 2 ? Kt[it % 2] : Qt[it % 2]);
  };
  auto whole = [](const bf4 (&x)[NK]) {
    f4 r = __builtin_convertvector(x[NK - 1], f4);
#pragma unroll
    for (int n = NK - 2; n >= 0; --n) r += __builtin_convertvector(x[n], f4);
    return r;
  };

  f4 Y[4], Z[4];  // dq', dk' of token 16 it + r16, keys 16 w + 4 kg + i
  for (int hg = 0; hg < group; ++hg) {
    const int h = hk * group + hg;
    const int64_t ch = ((int64_t)c * p.B + b) * p.H + h;
    const IT *dop = (const IT *)p.dout.p + b * p.dout.s0 + h * p.dout.s2 + t0 * p.dout.s1;
    const float *Sp = state_of(p.states, p, ch, 0) + (keys ? 256 * w : 0), *Dp = state_of(p.dstates, p, ch, 0) + (keys ? 256 * w : 0);
    const float *yp = value_of(p.y, p, ch, 0), *xp = value_of(p.dr, p, ch, 0);
    f4 F1[4], F2[4], F3[4], A[NJ], N[NJ];  // S0 dO^T, D U^T, S0 dR^T; tiles of dO U^T, dR U^T, transposed
#pragma unroll
    for (int it = 0; it < 4; ++it) F1[it] = F2[it] = F3[it] = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) A[j] = N[j] = 0;
    float sd = 0, rb[PT];  // <S0, D>; dR.Y of the staged tokens
    f4 sv[2], dv[2], yv[PT], xv[PT];
    Raw4<IT> go[PT];
    // staged piece x of this wavefront: half (w + x NW) / 4 of the slab, tokens 16 (w + x NW) % 4 + r16, columns 4 kg + i
    auto load_values = [&](int s) {
#pragma unroll
      for (int x = 0; x < PT; ++x) {
        const int vt = 2 * s + (w + x * NW) / 4, it = (w + x * NW) % 4, at = (vt < p.VT ? vt : 0) * (kC * 16) + 256 * it;
        yv[x] = *(const f4 *)(yp + at + at16);
        xv[x] = *(const f4 *)(xp + at + at16);
      }
    };
    auto load_inputs = [&](int s) {
#pragma unroll
      for (int x = 0; x < PT; ++x) {
        const int vt = 2 * s + (w + x * NW) / 4, it = (w + x * NW) % 4, have = t0 + 16 * it + r16 < p.L ? p.Dv - 16 * vt - 4 * kg : 0;
        go[x] = load4(dop + 16 * it * p.dout.s1 + 16 * vt + ao, (const IT *)p.dout.p, have, p.vdo);
      }
    };
    auto load_states = [&](int s, const float *m, f4 (&v)[2]) {
#pragma unroll
      for (int x = 0; x < 2; ++x) v[x] = *(const f4 *)(m + (2 * s + x < p.VT ? 2 * s + x : 0) * (int64_t)(p.Dkp * 16) + at16);
    };
    bf8 SA[NM], DA[NM];
    auto stage = [&](int s) {
      __bf16 *const Os = buf + (s & 1) * kStage, *const Us = Os + NK * SF, *const Rs = Us + NM * SF;
#pragma unroll
      for (int x = 0; x < PT; ++x) {
        const int sh = (w + x * NW) / 4, it = (w + x * NW) % 4, at = (it * 64 + lane) * 8 + 4 * sh;
        const bool in = 2 * s + sh < p.VT, live = t0 + 16 * it + r16 < p.L && p.Dv - 32 * s - 16 * sh - 4 * kg > 0;
        const float be = rows[4 * (16 * it + r16) + 1];
        const f4 yy = in ? yv[x] : (f4)0.0f, xx = in ? xv[x] : (f4)0.0f;
        bf4 o[NK], u[NM], r[NM];
        to_parts<IT, NK>(go[x], live, o);
        split_parts<NM>((f4)(be * yy), u);
        split_parts<NM>(xx, r);
#pragma unroll
        for (int i = 0; i < 4; ++i) rb[x] = fmaf(xx[i], yy[i], rb[x]);
#pragma unroll
        for (int n = 0; n < NK; ++n) *(bf4 *)(Os + n * SF + at) = o[n];
#pragma unroll
        for (int n = 0; n < NM; ++n) *(bf4 *)(Us + n * SF + at) = u[n];
#pragma unroll
        for (int n = 0; n < NM; ++n) *(bf4 *)(Rs + n * SF + at) = r[n];
      }
    };
    auto split_states = [&](int s) {
      f8 x = __builtin_shufflevector(sv[0], sv[1], 0, 1, 2, 3, 4, 5, 6, 7);
      f8 y = __builtin_shufflevector(dv[0], dv[1], 0, 1, 2, 3, 4, 5, 6, 7);
      if (!keys || 2 * s + 1 >= p.VT) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!keys || j >= 4) x[j] = y[j] = 0;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sd = fmaf(x[j], y[j], sd);
      split_parts<NM>(x, SA);
      split_parts<NM>(y, DA);
    };
    // The slab's products; after those of token tile `it` comes read(it), so that the reads' issue (16 cycles of
    // the compute unit's address unit each) falls into the time of the products.
    auto multiply = [&](int s, auto read) {
      const __bf16 *const Os = buf + (s & 1) * kStage, *const Us = Os + NK * SF, *const Rs = Us + NM * SF;
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        bf8 O[NK], U[NM], R[NM];
        load_frag<NK>(Os, SF, it, lane, O);
        load_frag<NM>(Us, SF, it, lane, U);
        load_frag<NM>(Rs, SF, it, lane, R);
        F1[it] = mma<NM>(SA, O, F1[it]);
        F3[it] = mma<NM>(SA, R, F3[it]);
        F2[it] = mma<NM>(DA, U, F2[it]);
        if (it == wi) {
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            if (wj + j <= wi) {
              bf8 Uj[NM];
              load_frag<NM>(Us, SF, wj + j, lane, Uj);
              A[j] = mma<NM>(Uj, O, A[j]);
              N[j] = mma<NM>(Uj, R, N[j]);
            }
        }
        read(it);
        __builtin_amdgcn_sched_barrier(0);  // one token tile's operands in registers at a time
      }
    };
    {
      const float *m = delta_rows(p, ch);
      float x[(kDeltaRows + NT - 1) / NT];
#pragma unroll
      for (int i = 0; i < (kDeltaRows + NT - 1) / NT; ++i) x[i] = m[tid + i * NT < kDeltaRows ? tid + i * NT : 0];
      load_values(0);
      load_inputs(0);
      load_states(0, Sp, sv);
      load_states(0, Dp, dv);
#pragma unroll
      for (int i = 0; i < (kDeltaRows + NT - 1) / NT; ++i)
        if (tid + i * NT < kDeltaRows) rows[tid + i * NT] = x[i];
    }
#pragma unroll
    for (int x = 0; x < PT; ++x) rb[x] = 0;
    lds_barrier();
    for (int s = 0; s + 1 < slabs; ++s) {
      stage(s);
      lds_barrier();  // the other buffer's readers are a barrier behind
      split_states(s);
      multiply(s, [&](int it) {
        if (it == 0) load_values(s + 1);
        else if (it == 1) load_inputs(s + 1);
        else if (it == 2) load_states(s + 1, Sp, sv);
        else load_states(s + 1, Dp, dv);
      });
    }
    stage(slabs - 1);
    lds_barrier();
    split_states(slabs - 1);
    multiply(slabs - 1, load_keys);

    sd = group_sum<64>(sd);
    if (lane == 0) sdot[w] = sd;
#pragma unroll
    for (int x = 0; x < PT; ++x) rb[x] = kg_sum(rb[x]);
    lds_barrier();  // the slabs are read
    // the two halves of the slabs are one wavefront's two pieces, or wavefronts 0..3 and 4..7
    if (kg == 0 && (PT == 2 || w >= 4)) rowb[16 * (w % 4) + r16] = PT == 2 ? rb[0] + rb[PT - 1] : rb[0];
    {  // J and H
      const int i = 16 * wi + r16;
      const float fqi = rows[5 * kC + i], fki = rows[4 * kC + i] * rows[4 * i + 1], gh = rows[6 * kC + i], gl = rows[7 * kC + i];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int at = 16 * (wj + j) + 4 * kg;
        f4 jv = 0, hv = 0;
        if (wj + j <= wi) {
          const f4 xk = *(const f4 *)(rows + 4 * kC + at), xh = *(const f4 *)(rows + 6 * kC + at), xl = *(const f4 *)(rows + 7 * kC + at);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float e = fexp((gh - xh[x]) + (gl - xl[x])) * xk[x];
            jv[x] = at + x < i ? fqi * e * A[j][x] : 0.0f;
            if (at + x == i) diag[i] = fqi * e * A[j][x];
            hv[x] = at + x < i ? -fki * e * N[j][x] : 0.0f;
          }
        }
        bf4 jp[NM], hp[NM];
        split_parts<NM>(jv, jp);
        split_parts<NM>(hv, hp);
#pragma unroll
        for (int n = 0; n < NM; ++n) *(bf4 *)(Jm + (n * kC + i) * JP + at) = jp[n];
#pragma unroll
        for (int n = 0; n < NM; ++n) *(bf4 *)(Hm + (n * kC + i) * JP + at) = hp[n];
      }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const f4 row = token_row(rows, 16 * it + r16), f2 = row[2] * F2[it], c = whole(Ke[it]) * f2;
      const float x = kg_sum((c[0] + c[1]) + (c[2] + c[3]));
      if (kg == 0) red[w][1][16 * it + r16] = x;
      Y[it] = rows[8 * kC + 16 * it + r16] * F1[it];
      Z[it] = f2;
      F2[it] = -(row[1] * row[0]) * F3[it];  // from here on F2 and F3 are what dG takes with a plus and with a minus
      F3[it] = 0;
    }
    lds_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const int at = (16 * it + r16) * JP + 32 * s + 4 * kg;                          // row it, columns of step s
        const int tr = (32 * s + 4 * kg + r16 / 4) * JP + 16 * it + 4 * (r16 % 4);      // rows of step s, column it
        if (s <= it / 2) {
          bf8 B[NM], C[NM];
#pragma unroll
          for (int n = 0; n < NM; ++n) {
            const __bf16 *m = Jm + n * kC * JP + at;
            B[n] = __builtin_shufflevector(*(const bf4 *)m, *(const bf4 *)(m + 16), 0, 1, 2, 3, 4, 5, 6, 7);
          }
#pragma unroll
          for (int n = 0; n < NM; ++n) {
            const __bf16 *m = Hm + n * kC * JP + at;
            C[n] = __builtin_shufflevector(*(const bf4 *)m, *(const bf4 *)(m + 16), 0, 1, 2, 3, 4, 5, 6, 7);
          }
          Y[it] = mma<NM>(Kt[s], B, Y[it]);
          F2[it] = mma<NM>(Kt[s], C, F2[it]);
        }
        if (s >= it / 2) {
          bf8 B[NM], C[NM];
#pragma unroll
          for (int n = 0; n < NM; ++n) {
            B[n] = read_tr(Jm + n * kC * JP + tr, Jm + (n * kC + 16) * JP + tr);
            C[n] = read_tr(Hm + n * kC * JP + tr, Hm + (n * kC + 16) * JP + tr);
          }
          F3[it] = mma<NM>(Qt[s], B, F3[it]);
          F3[it] = mma<NM>(Kt[s], C, F3[it]);
        }
      }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const f4 q = whole(Qe[it]), k = whole(Ke[it]), z = q * Y[it] + k * (F2[it] - F3[it]);
      const float x = kg_sum((z[0] + z[1]) + (z[2] + z[3])), own = diag[16 * it + r16];
      if (kg == 0) red[w][0][16 * it + r16] = x;
      Y[it] += own * k;
      Z[it] += (F2[it] + F3[it]) + own * q;
    }
    if (PT == 1 && w < 4 && kg == 0) rowb[16 * w + r16] += rb[0];
    if (SHARED) {
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        if (hg) {
          Y[it] += sum[it][tid];
          Z[it] += sum[4 + it][tid];
        }
        sum[it][tid] = Y[it];
        sum[4 + it][tid] = Z[it];
      }
    }
    if (p.qk_norm && hg + 1 == group) {
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const f4 q = whole(Qe[it]) * Y[it], k = whole(Ke[it]) * Z[it];
        const float sq = kg_sum((q[0] + q[1]) + (q[2] + q[3])), sk = kg_sum((k[0] + k[1]) + (k[2] + k[3]));
        if (kg == 0) {
          norm[w][0][16 * it + r16] = sq;
          norm[w][1][16 * it + r16] = sk;
        }
      }
    }
    lds_barrier();
    if (w == 0) {  // dbeta and dg of the head
      double s = 0, k = 0, ss = 0;  // s of token 63 - lane, k of token lane - 1
#pragma unroll
      for (int n = 0; n < NW; ++n) {
        s += red[n][0][63 - lane];
        k += lane ? red[n][1][lane - 1] : 0.0f;
        ss += sdot[n];
      }
      double rest = __shfl(wave_scan_f64(s), 63 - lane);  // sum over i >= t of dG_i
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(fabs(rest) < INFINITY)) != 0, 0) && fabs(ss) < INFINITY) {
        // A pair after t is in rows and columns of the sum and cancels, but not where it is infinite or NaN.  The sum of
        // all tokens less those before t is the same from finite terms: in that of all every pair cancels, and what is
        // left is the entering state's share, <S0, dS0 - e^{G_C} D>.
        const float *S = state_of(p.states, p, ch, 0), *D = state_of(p.dstates, p, ch, 0);
        const float *E = state_of(p.dstates, p, c ? ch - p.B * p.H : ch + (int64_t)p.NC * p.B * p.H, 0);
        double g = 0, all = 0;
#pragma unroll
        for (int n = 0; n < NW; ++n) g += lane ? red[n][0][lane - 1] : 0.0f;
#pragma unroll 1
        for (int64_t i = lane; i < (int64_t)p.VT * p.Dkp * 16; i += 64) all += S[i] * ((double)E[i] - (double)rows[3] * D[i]);
        all = __shfl(wave_scan_f64(all), 63);
        const double less = all - wave_scan_f64(g);
        if (!(fabs(rest) < INFINITY)) rest = less;
      }
      const double from = rest + wave_scan_f64(k) + (double)rows[3] * ss;
      const int64_t t = t0 + lane;
      if (t < p.L) {
        ((float *)p.dg.p)[b * p.dg.s0 + t * p.dg.s1 + h * p.dg.s2] = (float)from;
        store_either<IT>((void *)p.dbeta.p, p.beta32, b * p.dbeta.s0 + t * p.dbeta.s1 + h * p.dbeta.s2, rowb[lane]);
      }
    }
    if (hg + 1 < group) lds_barrier();  // J, H, rows and the sums are read
  }

  IT *dqb = (IT *)p.dq.p + b * p.dq.s0 + hk * p.dq.s2, *dkb = (IT *)p.dk.p + b * p.dk.s0 + hk * p.dk.s2;
  const int e = 16 * w + 4 * kg;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int tok = 16 * it + r16, have = t0 + tok < p.L ? p.Dk - e : 0;
    if (p.qk_norm) {  // through the norms
      float sq = 0, sk = 0;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        sq += norm[k][0][tok];
        sk += norm[k][1][tok];
      }
      const float fk = rows[4 * kC + tok], nq = rows[9 * kC + tok];
      Y[it] -= (nq * nq * sq) * whole(Qe[it]);
      Z[it] -= (fk * fk * sk) * whole(Ke[it]);
    }
    store4(dqb + (t0 + tok) * p.dq.s1 + e, Y[it], have, p.vdq);
    store4(dkb + (t0 + tok) * p.dk.s1 + e, Z[it], have, p.vdk);
  }
}

template <typename IT, int DK>
static hipError_t delta_bwd(const DeltaParams &p, hipStream_t s) {
  if (delta_pairs(p))
    delta_walk(p, 2, [&](const DeltaParams &part, dim3 grid) { hipLaunchKernelGGL((k_delta_bwd<IT, DK, 2>), grid, dim3(2 * kDT), 0, s, part); });
  else
    delta_walk(p, 1, [&](const DeltaParams &part, dim3 grid) { hipLaunchKernelGGL((k_delta_bwd<IT, DK, 1>), grid, dim3(2 * kDT), 0, s, part); });
  const dim3 grid((unsigned)(p.B * p.Hk) * (unsigned)p.NC);
  if (p.H > p.Hk) hipLaunchKernelGGL((k_delta_grad<IT, DK, true>), grid, dim3(4 * DK), 0, s, p);
  else hipLaunchKernelGGL((k_delta_grad<IT, DK, false>), grid, dim3(4 * DK), 0, s, p);
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
