// Gated delta rule, one token per stream, the state updated in place.
//   S' = e^g S,  u = beta (v - S'^T k),  S <- S' + k u^T,  o = scale S^T q = scale (S'^T q + (k.q) u)
// The state's bytes, read and written once, bound it (8 of every 8.1 bytes at 128 x 128), so a thread
// loads its part of the state before anything else and both products with the old state are taken
// from the same registers: one pass, one barrier.  A workgroup owns 64 columns of v of one head; lane
// l holds 4 columns, (l % 16), of the key rows 4 w + l / 16 + 16 j.
// 64 streams of 8 heads of 128 x 128: 13.9 us, 4.9 TB/s (a copy reaches 5.15); one stream of 8 heads of 64 x 64:
// 4.5 us, a launch's own time.
#include "ssm_delta.hpp"

namespace ssm {

template <int V>
__device__ __forceinline__ void load_cols(const float *p, int have, float (&x)[4]) {
  if (V == 4) {
    const float4 v = have > 0 ? *(const float4 *)p : make_float4(0, 0, 0, 0);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = i < have ? p[i] : 0.0f;
  }
}

template <typename IT, int JR, int V>
__global__ void __launch_bounds__(256) k_delta_step(const DeltaStepParams p) {
  __shared__ float red[4][2][64];
  const int tid = threadIdx.x, lane = tid % 64, w = tid / 64, c4 = 4 * (lane % 16), kr = 4 * w + lane / 16;
  const unsigned tiles = (p.Dv + 63) / 64, x = (unsigned)p.first + blockIdx.x;
  const int bh = x / tiles, v0 = 64 * (x % tiles);
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk), have = p.Dv - v0 - c4;
  float *hp = p.h + (int64_t)bh * p.Dk * p.Dv + v0 + c4;
  float S[JR][4], k[JR], q[JR];
#pragma unroll
  for (int j = 0; j < JR; ++j) load_cols<V>(hp + (int64_t)(kr + 16 * j) * p.Dv, kr + 16 * j < p.Dk ? have : 0, S[j]);
  const IT *kp = (const IT *)p.k.p + b * p.k.s0 + hk * p.k.s1, *qp = (const IT *)p.q.p + b * p.q.s0 + hk * p.q.s1;
  const float g = ((const float *)p.g.p)[b * p.g.s0 + h * p.g.s1];
  const float beta = load_either<IT>(p.beta.p, p.beta32, b * p.beta.s0 + h * p.beta.s1);
#pragma unroll
  for (int j = 0; j < JR; ++j) {
    const int r = kr + 16 * j;
    k[j] = r < p.Dk ? Conv<IT>::load(kp + r) : 0.0f;
    q[j] = r < p.Dk ? Conv<IT>::load(qp + r) : 0.0f;
  }
  // every wavefront forms k.k, q.q and k.q of the head for itself
  float kk = 0, qq = 0, kq = 0;
#pragma unroll
  for (int j = 0; j < JR / 4; ++j) {
    const int r = lane + 64 * j;
    const float a = r < p.Dk ? Conv<IT>::load(kp + r) : 0.0f, c = r < p.Dk ? Conv<IT>::load(qp + r) : 0.0f;
    kk = fmaf(a, a, kk);
    qq = fmaf(c, c, qq);
    kq = fmaf(a, c, kq);
  }
  kk = group_sum<64>(kk);
  qq = group_sum<64>(qq);
  kq = group_sum<64>(kq);
  const float rk = p.qk_norm ? 1.0f / sqrtf(kk + 1e-6f) : 1.0f, rq = p.qk_norm ? p.scale / sqrtf(qq + 1e-6f) : p.scale;
  float a[4] = {0, 0, 0, 0}, c[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < JR; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = fmaf(k[j], S[j][i], a[i]);
      c[i] = fmaf(q[j], S[j][i], c[i]);
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] += __shfl_xor(a[i], 16);
    c[i] += __shfl_xor(c[i], 16);
    a[i] += __shfl_xor(a[i], 32);
    c[i] += __shfl_xor(c[i], 32);
  }
  if (lane < 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      red[w][0][c4 + i] = a[i];
      red[w][1][c4 + i] = c[i];
    }
  }
  __syncthreads();
  const float eg = fast_exp2(g * LOG2E);
  const IT *vp = (const IT *)p.v.p + b * p.v.s0 + h * p.v.s1 + v0 + c4;
  IT *op = (IT *)p.o.p + b * p.o.s0 + h * p.o.s1 + v0 + c4;
  float u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float sk = (red[0][0][c4 + i] + red[1][0][c4 + i]) + (red[2][0][c4 + i] + red[3][0][c4 + i]);
    const float sq = (red[0][1][c4 + i] + red[1][1][c4 + i]) + (red[2][1][c4 + i] + red[3][1][c4 + i]);
    const float v = i < have ? Conv<IT>::load(vp + i) : 0.0f;
    u[i] = beta * fmaf(-eg * rk, sk, v);
    if (kr == 0 && i < have) Conv<IT>::store(op + i, rq * fmaf(rk * kq, u[i], eg * sq));
    u[i] *= rk;
  }
#pragma unroll
  for (int j = 0; j < JR; ++j) {
    if (kr + 16 * j >= p.Dk || have <= 0) continue;
    float *d = hp + (int64_t)(kr + 16 * j) * p.Dv;
#pragma unroll
    for (int i = 0; i < 4; ++i) S[j][i] = fmaf(k[j], u[i], eg * S[j][i]);
    if (V == 4) {
      *(float4 *)d = make_float4(S[j][0], S[j][1], S[j][2], S[j][3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < have) d[i] = S[j][i];
    }
  }
}

template <typename IT>
static hipError_t delta_step(const DeltaStepParams &p, hipStream_t s) {
  const int64_t all = (int64_t)p.B * p.H * ((p.Dv + 63) / 64), most = kGridThreads / 256;
  const bool v4 = p.Dv % 4 == 0 && (uintptr_t)p.h % 16 == 0;
  DeltaStepParams part = p;
  for (; part.first < all; part.first += most) {
    const dim3 grid((unsigned)(all - part.first < most ? all - part.first : most));
    if (p.Dk <= 64 && v4) hipLaunchKernelGGL((k_delta_step<IT, 4, 4>), grid, dim3(256), 0, s, part);
    else if (p.Dk <= 64) hipLaunchKernelGGL((k_delta_step<IT, 4, 1>), grid, dim3(256), 0, s, part);
    else if (v4) hipLaunchKernelGGL((k_delta_step<IT, 8, 4>), grid, dim3(256), 0, s, part);
    else hipLaunchKernelGGL((k_delta_step<IT, 8, 1>), grid, dim3(256), 0, s, part);
  }
  return hipGetLastError();
}
hipError_t launch_delta_step(const DeltaStepParams &p, int dtype, hipStream_t s) {
  return dtype == 0 ? delta_step<float>(p, s) : dtype == 1 ? delta_step<bf16_t>(p, s) : delta_step<f16_t>(p, s);
}

}  // namespace ssm
