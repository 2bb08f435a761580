// Root-mean-square norm with the residual's addition, over rows of C channels:
//   s = x + residual, rounded to the residual's type;   y = s r w,  r = 1 / sqrt(mean(s^2) + eps)
// and, in place of y, its 8-bit form  q = e4m3(y / scale),  scale = max |y| / 448  (norm = 0: of x itself).
// Backward, with h = dy w (both gradients of s meet in one pass over the stored s):
//   ds' = ds + r (h - s r^2 mean(h s)),  dx = dresidual = ds',  dw = sum over rows of dy s r.
// The norm is of the stored sum, so that the backward, which has only that, is the adjoint of what was computed.
#include "ssm_device.hpp"
#include "ssm_internal.hpp"
#include "ssm_tiles.hpp"

namespace ssm {

template <typename IT, int V>
__device__ __forceinline__ void rn_load(const IT *src, float (&v)[V]) {
  struct alignas(V * sizeof(IT) < 16 ? V * sizeof(IT) : 16) Pack { IT e[V]; };
  const Pack k = *(const Pack *)src;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = Conv<IT>::load(&k.e[i]);
}
template <typename IT, int V>
__device__ __forceinline__ void rn_store(IT *dst, const float (&v)[V]) {
  struct alignas(V * sizeof(IT) < 16 ? V * sizeof(IT) : 16) Pack { IT e[V]; };
  Pack k;
#pragma unroll
  for (int i = 0; i < V; ++i) Conv<IT>::store(&k.e[i], v[i]);
  *(Pack *)dst = k;
}
template <typename IT>
__device__ __forceinline__ float rn_round(float v) {
  IT t;
  Conv<IT>::store(&t, v);
  return Conv<IT>::load(&t);
}
// V e4m3 values (OCP, to nearest even; |v| <= 448 but for its rounding).
template <int V>
__device__ __forceinline__ void rn_store8(uint8_t *dst, const float (&v)[V]) {
  if constexpr (V == 1) {
    *dst = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[0], 0, false);
  } else {
    struct alignas(V) Pack { int w[V / 4]; } k;
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      k.w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3],
                                               __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false), true);
    *(Pack *)dst = k;
  }
}

// Sums (max = 0) or maxima of N values over the W wavefronts of a row; every lane gets the same bits.
template <int W, int N, bool MAX>
__device__ __forceinline__ void rn_reduce(float (&v)[N], float (*lds)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if constexpr (MAX) {
#pragma unroll
      for (int d = 1; d < 64; d *= 2) v[n] = fmaxf(v[n], __shfl_xor(v[n], d));
    } else {
      v[n] = group_sum<64>(v[n]);
    }
  }
  if constexpr (W > 1) {
    __syncthreads();   // what an earlier reduction read
    if (threadIdx.x % 64 == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) lds[threadIdx.x / 64][n] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = lds[0][n];
#pragma unroll
      for (int k = 1; k < W; ++k) v[n] = MAX ? fmaxf(v[n], lds[k][n]) : v[n] + lds[k][n];
    }
  }
}

// W wavefronts a row, which they hold in registers between the sum and the scaling: each operand passes HBM once, and
// that is the bound.  16384 x 2048 in bf16 with a residual: 268 MB in 48-50 us, 5.4 TB/s; 64 rows of 4096 in 8 bits 4.6 us,
// the launch.  Workgroups of 4 rows (W = 1) or one.
template <typename IT, typename RT, int V, int W, int K>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W) k_rnorm_fwd(const RnormParams p) {
  constexpr int NT = 64 * W;
  __shared__ float lds[W][1];
  const int l = threadIdx.x % NT;
  const int64_t id = p.first + (int64_t)blockIdx.x * (W == 1 ? 4 : 1) + threadIdx.x / NT;
  if (id >= p.R) return;   // whole rows
  const IT *x = (const IT *)p.x + id * p.sx;
  const RT *r = p.res ? (const RT *)p.res + id * p.sr : nullptr;
  float t[K][V], w[K][V], ss[1] = {0};
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = (k * NT + l) * V;
    if (j < p.C) {
      rn_load<IT, V>(x + j, t[k]);
      if (p.w) rn_load<float, V>(p.w + j, w[k]);
      if (r) {
        float a[V];
        rn_load<RT, V>(r + j, a);
#pragma unroll
        for (int i = 0; i < V; ++i) t[k][i] = rn_round<RT>(t[k][i] + a[i]);
        rn_store<RT, V>((RT *)p.s + id * p.ss + j, t[k]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) t[k][i] = w[k][i] = 0;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) ss[0] = fmaf(t[k][i], t[k][i], ss[0]);
  }
  if (p.w) {   // without weights: the rows as they are
    rn_reduce<W, 1, false>(ss, lds);
    const float rs = 1.0f / sqrtf(ss[0] / (float)p.C + p.eps);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) t[k][i] = t[k][i] * rs * w[k][i];
  }
  if (!p.q) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = (k * NT + l) * V;
      if (j < p.C) rn_store<IT, V>((IT *)p.y + id * p.sy + j, t[k]);
    }
    return;
  }
  float top[1] = {0};
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) top[0] = fmaxf(top[0], fabsf(t[k][i]));   // a NaN is left out
  rn_reduce<W, 1, true>(top, lds);
  // at least the smallest normal number, so that the quotient below stays finite
  const float scale = top[0] > 0 ? fmaxf(top[0] / 448.0f, 1.17549435e-38f) : 1.0f, inv = 1.0f / scale;
  if (l == 0) p.scale[id] = scale;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = (k * NT + l) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) t[k][i] *= inv;
    if (j < p.C) rn_store8<V>(p.q + id * p.sq + j, t[k]);
  }
}

// Persistent: a row slot keeps its lanes' columns of dw in float32 registers over the rows slot, slot + nslot, ...
// The four slots of a workgroup of single wavefronts add theirs in LDS, so a workgroup leaves one partial row.
// 16384 x 2048 in bf16, ds and dw included: 268 MB in 52 us, 5.2 TB/s, HBM again; 8192 x 256 in float32 33 MB in 8 us.
template <typename IT, typename RT, int V, int W, int K>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W) k_rnorm_bwd(const RnormParams p) {
  constexpr int NT = 64 * W, Q = W == 1 ? 4 : 1;
  __shared__ float lds[W][2];
  __shared__ float part[W == 1 ? 3 : 1][W == 1 ? K * NT * V : 1];
  const int l = threadIdx.x % NT, sub = threadIdx.x / NT;
  float w[K][V], aw[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = (k * NT + l) * V;
    if (j < p.C) {
      rn_load<float, V>(p.w + j, w[k]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) w[k][i] = 0;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) aw[k][i] = 0;
  }
  for (int64_t row = (int64_t)blockIdx.x * Q + sub; row < p.R; row += (int64_t)p.nblk * Q) {
    float t[K][V], d[K][V], a[K][V], sum[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = (k * NT + l) * V;
      if (j < p.C) {
        rn_load<RT, V>((const RT *)p.s + row * p.ss + j, t[k]);
        rn_load<IT, V>((const IT *)p.dy + row * p.sdy + j, d[k]);
        if (p.ds) rn_load<RT, V>((const RT *)p.ds + row * p.sds + j, a[k]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) t[k][i] = d[k][i] = 0;
      }
      if (!p.ds || j >= p.C)
#pragma unroll
        for (int i = 0; i < V; ++i) a[k][i] = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        sum[0] = fmaf(t[k][i], t[k][i], sum[0]);
        sum[1] = fmaf(d[k][i] * w[k][i], t[k][i], sum[1]);
      }
    }
    rn_reduce<W, 2, false>(sum, lds);
    const float r = 1.0f / sqrtf(sum[0] / (float)p.C + p.eps), c = r * r * sum[1] / (float)p.C;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = (k * NT + l) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        aw[k][i] = fmaf(d[k][i], t[k][i] * r, aw[k][i]);
        a[k][i] = fmaf(r, fmaf(-t[k][i], c, d[k][i] * w[k][i]), a[k][i]);
      }
      if (j < p.C) {
        rn_store<IT, V>((IT *)p.dx + row * p.sdx + j, a[k]);
        if (p.dres) rn_store<RT, V>((RT *)p.dres + row * p.sdr + j, a[k]);
      }
    }
  }
  if (!p.dw) return;
  if constexpr (W == 1) {
    if (sub)
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) part[sub - 1][(k * V + i) * NT + l] = aw[k][i];
    __syncthreads();
    if (sub) return;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int n = 0; n < 3; ++n) aw[k][i] += part[n][(k * V + i) * NT + l];
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = (k * NT + l) * V;
    if (j < p.C) rn_store<float, V>(p.ws + (int64_t)blockIdx.x * p.C + j, aw[k]);
  }
}

// dw_j = the sum of the partial rows in order, in float64: 16 columns by 64 ranges of rows per workgroup.  3-5 us, latency.
__global__ void __launch_bounds__(1024) k_rnorm_fin(const RnormParams p) {
  __shared__ double part[64][17];
  const int col = threadIdx.x, q = threadIdx.y;
  const int64_t j = (int64_t)blockIdx.x * 16 + col, per = (p.nblk + 63) / 64, s0 = q * per;
  double s = 0;
  if (j < p.C && s0 < p.nblk) s = ordered_sum<8, float, double>(p.ws + s0 * p.C + j, p.C, s0 + per < p.nblk ? per : p.nblk - s0);
  part[q][col] = s;
  __syncthreads();
  if (q == 0 && j < p.C) {
    double t = 0;
    for (int k = 0; k < 64; ++k) t += part[k][col];
    p.dw[j] = (float)t;
  }
}

template <typename IT, typename RT, int V, int W, int K>
static hipError_t rnorm_v(const RnormParams &p, bool bwd, hipStream_t s) {
  constexpr int threads = W == 1 ? 256 : 64 * W, Q = W == 1 ? 4 : 1;
  if (!bwd) {
    constexpr int64_t most = kGridThreads / threads * Q;
    RnormParams part = p;
    for (; part.first < p.R; part.first += most) {
      const int64_t left = p.R - part.first, n = left < most ? left : most;
      hipLaunchKernelGGL((k_rnorm_fwd<IT, RT, V, W, K>), dim3((unsigned)((n + Q - 1) / Q)), dim3(threads), 0, s, part);
    }
    return hipGetLastError();
  }
  RnormParams b = p;
  b.nblk = (int)rnorm_blocks(p.R, W);
  hipLaunchKernelGGL((k_rnorm_bwd<IT, RT, V, W, K>), dim3((unsigned)b.nblk), dim3(threads), 0, s, b);
  if (b.dw) hipLaunchKernelGGL(k_rnorm_fin, dim3((unsigned)((p.C + 15) / 16)), dim3(16, 64), 0, s, b);
  return hipGetLastError();
}

template <typename IT, typename RT>
static hipError_t rnorm_t(const RnormParams &p, bool bwd, hipStream_t s) {
  constexpr int V = 16 / sizeof(IT);
  const int W = rnorm_waves(p.R, p.C, p.vec ? V : 1);
  if (!p.vec) {
    if (W == 1) return rnorm_v<IT, RT, 1, 1, 4>(p, bwd, s);
    if (W == 4) return rnorm_v<IT, RT, 1, 4, 4>(p, bwd, s);
    return rnorm_v<IT, RT, 1, 16, 16>(p, bwd, s);
  }
  const int per = (p.C + 64 * W * V - 1) / (64 * W * V);
  if (W == 1) return per == 1 ? rnorm_v<IT, RT, V, 1, 1>(p, bwd, s) : per == 2 ? rnorm_v<IT, RT, V, 1, 2>(p, bwd, s) : rnorm_v<IT, RT, V, 1, 4>(p, bwd, s);
  if (W == 4) return per == 1 ? rnorm_v<IT, RT, V, 4, 1>(p, bwd, s) : per == 2 ? rnorm_v<IT, RT, V, 4, 2>(p, bwd, s) : rnorm_v<IT, RT, V, 4, 4>(p, bwd, s);
  return per <= 2 ? rnorm_v<IT, RT, V, 16, 2>(p, bwd, s) : rnorm_v<IT, RT, V, 16, 4>(p, bwd, s);
}
hipError_t launch_rnorm(const RnormParams &p, int dtype, int rdtype, bool bwd, hipStream_t s) {
  if (dtype == 0) return rnorm_t<float, float>(p, bwd, s);
  if (dtype == 1) return rdtype == 0 ? rnorm_t<bf16_t, float>(p, bwd, s) : rnorm_t<bf16_t, bf16_t>(p, bwd, s);
  return rdtype == 0 ? rnorm_t<f16_t, float>(p, bwd, s) : rnorm_t<f16_t, f16_t>(p, bwd, s);
}

}  // namespace ssm
