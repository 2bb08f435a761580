// Grouped norm over the last dimension, with a gate or an activation: per row and group of n channels
//   xh = (x - mean) r,  r = 1 / sqrt(mean((x - mean)^2) + eps)     (center = 0: without the mean)
//   z = xh w + b,  y = z silu(gate), silu(z) or z.
// Backward, with dz = dy silu(gate), dy silu'(z) or dy and h = dz w:
//   dx = r (h - xh mean(h xh) - [center] mean(h)),  dw = sum over rows of dz xh,  db = sum of dz,
//   dgate = dy z silu'(gate).
// NP lanes own a group: lane l holds channels (k NP + l) V + i, so a group is read once, in 16-byte
// loads where its rows allow, and its sums are reductions over NP lanes.  Everything is float32 in
// between.  The backward recomputes mean and r from the x that it needs anyway, so the forward saves
// nothing; it is persistent, a lane group keeping one group of channels over its rows, with dw and db in
// float32 registers and one partial row per row slot that a second kernel adds in order, in float64: no float
// atomics, bitwise reproducible.  HBM bounds both directions from some 8 MB on:
// 16384 rows of 16 groups of 128, bf16, gate: forward 39 us (5.2 TB/s), backward 76 us (4.4 TB/s; with 2
// wavefronts a SIMD 104, with 8 the same 77 and twice the partial rows; reading a row ahead changed nothing).
#include "ssm_device.hpp"
#include "ssm_internal.hpp"
#include "ssm_tiles.hpp"

namespace ssm {

template <typename IT, int V>
__device__ __forceinline__ void g_load(const IT *src, float (&v)[V]) {
  struct alignas(V * sizeof(IT)) Pack { IT e[V]; };
  const Pack k = *(const Pack *)src;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = Conv<IT>::load(&k.e[i]);
}
template <typename IT, int V>
__device__ __forceinline__ void g_store(IT *dst, const float (&v)[V]) {
  struct alignas(V * sizeof(IT)) Pack { IT e[V]; };
  Pack k;
#pragma unroll
  for (int i = 0; i < V; ++i) Conv<IT>::store(&k.e[i], v[i]);
  *(Pack *)dst = k;
}
// The lane's channels of a group (`fill` past its end).
template <typename IT, int V, int NP, int K>
__device__ __forceinline__ void g_cols(const IT *src, int l, int n, float (&v)[K][V], float fill = 0.0f) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = (k * NP + l) * V;
    if (src && j < n) {
      g_load<IT, V>(src + j, v[k]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = fill;
    }
  }
}
template <typename IT, int V, int NP, int K>
__device__ __forceinline__ void g_put(IT *dst, int l, int n, const float (&v)[K][V]) {
#pragma unroll
  for (int k = 0; k < K; ++k)
    if ((k * NP + l) * V < n) g_store<IT, V>(dst + (k * NP + l) * V, v[k]);
}
// x -> (x - mean) r in place (0 past the end); returns r.
template <int V, int NP, int K>
__device__ __forceinline__ float g_normalize(float (&x)[K][V], int l, int n, bool center, float eps) {
  float m = 0;
  if (center) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) m += x[k][i];
    m = group_sum<NP>(m) / (float)n;
  }
  float ss = 0;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[k][i] = (k * NP + l) * V < n ? x[k][i] - m : 0.0f;
      ss = fmaf(x[k][i], x[k][i], ss);
    }
  const float r = 1.0f / sqrtf(group_sum<NP>(ss) / (float)n + eps);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) x[k][i] *= r;
  return r;
}

template <typename IT, int V, int NP, int K>
__global__ void __launch_bounds__(256) k_gnorm_fwd(const GnormParams p) {
  const int l = threadIdx.x % NP;
  const int64_t id = p.first + (int64_t)blockIdx.x * (256 / NP) + threadIdx.x / NP;
  const int64_t at = id < p.R * p.G ? id : p.R * p.G - 1;  // lane groups past the end write nothing
  const int64_t row = at / p.G;
  const int c0 = (int)(at % p.G) * p.n;
  float x[K][V], t[K][V], w[K][V], b[K][V];
  g_cols<IT, V, NP, K>((const IT *)p.x + row * p.sx + c0, l, p.n, x);
  if (p.act == 2) g_cols<IT, V, NP, K>((const IT *)p.gate + row * p.sg + c0, l, p.n, t);
  g_cols<float, V, NP, K>(p.w ? p.w + c0 : nullptr, l, p.n, w, 1.0f);
  g_cols<float, V, NP, K>(p.b ? p.b + c0 : nullptr, l, p.n, b);
  g_normalize<V, NP, K>(x, l, p.n, p.center, p.eps);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float z = fmaf(x[k][i], w[k][i], b[k][i]);
      const float a = p.act == 2 ? t[k][i] : z;
      x[k][i] = p.act == 0 ? z : p.act == 2 ? z * a * sigmoidf(a) : a * sigmoidf(a);
    }
  if (id < p.R * p.G) g_put<IT, V, NP, K>((IT *)p.y + row * p.sy + c0, l, p.n, x);
}

template <typename IT, int V, int NP, int K>
__global__ void __launch_bounds__(256) k_gnorm_bwd(const GnormParams p) {
  const int l = threadIdx.x % NP;
  const int64_t id = (int64_t)blockIdx.x * (256 / NP) + threadIdx.x / NP;
  const int64_t slot = id / p.G;
  if (slot >= p.nblk) return;  // whole lane groups
  const int c0 = (int)(id % p.G) * p.n;
  float w[K][V], b[K][V], aw[K][V], ab[K][V];
  g_cols<float, V, NP, K>(p.w ? p.w + c0 : nullptr, l, p.n, w, 1.0f);
  g_cols<float, V, NP, K>(p.b ? p.b + c0 : nullptr, l, p.n, b);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) aw[k][i] = ab[k][i] = 0;
  for (int64_t row = slot; row < p.R; row += p.nblk) {
    float x[K][V], t[K][V], d[K][V];
    g_cols<IT, V, NP, K>((const IT *)p.x + row * p.sx + c0, l, p.n, x);
    g_cols<IT, V, NP, K>((const IT *)p.dout + row * p.sdo + c0, l, p.n, d);
    if (p.act == 2) g_cols<IT, V, NP, K>((const IT *)p.gate + row * p.sg + c0, l, p.n, t);
    const float r = g_normalize<V, NP, K>(x, l, p.n, p.center, p.eps);
    float hx = 0, hs = 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = fmaf(x[k][i], w[k][i], b[k][i]), dy = d[k][i];
        float dz = dy;
        if (p.act) {
          const float a = p.act == 2 ? t[k][i] : z, s = sigmoidf(a), ds = s * fmaf(a, 1.0f - s, 1.0f);
          dz = dy * (p.act == 2 ? a * s : ds);
          t[k][i] = dy * z * ds;
        }
        aw[k][i] = fmaf(dz, x[k][i], aw[k][i]);
        ab[k][i] += dz;
        d[k][i] = dz * w[k][i];
        hx = fmaf(d[k][i], x[k][i], hx);
        hs += d[k][i];
      }
    hx = group_sum<NP>(hx) / (float)p.n;
    hs = p.center ? group_sum<NP>(hs) / (float)p.n : 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) d[k][i] = r * (fmaf(-x[k][i], hx, d[k][i]) - hs);
    g_put<IT, V, NP, K>((IT *)p.dx + row * p.sdx + c0, l, p.n, d);
    if (p.act == 2) g_put<IT, V, NP, K>((IT *)p.dgate + row * p.sdg + c0, l, p.n, t);
  }
  const int64_t C = (int64_t)p.G * p.n;
  if (p.dw) g_put<float, V, NP, K>(p.ws + slot * C + c0, l, p.n, aw);
  if (p.db) g_put<float, V, NP, K>(p.ws + (p.dw ? p.nblk * C : 0) + slot * C + c0, l, p.n, ab);
}

// dw_j, db_j = sum over the row slots in order: 16 columns by 64 ranges of slots per workgroup.
__global__ void __launch_bounds__(1024) k_gnorm_fin(const GnormParams p) {
  __shared__ double part[64][17];
  const int64_t C = (int64_t)p.G * p.n;
  const int col = threadIdx.x, q = threadIdx.y;
  const int64_t j = (int64_t)blockIdx.x * 16 + col, per = (p.nblk + 63) / 64, s0 = q * per;
  const bool second = blockIdx.y || !p.dw;
  const float *ws = p.ws + (second && p.dw ? p.nblk * C : 0);
  double s = 0;
  if (j < C && s0 < p.nblk) s = ordered_sum<8, float, double>(ws + s0 * C + j, C, s0 + per < p.nblk ? per : p.nblk - s0);
  part[q][col] = s;
  __syncthreads();
  if (q == 0 && j < C) {
    double t = 0;
    for (int k = 0; k < 64; ++k) t += part[k][col];
    (second ? p.db : p.dw)[j] = (float)t;
  }
}

template <typename IT, int V, int NP, int K>
static hipError_t gnorm_v(const GnormParams &p, bool bwd, hipStream_t s) {
  constexpr int64_t Q = 256 / NP;  // lane groups of a workgroup
  if (!bwd) {
    constexpr int64_t most = kGridThreads / NP;
    GnormParams part = p;
    for (; part.first < p.R * p.G; part.first += most) {
      const int64_t left = p.R * p.G - part.first, n = left < most ? left : most;
      hipLaunchKernelGGL((k_gnorm_fwd<IT, V, NP, K>), dim3((unsigned)((n + Q - 1) / Q)), dim3(256), 0, s, part);
    }
    return hipGetLastError();
  }
  hipLaunchKernelGGL((k_gnorm_bwd<IT, V, NP, K>), dim3((unsigned)(((int64_t)p.nblk * p.G + Q - 1) / Q)), dim3(256), 0, s, p);
  if (p.dw || p.db)  // (16, 64) threads: a grid row counts channels alone
    hipLaunchKernelGGL(k_gnorm_fin, dim3((unsigned)(((int64_t)p.G * p.n + 15) / 16), p.dw && p.db ? 2 : 1), dim3(16, 64), 0, s, p);
  return hipGetLastError();
}

template <typename IT>
static hipError_t gnorm_t(const GnormParams &p, bool bwd, hipStream_t s) {
  constexpr int V = 16 / sizeof(IT);
  if (p.vec) {  // the fewest lanes that hold a group in one load each
    if (p.n <= 8 * V) return gnorm_v<IT, V, 8, 1>(p, bwd, s);
    if (p.n <= 16 * V) return gnorm_v<IT, V, 16, 1>(p, bwd, s);
    if (p.n <= 32 * V) return gnorm_v<IT, V, 32, 1>(p, bwd, s);
    if (p.n <= 64 * V) return gnorm_v<IT, V, 64, 1>(p, bwd, s);
    return gnorm_v<IT, V, 64, kGnormMaxGroup / (64 * V)>(p, bwd, s);
  }
  if (p.n <= 16) return gnorm_v<IT, 1, 16, 1>(p, bwd, s);
  if (p.n <= 64) return gnorm_v<IT, 1, 64, 1>(p, bwd, s);
  if (p.n <= 256) return gnorm_v<IT, 1, 64, 4>(p, bwd, s);
  return gnorm_v<IT, 1, 64, 16>(p, bwd, s);
}
hipError_t launch_gnorm(const GnormParams &p, int dtype, bool bwd, hipStream_t s) {
  return dtype == 0 ? gnorm_t<float>(p, bwd, s) : dtype == 1 ? gnorm_t<bf16_t>(p, bwd, s) : gnorm_t<f16_t>(p, bwd, s);
}

}  // namespace ssm
