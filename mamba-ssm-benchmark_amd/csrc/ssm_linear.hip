// Linear layer with its epilogue, in 16 and 8 bits:
//   z = (x W^T) [xs ws] + bias,   y = act(z) + residual          (8 bits: rows of x and W are q scale)
//   backward: dz = dy act'(z), dx = dz W, dW = dz^T x, dbias = sum over rows of dz.
// All products are of the form C[m, n] = sum over k of A(m, k) B(n, k) with each operand stored along k or along its
// rows; sums are float32 in the matrix cores, z meets bias, activation and residual in float32 and is rounded once.
#include "ssm_device.hpp"
#include "ssm_internal.hpp"
#include "ssm_tiles.hpp"
#include "ssm_wave.hpp"

namespace ssm {

typedef float lf4 __attribute__((ext_vector_type(4)));
typedef __bf16 lbf8 __attribute__((ext_vector_type(8)));
typedef _Float16 lh8 __attribute__((ext_vector_type(8)));

struct fp8_t { uint8_t bits; };

template <typename T> struct Mma;
template <> struct Mma<bf16_t> {
  typedef lbf8 Frag;   // 8 consecutive k of a row
  __device__ __forceinline__ static lf4 mul(Frag a, Frag b, lf4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<f16_t> {
  typedef lh8 Frag;
  __device__ __forceinline__ static lf4 mul(Frag a, Frag b, lf4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<fp8_t> {
  typedef long Frag;
  __device__ __forceinline__ static lf4 mul(Frag a, Frag b, lf4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ float lin_act(float z, int act) {
  if (act == kActSilu) return z * sigmoidf(z);
  if (act == kActGelu) return 0.5f * z * (1.0f + erff(z * 0.70710678f));
  return z;
}
__device__ __forceinline__ float lin_slope(float z, int act) {
  if (act == kActSilu) {
    const float s = sigmoidf(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
  }
  if (act == kActGelu) return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * 0.39894228f * __expf(-0.5f * z * z);
  return 1.0f;
}

// ------------------------------------------------------------------ any size, stride and alignment
// A workgroup of four wavefronts takes 64 x 64 of C, a wavefront 32 x 32 of it; both operands' 64 x 32 tiles pass
// through registers into LDS, [row][k] whatever their storage, zeros past their ends.
template <typename T> __device__ __forceinline__ T lin_zero() { return T{}; }
template <typename T, typename OT>
__global__ void __launch_bounds__(256) k_linear_any(const GemmParams p) {
  constexpr int BK = 32, LD = BK + 8;
  __shared__ __attribute__((aligned(16))) T As[64][LD], Bs[64][LD];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int64_t tn = (p.N + 63) / 64, m0 = blockIdx.x / tn * 64, n0 = blockIdx.x % tn * 64;
  const int wm = (wave / 2) * 32, wn = (wave % 2) * 32;
  lf4 acc[2][2] = {};
  for (int64_t k0 = 0; k0 < p.K; k0 += BK) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int id = threadIdx.x + 256 * e;
      {
        const int row = p.a_along ? id / BK : id % 64, k = p.a_along ? id % BK : id / 64;
        As[row][k] = m0 + row < p.M && k0 + k < p.K ? ((const T *)p.A)[(m0 + row) * (p.a_along ? p.sa : 1) + (k0 + k) * (p.a_along ? 1 : p.sa)] : lin_zero<T>();
      }
      {
        const int row = p.b_along ? id / BK : id % 64, k = p.b_along ? id % BK : id / 64;
        Bs[row][k] = n0 + row < p.N && k0 + k < p.K ? ((const T *)p.B)[(n0 + row) * (p.b_along ? p.sb : 1) + (k0 + k) * (p.b_along ? 1 : p.sb)] : lin_zero<T>();
      }
    }
    __syncthreads();
    typename Mma<T>::Frag a[2], b[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      a[i] = *(const typename Mma<T>::Frag *)&As[wm + 16 * i + lane % 16][8 * (lane / 16)];
      b[i] = *(const typename Mma<T>::Frag *)&Bs[wn + 16 * i + lane % 16][8 * (lane / 16)];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = Mma<T>::mul(b[j], a[i], acc[i][j]);   // rows of the result: n
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t m = m0 + wm + 16 * i + lane % 16, n = n0 + wn + 16 * j + 4 * (lane / 16) + q;
        if (m >= p.M || n >= p.N) continue;
        float z = acc[i][j][q];
        if (p.xs) z *= p.xs[m] * p.ws[n];
        if (p.bias) z += Conv<OT>::load((const OT *)p.bias + n);
        if (p.pre) Conv<OT>::store((OT *)p.pre + m * p.spre + n, z);
        z = lin_act(z, p.act);
        if (p.residual) z += Conv<OT>::load((const OT *)p.residual + m * p.sr + n);
        Conv<OT>::store((OT *)p.C + m * p.sc + n, z);
      }
}

// ------------------------------------------------------------------ dz and dbias
// dz = dy act'(z), 64 columns by a range of rows per workgroup, and that range's column sums of dz.
template <typename T>
__global__ void __launch_bounds__(256) k_linear_dz(const LinearDzParams p) {
  __shared__ float part[4][64];
  const int col = threadIdx.x % 64, sub = threadIdx.x / 64;
  const int64_t n = (int64_t)blockIdx.x * 64 + col, per = (p.M + gridDim.y - 1) / gridDim.y, m0 = blockIdx.y * per;
  const int64_t m1 = m0 + per < p.M ? m0 + per : p.M;
  float s = 0;
  if (n < p.N)
    for (int64_t m = m0 + sub; m < m1; m += 4) {
      float d = Conv<T>::load((const T *)p.dy + m * p.sdy + n);
      if (p.act) {
        d *= lin_slope(Conv<T>::load((const T *)p.pre + m * p.N + n), p.act);
        Conv<T>::store((T *)p.dz + m * p.N + n, d);
      }
      s += d;
    }
  part[sub][col] = s;
  __syncthreads();
  if (p.partial && sub == 0 && n < p.N)
    p.partial[blockIdx.y * p.N + n] = (part[0][col] + part[1][col]) + (part[2][col] + part[3][col]);
}
template <typename T>
__global__ void __launch_bounds__(256) k_linear_dbias(const LinearDzParams p) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n < p.N) Conv<T>::store((T *)p.dbias + n, (float)ordered_sum<8, float, double>(p.partial + n, p.N, p.slots));
}

template <typename T, typename OT>
static hipError_t gemm_t(const GemmParams &p, hipStream_t s) {
  hipLaunchKernelGGL((k_linear_any<T, OT>), dim3((unsigned)(((p.N + 63) / 64) * ((p.M + 63) / 64))), dim3(256), 0, s, p);
  return hipGetLastError();
}
hipError_t launch_gemm(const GemmParams &p, int dtype, hipStream_t s) {
  if (p.fp8) return dtype == 1 ? gemm_t<fp8_t, bf16_t>(p, s) : gemm_t<fp8_t, f16_t>(p, s);
  return dtype == 1 ? gemm_t<bf16_t, bf16_t>(p, s) : gemm_t<f16_t, f16_t>(p, s);
}
template <typename T>
static hipError_t dz_t(const LinearDzParams &p, hipStream_t s) {
  hipLaunchKernelGGL((k_linear_dz<T>), dim3((unsigned)((p.N + 63) / 64), (unsigned)p.slots), dim3(256), 0, s, p);
  if (p.dbias) hipLaunchKernelGGL((k_linear_dbias<T>), dim3((unsigned)((p.N + 255) / 256)), dim3(256), 0, s, p);
  return hipGetLastError();
}
hipError_t launch_linear_dz(const LinearDzParams &p, int dtype, hipStream_t s) {
  return dtype == 1 ? dz_t<bf16_t>(p, s) : dz_t<f16_t>(p, s);
}

}  // namespace ssm
