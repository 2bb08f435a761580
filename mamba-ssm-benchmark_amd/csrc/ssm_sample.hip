// The next token of every row of logits, from given random numbers.  With m the row's largest logit and
// w_i = exp((l_i - m) / T): of the order by falling logit (ties: the lower index first) the first top_k are kept, of
// those the shortest prefix that holds top_p of their mass, of those the ones with w_i >= min_p, and always the first;
// the token is the first kept index at which the running sum of the kept weights, by index, passes u times their sum.
//
// Weights are 64-bit integers, w_i 2^S rounded, S as large as the sum of V of them allows (52 at most): their sums
// are exact in any order, so LDS atomics give the same token every time, and what is rounded is 2^-S of the largest
// weight, below what a float64 sum of as many terms loses for V <= 2^17.
#include "ssm_device.hpp"
#include "ssm_internal.hpp"
#include "ssm_wave.hpp"

namespace ssm {

typedef unsigned long long u64;

// Keys in the order of the values, -0 and 0 alike.
__device__ __forceinline__ uint32_t sm_key(float l) {
  const uint32_t u = __float_as_uint(l + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sm_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// E consecutive logits from index i (those past the row's end are -inf), read whole whatever their alignment.
constexpr int kSampleE = 8;
template <typename IT>
__device__ __forceinline__ void sm_load(const IT *row, int64_t i, int64_t V, float (&v)[kSampleE]) {
  if (i + kSampleE <= V) {
    IT e[kSampleE];
    __builtin_memcpy(e, row + i, sizeof(e));
#pragma unroll
    for (int k = 0; k < kSampleE; ++k) v[k] = to_f32(e[k]);
  } else {
#pragma unroll
    for (int k = 0; k < kSampleE; ++k) v[k] = i + k < V ? to_f32(row[i + k]) : -INFINITY;
  }
}

struct SampleRow {
  double inv_t, scale;   // 1 / T; 2^S
  float top;             // the largest logit
  double temperature;
  __device__ __forceinline__ double z(float l) const { return l == top ? 0.0 : ((double)l - (double)top) / temperature; }
  __device__ __forceinline__ u64 weight(float l) const { return (u64)(exp(z(l)) * scale + 0.5); }
};

template <int NT, typename T, typename F>
__device__ __forceinline__ T sm_block(T v, T *lds, F f) {   // f over all threads' values, to all of them
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = f(v, (T)__shfl_xor(v, d));
  __syncthreads();
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
  __syncthreads();
  v = lds[0];
  for (int k = 1; k < NT / 64; ++k) v = f(v, lds[k]);
  return v;
}

// Walks the NB bins of `hist` from the highest down to the one at which the sum reaches `target` (> 0, at most the
// whole): its index, and the sum above it.
template <int NT>
__device__ __forceinline__ void sm_find(const u64 *hist, int nb, u64 target, u64 *lds, int *bin, u64 *above) {
  const int per = (nb + NT - 1) / NT, hi = nb - (int)threadIdx.x * per;   // bins [hi - per, hi) of this thread
  u64 mine = 0;
  for (int b = hi - 1; b >= hi - per; --b)
    if (b >= 0 && b < nb) mine += hist[b];
  u64 upto = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64 t = __shfl_up(upto, d);
    if (threadIdx.x % 64 >= d) upto += t;
  }
  __syncthreads();
  if (threadIdx.x % 64 == 63) lds[threadIdx.x / 64] = upto;
  __syncthreads();
  for (int k = 0; k < (int)threadIdx.x / 64; ++k) upto += lds[k];
  u64 sum = upto - mine;
  if (sum < target && upto >= target)
    for (int b = hi - 1; b >= hi - per; --b) {
      if (b < 0 || b >= nb) continue;
      if (sum + hist[b] >= target) {
        *bin = b;
        *above = sum;
        break;
      }
      sum += hist[b];
    }
  __syncthreads();
}

template <typename IT, int NT>
__global__ void __launch_bounds__(NT) k_sample(const SampleParams p) {
  constexpr int kBits = 11, kBins = 1 << kBits, kSteps = 2048;
  __shared__ u64 hist[kBins];          // also: masses of the steps
  __shared__ uint32_t ties[kSteps];
  __shared__ u64 red[NT / 64];
  __shared__ int bin;
  __shared__ u64 above;
  const int64_t row = p.first + blockIdx.x, V = p.V;
  const IT *logits = (const IT *)p.logits + row * p.sl;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  constexpr int64_t kStride = (int64_t)NT * kSampleE;
  auto each = [&](auto f) {   // f(index, logit) over the row
    for (int64_t i = (int64_t)threadIdx.x * kSampleE; i < V; i += kStride) {
      float v[kSampleE];
      sm_load<IT>(logits, i, V, v);
#pragma unroll
      for (int k = 0; k < kSampleE; ++k)
        if (i + k < V) f(i + k, v[k]);
    }
  };

  uint32_t top = 0;
  each([&](int64_t, float l) { top = max(top, l == l ? sm_key(l) : 0xffffffffu); });   // above infinity's: a NaN
  top = (uint32_t)sm_block<NT>((u64)top, red, [](u64 a, u64 b) { return a > b ? a : b; });
  SampleRow r;
  r.top = sm_value(top);
  if (top == 0xffffffffu || r.top == -INFINITY) {   // no distribution
    if (threadIdx.x == 0) {
      p.token[row] = -1;
      p.logprob[row] = NAN;
    }
    return;
  }
  r.temperature = p.temperatures ? (double)p.temperatures[row] : p.temperature;
  int64_t k = p.top_ks ? p.top_ks[row] : p.top_k;
  double top_p = p.top_ps ? (double)p.top_ps[row] : p.top_p;
  const double min_p = p.min_ps ? (double)p.min_ps[row] : p.min_p;
  if (!(r.temperature > 0)) {
    r.temperature = 1;
    k = 1;
  }
  r.scale = ldexp(1.0, p.shift);
  const double lowest = min_p > 0 ? log(min_p < 1 ? min_p : 1.0) : -INFINITY;

  uint32_t cut = 0;              // kept: keys above the cut, and the first `at_cut` of it
  u64 at_cut = ~0ull;
  auto select = [&](auto value, u64 target) {   // the key at which the values' sum, by falling key, reaches the target
    uint32_t prefix = 0;
    u64 sum = 0;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int b = threadIdx.x; b < kBins; b += NT) hist[b] = 0;
      __syncthreads();
      each([&](int64_t, float l) {
        const uint32_t key = sm_key(l);
        if (pass == 0 || key >> (shift + bits) == prefix >> (shift + bits))
          atomicAdd(&hist[(key >> shift) & ((1 << bits) - 1)], value(l, key));
      });
      __syncthreads();
      sm_find<NT>(hist, 1 << bits, target - sum, red, &bin, &above);
      prefix |= (uint32_t)bin << shift;
      sum += above;
      __syncthreads();
    }
    cut = prefix;
    return sum;   // above the cut
  };
  if (k == 1) {
    cut = top;
    at_cut = 1;
  } else if (k > 0 && k < V) {
    at_cut = (u64)k - select([&](float, uint32_t) { return (u64)1; }, (u64)k);
  }
  if (top_p < 1 && k != 1) {
    // the mass that is kept so far
    u64 mass = 0, at = 0;
    each([&](int64_t, float l) {
      const uint32_t key = sm_key(l);
      if (key > cut) mass += r.weight(l);
      at += key == cut;
    });
    mass = sm_block<NT>(mass, red, [](u64 a, u64 b) { return a + b; });
    at = sm_block<NT>(at, red, [](u64 a, u64 b) { return a + b; });
    const u64 wcut = cut ? r.weight(sm_value(cut)) : 0;
    mass += (at < at_cut ? at : at_cut) * wcut;
    const uint32_t kcut = cut;
    const u64 at_kcut = at_cut;
    const double want = top_p > 0 ? top_p * (double)mass : 0.0;
    u64 target = (u64)ceil(want);   // the first place at which the sum reaches it is the last one kept
    target = target < 1 ? 1 : target > mass ? mass : target;
    // of the ties at top_k's cut only the first count: the sum may be reached among them, before those that do not
    const u64 sum = select([&](float l, uint32_t key) { return key >= kcut ? r.weight(l) : (u64)0; }, target);
    const u64 w = r.weight(sm_value(cut));
    at_cut = (target - sum + w - 1) / w;
    if (cut == kcut && at_kcut < at_cut) at_cut = at_kcut;
  }

  // Masses and ties of every step of 64 x E consecutive logits; steps grow with V so that kSteps of them hold a row.
  const int64_t unit = 64 * kSampleE;
  const int64_t fold = (V + unit * kSteps - 1) / (unit * kSteps), step = unit * fold;   // logits a step
  const int steps = (int)((V + step - 1) / step);
  auto kept = [&](float l, uint32_t key) { return key >= cut && (key == top || r.z(l) >= lowest); };
  for (int s = wave; s < steps; s += NT / 64) {
    u64 m = 0, t = 0;
    for (int64_t f = 0; f < fold; ++f) {
      const int64_t i = s * step + f * unit + lane * kSampleE;
      float v[kSampleE];
      if (i < V) sm_load<IT>(logits, i, V, v);
#pragma unroll
      for (int q = 0; q < kSampleE; ++q)
        if (i + q < V) {
          const uint32_t key = sm_key(v[q]);
          if (kept(v[q], key)) {
            t += key == cut;
            if (key != cut) m += r.weight(v[q]);
          }
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      m += __shfl_xor(m, d);
      t += __shfl_xor(t, d);
    }
    if (lane == 0) {
      hist[s] = m;
      ties[s] = (uint32_t)t;
    }
  }
  __syncthreads();
  if (wave) return;
  // one wavefront: the total, the step of the token, then the token
  const float vcut = sm_value(cut);
  const u64 wcut = cut ? r.weight(vcut) : 0;
  auto ties_kept = [&](u64 before, u64 n) { return before >= at_cut ? (u64)0 : n < at_cut - before ? n : at_cut - before; };
  u64 total = 0, tie_run = 0;
  for (int s0 = 0; s0 < steps; s0 += 64) {   // ties before each step, in place of them; kept masses
    const int s = s0 + lane;
    const u64 n = s < steps ? ties[s] : 0;
    u64 upto = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const u64 t = __shfl_up(upto, d);
      if (lane >= d) upto += t;
    }
    const u64 before = tie_run + upto - n;
    u64 m = s < steps ? hist[s] + ties_kept(before, n) * wcut : 0;
    if (s < steps) {
      hist[s] = m;
      ties[s] = (uint32_t)before;
    }
    tie_run += __shfl(upto, 63);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) m += __shfl_xor(m, d);
    total += m;
  }
  wave_lds_sync();
  const double u = p.u_f64 ? ((const double *)p.u)[row] : (double)((const float *)p.u)[row];
  const double x = u * (double)total;
  u64 goal = x > 0 ? (u64)x : 0;   // the first sum above it
  if (goal >= total || u != u) goal = total - 1;
  u64 run = 0;
  int at = 0;
  for (int s0 = 0; s0 < steps; s0 += 64) {
    const int s = s0 + lane;
    const u64 m = s < steps ? hist[s] : 0;
    u64 upto = m;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const u64 t = __shfl_up(upto, d);
      if (lane >= d) upto += t;
    }
    const u64 past = __ballot(run + upto > goal);
    if (past) {
      const int l = __ffsll((long long)past) - 1;
      at = s0 + l;
      run += __shfl(upto - m, l);
      break;
    }
    run += __shfl(upto, 63);
  }
  u64 tie_before = ties[at];
  for (int64_t f = 0; f < fold; ++f) {
    const int64_t i = at * step + f * unit + lane * kSampleE;
    float v[kSampleE];
    u64 w[kSampleE], m = 0, t = 0;
    if (i < V) sm_load<IT>(logits, i, V, v);
#pragma unroll
    for (int q = 0; q < kSampleE; ++q) t += i + q < V && sm_key(v[q]) == cut && kept(v[q], cut);
    u64 upto = t;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const u64 a = __shfl_up(upto, d);
      if (lane >= d) upto += a;
    }
    u64 before = tie_before + upto - t;
    tie_before += __shfl(upto, 63);
#pragma unroll
    for (int q = 0; q < kSampleE; ++q) {
      w[q] = 0;
      if (i + q < V) {
        const uint32_t key = sm_key(v[q]);
        if (kept(v[q], key)) {
          w[q] = key != cut || before < at_cut ? r.weight(v[q]) : 0;
          before += key == cut;
        }
      }
      m += w[q];
    }
    upto = m;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const u64 a = __shfl_up(upto, d);
      if (lane >= d) upto += a;
    }
    const u64 past = __ballot(run + upto > goal);
    if (past) {
      if (lane == __ffsll((long long)past) - 1) {
        u64 sum = run + upto - m;
        int q = 0;
        for (; q < kSampleE - 1 && sum + w[q] <= goal; ++q) sum += w[q];
        p.token[row] = i + q;
        p.logprob[row] = (float)(r.z(v[q]) - log((double)total / r.scale));
      }
      return;
    }
    run += __shfl(upto, 63);
  }
}

template <typename IT>
static hipError_t sample_t(SampleParams p, hipStream_t s) {
  const int64_t most = kGridThreads / 1024;
  for (; p.first < p.R; p.first += most) {
    const dim3 grid((unsigned)(p.R - p.first < most ? p.R - p.first : most));
    if (p.V <= 4096) hipLaunchKernelGGL((k_sample<IT, 256>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((k_sample<IT, 1024>), grid, dim3(1024), 0, s, p);
  }
  return hipGetLastError();
}
hipError_t launch_sample(const SampleParams &p, int dtype, hipStream_t s) {
  return dtype == 0 ? sample_t<float>(p, s) : dtype == 1 ? sample_t<bf16_t>(p, s) : sample_t<f16_t>(p, s);
}

}  // namespace ssm
