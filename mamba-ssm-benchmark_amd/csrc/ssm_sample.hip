// The next token of every row of logits, from given random numbers.  With m the row's largest logit and
// w_i = exp((l_i - m) / T): of the order by falling logit (ties: the lower index first) the first top_k are kept, of
// those the shortest prefix that holds top_p of their mass, of those the ones with w_i >= min_p, and always the first;
// the token is the first kept index at which the running sum of the kept weights, by index, passes u times their sum.
//
// Weights are 64-bit integers, w_i 2^S rounded, S as large as the sum of V of them allows (51 at most): their sums
// are exact in any order, so atomics in LDS give the same token every time.  Each is off by 2^-(S+1) of the largest weight at
// most, so V of them by V 2^-(S+1): 4e-9 of it at V = 2^17 (S = 44), 2.4e-7 at 2^20, 6e-5 at 2^24 (S = 37).
//
// The row is not sorted.  What is kept is a prefix of the order, so it ends at one element, the cut (key, index).  A
// histogram of 2048 bins by falling logit, of counts for top_k and of weights for top_p, gives the bin that the cut is
// in; the elements of that bin (some hundred) are gathered and sorted in LDS.  A bin of more than kCandidates is cut
// by digits of (key, index) instead, 11 bits a pass.  What min_p leaves out is a range of keys, so it only moves the cut.
//
// A row of up to 32768 logits is one workgroup's from the maximum to the token.  Longer ones are walked by a workgroup a
// chunk, in five launches: maxima, histograms, cut (a workgroup a row), kept masses, token.  One workgroup against five
// launches, top_p, us: 64 x 8192 34 against 52, 64 x 16384 40 against 56, 64 x 32768 51 against 64 (1 x 32768, all kept, 23
// against 21).
//
// What bounds it is latency: a chain of passes over a row with barriers between them, by few workgroups.  64 rows of 131072
// in bf16 are 16.8 MB (3.3 us at 5 TB/s); top_k 40 and top_p 0.9 take 104 us, most of it in the cut's kernel, whose
// workgroup gathers twice from its whole row.  A row of 256 takes 4.8 us with all kept, the launch itself, and 11 with top_p.
#include <type_traits>

#include "ssm_device.hpp"
#include "ssm_internal.hpp"
#include "ssm_wave.hpp"

namespace ssm {

typedef unsigned long long u64;
constexpr int kE = 8;                  // consecutive logits a lane reads at once
constexpr int kTile = 64 * kE;         // and a wavefront
constexpr int kCandidates = 2048;   // and places of the sort

// Keys in the order of the values, -0 and 0 alike; a NaN's is above infinity's.
__device__ __forceinline__ uint32_t sm_key(float l) {
  const uint32_t u = __float_as_uint(l + 0.0f);
  return l == l ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0xffffffffu;
}
__device__ __forceinline__ float sm_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// kE consecutive logits from index i, read whole whatever their alignment; those past the row's end are not there.
template <typename IT>
__device__ __forceinline__ void sm_load(const IT *row, int64_t i, int64_t V, float (&v)[kE]) {
  if (i + kE <= V) {
    IT e[kE];
    __builtin_memcpy(e, row + i, sizeof(e));
#pragma unroll
    for (int k = 0; k < kE; ++k) v[k] = to_f32(e[k]);
  } else {
#pragma unroll
    for (int k = 0; k < kE; ++k) v[k] = i + k < V ? to_f32(row[i + k]) : -INFINITY;
  }
}

// A row's settings and its weights.  exp2(t / 256) = 2^(i / 256) e^x with i the nearest whole number, |x| <= ln 2 / 512: the
// first factor from a table in LDS and the exponent, the second as its series to x^4 (the rest is below 4e-17).
constexpr int kTable = 256;
struct SampleRow {
  double top, step;   // the largest logit; 256 / (T ln 2)
  double temperature, lowest;
  float topf, octave64;   // 64 / (T ln 2)
  int shift;
  uint32_t top_key;
  const double *table;
  __device__ __forceinline__ double z(float l) const { return l == topf ? 0.0 : ((double)l - top) / temperature; }
  __device__ __forceinline__ u64 weight(float l) const {
    constexpr double whole = 6755399441055744.0, one = 4503599627370496.0, h = 0.0027076061740622863;   // 1.5 2^52, 2^52, ln 2 / 256
    const double t = l == topf ? 0.0 : fmax(((double)l - top) * step, -2e5);
    const double n = t + whole, x = t - (n - whole);
    const int i = (int)(uint32_t)__builtin_bit_cast(u64, n);
    double e = fma(x, h * h * h * h / 24, h * h * h / 6);
    e = fma(x, e, h * h / 2);
    e = fma(x, e, h);
    e = fma(x, e, 1.0);
    // w 2^shift + 2^52, whose low bits are the number: w < 2^52
    const u64 f = __builtin_bit_cast(u64, table[i & (kTable - 1)]) + ((u64)(uint32_t)(i >> 8) << 52);
    return __builtin_bit_cast(u64, fma(__builtin_bit_cast(double, f), e, one)) - __builtin_bit_cast(u64, one);
  }
  // 1/64 octaves of weight down from the top: 1792 bins of one, then 32 a doubling; falling logits, rising bins.
  __device__ __forceinline__ int bin(float l) const {
    if (l == topf) return 0;
    const float d = (topf - l) * octave64;
    return d < 1792.0f ? (int)d : d < 458752.0f ? 1792 + (int)((__float_as_uint(d) - __float_as_uint(1792.0f)) >> 18) : 2047;
  }
};
constexpr int kBins = 2048;
struct SampleSettings {
  int64_t k;          // 0: all
  double top_p;       // >= 1: all
};
__device__ __forceinline__ SampleSettings sm_settings(const SampleParams &p, int64_t row, SampleRow &r) {
  SampleSettings s;
  r.temperature = p.temperatures ? (double)p.temperatures[row] : p.temperature;
  s.k = p.top_ks ? p.top_ks[row] : p.top_k;
  s.top_p = p.top_ps ? (double)p.top_ps[row] : p.top_p;
  const double min_p = p.min_ps ? (double)p.min_ps[row] : p.min_p;
  if (!(r.temperature > 0)) {
    r.temperature = 1;
    s.k = 1;
  }
  if (min_p > 1) s.k = 1;   // no weight reaches it: the first alone, of ties too
  if (s.k < 0 || s.k >= p.V) s.k = 0;
  if (!(s.top_p < 1)) s.top_p = 1;
  r.lowest = min_p > 0 ? log(min_p < 1 ? min_p : 1.0) : -INFINITY;
  r.step = 369.3299304757465 / r.temperature;   // 256 / ln 2
  r.octave64 = (float)(r.step / 4);
  r.shift = p.shift;
  return s;
}
// (key, first index) of the row's largest logit, as a number that is larger the earlier in the order
__device__ __forceinline__ u64 sm_place(uint32_t key, uint32_t i) { return (u64)key << 32 | (uint32_t)~i; }
__device__ __forceinline__ bool sm_top(SampleRow &r, u64 best) {   // false: no distribution
  r.top_key = (uint32_t)(best >> 32);
  r.topf = sm_value(r.top_key);
  r.top = r.topf;
  return r.top_key != 0xffffffffu && r.topf != -INFINITY;
}

template <int NT, typename T, typename F>
__device__ __forceinline__ T sm_block(T v, T *lds, F f) {   // f over all threads' values, to all of them
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = f(v, (T)__shfl_xor(v, d));
  if constexpr (NT > 64) {
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    v = lds[0];
    for (int k = 1; k < NT / 64; ++k) v = f(v, lds[k]);
  }
  return v;
}
__device__ __forceinline__ u64 sm_scan(u64 v) {   // inclusive, over the wavefront
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64 t = __shfl_up(v, d);
    if ((int)(threadIdx.x % 64) >= d) v += t;
  }
  return v;
}

template <int NT> struct SampleLds {
  u64 mass[kBins];
  uint32_t count[kBins];
  u64 place[kCandidates];
  double table[kTable];
  u64 red[NT / 64];
  u64 above, cut;
  int bin, n;
};
template <int NT>
__device__ __forceinline__ void sm_table(double *table, SampleRow &r) {   // before a barrier
  for (int i = threadIdx.x; i < kTable; i += NT) table[i] = ldexp(exp2((double)i / kTable), r.shift);
  r.table = table;
}

// The first of kBins bins of the counts, or of the masses, at which the running sum reaches `target` (1 .. the whole),
// into m.bin, and the sum before it, into m.above.
template <int NT>
__device__ __forceinline__ void sm_find(SampleLds<NT> &m, int by_mass, u64 target) {
  constexpr int per = kBins / NT;
  u64 v[per], mine = 0;
#pragma unroll
  for (int k = 0; k < per; ++k) mine += v[k] = by_mass ? m.mass[threadIdx.x * per + k] : m.count[threadIdx.x * per + k];
  u64 upto = sm_scan(mine);
  __syncthreads();
  if (threadIdx.x % 64 == 63) m.red[threadIdx.x / 64] = upto;
  __syncthreads();
  for (int k = 0; k < (int)threadIdx.x / 64; ++k) upto += m.red[k];
  u64 sum = upto - mine;
  if (sum < target && upto >= target) {
#pragma unroll
    for (int k = 0; k < per; ++k) {
      if (sum < target && sum + v[k] >= target) {
        m.bin = threadIdx.x * per + k;
        m.above = sum;
      }
      sum += v[k];
    }
  }
  __syncthreads();
}

// The smallest keys from -inf's to the top's at which in(l, 0) and in(l, 1) hold, which do from there on.  A wavefront
// tries 64 keys at once, for both.
template <typename F>
__device__ __forceinline__ void sm_borders(const SampleRow &r, F in, uint32_t (&from)[2]) {
  const uint32_t lane = threadIdx.x % 64;
  uint32_t n[2];   // it is one of from .. from + n
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    from[h] = 0x007fffffu;
    n[h] = r.top_key - from[h];
  }
  while (n[0] | n[1])
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t step = n[h] / 64 + 1, mine = lane * step;
      const u64 yes = __ballot(mine <= n[h] && in(sm_value(from[h] + mine), h));
      const uint32_t l = yes ? __ffsll((long long)yes) - 1 : n[h] / step + 1;   // the first lane that it holds for, or past the last one tried
      const uint32_t lower = l ? (l - 1) * step + 1 : 0, upper = yes ? l * step : n[h];
      from[h] += lower;
      n[h] = upper - lower;
    }
}
// The logits of bin `bin`, from hi down to lo: bins rise with falling keys, so each is a range of them.
__device__ __forceinline__ void sm_range(const SampleRow &r, int bin, float &lo, float &hi) {
  uint32_t from[2];
  sm_borders(r, [&](float l, int h) { return r.bin(l) <= bin - (h && bin); }, from);
  lo = sm_value(from[0]);
  hi = bin ? sm_value(from[1] - 1) : r.topf;
}
// Gathers the elements of a range of logits; m.n counts them, the first kCandidates are kept.
template <int NT, typename Each>
__device__ __forceinline__ int sm_gather(SampleLds<NT> &m, Each each, float lo, float hi) {
  if (threadIdx.x == 0) m.n = 0;
  __syncthreads();
  each([&](uint32_t i, float l) {
    if (!(l >= lo && l <= hi)) return;
    const int at = atomicAdd(&m.n, 1);
    if (at < kCandidates) m.place[at] = sm_place(sm_key(l), i);
  });
  __syncthreads();
  return m.n;
}
// The first n of NT E elements in falling order, by a bitonic network: E consecutive ones a thread in registers, pairs of
// one thread and (by lane exchanges) of one wavefront without LDS, so 1024 elements pass LDS in 3 of 55 steps.
template <int NT, int E>
__device__ __forceinline__ void sm_sort(u64 *place, int n) {
  int P = 64 * E;
  while (P < n) P *= 2;
  const int i0 = threadIdx.x * E;
  const bool active = i0 < P;   // whole wavefronts
  u64 v[E];
#pragma unroll
  for (int q = 0; q < E; ++q) v[q] = i0 + q < n ? place[i0 + q] : 0;   // 0: below any element
  auto keep = [](u64 &x, u64 o, bool larger) { x = (x > o) == larger ? x : o; };
  auto own = [&](int k) {   // the steps between a thread's elements, up to k / 2 apart
#pragma unroll
    for (int d = E / 2; d; d /= 2) {
      if (d >= k) continue;
#pragma unroll
      for (int q = 0; q < E; ++q) {
        if (q & d) continue;
        const bool falling = !((i0 + q) & k);
        const u64 x = v[q], y = v[q | d];
        v[q] = (x > y) == falling ? x : y;
        v[q | d] = (x > y) == falling ? y : x;
      }
    }
  };
#pragma unroll
  for (int k = 2; k < E; k *= 2) own(k);
#pragma unroll 1
  for (int k = E; k <= P; k *= 2) {
#pragma unroll 1
    for (int d = k / 2; d >= E; d /= 2) {
      const bool larger = !(i0 & k) == !(i0 & d);
      if (d < 64 * E) {
        if (active)
#pragma unroll
          for (int q = 0; q < E; ++q) keep(v[q], __shfl_xor(v[q], d / E), larger);
      } else {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < E; ++q) place[i0 + q] = v[q];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < E; ++q) keep(v[q], place[(i0 + q) ^ d], larger);
      }
    }
    own(k);
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < E; ++q) place[i0 + q] = v[q];
  __syncthreads();
}
// Of sorted elements the one at which the running sum of value(l, place) reaches `target` (1 .. the whole).
template <int NT, typename M, typename Value>
__device__ __forceinline__ u64 sm_reach(M &m, int n, u64 target, Value value) {
  u64 sum = 0;   // of the elements before this turn's
  for (int c0 = 0; c0 < n; c0 += NT) {
    const int c = c0 + threadIdx.x;
    const u64 at = c < n ? m.place[c] : 0, own = c < n ? value(sm_value((uint32_t)(at >> 32)), at) : 0;
    u64 upto = sm_scan(own);
    if (threadIdx.x % 64 == 63) m.red[threadIdx.x / 64] = upto;
    __syncthreads();
    u64 all = 0;
    for (int k = 0; k < NT / 64; ++k) {
      if (k == (int)threadIdx.x / 64) upto += all;
      all += m.red[k];
    }
    upto += sum;
    if (upto - own < target && upto >= target) m.cut = at;
    sum += all;
    __syncthreads();
  }
  return m.cut;
}
// Of the elements of a range of logits the one at which the running sum of value(l, place), by falling place, reaches
// `target` (1 .. the whole), as its place.  n: how many there are, of which up to kCandidates have been gathered; ones:
// every value is one.
template <int NT, typename Each, typename Value>
__device__ __forceinline__ u64 sm_cut(SampleLds<NT> &m, Each each, float lo, float hi, int n, u64 target, bool ones, Value value) {
  if (n <= kCandidates) {
    if (n <= 256) {   // each element's rank by comparing it with all: 0.7 us for 100 where the network takes 4.6
      u64 mine = 0;
      int rank = 0;
      if ((int)threadIdx.x < n) {
        mine = m.place[threadIdx.x];
#pragma unroll 8
        for (int o = 0; o < n; ++o) rank += m.place[o] > mine;
      }
      __syncthreads();
      if ((int)threadIdx.x < n) m.place[rank] = mine;
      __syncthreads();
    } else {
      sm_sort<NT, kCandidates / NT>(m.place, n);
    }
    if (ones) return m.place[target - 1];
    return sm_reach<NT>(m, n, target, value);
  }
  u64 prefix = 0, sum = 0;
  for (int shift = 53; shift > -11; shift -= 11) {   // digits of 11 bits, the last of 9
    const int s = shift < 0 ? 0 : shift, bits = shift < 0 ? 11 + shift : 11;
    for (int b = threadIdx.x; b < kBins; b += NT) m.mass[b] = 0;
    __syncthreads();
    each([&](uint32_t i, float l) {
      if (!(l >= lo && l <= hi)) return;
      const u64 at = sm_place(sm_key(l), i);
      if (shift < 53 && at >> (s + bits) != prefix >> (s + bits)) return;
      atomicAdd(&m.mass[(1 << bits) - 1 - (int)(at >> s & ((1 << bits) - 1))], value(l, at));   // falling
    });
    __syncthreads();
    sm_find<NT>(m, 1, target - sum);
    prefix |= (u64)((1 << bits) - 1 - m.bin) << s;
    sum += m.above;
    __syncthreads();
  }
  return prefix;
}

// The sum that the last place kept by top_p is the first to reach.
__device__ __forceinline__ u64 sm_target(const SampleSettings &s, u64 mass) {
  const u64 target = s.top_p > 0 ? (u64)ceil(s.top_p * (double)mass) : 1;
  return target < 1 ? 1 : target > mass ? mass : target;
}
// The cut of a row whose histograms are in m (of counts if k, of weights if top_p): the place of the last kept element,
// min_p aside.  One after the other top_k's cut by counts and top_p's by what that leaves of the weights, in one loop: the
// code of a walk is long, and a kernel of one workgroup a row waits for every line of it.
template <int NT, typename Each>
__device__ __forceinline__ u64 sm_select(SampleLds<NT> &m, const SampleRow &r, const SampleSettings &s, Each each) {
  auto add = [](u64 a, u64 b) { return a + b; };
  u64 cut = 0, target = (u64)s.k;
  int have = -1, n = 0;   // the bin whose elements are gathered
  float lo = 0, hi = 0;
#pragma unroll 1
  for (int by_mass = s.k > 1 ? 0 : 1; by_mass < (s.top_p < 1 ? 2 : 1); ++by_mass) {
    if (by_mass) {
      u64 mass = 0;
#pragma unroll 1
      for (int b = threadIdx.x; b < kBins; b += NT) mass += m.mass[b];
      target = sm_target(s, sm_block<NT>(mass, m.red, add));
      __syncthreads();
    }
    sm_find<NT>(m, by_mass, target);
    const int bin = m.bin;
    const u64 rest = target - m.above, kcut = cut;
    __syncthreads();
    if (bin != have) {
      sm_range(r, bin, lo, hi);
      n = sm_gather<NT>(m, each, lo, hi);
      have = bin;
    }
    u64 save[kBins / NT];   // cutting by digits takes the histogram's place
#pragma unroll
    for (int b = 0; b < kBins / NT; ++b) save[b] = m.mass[b * NT + threadIdx.x];
    __syncthreads();
    cut = sm_cut<NT>(m, each, lo, hi, n, rest, !by_mass, [&](float l, u64 at) { return !by_mass ? 1 : at >= kcut ? r.weight(l) : (u64)0; });
    __syncthreads();
    if (by_mass || !(s.top_p < 1)) continue;
    u64 kept = 0;   // what top_k has left of the weights
    if (n <= kCandidates) {
#pragma unroll 1
      for (int c = threadIdx.x; c < n; c += NT) kept += m.place[c] >= cut ? r.weight(sm_value((uint32_t)(m.place[c] >> 32))) : 0;
    } else {
      each([&](uint32_t i, float l) {
        if (l >= lo && l <= hi && sm_place(sm_key(l), i) >= cut) kept += r.weight(l);
      });
    }
    kept = sm_block<NT>(kept, m.red, add);
#pragma unroll
    for (int b = 0; b < kBins / NT; ++b) {
      const int at = b * NT + threadIdx.x;
      m.mass[at] = at < have ? save[b] : at == have ? kept : 0;
    }
    __syncthreads();
  }
  return cut;
}

// The cut with min_p: the smallest key that it keeps, at any index.
__device__ __forceinline__ u64 sm_min_p(const SampleRow &r, u64 cut, u64 first) {
  if (r.lowest == -INFINITY) return cut;
  uint32_t from[2];
  sm_borders(r, [&](float l, int) { return r.z(l) >= r.lowest; }, from);
  const u64 lowest = (u64)from[0] << 32;
  cut = cut > lowest ? cut : lowest;
  return cut < first ? cut : first;   // the first stays
}
// The weight of element i in the draw.
struct SampleCut {
  float l;
  uint32_t i;
  __device__ __forceinline__ explicit SampleCut(u64 cut) : l(sm_value((uint32_t)(cut >> 32))), i((uint32_t)~cut) {
    if (cut == 0) l = -INFINITY;   // all: -inf has no weight
  }
  __device__ __forceinline__ u64 weight(const SampleRow &r, uint32_t at, float v) const {
    return v > l || (v == l && at <= i) ? r.weight(v) : 0;
  }
};

// The running sum that the token's is the first to pass.
__device__ __forceinline__ u64 sm_goal(const SampleParams &p, int64_t row, u64 total) {
  const double u = p.u_f64 ? ((const double *)p.u)[row] : (double)((const float *)p.u)[row], x = u * (double)total;
  const u64 goal = x > 0 ? (u64)x : 0;
  return goal >= total || u != u ? total - 1 : goal;
}
// One wavefront: the tile of `tiles` in which the running sum of their masses passes u times the whole, and the sum
// before it.
__device__ __forceinline__ void sm_tile(const SampleParams &p, int64_t row, const u64 *masses, int64_t tiles, int64_t &tile, u64 &run,
                                        u64 &goal, u64 &total) {
  const int lane = threadIdx.x % 64;
  total = 0;
  for (int64_t t = lane; t < tiles; t += 64) total += masses[t];
#pragma unroll
  for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
  goal = sm_goal(p, row, total);
  run = 0;
  for (int64_t t0 = 0; t0 < tiles; t0 += 64) {
    const u64 m = t0 + lane < tiles ? masses[t0 + lane] : 0, upto = sm_scan(m), past = __ballot(run + upto > goal);
    if (past) {
      const int l = __ffsll((long long)past) - 1;
      tile = t0 + l;
      run += __shfl(upto - m, l);
      return;
    }
    run += __shfl(upto, 63);
  }
  tile = tiles - 1;   // not reached: the sums end at the total
}
__device__ __forceinline__ float sm_logprob(const SampleRow &r, float l, u64 total) {
  return (float)(r.z(l) - log(ldexp((double)total, -r.shift)));   // 0 where the token is all that is kept
}
// One wavefront: the token, in the tile whose logits its lanes hold.
__device__ __forceinline__ void sm_pick(const SampleParams &p, const SampleRow &r, int64_t row, const SampleCut &cut, int64_t i, const float (&v)[kE],
                                        u64 run, u64 goal, u64 total) {
  u64 w[kE], m = 0;
#pragma unroll
  for (int q = 0; q < kE; ++q) m += w[q] = i + q < p.V ? cut.weight(r, (uint32_t)(i + q), v[q]) : 0;
  const u64 upto = sm_scan(m), past = __ballot(run + upto > goal);
  if ((int)(threadIdx.x % 64) != __ffsll((long long)past) - 1) return;
  u64 sum = run + upto - m;
  int at = 0;
  float l = v[0];
#pragma unroll
  for (int q = 0; q < kE - 1; ++q) {   // the first q whose sum passes
    sum += w[q];
    if (sum <= goal) {
      at = q + 1;
      l = v[q + 1];
    }
  }
  p.token[row] = i + at;
  p.logprob[row] = sm_logprob(r, l, total);
}

// ------------------------------------------------------------------ short rows
// Up to kShort logits: the whole row is sorted, and nothing is unrolled (see sm_select).
// 64 rows of 1000, top_p 19 us against 30 in k_sample_row, which holds more than a short row needs; all kept 5.7 against 17.
// A row of 256 with top_k 10 us, the chain of the sort's exchanges.
constexpr int kShort = 1024;
template <typename IT>
__global__ void __launch_bounds__(256) k_sample_short(const SampleParams p) {
  constexpr int NT = 256, per = kShort / NT;
  __shared__ struct {
    u64 place[kShort], weight[kShort], red[NT / 64], cut;
    double table[kTable];
  } m;
  const int64_t row = p.first + blockIdx.x;
  const IT *logits = (const IT *)p.logits + row * p.sl;
  const int V = (int)p.V, t = threadIdx.x;
  u64 first = 0;
#pragma unroll 1
  for (int c = t; c < V; c += NT) {
    const u64 at = sm_place(sm_key(to_f32(logits[c])), c);
    m.place[c] = at;
    first = at > first ? at : first;
  }
  SampleRow r;
  const SampleSettings s = sm_settings(p, row, r);
  sm_table<NT>(m.table, r);
  first = sm_block<NT>(first, m.red, [](u64 a, u64 b) { return a > b ? a : b; });
  const bool there = sm_top(r, first);
  if (!there || s.k == 1) {
    if (t == 0) {
      p.token[row] = there ? (int64_t)(uint32_t)~first : -1;
      p.logprob[row] = there ? 0.0f : NAN;
    }
    return;
  }
  __syncthreads();
#pragma unroll 1
  for (int c = t; c < kShort; c += NT) m.weight[c] = c < V ? r.weight(sm_value((uint32_t)(m.place[c] >> 32))) : 0;
  __syncthreads();
  u64 w[per];   // of consecutive logits
#pragma unroll
  for (int q = 0; q < per; ++q) w[q] = m.weight[t * per + q];
  u64 cut = 0;
  if (s.k > 1 || s.top_p < 1 || r.lowest > -INFINITY) {
    u64 at[per];
#pragma unroll
    for (int q = 0; q < per; ++q) at[q] = t * per + q < V ? m.place[t * per + q] : 0;
    __syncthreads();
    if (s.k > 1 || s.top_p < 1) {
      sm_sort<NT, per>(m.place, V);
      const int n = s.k > 1 ? (int)s.k : V;
      cut = m.place[n - 1];
      if (s.top_p < 1) {
        u64 mass = 0;
#pragma unroll
        for (int q = 0; q < per; ++q) mass += at[q] >= cut ? w[q] : 0;
        mass = sm_block<NT>(mass, m.red, [](u64 a, u64 b) { return a + b; });
        __syncthreads();
        cut = sm_reach<NT>(m, n, sm_target(s, mass), [&](float, u64 at) { return m.weight[(uint32_t)~at]; });
      }
    }
#pragma unroll
    for (int q = 0; q < per; ++q) {   // without branches: with them the compiler loses the zeros
      const double z = r.z(sm_value((uint32_t)(at[q] >> 32)));
      w[q] = (at[q] >= cut) & ((at[q] == first) | (z >= r.lowest)) ? w[q] : 0;
    }
  }
  u64 mine = 0;
#pragma unroll
  for (int q = 0; q < per; ++q) mine += w[q];
  u64 upto = sm_scan(mine), total = 0;
  __syncthreads();
  if (t % 64 == 63) m.red[t / 64] = upto;
  __syncthreads();
  for (int k = 0; k < NT / 64; ++k) {
    if (k == t / 64) upto += total;
    total += m.red[k];
  }
  const u64 goal = sm_goal(p, row, total);
  if (!(upto > goal && upto - mine <= goal)) return;   // one thread has it
  u64 run = upto - mine;
  int q = 0;
#pragma unroll
  for (int k = 0; k < per - 1; ++k) {
    run += w[k];
    if (run <= goal) q = k + 1;
  }
  p.token[row] = t * per + q;
  p.logprob[row] = sm_logprob(r, to_f32(logits[t * per + q]), total);
}

// ------------------------------------------------------------------ rows of one workgroup
// Bound by the chain of its passes (maximum, histogram, gather and sort, sums, token): 64 rows of 5000 17.5 us with all kept,
// 27 with top_k, 31 with top_p; of 20000 22, 32, 41.
template <typename IT, int NT, int J>   // J tiles a wavefront: the first stays in registers, the others are read anew (from L2) each time
__global__ void __launch_bounds__(NT) k_sample_row(const SampleParams p) {
  __shared__ SampleLds<NT> m;
  __shared__ u64 tiles[J * NT / 64];
  const int64_t row = p.first + blockIdx.x, V = p.V;
  const IT *logits = (const IT *)p.logits + row * p.sl;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  float held[kE];
  if (threadIdx.x * kE < V) sm_load<IT>(logits, threadIdx.x * kE, V, held);
  auto tile_at = [&](int j, float (&v)[kE]) {   // the lane's first index
    const int64_t i = (int64_t)(j * (NT / 64) + wave) * kTile + lane * kE;
    if (j == 0) {
#pragma unroll
      for (int q = 0; q < kE; ++q) v[q] = held[q];
    } else if (i < V) {
      sm_load<IT>(logits, i, V, v);
    }
    return i;
  };
  auto each = [&](auto f) {
#pragma unroll 2
    for (int j = 0; j < J; ++j) {
      float v[kE];
      const int64_t i = tile_at(j, v);
#pragma unroll
      for (int q = 0; q < kE; ++q)
        if (i + q < V) f((uint32_t)(i + q), v[q]);
    }
  };
  u64 first = 0;
  each([&](uint32_t i, float l) {
    const u64 at = sm_place(sm_key(l), i);
    first = at > first ? at : first;
  });
  first = sm_block<NT>(first, m.red, [](u64 a, u64 b) { return a > b ? a : b; });
  SampleRow r;
  const SampleSettings s = sm_settings(p, row, r);
  if (!sm_top(r, first)) {
    if (threadIdx.x == 0) {
      p.token[row] = -1;
      p.logprob[row] = NAN;
    }
    return;
  }
  if (s.k == 1) {
    if (threadIdx.x == 0) {
      p.token[row] = (uint32_t)~first;
      p.logprob[row] = 0.0f;
    }
    return;
  }
  sm_table<NT>(m.table, r);
  u64 cut = 0;
  if (s.k > 1 || s.top_p < 1) {
    for (int b = threadIdx.x; b < kBins; b += NT) m.mass[b] = m.count[b] = 0;
    __syncthreads();
    each([&](uint32_t, float l) {
      const int b = r.bin(l);
      if (s.k > 1) atomicAdd(&m.count[b], 1u);
      if (s.top_p < 1) atomicAdd(&m.mass[b], r.weight(l));
    });
    __syncthreads();
    cut = sm_select<NT>(m, r, s, each);
  }
  const SampleCut kept(sm_min_p(r, cut, first));
  __syncthreads();
#pragma unroll 1
  for (int j = 0; j < J; ++j) {
    float v[kE];
    const int64_t i = tile_at(j, v);
    u64 sum = 0;
#pragma unroll
    for (int q = 0; q < kE; ++q) sum += i + q < V ? kept.weight(r, (uint32_t)(i + q), v[q]) : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    if (lane == 0) tiles[j * (NT / 64) + wave] = sum;
  }
  __syncthreads();
  int64_t tile;
  u64 run, goal, total;
  sm_tile(p, row, tiles, J * NT / 64, tile, run, goal, total);
  if (wave != tile % (NT / 64)) return;   // the wavefront that holds it
  float v[kE];
  const int64_t i = tile_at((int)(tile / (NT / 64)), v);
  sm_pick(p, r, row, kept, i, v, run, goal, total);
}

// ------------------------------------------------------------------ longer rows
template <int NT> constexpr int sm_chunk() { return 4 * NT * kE; }   // logits a workgroup
template <typename IT, int NT>
struct SampleChunk {
  float v[4][kE];
  int64_t row, c, at;   // at: the lane's first index
  __device__ __forceinline__ SampleChunk(const SampleParams &p, int64_t chunks) {
    const int64_t b = p.first + blockIdx.x;
    row = b / chunks;
    c = b % chunks;
    const IT *logits = (const IT *)p.logits + row * p.sl;
    at = c * sm_chunk<NT>() + (threadIdx.x / 64) * kTile + (threadIdx.x % 64) * kE;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (index(j) < p.V) sm_load<IT>(logits, index(j), p.V, v[j]);
  }
  __device__ __forceinline__ int64_t index(int j) const { return at + (int64_t)j * (NT / 64) * kTile; }
  template <typename F>
  __device__ __forceinline__ void each(int64_t V, F f) const {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < kE; ++q)
        if (index(j) + q < V) f((uint32_t)(index(j) + q), v[j][q]);
  }
};
__device__ __forceinline__ u64 sm_first(const SampleParams &p, int64_t row) {   // the row's, of its chunks'; for a whole wavefront
  u64 best = 0;
  for (int64_t c = threadIdx.x % 64; c < p.parts; c += 64) best = max(best, (u64)p.firsts[row * p.parts + c]);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) best = max(best, (u64)__shfl_xor(best, d));
  return best;
}
// The five kernels at 64 x 131072 in bf16 (16.8 MB; once from HBM, then from L2 and the memory-side cache): 9, 19, 64, 14, 10 us.
template <typename IT>
__global__ void __launch_bounds__(256) k_sample_first(const SampleParams p) {
  __shared__ u64 red[4];
  const SampleChunk<IT, 256> x(p, p.parts);
  u64 first = 0;
  x.each(p.V, [&](uint32_t i, float l) {
    const u64 at = sm_place(sm_key(l), i);
    first = at > first ? at : first;
  });
  first = sm_block<256>(first, red, [](u64 a, u64 b) { return a > b ? a : b; });
  if (threadIdx.x == 0) p.firsts[x.row * p.parts + x.c] = first;
}
template <typename IT, int NT>
__global__ void __launch_bounds__(NT) k_sample_bins(const SampleParams p) {
  __shared__ u64 mass[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ double table[kTable];
  const SampleChunk<IT, NT> x(p, p.chunks);
  SampleRow r;
  const SampleSettings s = sm_settings(p, x.row, r);
  if (!sm_top(r, sm_first(p, x.row)) || s.k == 1 || (s.k == 0 && s.top_p >= 1)) return;   // the whole workgroup
  sm_table<NT>(table, r);
  for (int b = threadIdx.x; b < kBins; b += NT) mass[b] = count[b] = 0;
  __syncthreads();
  x.each(p.V, [&](uint32_t, float l) {
    const int b = r.bin(l);
    if (s.k > 1) atomicAdd(&count[b], 1u);
    if (s.top_p < 1) atomicAdd(&mass[b], r.weight(l));
  });
  __syncthreads();
  const int64_t at = (x.row * p.chunks + x.c) * kBins;
  for (int b = threadIdx.x; b < kBins; b += NT) {
    if (s.k > 1) p.counts[at + b] = count[b];
    if (s.top_p < 1) p.masses[at + b] = mass[b];
  }
}
// A workgroup a row: each stage (top_k, then top_p) adds the chunks' histograms, finds the bin and gathers its logits from
// the whole row, 17 of 29 us; 32 registers of loads are under way at once (64 spill: the five kernels 137 us with both stages against 104).
template <typename IT, int NT>
__global__ void __launch_bounds__(NT) k_sample_cut(const SampleParams p) {
  __shared__ SampleLds<NT> m;
  const int64_t row = p.first + blockIdx.x, V = p.V;
  const IT *logits = (const IT *)p.logits + row * p.sl;
  SampleRow r;
  const SampleSettings s = sm_settings(p, row, r);
  const u64 first = sm_first(p, row);
  u64 cut = s.k == 1 ? first : 0;
  if (sm_top(r, first) && s.k != 1 && (s.k > 1 || s.top_p < 1)) {
    sm_table<NT>(m.table, r);
    for (int b = threadIdx.x; b < kBins; b += NT) {
      uint32_t n = 0;
      u64 w = 0;
      const int64_t at = row * p.chunks * kBins + b;
      if (s.k > 1)
#pragma unroll 4
        for (int64_t c = 0; c < p.chunks; ++c) n += p.counts[at + c * kBins];
      if (s.top_p < 1)
#pragma unroll 4
        for (int64_t c = 0; c < p.chunks; ++c) w += p.masses[at + c * kBins];
      m.count[b] = n;
      m.mass[b] = w;
    }
    __syncthreads();
    auto each = [&](auto f) {
      constexpr int64_t stride = NT * kE;
      constexpr int U = 16 / sizeof(IT);   // loads under way together: 32 registers
      struct Raw { IT e[kE]; };
#pragma unroll 1
      for (int64_t i0 = (int64_t)threadIdx.x * kE; i0 < V; i0 += U * stride) {
        Raw raw[U];
#pragma unroll
        for (int j = 0; j < U; ++j)
          if (i0 + j * stride + kE <= V) __builtin_memcpy(&raw[j], logits + i0 + j * stride, sizeof(Raw));
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int64_t i = i0 + j * stride;
          if (i >= V) break;
          if (i + kE > V)
            for (int q = 0; q < kE; ++q) raw[j].e[q] = logits[i + q < V ? i + q : V - 1];
#pragma unroll
          for (int q = 0; q < kE; ++q)
            if (i + q < V) f((uint32_t)(i + q), to_f32(raw[j].e[q]));
        }
      }
    };
    cut = sm_select<NT>(m, r, s, each);
  }
  if (sm_top(r, first)) cut = sm_min_p(r, cut, first);
  if (threadIdx.x == 0) p.cuts[row] = cut;
}
template <typename IT>
__global__ void __launch_bounds__(256) k_sample_tiles(const SampleParams p) {
  __shared__ double table[kTable];
  const SampleChunk<IT, 256> x(p, p.parts);
  SampleRow r;
  sm_settings(p, x.row, r);
  sm_table<256>(table, r);
  const SampleCut cut(p.filtered ? p.cuts[x.row] : 0);
  if (!sm_top(r, sm_first(p, x.row))) return;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t i = x.index(j);
    u64 sum = 0;
#pragma unroll
    for (int q = 0; q < kE; ++q) sum += i + q < p.V ? cut.weight(r, (uint32_t)(i + q), x.v[j][q]) : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    if (threadIdx.x % 64 == 0 && i < p.V) p.tiles[x.row * p.ntiles + i / kTile] = sum;
  }
}
template <typename IT>
__global__ void __launch_bounds__(256) k_sample_token(const SampleParams p) {
  __shared__ double table[kTable];
  __shared__ u64 red[4], found[2];
  const int64_t row = p.first + blockIdx.x;
  const u64 *masses = (const u64 *)p.tiles + row * p.ntiles;
  SampleRow r;
  sm_settings(p, row, r);
  sm_table<256>(table, r);
  // consecutive tiles a thread
  const int64_t per = (p.ntiles + 255) / 256, t0 = threadIdx.x * per, t1 = t0 + per < p.ntiles ? t0 + per : p.ntiles;
  u64 mine = 0;
  for (int64_t t = t0; t < t1; ++t) mine += masses[t];
  const SampleCut cut(p.filtered ? p.cuts[row] : 0);
  if (!sm_top(r, sm_first(p, row))) {
    if (threadIdx.x == 0) {
      p.token[row] = -1;
      p.logprob[row] = NAN;
    }
    return;
  }
  u64 upto = sm_scan(mine);
  if (threadIdx.x % 64 == 63) red[threadIdx.x / 64] = upto;
  __syncthreads();
  u64 total = 0;
  for (int k = 0; k < 4; ++k) {
    if (k == (int)threadIdx.x / 64) upto += total;
    total += red[k];
  }
  const u64 goal = sm_goal(p, row, total);
  if (upto > goal && upto - mine <= goal) {   // one thread
    u64 run = upto - mine;
    int64_t t = t0;
    for (; t + 1 < t1 && run + masses[t] <= goal; ++t) run += masses[t];
    found[0] = t;
    found[1] = run;
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const int64_t i = found[0] * kTile + threadIdx.x * kE;
  float v[kE] = {};
  if (i < p.V) sm_load<IT>((const IT *)p.logits + row * p.sl, i, p.V, v);
  sm_pick(p, r, row, cut, i, v, found[1], goal, total);
}

template <typename IT, int NT>
static void sample_long(SampleParams p, hipStream_t s) {
  auto launch = [&](auto kernel, int64_t all, int threads) {
    const int64_t most = kGridThreads / threads;
    for (p.first = 0; p.first < all; p.first += most)
      hipLaunchKernelGGL(kernel, dim3((unsigned)(all - p.first < most ? all - p.first : most)), dim3(threads), 0, s, p);
  };
  launch(k_sample_first<IT>, p.R * p.parts, 256);
  if (p.filtered) {
    launch(k_sample_bins<IT, NT>, p.R * p.chunks, NT);
    launch(k_sample_cut<IT, 1024>, p.R, 1024);
  }
  launch(k_sample_tiles<IT>, p.R * p.parts, 256);
  launch(k_sample_token<IT>, p.R, 256);
}
template <typename IT>
static hipError_t sample_t(SampleParams p, hipStream_t s) {
  if (p.chunks) {
    if (p.chunk == sm_chunk<256>()) sample_long<IT, 256>(p, s);
    else sample_long<IT, 1024>(p, s);
    return hipGetLastError();
  }
  const int64_t most = kGridThreads / 1024;
  for (; p.first < p.R; p.first += most) {
    const dim3 grid((unsigned)(p.R - p.first < most ? p.R - p.first : most));
    if (p.V <= kShort) hipLaunchKernelGGL((k_sample_short<IT>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((k_sample_row<IT, 1024, 4>), grid, dim3(1024), 0, s, p);
  }
  return hipGetLastError();
}
hipError_t launch_sample(const SampleParams &p, int dtype, hipStream_t s) {
  return dtype == 0 ? sample_t<float>(p, s) : dtype == 1 ? sample_t<bf16_t>(p, s) : sample_t<f16_t>(p, s);
}

}  // namespace ssm
