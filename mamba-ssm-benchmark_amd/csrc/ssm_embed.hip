// Token embedding with a scale, and its gradient by sorted tokens:
//   out_i = scale w[token_i]  (zeros for a token outside [0, V)),   dw_v = scale sum over i with token_i = v of dout_i.
// The gradient sorts the tokens (stable radix sort, so equal tokens keep their order), adds the rows of dout that belong
// to one token in that order and writes every row of dw once, zeros included: no float atomics, bitwise repeatable,
// nothing is read back on the host.
#include <algorithm>

#include "ssm_device.hpp"
#include "ssm_internal.hpp"

namespace ssm {

template <typename IT, int V>
__device__ __forceinline__ void em_load(const IT *src, float (&v)[V]) {
  struct alignas(V * sizeof(IT)) Pack { IT e[V]; };
  const Pack k = *(const Pack *)src;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = Conv<IT>::load(&k.e[i]);
}
template <typename IT, int V>
__device__ __forceinline__ void em_store(IT *dst, const float (&v)[V]) {
  struct alignas(V * sizeof(IT)) Pack { IT e[V]; };
  Pack k;
#pragma unroll
  for (int i = 0; i < V; ++i) Conv<IT>::store(&k.e[i], v[i]);
  *(Pack *)dst = k;
}

// `lanes` threads a row (a power of two), 256 / lanes rows a workgroup, a row in as few loads as its threads allow.  Bound
// by HBM: 16384 rows of 1024 in bf16 67 MB in 12 us, 5.6 TB/s (8192 of 256 in float32 4.5 us: rows of 256 tokens stay in L2).
template <typename IT, int V>
__global__ void __launch_bounds__(256) k_embed_fwd(const EmbedParams p) {
  const int l = threadIdx.x & (p.lanes - 1);
  const int64_t i = p.first + (int64_t)blockIdx.x * (256 / p.lanes) + threadIdx.x / p.lanes;
  if (i >= p.n) return;
  const int64_t v = p.tokens[i];
  const bool there = v >= 0 && v < p.V;
  const IT *src = (const IT *)p.w + (there ? v : 0) * p.sw;
  IT *dst = (IT *)p.out + i * p.so;
  for (int64_t j = (int64_t)l * V; j < p.D; j += (int64_t)p.lanes * V) {
    float e[V];
    em_load<IT, V>(src + j, e);
#pragma unroll
    for (int k = 0; k < V; ++k) e[k] = there ? e[k] * p.scale : 0.0f;
    em_store<IT, V>(dst + j, e);
  }
}

// ------------------------------------------------------------------ sort
// One stable pass over a digit of `bits` bits.  Each of nw wavefronts owns `per` consecutive items: k_embed_count counts
// its digits, k_embed_place finds where each digit's items of each wavefront begin and writes them, 64 at a time; within
// those, a lane's place among the lanes of its digit comes from ballots of the digit's bits.
__device__ __forceinline__ uint32_t em_key(const EmbedParams &p, int64_t i) {
  if (p.pass) return p.key_in[i];
  const int64_t v = p.tokens[i];
  return v >= 0 && v < p.V ? (uint32_t)v : (uint32_t)p.V;   // tokens outside the vocabulary come last
}
// A pass of the sort over 9 bits of the keys at most, as few passes as those allow, evenly shared: counts, then places.  Up
// to 64 wavefronts, each with a run of the tokens, of which the second kernel adds the earlier ones' counts by itself: no
// third launch and no flags to wait for.  16384 tokens: 3.4-4.2 us and 10-11, both latency (0.2 MB).
__global__ void __launch_bounds__(256) k_embed_count(const EmbedParams p) {
  __shared__ uint32_t count[4][1 << kEmbedBits];
  const int lane = threadIdx.x % 64, w = threadIdx.x / 64, B = 1 << p.bits;
  const int64_t wave = (int64_t)blockIdx.x * 4 + w;
  for (int b = lane; b < B; b += 64) count[w][b] = 0;
  __syncthreads();
  if (wave < p.nw)
    for (int64_t i = wave * p.per + lane; i < p.n && i < (wave + 1) * p.per; i += 64)
      atomicAdd(&count[w][(em_key(p, i) >> p.shift) & (B - 1)], 1u);
  __syncthreads();
  if (wave < p.nw)
    for (int b = lane; b < B; b += 64) p.hist[wave * B + b] = count[w][b];
}
__global__ void __launch_bounds__(256) k_embed_place(const EmbedParams p) {
  __shared__ uint32_t base[4][1 << kEmbedBits];
  __shared__ uint32_t sums[256];
  const int lane = threadIdx.x % 64, w = threadIdx.x / 64, B = 1 << p.bits;
  const int64_t wave0 = (int64_t)blockIdx.x * 4;
  // items of the digits below, then of this digit in the wavefronts before: two digits a thread
  constexpr int per = 2;
  static_assert(per * 256 == 1 << kEmbedBits, "digits");
  uint32_t total[per] = {}, run = 0, mine[per][4] = {};
  if ((int)threadIdx.x * per < B) {
    const uint2 *h = (const uint2 *)p.hist + threadIdx.x;
#pragma unroll 32
    for (int v = 0; v < (int)p.nw; ++v) {
      const uint2 c = h[(int64_t)v * (B / 2)];
      total[0] += c.x;
      total[1] += c.y;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        mine[0][q] += v < wave0 + q ? c.x : 0;
        mine[1][q] += v < wave0 + q ? c.y : 0;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < per; ++k) {
    run += total[k];
#pragma unroll
    for (int q = 0; q < 4; ++q) base[q][threadIdx.x * per + k] = mine[k][q];
  }
  sums[threadIdx.x] = run;
  __syncthreads();
  for (int d = 1; d < 256; d *= 2) {
    const uint32_t t = threadIdx.x >= d ? sums[threadIdx.x - d] : 0;
    __syncthreads();
    sums[threadIdx.x] += t;
    __syncthreads();
  }
  run = sums[threadIdx.x] - run;
#pragma unroll
  for (int k = 0; k < per; ++k) {
#pragma unroll
    for (int q = 0; q < 4; ++q) base[q][threadIdx.x * per + k] += run;
    run += total[k];
  }
  __syncthreads();
  const int64_t wave = wave0 + w, end = (wave + 1) * p.per < p.n ? (wave + 1) * p.per : p.n;
  constexpr int U = 4;   // steps whose items are loaded together
  for (int64_t i0 = wave * p.per; i0 < end; i0 += 64 * U) {   // no barrier in here: wavefronts may differ in their steps
    uint32_t keys[U], places[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + 64 * u + lane;
      keys[u] = i < end ? em_key(p, i) : 0;
      places[u] = i < end ? (p.pass ? p.pos_in[i] : (uint32_t)i) : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = i0 + 64 * u + lane < end;
      const uint32_t digit = (keys[u] >> p.shift) & (B - 1);
      uint64_t same = __ballot(there);
      for (int b = 0; b < p.bits; ++b) {
        const uint64_t set = __ballot((digit >> b) & 1);
        same &= (digit >> b) & 1 ? set : ~set;
      }
      const int before = __popcll(same & ((1ull << lane) - 1));
      uint32_t at = 0;
      if (there) at = base[w][digit] + before;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (there && before == 0) base[w][digit] += __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (there) {
        p.key_out[at] = keys[u];
        p.pos_out[at] = places[u];
      }
    }
  }
}

// Place i is the first of the tokens above its forerunner's up to its own: mostly few, else the wavefront's work.
__device__ __forceinline__ void em_bounds(const EmbedParams &p, int64_t i, bool there, int64_t before, int64_t own) {
  const int64_t v0 = before + 1, v1 = there ? own : before;
  uint64_t wide = __ballot(v1 - v0 >= 16);
  if (v1 - v0 < 16)
    for (int64_t v = v0; v <= v1; ++v) p.start[v] = (uint32_t)i;
  while (wide) {
    const int l = __ffsll((unsigned long long)wide) - 1;
    wide &= wide - 1;
    const int64_t w1 = __shfl(v1, l), at = __shfl(i, l);
    for (int64_t v = __shfl(v0, l) + threadIdx.x % 64; v <= w1; v += 64) p.start[v] = (uint32_t)at;
  }
}

// All passes in one workgroup, for up to kEmbedShort tokens: keys and places stay in LDS, a wavefront's items pass through
// its registers.  The same steps as above, and the first place of every token with them.  8192 tokens, a pass: 13.5 us,
// the chain of its barriers.
__global__ void __launch_bounds__(1024) k_embed_sort(const EmbedParams p) {
  constexpr int U = kEmbedShort / 1024, B = 1 << kEmbedBits;
  __shared__ uint32_t keys[kEmbedShort];
  __shared__ uint16_t places[kEmbedShort];
  __shared__ uint32_t base[16][B];
  __shared__ uint32_t sums[16];
  const int lane = threadIdx.x % 64, w = threadIdx.x / 64, n = (int)p.n;
  const int steps = (n + 1023) / 1024, i0 = w * steps * 64;   // of a wavefront
  for (int pass = 0; pass * p.bits < p.all_bits; ++pass) {
    const int shift = pass * p.bits;
    for (int b = threadIdx.x; b < 16 * B; b += 1024) base[b / B][b % B] = 0;
    uint32_t key[U], place[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 64 * u + lane;
      if (u >= steps || i >= n) continue;
      if (pass) {
        key[u] = keys[i];
        place[u] = places[i];
      } else {
        const int64_t v = p.tokens[i];
        key[u] = v >= 0 && v < p.V ? (uint32_t)v : (uint32_t)p.V;
        place[u] = i;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < steps && i0 + 64 * u + lane < n) atomicAdd(&base[w][(key[u] >> shift) & (B - 1)], 1u);
    __syncthreads();
    uint32_t all = 0, before = 0;
    if (threadIdx.x < B)
      for (int v = 0; v < 16; ++v) all += base[v][threadIdx.x];
    uint32_t upto = all;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t t = __shfl_up(upto, d);
      if (lane >= d) upto += t;
    }
    if (lane == 63) sums[w] = upto;
    __syncthreads();
    for (int v = 0; v < w; ++v) before += sums[v];
    if (threadIdx.x < B) {
      uint32_t at = before + upto - all;
      for (int v = 0; v < 16; ++v) {
        const uint32_t c = base[v][threadIdx.x];
        base[v][threadIdx.x] = at;
        at += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= steps) continue;
      const bool there = i0 + 64 * u + lane < n;
      const uint32_t digit = there ? (key[u] >> shift) & (B - 1) : 0;
      uint64_t same = __ballot(there);
      for (int b = 0; b < p.bits; ++b) {
        const uint64_t set = __ballot((digit >> b) & 1);
        same &= (digit >> b) & 1 ? set : ~set;
      }
      const int ahead = __popcll(same & ((1ull << lane) - 1));
      uint32_t at = 0;
      if (there) at = base[w][digit] + ahead;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (there && ahead == 0) base[w][digit] += __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (there) {
        keys[at] = key[u];
        places[at] = (uint16_t)place[u];
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i - (int)threadIdx.x <= n; i += 1024) {   // whole wavefronts, and place n too
    if (i < n) {
      p.key[0][i] = keys[i];
      p.pos[0][i] = places[i];
    }
    em_bounds(p, i, i <= n, i && i <= n ? (int64_t)keys[i - 1] : -1, i < n ? (int64_t)keys[i] : p.V);
  }
}

// ------------------------------------------------------------------ sums
// Sum of dout's rows at sorted places [from, to), columns j .. j + V, in order; up to 16 rows are read together.
template <int U, typename IT, int V>
__device__ __forceinline__ void em_some(const EmbedParams &p, int64_t from, int64_t j, float (&acc)[V]) {
  struct alignas(V * sizeof(IT)) Pack { IT e[V]; };
  Pack e[U];
#pragma unroll
  for (int u = 0; u < U; ++u) e[u] = *(const Pack *)((const IT *)p.dout + (int64_t)p.pos_in[from + u] * p.sd + j);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += to_f32(e[u].e[i]);
}
template <typename IT, int V>
__device__ __forceinline__ void em_rows(const EmbedParams &p, int64_t from, int64_t to, int64_t j, float (&acc)[V]) {
  int64_t k = from;
  for (; k + 16 <= to; k += 16) em_some<16, IT, V>(p, k, j, acc);
  if (k + 8 <= to) {
    em_some<8, IT, V>(p, k, j, acc);
    k += 8;
  }
  if (k + 4 <= to) {
    em_some<4, IT, V>(p, k, j, acc);
    k += 4;
  }
  if (k + 2 <= to) {
    em_some<2, IT, V>(p, k, j, acc);
    k += 2;
  }
  if (k < to) em_some<1, IT, V>(p, k, j, acc);
}
template <int V>
__device__ __forceinline__ void em_parts(const float *src, int64_t from, int64_t to, int64_t D, int64_t j, float (&acc)[V]) {
  for (int64_t k = from; k < to; k += 8) {
    float e[8][V];
#pragma unroll
    for (int u = 0; u < 8; ++u) em_load<float, V>(src + (k + u < to ? k + u : to - 1) * D + j, e[u]);
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += k + u < to ? e[u][i] : 0.0f;
  }
}

// The sums of those pieces of kEmbedPiece sorted places that hold one token alone, and the first place of every token.
// Without them a token that fills a batch is one lane group's chain of loads: 2048 of one token 131 us against 24.
template <typename IT, int V>
__global__ void __launch_bounds__(256) k_embed_pieces(const EmbedParams p) {
  if ((int64_t)blockIdx.x >= p.npiece_blocks) {
    const int64_t i = ((int64_t)blockIdx.x - p.npiece_blocks) * 256 + threadIdx.x;
    em_bounds(p, i, i <= p.n, i && i <= p.n ? (int64_t)p.key_in[i - 1] : -1, i < p.n ? (int64_t)p.key_in[i] : p.V);
    return;
  }
  const int l = threadIdx.x & (p.lanes - 1);
  const int64_t piece = (int64_t)blockIdx.x * (256 / p.lanes) + threadIdx.x / p.lanes, from = piece * kEmbedPiece;
  if (from + kEmbedPiece > p.n) return;
  const uint32_t key = p.key_in[from];
  if (key >= (uint32_t)p.V || p.key_in[from + kEmbedPiece - 1] != key) return;
  for (int64_t j = (int64_t)l * V; j < p.D; j += (int64_t)p.lanes * V) {
    float acc[V] = {};
    em_rows<IT, V>(p, from, from + kEmbedPiece, j, acc);
    em_store<float, V>(p.piece + piece * p.D + j, acc);
  }
}
// The same of kEmbedGroup pieces, where the batch is long.
template <int V>
__global__ void __launch_bounds__(256) k_embed_groups(const EmbedParams p) {
  constexpr int64_t whole = (int64_t)kEmbedPiece * kEmbedGroup;
  const int l = threadIdx.x & (p.lanes - 1);
  const int64_t group = (int64_t)blockIdx.x * (256 / p.lanes) + threadIdx.x / p.lanes, from = group * whole;
  if (from + whole > p.n) return;
  const uint32_t key = p.key_in[from];
  if (key >= (uint32_t)p.V || p.key_in[from + whole - 1] != key) return;
  for (int64_t j = (int64_t)l * V; j < p.D; j += (int64_t)p.lanes * V) {
    float acc[V] = {};
    em_parts<V>(p.piece, group * kEmbedGroup, (group + 1) * kEmbedGroup, p.D, j, acc);
    em_store<float, V>(p.group + group * p.D + j, acc);
  }
}
// Every row of dw: those of the tokens that come, by the first of their places (a lane group looks at each), with
// whole pieces (and groups of them) in their sums' place; zeros by the first workgroups, which wait for nothing.  Each row
// of dw is written once, with no pass of zeros before: 50001 rows of 1024 in bf16 from 16384 rows of dout 136 MB in 27 us,
// 5 TB/s, HBM; 256 rows of 256 in float32 from 8192 6 us, the longest run of one token.
template <typename IT, int V>
__global__ void __launch_bounds__(256) k_embed_rows(const EmbedParams p) {
  constexpr int64_t P = kEmbedPiece, G = kEmbedGroup;
  const int l = threadIdx.x & (p.lanes - 1), group = threadIdx.x / p.lanes, groups = 256 / p.lanes;
  if ((int64_t)blockIdx.x < p.nzero_blocks) {
    const int64_t v0 = (int64_t)blockIdx.x * kEmbedRows;
    __shared__ uint32_t start[kEmbedRows + 1];
    for (int i = threadIdx.x; i <= kEmbedRows && v0 + i <= p.V; i += 256) start[i] = p.start[v0 + i];
    __syncthreads();
    const float zero[V] = {};
    for (int i = group; i < kEmbedRows && v0 + i < p.V; i += groups)
      if (start[i] == start[i + 1])
        for (int64_t j = (int64_t)l * V; j < p.D; j += (int64_t)p.lanes * V) em_store<IT, V>((IT *)p.dw + (v0 + i) * p.D + j, zero);
    return;
  }
  const int64_t i = p.first + ((int64_t)blockIdx.x - p.nzero_blocks) * groups + group;
  if (i >= p.n) return;
  {
    const uint32_t v = p.key_in[i], last = i ? p.key_in[i - 1] : v + 1;
    if (v >= (uint32_t)p.V || last == v) return;
    const int64_t s = i, e = p.start[v + 1];
    int64_t p0 = (s + P - 1) / P, p1 = e / P;         // whole pieces
    if (p0 >= p1 || !p.pieces) p0 = p1 = -1;
    int64_t g0 = (p0 + G - 1) / G, g1 = p1 / G;       // whole groups
    if (!p.group || p0 < 0 || g0 >= g1) g0 = g1 = -1;
    for (int64_t j = (int64_t)l * V; j < p.D; j += (int64_t)p.lanes * V) {
      float acc[V] = {};
      if (p0 < 0) {
        em_rows<IT, V>(p, s, e, j, acc);
      } else {
        em_rows<IT, V>(p, s, p0 * P, j, acc);
        em_parts<V>(p.piece, p0, g0 < 0 ? p1 : g0 * G, p.D, j, acc);
        if (g0 >= 0) {
          em_parts<V>(p.group, g0, g1, p.D, j, acc);
          em_parts<V>(p.piece, g1 * G, p1, p.D, j, acc);
        }
        em_rows<IT, V>(p, p1 * P, e, j, acc);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] *= p.scale;
      em_store<IT, V>((IT *)p.dw + (int64_t)v * p.D + j, acc);
    }
  }
}

template <typename IT, int V>
static hipError_t embed_v(EmbedParams p, bool bwd, hipStream_t s) {
  p.lanes = 1;   // a row in as few loads as 256 threads allow
  while (p.lanes < 256 && (int64_t)p.lanes * V < p.D) p.lanes *= 2;
  const int64_t Q = 256 / p.lanes, most = kGridThreads / p.lanes;
  auto blocks = [&](int64_t rows) { return dim3((unsigned)((rows + Q - 1) / Q)); };
  if (!bwd) {
    for (; p.first < p.n; p.first += most)
      hipLaunchKernelGGL((k_embed_fwd<IT, V>), blocks(p.n - p.first < most ? p.n - p.first : most), dim3(256), 0, s, p);
    return hipGetLastError();
  }
  while ((p.V >> p.all_bits) > 0) ++p.all_bits;   // keys 0 .. V
  const int passes = (p.all_bits + kEmbedBits - 1) / kEmbedBits;
  p.bits = (p.all_bits + passes - 1) / passes;
  // One launch in place of two a pass and the bounds.  The gradient of 512 tokens of 256 12.4 us against 17.9, of 2048 16.1
  // against 20.3, of 8192 30.4 against 30.1, where the fewer launches save the host's time; with two passes (50000 rows)
  // 1024 tokens 43 against 53, 2048 50 against 48, 4096 57 against 53.
  const bool one = p.n <= (passes == 1 ? kEmbedShort : 2048);
  if (one) {
    p.bits = kEmbedBits;
    hipLaunchKernelGGL(k_embed_sort, dim3(1), dim3(1024), 0, s, p);
    p.key_in = p.key[0];
    p.pos_in = p.pos[0];
  } else {
    for (p.pass = 0; p.pass < passes; ++p.pass) {
      p.shift = p.pass * p.bits;
      p.key_out = p.key[p.pass & 1];
      p.pos_out = p.pos[p.pass & 1];
      hipLaunchKernelGGL(k_embed_count, dim3((unsigned)((p.nw + 3) / 4)), dim3(256), 0, s, p);
      hipLaunchKernelGGL(k_embed_place, dim3((unsigned)((p.nw + 3) / 4)), dim3(256), 0, s, p);
      p.key_in = p.key_out;
      p.pos_in = p.pos_out;
    }
  }
  // a few hundred places are summed one by one: 512 tokens 12.2 us against 13.8, but 41 against 17 if all are one token
  const int64_t pieces = p.n <= 512 ? 0 : p.n / kEmbedPiece, bounds = one ? 0 : (p.n + 256) / 256;
  p.pieces = pieces > 0;
  p.npiece_blocks = (pieces + Q - 1) / Q;
  if (pieces || bounds) hipLaunchKernelGGL((k_embed_pieces<IT, V>), dim3((unsigned)(p.npiece_blocks + bounds)), dim3(256), 0, s, p);
  if (p.group) hipLaunchKernelGGL((k_embed_groups<V>), blocks(pieces / kEmbedGroup), dim3(256), 0, s, p);
  p.nzero_blocks = (p.V + kEmbedRows - 1) / kEmbedRows;
  for (; p.first < p.n; p.first += most, p.nzero_blocks = 0)
    hipLaunchKernelGGL((k_embed_rows<IT, V>), dim3((unsigned)(p.nzero_blocks + (std::min(p.n - p.first, most) + Q - 1) / Q)), dim3(256), 0, s, p);
  return hipGetLastError();
}
template <typename IT>
static hipError_t embed_t(const EmbedParams &p, bool bwd, hipStream_t s) {
  return p.vec ? embed_v<IT, 16 / sizeof(IT)>(p, bwd, s) : embed_v<IT, 1>(p, bwd, s);
}
hipError_t launch_embed(const EmbedParams &p, int dtype, bool bwd, hipStream_t s) {
  return dtype == 0 ? embed_t<float>(p, bwd, s) : dtype == 1 ? embed_t<bf16_t>(p, bwd, s) : embed_t<f16_t>(p, bwd, s);
}

}  // namespace ssm
