// Token embedding with a scale, and its gradient by sorted tokens:
//   out_i = scale w[token_i]  (zeros for a token outside [0, V)),   dw_v = scale sum over i with token_i = v of dout_i.
// The gradient sorts the tokens (stable radix sort, so equal tokens keep their order), adds the rows of dout that belong
// to one token in that order and writes every row of dw once, zeros included: no float atomics, bitwise repeatable,
// nothing is read back on the host.
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

// `lanes` threads a row (a power of two), 256 / lanes rows a workgroup.
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
  // items of the digits below, then of this digit in the wavefronts before
  constexpr int per = (1 << kEmbedBits) / 256;
  uint32_t total[per], run = 0;
#pragma unroll
  for (int k = 0; k < per; ++k) {
    const int b = threadIdx.x * per + k;
    uint32_t all = 0, mine[4] = {0, 0, 0, 0};
    if (b < B)
#pragma unroll 8
      for (int64_t v = 0; v < p.nw; ++v) {
        const uint32_t c = p.hist[v * B + b];
        all += c;
#pragma unroll
        for (int q = 0; q < 4; ++q) mine[q] += v < wave0 + q ? c : 0;
      }
    total[k] = all;
    run += all;
#pragma unroll
    for (int q = 0; q < 4; ++q) base[q][b] = mine[q];
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
  for (int64_t i0 = wave * p.per; i0 < end; i0 += 64) {   // no barrier in here: wavefronts may differ in their steps
    const int64_t i = i0 + lane;
    const bool there = i < end;
    const uint32_t key = there ? em_key(p, i) : 0, pos = there ? (p.pass ? p.pos_in[i] : (uint32_t)i) : 0;
    const uint32_t digit = (key >> p.shift) & (B - 1);
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
      p.key_out[at] = key;
      p.pos_out[at] = pos;
    }
  }
}

// ------------------------------------------------------------------ sums
// Sum of dout's rows at sorted places [from, to), columns j .. j + V, in order; 8 rows are read together.
template <typename IT, int V>
__device__ __forceinline__ void em_rows(const EmbedParams &p, int64_t from, int64_t to, int64_t j, float (&acc)[V]) {
  for (int64_t k = from; k < to; k += 8) {
    float e[8][V];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t at = k + u < to ? k + u : to - 1;
      em_load<IT, V>((const IT *)p.dout + (int64_t)p.pos_in[at] * p.sd + j, e[u]);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += k + u < to ? e[u][i] : 0.0f;
  }
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
template <typename IT, int V>
__global__ void __launch_bounds__(256) k_embed_pieces(const EmbedParams p) {
  if ((int64_t)blockIdx.x >= p.npiece_blocks) {
    const int64_t v = ((int64_t)blockIdx.x - p.npiece_blocks) * 256 + threadIdx.x;
    if (v > p.V) return;
    int64_t lo = 0, hi = p.n;   // the first place whose key is not below v
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (p.key_in[mid] < (uint32_t)v) lo = mid + 1;
      else hi = mid;
    }
    p.start[v] = (uint32_t)lo;
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
// Every row of dw: the places of its token, with whole pieces (and groups of them) in their sums' place.
template <typename IT, int V>
__global__ void __launch_bounds__(256) k_embed_rows(const EmbedParams p) {
  const int l = threadIdx.x & (p.lanes - 1);
  const int64_t v = p.first + (int64_t)blockIdx.x * (256 / p.lanes) + threadIdx.x / p.lanes;
  if (v >= p.V) return;
  const int64_t s = p.start[v], e = p.start[v + 1];
  constexpr int64_t P = kEmbedPiece, G = kEmbedGroup;
  int64_t p0 = (s + P - 1) / P, p1 = e / P;         // whole pieces
  if (p0 >= p1) p0 = p1 = -1;
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
    for (int i = 0; i < V; ++i) acc[i] *= p.scale;
    em_store<IT, V>((IT *)p.dw + v * p.D + j, acc);
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
  int bits = 0;
  while ((p.V >> bits) > 0) ++bits;   // keys 0 .. V
  const int passes = (bits + kEmbedBits - 1) / kEmbedBits;
  p.bits = (bits + passes - 1) / passes;
  for (p.pass = 0; p.pass < passes; ++p.pass) {
    p.shift = p.pass * p.bits;
    p.key_out = p.key[p.pass & 1];
    p.pos_out = p.pos[p.pass & 1];
    hipLaunchKernelGGL(k_embed_count, dim3((unsigned)((p.nw + 3) / 4)), dim3(256), 0, s, p);
    hipLaunchKernelGGL(k_embed_place, dim3((unsigned)((p.nw + 3) / 4)), dim3(256), 0, s, p);
    p.key_in = p.key_out;
    p.pos_in = p.pos_out;
  }
  const int64_t pieces = p.n / kEmbedPiece;
  p.npiece_blocks = (pieces + Q - 1) / Q;
  hipLaunchKernelGGL((k_embed_pieces<IT, V>), dim3((unsigned)(p.npiece_blocks + (p.V + 256) / 256)), dim3(256), 0, s, p);
  if (p.group) hipLaunchKernelGGL((k_embed_groups<V>), blocks(pieces / kEmbedGroup), dim3(256), 0, s, p);
  for (; p.first < p.V; p.first += most)
    hipLaunchKernelGGL((k_embed_rows<IT, V>), blocks(p.V - p.first < most ? p.V - p.first : most), dim3(256), 0, s, p);
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
