// logits.cu -- per-request rules on logits before the sampler: penalties for repeated tokens, biases, grammar masks.
//
// LlmSampler.Sample applies one repetition penalty, once per occurrence (LlmSampler.cs:39-57); a server's requests
// each bring their own rules.  For token t of row r, with c the times t stands in the row's generated history and
// seen whether it stands anywhere in it (prompt included), in fp32 and in this order:
//   v = x[t];  seen: v = v > 0 ? v / repetition : v * repetition;   v -= frequency * c;   c > 0: v -= presence;
//   v += the row's biases of t, summed in list order;   a token whose mask bit is 0 becomes -inf, whatever v is.
//
// A row's histogram of its history would cost a zeroed vocab-sized buffer in memory; here a cluster of 1 to 8 CTAs holds
// it in distributed shared memory.  Each CTA owns a slice of the vocabulary, reads its share of the history once and
// counts each token in the owner's slice (integer atomics: the result does not depend on their order); after the
// cluster barrier one pass over the slice reads the logits, applies every rule and writes.  In place, 4-token groups
// that no rule touches are neither read nor written.  Bound: HBM (input and output once) for batches, the chain
// zero -> count -> pass of one launch for single rows.

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <math.h>

#include <utility>

#include "batch_ops.h"
#include "common.cuh"

namespace cg = cooperative_groups;

namespace zc {

namespace {

constexpr int LG_SMEM_MAX = 200 * 1024;
constexpr int LG_AHEAD = 8;  // 4-token groups per thread that are on their way while the history is counted

// A token's count: the top bit marks a history token, the others its generated occurrences.  16 bits hold it (and four
// CTAs an SM their slices of a vocabulary of 131,072) unless a history or a bias list is longer than 32767.
template <typename H>
struct Count;
template <>
struct Count<uint16_t> {
  static constexpr unsigned SEEN = 0x8000u;
  static __device__ __forceinline__ void note(unsigned* word_base, int i, bool generated) {  // word_base may be remote
    unsigned* w = word_base + (i >> 1);
    const int sh = 16 * (i & 1);
    if (generated) atomicAdd(w, 1u << sh);
    atomicOr(w, SEEN << sh);
  }
  static __device__ __forceinline__ void load(const uint16_t* p, unsigned (&h)[4]) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    h[0] = u.x & 0xffffu, h[1] = u.x >> 16, h[2] = u.y & 0xffffu, h[3] = u.y >> 16;
  }
  static __device__ __forceinline__ void raise(uint16_t* p, unsigned v) {
    for (unsigned old = *p; old < v;) {
      const unsigned was = atomicCAS(p, (unsigned short)old, (unsigned short)v);
      if (was == old) break;
      old = was;
    }
  }
  static __device__ __forceinline__ void mark(uint16_t* p) {
    for (unsigned old = *p; !(old & SEEN);) {
      const unsigned was = atomicCAS(p, (unsigned short)old, (unsigned short)(old | SEEN));
      if (was == old) break;
      old = was;
    }
  }
};
template <>
struct Count<uint32_t> {
  static constexpr unsigned SEEN = 0x80000000u;
  static __device__ __forceinline__ void note(unsigned* word_base, int i, bool generated) {
    if (generated) atomicAdd(word_base + i, 1u);
    atomicOr(word_base + i, SEEN);
  }
  static __device__ __forceinline__ void load(const uint32_t* p, unsigned (&h)[4]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    h[0] = u.x, h[1] = u.y, h[2] = u.z, h[3] = u.w;
  }
  static __device__ __forceinline__ void raise(uint32_t* p, unsigned v) { atomicMax(p, v); }
  static __device__ __forceinline__ void mark(uint32_t* p) { atomicOr(p, SEEN); }
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// Four logits as they lie in memory.
template <typename T>
struct Group {
  uint2 v;
};
template <>
struct Group<float> {
  float4 v;
};
__device__ __forceinline__ Group<float> fetch(const float* p) { return {*reinterpret_cast<const float4*>(p)}; }
template <typename T>
__device__ __forceinline__ Group<T> fetch(const T* p) {
  return {*reinterpret_cast<const uint2*>(p)};
}
__device__ __forceinline__ void floats(const Group<float>& g, float (&v)[4]) {
  v[0] = g.v.x, v[1] = g.v.y, v[2] = g.v.z, v[3] = g.v.w;
}
template <typename T>
__device__ __forceinline__ void floats(const Group<T>& g, float (&v)[4]) {
  const T* e = reinterpret_cast<const T*>(&g.v);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_f(e[i]);
}

struct Rules {
  float repetition, frequency, presence;
};

template <unsigned SEEN>
__device__ __forceinline__ float apply(float v, unsigned h, const Rules& r) {
  if (h) {
    v = v > 0.f ? __fdiv_rn(v, r.repetition) : v * r.repetition;
    const unsigned c = h & ~SEEN;
    if (c) v = (v - r.frequency * (float)c) - r.presence;
  }
  return v;
}

// VEC: both row starts are 16-byte (8-byte for 16-bit input) aligned, so 4 tokens move per access.
template <typename T, typename H, bool VEC, int LG_THREADS>
__global__ void __launch_bounds__(LG_THREADS, 1024 / LG_THREADS) logits_kernel(LogitsArgs a, int slice, bool in_place) {
  constexpr unsigned SEEN = Count<H>::SEEN;
  extern __shared__ __align__(16) unsigned smem[];
  H* hist = reinterpret_cast<H*>(smem);  // [slice]
  pdl_trigger();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const int row = blockIdx.x / ranks;
  const int v0 = min(a.vocab, rank * slice), v1 = min(a.vocab, v0 + slice);
  const T* x = reinterpret_cast<const T*>(a.x) + (size_t)row * a.x_stride;
  float* out = a.out + (size_t)row * a.out_stride;
  Rules rules{a.repetition ? a.repetition[row] : 1.f, a.frequency ? a.frequency[row] : 0.f,
              a.presence ? a.presence[row] : 0.f};

  // the row's history
  const int32_t* past = nullptr;
  int n_past = 0, n_prompt = 0;
  if (a.past) {
    const int pr = a.past_rows ? a.past_rows[row] : row;
    if ((unsigned)pr < (unsigned)a.past_count) {
      past = a.past + (size_t)pr * a.past_cap;
      n_past = min(max(a.past_len[pr], 0), a.past_cap);
      n_prompt = a.prompt_len ? min(max(a.prompt_len[pr], 0), n_past) : 0;
    }
    if (rules.repetition == 1.f && rules.frequency == 0.f && rules.presence == 0.f) n_past = 0;
  }
  const uint32_t* mask = nullptr;
  if (a.mask) {
    const int m = a.mask_rows ? a.mask_rows[row] : row;
    if ((unsigned)m < (unsigned)a.masks) mask = a.mask + (size_t)m * a.mask_stride;
  }
  // the first groups of the slice and their mask words, unless in place, where most logits are not needed
  const int n4 = VEC ? (v1 - v0) / 4 : 0;
  Group<T> ahead[LG_AHEAD];
  uint32_t words[LG_AHEAD];
  auto load_ahead = [&](int i0) {
#pragma unroll
    for (int u = 0; u < LG_AHEAD; ++u) {
      const int i = i0 + u * LG_THREADS;
      if (i < n4 && !in_place) ahead[u] = fetch(x + v0 + 4 * i);
      words[u] = mask && i < n4 ? __ldg(mask + ((v0 + 4 * i) >> 5)) : 0xffffffffu;
    }
  };
  load_ahead(threadIdx.x);
  if (n_past > 0) {  // the same for every CTA of the cluster
    constexpr int PER = 16 / sizeof(H);
    for (int i = threadIdx.x * PER; i < slice; i += LG_THREADS * PER)  // slice is a multiple of 32
      *reinterpret_cast<uint4*>(hist + i) = make_uint4(0, 0, 0, 0);
    cluster.sync();
    for (int i = rank * LG_THREADS + threadIdx.x; i < n_past; i += ranks * LG_THREADS) {
      const int t = past[i];
      if ((unsigned)t >= (unsigned)a.vocab) continue;
      const int owner = t / slice;
      Count<H>::note(cluster.map_shared_rank(smem, owner), t - owner * slice, i >= n_prompt);
    }
    cluster.sync();
  }

  const bool hashed = n_past > 0;
  for (int i0 = threadIdx.x; i0 < n4;) {
#pragma unroll
    for (int u = 0; u < LG_AHEAD; ++u) {
      const int i = i0 + u * LG_THREADS, t = v0 + 4 * i;
      if (i >= n4) break;
      const unsigned bits = (words[u] >> (t & 31)) & 15u;
      unsigned h[4] = {0, 0, 0, 0};
      if (hashed) Count<H>::load(hist + 4 * i, h);
      if (in_place) {
        if (bits == 15u && !(h[0] | h[1] | h[2] | h[3])) continue;
        ahead[u] = fetch(x + t);
      }
      float v[4];
      floats(ahead[u], v);
      if (h[0] | h[1] | h[2] | h[3]) {  // few groups hold a token of the history
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = apply<SEEN>(v[k], h[k], rules);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = bits >> k & 1u ? v[k] : -INFINITY;
      *reinterpret_cast<float4*>(out + t) = make_float4(v[0], v[1], v[2], v[3]);
    }
    i0 += LG_AHEAD * LG_THREADS;
    load_ahead(i0);
  }
  for (int t = v0 + (VEC ? (v1 - v0) / 4 * 4 : 0) + threadIdx.x; t < v1; t += LG_THREADS) {
    const bool ok = !mask || (__ldg(mask + (t >> 5)) >> (t & 31)) & 1u;
    const unsigned h = hashed ? hist[t - v0] : 0u;
    if (in_place && ok && !h) continue;
    out[t] = ok ? apply<SEEN>(to_f(x[t]), h, rules) : -INFINITY;
  }

  if (a.bias_start) {
    // Biases of this slice, onto the values just written.  The histogram is reused: a token's slot holds n - i of the
    // first list entry i that names it, with the top bit set when there are more, whose sum that entry takes.
    const int lo = min(max(a.bias_start[row], 0), a.n_bias), hi = min(max(a.bias_start[row + 1], lo), a.n_bias);
    const int n = hi - lo;
    const int32_t* ids = a.bias_ids + lo;
    const float* add = a.bias + lo;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += LG_THREADS) {
      const int t = ids[i];
      if (t >= v0 && t < v1) hist[t - v0] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += LG_THREADS) {
      const int t = ids[i];
      if (t >= v0 && t < v1) Count<H>::raise(hist + (t - v0), (unsigned)(n - i));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += LG_THREADS) {
      const int t = ids[i];
      if (t >= v0 && t < v1 && (hist[t - v0] & ~SEEN) != (unsigned)(n - i))
        Count<H>::mark(hist + (t - v0));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += LG_THREADS) {
      const int t = ids[i];
      if (t < v0 || t >= v1 || (hist[t - v0] & ~SEEN) != (unsigned)(n - i)) continue;
      if (mask && !((__ldg(mask + (t >> 5)) >> (t & 31)) & 1u)) continue;
      float sum = add[i];
      if (hist[t - v0] & SEEN)
        for (int j = i + 1; j < n; ++j)
          if (ids[j] == t) sum += add[j];
      out[t] += sum;
    }
  }
}

template <typename T, typename H>
int launch(const LogitsArgs& a, cudaStream_t s) {
  // CTAs per row: 8, fewer for small vocabularies, whose slices would be a few loads a thread.
  int ranks = 8;
  while (ranks > 1 && a.vocab <= ranks * 2048) ranks >>= 1;
  const int slice = ((a.vocab + ranks - 1) / ranks + 31) / 32 * 32;
  if ((size_t)slice * 4 > LG_SMEM_MAX) return kTooLarge;  // by the wider count, whichever is used
  if ((long long)a.rows * ranks > 0x7fffffffLL) return kTooLarge;
  const size_t smem = a.past || a.bias_start ? (size_t)slice * sizeof(H) : 0;
  const bool in_place = (const void*)a.out == a.x;
  const bool vec = (uintptr_t)a.x % (4 * sizeof(T)) == 0 && (uintptr_t)a.out % 16 == 0 &&
                   (a.rows == 1 || (a.x_stride % 4 == 0 && a.out_stride % 4 == 0));
  // 512 threads a CTA while all clusters are resident with two of them an SM (32 of 8 CTAs), else 256 and four an SM:
  // a vocabulary of 131,072 in bf16 takes 10.9 us so for 32 rows (13.6 with 256 threads), 17.8 for 64 rows (23.1 with
  // 512).
  const bool few = (long long)a.rows * ranks <= 256;
  auto kernel = few ? (vec ? logits_kernel<T, H, true, 512> : logits_kernel<T, H, false, 512>)
                    : (vec ? logits_kernel<T, H, true, 256> : logits_kernel<T, H, false, 256>);
  if (allow_smem(kernel, smem, LG_SMEM_MAX)) return kCudaError;
  return launch_cluster_pdl(kernel, dim3(a.rows * ranks), dim3(few ? 512 : 256), ranks, smem, s, a, slice, in_place) ==
                 cudaSuccess
             ? kOk
             : kCudaError;
}

template <typename T>
int launch(const LogitsArgs& a, cudaStream_t s) {
  return a.past_cap > 32767 || a.n_bias > 32767 ? launch<T, uint32_t>(a, s) : launch<T, uint16_t>(a, s);
}

}  // namespace

int process_logits(const LogitsArgs& a, cudaStream_t s) {
  if (a.rows < 0 || a.vocab <= 0 || a.x_type < 0 || a.x_type > 2) return kBadArgument;
  if (a.rows == 0) return kOk;
  if (a.past_cap > 1 << 30 || a.n_bias > 1 << 30) return kTooLarge;
  if (!a.x || !a.out) return kBadArgument;
  if (a.rows > 1 && (a.x_stride < a.vocab || a.out_stride < a.vocab)) return kBadArgument;
  if (a.past && (!a.past_len || a.past_cap < 0 || a.past_count <= 0)) return kBadArgument;
  if (a.bias_start && (a.n_bias < 0 || (a.n_bias > 0 && (!a.bias_ids || !a.bias)))) return kBadArgument;
  if (a.mask && (a.masks <= 0 || a.mask_stride < (a.vocab + 31) / 32)) return kBadArgument;
  if (a.mask && !a.mask_rows && a.masks < a.rows) return kBadArgument;
  // in place only where input and output are the same elements
  if ((const void*)a.out == a.x && (a.x_type != 0 || (a.rows > 1 && a.x_stride != a.out_stride))) return kBadArgument;
  switch (a.x_type) {
    case 0: return launch<float>(a, s);
    case 1: return launch<__half>(a, s);
    default: return launch<__nv_bfloat16>(a, s);
  }
}

}  // namespace zc
