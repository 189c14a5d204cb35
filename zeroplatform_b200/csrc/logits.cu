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

constexpr int LG_THREADS = 512;
constexpr int LG_SMEM_MAX = 200 * 1024;
constexpr unsigned SEEN = 0x80000000u;  // a history token; the other bits count its generated occurrences

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ void load_vec(const float* p, float* v) {
  const float4 f = *reinterpret_cast<const float4*>(p);
  v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
}
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_f(e[i]);
}

struct Rules {
  float repetition, frequency, presence;
};

__device__ __forceinline__ float apply(float v, unsigned h, const Rules& r) {
  if (h) {
    v = v > 0.f ? __fdiv_rn(v, r.repetition) : v * r.repetition;
    const unsigned c = h & ~SEEN;
    if (c) v = (v - r.frequency * (float)c) - r.presence;
  }
  return v;
}

// VEC: both row starts are 16-byte (8-byte for 16-bit input) aligned, so 4 tokens move per access.
template <typename T, bool VEC>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(LogitsArgs a, int slice, bool in_place) {
  extern __shared__ __align__(16) unsigned hist[];  // [slice]
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
  if (n_past > 0) {  // the same for every CTA of the cluster
    for (int i = threadIdx.x * 4; i < slice; i += LG_THREADS * 4)  // slice is a multiple of 32
      *reinterpret_cast<uint4*>(hist + i) = make_uint4(0, 0, 0, 0);
    cluster.sync();
    for (int i = rank * LG_THREADS + threadIdx.x; i < n_past; i += ranks * LG_THREADS) {
      const int t = past[i];
      if ((unsigned)t >= (unsigned)a.vocab) continue;
      const int owner = t / slice;
      unsigned* h = cluster.map_shared_rank(hist, owner) + (t - owner * slice);
      if (i >= n_prompt) atomicAdd(h, 1u);
      atomicOr(h, SEEN);
    }
    cluster.sync();
  }
  const uint32_t* mask = nullptr;
  if (a.mask) {
    const int m = a.mask_rows ? a.mask_rows[row] : row;
    if ((unsigned)m < (unsigned)a.masks) mask = a.mask + (size_t)m * a.mask_stride;
  }

  const bool hashed = n_past > 0;
  if (VEC) {
    const int n4 = (v1 - v0) / 4;
    for (int i = threadIdx.x; i < n4; i += LG_THREADS) {
      const int t = v0 + 4 * i;
      const unsigned bits = mask ? (__ldg(mask + (t >> 5)) >> (t & 31)) & 15u : 15u;
      uint4 h = make_uint4(0, 0, 0, 0);
      if (hashed) h = *reinterpret_cast<const uint4*>(hist + 4 * i);
      if (in_place && bits == 15u && !(h.x | h.y | h.z | h.w)) continue;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (bits) load_vec(x + t, v);
      float4 r;
      r.x = bits & 1u ? apply(v[0], h.x, rules) : -INFINITY;
      r.y = bits & 2u ? apply(v[1], h.y, rules) : -INFINITY;
      r.z = bits & 4u ? apply(v[2], h.z, rules) : -INFINITY;
      r.w = bits & 8u ? apply(v[3], h.w, rules) : -INFINITY;
      *reinterpret_cast<float4*>(out + t) = r;
    }
  }
  for (int t = v0 + (VEC ? (v1 - v0) / 4 * 4 : 0) + threadIdx.x; t < v1; t += LG_THREADS) {
    const bool ok = !mask || (__ldg(mask + (t >> 5)) >> (t & 31)) & 1u;
    const unsigned h = hashed ? hist[t - v0] : 0u;
    if (in_place && ok && !h) continue;
    out[t] = ok ? apply(to_f(x[t]), h, rules) : -INFINITY;
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
      if (t >= v0 && t < v1) atomicMax(hist + (t - v0), (unsigned)(n - i));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += LG_THREADS) {
      const int t = ids[i];
      if (t >= v0 && t < v1 && (hist[t - v0] & ~SEEN) != (unsigned)(n - i)) atomicOr(hist + (t - v0), SEEN);
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

template <typename T>
int launch(const LogitsArgs& a, cudaStream_t s) {
  // CTAs per row: 8 while the rows alone do not fill the GPU or a row's slice would not leave room for three CTAs an SM
  // (64 KB of counts), fewer for small vocabularies, whose slices would be a few loads a thread.
  int ranks = 8;
  while (ranks > 1 && a.vocab <= ranks * 2 * LG_THREADS) ranks >>= 1;
  const int slice = ((a.vocab + ranks - 1) / ranks + 31) / 32 * 32;
  if ((size_t)slice * 4 > LG_SMEM_MAX) return kTooLarge;
  if ((long long)a.rows * ranks > 0x7fffffffLL) return kTooLarge;
  const size_t smem = a.past || a.bias_start ? (size_t)slice * 4 : 0;
  const bool in_place = (const void*)a.out == a.x;
  const bool vec = (uintptr_t)a.x % (4 * sizeof(T)) == 0 && (uintptr_t)a.out % 16 == 0 &&
                   (a.rows == 1 || (a.x_stride % 4 == 0 && a.out_stride % 4 == 0));
  auto kernel = vec ? logits_kernel<T, true> : logits_kernel<T, false>;
  if (allow_smem(kernel, smem)) return kCudaError;
  return launch_cluster_pdl(kernel, dim3(a.rows * ranks), dim3(LG_THREADS), ranks, smem, s, a, slice, in_place) ==
                 cudaSuccess
             ? kOk
             : kCudaError;
}

}  // namespace

int process_logits(const LogitsArgs& a, cudaStream_t s) {
  if (a.rows < 0 || a.vocab <= 0 || a.x_type < 0 || a.x_type > 2) return kBadArgument;
  if (a.rows == 0) return kOk;
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
