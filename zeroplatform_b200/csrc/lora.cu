// lora.cu -- low-rank adapters of many requests at once beside a shared projection.
//
//   out[r] = y[r] + scale_a * (x[r] A_a^T) B_a^T      a = adapter[r];  rows without an adapter: out[r] = y[r]
//
// with y the shared projection's output (zcu_gemv / zcu_gemm of quantized weights), A_a [rank][k] and B_a [n][rank] in
// fp32, fp16 or bf16, and adapters whose own rank is below the stored one.  Both products in one launch: a cluster of
// up to 8 CTAs owns a row (or a tile of rows), splits k for the first product, sums the partial t = x A^T through
// distributed shared memory in a fixed order, and splits n for the second.  t never leaves the chip, there is no
// scratch in memory, and no atomics: the result does not depend on what shares the batch.
//
// lora_row_kernel (few rows, as in decode): fp32 arithmetic, one cluster per row.  A warp's lanes read along k, a row of
//   B is read by rank / 8 lanes, and the first rows of B are on their way before the cluster has summed t.  Bound: the
//   adapters' bytes (each row reads its own; rows that share an adapter meet in L2), at small sizes the chain
//   A -> t -> B of one launch.
// lora_tile_kernel (many rows, as in prefill): 64 rows per cluster on the tensor cores, mma m16n8k8 with x, t (and fp32
//   weights) as tf32 hi + lo pairs, which hold fp32 to 2^-22 and any range; 16-bit weights are exact in tf32.  A warp
//   takes its 16 rows one adapter at a time, usually one.  Bound: x, y and out once, or the tensor pipe at large ranks.

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <utility>

#include "batch_ops.h"
#include "common.cuh"

namespace cg = cooperative_groups;

namespace zc {

namespace {

constexpr int LR_THREADS = 256;
constexpr int LR_WARPS = LR_THREADS / 32;
constexpr int LR_CLUSTER = 8;
constexpr int LR_MAX_RANK = 128;

// Eight weights as floats; p is 16-byte aligned.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <typename W>
struct Raw;  // eight weights as they lie in memory
template <>
struct Raw<float> {
  float4 a, b;
};
template <>
struct Raw<__half> {
  uint4 a;
};
template <>
struct Raw<__nv_bfloat16> {
  uint4 a;
};
__device__ __forceinline__ void fetch(const float* p, Raw<float>& r) {
  r.a = __ldg(reinterpret_cast<const float4*>(p));
  r.b = __ldg(reinterpret_cast<const float4*>(p) + 1);
}
template <typename W>
__device__ __forceinline__ void fetch(const W* p, Raw<W>& r) {
  r.a = __ldg(reinterpret_cast<const uint4*>(p));
}
__device__ __forceinline__ void clear(Raw<float>& r) { r.a = r.b = make_float4(0.f, 0.f, 0.f, 0.f); }
template <typename W>
__device__ __forceinline__ void clear(Raw<W>& r) {
  r.a = make_uint4(0, 0, 0, 0);
}
// keeps the first n (1 to 7) weights
__device__ __forceinline__ void cut(Raw<float>& r, int n) {
  if (n < 2) r.a.y = 0.f;
  if (n < 3) r.a.z = 0.f;
  if (n < 4) r.a.w = 0.f;
  if (n < 5) r.b.x = 0.f;
  if (n < 6) r.b.y = 0.f;
  if (n < 7) r.b.z = 0.f;
  if (n < 8) r.b.w = 0.f;
}
template <typename W>
__device__ __forceinline__ void cut(Raw<W>& r, int n) {
  r.a.x &= n < 2 ? 0x0000ffffu : 0xffffffffu;
  r.a.y &= n < 3 ? 0u : n < 4 ? 0x0000ffffu : 0xffffffffu;
  r.a.z &= n < 5 ? 0u : n < 6 ? 0x0000ffffu : 0xffffffffu;
  r.a.w &= n < 7 ? 0u : n < 8 ? 0x0000ffffu : 0xffffffffu;
}
__device__ __forceinline__ float2 pair_of(const Raw<float>& r, int i) {  // weights 2i, 2i + 1
  return i == 0 ? make_float2(r.a.x, r.a.y) : i == 1 ? make_float2(r.a.z, r.a.w) : i == 2 ? make_float2(r.b.x, r.b.y)
                                                                                         : make_float2(r.b.z, r.b.w);
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}
__device__ __forceinline__ float2 pair_of(const Raw<__half>& r, int i) {
  const uint32_t w = word_of(r.a, i);
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 pair_of(const Raw<__nv_bfloat16>& r, int i) {
  const uint32_t w = word_of(r.a, i);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// The adapter of a row: -1 where it has none.
__device__ __forceinline__ int adapter_of(const LoraArgs& a, int row) {
  const int i = row < a.rows ? a.adapter[row] : -1;
  return (unsigned)i < (unsigned)a.adapters ? i : -1;
}
__device__ __forceinline__ int rank_of(const LoraArgs& a, int adapter) {
  return a.ranks ? min(max(a.ranks[adapter], 0), a.rank) : a.rank;
}

// LG: lanes that share a row of B, 8 ranks each, and rank rows of A that a warp sums; 8 LG >= rank.
template <typename W, int LG>
__global__ void __launch_bounds__(LR_THREADS) lora_row_kernel(LoraArgs a) {
  __shared__ __align__(16) float part[8 * LG], t[8 * LG];
  pdl_trigger();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int c = cluster.block_rank(), C = cluster.num_blocks();
  const int row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float* x = a.x + (size_t)row * a.x_stride;
  const float* y = a.y + (size_t)row * a.y_stride;
  float* out = a.out + (size_t)row * a.out_stride;
  const int n0 = (int)((long long)a.n * c / C), n1 = (int)((long long)a.n * (c + 1) / C);
  const int ad = adapter_of(a, row);
  const int R = ad >= 0 ? rank_of(a, ad) : 0;
  if (R == 0) {  // the same for the whole cluster
    if (out != y)
      for (int i = n0 + tid; i < n1; i += LR_THREADS) out[i] = y[i];
    return;
  }
  const W* A = reinterpret_cast<const W*>(a.a) + (size_t)ad * a.rank * a.k;
  const W* B = reinterpret_cast<const W*>(a.b) + (size_t)ad * a.n * a.rank;

  // ---- t = x A^T over this CTA's part of k, in pieces of 8 ----
  const int kv = a.k / 8, k0 = (int)((long long)kv * c / C), k1 = (int)((long long)kv * (c + 1) / C);
  float acc[LG];
#pragma unroll
  for (int i = 0; i < LG; ++i) acc[i] = 0.f;
  for (int u = k0 + lane; u < k1; u += 32) {
    constexpr int BATCH = LG < 4 ? LG : 4;  // rows of A in flight
    const float4 xa = *reinterpret_cast<const float4*>(x + 8 * u), xb = *reinterpret_cast<const float4*>(x + 8 * u + 4);
    const float2 xv[4] = {make_float2(xa.x, xa.y), make_float2(xa.z, xa.w), make_float2(xb.x, xb.y),
                          make_float2(xb.z, xb.w)};
#pragma unroll
    for (int i0 = 0; i0 < LG; i0 += BATCH) {
      Raw<W> w[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int j = (i0 + i) * LR_WARPS + warp;
        if (j < R)
          fetch(A + (size_t)j * a.k + 8 * u, w[i]);
        else
          clear(w[i]);
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        float2 s = make_float2(acc[i0 + i], 0.f);
#pragma unroll
        for (int q = 0; q < 4; ++q) s = __ffma2_rn(pair_of(w[i], q), xv[q], s);
        acc[i0 + i] = s.x + s.y;
      }
    }
  }
  // the first rows of B, before t is known
  constexpr int GROUPS = LR_THREADS / LG, AHEAD = 4;
  const int grp = tid / LG, piece = tid % LG;
  const bool mine = 8 * piece < R;
  Raw<W> ahead[AHEAD];
  float y_ahead[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int n = n0 + grp + i * GROUPS;
    if (mine && n < n1)
      fetch(B + (size_t)n * a.rank + 8 * piece, ahead[i]);
    else
      clear(ahead[i]);
    y_ahead[i] = piece == 0 && n < n1 ? y[n] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < LG; ++i) {
    const float s = warp_sum(acc[i]);
    if (lane == 0) part[i * LR_WARPS + warp] = s;
  }
  cluster.sync();
  for (int j = tid; j < 8 * LG; j += LR_THREADS) {
    float v[LR_CLUSTER];
#pragma unroll
    for (int r = 0; r < LR_CLUSTER; ++r) v[r] = r < C ? cluster.map_shared_rank(part, r)[j] : 0.f;
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < LR_CLUSTER; ++r) s += v[r];
    t[j] = j < R ? s * (a.scales ? a.scales[ad] : 1.f) : 0.f;
  }
  cluster.sync();  // t is complete, and no CTA's partial sums are read any more

  // ---- out = y + t B^T over this CTA's rows of B ----
  float2 tv[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) tv[q] = *reinterpret_cast<const float2*>(t + 8 * piece + 2 * q);
  const int valid = R - 8 * piece;  // ranks at and past R are 0 in t; what B holds there must not turn them into NaN
  auto dot = [&](Raw<W> w) {
    if (valid > 0 && valid < 8) cut(w, valid);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int q = 0; q < 4; ++q) s = __ffma2_rn(pair_of(w, q), tv[q], s);
    float v = s.x + s.y;
#pragma unroll
    for (int o = LG / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int n = n0 + grp + i * GROUPS;
    const float v = dot(ahead[i]);
    if (piece == 0 && n < n1) out[n] = y_ahead[i] + v;
  }
  for (int nb = n0 + AHEAD * GROUPS; nb < n1; nb += AHEAD * GROUPS) {
    Raw<W> w[AHEAD];
    float yv[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int n = nb + grp + i * GROUPS;
      if (mine && n < n1)
        fetch(B + (size_t)n * a.rank + 8 * piece, w[i]);
      else
        clear(w[i]);
      yv[i] = piece == 0 && n < n1 ? y[n] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int n = nb + grp + i * GROUPS;
      const float v = dot(w[i]);
      if (piece == 0 && n < n1) out[n] = yv[i] + v;
    }
  }
}

// ---- tiles of 64 rows ----

constexpr int LT_ROWS = 64;

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tf32_of(float v) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return r;
}

// The A operand of a 16-row, 32-deep step: lane (g, c) gives elements 8 c .. 8 c + 7 of rows g and g + 8; k-step s takes
// elements 2 s and 2 s + 1 of each lane.  The B operand's lane (g, c) gives the same elements of column g.
struct Step {
  uint32_t hi[4][4], lo[4][4];
};
__device__ __forceinline__ void split_step(const float (&r0)[8], const float (&r1)[8], Step& s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v[4] = {r0[2 * i], r1[2 * i], r0[2 * i + 1], r1[2 * i + 1]};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s.hi[i][q] = tf32_of(v[q]);
      s.lo[i][q] = tf32_of(v[q] - __uint_as_float(s.hi[i][q]));
    }
  }
}
template <typename W>
__device__ __forceinline__ void step_mma(float (&d)[4], const Step& s, const Raw<W>& w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = pair_of(w, i);
    if constexpr (sizeof(W) == 4) {
      const uint32_t h0 = tf32_of(p.x), h1 = tf32_of(p.y);
      mma_tf32(d, s.hi[i], tf32_of(p.x - __uint_as_float(h0)), tf32_of(p.y - __uint_as_float(h1)));
      mma_tf32(d, s.lo[i], h0, h1);
      mma_tf32(d, s.hi[i], h0, h1);
    } else {
      mma_tf32(d, s.lo[i], __float_as_uint(p.x), __float_as_uint(p.y));
      mma_tf32(d, s.hi[i], __float_as_uint(p.x), __float_as_uint(p.y));
    }
  }
}

// NT: column tiles of 8 ranks, 8 NT >= rank.
template <typename W, int NT>
__global__ void __launch_bounds__(LR_THREADS) lora_tile_kernel(LoraArgs a) {
  constexpr int TS = 8 * NT + 4;  // floats of a row of t
  constexpr int STEPS = (8 * NT + 31) / 32;
  extern __shared__ __align__(16) float sm[];
  float* part = sm;                        // [2][LT_ROWS][TS]: the two k halves' sums, then [0] all of this CTA's
  float* t = sm + 2 * LT_ROWS * TS;        // [LT_ROWS][TS]
  pdl_trigger();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int cr = cluster.block_rank(), C = cluster.num_blocks();
  const int row0 = (int)(blockIdx.x / C) * LT_ROWS, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int mt = warp & 3, half = warp >> 2;  // 16 rows, and a half of k or n
  const int ra = row0 + mt * 16 + g, rb = ra + 8;
  const int ida = adapter_of(a, ra), idb = adapter_of(a, rb);
  for (int i = tid; i < 2 * LT_ROWS * TS; i += LR_THREADS) part[i] = 0.f;
  __syncthreads();

  // ---- t = x A^T ----
  {
    const int steps = a.k / 32, u0 = (int)((long long)steps * (2 * cr + half) / (2 * C)),
              u1 = (int)((long long)steps * (2 * cr + half + 1) / (2 * C));
    unsigned todo_a = ida >= 0, todo_b = idb >= 0;
    for (;;) {  // one adapter of the 16 rows at a time
      const unsigned ad = __reduce_min_sync(0xffffffffu, min(todo_a ? (unsigned)ida : 0xffffffffu,
                                                             todo_b ? (unsigned)idb : 0xffffffffu));
      if (ad == 0xffffffffu) break;
      const bool ma = todo_a && ida == (int)ad, mb = todo_b && idb == (int)ad;
      if (ma) todo_a = 0;
      if (mb) todo_b = 0;
      const int R = rank_of(a, (int)ad), tiles = (R + 7) / 8;
      const W* A = reinterpret_cast<const W*>(a.a) + (size_t)ad * a.rank * a.k + 8 * c;
      const float* xa = a.x + (size_t)ra * a.x_stride + 8 * c;
      const float* xb = a.x + (size_t)rb * a.x_stride + 8 * c;
      float acc[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
      for (int u = u0; u < u1; ++u) {
        float va[8] = {}, vb[8] = {};
        if (ma) load8(xa + 32 * u, va);
        if (mb) load8(xb + 32 * u, vb);
        Raw<W> w[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          if (8 * i + g < R)
            fetch(A + (size_t)(8 * i + g) * a.k + 32 * u, w[i]);
          else
            clear(w[i]);
        }
        Step s;
        split_step(va, vb, s);
#pragma unroll
        for (int i = 0; i < NT; ++i)
          if (i < tiles) step_mma<W>(acc[i], s, w[i]);
      }
      float* pa = part + (half * LT_ROWS + mt * 16 + g) * TS;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (ma) *reinterpret_cast<float2*>(pa + 8 * i + 2 * c) = make_float2(acc[i][0], acc[i][1]);
        if (mb) *reinterpret_cast<float2*>(pa + 8 * TS + 8 * i + 2 * c) = make_float2(acc[i][2], acc[i][3]);
      }
    }
  }
  cluster.sync();
  // ---- every CTA sums a part of t over the cluster and gives it to the others ----
  for (int i = cr * LR_THREADS + tid; i < LT_ROWS * 2 * NT; i += C * LR_THREADS) {  // 4 ranks of a row
    const int r = i / (2 * NT), j = i % (2 * NT) * 4;
    float4 v[LR_CLUSTER][2];
#pragma unroll
    for (int q = 0; q < LR_CLUSTER; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        v[q][h] = q < C ? *reinterpret_cast<const float4*>(cluster.map_shared_rank(part, q) + (h * LT_ROWS + r) * TS + j)
                        : make_float4(0.f, 0.f, 0.f, 0.f);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int q = 0; q < LR_CLUSTER; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) s.x += v[q][h].x, s.y += v[q][h].y, s.z += v[q][h].z, s.w += v[q][h].w;
    const int ad = adapter_of(a, row0 + r);
    if (ad >= 0) {
      const int R = rank_of(a, ad);
      const float f = a.scales ? a.scales[ad] : 1.f;
      s.x = j < R ? s.x * f : 0.f, s.y = j + 1 < R ? s.y * f : 0.f;
      s.z = j + 2 < R ? s.z * f : 0.f, s.w = j + 3 < R ? s.w * f : 0.f;
    }
    for (int q = 0; q < C; ++q) *reinterpret_cast<float4*>(cluster.map_shared_rank(t, q) + r * TS + j) = s;
  }
  cluster.sync();

  // ---- out = y + t B^T ----
  const int tiles = (a.n + 7) / 8, t0 = (int)((long long)tiles * (2 * cr + half) / (2 * C)),
            t1 = (int)((long long)tiles * (2 * cr + half + 1) / (2 * C));
  const float* ya = a.y + (size_t)ra * a.y_stride;
  const float* yb = a.y + (size_t)rb * a.y_stride;
  float* oa = a.out + (size_t)ra * a.out_stride;
  float* ob = a.out + (size_t)rb * a.out_stride;
  auto add = [&](const float* y, float* o, int n, float d0, float d1) {
    if (n < a.n) o[n] = y[n] + d0;
    if (n + 1 < a.n) o[n + 1] = y[n + 1] + d1;
  };
  // both row starts on 8 bytes: two columns an access
  const bool wide = ((uintptr_t)a.y | (uintptr_t)a.out) % 8 == 0 && a.y_stride % 2 == 0 && a.out_stride % 2 == 0;
  unsigned todo_a = ida >= 0, todo_b = idb >= 0;
  for (;;) {
    const unsigned ad = __reduce_min_sync(0xffffffffu, min(todo_a ? (unsigned)ida : 0xffffffffu,
                                                           todo_b ? (unsigned)idb : 0xffffffffu));
    if (ad == 0xffffffffu) break;
    const bool ma = todo_a && ida == (int)ad, mb = todo_b && idb == (int)ad;
    if (ma) todo_a = 0;
    if (mb) todo_b = 0;
    const int R = rank_of(a, (int)ad);
    const W* B = reinterpret_cast<const W*>(a.b) + (size_t)ad * a.n * a.rank + 8 * c;
    Step s[STEPS];
#pragma unroll
    for (int q = 0; q < STEPS; ++q) {
      float va[8] = {}, vb[8] = {};
      const float* p = t + (mt * 16 + g) * TS + 32 * q + 8 * c;
      if (32 * q + 8 * c < 8 * NT) {
        if (ma)
          for (int i = 0; i < 8; ++i) va[i] = p[i];
        if (mb)
          for (int i = 0; i < 8; ++i) vb[i] = p[8 * TS + i];
      }
      split_step(va, vb, s[q]);
    }
    constexpr int COLS = 4;  // column tiles in flight
    for (int i0 = t0; i0 < t1; i0 += COLS) {
      Raw<W> w[COLS][STEPS];
      float2 y0[COLS], y1[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) {
        const int n = 8 * (i0 + i) + g, col = 8 * (i0 + i) + 2 * c;
        const bool in = i0 + i < t1;
#pragma unroll
        for (int q = 0; q < STEPS; ++q) {
          if (in && n < a.n && 32 * q + 8 * c < R)
            fetch(B + (size_t)n * a.rank + 32 * q, w[i][q]);
          else
            clear(w[i][q]);
          // ranks at and past R are 0 in t; what B holds there must not turn them into NaN
          if (32 * q + 8 * c < R && 32 * q + 8 * c + 8 > R) cut(w[i][q], R - 32 * q - 8 * c);
        }
        if (wide && in && col + 1 < a.n) {
          if (ma) y0[i] = *reinterpret_cast<const float2*>(ya + col);
          if (mb) y1[i] = *reinterpret_cast<const float2*>(yb + col);
        }
      }
#pragma unroll
      for (int i = 0; i < COLS; ++i) {
        if (i0 + i >= t1) break;
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < STEPS; ++q)
          if (32 * q < R) step_mma<W>(d, s[q], w[i][q]);
        const int col = 8 * (i0 + i) + 2 * c;
        if (wide && col + 1 < a.n) {
          if (ma) *reinterpret_cast<float2*>(oa + col) = make_float2(y0[i].x + d[0], y0[i].y + d[1]);
          if (mb) *reinterpret_cast<float2*>(ob + col) = make_float2(y1[i].x + d[2], y1[i].y + d[3]);
        } else {
          if (ma) add(ya, oa, col, d[0], d[1]);
          if (mb) add(yb, ob, col, d[2], d[3]);
        }
      }
    }
  }
  if (a.out != a.y)  // rows without an adapter
    for (int r = mt * 16; r < mt * 16 + 16 && row0 + r < a.rows; ++r) {
      if (adapter_of(a, row0 + r) >= 0) continue;
      const float* y = a.y + (size_t)(row0 + r) * a.y_stride;
      float* o = a.out + (size_t)(row0 + r) * a.out_stride;
      for (int n = 8 * t0 + lane; n < min(8 * t1, a.n); n += 32) o[n] = y[n];
    }
}

template <typename W, int LG>
int launch_row(const LoraArgs& a, cudaStream_t s) {
  // 8 CTAs a row while their parts of k and n are worth a cluster's two barriers (at least a warp's lanes along k)
  int C = LR_CLUSTER;
  while (C > 1 && a.k < 256 * C && a.n < 256 * C) C >>= 1;
  if ((long long)a.rows * C > 0x7fffffffLL) return kTooLarge;
  return launch_cluster_pdl(lora_row_kernel<W, LG>, dim3(a.rows * C), dim3(LR_THREADS), C, 0, s, a) == cudaSuccess
             ? kOk
             : kCudaError;
}

template <typename W, int NT>
int launch_tile(const LoraArgs& a, cudaStream_t s) {
  const int tiles = (a.rows + LT_ROWS - 1) / LT_ROWS;
  const size_t smem = (size_t)3 * LT_ROWS * (8 * NT + 4) * 4;
  auto kernel = lora_tile_kernel<W, NT>;
  if (allow_smem(kernel, smem)) return kCudaError;
  if ((long long)tiles * LR_CLUSTER > 0x7fffffffLL) return kTooLarge;
  return launch_cluster_pdl(kernel, dim3(tiles * LR_CLUSTER), dim3(LR_THREADS), LR_CLUSTER, smem, s, a) == cudaSuccess
             ? kOk
             : kCudaError;
}

template <typename W, int LG>
int launch(const LoraArgs& a, cudaStream_t s) {
  return a.rows <= 256 ? launch_row<W, LG>(a, s) : launch_tile<W, LG>(a, s);
}

template <typename W>
int launch_rank(const LoraArgs& a, cudaStream_t s) {
  if (a.rank <= 8) return launch<W, 1>(a, s);
  if (a.rank <= 16) return launch<W, 2>(a, s);
  if (a.rank <= 32) return launch<W, 4>(a, s);
  if (a.rank <= 64) return launch<W, 8>(a, s);
  return launch<W, 16>(a, s);
}

}  // namespace

int lora_add(const LoraArgs& a, cudaStream_t s) {
  if (a.rows < 0 || a.k <= 0 || a.n <= 0 || a.adapters <= 0 || a.rank <= 0 || a.w_type < 0 || a.w_type > 2)
    return kBadArgument;
  if (a.rows == 0) return kOk;
  if (!a.x || !a.y || !a.out || !a.a || !a.b || !a.adapter) return kBadArgument;
  if (a.rows > 1 && (a.x_stride < a.k || a.y_stride < a.n || a.out_stride < a.n)) return kBadArgument;
  if ((const void*)a.out == (const void*)a.y && a.rows > 1 && a.y_stride != a.out_stride) return kBadArgument;
  if (a.rank % 8 || a.rank > LR_MAX_RANK || a.k % 32) return kUnsupported;
  if (((uintptr_t)a.x | (uintptr_t)a.a | (uintptr_t)a.b) % 16 || (a.rows > 1 && a.x_stride % 4)) return kBadArgument;
  switch (a.w_type) {
    case 0: return launch_rank<float>(a, s);
    case 1: return launch_rank<__half>(a, s);
    default: return launch_rank<__nv_bfloat16>(a, s);
  }
}

}  // namespace zc
