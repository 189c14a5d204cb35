// lora.cu -- low-rank adapters of many requests at once beside a shared projection.
//
//   out[r] = y[r] + scale_a * (x[r] A_a^T) B_a^T      a = adapter[r];  rows without an adapter: out[r] = y[r]
//
// with y the shared projection's output (zcu_gemv / zcu_gemm of quantized weights), A_a [rank][k] and B_a [n][rank] in
// fp32, fp16 or bf16, and adapters whose own rank is below the stored one.  Both products in one launch: a cluster of
// up to 8 CTAs owns a row (or a tile of rows), splits k for the first product, sums the partial t = x A^T through
// distributed shared memory in a fixed order, and splits n for the second.  t never leaves the chip, there is no
// scratch in memory and no atomics on results: the same call gives the same bits.
//
// lora_row_kernel (few rows, as in decode): fp32 arithmetic, one cluster per row.  A warp's lanes read along k, a row
//   of B is read by rank / 8 lanes, and the first rows of B are on their way before the cluster has summed t.  Bound:
//   the adapters' bytes from L2 (each row reads its own; rows that share an adapter meet there), at small sizes the
//   chain A -> t -> B of one launch.  k = n = 4096: one row of rank 16 4.1 us; 64 rows of rank 64 12.6 us, 64 MB from
//   L2 at 5.3 TB/s.
// lora_tile_kernel (many rows, as in prefill): 64 rows per cluster, sorted by adapter, on the tensor cores (mma.sync), x
//   and t split into terms of the weights' type that hold fp32 to 2^-22 (Step); the accumulator truncates, so 32 columns
//   are summed there and the sums added with rounding (k 16,384: 2e-7 off instead of 2.4e-6, 1 us of 44).  x and A, then
//   y and B, pass through one cp.async ring, whose second filling starts before the cluster has summed t.  The adapter
//   that most of a tile's rows name is staged; warps whose rows name others fetch those weights themselves, the first
//   one's a turn ahead.  2048 rows of rank 64, k = n = 4096, all but 250 with the same adapter: fp16 44 us (2.3 TB/s of
//   x, y and out), bf16 57, fp32 109; bound by the instructions and barriers of a turn (about 300 per warp and 64
//   columns, 14 warps an SM), not by HBM (16 us) or the tensor pipe (9 us).

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
constexpr int LR_AHEAD = 4;  // rows of B that a lane group has in flight
constexpr int LR_MAX_RANK = 128;

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
__global__ void __launch_bounds__(LR_THREADS) lora_row_kernel(LoraArgs a, int parts) {
  __shared__ __align__(16) float part[8 * LG], t[8 * LG];
  pdl_trigger();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int c = cluster.block_rank(), C = cluster.num_blocks();
  const int row = blockIdx.x / (C * parts), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nc = blockIdx.x % (C * parts), ncs = C * parts;  // this CTA's part of n; k is split over the cluster
  const float* x = a.x + (size_t)row * a.x_stride;
  const float* y = a.y + (size_t)row * a.y_stride;
  float* out = a.out + (size_t)row * a.out_stride;
  const int n0 = (int)((long long)a.n * nc / ncs), n1 = (int)((long long)a.n * (nc + 1) / ncs);
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
  constexpr int GROUPS = LR_THREADS / LG, AHEAD = LR_AHEAD;
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

constexpr int LT_ROWS = 64, LT_K = 64, LT_STAGES = 3;
constexpr int LT_XROW = LT_K * 4 + 16;  // bytes of a staged row of x: 16 more put an access's two rows on other banks

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tf32_of(float v) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return r;
}
// 16 bytes from memory into shared memory, zeros where !ok (nothing is read then)
__device__ __forceinline__ void copy16(void* dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
               "r"(ok ? 16 : 0)
               : "memory");
}

// A 16-row, 32-deep step of a product with fp32 rows.  Lane (g, c) holds elements 8 c .. 8 c + 7 of rows g and g + 8 and
// the same elements of weight row (column) g: the contraction index is permuted alike on both sides.  The rows are
// split into terms of the weights' type that hold them to at least 2^-22:
//   fp16   hi + lo, with a power of two of the row's own that keeps it in range;  2 terms, k-steps of 16
//   bf16   three terms, in fp32's range;                                          3 terms, k-steps of 16
//   fp32   tf32 hi + lo of both sides, lo x lo left out;                          3 products, k-steps of 8
// (a k-step of either kind takes the tensor cores the same time: 540 TFLOP/s at k 16, 270 at k 8).
template <typename W>
struct Step;
template <>
struct Step<__half> {
  static constexpr bool SCALED = true;
  uint32_t hi[2][4], lo[2][4];
  __device__ __forceinline__ void split(const float (&r0)[8], const float (&r1)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // row g or g + 8, elements 4 i + (0, 1) or (2, 3)
        const float(&r)[8] = q & 1 ? r1 : r0;
        const float u = r[4 * i + (q >> 1) * 2], v = r[4 * i + (q >> 1) * 2 + 1];
        const __half2 h = __floats2half2_rn(u, v);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(u - f.x, v - f.y);
        hi[i][q] = *reinterpret_cast<const uint32_t*>(&h);
        lo[i][q] = *reinterpret_cast<const uint32_t*>(&l);
      }
  }
  __device__ __forceinline__ void mma(float (&d)[4], const Raw<__half>& w) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) mma_f16(d, lo[i], word_of(w.a, 2 * i), word_of(w.a, 2 * i + 1));
#pragma unroll
    for (int i = 0; i < 2; ++i) mma_f16(d, hi[i], word_of(w.a, 2 * i), word_of(w.a, 2 * i + 1));
  }
};
template <>
struct Step<__nv_bfloat16> {
  static constexpr bool SCALED = false;
  uint32_t t[3][2][4];
  __device__ __forceinline__ void split(const float (&r0)[8], const float (&r1)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float(&r)[8] = q & 1 ? r1 : r0;
        float u = r[4 * i + (q >> 1) * 2], v = r[4 * i + (q >> 1) * 2 + 1];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(u, v);
          t[k][i][q] = *reinterpret_cast<const uint32_t*>(&h);
          u -= __uint_as_float(t[k][i][q] << 16);
          v -= __uint_as_float(t[k][i][q] & 0xffff0000u);
        }
      }
  }
  __device__ __forceinline__ void mma(float (&d)[4], const Raw<__nv_bfloat16>& w) const {
#pragma unroll
    for (int k = 2; k >= 0; --k)
#pragma unroll
      for (int i = 0; i < 2; ++i) mma_bf16(d, t[k][i], word_of(w.a, 2 * i), word_of(w.a, 2 * i + 1));
  }
};
template <>
struct Step<float> {
  static constexpr bool SCALED = false;
  uint32_t hi[4][4], lo[4][4];
  __device__ __forceinline__ void split(const float (&r0)[8], const float (&r1)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v[4] = {r0[2 * i], r1[2 * i], r0[2 * i + 1], r1[2 * i + 1]};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        hi[i][q] = tf32_of(v[q]);
        lo[i][q] = tf32_of(v[q] - __uint_as_float(hi[i][q]));
      }
    }
  }
  __device__ __forceinline__ void mma(float (&d)[4], const Raw<float>& w) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = pair_of(w, i);
      const uint32_t h0 = tf32_of(p.x), h1 = tf32_of(p.y);
      mma_tf32(d, hi[i], tf32_of(p.x - __uint_as_float(h0)), tf32_of(p.y - __uint_as_float(h1)));
      mma_tf32(d, lo[i], h0, h1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = pair_of(w, i);
      mma_tf32(d, hi[i], tf32_of(p.x), tf32_of(p.y));
    }
  }
};

__device__ __forceinline__ float top8(const float (&v)[8]) {
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) t = fmaxf(t, fabsf(v[i]));
  return t;
}
__device__ __forceinline__ float top_quad(float t) {
  t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
  return fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
}
// The power of two that brings `top` to 2^6 .. 2^7 (fp16 holds up to 2^16 and 2^-24): 1 for 0 and what is not finite.
__device__ __forceinline__ float scale_for(float top) {
  if (!(top > 0.f && top < INFINITY)) return 1.f;
  const int e = (int)((__float_as_uint(top) >> 23) & 255u) - 127;
  return __uint_as_float((uint32_t)(127 + min(max(6 - e, -126), 126)) << 23);
}
__device__ __forceinline__ void times(float (&v)[8], float f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= f;
}
__device__ __forceinline__ void load_row8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load_raw(const unsigned char* p, Raw<float>& r) {
  r.a = *reinterpret_cast<const float4*>(p);
  r.b = *reinterpret_cast<const float4*>(p + 16);
}
template <typename W>
__device__ __forceinline__ void load_raw(const unsigned char* p, Raw<W>& r) {
  r.a = *reinterpret_cast<const uint4*>(p);
}

// 4 bytes likewise, for rows that do not start on 16
__device__ __forceinline__ void copy4(void* dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
               "r"(ok ? 4 : 0)
               : "memory");
}

// Shared memory of a tile: a ring of stages, then this CTA's part of t.  A stage is 64 columns of x and of A, or of y and
// of B's rows.  NT: column tiles of 8 ranks, 8 NT >= rank.  Rows are padded so that operand reads (row g, piece c)
// spread over all banks.
template <typename W, int NT>
struct Tile {
  static constexpr int TS = 8 * NT + 4;                                                // floats of a row of t
  static constexpr int AROW = LT_K * (int)sizeof(W) + (sizeof(W) == 4 ? 16 : 64);      // bytes of a staged row of A
  static constexpr int BROW = 8 * NT * (int)sizeof(W) + (sizeof(W) == 4 ? 16 : NT >= 8 ? 64 : 0);  // and of B
  static constexpr int WBYTES = 8 * NT * AROW > LT_K * BROW ? 8 * NT * AROW : LT_K * BROW;
  static constexpr int STAGE = LT_ROWS * LT_XROW + WBYTES;
  static constexpr int BYTES = LT_STAGES * STAGE + LT_ROWS * TS * 4;
  static_assert(LT_ROWS * TS * 4 <= STAGE, "t takes the last stage's place");
};

// The rows of a tile: LT_CHUNK rows at a time are put in the order of their adapters (those that share a bucket stay in
// the batch's order, rows without an adapter come last), so that a tile's rows name few of them whatever the batch's
// order is: 2048 rows, k = n = 4096, six of seven with one of 12 adapters of rank 64, take 56 us, in their own order 234.  A
// stable counting sort that every CTA repeats for itself, about 1 us; a bucket may hold several adapters, which only
// mixes them.  row[i] is the tile's i-th row, -1 behind the last one.  work: 8 x 256 counts.
constexpr int LT_CHUNK = 1024;
__device__ __forceinline__ void rows_of_tile(const LoraArgs& a, int tile, unsigned short* work, int (&row)[LT_ROWS]) {
  static_assert(LR_THREADS == 256 && LT_CHUNK % (LR_WARPS * 32) == 0 && LT_CHUNK % LT_ROWS == 0, "");
  constexpr int EACH = LT_CHUNK / LR_THREADS;
  __shared__ int sums[LR_WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int chunk0 = tile / (LT_CHUNK / LT_ROWS) * LT_CHUNK, first = tile * LT_ROWS - chunk0;
  int key[EACH], at[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {  // a warp's rows in order: 32 j + lane
    const int k = warp * (LT_CHUNK / LR_WARPS) + 32 * j + lane;
    const int ad = k < a.rows - chunk0 ? adapter_of(a, chunk0 + k) : -2;
    key[j] = ad >= 0 ? ad % 255 : ad == -1 ? 255 : -1;
  }
  unsigned short* mine = work + warp * 256;
#pragma unroll
  for (int i = 0; i < 8; ++i) mine[lane + 32 * i] = 0;
  if (tid < LT_ROWS) row[tid] = -1;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const unsigned same = __match_any_sync(0xffffffffu, key[j]);
    const int before = key[j] >= 0 ? mine[key[j]] : 0;
    at[j] = before + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (key[j] >= 0 && (same >> lane) == 1u) mine[key[j]] = (unsigned short)(at[j] + 1);  // the last of them
    __syncwarp();
  }
  __syncthreads();
  int total = 0;  // of bucket tid; the warps' counts become what comes before them
#pragma unroll
  for (int w = 0; w < LR_WARPS; ++w) {
    const int n = work[w * 256 + tid];
    work[w * 256 + tid] = (unsigned short)total;
    total += n;
  }
  int upto = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  int start = upto - total;
#pragma unroll
  for (int w = 0; w < LR_WARPS; ++w) start += w < warp ? sums[w] : 0;
#pragma unroll
  for (int w = 0; w < LR_WARPS; ++w) work[w * 256 + tid] += (unsigned short)start;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int p = key[j] >= 0 ? mine[key[j]] + at[j] - first : -1;
    if (p >= 0 && p < LT_ROWS) row[p] = chunk0 + warp * (LT_CHUNK / LR_WARPS) + 32 * j + lane;
  }
  __syncthreads();
}

template <typename W, int NT>
__global__ void __launch_bounds__(LR_THREADS, sizeof(W) == 2 && NT <= 8 ? 2 : 1) lora_tile_kernel(LoraArgs a) {
  using T = Tile<W, NT>;
  constexpr int TS = T::TS, STEPS = (8 * NT + 31) / 32, EPP = 16 / (int)sizeof(W);  // weights of a 16-byte piece
  extern __shared__ __align__(16) unsigned char smem[];
  float* t = reinterpret_cast<float*>(smem + (LT_STAGES - 1) * T::STAGE);  // [LT_ROWS][TS]
  float* part = reinterpret_cast<float*>(smem + LT_STAGES * T::STAGE);     // [LT_ROWS][TS]: this CTA's part of k
  __shared__ int ids[LT_ROWS], rows[LT_ROWS];
  __shared__ int s_main;
  pdl_trigger();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int cr = cluster.block_rank(), C = cluster.num_blocks();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int mt = warp & 3, half = warp >> 2;  // 16 rows, and a half of every 64 k or of the columns
  rows_of_tile(a, (int)(blockIdx.x / C), reinterpret_cast<unsigned short*>(smem), rows);
  if (tid < LT_ROWS) ids[tid] = rows[tid] >= 0 ? adapter_of(a, rows[tid]) : -1;
  if (tid == 0) s_main = 0;
  __syncthreads();
  if (tid < LT_ROWS && ids[tid] >= 0) {  // the adapter that most rows name, the lowest row among equals
    int same = 0;
#pragma unroll 8
    for (int i = 0; i < LT_ROWS; ++i) same += ids[i] == ids[tid];
    atomicMax(&s_main, same * LT_ROWS + (LT_ROWS - 1 - tid));
  }
  __syncthreads();
  // Its weights are staged with the rows; a warp whose rows name others fetches those weights itself.
  const int main_ad = s_main ? ids[LT_ROWS - 1 - s_main % LT_ROWS] : -1;
  const int main_rank = main_ad >= 0 ? rank_of(a, main_ad) : 0;
  const int la = mt * 16 + g, lb = la + 8, ra = rows[la], rb = rows[lb];
  const int ida = ids[la], idb = ids[lb];
  const unsigned low_id = __reduce_min_sync(0xffffffffu, min((unsigned)ida, (unsigned)idb));  // -1 is the highest
  const int high_id = __reduce_max_sync(0xffffffffu, max(ida, idb));
  const bool none = high_id < 0;                                  // no row of this warp has an adapter
  const bool only_main = low_id == (unsigned)main_ad && high_id == main_ad;  // all of them the staged one
  const bool has_main = __any_sync(0xffffffffu, main_ad >= 0 && (ida == main_ad || idb == main_ad));
  // The warp's other adapters in ascending order; -1 where there is none.  The first one's weights are fetched ahead.
  auto other_after = [&](int prev) {
    const unsigned na = ida > prev && ida != main_ad ? (unsigned)ida : 0xffffffffu;
    const unsigned nb = idb > prev && idb != main_ad ? (unsigned)idb : 0xffffffffu;
    return (int)__reduce_min_sync(0xffffffffu, min(na, nb));
  };
  const int other = other_after(-1);
  const int other_rank = other >= 0 ? rank_of(a, other) : 0;

  // ---- t = x A^T: the cluster's CTAs take 64 columns in turn, so that they read a row's neighbouring pieces together ----
  const int chunks = (a.k + LT_K - 1) / LT_K, turns = (chunks - cr + C - 1) / C;
  // This thread's pieces of a stage: of x (and y) rows r16, r16 + 16, .., piece p16; of A rows wr, wr + WSTEP, .., piece
  // wp.  Sources advance by a turn's columns.
  constexpr int XROWS = LR_THREADS / 16, XN = LT_ROWS / XROWS;
  constexpr int APR = LT_K / EPP, WSTEP = LR_THREADS / APR, AN = (8 * NT + WSTEP - 1) / WSTEP;
  const int r16 = tid / 16, p16 = tid % 16, wr = tid / APR, wp = tid % APR;
  unsigned have = 0;  // bit i: row r16 + 16 i has an adapter
#pragma unroll
  for (int i = 0; i < XN; ++i) have |= (ids[r16 + XROWS * i] >= 0 ? 1u : 0u) << i;
  auto row_at = [&](int i) { return (size_t)max(rows[r16 + XROWS * i], 0); };
  const float* x_src = a.x + cr * LT_K + p16 * 4;
  const W* a_src = reinterpret_cast<const W*>(a.a) + ((size_t)max(main_ad, 0) * a.rank + wr) * a.k + cr * LT_K + wp * EPP;
  unsigned char* const x_dst = smem + r16 * LT_XROW + p16 * 16;
  unsigned char* const a_dst = smem + LT_ROWS * LT_XROW + wr * T::AROW + wp * 16;
  int k_left = a.k - cr * LT_K, fill = 0;  // columns from this turn's first; stage that is filled next
  auto issue = [&]() {
    if (k_left > 0) {
      const bool in_x = p16 * 4 < k_left, in_a = wp * EPP < k_left;
#pragma unroll
      for (int i = 0; i < XN; ++i)
        copy16(x_dst + fill * T::STAGE + i * XROWS * LT_XROW, x_src + row_at(i) * a.x_stride,
               in_x && (have >> i & 1u));
#pragma unroll
      for (int i = 0; i < AN; ++i)
        if ((8 * NT) % WSTEP == 0 || wr + i * WSTEP < 8 * NT)
          copy16(a_dst + fill * T::STAGE + i * WSTEP * T::AROW, a_src + (size_t)i * WSTEP * a.k,
                 in_a && wr + i * WSTEP < main_rank);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    x_src += C * LT_K;
    a_src += C * LT_K;
    k_left -= C * LT_K;
    fill = fill == LT_STAGES - 1 ? 0 : fill + 1;
  };
  {
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    // Powers of two of the two rows: no element times them passes 2^15.  They start so high that the first element
    // which is not 0 (or below 2^-85) chooses them.
    constexpr float UNSET = 1.2676506e30f;  // 2^100
    float sa = UNSET, sb = UNSET;
    issue();
    issue();
    int use = 0;  // stage that is read next
    auto fetch_a = [&](int ad, int R, int q, Raw<W>(&w)[NT]) {
      const int k = (q * C + cr) * LT_K + half * 32 + 8 * c;
      const W* A = reinterpret_cast<const W*>(a.a) + ((size_t)ad * a.rank + g) * a.k + k;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (8 * i + g < R && k < a.k)
          fetch(A + (size_t)8 * i * a.k, w[i]);
        else
          clear(w[i]);
      }
    };
    for (int q = 0; q < turns; ++q) {
      Raw<W> w[NT];
      if (other >= 0) fetch_a(other, other_rank, q, w);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
      issue();
      const unsigned char* st = smem + use * T::STAGE;
      use = use == LT_STAGES - 1 ? 0 : use + 1;
      if (none) continue;
      float va[8], vb[8];
      load_row8(reinterpret_cast<const float*>(st + la * LT_XROW) + half * 32 + 8 * c, va);
      load_row8(reinterpret_cast<const float*>(st + lb * LT_XROW) + half * 32 + 8 * c, vb);
      if constexpr (Step<W>::SCALED) {
        // A row's power of two comes from its first 32 elements, with room for 2^8 times as much; where more comes, the
        // sums so far follow.
        float ta = top8(va), tb = top8(vb);
        if (__any_sync(0xffffffffu, fmaxf(ta * sa, tb * sb) > 32768.f)) {
          ta = top_quad(ta);
          tb = top_quad(tb);
          auto follow = [&](float& s, float top, int k) {
            if (top * s > 32768.f && top < INFINITY) {
              const float n = scale_for(top), f = n / s;
#pragma unroll
              for (int i = 0; i < NT; ++i) acc[i][k] *= f, acc[i][k + 1] *= f;
              s = n;
            }
          };
          follow(sa, ta, 0);
          follow(sb, tb, 2);
        }
        times(va, sa);
        times(vb, sb);
      }
      Step<W> s;
      s.split(va, vb);
      const unsigned char* wt = st + LT_ROWS * LT_XROW + g * T::AROW + (half * 32 + 8 * c) * (int)sizeof(W);
      if (only_main) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
          if (8 * i < main_rank) {
            Raw<W> m;
            load_raw(wt + i * 8 * T::AROW, m);
            float d[4] = {0.f, 0.f, 0.f, 0.f};  // the tensor core's accumulator truncates: 32 columns a sum
            s.mma(d, m);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[i][k] += d[k];
          }
      } else {
        // Sums of their own: what an adapter holds reaches its own rows only.
        auto put = [&](int i, const Raw<W>& m, int ad) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          s.mma(d, m);
          if (ida == ad) acc[i][0] += d[0], acc[i][1] += d[1];
          if (idb == ad) acc[i][2] += d[2], acc[i][3] += d[3];
        };
        int R = other_rank;
        for (int ad = other; ad >= 0;) {
#pragma unroll
          for (int i = 0; i < NT; ++i)
            if (8 * i < R) put(i, w[i], ad);
          ad = other_after(ad);
          if (ad >= 0) fetch_a(ad, R = rank_of(a, ad), q, w);
        }
        if (has_main)
#pragma unroll
          for (int i = 0; i < NT; ++i)
            if (8 * i < main_rank) {
              Raw<W> m;
              load_raw(wt + i * 8 * T::AROW, m);
              put(i, m, main_ad);
            }
      }
    }
    // the two halves of each 64, in turn
    const float ia = Step<W>::SCALED ? 1.f / sa : 1.f, ib = Step<W>::SCALED ? 1.f / sb : 1.f;
#pragma unroll
    for (int h = 1; h >= 0; --h) {
      if (half == h) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float2* pa = reinterpret_cast<float2*>(part + la * TS + 8 * i + 2 * c);
          float2* pb = reinterpret_cast<float2*>(part + lb * TS + 8 * i + 2 * c);
          float2 u = make_float2(acc[i][0] * ia, acc[i][1] * ia), v = make_float2(acc[i][2] * ib, acc[i][3] * ib);
          if (h == 0) u.x += pa->x, u.y += pa->y, v.x += pb->x, v.y += pb->y;
          *pa = u;
          *pb = v;
        }
      }
      __syncthreads();
    }
  }

  // ---- out = y + t B^T: 64 columns in turn ----
  const int pieces64 = (a.n + 63) / 64, passes = (pieces64 - cr + C - 1) / C;
  const bool y16 = (uintptr_t)a.y % 16 == 0 && a.y_stride % 4 == 0;
  const bool out8 = (uintptr_t)a.out % 8 == 0 && a.out_stride % 2 == 0;
  const bool move = a.out != a.y;  // rows without an adapter are copied
  constexpr int BPR = 8 * NT / EPP, BSTEP = LR_THREADS / BPR, BN = (64 + BSTEP - 1) / BSTEP;
  const int br = tid / BPR, bp = tid % BPR;
  unsigned need = 0;  // bit i: row r16 + 16 i passes through
#pragma unroll
  for (int i = 0; i < XN; ++i)
    need |= (rows[r16 + XROWS * i] >= 0 && (move || ids[r16 + XROWS * i] >= 0) ? 1u : 0u) << i;
  const float* y_src = a.y + cr * 64 + p16 * 4;
  const W* b_src = reinterpret_cast<const W*>(a.b) + ((size_t)max(main_ad, 0) * a.n + cr * 64 + br) * a.rank + bp * EPP;
  unsigned char* const b_dst = smem + LT_ROWS * LT_XROW + br * T::BROW + bp * 16;
  int n_left = a.n - cr * 64;
  fill = 0;
  auto issue_cols = [&]() {
    if (n_left > 0) {
      unsigned char* to = x_dst + fill * T::STAGE;
      const int in = n_left - p16 * 4;  // columns from this piece's first
#pragma unroll
      for (int i = 0; i < XN; ++i) {
        const float* from = y_src + row_at(i) * a.y_stride;
        if (y16 && in >= 4) {
          copy16(to + i * XROWS * LT_XROW, from, need >> i & 1u);
        } else {
          for (int k = 0; k < 4; ++k)
            copy4(to + i * XROWS * LT_XROW + 4 * k, k < in ? from + k : a.y, k < in && (need >> i & 1u));
        }
      }
#pragma unroll
      for (int i = 0; i < BN; ++i)
        if (64 % BSTEP == 0 || br + i * BSTEP < 64)
          copy16(b_dst + fill * T::STAGE + i * BSTEP * T::BROW, b_src + (size_t)i * BSTEP * a.rank,
                 br + i * BSTEP < n_left && bp * EPP < main_rank);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    y_src += C * 64;
    b_src += (size_t)C * 64 * a.rank;
    n_left -= C * 64;
    fill = fill == LT_STAGES - 1 ? 0 : fill + 1;
  };
  issue_cols();  // while the cluster sums t, whose place is the last stage
  issue_cols();
  cluster.sync();
  // every CTA sums a part of t over the cluster and gives it to the others
  for (int i = cr * LR_THREADS + tid; i < LT_ROWS * 2 * NT; i += C * LR_THREADS) {  // 4 ranks of a row
    const int r = i / (2 * NT), j = i % (2 * NT) * 4;
    float4 v[LR_CLUSTER];
#pragma unroll
    for (int q = 0; q < LR_CLUSTER; ++q)
      v[q] = q < C ? *reinterpret_cast<const float4*>(cluster.map_shared_rank(part, q) + r * TS + j)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int q = 0; q < LR_CLUSTER; ++q) s.x += v[q].x, s.y += v[q].y, s.z += v[q].z, s.w += v[q].w;
    const int ad = ids[r];
    if (ad >= 0) {
      const int R = rank_of(a, ad);
      const float f = a.scales ? a.scales[ad] : 1.f;
      s.x = j < R ? s.x * f : 0.f, s.y = j + 1 < R ? s.y * f : 0.f;
      s.z = j + 2 < R ? s.z * f : 0.f, s.w = j + 3 < R ? s.w * f : 0.f;
    }
#pragma unroll
    for (int q = 0; q < LR_CLUSTER; ++q)
      if (q < C) *reinterpret_cast<float4*>(cluster.map_shared_rank(t, q) + r * TS + j) = s;
  }
  cluster.sync();

  // this warp's rows of t, as operands: each row belongs to one pass only
  Step<W> s[STEPS];
  float ia = 1.f, ib = 1.f;
  {
    float va[STEPS][8], vb[STEPS][8], ta = 0.f, tb = 0.f;
#pragma unroll
    for (int q = 0; q < STEPS; ++q) {
      const float* p = t + la * TS + 32 * q + 8 * c;
#pragma unroll
      for (int i = 0; i < 8; ++i) va[q][i] = vb[q][i] = 0.f;
      if (32 * q + 8 * c < 8 * NT) {
        load_row8(p, va[q]);
        load_row8(p + 8 * TS, vb[q]);
      }
      ta = fmaxf(ta, top8(va[q]));
      tb = fmaxf(tb, top8(vb[q]));
    }
    if constexpr (Step<W>::SCALED) {
      const float fa = scale_for(top_quad(ta)), fb = scale_for(top_quad(tb));
      ia = 1.f / fa;
      ib = 1.f / fb;
#pragma unroll
      for (int q = 0; q < STEPS; ++q) times(va[q], fa), times(vb[q], fb);
    }
#pragma unroll
    for (int q = 0; q < STEPS; ++q) s[q].split(va[q], vb[q]);
  }
  float* oa = a.out + (size_t)max(ra, 0) * a.out_stride;
  float* ob = a.out + (size_t)max(rb, 0) * a.out_stride;
  constexpr int AT = STEPS * (int)sizeof(W) > 4 ? 1 : 4;  // column tiles whose weights are fetched at once
  const bool wa = ra >= 0 && (ida >= 0 || move), wb = rb >= 0 && (idb >= 0 || move);
  __syncthreads();  // t is in registers
  const bool ragged = main_rank % 8 != 0;  // the last piece of B's rows holds ranks that are not this adapter's
  const bool bare = __any_sync(0xffffffffu, ida < 0 || idb < 0);
  int use = 0;
  auto fetch_b = [&](int ad, int R, int n0, int i0, Raw<W>(&w)[AT][STEPS]) {
    const int n = n0 + 32 * half + g;
    const W* B = reinterpret_cast<const W*>(a.b) + ((size_t)ad * a.n + n) * a.rank + 8 * c;
#pragma unroll
    for (int i = 0; i < AT; ++i)
#pragma unroll
      for (int q = 0; q < STEPS; ++q) {
        const int valid = R - 32 * q - 8 * c;  // ranks of this lane's piece; B may hold anything behind them
        if (valid > 0 && n + 8 * (i0 + i) < a.n)
          fetch(B + (size_t)8 * (i0 + i) * a.rank + 32 * q, w[i][q]);
        else
          clear(w[i][q]);
        if (valid > 0 && valid < 8) cut(w[i][q], valid);
      }
  };
  for (int p = 0; p < passes; ++p) {
    Raw<W> w[AT][STEPS];
    if (other >= 0) fetch_b(other, other_rank, (p * C + cr) * 64, 0, w);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    issue_cols();
    const unsigned char* st = smem + use * T::STAGE;
    use = use == LT_STAGES - 1 ? 0 : use + 1;
    const int n0 = (p * C + cr) * 64;
    float d[4][4];  // this warp's four column tiles
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0.f;
    const unsigned char* wt = st + LT_ROWS * LT_XROW + (32 * half + g) * T::BROW + 8 * c * (int)sizeof(W);
    if (has_main) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < STEPS; ++q) {
          if (32 * q >= main_rank) break;
          Raw<W> m;
          if (8 * NT >= 32 || 8 * c < 8 * NT)
            load_raw(wt + 8 * i * T::BROW + 32 * q * (int)sizeof(W), m);
          else
            clear(m);
          if (ragged) {  // t is 0 there, but B may hold anything
            const int valid = main_rank - 32 * q - 8 * c;
            if (valid > 0 && valid < 8) cut(m, valid);
          }
          s[q].mma(d[i], m);
        }
    }
    int R = other_rank;
    for (int ad = other; ad >= 0;) {  // each row's sum is its own adapter's
#pragma unroll
      for (int i0 = 0; i0 < 4; i0 += AT) {
        if (i0 > 0) fetch_b(ad, R, n0, i0, w);
#pragma unroll
        for (int i = 0; i < AT; ++i) {
          float e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < STEPS; ++q)
            if (32 * q < R) s[q].mma(e, w[i][q]);
          if (ida == ad) d[i0 + i][0] = e[0], d[i0 + i][1] = e[1];
          if (idb == ad) d[i0 + i][2] = e[2], d[i0 + i][3] = e[3];
        }
      }
      ad = other_after(ad);
      if (ad >= 0) fetch_b(ad, R = rank_of(a, ad), n0, 0, w);
    }
    const bool whole = out8 && n0 + 64 <= a.n;
    float* const pa = oa + n0 + 32 * half + 2 * c;
    float* const pb = ob + n0 + 32 * half + 2 * c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 y0 = *reinterpret_cast<const float2*>(st + la * LT_XROW + (32 * half + 8 * i + 2 * c) * 4);
      const float2 y1 = *reinterpret_cast<const float2*>(st + lb * LT_XROW + (32 * half + 8 * i + 2 * c) * 4);
      float2 u = make_float2(fmaf(d[i][0], ia, y0.x), fmaf(d[i][1], ia, y0.y));
      float2 v = make_float2(fmaf(d[i][2], ib, y1.x), fmaf(d[i][3], ib, y1.y));
      if (bare) {  // rows without an adapter among rows that have one: whatever its weights times 0 are stays out
        if (ida < 0) u = y0;
        if (idb < 0) v = y1;
      }
      if (whole) {
        if (wa) *reinterpret_cast<float2*>(pa + 8 * i) = u;
        if (wb) *reinterpret_cast<float2*>(pb + 8 * i) = v;
      } else {
        const int col = n0 + 32 * half + 8 * i + 2 * c;
        if (wa && col < a.n) pa[8 * i] = u.x;
        if (wb && col < a.n) pb[8 * i] = v.x;
        if (wa && col + 1 < a.n) pa[8 * i + 1] = u.y;
        if (wb && col + 1 < a.n) pb[8 * i + 1] = v.y;
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename W, int LG>
int launch_row(const LoraArgs& a, cudaStream_t s) {
  // 8 CTAs a row while their parts of k and n are worth a cluster's two barriers (at least a warp's lanes along k).
  // Many rows take smaller clusters; with 8 their CTAs come in waves of about 5 us.  200 rows of rank 64, k 1088, n 2317
  // take 30 us with clusters of 8, 22 with 4, 18 with 2 (120 rows 12.8 with 4); of rank 16, k = n = 4096, where four CTAs
  // fit an SM, 14.0, 10.5 and 13.7.  The cluster's size sets the order of t's sum, so up to 112 rows it stays 8: a row
  // then has the same bits in all those batches (100 rows of the two shapes: 15.9 and 8.8 us with 8, 11.9 and 8.9 with
  // 4).
  int C = a.rows <= 112 ? LR_CLUSTER : a.rows <= (LG <= 2 ? 208 : 128) ? 4 : 2;
  while (C > 1 && a.k < 256 * C && a.n < 256 * C) C >>= 1;
  // Few rows take several clusters each, which all sum t and share n, until a CTA's part of n is what it fetches ahead
  // or the clusters (32 of 8 CTAs) no longer fit two CTAs an SM: one row of rank 32, n 11008, k 4096 takes 7.7 us with
  // one cluster, 5.3 with six.
  const int fetched = C * LR_AHEAD * (LR_THREADS / LG);
  const int parts = std::max(1, std::min((a.n + fetched - 1) / fetched, 32 * 8 / (a.rows * C)));
  if ((long long)a.rows * C * parts > 0x7fffffffLL) return kTooLarge;
  return launch_cluster_pdl(lora_row_kernel<W, LG>, dim3(a.rows * C * parts), dim3(LR_THREADS), C, 0, s, a, parts) ==
                 cudaSuccess
             ? kOk
             : kCudaError;
}

template <typename W, int NT>
int launch_tile(const LoraArgs& a, cudaStream_t s) {
  const int tiles = (a.rows + LT_ROWS - 1) / LT_ROWS;
  const size_t smem = Tile<W, NT>::BYTES;
  auto kernel = lora_tile_kernel<W, NT>;
  if (allow_smem(kernel, smem, smem)) return kCudaError;
  if ((long long)tiles * LR_CLUSTER > 0x7fffffffLL) return kTooLarge;
  return launch_cluster_pdl(kernel, dim3(tiles * LR_CLUSTER), dim3(LR_THREADS), LR_CLUSTER, smem, s, a) == cudaSuccess
             ? kOk
             : kCudaError;
}

template <typename W, int LG>
int launch(const LoraArgs& a, cudaStream_t s) {
  // A cluster per row up to 256 rows, whatever adapters they use: 256 rows of rank 64, k = n = 4096 take 34 us with 8
  // adapters and 56 with 64 (of rank 16: 14 and 16).  Tiles take 31 us (22) for 64 to 256 rows in runs and 40 (29) for
  // 1024, and where each row names one of 8 or 64 adapters 48 and 150 (33 and 81) for 256 rows, 88 (61) for 1024 and 64:
  // how many meet in a tile only the device knows.
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
