// attention_sparse.cu -- decode attention over the pages of a paged K/V cache that a cheap score selects, one launch.
//
// For a query row and a KV head, with the 8-bit key bounds lo, hi and scale s of every page (kv_append.cu):
//   score(page) = s * max over the head's query heads of  s_q * sum_d max(qi_d lo_d, qi_d hi_d)
// where qi = rint(q / s_q), s_q = max|q| / 32512: an upper bound of q.k over the page, up to the rounding of q.  The
// sum is a whole number below 2^30 and the two factors are one fp32 rounding each, so the selection does not depend
// on any order of summation.  The first `sink` and the last `recent` pages and the highest scores fill the budget, the
// lower page first among equals; softmax attention (as paged decode attention, GqaAttention.cs:29-130) then runs over
// the tokens of these pages.  A row that has no more pages than the budget is attended whole and scores nothing.
//
// One cluster of S CTAs per (query row, KV head), from score to output, with no scratch in memory:
//   score   each CTA scores its share of the pages.  max(qi lo, qi hi) = max(qi, 0) hi + min(qi, 0) lo, so a score
//           is one product of 2 hd signed bytes: mma m16n8k32.s8, eight heads' high bytes of qi in rows 0-7 and their
//           low bytes in rows 8-15, eight pages as columns.  Records pass through a cp.async buffer of the warp's own,
//           sixteen pages a stage, two stages in flight; their ids come from shared memory, so that no load waits for
//           another.
//   select  the CTAs exchange their scores through distributed shared memory; each finds the threshold by radix
//           select on the order-preserving bits, and takes its part of the chosen pages, in page order.
//   attend  mma m16n8k16 on the raw fp16 keys and values, from the same buffer, with the fp32 query as hi + lo halves in
//           rows 0-7 and 8-15 (a power of two of its own brings each head's query into fp16's range) and the fp32
//           weights split likewise, relative to the block's largest one: products are exact, and scores and weights
//           hold fp32 to about 2^-22 (weights down to 2^-28 of their 16 neighbours' largest).  The accumulator
//           layout of q.k is the operand layout of p.v, and the contraction index is permuted alike on both sides, so
//           operands are 16-byte reads and nothing is exchanged between lanes but the row maxima.  fp32 pools take
//           the same path with tf32 hi + lo pairs of both sides.
//   join    warps, then the cluster's CTAs, merge their (max, sum, output) states in shared memory.
// Bound: HBM, bytes = pages * (2 hd + 4) + selected tokens * hd * 2 * sizeof(kv) per (row, KV head), behind a chain of
// about 10 us that every row has (lengths, ids, bounds, threshold, keys, join).  32 sequences of 4k to 32k tokens,
// 32 / 8 heads of 128, 128 pages of 16: 82 us for 350 MB (4.3 TB/s); 24 sequences of up to 2k tokens, 12 heads of 64,
// fp32 pools, 32 pages: 26 us for 70 MB; one sequence of 8k tokens: 13.8 us, the chain.

#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>
#include <utility>

#include "batch_ops.h"
#include "common.cuh"

namespace cg = cooperative_groups;

namespace zc {

namespace {

constexpr int SP_WARPS = 8;
constexpr int SP_THREADS = SP_WARPS * 32;
constexpr int SP_CLUSTER = 8;  // most CTAs of a cluster
constexpr int SP_HEADS = 8;  // query heads per pass: half of an mma's 16 rows
constexpr float SP_LOG2E = 1.4426950408889634f;
constexpr float SP_P_BITS = 14.f, SP_LO = 2048.f;  // fp16 pools: power of two of a block's weights, factor of their lo halves
constexpr size_t SP_SMEM_MAX = 220 * 1024;

struct SparseDev {
  SparseAttnArgs a;
  int cap_pages;  // pages that max_ctx allows
  int share;      // list entries of a CTA: ceil(budget / S)
  int key_words;  // scores a CTA holds: all pages', where there may be more than the budget
  int id_words;   // page ids it holds beside them: as many, or 0 where shared memory does not have the room
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t tf32_of(float v) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return r;
}
// v = hi + lo with both in tf32 (v - hi is exact in fp32)
__device__ __forceinline__ void tf32_pair(float v, uint32_t& hi, uint32_t& lo) {
  hi = tf32_of(v);
  lo = tf32_of(v - __uint_as_float(hi));
}

// 16 bytes from memory into shared memory, zeros where !ok (nothing is read then)
__device__ __forceinline__ void copy16(void* dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
               "r"(ok ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>  // all but the last N groups of this thread have landed
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// 16-byte piece of a row in a warp's buffer.  Operand reads of keys and bounds take rows g, pieces 4 j + c, those of
// values rows 2 c and 2 c + 1, pieces 8 j + g: either exchange puts the eight lanes of an access on all banks.
__device__ __forceinline__ int key_piece(int row, int piece) { return piece ^ ((row & 1) * 4); }
__device__ __forceinline__ int value_piece(int row, int piece) { return piece ^ (row & 6); }
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Unsigned key whose order is the float's (NaN, the score of a page with an infinite key, above everything; -0 below 0:
// callers pass sums that are never -0).  The asm keeps these bits from the compiler, which would set the sign by a
// floating-point negation and so lose a NaN's.
__device__ __forceinline__ uint32_t order_key(float f) {
  uint32_t u;
  asm("mov.b32 %0, %1;" : "=r"(u) : "f"(f));
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// The score operand of a head tile: rows 0-7 the high bytes of qi, rows 8-15 the low bytes (qi = 256 high + low, both
// signed), columns [min(qi, 0) per dim | max(qi, 0) per dim].  sq: s_q per head, -inf factor handled by the caller.
template <int HD>
__device__ void stage_score_query(const float* q, int heads, int8_t* qs, int stride, float* sq) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int h = threadIdx.x >> 5; h < SP_HEADS; h += SP_WARPS) {  // one warp per head
    float v[HD / 32], top = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      v[i] = h < heads ? q[h * HD + lane + 32 * i] : 0.f;
      top = fmaxf(top, fabsf(v[i]));
    }
    top = warp_max(top);
    const float s = __fdiv_rn(top, 32512.f);
    if (lane == 0) sq[h] = s;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const int qi = s > 0.f ? min(max(__float2int_rn(__fdiv_rn(v[i], s)), -32512), 32512) : 0;
      const int neg = min(qi, 0), pos = max(qi, 0), d = lane + 32 * i;
      const int8_t nl = (int8_t)(neg & 255), pl = (int8_t)(pos & 255);
      qs[h * stride + d] = (int8_t)((neg - nl) >> 8);
      qs[(h + 8) * stride + d] = nl;
      qs[h * stride + HD + d] = (int8_t)((pos - pl) >> 8);
      qs[(h + 8) * stride + HD + d] = pl;
    }
  }
}

// The attention operand of a head tile: q * scale * log2(e) * 2^e, hi parts in rows 0-7, lo parts in rows 8-15.
// ex[head] = 2^-e undoes the power of two, which puts the largest |q| of the head at 2^7 .. 2^8.
template <int HD, bool HALF>
__device__ void stage_query(const float* q, int heads, float scale_log2, void* qa, int stride, float* ex) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int h = threadIdx.x >> 5; h < SP_HEADS; h += SP_WARPS) {
    float v[HD / 32], top = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      v[i] = h < heads ? q[h * HD + lane + 32 * i] * scale_log2 : 0.f;
      top = fmaxf(top, fabsf(v[i]));
    }
    top = warp_max(top);
    float up = 1.f, down = 1.f;
    const int e = (int)((__float_as_uint(top) >> 23) & 255u) - 127;  // floor(log2(top)) of a normal number
    if (HALF && top > 0.f && top < INFINITY) {
      const int k = min(max(7 - e, -126), 126);
      up = __uint_as_float((uint32_t)(127 + k) << 23);
      down = __uint_as_float((uint32_t)(127 - k) << 23);
    }
    if (lane == 0) ex[h] = down;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const int d = lane + 32 * i;
      if (HALF) {
        store_hl(reinterpret_cast<__half*>(qa) + h * stride + d, (size_t)8 * stride, v[i] * up);
      } else {
        uint32_t hi, lo;
        tf32_pair(v[i], hi, lo);
        uint32_t* o = reinterpret_cast<uint32_t*>(qa);
        o[h * stride + d] = hi;
        o[(h + 8) * stride + d] = lo;
      }
    }
  }
}

// One warp's attention state: outputs of head lane / 4, two dims per tile of eight.  The tensor core's accumulator
// truncates, so it holds one block's products only; a block's hi and lo rows are added to the state with rounding.
template <int HD, bool HALF>
struct State {
  static constexpr int NT = HD / 8;
  float acc[NT][2];
  float m, l;  // head lane / 4: running maximum (log2 domain), this lane's share of the sum

  __device__ void init() {
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }
  // The new maximum over the tile's scores (N per lane), whose own maximum is t; rescales what was summed so far.
  template <int N>
  __device__ float raise(const float (&s)[N], float& t) {
    t = s[0];
#pragma unroll
    for (int i = 1; i < N; ++i) t = fmaxf(t, s[i]);
    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
    const float mn = fmaxf(m, t);
    const float base = mn == -INFINITY ? 0.f : mn;  // no token yet: every weight below is exp2(-inf) = 0
    const bool moved = mn > m;
    if (__any_sync(0xffffffffu, moved)) {
      const float alpha = exp2f(m - base);
      l *= alpha;
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i][0] *= alpha, acc[i][1] *= alpha;
    }
    m = mn;
    return base;
  }
};

template <int HD, bool HALF, int CTAS>
__global__ void __launch_bounds__(SP_THREADS, CTAS) sparse_attn_kernel(SparseDev dv) {
  const SparseAttnArgs& a = dv.a;
  constexpr int QS = 2 * HD + 16;                    // bytes of a score operand row
  constexpr int QA = HALF ? HD + 8 : HD + 4;         // elements of an attention operand row
  constexpr int ES = HALF ? 2 : 4;
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int RING = 64 * HD;                      // a warp's buffer: 32 bounds records, or a block's keys and values
  unsigned char* ring = smem + (threadIdx.x >> 5) * RING;
  float* so = reinterpret_cast<float*>(smem);                      // at the end: each warp's outputs
  unsigned char* at = smem + SP_WARPS * RING;
  uint32_t* keys = reinterpret_cast<uint32_t*>(at);                // [key_words]: scores of all pages
  at += (size_t)dv.key_words * 4;
  int32_t* ids = reinterpret_cast<int32_t*>(at);                   // [id_words]: page ids of the table row
  at += (size_t)dv.id_words * 4;
  float* part = reinterpret_cast<float*>(at);                      // this CTA's output, 8 HD floats
  at += SP_HEADS * HD * 4;
  int8_t* qs = reinterpret_cast<int8_t*>(at);                      // [16][QS]
  at += 16 * QS;
  unsigned char* qa = at;                                          // [16][QA]
  at += 16 * QA * ES;
  int2* list = reinterpret_cast<int2*>(at);                        // [share]: (page id, page of the sequence)
  __shared__ uint32_t hist[4][256];
  __shared__ float sq[SP_HEADS], ex[SP_HEADS];
  __shared__ float wm[SP_WARPS][SP_HEADS], wl[SP_WARPS][SP_HEADS];
  __shared__ float pm[SP_HEADS], pl[SP_HEADS];
  __shared__ int red[2][SP_WARPS];
  __shared__ int s_digit, s_rem, s_all;
  pdl_trigger();
  pdl_wait();

  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();
  const int rank = cluster.block_rank(), S = cluster.num_blocks();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int g = lane >> 2, c = lane & 3;
  const long long pair = blockIdx.x / S;
  const int b = (int)(pair / a.hkv), kvh = (int)(pair % a.hkv);
  const int P = a.page_size, group = a.hq / a.hkv;
  const int row = a.rows ? a.rows[b] : b;
  int ctx = (unsigned)row < (unsigned)a.table_rows ? min(max(a.ctx_len[b], 0), a.max_ctx) : 0;
  const int n = min((ctx + P - 1) / P, dv.cap_pages);  // max_ctx and a page are within 2^30
  ctx = (int)min((long long)ctx, (long long)n * P);    // a table shorter than max_ctx
  const int want = min(a.budget, n);
  const float* q = a.q + (size_t)b * a.q_stride + (size_t)kvh * group * HD;
  float* out = a.out + ((size_t)b * a.hq + (size_t)kvh * group) * HD;
  const bool wide = (uintptr_t)a.out % 16 == 0;  // 16-byte stores
  int32_t* sel = a.sel + ((size_t)b * a.hkv + kvh) * a.budget;
  for (int i = want + rank * SP_THREADS + tid; i < a.budget; i += S * SP_THREADS) sel[i] = -1;
  if (n == 0) {  // the same for the whole cluster
    for (int i = rank * SP_THREADS + tid; i < group * HD; i += S * SP_THREADS) out[i] = 0.f;
    cluster.barrier_wait();
    return;
  }
  const int32_t* pt = a.page_table + (size_t)row * a.max_pages;
  const bool keep_ids = dv.id_words > 0 && n > a.budget;
  if (keep_ids) {
    for (int i = tid; i < n; i += SP_THREADS)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(ids + i)),
                   "l"(pt + i)
                   : "memory");
  }
  copies_commit();
  // the first head tile's operands, while the ids are on their way
  stage_score_query<HD>(q, min(SP_HEADS, group), qs, QS, sq);
  stage_query<HD, HALF>(q, min(SP_HEADS, group), a.scale * SP_LOG2E, qa, QA, ex);
  auto id_of = [&](int p) { return keep_ids ? ids[p] : pt[p]; };
  const int share = (want + S - 1) / S;

  if (n <= a.budget) {
    for (int i = rank * share + tid; i < min(want, (rank + 1) * share); i += SP_THREADS) {
      list[i - rank * share] = make_int2(pt[i], i);
      sel[i] = i;
    }
    cluster.barrier_wait();
  } else {
    // ---- score ----
    const int cs = (n + S - 1) / S, p_begin = min(n, rank * cs), p_end = min(n, p_begin + cs);
    for (int i = tid; i < 4 * 256; i += SP_THREADS) hist[0][i] = 0;
    constexpr int KS = 2 * HD / 64;      // 16-byte pieces of a record per lane; two k-steps of 32 each
    constexpr int RP = 2 * HD / 16;      // pieces of a record
    for (int h0 = 0; h0 < group; h0 += SP_HEADS) {
      const int heads = min(SP_HEADS, group - h0);
      if (h0 > 0) {
        __syncthreads();  // the last tile's operand is no longer read
        stage_score_query<HD>(q + (size_t)h0 * HD, heads, qs, QS, sq);
      }
      copies_wait<0>();
      __syncthreads();  // staged, the ids there, and the histograms cleared
      uint4 ah[KS], al[KS];
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        ah[j] = *reinterpret_cast<const uint4*>(qs + g * QS + 64 * j + 16 * c);
        al[j] = *reinterpret_cast<const uint4*>(qs + (g + 8) * QS + 64 * j + 16 * c);
      }
      const float s_q = sq[g];
      const bool last = h0 + SP_HEADS >= group;
      // Sixteen pages a stage, two stages in flight (four measured no better); lanes 0-15 hold the pages' ids, scales and
      // whether they exist.
      constexpr int STAGES = 2;
      int id = -1;
      float scale[STAGES];
      bool ok[STAGES];
#pragma unroll
      for (int i = 0; i < STAGES; ++i) scale[i] = 0.f, ok[i] = false;
      auto fetch_ids = [&](int p0) {
        const int p = p0 + lane;
        id = lane < 16 && p < p_end ? id_of(p) : -1;
      };
      auto issue = [&](int p0, int buf) {
        const bool in_pool = (unsigned)id < (unsigned)a.num_pages;
        const size_t rec = in_pool ? (size_t)id * a.hkv + kvh : 0;
        if (p0 < p_end) {
#pragma unroll
          for (int i = 0; i < RP / 2; ++i) {
            const int r = (i * 32 + lane) / RP, piece = (i * 32 + lane) % RP;
            const size_t from = __shfl_sync(0xffffffffu, rec, r);
            copy16(ring + buf * 16 * 2 * HD + r * 2 * HD + key_piece(r, piece) * 16,
                   a.bounds + from * (2 * HD) + piece * 16, __shfl_sync(0xffffffffu, (int)in_pool, r));
          }
        }
        copies_commit();
#pragma unroll
        for (int i = 0; i + 1 < STAGES; ++i) scale[i] = scale[i + 1], ok[i] = ok[i + 1];
        ok[STAGES - 1] = in_pool;
        scale[STAGES - 1] = in_pool && last ? __ldg(a.scales + rec) : 0.f;
      };
      constexpr int STEP = SP_WARPS * 16;
      const int first = p_begin + warp * 16;
#pragma unroll
      for (int i = 0; i < STAGES; ++i) {
        fetch_ids(first + i * STEP);
        issue(first + i * STEP, i);
      }
      fetch_ids(first + STAGES * STEP);
      int buf = 0;
      for (int p0 = first; p0 < p_end; p0 += STEP) {
        copies_wait<STAGES - 1>();
        __syncwarp();
        int d2[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          int d[4] = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            const int r = 8 * u + g;
            const uint4 rec = *reinterpret_cast<const uint4*>(ring + buf * 16 * 2 * HD + r * 2 * HD +
                                                              key_piece(r, 4 * j + c) * 16);
            mma_s8(d, ah[j].x, al[j].x, ah[j].y, al[j].y, rec.x, rec.y);
            mma_s8(d, ah[j].z, al[j].z, ah[j].w, al[j].w, rec.z, rec.w);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) d2[u][i] = d[i];
        }
        __syncwarp();
        const float sc = scale[0];
        const bool exists = ok[0];
        issue(p0 + STAGES * STEP, buf);
        fetch_ids(p0 + (STAGES + 1) * STEP);
        buf = buf + 1 == STAGES ? 0 : buf + 1;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int(&d)[4] = d2[u];
          // columns (pages) 2c and 2c + 1 of head g; the maximum over the tile's heads
          float f0 = g < heads ? __fmul_rn((float)(d[0] * 256 + d[2]), s_q) : -INFINITY;
          float f1 = g < heads ? __fmul_rn((float)(d[1] * 256 + d[3]), s_q) : -INFINITY;
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            f0 = fmaxf(f0, __shfl_xor_sync(0xffffffffu, f0, o));
            f1 = fmaxf(f1, __shfl_xor_sync(0xffffffffu, f1, o));
          }
          // lanes 0-3 take the pages 2c and 2c + 1
          const int at0 = 8 * u + 2 * c;
          const float c0 = __shfl_sync(0xffffffffu, sc, at0), c1 = __shfl_sync(0xffffffffu, sc, at0 + 1);
          const int v0 = __shfl_sync(0xffffffffu, (int)exists, at0), v1 = __shfl_sync(0xffffffffu, (int)exists, at0 + 1);
          if (g == 0) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int p = p0 + 8 * u + 2 * c + k;
              if (p >= p_end) continue;
              float f = k ? f1 : f0;
              if (h0 > 0) f = fmaxf(f, __uint_as_float(keys[p]));
              if (last)  // + 0: -0 orders as 0
                keys[p] = (k ? v1 : v0) ? order_key(__fmul_rn(f, k ? c1 : c0) + 0.f) : 0u;
              else
                keys[p] = __float_as_uint(f);
            }
          }
        }
      }
    }
    // ---- every CTA gets every key ----
    __syncthreads();
    cluster.barrier_wait();  // the other CTAs have started
    for (int r = 0; r < S; ++r)
      if (r != rank) {
        uint32_t* to = cluster.map_shared_rank(keys, r);
        for (int i = p_begin + tid; i < p_end; i += SP_THREADS) to[i] = keys[i];
      }
    cluster.sync();
    // ---- select: the forced pages, and the `rem` largest keys of the pages [f0, f1) between them ----
    const int f0 = min(a.sink, n), f1 = max(f0, n - a.recent);
    int rem = want - (n - (f1 - f0));
    uint32_t kmin = 0xffffffffu, kmax = 0;
    for (int i = f0 + tid; i < f1; i += SP_THREADS) {
      kmin = min(kmin, keys[i]);
      kmax = max(kmax, keys[i]);
    }
    kmin = __reduce_min_sync(0xffffffffu, kmin);
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if (lane == 0) red[0][warp] = (int)kmin, red[1][warp] = (int)kmax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SP_WARPS; ++w) {
      kmin = min(kmin, (uint32_t)red[0][w]);
      kmax = max(kmax, (uint32_t)red[1][w]);
    }
    // Radix select on key - kmin from its highest bit in use (scores share their leading bits): after a pass `cur` are
    // the leading bits of the threshold, down to bit `shift`.
    uint32_t cur = 0;
    int shift = f1 > f0 ? 32 - __clz((int)(kmax - kmin)) : 0;
    for (int pass = 0; rem > 0; ++pass) {  // at most four: 8 bits each
      const int bits = min(8, shift);
      shift -= bits;
      for (int i = f0 + tid; i < f1; i += SP_THREADS) {
        const uint32_t k = (keys[i] - kmin) >> shift;
        if (k >> bits == cur) atomicAdd(&hist[pass][k & ((1u << bits) - 1u)], 1u);
      }
      __syncthreads();
      constexpr int DG = 256 / SP_THREADS;  // digits a thread, the highest first
      int tot[DG], inc = 0;
#pragma unroll
      for (int k = 0; k < DG; ++k) {
        tot[k] = (int)hist[pass][255 - (tid * DG + k)];
        inc += tot[k];
      }
      const int own = inc;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      if (lane == 31) red[0][warp] = inc;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < SP_WARPS; ++w) inc += w < warp ? red[0][w] : 0;
      inc -= own;  // keys with a higher digit than this thread's
#pragma unroll
      for (int k = 0; k < DG; ++k) {
        if (inc < rem && inc + tot[k] >= rem) {
          s_digit = 255 - (tid * DG + k);
          s_rem = rem - inc;
          s_all = rem - inc == tot[k];
        }
        inc += tot[k];
      }
      __syncthreads();
      cur = cur << bits | (uint32_t)s_digit;
      rem = s_rem;
      if (s_all || shift == 0) break;  // every key with these leading bits is taken, or they are all its bits
    }
    // ---- this CTA's part of the list, in page order: forced, above the threshold, the first `rem` equal to it ----
    const bool some = want > n - (f1 - f0);  // a threshold was found
    const int seg = ((n + SP_WARPS - 1) / SP_WARPS + 31) / 32 * 32, w0 = min(n, warp * seg), w1 = min(n, w0 + seg);
    auto kind = [&](int i) {  // 2: taken, 1: equal to the threshold, 0: not
      if (i >= w1) return 0;
      if (i < f0 || i >= f1) return 2;
      if (!some) return 0;
      const uint32_t k = (keys[i] - kmin) >> shift;
      return k > cur ? 2 : k == cur ? 1 : 0;
    };
    int gt = 0, eq = 0;
    for (int i = w0; i < w1; i += 32) {
      const int k = kind(i + lane);
      gt += __popc(__ballot_sync(0xffffffffu, k == 2));
      eq += __popc(__ballot_sync(0xffffffffu, k == 1));
    }
    __syncthreads();
    if (lane == 0) red[0][warp] = gt, red[1][warp] = eq;
    __syncthreads();
    int gt_seen = 0, eq_seen = 0;
    for (int w = 0; w < warp; ++w) gt_seen += red[0][w], eq_seen += red[1][w];
    const int l0 = rank * share, l1 = min(want, l0 + share);
    for (int i = w0; i < w1; i += 32) {
      const int k = kind(i + lane);
      const unsigned bgt = __ballot_sync(0xffffffffu, k == 2), beq = __ballot_sync(0xffffffffu, k == 1);
      const unsigned below = (1u << lane) - 1u;
      const int e = eq_seen + __popc(beq & below);  // rank among the equal ones
      const int to = gt_seen + __popc(bgt & below) + min(e, rem);
      if ((k == 2 || (k == 1 && e < rem)) && to >= l0 && to < l1) {
        sel[to] = i + lane;
        list[to - l0] = make_int2(id_of(i + lane), i + lane);
      }
      gt_seen += __popc(bgt);
      eq_seen += __popc(beq);
    }
  }

  // ---- attend ----
  const int mine = max(0, min(want, (rank + 1) * share) - rank * share);
  const int tokens = mine * P;
  const unsigned char* kb = reinterpret_cast<const unsigned char*>(a.k_pool) + (long long)kvh * a.head_stride * ES;
  const unsigned char* vb = reinterpret_cast<const unsigned char*>(a.v_pool) + (long long)kvh * a.head_stride * ES;
  // Eight tokens from flat index i8 (a multiple of 8, as the page size is): their offset in the pools and how many of
  // them the sequence has.
  auto locate = [&](int i8, long long& off) {
    off = 0;
    if (i8 >= tokens) return 0;
    const int e = i8 / P, slot = i8 - e * P;
    const int2 p = list[e];
    if ((unsigned)p.x >= (unsigned)a.num_pages) return 0;
    off = ((long long)p.x * a.page_stride + (long long)slot * a.slot_stride) * ES;
    return min(max(ctx - (p.y * P + slot), 0), 8);
  };
  for (int h0 = 0; h0 < group; h0 += SP_HEADS) {
    const int heads = min(SP_HEADS, group - h0);
    __syncthreads();  // the list is written; the last tile's operand and outputs are no longer read
    if (h0 > 0) {
      stage_query<HD, HALF>(q + (size_t)h0 * HD, heads, a.scale * SP_LOG2E, qa, QA, ex);
      __syncthreads();
    }
    const float down = ex[g];
    State<HD, HALF> st;
    st.init();
    // A block is 16 tokens (fp32 pools: 8) of keys and as many of values in the warp's buffer.  The next block's keys
    // are on their way from when this block's have been read, its values likewise.
    constexpr int TB = HALF ? 16 : 8, NB = TB / 8;
    constexpr int ROWB = HD * ES, RPC = ROWB / 16;  // bytes and 16-byte pieces of a row
    constexpr int HALF_RING = TB * ROWB;            // keys, then values
    static_assert(2 * HALF_RING == RING, "a block's keys and values fill the warp's buffer");
    const long long row_bytes = a.slot_stride * ES;
    constexpr int RPI = 32 / RPC > 0 ? 32 / RPC : 1;  // rows that a warp's copy instruction covers
    constexpr int IPR = RPC > 32 ? RPC / 32 : 1;      // instructions per row where a row has more than 32 pieces
    const int row0 = IPR > 1 ? 0 : lane / RPC, piece0 = IPR > 1 ? lane : lane % RPC;
    const unsigned char* const k_lane = kb + row0 * row_bytes + piece0 * 16;
    const unsigned char* const v_lane = vb + row0 * row_bytes + piece0 * 16;
    auto copy_rows = [&](const unsigned char* from, unsigned char* to, const long long (&off)[NB], const int (&nv)[NB],
                         bool keys_) {
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const unsigned char* src = from + off[u];
#pragma unroll
        for (int i = 0; i < 8; i += RPI) {
          const int r = i + row0;
#pragma unroll
          for (int k = 0; k < IPR; ++k) {
            const int piece = piece0 + 32 * k;
            copy16(to + (8 * u + r) * ROWB + (keys_ ? key_piece(r, piece) : value_piece(r, piece)) * 16, src + 512 * k,
                   r < nv[u]);
          }
          src += RPI * row_bytes;
        }
      }
      copies_commit();
    };
    constexpr int STRIDE = SP_WARPS * TB;  // tokens between a warp's blocks
    unsigned char* const kbuf = ring;
    unsigned char* const vbuf = ring + HALF_RING;
    int nv[NB];  // tokens that the block in the buffer has
    int i0 = warp * TB;
    if (i0 < tokens) {
      long long off[NB];
#pragma unroll
      for (int u = 0; u < NB; ++u) nv[u] = locate(i0 + 8 * u, off[u]);
      copy_rows(k_lane, kbuf, off, nv, true);
      copy_rows(v_lane, vbuf, off, nv, false);
    }
    for (; i0 < tokens; i0 += STRIDE) {
      const bool more = i0 + STRIDE < tokens;
      long long off_next[NB];
      int nv_next[NB];
#pragma unroll
      for (int u = 0; u < NB; ++u) nv_next[u] = locate(i0 + STRIDE + 8 * u, off_next[u]);
      copies_wait<1>();  // the keys
      __syncwarp();
      float s[2 * NB];
      if constexpr (HALF) {
        const __half* qh = reinterpret_cast<const __half*>(qa);
        float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          const uint4 ah = *reinterpret_cast<const uint4*>(qh + g * QA + 32 * j + 8 * c);
          const uint4 al = *reinterpret_cast<const uint4*>(qh + (g + 8) * QA + 32 * j + 8 * c);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            // 32 dims a sum in the tensor core, whose accumulator truncates; the sums are added with rounding
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            const uint4 k = *reinterpret_cast<const uint4*>(kbuf + (8 * u + g) * ROWB + key_piece(g, 4 * j + c) * 16);
            mma_f16(d, ah.x, al.x, ah.y, al.y, k.x, k.y);
            mma_f16(d, ah.z, al.z, ah.w, al.w, k.z, k.w);
            z[2 * u] += d[0] + d[2];
            z[2 * u + 1] += d[1] + d[3];
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[2 * u] = 2 * c < nv[u] ? z[2 * u] * down : -INFINITY;
          s[2 * u + 1] = 2 * c + 1 < nv[u] ? z[2 * u + 1] * down : -INFINITY;
        }
      } else {
        const uint32_t* qt = reinterpret_cast<const uint32_t*>(qa);
        float z0 = 0.f, z1 = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
          float d[4] = {0.f, 0.f, 0.f, 0.f}, dl[4] = {0.f, 0.f, 0.f, 0.f};
          const uint4 ah = *reinterpret_cast<const uint4*>(qt + g * QA + 16 * j + 4 * c);
          const uint4 al = *reinterpret_cast<const uint4*>(qt + (g + 8) * QA + 16 * j + 4 * c);
          const uint4 k = *reinterpret_cast<const uint4*>(kbuf + g * ROWB + key_piece(g, 4 * j + c) * 16);
          uint32_t h[4], l[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) tf32_pair(__uint_as_float(word(k, i)), h[i], l[i]);
          mma_tf32(d, ah.x, al.x, ah.y, al.y, h[0], h[1]);
          mma_tf32(dl, ah.x, al.x, ah.y, al.y, l[0], l[1]);
          mma_tf32(d, ah.z, al.z, ah.w, al.w, h[2], h[3]);
          mma_tf32(dl, ah.z, al.z, ah.w, al.w, l[2], l[3]);
          z0 += d[0] + ((dl[0] + dl[2]) + d[2]);
          z1 += d[1] + ((dl[1] + dl[3]) + d[3]);
        }
        s[0] = 2 * c < nv[0] ? z0 : -INFINITY;
        s[1] = 2 * c + 1 < nv[0] ? z1 : -INFINITY;
      }
      __syncwarp();
      if (more)
        copy_rows(k_lane, kbuf, off_next, nv_next, true);
      else
        copies_commit();  // an empty group, so that the wait below counts the same
      float top;
      const float base = st.raise(s, top);
      if constexpr (HALF) {
        // fp16 ends at 2^-24, and a row may be carried by weights far below its largest one, whose value is 0 (an
        // attention sink).  So a block's weights are relative to its own maximum, which gets 2^14 (SP_P_BITS); lo
        // halves, below 2^3, are held times 2^11 (SP_LO).  That keeps 2^-22 of a weight down to 2^-28 of the largest
        // among the block's 16 tokens, and 2^-50 of that one below.  `back` returns the block to the state's maximum.
        const bool none = top == -INFINITY;
        const float from = none ? 0.f : top - SP_P_BITS, back = none ? 0.f : exp2f(from - base);
        uint32_t p_hi[2], p_lo[2];
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float p0 = exp2f(s[2 * u] - from), p1 = exp2f(s[2 * u + 1] - from);
          sum += p0 + p1;
          const __half2 h = __floats2half2_rn(p0, p1);
          const float2 hf = __half22float2(h);
          const __half2 lo = __floats2half2_rn((p0 - hf.x) * SP_LO, (p1 - hf.y) * SP_LO);
          p_hi[u] = *reinterpret_cast<const uint32_t*>(&h);
          p_lo[u] = *reinterpret_cast<const uint32_t*>(&lo);
        }
        st.l = fmaf(sum, back, st.l);
        copies_wait<1>();  // the values
        __syncwarp();
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
          uint4 v[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int r = 2 * c + (u & 1) + 8 * (u >> 1);
            v[u] = *reinterpret_cast<const uint4*>(vbuf + r * ROWB + value_piece(r, 8 * j + g) * 16);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {  // column n of tile (j, e) is dim 64 j + 8 n + e
            const uint32_t b0 = __byte_perm(word(v[0], e / 2), word(v[1], e / 2), e & 1 ? 0x7632 : 0x5410);
            const uint32_t b1 = __byte_perm(word(v[2], e / 2), word(v[3], e / 2), e & 1 ? 0x7632 : 0x5410);
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            mma_f16(d, p_hi[0], p_lo[0], p_hi[1], p_lo[1], b0, b1);
            st.acc[8 * j + e][0] = fmaf(fmaf(d[2], 1.f / SP_LO, d[0]), back, st.acc[8 * j + e][0]);
            st.acc[8 * j + e][1] = fmaf(fmaf(d[3], 1.f / SP_LO, d[1]), back, st.acc[8 * j + e][1]);
          }
        }
      } else {
        const float p0 = exp2f(s[0] - base), p1 = exp2f(s[1] - base);
        st.l += p0 + p1;
        uint32_t h0w, l0w, h1w, l1w;
        tf32_pair(p0, h0w, l0w);
        tf32_pair(p1, h1w, l1w);
        copies_wait<1>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          uint4 v[2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
            v[u] = *reinterpret_cast<const uint4*>(vbuf + (2 * c + u) * ROWB +
                                                   value_piece(2 * c + u, 8 * j + g) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // column n of tile (j, e) is dim 32 j + 4 n + e
            uint32_t vh0, vl0, vh1, vl1;
            tf32_pair(__uint_as_float(word(v[0], e)), vh0, vl0);
            tf32_pair(__uint_as_float(word(v[1], e)), vh1, vl1);
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            mma_tf32(d, h0w, l0w, h1w, l1w, vl0, vl1);
            mma_tf32(d, h0w, l0w, h1w, l1w, vh0, vh1);
            st.acc[4 * j + e][0] += d[0] + d[2];
            st.acc[4 * j + e][1] += d[1] + d[3];
          }
        }
      }
      __syncwarp();
      if (more)
        copy_rows(v_lane, vbuf, off_next, nv_next, false);
      else
        copies_commit();
#pragma unroll
      for (int u = 0; u < NB; ++u) nv[u] = nv_next[u];
    }
    copies_wait<0>();
    __syncthreads();  // every warp is done with its buffer, where the outputs go now
    // ---- join: this CTA's warps ----
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
    if (c == 0) wm[warp][g] = st.m, wl[warp][g] = st.l;
    // Outputs stay in accumulator order, 4 at a time: piece (slot, lane) with slot = (j, k, e / 4) is dims
    // 8 E j + (2 c + k) E + e .. + 3 of head g (lane = 4 g + c), so that every access below is 16 bytes a lane in a row.
    constexpr int E = HALF ? 8 : 4;  // column n of tile E j + e is dim 8 E j + E n + e
    constexpr int PIECES = SP_HEADS * HD / 4;
    float4* so4 = reinterpret_cast<float4*>(so);
    float4* part4 = reinterpret_cast<float4*>(part);
#pragma unroll
    for (int j = 0; j < HD / (8 * E); ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          float4 o;
          o.x = st.acc[E * j + e][k];
          o.y = st.acc[E * j + e + 1][k];
          o.z = st.acc[E * j + e + 2][k];
          o.w = st.acc[E * j + e + 3][k];
          so4[warp * PIECES + (((j * 2 + k) * (E / 4) + e / 4) * 32 + lane)] = o;
        }
    auto store = [&](int i, float4 O, float L) {  // piece i of the result
      const int h = (i & 31) >> 2;
      if (h >= heads) return;
      const int slot = i >> 5, j = slot / (2 * (E / 4)), k = slot / (E / 4) % 2, e = slot % (E / 4) * 4;
      float* to = out + (size_t)(h0 + h) * HD + 8 * E * j + (2 * (i & 3) + k) * E + e;
      const float d = L == 0.f ? 1.f : L;  // 0: none of the row's pages exists, and O is 0
      O = make_float4(O.x / d, O.y / d, O.z / d, O.w / d);
      if (wide)
        *reinterpret_cast<float4*>(to) = O;
      else
        to[0] = O.x, to[1] = O.y, to[2] = O.z, to[3] = O.w;
    };
    __syncthreads();
    for (int i = tid; i < PIECES; i += SP_THREADS) {
      const int h = (i & 31) >> 2;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < SP_WARPS; ++w) M = fmaxf(M, wm[w][h]);
      const float base = M == -INFINITY ? 0.f : M;  // no token: the factors are exp2(-inf) = 0, and a NaN stays one
      float L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < SP_WARPS; ++w) {
        const float f = exp2f(wm[w][h] - base);
        const float4 o = so4[w * PIECES + i];
        L = fmaf(wl[w][h], f, L);
        O.x = fmaf(o.x, f, O.x), O.y = fmaf(o.y, f, O.y), O.z = fmaf(o.z, f, O.z), O.w = fmaf(o.w, f, O.w);
      }
      if (S == 1) {
        store(i, O, L);
      } else {
        part4[i] = O;
        if (i < 32 && (i & 3) == 0) pm[h] = M, pl[h] = L;
      }
    }
    if (S == 1) continue;
    // ---- and the cluster's CTAs, each of them a share of the outputs ----
    cluster.sync();
    for (int i = rank * SP_THREADS + tid; i < PIECES; i += S * SP_THREADS) {
      const int h = (i & 31) >> 2;
      if (h >= heads) continue;
      float M = -INFINITY;
#pragma unroll
      for (int r = 0; r < SP_CLUSTER; ++r)
        if (r < S) M = fmaxf(M, cluster.map_shared_rank(pm, r)[h]);
      const float base = M == -INFINITY ? 0.f : M;
      float L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int r = 0; r < SP_CLUSTER; ++r) {
        if (r >= S) break;
        const float f = exp2f(cluster.map_shared_rank(pm, r)[h] - base);
        const float4 o = cluster.map_shared_rank(part4, r)[i];
        L = fmaf(cluster.map_shared_rank(pl, r)[h], f, L);
        O.x = fmaf(o.x, f, O.x), O.y = fmaf(o.y, f, O.y), O.z = fmaf(o.z, f, O.z), O.w = fmaf(o.w, f, O.w);
      }
      store(i, O, L);
    }
    cluster.sync();  // no CTA leaves, or writes its state again, while another reads it
  }
}

template <int HD, bool HALF>
int launch(const SparseAttnArgs& a, cudaStream_t s) {
  SparseDev d;
  d.a = a;
  d.cap_pages = (int)std::min<long long>(((long long)a.max_ctx + a.page_size - 1) / a.page_size, a.max_pages);
  const long long pairs = (long long)a.batch * a.hkv;
  // CTAs per pair: as many as are all resident at once, one an SM, since each pays a chain of about 10 us (lengths, ids,
  // threshold, joins) whatever its share.  A cluster lives in one GPC, so the 148 SMs hold 14 clusters of 8, 32 of 4
  // and 74 of 2; one more starts a second wave.  Sequences of 8k tokens, 64 pages: 14 pairs 14.1 us with 8 CTAs each,
  // 15.1 with 4; 18 pairs 26.6 and 15.4; 32 pairs (16k, 128 pages) 24.4 and 22.1; 64 pairs 32.4 with 4, 30.2 with 2;
  // 128 pairs 48.6 with 2, 45.2 with 1.
  const int S = pairs <= 14 ? 8 : pairs <= 32 ? 4 : pairs <= 74 ? 2 : 1;
  d.key_words = d.cap_pages > a.budget ? (d.cap_pages + 3) / 4 * 4 : 0;
  d.share = (std::min(a.budget, d.cap_pages) + S - 1) / S;
  size_t smem = (size_t)SP_WARPS * 64 * HD + (size_t)d.key_words * 4 + SP_HEADS * HD * 4 + 16 * (2 * HD + 16) +
                16 * (HALF ? (HD + 8) * 2 : (HD + 4) * 4) + (size_t)d.share * 8;
  d.id_words = smem + (size_t)d.key_words * 4 <= SP_SMEM_MAX ? d.key_words : 0;
  smem += (size_t)d.id_words * 4;
  if (smem > SP_SMEM_MAX || pairs * S > 0x7fffffffLL) return kTooLarge;
  // One CTA an SM is left its registers (8 pairs of 8k tokens 13.9 us so, 16.3 us within the 128 that two CTAs an SM
  // need); more pairs than SMs share them.  Outputs of 256 dims leave room for one only.
  const bool two = HD <= 128 && pairs * S > 148;
  auto kernel = two ? sparse_attn_kernel<HD, HALF, HD <= 128 ? 2 : 1> : sparse_attn_kernel<HD, HALF, 1>;
  if (allow_smem(kernel, smem, SP_SMEM_MAX)) return kCudaError;
  return launch_cluster_pdl(kernel, dim3((unsigned)(pairs * S)), dim3(SP_THREADS), S, smem, s, d) == cudaSuccess
             ? kOk
             : kCudaError;
}

template <bool HALF>
int launch_hd(const SparseAttnArgs& a, cudaStream_t s) {
  switch (a.hd) {
    case 64: return launch<64, HALF>(a, s);
    case 128: return launch<128, HALF>(a, s);
    case 256: return launch<256, HALF>(a, s);
    default: return kUnsupported;
  }
}

}  // namespace

int sparse_attention(const SparseAttnArgs& a, cudaStream_t s) {
  if (a.batch < 0 || a.hq <= 0 || a.hkv <= 0 || a.hq % a.hkv || a.hd <= 0 || a.page_size <= 0 || a.max_pages <= 0 ||
      a.num_pages <= 0 || a.table_rows <= 0 || a.max_ctx < 0)
    return kBadArgument;
  if (a.budget <= 0 || a.sink < 0 || a.recent < 0 || (long long)a.sink + a.recent > a.budget) return kBadArgument;
  if (a.batch == 0) return kOk;
  if (!a.q || !a.k_pool || !a.v_pool || !a.bounds || !a.scales || !a.page_table || !a.ctx_len || !a.out || !a.sel)
    return kBadArgument;
  if (!a.rows && a.batch > a.table_rows) return kBadArgument;
  if (((uintptr_t)a.k_pool | (uintptr_t)a.v_pool | (uintptr_t)a.bounds) % 16) return kBadArgument;
  const int vec = a.kv_half ? 8 : 4;  // elements of a 16-byte load
  if (a.page_stride % vec || a.slot_stride % vec || a.head_stride % vec) return kBadArgument;
  if (a.page_size % 8) return kUnsupported;
  if ((long long)a.max_ctx + a.page_size > 1 << 30) return kTooLarge;  // token indices stay within 32 bits
  return a.kv_half ? launch_hd<true>(a, s) : launch_hd<false>(a, s);
}

}  // namespace zc
