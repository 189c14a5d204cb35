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
//           low bytes in rows 8-15, eight pages as columns.  A page's record goes straight from memory into the
//           operand registers (16 bytes a lane; the contraction index is permuted alike on both sides).
//   select  radix select on the order-preserving bits of the scores, 8 bits a pass, histograms summed over the
//           cluster through distributed shared memory; the chosen pages are handed out in page order.
//   attend  mma m16n8k16 on the raw fp16 keys and values, again from memory into operand registers, with the fp32
//           query as hi + lo halves in rows 0-7 and 8-15 (a power of two of its own brings each head's query into
//           fp16's range) and the fp32 weights split the same way: products are exact and the result is fp32 to about
//           2^-22.  The accumulator layout of q.k is the operand layout of p.v, so nothing is exchanged between
//           lanes but the row maxima.  fp32 pools take the same path with tf32 hi + lo pairs of both sides.
//   join    warps, then the cluster's CTAs, merge their (max, sum, output) states in shared memory.
// Bound: HBM, bytes = pages * (2 hd + 4) + selected tokens * hd * 2 * sizeof(kv) per (row, KV head).

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
constexpr int SP_HEADS = 8;  // query heads per pass: half of an mma's 16 rows
constexpr float SP_LOG2E = 1.4426950408889634f;
constexpr size_t SP_SMEM_MAX = 220 * 1024;

struct SparseDev {
  SparseAttnArgs a;
  int cap_pages;  // pages that max_ctx allows
  int share;      // list entries of a CTA: ceil(budget / S)
  int key_words;  // words of the region that holds a CTA's scores, later the warps' outputs
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

__device__ __forceinline__ uint4 ld_once(const void* p) {
  const int4 v = ld_stream_v4(p);
  return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Unsigned key whose order is the float's (NaN above everything, -0 below 0: callers pass sums that are never -0).
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The score operand of a head tile: rows 0-7 the high bytes of qi, rows 8-15 the low bytes (qi = 256 high + low, both
// signed), columns [min(qi, 0) per dim | max(qi, 0) per dim].  sq: s_q per head, -inf factor handled by the caller.
template <int HD>
__device__ void stage_score_query(const float* q, int heads, int8_t* qs, int stride, float* sq) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;  // one warp per head
  float v[HD / 32], top = 0.f;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) {
    v[i] = warp < heads ? q[warp * HD + lane + 32 * i] : 0.f;
    top = fmaxf(top, fabsf(v[i]));
  }
  top = warp_max(top);
  const float s = __fdiv_rn(top, 32512.f);
  if (lane == 0) sq[warp] = s;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) {
    const int qi = s > 0.f ? min(max(__float2int_rn(__fdiv_rn(v[i], s)), -32512), 32512) : 0;
    const int neg = min(qi, 0), pos = max(qi, 0), d = lane + 32 * i;
    const int8_t nl = (int8_t)(neg & 255), pl = (int8_t)(pos & 255);
    qs[warp * stride + d] = (int8_t)((neg - nl) >> 8);
    qs[(warp + 8) * stride + d] = nl;
    qs[warp * stride + HD + d] = (int8_t)((pos - pl) >> 8);
    qs[(warp + 8) * stride + HD + d] = pl;
  }
}

// The attention operand of a head tile: q * scale * log2(e) * 2^e, hi parts in rows 0-7, lo parts in rows 8-15.
// ex[head] = 2^-e undoes the power of two, which puts the largest |q| of the head at 2^7 .. 2^8.
template <int HD, bool HALF>
__device__ void stage_query(const float* q, int heads, float scale_log2, void* qa, int stride, float* ex) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float v[HD / 32], top = 0.f;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) {
    v[i] = warp < heads ? q[warp * HD + lane + 32 * i] * scale_log2 : 0.f;
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
  if (lane == 0) ex[warp] = down;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) {
    const int d = lane + 32 * i;
    if (HALF) {
      __half* o = reinterpret_cast<__half*>(qa);
      store_hl(o + warp * stride + d, (size_t)8 * stride, v[i] * up);
    } else {
      uint32_t hi, lo;
      tf32_pair(v[i], hi, lo);
      uint32_t* o = reinterpret_cast<uint32_t*>(qa);
      o[warp * stride + d] = hi;
      o[(warp + 8) * stride + d] = lo;
    }
  }
}

// One warp's attention state: rows of the accumulators are heads g (hi products) and g + 8 (lo products).
template <int HD, bool HALF>
struct State {
  static constexpr int NT = HD / 8;
  float acc[NT][4];
  float m, l;  // head lane / 4: running maximum (log2 domain), this lane's share of the sum

  __device__ void init() {
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }
  // The new maximum over the tile's scores (N per lane); rescales what was summed so far.
  template <int N>
  __device__ float raise(const float (&s)[N]) {
    float t = s[0];
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
      for (int i = 0; i < NT; ++i) acc[i][0] *= alpha, acc[i][1] *= alpha, acc[i][2] *= alpha, acc[i][3] *= alpha;
    }
    m = mn;
    return base;
  }
};

template <int HD, bool HALF>
__global__ void __launch_bounds__(SP_THREADS) sparse_attn_kernel(SparseDev dv) {
  const SparseAttnArgs& a = dv.a;
  constexpr int QS = 2 * HD + 16;                    // bytes of a score operand row
  constexpr int QA = HALF ? HD + 8 : HD + 4;         // elements of an attention operand row
  constexpr int ES = HALF ? 2 : 4;
  extern __shared__ __align__(16) unsigned char smem[];
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);              // [key_words]: scores of this CTA's pages,
  float* so = reinterpret_cast<float*>(smem);                      // then [warp][head][HD] outputs
  unsigned char* at = smem + (size_t)dv.key_words * 4;
  float* part = reinterpret_cast<float*>(at);                      // [8][HD] this CTA's output
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
  __shared__ int2 counts;
  __shared__ int s_digit, s_rem, s_all;
  pdl_trigger();
  pdl_wait();

  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), S = cluster.num_blocks();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int g = lane >> 2, c = lane & 3;
  const long long pair = blockIdx.x / S;
  const int b = (int)(pair / a.hkv), kvh = (int)(pair % a.hkv);
  const int P = a.page_size, group = a.hq / a.hkv;
  const int row = a.rows ? a.rows[b] : b;
  int ctx = (unsigned)row < (unsigned)a.table_rows ? max(a.ctx_len[b], 0) : 0;
  const int n = min((ctx + P - 1) / P, dv.cap_pages);
  ctx = min(ctx, (int)min((long long)n * P, 0x7fffffffLL));
  const int want = min(a.budget, n);
  const float* q = a.q + (size_t)b * a.q_stride + (size_t)kvh * group * HD;
  float* out = a.out + ((size_t)b * a.hq + (size_t)kvh * group) * HD;
  int32_t* sel = a.sel + ((size_t)b * a.hkv + kvh) * a.budget;
  for (int i = want + rank * SP_THREADS + tid; i < a.budget; i += S * SP_THREADS) sel[i] = -1;
  if (n == 0) {  // the same for the whole cluster
    for (int i = rank * SP_THREADS + tid; i < group * HD; i += S * SP_THREADS) out[i] = 0.f;
    return;
  }
  const int32_t* pt = a.page_table + (size_t)row * a.max_pages;
  const int share = (want + S - 1) / S;

  if (n <= a.budget) {
    for (int i = rank * share + tid; i < min(want, (rank + 1) * share); i += SP_THREADS) {
      list[i - rank * share] = make_int2(pt[i], i);
      sel[i] = i;
    }
  } else {
    // ---- score ----
    const int cs = (n + S - 1) / S, p_begin = min(n, rank * cs), p_end = min(n, p_begin + cs);
    for (int i = tid; i < 4 * 256; i += SP_THREADS) hist[0][i] = 0;
    constexpr int KS = 2 * HD / 64;  // 16-byte pieces of a record per lane; two k-steps of 32 each
    for (int h0 = 0; h0 < group; h0 += SP_HEADS) {
      const int heads = min(SP_HEADS, group - h0);
      __syncthreads();  // hist cleared, the last tile's operand no longer read
      stage_score_query<HD>(q + (size_t)h0 * HD, heads, qs, QS, sq);
      __syncthreads();
      uint4 ah[KS], al[KS];
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        ah[j] = *reinterpret_cast<const uint4*>(qs + g * QS + 64 * j + 16 * c);
        al[j] = *reinterpret_cast<const uint4*>(qs + (g + 8) * QS + 64 * j + 16 * c);
      }
      const float s_q = sq[g];
      const bool last = h0 + SP_HEADS >= group;
      int ph[2];
      auto page_at = [&](int p) { return p < p_end ? pt[p] : -1; };
      ph[0] = page_at(p_begin + warp * 16 + g);
      ph[1] = page_at(p_begin + warp * 16 + 8 + g);
      for (int p0 = p_begin + warp * 16; p0 < p_end; p0 += SP_WARPS * 16) {
        uint4 r[2][KS];
        float scale[2];
        bool ok[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          ok[u] = (unsigned)ph[u] < (unsigned)a.num_pages;
          const size_t rec = ok[u] ? (size_t)ph[u] * a.hkv + kvh : 0;
          const int8_t* src = a.bounds + rec * (2 * HD) + 16 * c;
#pragma unroll
          for (int j = 0; j < KS; ++j) r[u][j] = ok[u] ? ld_once(src + 64 * j) : make_uint4(0, 0, 0, 0);
          scale[u] = ok[u] && last ? __ldg(a.scales + rec) : 0.f;
        }
        ph[0] = page_at(p0 + SP_WARPS * 16 + g);
        ph[1] = page_at(p0 + SP_WARPS * 16 + 8 + g);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          int d[4] = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            mma_s8(d, ah[j].x, al[j].x, ah[j].y, al[j].y, r[u][j].x, r[u][j].y);
            mma_s8(d, ah[j].z, al[j].z, ah[j].w, al[j].w, r[u][j].z, r[u][j].w);
          }
          // columns (pages) 2c and 2c + 1 of head g; the maximum over the tile's heads
          float f0 = g < heads ? __fmul_rn((float)(d[0] * 256 + d[2]), s_q) : -INFINITY;
          float f1 = g < heads ? __fmul_rn((float)(d[1] * 256 + d[3]), s_q) : -INFINITY;
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            f0 = fmaxf(f0, __shfl_xor_sync(0xffffffffu, f0, o));
            f1 = fmaxf(f1, __shfl_xor_sync(0xffffffffu, f1, o));
          }
          // lanes 4i hold page i's scale and validity; lanes 0-3 take the pages 2c and 2c + 1
          const float c0 = __shfl_sync(0xffffffffu, scale[u], 8 * c), c1 = __shfl_sync(0xffffffffu, scale[u], 8 * c + 4);
          const int v0 = __shfl_sync(0xffffffffu, (int)ok[u], 8 * c), v1 = __shfl_sync(0xffffffffu, (int)ok[u], 8 * c + 4);
          if (g == 0) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int p = p0 + 8 * u + 2 * c + k;
              if (p >= p_end) continue;
              float f = k ? f1 : f0;
              if (h0 > 0) f = fmaxf(f, __uint_as_float(keys[p - p_begin]));
              if (!last) {
                keys[p - p_begin] = __float_as_uint(f);
                continue;
              }
              uint32_t key = order_key(__fmul_rn(f, k ? c1 : c0) + 0.f);  // + 0: -0 orders as 0
              if (!(k ? v1 : v0)) key = 0;
              if (p < a.sink || p >= n - a.recent) key = 0xffffffffu;
              keys[p - p_begin] = key;
              atomicAdd(&hist[0][key >> 24], 1u);
            }
          }
        }
      }
    }
    // ---- select the `want` largest keys ----
    uint32_t prefix = 0, mask = 0;
    int rem = want;
    for (int pass = 0; pass < 4; ++pass) {
      const int shift = 24 - 8 * pass;
      if (pass > 0)
        for (int i = p_begin + tid; i < p_end; i += SP_THREADS) {
          const uint32_t k = keys[i - p_begin];
          if ((k & mask) == prefix) atomicAdd(&hist[pass][(k >> shift) & 255u], 1u);
        }
      cluster.sync();
      const int digit = 255 - tid;  // SP_THREADS == 256: thread 0 has the highest digit
      int tot = 0;
      for (int r = 0; r < S; ++r) tot += (int)cluster.map_shared_rank(&hist[pass][0], r)[digit];
      int inc = tot;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      if (lane == 31) red[0][warp] = inc;
      __syncthreads();
      for (int w = 0; w < warp; ++w) inc += red[0][w];
      if (inc >= rem && inc - tot < rem) {
        s_digit = digit;
        s_rem = rem - (inc - tot);
        s_all = s_rem == tot;
      }
      __syncthreads();
      prefix |= (uint32_t)s_digit << shift;
      mask |= 255u << shift;
      rem = s_rem;
      const bool all = s_all;
      __syncthreads();
      if (all) break;  // every key with this prefix is taken
    }
    // ---- hand them out in page order: keys above the prefix, and the first `rem` equal to it ----
    int gt = 0, eq = 0;
    for (int i = p_begin + tid; i < p_end; i += SP_THREADS) {
      const uint32_t k = keys[i - p_begin] & mask;
      gt += k > prefix;
      eq += k == prefix;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      gt += __shfl_xor_sync(0xffffffffu, gt, o);
      eq += __shfl_xor_sync(0xffffffffu, eq, o);
    }
    if (lane == 0) red[0][warp] = gt, red[1][warp] = eq;
    __syncthreads();
    if (tid == 0) {
      int2 t = make_int2(0, 0);
      for (int w = 0; w < SP_WARPS; ++w) t.x += red[0][w], t.y += red[1][w];
      counts = t;
    }
    cluster.sync();
    int eq_seen = 0, pos = 0;  // before this CTA: keys equal to the prefix, entries handed out
    for (int r = 0; r < rank; ++r) {
      const int2 t = *cluster.map_shared_rank(&counts, r);
      pos += t.x;
      eq_seen += t.y;
    }
    pos += min(eq_seen, rem);
    for (int i0 = p_begin; i0 < p_end; i0 += SP_THREADS) {
      const int i = i0 + tid;
      const uint32_t k = i < p_end ? keys[i - p_begin] & mask : 0u;
      const bool is_eq = i < p_end && k == prefix, is_gt = i < p_end && k > prefix;
      const unsigned beq = __ballot_sync(0xffffffffu, is_eq), bgt = __ballot_sync(0xffffffffu, is_gt);
      __syncthreads();
      if (lane == 0) red[0][warp] = __popc(bgt), red[1][warp] = __popc(beq);
      __syncthreads();
      int before_gt = __popc(bgt & ((1u << lane) - 1u)), before_eq = __popc(beq & ((1u << lane) - 1u));
      int all_gt = 0, all_eq = 0;
      for (int w = 0; w < SP_WARPS; ++w) {
        if (w < warp) before_gt += red[0][w], before_eq += red[1][w];
        all_gt += red[0][w];
        all_eq += red[1][w];
      }
      const int e = eq_seen + before_eq;  // rank among the equal ones
      if (is_gt || (is_eq && e < rem)) {
        const int to = pos + before_gt + min(e, rem) - min(eq_seen, rem);
        sel[to] = i;
        cluster.map_shared_rank(list, to / share)[to % share] = make_int2(pt[i], i);
      }
      pos += all_gt + min(eq_seen + all_eq, rem) - min(eq_seen, rem);
      eq_seen += all_eq;
    }
    cluster.sync();
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
    stage_query<HD, HALF>(q + (size_t)h0 * HD, heads, a.scale * SP_LOG2E, qa, QA, ex);
    __syncthreads();
    const float down = ex[g];
    State<HD, HALF> st;
    st.init();
    const long long row_bytes = a.slot_stride * ES;
    if constexpr (HALF) {
      const __half* qh = reinterpret_cast<const __half*>(qa);
      for (int i0 = warp * 16; i0 < tokens; i0 += SP_WARPS * 16) {
        long long off[2];
        int nv[2];
        nv[0] = locate(i0, off[0]);
        nv[1] = locate(i0 + 8, off[1]);
        uint4 kr[2][HD / 32], vr[4][HD / 64];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < HD / 32; ++j)
            kr[u][j] = g < nv[u] ? ld_once(kb + off[u] + g * row_bytes + 64 * j + 16 * c) : make_uint4(0, 0, 0, 0);
        auto load_v = [&]() {
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < HD / 64; ++j) {
              const int t = 2 * c + (u & 1);
              vr[u][j] = t < nv[u >> 1] ? ld_once(vb + off[u >> 1] + t * row_bytes + 128 * j + 16 * g)
                                        : make_uint4(0, 0, 0, 0);
            }
        };
        if (HD <= 128) load_v();
        float s[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < HD / 32; ++j) {
            const uint4 ah = *reinterpret_cast<const uint4*>(qh + g * QA + 32 * j + 8 * c);
            const uint4 al = *reinterpret_cast<const uint4*>(qh + (g + 8) * QA + 32 * j + 8 * c);
            mma_f16(d, ah.x, al.x, ah.y, al.y, kr[u][j].x, kr[u][j].y);
            mma_f16(d, ah.z, al.z, ah.w, al.w, kr[u][j].z, kr[u][j].w);
          }
          s[2 * u] = 2 * c < nv[u] ? (d[0] + d[2]) * down : -INFINITY;
          s[2 * u + 1] = 2 * c + 1 < nv[u] ? (d[1] + d[3]) * down : -INFINITY;
        }
        if (HD > 128) load_v();  // 256: keys and values do not fit the registers together
        const float base = st.raise(s);
        uint32_t p_hi[2], p_lo[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float p0 = exp2f(s[2 * u] - base), p1 = exp2f(s[2 * u + 1] - base);
          st.l += p0 + p1;
          const __half2 h = __floats2half2_rn(p0, p1);
          const float2 hf = __half22float2(h);
          const __half2 lo = __floats2half2_rn(p0 - hf.x, p1 - hf.y);
          p_hi[u] = *reinterpret_cast<const uint32_t*>(&h);
          p_lo[u] = *reinterpret_cast<const uint32_t*>(&lo);
        }
#pragma unroll
        for (int j = 0; j < HD / 64; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) {  // column n of tile (j, e) is dim 64 j + 8 n + e
            const uint32_t b0 = __byte_perm(word(vr[0][j], e / 2), word(vr[1][j], e / 2), e & 1 ? 0x7632 : 0x5410);
            const uint32_t b1 = __byte_perm(word(vr[2][j], e / 2), word(vr[3][j], e / 2), e & 1 ? 0x7632 : 0x5410);
            mma_f16(st.acc[8 * j + e], p_hi[0], p_lo[0], p_hi[1], p_lo[1], b0, b1);
          }
      }
    } else {
      const uint32_t* qt = reinterpret_cast<const uint32_t*>(qa);
      for (int i0 = warp * 8; i0 < tokens; i0 += SP_WARPS * 8) {
        long long off;
        const int nv = locate(i0, off);
        uint4 kr[HD / 16], vr[2][HD / 32];
#pragma unroll
        for (int j = 0; j < HD / 16; ++j)
          kr[j] = g < nv ? ld_once(kb + off + g * row_bytes + 64 * j + 16 * c) : make_uint4(0, 0, 0, 0);
        auto load_v = [&]() {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < HD / 32; ++j)
              vr[u][j] = 2 * c + u < nv ? ld_once(vb + off + (2 * c + u) * row_bytes + 128 * j + 16 * g)
                                        : make_uint4(0, 0, 0, 0);
        };
        if (HD <= 128) load_v();
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
          const uint4 ah = *reinterpret_cast<const uint4*>(qt + g * QA + 16 * j + 4 * c);
          const uint4 al = *reinterpret_cast<const uint4*>(qt + (g + 8) * QA + 16 * j + 4 * c);
          uint32_t h[4], l[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) tf32_pair(__uint_as_float(word(kr[j], i)), h[i], l[i]);
          mma_tf32(d, ah.x, al.x, ah.y, al.y, h[0], h[1]);
          mma_tf32(d, ah.x, al.x, ah.y, al.y, l[0], l[1]);
          mma_tf32(d, ah.z, al.z, ah.w, al.w, h[2], h[3]);
          mma_tf32(d, ah.z, al.z, ah.w, al.w, l[2], l[3]);
        }
        if (HD > 128) load_v();
        float s[2];
        s[0] = 2 * c < nv ? d[0] + d[2] : -INFINITY;
        s[1] = 2 * c + 1 < nv ? d[1] + d[3] : -INFINITY;
        const float base = st.raise(s);
        const float p0 = exp2f(s[0] - base), p1 = exp2f(s[1] - base);
        st.l += p0 + p1;
        uint32_t h0w, l0w, h1w, l1w;
        tf32_pair(p0, h0w, l0w);
        tf32_pair(p1, h1w, l1w);
#pragma unroll
        for (int j = 0; j < HD / 32; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // column n of tile (j, e) is dim 32 j + 4 n + e
            uint32_t vh0, vl0, vh1, vl1;
            tf32_pair(__uint_as_float(word(vr[0][j], e)), vh0, vl0);
            tf32_pair(__uint_as_float(word(vr[1][j], e)), vh1, vl1);
            mma_tf32(st.acc[4 * j + e], h0w, l0w, h1w, l1w, vh0, vh1);
            mma_tf32(st.acc[4 * j + e], h0w, l0w, h1w, l1w, vl0, vl1);
          }
      }
    }
    // ---- join: this CTA's warps ----
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
    if (c == 0) wm[warp][g] = st.m, wl[warp][g] = st.l;
    constexpr int E = HALF ? 8 : 4;  // tiles whose column n is dims E n + e of a block of 8 E dims
#pragma unroll
    for (int j = 0; j < HD / (8 * E); ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          float4 o;
          o.x = st.acc[E * j + e][k] + st.acc[E * j + e][k + 2];
          o.y = st.acc[E * j + e + 1][k] + st.acc[E * j + e + 1][k + 2];
          o.z = st.acc[E * j + e + 2][k] + st.acc[E * j + e + 2][k + 2];
          o.w = st.acc[E * j + e + 3][k] + st.acc[E * j + e + 3][k + 2];
          *reinterpret_cast<float4*>(so + (warp * SP_HEADS + g) * HD + 8 * E * j + (2 * c + k) * E + e) = o;
        }
    __syncthreads();
    for (int i = tid; i < SP_HEADS * HD; i += SP_THREADS) {
      const int h = i / HD;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < SP_WARPS; ++w) M = fmaxf(M, wm[w][h]);
      const float base = M == -INFINITY ? 0.f : M;  // no token: the factors are exp2(-inf) = 0, and a NaN stays one
      float L = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < SP_WARPS; ++w) {
        const float f = exp2f(wm[w][h] - base);
        L = fmaf(wl[w][h], f, L);
        O = fmaf(so[w * SP_HEADS * HD + i], f, O);
      }
      part[i] = O;
      if (i % HD == 0) pm[h] = M, pl[h] = L;
    }
    // ---- and the cluster's CTAs, each of them a share of the outputs ----
    cluster.sync();
    for (int i = rank * SP_THREADS + tid; i < heads * HD; i += S * SP_THREADS) {
      const int h = i / HD;
      float M = -INFINITY;
      for (int r = 0; r < S; ++r) M = fmaxf(M, cluster.map_shared_rank(pm, r)[h]);
      const float base = M == -INFINITY ? 0.f : M;
      float L = 0.f, O = 0.f;
      for (int r = 0; r < S; ++r) {
        const float f = exp2f(cluster.map_shared_rank(pm, r)[h] - base);
        L = fmaf(cluster.map_shared_rank(pl, r)[h], f, L);
        O = fmaf(cluster.map_shared_rank(part, r)[i], f, O);
      }
      out[(size_t)h0 * HD + i] = L == 0.f ? 0.f : O / L;  // 0: none of the row's pages exists
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
  int S = 1;
  while (S < 8 && pairs * S < 4 * 148) S <<= 1;
  size_t smem = 0;
  for (;; S <<= 1) {  // more CTAs where one CTA's scores would not fit
    const int scored = d.cap_pages > a.budget ? (d.cap_pages + S - 1) / S : 0;
    d.key_words = (std::max(scored, SP_WARPS * SP_HEADS * HD) + 3) / 4 * 4;
    d.share = (std::min(a.budget, d.cap_pages) + S - 1) / S;
    smem = (size_t)d.key_words * 4 + SP_HEADS * HD * 4 + 16 * (2 * HD + 16) + 16 * (HALF ? (HD + 8) * 2 : (HD + 4) * 4) +
           (size_t)d.share * 8;
    if (smem <= SP_SMEM_MAX || S == 8) break;
  }
  if (smem > SP_SMEM_MAX || pairs * S > 0x7fffffffLL) return kTooLarge;
  auto kernel = sparse_attn_kernel<HD, HALF>;
  if (allow_smem(kernel, smem)) return kCudaError;
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
  return a.kv_half ? launch_hd<true>(a, s) : launch_hd<false>(a, s);
}

}  // namespace zc
