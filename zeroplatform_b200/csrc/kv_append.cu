// kv_append.cu -- a step's keys and values into the paged pools through a slot map, with 8-bit bounds of the keys of
// every page they touch.
//
// PagedKvCache.AppendTokenAt (PagedKvCache.cs:149-183) for many sequences at once, on device slots.  The bounds are
// what page-sparse attention scores pages by: over the keys that a page stores, per KV head and dimension,
//   s = max |k| / 127 (fp32, rounded to nearest),   lo = floor(min k / s),   hi = ceil(max k / s),
// so that lo * s <= k <= hi * s (a largest |k| that the rounding of s leaves an ulp outside is clamped to 127).  The
// quotients are floored exactly: the sign of the fused residual tells on which side of an integer the real one lies.
//
// One warp takes all tokens of one page and one head, run by run (consecutive entries in consecutive slots; entries that
// are skipped and gaps between slots may lie between runs): it stores a run, keeps the running min and max in
// registers, adds the keys that the page held before, and writes the codes after the last run.  The keys are therefore
// read once and the bounds need no state of their own, no atomics and no second pass.  Bound: HBM for prompts
// (8 bytes of input and 4 of pool per element with fp32 rows and fp16 pools), latency for single tokens.

#include <math.h>

#include "batch_ops.h"
#include "common.cuh"

namespace zc {

namespace {

constexpr int KA_WARPS = 8;
constexpr int KA_UNROLL = 4;  // token rows of K and V in flight per lane
constexpr int KA_HELD = 8;    // stored keys likewise
constexpr int KA_SKIP = 32;   // windows of 32 slots likewise, over skipped entries

// Four elements of a row as they lie in memory.
template <typename T>
struct Row;
template <>
struct Row<float> {
  float4 v;
};
template <>
struct Row<__half> {
  uint2 v;
};
__device__ __forceinline__ Row<float> fetch(const float* p) { return {*reinterpret_cast<const float4*>(p)}; }
__device__ __forceinline__ Row<__half> fetch(const __half* p) { return {*reinterpret_cast<const uint2*>(p)}; }
__device__ __forceinline__ float4 floats(const Row<float>& r) { return r.v; }
__device__ __forceinline__ float4 floats(const Row<__half>& r) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.v.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.v.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
// Stores v in the pool's type and returns what was stored.
__device__ __forceinline__ float4 store4(float* p, float4 v) {
  *reinterpret_cast<float4*>(p) = v;
  return v;
}
__device__ __forceinline__ float4 store4(__half* p, float4 v) {
  const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
  uint2 u;
  u.x = *reinterpret_cast<const uint32_t*>(&a);
  u.y = *reinterpret_cast<const uint32_t*>(&b);
  *reinterpret_cast<uint2*>(p) = u;
  const float2 c = __half22float2(a), d = __half22float2(b);
  return make_float4(c.x, c.y, d.x, d.y);
}

__device__ __forceinline__ void widen(float4& lo, float4& hi, float4 k) {
  lo.x = fminf(lo.x, k.x), lo.y = fminf(lo.y, k.y), lo.z = fminf(lo.z, k.z), lo.w = fminf(lo.w, k.w);
  hi.x = fmaxf(hi.x, k.x), hi.y = fmaxf(hi.y, k.y), hi.z = fmaxf(hi.z, k.z), hi.w = fmaxf(hi.w, k.w);
}

// floor(x / s) of the real quotient, |x / s| <= 128, clamped to [-127, 127]; inv = 1 / s rounded.  The product is off by
// less than 2^-15, so only an integer next to it can be wrong: fma gives the residual's sign exactly.
__device__ __forceinline__ int floor_code(float x, float s, float inv) {
  float f = floorf(inv > 0.f ? x * inv : __fdiv_rn(x, s));  // 0: s so small that 1 / s may not be finite
  if (__fmaf_rn(-f, s, x) < 0.f) f -= 1.f;
  else if (__fmaf_rn(-(f + 1.f), s, x) >= 0.f) f += 1.f;
  return (int)fminf(fmaxf(f, -127.f), 127.f);
}

template <int HD, typename IN, typename KV>
__global__ void __launch_bounds__(KA_WARPS * 32, 2) kv_append_kernel(KvAppendArgs a, int tile, long long units) {
  constexpr int VEC = HD / 4;                       // 4-element pieces of a row
  constexpr int LPR = VEC < 32 ? VEC : 32;          // lanes per row
  constexpr int ROWS = 32 / LPR;                    // rows a warp takes at once
  constexpr int PCS = VEC / LPR;                    // pieces per lane
  // rows: fp32 rows of 256 dims would spill with as many as 128 take
  constexpr int UNROLL = sizeof(IN) == 4 ? KA_UNROLL / PCS : KA_UNROLL, HELD = KA_HELD / PCS;
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / LPR, col = (lane % LPR) * 4;
  const long long unit = (long long)blockIdx.x * KA_WARPS + warp;  // (token tile, head), heads fastest
  if (unit >= units) return;
  const int h = (int)(unit % a.hkv);
  const int t_begin = (int)(unit / a.hkv) * tile, t_end = min(a.tokens, t_begin + tile);
  const int P = a.page_size;
  const int64_t pool_slots = (int64_t)a.num_pages * P;
  const IN* kin = reinterpret_cast<const IN*>(a.k) + (size_t)h * HD + col;
  const IN* vin = reinterpret_cast<const IN*>(a.v) + (size_t)h * HD + col;

  auto slot_at = [&](int t) -> int64_t {  // -1 where an entry is skipped or there is none
    const int64_t s = (unsigned)t < (unsigned)a.tokens ? a.slots[t] : -1;
    return s < pool_slots ? s : -1;
  };
  // Over skipped entries, which may be many: windows at, at +- 32, .. of 32 entries (at +- lane), up to the first that has
  // an entry; w: that window.  Returns its start, outside [0, tokens) if none.  Padding is negative, which the high
  // words tell: KA_SKIP windows of them are on their way at once.
  auto look = [&](int at, int step, int64_t& w) {
    for (;;) {
      int high[KA_SKIP];
#pragma unroll
      for (int u = 0; u < KA_SKIP; ++u) {
        const int t = at + step * (32 * u + lane);
        high[u] = (unsigned)t < (unsigned)a.tokens ? reinterpret_cast<const int*>(a.slots + t)[1] : -1;
      }
      int first = KA_SKIP;  // this lane's first window with a candidate
#pragma unroll
      for (int u = KA_SKIP - 1; u >= 0; --u)
        if (high[u] >= 0) first = u;
      first = __reduce_min_sync(0xffffffffu, first);
      at += step * 32 * first;
      if ((unsigned)at >= (unsigned)a.tokens) break;
      if (first == KA_SKIP) continue;
      w = slot_at(at + step * lane);
      if (__any_sync(0xffffffffu, w >= 0)) return at;
      at += 32 * step;  // slots behind the pool
    }
    w = -1;
    return at;
  };
  int base = t_begin;
  int64_t win = slot_at(base + lane);  // entries base .. base + 31, one a lane
  int64_t w = slot_at(t_begin - 1 - lane);
  unsigned mine = __ballot_sync(0xffffffffu, win >= 0 && lane < t_end - t_begin);
  if (!mine) return;
  int t = t_begin + __ffs(mine) - 1;
  int64_t slot = __shfl_sync(0xffffffffu, win, t - base);
  // A page belongs to the warp of its first entry: what continues the page of the entry before this tile is not ours.
  if (t_begin > 32 && !__any_sync(0xffffffffu, w >= 0)) look(t_begin - 33, -1, w);
  int page = (int)(slot / P);
  int64_t page0 = (int64_t)page * P;
  if (const unsigned some = __ballot_sync(0xffffffffu, w >= 0)) {
    const int64_t prev = __shfl_sync(0xffffffffu, w, __ffs(some) - 1);
    if ((uint64_t)(prev - page0) < (uint64_t)P) {
      mine &= __ballot_sync(0xffffffffu, (uint64_t)(win - page0) >= (uint64_t)P);
      if (!mine) return;
      t = t_begin + __ffs(mine) - 1;
      slot = __shfl_sync(0xffffffffu, win, t - base);
      page = (int)(slot / P);
      page0 = (int64_t)page * P;
    }
  }
  for (;;) {
    KV* kp = reinterpret_cast<KV*>(a.k_pool) + page * a.page_stride + h * a.head_stride + col;
    KV* vp = reinterpret_cast<KV*>(a.v_pool) + page * a.page_stride + h * a.head_stride + col;
    float4 lo[PCS], hi[PCS];
#pragma unroll
    for (int p = 0; p < PCS; ++p) {
      lo[p] = make_float4(INFINITY, INFINITY, INFINITY, INFINITY);
      hi[p] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
    int seen = 0;  // slots of the page up to here are in lo and hi
    do {
      const int s0 = (int)(slot - page0), most = P - s0;
      int n;  // tokens of this run
      for (;;) {
        const int i = base + lane - t;
        const unsigned in = __ballot_sync(0xffffffffu, i <= 0 || (i < most && win == slot + i));
        n = base - t + __ffs(~in) - 1;
        if (in != 0xffffffffu) break;
        base += 32;
        win = slot_at(base + lane);
      }
      // the run's first rows and the keys that earlier calls stored are on their way together
      Row<IN> kr[UNROLL][PCS], vr[UNROLL][PCS];
      auto load_run = [&](int i0) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          const int i = i0 + u * ROWS;
          if (i < n)
#pragma unroll
            for (int p = 0; p < PCS; ++p) {
              kr[u][p] = fetch(kin + (long long)(t + i) * a.k_stride + p * 128);
              vr[u][p] = fetch(vin + (long long)(t + i) * a.v_stride + p * 128);
            }
        }
      };
      load_run(sub);
      const int end = t + n;  // the next entry, of this page or another
      unsigned some = __ballot_sync(0xffffffffu, win >= 0 && base + lane >= end);
      if (a.bounds)
        for (int i0 = seen + sub; i0 < s0; i0 += ROWS * HELD) {
          Row<KV> hr[HELD][PCS];
#pragma unroll
          for (int u = 0; u < HELD; ++u)
            if (i0 + u * ROWS < s0)
#pragma unroll
              for (int p = 0; p < PCS; ++p) hr[u][p] = fetch(kp + (long long)(i0 + u * ROWS) * a.slot_stride + p * 128);
#pragma unroll
          for (int u = 0; u < HELD; ++u)
            if (i0 + u * ROWS < s0)
#pragma unroll
              for (int p = 0; p < PCS; ++p) widen(lo[p], hi[p], floats(hr[u][p]));
        }
      for (int i0 = sub;;) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          const int i = i0 + u * ROWS;
          if (i < n)
#pragma unroll
            for (int p = 0; p < PCS; ++p) {
              const long long at = (long long)(s0 + i) * a.slot_stride + p * 128;
              widen(lo[p], hi[p], store4(kp + at, floats(kr[u][p])));
              store4(vp + at, floats(vr[u][p]));
            }
        }
        i0 += ROWS * UNROLL;
        if (i0 >= n) break;
        load_run(i0);
      }
      seen = max(seen, s0 + n);
      if (!some && base + 32 < a.tokens) {
        base = look(base + 32, 1, win);
        some = __ballot_sync(0xffffffffu, win >= 0);
      }
      if (!some) {  // no entry is left
        t = a.tokens;
        break;
      }
      t = base + __ffs(some) - 1;
      slot = __shfl_sync(0xffffffffu, win, t - base);
    } while ((uint64_t)(slot - page0) < (uint64_t)P);
    if (a.bounds) {
      float top = 0.f;
#pragma unroll
      for (int p = 0; p < PCS; ++p) {
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) {
          lo[p].x = fminf(lo[p].x, __shfl_xor_sync(0xffffffffu, lo[p].x, o));
          lo[p].y = fminf(lo[p].y, __shfl_xor_sync(0xffffffffu, lo[p].y, o));
          lo[p].z = fminf(lo[p].z, __shfl_xor_sync(0xffffffffu, lo[p].z, o));
          lo[p].w = fminf(lo[p].w, __shfl_xor_sync(0xffffffffu, lo[p].w, o));
          hi[p].x = fmaxf(hi[p].x, __shfl_xor_sync(0xffffffffu, hi[p].x, o));
          hi[p].y = fmaxf(hi[p].y, __shfl_xor_sync(0xffffffffu, hi[p].y, o));
          hi[p].z = fmaxf(hi[p].z, __shfl_xor_sync(0xffffffffu, hi[p].z, o));
          hi[p].w = fmaxf(hi[p].w, __shfl_xor_sync(0xffffffffu, hi[p].w, o));
        }
        top = fmaxf(top, fmaxf(fmaxf(fmaxf(fabsf(lo[p].x), fabsf(lo[p].y)), fmaxf(fabsf(lo[p].z), fabsf(lo[p].w))),
                               fmaxf(fmaxf(fabsf(hi[p].x), fabsf(hi[p].y)), fmaxf(fabsf(hi[p].z), fabsf(hi[p].w)))));
      }
      const float s = __fdiv_rn(warp_max(top), 127.f);
      const float inv = s > 1e-30f ? 1.f / s : 0.f;
      int8_t* codes = a.bounds + ((size_t)page * a.hkv + h) * 2 * HD + col;
      if (sub == 0)
#pragma unroll
        for (int p = 0; p < PCS; ++p) {
          char4 l = make_char4(0, 0, 0, 0), u = l;
          if (s > 0.f && s < INFINITY) {
            l = make_char4(floor_code(lo[p].x, s, inv), floor_code(lo[p].y, s, inv), floor_code(lo[p].z, s, inv),
                           floor_code(lo[p].w, s, inv));
            u = make_char4(-floor_code(-hi[p].x, s, inv), -floor_code(-hi[p].y, s, inv),
                           -floor_code(-hi[p].z, s, inv), -floor_code(-hi[p].w, s, inv));
          }
          *reinterpret_cast<char4*>(codes + p * 128) = l;
          *reinterpret_cast<char4*>(codes + HD + p * 128) = u;
        }
      if (lane == 0) a.scales[(size_t)page * a.hkv + h] = s;
    }
    if (t >= t_end) return;
    page = (int)(slot / P);
    page0 = (int64_t)page * P;
  }
}

template <int HD, typename IN, typename KV>
int launch(const KvAppendArgs& a, cudaStream_t s) {
  // Tokens per warp: it walks its tile's runs one after another, so single tokens while that leaves fewer than 64
  // warps an SM (a decode step), and a common page's worth of a prompt beyond, where most warps of a finer split would
  // find that their token belongs to a page before it.
  const int tile = (long long)a.tokens * a.hkv <= 148 * 64 ? 1 : 16;
  const long long units = (long long)((a.tokens + tile - 1) / tile) * a.hkv;
  const long long blocks = (units + KA_WARPS - 1) / KA_WARPS;
  if (blocks > 0x7fffffffLL) return kTooLarge;
  return launch_pdl(kv_append_kernel<HD, IN, KV>, dim3((unsigned)blocks), dim3(KA_WARPS * 32), 0, s, a, tile,
                    units) == cudaSuccess
             ? kOk
             : kCudaError;
}

template <int HD>
int launch_hd(const KvAppendArgs& a, cudaStream_t s) {
  if (a.half_input) return a.kv_half ? launch<HD, __half, __half>(a, s) : launch<HD, __half, float>(a, s);
  return a.kv_half ? launch<HD, float, __half>(a, s) : launch<HD, float, float>(a, s);
}

}  // namespace

int kv_append(const KvAppendArgs& a, cudaStream_t s) {
  if (a.tokens < 0 || a.hkv <= 0 || a.hd <= 0 || a.page_size <= 0 || a.num_pages <= 0) return kBadArgument;
  if (a.tokens == 0) return kOk;
  if (a.tokens > 0x7fffffff - 4096) return kTooLarge;  // windows of slots reach past the last entry
  if (!a.k || !a.v || !a.slots || !a.k_pool || !a.v_pool || (!a.bounds != !a.scales)) return kBadArgument;
  // 4-element pieces of every row and 4-byte code words
  const size_t ia = a.half_input ? 8 : 16, pa = a.kv_half ? 8 : 16;
  if (((uintptr_t)a.k | (uintptr_t)a.v) % ia || ((uintptr_t)a.k_pool | (uintptr_t)a.v_pool) % pa) return kBadArgument;
  if (a.k_stride % 4 || a.v_stride % 4 || a.page_stride % 4 || a.slot_stride % 4 || a.head_stride % 4)
    return kBadArgument;
  if (a.bounds && ((uintptr_t)a.bounds % 4 || (uintptr_t)a.scales % 4)) return kBadArgument;
  switch (a.hd) {
    case 32: return launch_hd<32>(a, s);
    case 64: return launch_hd<64>(a, s);
    case 128: return launch_hd<128>(a, s);
    case 256: return launch_hd<256>(a, s);
    default: return kUnsupported;
  }
}

}  // namespace zc
