// pages.cu -- block tables and slot maps from request lengths, on the device.
//
// The engine's PagedKvCache bookkeeping (PagedKvCache.cs:105-271: a page stack, a table row per sequence) for callers
// whose lengths live on the GPU: a step that decides on the device how many tokens each request adds (speculative
// drafts, sampled stops, padded graphs) gets its pages, slots and positions without a host round trip.
//
//   reserve  request b on table row r: old = len[r], n = max(n_new, 0); more = ceil((old + n) / P) - ceil(old / P)
//            pages, the j-th of them free[count - 1 - (pages of the requests before it) - j]; token t of the step
//            belongs to the request whose [start[b], start[b + 1]) holds it.
//   trim     pages past ceil(min(new, old) / P) go back to the stack, the last request's last page first, so that a
//            reserve taken back leaves the stack as it was.
//
// Both are chains of a few dependent loads (row -> length -> scan -> stack -> store): latency bound at every size that
// a step has, so each is one launch.  A cluster of up to 8 CTAs shares the tokens; every CTA does the whole scan
// (2 loads per request), and the cluster barrier separates these reads from the new lengths and count, which only the
// first CTA writes.  No atomics on global memory: the result does not depend on the order of anything.

#include <cooperative_groups.h>

#include <algorithm>
#include <utility>

#include "batch_ops.h"
#include "common.cuh"

namespace cg = cooperative_groups;

namespace zc {

namespace {

constexpr size_t PG_SMEM_MAX = 220 * 1024;

// Exclusive prefix of v over the block's PG_THREADS threads (red: 33 words); *total gets the sum.
template <int PG_THREADS>
__device__ __forceinline__ long long block_prefix(long long v, long long* red, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    long long w = lane < PG_THREADS / 32 ? red[lane] : 0;
    long long wi = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, wi, o);
      if (lane >= o) wi += u;
    }
    red[lane] = wi - w;
    if (lane == 31) red[32] = wi;
  }
  __syncthreads();
  const long long r = red[warp] + inc - v;
  *total = red[32];
  __syncthreads();
  return r;
}

__device__ __forceinline__ int pages_of(long long tokens, int page) { return (int)((tokens + page - 1) / page); }

// What both kernels keep per request in shared memory.
struct Req {
  int* row;    // table row, -1: not usable (out of range, or a row that an earlier request of the call names)
  int* arg;    // tokens to add, or the length to keep
  int* old;    // tokens stored (trim: pages stored)
  int* first;  // pages stored (reserve) or kept (trim)
  int* poff;   // pages moved by the requests before it (trim: by reverse index, behind it)
  int* start;  // [batch + 1] first token (reserve only)
};

// Table rows, arguments and lengths of the requests: two loads one after the other, whatever else is checked.  A row
// named twice belongs to the first request that names it.
template <int PG_THREADS>
__device__ void load_requests(const PagePool& p, const int32_t* rows, const int32_t* args, int batch, const Req& q,
                              int* owner) {
  for (int b = threadIdx.x; b < batch; b += PG_THREADS) {
    const int r = rows ? rows[b] : b;  // without rows batch <= max_rows
    q.arg[b] = max(args[b], 0);
    const bool in = (unsigned)r < (unsigned)p.max_rows;
    q.row[b] = in ? r : -1;
    q.old[b] = in ? max(p.len[r], 0) : 0;
    if (in && rows) owner[r] = 0x7fffffff;
  }
  __syncthreads();
  if (!rows) return;
  for (int b = threadIdx.x; b < batch; b += PG_THREADS)
    if (q.row[b] >= 0) atomicMin(&owner[q.row[b]], b);
  __syncthreads();
  for (int b = threadIdx.x; b < batch; b += PG_THREADS)
    if (q.row[b] >= 0 && owner[q.row[b]] != b) {
      q.row[b] = -1;
      q.old[b] = 0;
    }
  __syncthreads();
}

// The last i in [0, n) with at[i] <= v (at ascending, at[0] <= v).
__device__ __forceinline__ int find(const int* at, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= v)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <int PG_THREADS>
__global__ void __launch_bounds__(PG_THREADS) reserve_kernel(PagePool p, const int32_t* __restrict__ rows,
                                                               const int32_t* __restrict__ n_new, int batch,
                                                               int tokens, PagePlanOut o) {
  extern __shared__ int sm[];
  __shared__ long long red[33];
  __shared__ int s_used;
  pdl_trigger();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const int P = p.page_size;
  const Req q{sm, sm + batch, sm + 2 * batch, sm + 3 * batch, sm + 4 * batch, sm + 5 * batch};
  const int held = *p.free_count;
  load_requests<PG_THREADS>(p, rows, n_new, batch, q, sm + 6 * batch + 1);
  const int count = min(max(held, 0), p.num_pages);

  // each thread owns `per` consecutive requests
  const int per = (batch + PG_THREADS - 1) / PG_THREADS;
  const int b0 = min(batch, (int)threadIdx.x * per), b1 = min(batch, b0 + per);
  long long sum = 0, total;
  for (int b = b0; b < b1; ++b) sum += q.arg[b];
  long long at = block_prefix<PG_THREADS>(sum, red, &total);
  const long long whole = total;
  long long more = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = q.arg[b], old = q.old[b];
    q.start[b] = (int)min(at, (long long)0x7fffffff);
    at += n;
    const bool fits = q.row[b] >= 0 && (long long)old + n <= min((long long)p.max_pages * P, 0x7fffffffLL) &&
                      at <= tokens;
    const int have = pages_of(old, P);
    q.first[b] = fits ? have : -1;
    if (fits) more += pages_of((long long)old + n, P) - have;
  }
  if (threadIdx.x == 0) q.start[batch] = (int)min(whole, (long long)0x7fffffff);
  if (threadIdx.x == 0) s_used = 0;
  long long off = block_prefix<PG_THREADS>(more, red, &total);
  for (int b = b0; b < b1; ++b) {
    q.poff[b] = (int)min(off, (long long)count);
    if (q.first[b] < 0) continue;
    const int m = pages_of((long long)q.old[b] + q.arg[b], P) - q.first[b];
    off += m;
    if (off > count)
      q.first[b] = -1;  // refused, as every later request, whether it needs a page or not
    else if (m > 0)
      atomicMax(&s_used, (int)off);
  }
  cluster.sync();  // every CTA has read the lengths and the count (and, as a block barrier, filled its shared memory)
  const int used = s_used;  // the granted requests' pages are the first `used` of the prefix

  if (rank == 0) {
    if (threadIdx.x == 0) *p.free_count = count - used;
    for (int b = threadIdx.x; b < batch; b += PG_THREADS) {
      const bool ok = q.first[b] >= 0;
      o.granted[b] = ok;
      o.start[b] = q.start[b];
      if (ok) p.len[q.row[b]] = q.old[b] + q.arg[b];
    }
    if (threadIdx.x == 0) o.start[batch] = q.start[batch];
  }
  const int tid = rank * PG_THREADS + threadIdx.x, step = ranks * PG_THREADS;
  // new pages into the tables: the i-th page popped belongs to the last request whose poff is <= i.  A refused
  // request's poff is at least `used`, a request without new pages is followed by one with the same poff.
  for (unsigned i = tid; i < (unsigned)used; i += step) {
    const int b = find(q.poff, batch, (int)i);
    p.table[(size_t)q.row[b] * p.max_pages + q.first[b] + (i - q.poff[b])] = p.free_list[count - 1 - i];
  }
  // Four tokens a thread: one search, and a page looked up when it changes.
  const bool wide = ((uintptr_t)o.slots | (uintptr_t)o.positions | (uintptr_t)o.token_rows | (uintptr_t)o.ctx_len) % 16 == 0;
  const int all = q.start[batch];
  for (unsigned u = 4 * tid; u < (unsigned)tokens; u += 4 * step) {  // unsigned: 2^31 and a step do not wrap
    const int t = (int)u;
    int64_t slot[4];
    int pos[4], row[4], ctx[4];
    int b = t < all ? find(q.start, batch, t) : batch, col = -1, page = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      slot[i] = -1;
      pos[i] = 0, row[i] = -1, ctx[i] = 0;
      while (b < batch && u + i >= (unsigned)q.start[b + 1]) ++b, col = -1;  // requests without tokens are passed over
      if (b == batch || q.first[b] < 0) continue;
      pos[i] = q.old[b] + (t + i - q.start[b]);
      row[i] = q.row[b];
      ctx[i] = pos[i] + 1;
      if (pos[i] / P != col) {
        col = pos[i] / P;
        const int fresh = col - q.first[b];
        page = fresh < 0 ? p.table[(size_t)row[i] * p.max_pages + col] : p.free_list[count - 1 - (q.poff[b] + fresh)];
      }
      slot[i] = (int64_t)page * P + (pos[i] - col * P);
    }
    if (wide && u + 4 <= (unsigned)tokens) {
      *reinterpret_cast<longlong2*>(o.slots + t) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(o.slots + t + 2) = make_longlong2(slot[2], slot[3]);
      *reinterpret_cast<int4*>(o.positions + t) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(o.token_rows + t) = make_int4(row[0], row[1], row[2], row[3]);
      *reinterpret_cast<int4*>(o.ctx_len + t) = make_int4(ctx[0], ctx[1], ctx[2], ctx[3]);
    } else {
      for (int i = 0; i < 4 && u + i < (unsigned)tokens; ++i) {
        o.slots[t + i] = slot[i];
        o.positions[t + i] = pos[i];
        o.token_rows[t + i] = row[i];
        o.ctx_len[t + i] = ctx[i];
      }
    }
  }
}

template <int PG_THREADS>
__global__ void __launch_bounds__(PG_THREADS) trim_kernel(PagePool p, const int32_t* __restrict__ rows,
                                                            const int32_t* __restrict__ new_len, int batch) {
  extern __shared__ int sm[];
  __shared__ long long red[33];
  pdl_trigger();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const int P = p.page_size;
  const Req q{sm, sm + batch, sm + 2 * batch, sm + 3 * batch, sm + 4 * batch, nullptr};
  const int held = *p.free_count;
  load_requests<PG_THREADS>(p, rows, new_len, batch, q, sm + 5 * batch);
  const int count = min(max(held, 0), p.num_pages);
  const int per = (batch + PG_THREADS - 1) / PG_THREADS;
  const int most = (int)min((long long)p.max_pages * P, 0x7fffffffLL);
  // requests in reverse order: index i is request batch - 1 - i
  const int i0 = min(batch, (int)threadIdx.x * per), i1 = min(batch, i0 + per);
  long long gone = 0, total;
  for (int i = i0; i < i1; ++i) {
    const int b = batch - 1 - i, old = min(q.old[b], most), keep = min(q.arg[b], old);
    q.arg[b] = keep;
    q.old[b] = pages_of(old, P);
    q.first[b] = pages_of(keep, P);
    gone += q.old[b] - q.first[b];
  }
  long long off = block_prefix<PG_THREADS>(gone, red, &total);
  for (int i = i0; i < i1; ++i) {
    const int b = batch - 1 - i;
    q.poff[i] = (int)min(off, 0x7fffffffLL);  // by reverse index: ascending
    off += q.old[b] - q.first[b];
  }
  // a stack never grows past the pool: what a broken table names beyond it is dropped
  const int back = (int)min(total, (long long)(p.num_pages - count));
  cluster.sync();
  if (rank == 0) {
    if (threadIdx.x == 0) *p.free_count = count + back;
    for (int b = threadIdx.x; b < batch; b += PG_THREADS)
      if (q.row[b] >= 0) p.len[q.row[b]] = q.arg[b];
  }
  const int tid = rank * PG_THREADS + threadIdx.x, step = ranks * PG_THREADS;
  const int moved = (int)min(total, 0x7fffffffLL);
  for (unsigned u = tid; u < (unsigned)moved; u += step) {
    const int j = (int)u, i = find(q.poff, batch, j), b = batch - 1 - i;
    int32_t* e = p.table + (size_t)q.row[b] * p.max_pages + (q.old[b] - 1 - (j - q.poff[i]));
    if (j < back) p.free_list[count + j] = *e;
    *e = -1;
  }
}

int check(const PagePool& p, int batch) {
  if (!p.table || !p.len || !p.free_list || !p.free_count || batch < 0) return kBadArgument;
  if (p.max_rows <= 0 || p.max_pages <= 0 || p.num_pages <= 0 || p.page_size <= 0) return kBadArgument;
  return kOk;
}

// A step that one CTA of 256 threads covers in a turn or two (a decode batch) is one, whose barriers are cheap;
// larger ones take up to 8 CTAs of 1024.  64 requests with one token each: 3.7 us against 4.3 with 1024 threads; 256
// requests with 65 thousand tokens: 8 CTAs 9 us, one CTA 27.
struct Shape {
  int threads, cluster;
};
Shape shape_for(int batch, long long items) {
  if (batch <= 256 && items <= 2048) return {256, 1};
  return {1024, items <= 4096 ? 1 : items <= 16384 ? 4 : 8};
}

}  // namespace

int pages_reserve(const PagePool& p, const int32_t* rows, const int32_t* n_new, int batch, int tokens,
                  const PagePlanOut& o, cudaStream_t s) {
  if (const int rc = check(p, batch)) return rc;
  if (tokens < 0 || !o.start || (batch > 0 && (!n_new || !o.granted))) return kBadArgument;
  if (tokens > 0 && (!o.slots || !o.positions || !o.token_rows || !o.ctx_len)) return kBadArgument;
  if (!rows && batch > p.max_rows) return kBadArgument;
  const size_t smem = ((size_t)6 * batch + 1 + (rows ? p.max_rows : 0)) * sizeof(int);
  if (smem > PG_SMEM_MAX) return kTooLarge;
  const Shape f = shape_for(batch, tokens);
  auto kernel = f.threads == 256 ? reserve_kernel<256> : reserve_kernel<1024>;
  if (allow_smem(kernel, smem, PG_SMEM_MAX)) return kCudaError;
  return launch_cluster_pdl(kernel, dim3(f.cluster), dim3(f.threads), f.cluster, smem, s, p, rows, n_new, batch,
                            tokens, o) == cudaSuccess
             ? kOk
             : kCudaError;
}

int pages_trim(const PagePool& p, const int32_t* rows, const int32_t* new_len, int batch, cudaStream_t s) {
  if (const int rc = check(p, batch)) return rc;
  if (batch == 0) return kOk;
  if (!new_len || (!rows && batch > p.max_rows)) return kBadArgument;
  const size_t smem = ((size_t)5 * batch + (rows ? p.max_rows : 0)) * sizeof(int);
  if (smem > PG_SMEM_MAX) return kTooLarge;
  const Shape f = shape_for(batch, (long long)batch * 16);  // the host does not know how many pages go back
  auto kernel = f.threads == 256 ? trim_kernel<256> : trim_kernel<1024>;
  if (allow_smem(kernel, smem, PG_SMEM_MAX)) return kCudaError;
  return launch_cluster_pdl(kernel, dim3(f.cluster), dim3(f.threads), f.cluster, smem, s, p, rows, new_len, batch) ==
                 cudaSuccess
             ? kOk
             : kCudaError;
}

}  // namespace zc
