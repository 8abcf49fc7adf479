// Step plan (tq_step_plan): from each request's cached and new token counts, the metadata that
// the other entry points of this library take, in one launch:
//   q_start = exclusive sum of new_len            kv_len = cached_len + new_len
//   request s grows from first = ceil(cached / 64) to last = ceil(kv_len / 64) pages; the o-th
//   page that the batch takes (request by request, in page order) is free[count - 1 - o]
//   token t of request s: seq_id = s, q_pos = cached[s] + t - q_start[s],
//   slot = page_table[s][q_pos / 64] * 64 + q_pos % 64
// Whole numbers only, so the result does not depend on timing.
//
// What bounds it: latency. A step moves a few KB (12 bytes a token), so everything happens in
// one launch without a barrier between CTAs. Up to kNear requests every CTA scans all of them
// itself, four a thread, into shared memory; it then writes the results of its share of the
// requests and fills its share of the tokens, finding a token's request by bisection in shared
// memory and a new page in the free stack rather than in the table that another CTA may be writing
// (512 requests with 14841 tokens: 4.4 us on the device, 10.5 with a scan split over a cluster and
// bisection in global memory; 5.6 us a call, 64 decode requests 4.9, 4096 requests 8.3).
// Beyond kNear, clusters of C CTAs split the requests: each CTA sums its share, the CTAs exchange
// their totals through distributed shared memory, scan their share with that base, and after a
// cluster barrier fill the tokens. With more than one cluster, every cluster does the whole scan
// (they write the same values) and the clusters split only the tokens. Back to back 16 us a call for
// 9001 requests with 13469 tokens, 25 for 4097 with 202793 (one request less, and the other form
// takes 8.3), 39 for 65536 with 163416, 15.5 for 300 over 2^19 token rows: three dependent passes
// over the requests, a bisection in global memory for each token, and no programmatic launch.

#include <cuda_runtime.h>

#include <climits>
#include <cstdint>

#include "tq_contracts.h"
#include "tq_ptx.cuh"

namespace tq {
namespace step {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kPage = 64;

struct Args {
  const int* cached;
  const int* fresh;
  const int* free_pages;
  const int* free_count;
  int* table;
  int* q_start;
  int* kv_len;
  int* seq_id;
  int* q_pos;
  int* slot;  // may be null
  int* free_left;
  int* flags;  // may be null
  int requests, columns, tokens, pool;
  int cluster;  // CTAs per cluster
};

struct Count {
  long long tokens, pages;
};

__device__ __forceinline__ Count operator+(Count a, Count b) {
  return {a.tokens + b.tokens, a.pages + b.pages};
}

// One request: its counts, and what is wrong with them.
struct Request {
  long long cached, total;
  int first, last;  // page columns: held, and held after this step
  int bad;
};

__device__ __forceinline__ Request request_of(const Args& a, int s) {
  Request r;
  const int c = a.cached[s], n = a.fresh[s];
  r.bad = (c < 0 || n < 0) ? TQ_DEV_SEQ_RANGE : 0;
  r.cached = c < 0 ? 0 : c;
  r.total = r.cached + (n < 0 ? 0 : n);
  const long long first = (r.cached + kPage - 1) / kPage, last = (r.total + kPage - 1) / kPage;
  if (last > a.columns) r.bad |= TQ_DEV_TABLE_SHORT;
  r.first = int(first < a.columns ? first : a.columns);
  r.last = int(last < a.columns ? last : a.columns);
  return r;
}

__device__ __forceinline__ Count warp_inclusive(Count v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xFFFFFFFFu, v.tokens, o);
    const long long p = __shfl_up_sync(0xFFFFFFFFu, v.pages, o);
    if (lane >= o) v = v + Count{t, p};
  }
  return v;
}

// Exclusive sum of `v` over the block's threads; `total` gets the whole sum.
__device__ __forceinline__ Count block_exclusive(Count v, Count* part, Count* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Count inc = warp_inclusive(v);
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const Count w = warp_inclusive(part[lane]);
    part[lane] = w;
  }
  __syncthreads();
  *total = part[kWarps - 1];
  Count before{0, 0};
  if (warp > 0) before = part[warp - 1];
  const Count out{before.tokens + inc.tokens - v.tokens, before.pages + inc.pages - v.pages};
  __syncthreads();  // part is reused
  return out;
}

// Limits of the near kernel: sums of kNear counts below kNearCount stay within 32 bits.
constexpr int kNear = 4096;
constexpr int kNearCount = 1 << 19;

template <int kN>
struct NearShared {
  uint32_t part[2][32];
  int start[kN + 1];  // first token of each request
  int page[kN + 1];   // pages taken by the requests before it
  int cached[kN];
};

__device__ __forceinline__ uint32_t warp_inclusive(uint32_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// The last i with start[i] <= x, of n ascending ones: of equal ones (empty requests) the last.
__device__ __forceinline__ int last_at_or_below(const int* start, int n, int x) {
  int b = 0, e = n;
  while (e - b > 1) {
    const int m = (b + e) >> 1;
    if (start[m] <= x) b = m; else e = m;
  }
  return b;
}

// kT threads, four consecutive requests each.
template <int kT>
__global__ void __launch_bounds__(kT) near_kernel(const Args a) {
  constexpr int kN = 4 * kT, kW = kT / 32;
  extern __shared__ __align__(16) uint8_t raw[];
  NearShared<kN>& sh = *reinterpret_cast<NearShared<kN>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Launched while the kernel before it ends; its results are waited for here.
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int pool = min(max(*a.free_count, 0), a.pool);
  int bad = 0;
  Request r[4];
  uint32_t tokens = 0, pages = 0;  // of this thread's requests, then before them
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = {0, 0, 0, 0, 0};
    if (4 * tid + i < a.requests) r[i] = request_of(a, 4 * tid + i);
    tokens += uint32_t(min(r[i].total - r[i].cached, (long long)a.tokens + 1));
    pages += uint32_t(r[i].last - r[i].first);
  }
  const uint32_t own_tokens = tokens, own_pages = pages;
  tokens = warp_inclusive(tokens);
  pages = warp_inclusive(pages);
  if (lane == 31) {
    sh.part[0][warp] = tokens;
    sh.part[1][warp] = pages;
  }
  __syncthreads();
  // Every warp sums the warps' totals itself: one barrier instead of three.
  const uint32_t t_warp = warp_inclusive(lane < kW ? sh.part[0][lane] : 0u);
  const uint32_t p_warp = warp_inclusive(lane < kW ? sh.part[1][lane] : 0u);
  const uint32_t all_tokens = __shfl_sync(0xFFFFFFFFu, t_warp, kW - 1);
  const uint32_t all_pages = __shfl_sync(0xFFFFFFFFu, p_warp, kW - 1);
  const uint32_t t_before = __shfl_sync(0xFFFFFFFFu, t_warp, (warp + 31) & 31);
  const uint32_t p_before = __shfl_sync(0xFFFFFFFFu, p_warp, (warp + 31) & 31);
  tokens += (warp ? t_before : 0u) - own_tokens;
  pages += (warp ? p_before : 0u) - own_pages;
  const int real = int(min(all_tokens, uint32_t(a.tokens)));
  // This CTA's share of the requests' own results.
  const int share = (a.requests + int(gridDim.x) - 1) / int(gridDim.x);
  const int lo = int(blockIdx.x) * share, hi = min(a.requests, lo + share);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = 4 * tid + i;
    const int need = r[i].last - r[i].first;
    if (s < a.requests) {
      const int start = int(min(tokens, uint32_t(a.tokens)));
      sh.start[s] = start;
      sh.page[s] = int(pages);
      sh.cached[s] = int(r[i].cached);
      if (s >= lo && s < hi) {
        const int left = pool - int(min(pages, uint32_t(INT_MAX)));
        const int got = left >= need ? need : max(left, 0);
        long long len = min(r[i].total, (long long)INT_MAX);
        // Pages held bound what the cache can hold: a short table or an empty pool cuts kv_len.
        if (got < need || (r[i].bad & TQ_DEV_TABLE_SHORT))
          len = min(len, (long long)kPage * (r[i].first + got));
        if (got < need) bad |= TQ_DEV_POOL_EMPTY;
        bad |= r[i].bad;
        a.q_start[s] = start;
        a.kv_len[s] = int(len);
      }
    }
    tokens += uint32_t(min(r[i].total - r[i].cached, (long long)a.tokens + 1));
    pages += uint32_t(need);
  }
  if (tid == 0) {
    sh.start[a.requests] = real;
    sh.page[a.requests] = int(all_pages);
    if (blockIdx.x == 0) {
      a.q_start[a.requests] = real;
      *a.free_left = pool - int(min(all_pages, uint32_t(pool)));
      if (all_tokens > uint32_t(a.tokens)) bad |= TQ_DEV_WORK_OVERFLOW;
    }
  }
  __syncthreads();

  // The new pages.
  const long long step = (long long)gridDim.x * kT, me = (long long)blockIdx.x * kT + tid;
  for (long long o64 = me; o64 < all_pages; o64 += step) {
    const int o = int(o64), s = last_at_or_below(sh.page, a.requests, o);
    const int held = sh.cached[s] / kPage + (sh.cached[s] % kPage != 0);
    const int col = held + o - sh.page[s];
    a.table[(long long)s * a.columns + col] = o < pool ? a.free_pages[pool - 1 - o] : -1;
  }

  // The tokens, four consecutive ones a thread where they are many.
  const bool wide = ((reinterpret_cast<uintptr_t>(a.seq_id) | reinterpret_cast<uintptr_t>(a.q_pos) |
                      reinterpret_cast<uintptr_t>(a.slot)) & 15) == 0;
  for (long long t64 = 4 * me; t64 < a.tokens; t64 += 4 * step) {
    const int t0 = int(t64);
    int seq[4], pos[4], slot[4];
    int b = t0 < real ? last_at_or_below(sh.start, a.requests, t0) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = t0 + i;
      seq[i] = pos[i] = slot[i] = -1;
      if (t >= real) continue;
      while (sh.start[b + 1] <= t) ++b;  // start[requests] = real > t
      const int cached = sh.cached[b];
      const long long p = (long long)cached + (t - sh.start[b]), col = p / kPage;
      seq[i] = b;
      pos[i] = int(min(p, (long long)INT_MAX));
      if (col < a.columns) {
        const int first = cached / kPage + (cached % kPage != 0);
        int page = -1;
        if (col < first) {
          page = a.table[(long long)b * a.columns + col];
        } else {
          // A new page: from the stack, since another CTA may still be writing the table.
          const long long o = (long long)sh.page[b] + col - first;
          if (o < pool) page = a.free_pages[pool - 1 - o];
        }
        const long long at = (long long)page * kPage + p % kPage;
        if (page >= 0 && at <= INT_MAX) slot[i] = int(at);
        if (at > INT_MAX) bad |= TQ_DEV_PAGE_RANGE;
      }
    }
    if (wide && t64 + 4 <= a.tokens) {
      *reinterpret_cast<int4*>(a.seq_id + t0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
      *reinterpret_cast<int4*>(a.q_pos + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      if (a.slot)
        *reinterpret_cast<int4*>(a.slot + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (t64 + i >= a.tokens) break;
        a.seq_id[t0 + i] = seq[i];
        a.q_pos[t0 + i] = pos[i];
        if (a.slot) a.slot[t0 + i] = slot[i];
      }
    }
  }
  if (bad && a.flags) atomicOr(a.flags, bad);
}

template <int kT>
cudaError_t launch_near(const Args& a, cudaStream_t stream) {
  long long ctas = (a.tokens + 4ll * kT - 1) / (4 * kT);
  ctas = ctas < 1 ? 1 : ctas > 296 ? 296 : ctas;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas), 1, 1);
  cfg.blockDim = dim3(kT, 1, 1);
  cfg.dynamicSmemBytes = sizeof(NearShared<4 * kT>);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, near_kernel<kT>, a);
}

__global__ void __launch_bounds__(kThreads) plan_kernel(const Args a) {
  __shared__ Count part[kWarps];
  __shared__ Count mine;  // this CTA's totals, read by its cluster
  const int tid = threadIdx.x, lane = tid & 31;
  const int rank = int(ptx::cluster_rank());
  const int share = (a.requests + a.cluster - 1) / a.cluster;
  const int lo = min(a.requests, rank * share), hi = min(a.requests, lo + share);
  const long long pool = min(max(*a.free_count, 0), a.pool);
  int bad = 0;

  // Totals of the shares before this CTA's.
  Count base{0, 0};
  {
    Count sum{0, 0}, total;
    for (int s = lo + tid; s < hi; s += kThreads) {
      const Request r = request_of(a, s);
      sum = sum + Count{r.total - r.cached, r.last - r.first};
    }
    block_exclusive(sum, part, &total);
    if (tid == 0) mine = total;
    ptx::cluster_sync();
    for (int c = 0; c < rank; ++c) {
      const uint32_t at = ptx::map_peer(ptx::smem_addr(&mine), uint32_t(c));
      base.tokens += ptx::ld_cluster_s64(at);
      base.pages += ptx::ld_cluster_s64(at + 8);
    }
  }

  // This CTA's share in request order, kThreads requests at a time.
  for (int s0 = lo; s0 < hi; s0 += kThreads) {
    const int s = s0 + tid;
    Request r{0, 0, 0, 0, 0};
    if (s < hi) r = request_of(a, s);
    Count total;
    const Count at =
        base + block_exclusive(Count{r.total - r.cached, r.last - r.first}, part, &total);
    base = base + total;
    const int need = r.last - r.first;
    const long long left = pool - at.pages;
    const int got = left >= need ? need : int(left > 0 ? left : 0);
    if (s < hi) {
      a.q_start[s] = int(min(at.tokens, (long long)a.tokens));
      // Pages held bound what the cache can hold: a short table or an empty pool cuts kv_len.
      long long len = min(r.total, (long long)INT_MAX);
      const long long room = (long long)kPage * (r.first + got);
      if (got < need || (r.bad & TQ_DEV_TABLE_SHORT)) len = min(len, room);
      a.kv_len[s] = int(len);
      if (got < need) bad |= TQ_DEV_POOL_EMPTY;
      bad |= r.bad;
    }
    // The pages: a warp fills the new columns of its requests one request after the other.
    unsigned grows = __ballot_sync(0xFFFFFFFFu, need > 0);
    while (grows) {
      const int src = __ffs(grows) - 1;
      grows &= grows - 1;
      const int row = __shfl_sync(0xFFFFFFFFu, s, src);
      const int first = __shfl_sync(0xFFFFFFFFu, r.first, src);
      const int n = __shfl_sync(0xFFFFFFFFu, need, src);
      const int have = __shfl_sync(0xFFFFFFFFu, got, src);
      const long long o = __shfl_sync(0xFFFFFFFFu, at.pages, src);
      int* dst = a.table + (long long)row * a.columns + first;
      for (int k = lane; k < n; k += 32) dst[k] = k < have ? a.free_pages[pool - 1 - o - k] : -1;
    }
  }
  // The last CTA with a share ends at the batch's totals.
  if (rank == a.cluster - 1 && tid == 0) {
    a.q_start[a.requests] = int(min(base.tokens, (long long)a.tokens));
    *a.free_left = int(pool > base.pages ? pool - base.pages : 0);
    if (base.tokens > a.tokens) bad |= TQ_DEV_WORK_OVERFLOW;
  }
  ptx::cluster_sync();

  // Tokens, over all CTAs of the grid.
  const int real = a.q_start[a.requests];
  for (long long t64 = (long long)blockIdx.x * kThreads + tid; t64 < a.tokens;
       t64 += (long long)gridDim.x * kThreads) {
    const int t = int(t64);
    int seq = -1, pos = -1, slot = -1;
    if (t < real) {
      // The last request that starts at or before t (requests without tokens are passed over).
      int b = 0, e = a.requests;
      while (e - b > 1) {
        const int m = (b + e) >> 1;
        if (a.q_start[m] <= t) b = m; else e = m;
      }
      seq = b;
      const int c = a.cached[seq];
      const long long p = (long long)(c < 0 ? 0 : c) + (t - a.q_start[seq]);
      pos = int(min(p, (long long)INT_MAX));
      const long long col = p / kPage;
      if (col < a.columns) {
        const int page = a.table[(long long)seq * a.columns + col];
        const long long at = (long long)page * kPage + p % kPage;
        if (page >= 0 && at <= INT_MAX) slot = int(at);
        if (at > INT_MAX) bad |= TQ_DEV_PAGE_RANGE;
      }
    }
    a.seq_id[t] = seq;
    a.q_pos[t] = pos;
    if (a.slot) a.slot[t] = slot;
  }
  if (bad && a.flags) atomicOr(a.flags, bad);
}

}  // namespace step
}  // namespace tq

extern "C" int32_t tq_step_plan(const TqStepPlanSpec* spec, int32_t* device_flags, void* stream,
                                TqContractError* err) {
  using namespace tq::step;
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  const int32_t st = tq::step_plan_validate(spec, err);
  if (st != TQ_OK) return st;
  const TqStepPlanSpec& s = *spec;
  auto ints = [](const TqTensorSpec& t) { return reinterpret_cast<int*>(t.device_address); };
  Args a;
  a.cached = ints(s.cached_len);
  a.fresh = ints(s.new_len);
  a.free_pages = ints(s.free_pages);
  a.free_count = ints(s.free_count);
  a.table = ints(s.page_table);
  a.q_start = ints(s.q_start);
  a.kv_len = ints(s.kv_len);
  a.seq_id = ints(s.seq_id);
  a.q_pos = ints(s.q_pos);
  a.slot = s.slot.rank ? ints(s.slot) : nullptr;
  a.free_left = ints(s.free_left);
  a.flags = device_flags;
  a.requests = int(s.cached_len.shape[0]);
  a.columns = int(s.page_table.shape[1]);
  a.tokens = int(s.seq_id.shape[0]);
  a.pool = int(s.free_pages.shape[0]);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (a.requests <= kNear && a.tokens < kNearCount && a.columns < kNearCount) {
    // A quarter of the threads where that many hold the requests: fewer to start and to wait for.
    // (The larger form's shared memory passes the 48 KB of a plain launch; its 1024 threads of 56
    // registers are one CTA an SM, and at kNearCount token rows it has 128 of them.)
    cudaError_t e;
    if (a.requests <= kNear / 4) {
      e = launch_near<kThreads / 4>(a, cs);
    } else {
      static_assert(sizeof(NearShared<kNear>) <= 232448, "shared memory per CTA");
      e = cudaFuncSetAttribute(near_kernel<kThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               int(sizeof(NearShared<kNear>)));
      if (e == cudaSuccess) e = launch_near<kThreads>(a, cs);
    }
    if (e != cudaSuccess) return fail("launch", TQ_ERR_CUDA);
    return fail(nullptr, TQ_OK);
  }
  a.cluster = 8;
  const long long per_cluster = 8ll * kThreads * 4;
  long long clusters = (a.tokens + per_cluster - 1) / per_cluster;
  if (clusters < 1) clusters = 1;
  if (clusters > 16) clusters = 16;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(clusters * a.cluster), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = cs;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = unsigned(a.cluster);
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, plan_kernel, a) != cudaSuccess) return fail("launch", TQ_ERR_CUDA);
  return fail(nullptr, TQ_OK);
}
