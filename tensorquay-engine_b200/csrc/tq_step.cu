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
// one launch: clusters of C CTAs split the requests, each CTA sums its share, the CTAs exchange
// their totals through distributed shared memory, scan their share with that base, and after a
// cluster barrier fill the tokens. With more than one cluster, every cluster does the whole scan
// (they write the same values) and the clusters split only the tokens, so no grid barrier and no
// workspace are needed.

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

__global__ void __launch_bounds__(kThreads) plan_kernel(const Args a) {
  __shared__ Count part[kWarps];
  __shared__ Count mine;  // this CTA's totals, read by its cluster
  const int tid = threadIdx.x, lane = tid & 31;
  const int rank = a.cluster > 1 ? int(ptx::cluster_rank()) : 0;
  const int share = (a.requests + a.cluster - 1) / a.cluster;
  const int lo = min(a.requests, rank * share), hi = min(a.requests, lo + share);
  const long long pool = min(max(*a.free_count, 0), a.pool);
  int bad = 0;

  // Totals of the shares before this CTA's.
  Count base{0, 0};
  if (a.cluster > 1) {
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
  if (a.cluster > 1)
    ptx::cluster_sync();
  else
    __syncthreads();

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
  // One CTA while one thread per request and four tokens per thread do; then clusters of eight.
  a.cluster = a.requests <= kThreads && a.tokens <= 4 * kThreads ? 1 : 8;
  const long long per_cluster = 8ll * kThreads * 4;
  long long clusters = a.cluster == 1 ? 1 : (a.tokens + per_cluster - 1) / per_cluster;
  if (clusters < 1) clusters = 1;
  if (clusters > 16) clusters = 16;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(clusters * a.cluster), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
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
