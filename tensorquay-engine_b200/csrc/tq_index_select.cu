// Index select (tq_index_select): each token's K best rows or pages, in ascending order.

#include <cuda_runtime.h>

#include <cstdint>

#include "tq_contracts.h"
#include "tq_ptx.cuh"

namespace tq {
namespace index_select {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPageRows = 64;

struct Args {
  const float* scores;
  const int* seq_id;
  const int* q_pos;
  const int* kv_len;
  const int* page_table;  // null: row form
  int* idx;
  int* len;
  int* flags;
  long long stride;  // bytes between rows of scores
  int columns, sequences, slots, k, keep_first, keep_last;
};

// Order of the selection as a whole number: larger scores larger, -0 as 0; 0 is never selected.
__device__ __forceinline__ uint32_t key_of(float v) {
  uint32_t u = __float_as_uint(v);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u || u == 0xFF800000u) return 0;  // NaN, -inf
  if (u == 0x80000000u) u = 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Row {
  const float* scores;
  const int* pages;  // of the token's sequence (page form)
  int seen;          // rows that the token sees
  int count;         // of them, or of their pages
};

// Candidate i's key.
__device__ __forceinline__ uint32_t key_at(const Args& a, const Row& r, int i) {
  if (i < a.keep_first || i >= r.count - a.keep_last) return 0xFFFFFFFFu;
  if (!a.page_table) return key_of(r.scores[i]);
  uint32_t best = 0;
  const int end = min(r.seen, (i + 1) * kPageRows);
  for (int n = i * kPageRows; n < end; ++n) best = max(best, key_of(r.scores[n]));
  return best;
}

__device__ __forceinline__ int block_inclusive(int v, int* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) part[warp] = v;
  __syncthreads();
  for (int i = 0; i < warp; ++i) v += part[i];
  __syncthreads();
  return v;
}

__global__ void __launch_bounds__(kThreads) index_select_kernel(const Args a) {
  __shared__ int hist[256];
  __shared__ int part[kWarps];
  __shared__ uint32_t found[2];  // digit, candidates above it
  const int t = blockIdx.x, tid = threadIdx.x;
  int* idx = a.idx + (long long)t * a.k;
  Row r = {reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.scores) + t * a.stride),
           nullptr, 0, 0};
  const int s = a.seq_id[t];
  int bad = 0;
  if (s < 0 || s >= a.sequences) {
    bad = TQ_DEV_SEQ_RANGE;
  } else {
    long long n = min((long long)a.kv_len[s], (long long)a.q_pos[t] + 1);
    if (a.page_table) {
      r.pages = a.page_table + (long long)s * a.slots;
      if (n > (long long)a.slots * kPageRows) bad |= TQ_DEV_TABLE_SHORT;
      n = min(n, (long long)a.slots * kPageRows);
    }
    if (n > a.columns) bad |= TQ_DEV_WORK_OVERFLOW;
    r.seen = int(max(0ll, min(n, (long long)a.columns)));
    r.count = a.page_table ? (r.seen + kPageRows - 1) / kPageRows : r.seen;
  }
  if (bad && tid == 0 && a.flags) atomicOr(a.flags, bad);

  // The K-th largest key, 8 bits at a time: candidates equal to `prefix` in the bits done.
  uint32_t prefix = 0;
  int need = a.k;  // still to be taken among them
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < r.count; i += kThreads) {
      const uint32_t key = key_at(a, r, i);
      if (shift == 24 || (key ^ prefix) >> (shift + 8) == 0) atomicAdd(&hist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int above = 0, d = 255;
      while (d > 0 && above + hist[d] < need) above += hist[d--];
      found[0] = uint32_t(d);
      found[1] = uint32_t(above);
    }
    __syncthreads();
    prefix |= found[0] << shift;
    need -= int(found[1]);
    __syncthreads();
  }
  // All above it and the first `need` that equal it, in order; keys of 0 never.
  int taken = 0, equal = 0, ends = 0;
  for (int i0 = 0; i0 < r.count; i0 += kThreads) {
    const int i = i0 + tid;
    const uint32_t key = i < r.count ? key_at(a, r, i) : 0;
    const bool tie = key != 0 && key == prefix;
    const int before = block_inclusive(tie, part);
    const bool take = key != 0 && (key > prefix || (tie && equal + before <= need));
    equal += __syncthreads_count(tie);
    const int at = taken + block_inclusive(take, part) - 1;
    if (take) idx[at] = a.page_table ? r.pages[i] : i;
    taken += __syncthreads_count(take);
    ends = __syncthreads_or(take && i == r.count - 1);
  }
  for (int i = taken + tid; i < a.k; i += kThreads) idx[i] = -1;
  if (tid == 0)
    a.len[t] = !a.page_table ? taken : taken * kPageRows - (ends ? r.count * kPageRows - r.seen : 0);
}

}  // namespace index_select
}  // namespace tq

extern "C" int32_t tq_index_select(const TqIndexSelectSpec* spec, int32_t* device_flags,
                                   void* stream, TqContractError* err) {
  using namespace tq::index_select;
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  const int32_t st = tq::index_select_validate(spec, err);
  if (st != TQ_OK) return st;
  const TqIndexSelectSpec& s = *spec;
  if (s.scores.shape[0] == 0) return fail(nullptr, TQ_OK);
  auto ints = [](const TqTensorSpec& t) {
    return t.rank ? reinterpret_cast<int*>(t.device_address) : nullptr;
  };
  Args a = {};
  a.scores = reinterpret_cast<const float*>(s.scores.device_address);
  a.seq_id = ints(s.seq_id);
  a.q_pos = ints(s.q_pos);
  a.kv_len = ints(s.kv_len);
  a.page_table = ints(s.page_table);
  a.idx = ints(s.idx);
  a.len = ints(s.len);
  a.flags = device_flags;
  a.stride = (long long)s.scores.strides_bytes[0];
  a.columns = int(s.scores.shape[1]);
  a.sequences = int(s.kv_len.shape[0]);
  a.slots = s.page_table.rank ? int(s.page_table.shape[1]) : 0;
  a.k = int(s.idx.shape[1]);
  a.keep_first = s.keep_first;
  a.keep_last = s.keep_last;
  index_select_kernel<<<unsigned(s.scores.shape[0]), kThreads, 0,
                        static_cast<cudaStream_t>(stream)>>>(a);
  if (cudaGetLastError() != cudaSuccess) return fail("launch", TQ_ERR_CUDA);
  return fail(nullptr, TQ_OK);
}
