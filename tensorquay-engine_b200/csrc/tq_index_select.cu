// Index select (tq_index_select): each token's K best rows or pages, in ascending order.
//
// One block a token. A row of scores is read once: a sample of it gives a threshold that a little more
// than K scores reach (how much more: six standard deviations of the sample's count), the row is
// streamed and what reaches the threshold is kept with its position (1 to 2 K candidates), and the K-th
// largest of them is searched by counting, with the candidates in registers. Where too few or too many
// reach the threshold it is moved and the row streamed again; where that does not help (more equal
// scores than candidates fit) the K-th largest is searched by counting over the whole row. Which
// candidates are taken, ties by position, is put into a bitmap of the row, and the bitmap's order is
// the order of the answer; nothing depends on the order in which candidates arrive.
// In the page form the scores are first reduced to a value a page, in shared memory, and the same is
// done with those.
//
// What bounds it: reading the scores (4 bytes a row seen) for many tokens, the chain of loads, counts
// and barriers for few.

#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "tq_contracts.h"
#include "tq_ptx.cuh"

namespace tq {
namespace index_select {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kPageRows = 64;
constexpr int kCandidates = 4096;
constexpr int kHeld = kCandidates / kThreads;  // candidates of a thread
constexpr int kSample = 8;                     // sampled scores of a thread, at a time
constexpr int kMaxSample = 16;
constexpr uint32_t kNever = 0x007FFFFFu;       // key of -inf: this and below is never selected

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
  int words;  // of the bitmap
};

// Scores in their order as whole numbers. (-0 is below 0 here; values are compared as floats, where
// they are equal.)
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

struct Shared {
  int sums[2][kWarps][2];  // block sums, two buffers taken in turn
  int count;
};

// Sums of two numbers over the block, the same in all threads. `turn` flips: one barrier a call.
__device__ __forceinline__ int2 block_sum(Shared& sh, int x, int y, int& turn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  x = __reduce_add_sync(0xFFFFFFFFu, x);
  y = __reduce_add_sync(0xFFFFFFFFu, y);
  if (lane == 0) *reinterpret_cast<int2*>(sh.sums[turn][warp]) = make_int2(x, y);
  __syncthreads();
  const int2 v = lane < kWarps ? *reinterpret_cast<const int2*>(sh.sums[turn][lane]) : make_int2(0, 0);
  turn ^= 1;
  return make_int2(__reduce_add_sync(0xFFFFFFFFu, v.x), __reduce_add_sync(0xFFFFFFFFu, v.y));
}

// A key between two whose counts are known: by the counts at first, then halfway in turn.
__device__ __forceinline__ uint32_t between(uint32_t lo, uint32_t hi, int above_lo, int above_hi,
                                            int want, int round) {
  const uint32_t gap = hi - lo;
  uint32_t step = gap >> 1;
  if (!(round & 1) && above_lo > above_hi)
    step = uint32_t(float(gap) * (float(above_lo - want) / float(above_lo - above_hi)));
  return lo + max(1u, min(step, gap - 1));
}

// What is searched: `want` of the values at x[0, count), of which those outside [lo, hi) are taken
// anyway.
struct Row {
  const float* x;
  int count, lo, hi, want;
};

// Calls fn(values, position of the first, number) for four neighbours at a time, all values of
// [lo, hi) once; the block's threads share them.
template <typename Fn>
__device__ __forceinline__ void each_four(const Row& r, Fn fn) {
  const int head = min(r.hi - r.lo, int((16 - (reinterpret_cast<uintptr_t>(r.x + r.lo) & 15)) & 15) / 4);
  const int body = (r.hi - r.lo - head) / 4, tail = r.hi - r.lo - head - 4 * body;
  const int first = r.lo + head;
  if (threadIdx.x == 0 && head) {
    float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    v.x = r.x[r.lo];
    if (head > 1) v.y = r.x[r.lo + 1];
    if (head > 2) v.z = r.x[r.lo + 2];
    fn(v, r.lo);
  }
  if (threadIdx.x == 32 && tail) {
    const int at = first + 4 * body;
    float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    v.x = r.x[at];
    if (tail > 1) v.y = r.x[at + 1];
    if (tail > 2) v.z = r.x[at + 2];
    fn(v, at);
  }
  const float4* x = reinterpret_cast<const float4*>(r.x + first);
  int i = threadIdx.x;
  for (; i + 3 * kThreads < body; i += 4 * kThreads) {
    float4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = x[i + j * kThreads];
#pragma unroll
    for (int j = 0; j < 4; ++j) fn(v[j], first + 4 * (i + j * kThreads));
  }
  for (; i < body; i += kThreads) fn(x[i], first + 4 * i);
}

__device__ __forceinline__ int reach(const float4& v, float t) {
  return (v.x >= t) + (v.y >= t) + (v.z >= t) + (v.w >= t);
}

// The threshold that about `rank` of the sampled values reach (at least; a tie may bring more).
template <int N>
__device__ __forceinline__ float sample_threshold(Shared& sh, const float* s, int rank, int* turn) {
  uint32_t lo = kNever + 1, hi = 0xFF800001u;  // all finite values and +inf; none
  int above_lo = INT_MAX, above_hi = 0;
  for (int round = 1; hi - lo > 1; ++round) {
    const uint32_t mid = between(lo, hi, above_lo, above_hi, rank, above_lo == INT_MAX ? 1 : round);
    const float t = value_of(mid);
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += s[i] >= t;
    const int above = block_sum(sh, n, 0, *turn).x;
    if (above >= rank) {
      lo = mid;
      above_lo = above;
      if (above <= rank + rank / 16) break;
    } else {
      hi = mid;
      above_hi = above;
    }
  }
  return value_of(lo);
}

__device__ __forceinline__ void mark(uint32_t* map, int i) { atomicOr(&map[i >> 5], 1u << (i & 31)); }

// Streams the row and keeps what reaches `t`; returns how many do (kCandidates of them are kept).
__device__ __forceinline__ int collect(Shared& sh, const Row& r, float t, float* cand_v, int* cand_i) {
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  each_four(r, [&](const float4& v, int at) {
    const int n = reach(v, t);
    if (n == 0) return;
    int to = atomicAdd(&sh.count, n);
    const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (x[j] >= t) {
        if (to < kCandidates) {
          cand_v[to] = x[j];
          cand_i[to] = at + j;
        }
        ++to;
      }
  });
  __syncthreads();
  return sh.count;
}

// Marks the `want` largest of `count` candidates, the lowest positions of equal ones.
__device__ __forceinline__ void mark_best(Shared& sh, const float* cand_v, const int* cand_i, int count,
                                          int want, int end, uint32_t* map, int* turn) {
  float v[kHeld];
  int at[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int j = i * kThreads + int(threadIdx.x);
    v[i] = j < count ? cand_v[j] : -INFINITY;
    at[i] = j < count ? cand_i[j] : INT_MAX;
  }
  float t = -INFINITY;       // all above it
  int last = INT_MAX;        // of those equal to it, up to this position
  bool none_equal = true;
  if (count > want) {
    uint32_t lo = kNever + 1, hi = 0xFF800001u;
    int above_lo = count, above_hi = 0;
    bool exact = false;
    // The range of the candidates' keys first.
    uint32_t least = 0xFFFFFFFFu, most = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (at[i] != INT_MAX) {
        least = min(least, key_of(v[i]));
        most = max(most, key_of(v[i]));
      }
    least = __reduce_min_sync(0xFFFFFFFFu, least);
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    if ((threadIdx.x & 31) == 0)
      *reinterpret_cast<int2*>(sh.sums[*turn][threadIdx.x >> 5]) = make_int2(int(least), int(most));
    __syncthreads();
    {
      const int lane = threadIdx.x & 31;
      const int2 m = *reinterpret_cast<const int2*>(sh.sums[*turn][lane & (kWarps - 1)]);
      lo = __reduce_min_sync(0xFFFFFFFFu, uint32_t(m.x));
      hi = __reduce_max_sync(0xFFFFFFFFu, uint32_t(m.y)) + 1;
      *turn ^= 1;
    }
    for (int round = 0; hi - lo > 1; ++round) {
      const uint32_t mid = between(lo, hi, above_lo, above_hi, want, round);
      const float m = value_of(mid);
      int n = 0;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) n += v[i] >= m;
      const int above = block_sum(sh, n, 0, *turn).x;
      if (above >= want) {
        lo = mid;
        above_lo = above;
        if (above == want) { exact = true; break; }
      } else {
        hi = mid;
        above_hi = above;
      }
    }
    t = value_of(lo);
    none_equal = false;
    if (!exact) {
      // Equal ones: `need` of them with the lowest positions. (As floats: 0 and -0 are equal, so the
      // counts are taken again.)
      int n = 0, m = 0;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        n += v[i] > t;
        m += v[i] == t;
      }
      const int2 both = block_sum(sh, n, m, *turn);
      const int need = want - both.x;
      if (need < both.y) {
        int a = -1, b = end;  // count(<= a) < need <= count(<= b)
        while (b - a > 1) {
          const int mid = a + (b - a) / 2;
          int c = 0;
#pragma unroll
          for (int i = 0; i < kHeld; ++i) c += v[i] == t && at[i] <= mid;
          if (block_sum(sh, c, 0, *turn).x >= need) b = mid; else a = mid;
        }
        last = b;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (at[i] != INT_MAX && (none_equal || v[i] > t || (v[i] == t && at[i] <= last)))
      mark(map, at[i]);
}

// The same over the whole row, for what the candidates do not hold.
__device__ __forceinline__ void mark_best_of_all(Shared& sh, const Row& r, float guess, uint32_t* map,
                                                 int* turn) {
  // The largest key that `want` values reach, if that many are above -inf; else the lowest.
  uint32_t lo = kNever + 1, hi = 0xFF800001u, key = lo;
  float t = value_of(lo);
  int need = 0;
  for (int round = 0;; ++round) {
    const float x = value_of(key);
    int n = 0, m = 0;
    each_four(r, [&](const float4& v, int) {
      m += reach(v, x);
      n += (v.x > x) + (v.y > x) + (v.z > x) + (v.w > x);
    });
    const int2 both = block_sum(sh, n, m, *turn);
    if (round == 0 || both.y >= r.want) {
      lo = key;
      t = x;
      need = r.want - both.x;
      if (need > 0) break;  // what equals t is enough, or all that there is
    } else {
      hi = key;
    }
    if (hi - lo <= 1) break;
    key = lo + (hi - lo) / 2;
    if (round == 0 && key_of(guess) > lo && key_of(guess) < hi) key = key_of(guess);
  }
  // In order, one position a thread at a time.
  for (int i0 = r.lo; i0 < r.hi; i0 += kThreads) {
    const int i = i0 + int(threadIdx.x), lane = threadIdx.x & 31;
    const float v = i < r.hi ? r.x[i] : -INFINITY;
    const bool tie = v == t && v > -INFINITY;
    const unsigned ties = __ballot_sync(0xFFFFFFFFu, tie);
    if (lane == 0) sh.sums[*turn][threadIdx.x >> 5][0] = __popc(ties);
    __syncthreads();
    int before = __popc(ties & ((1u << lane) - 1)), all = 0;
    for (int w = 0; w < kWarps; ++w) {
      const int c = sh.sums[*turn][w][0];
      if (w < int(threadIdx.x >> 5)) before += c;
      all += c;
    }
    *turn ^= 1;
    if (v > t || (tie && before < need)) mark(map, i);
    need -= min(need, all);
  }
}

template <bool kPages>
__global__ void __launch_bounds__(kThreads, 2) index_select_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t raw[];
  float* cand_v = reinterpret_cast<float*>(raw);
  int* cand_i = reinterpret_cast<int*>(cand_v + kCandidates);
  uint32_t* map = reinterpret_cast<uint32_t*>(cand_i + kCandidates);
  float* page_best = reinterpret_cast<float*>(map + a.words);
  __shared__ Shared sh;
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int turn = 0;
  for (int i = tid; i < a.words; i += kThreads) map[i] = 0;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const float* scores = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.scores) + t * a.stride);
  const int s = a.seq_id[t], pos = a.q_pos[t];
  int bad = 0, seen = 0;
  if (s < 0 || s >= a.sequences) {
    bad = TQ_DEV_SEQ_RANGE;
  } else {
    long long n = min((long long)a.kv_len[s], (long long)pos + 1);
    if (kPages) {
      if (n > (long long)a.slots * kPageRows) bad |= TQ_DEV_TABLE_SHORT;
      n = min(n, (long long)a.slots * kPageRows);
    }
    if (n > a.columns) bad |= TQ_DEV_WORK_OVERFLOW;
    seen = int(max(0ll, min(n, (long long)a.columns)));
  }
  if (bad && tid == 0 && a.flags) atomicOr(a.flags, bad);
  Row r;
  r.x = scores;
  r.count = seen;
  if (kPages) {
    // The largest score of each page, 16 lanes a page; NaN does not count.
    r.x = page_best;
    r.count = (seen + kPageRows - 1) / kPageRows;
    const bool aligned = (reinterpret_cast<uintptr_t>(scores) & 15) == 0;
    constexpr int kBatch = 4;
    for (int p0 = 2 * warp + (lane >> 4); (p0 & ~1) < r.count; p0 += 2 * kWarps * kBatch) {
      float4 v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int p = p0 + 2 * kWarps * j, at = p * kPageRows + 4 * (lane & 15);
        v[j] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (aligned && at + 4 <= seen) {
          v[j] = *reinterpret_cast<const float4*>(scores + at);
        } else {
          if (at < seen) v[j].x = scores[at];
          if (at + 1 < seen) v[j].y = scores[at + 1];
          if (at + 2 < seen) v[j].z = scores[at + 2];
          if (at + 3 < seen) v[j].w = scores[at + 3];
        }
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int p = p0 + 2 * kWarps * j;
        float m = fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        if ((lane & 15) == 0 && p < r.count) page_best[p] = m;
      }
    }
  }
  __syncthreads();
  // What is kept anyway is marked, and the rest is searched.
  r.lo = min(a.keep_first, r.count);
  r.hi = max(r.lo, r.count - a.keep_last);
  r.want = a.k - r.lo - (r.count - r.hi);
  for (int i = tid; i < r.lo; i += kThreads) mark(map, i);
  for (int i = r.hi + tid; i < r.count; i += kThreads) mark(map, i);
  const int n = r.hi - r.lo;
  const float lowest = -3.402823466e38f;
  if (n > 0 && r.want > 0) {
    if (n <= kCandidates) {
      const int count = collect(sh, r, lowest, cand_v, cand_i);
      mark_best(sh, cand_v, cand_i, count, r.want, r.hi, map, &turn);
    } else {
      // Sampled in runs of eight neighbours, evenly over the row.
      float x[kMaxSample];
      const int rounds = n > 65536 ? kMaxSample / kSample : 1;
#pragma unroll
      for (int j = 0; j < kMaxSample / kSample; ++j) {
        const int run = j * kThreads + tid;
        const int at = r.lo + int((long long)run * (n - kSample) / (rounds * kThreads));
#pragma unroll
        for (int i = 0; i < kSample; ++i) {
          x[j * kSample + i] = -INFINITY;
          if (j < rounds) {
            const float v = r.x[at + i];
            x[j * kSample + i] = v >= lowest ? v : -INFINITY;  // no NaN
          }
        }
      }
      const float sampled = float(rounds * kThreads * kSample), share = sampled / float(n);
      const float expect = float(r.want) * share;
      float rank = expect + 6.f * sqrtf(expect) + 16.f, t0 = lowest;
      rank = fmaxf(fminf(rank, 0.8f * float(kCandidates) * share), expect + 1.f);
      bool found = false;
      for (int attempt = 0; attempt < 3 && !found; ++attempt) {
        t0 = rank >= sampled ? lowest
             : rounds > 1    ? sample_threshold<kMaxSample>(sh, x, int(rank), &turn)
                             : sample_threshold<kSample>(sh, x, int(rank), &turn);
        const int count = collect(sh, r, t0, cand_v, cand_i);
        if (count <= kCandidates && (count >= r.want || t0 == lowest)) {
          mark_best(sh, cand_v, cand_i, count, r.want, r.hi, map, &turn);
          found = true;
        } else if (count < r.want) {
          rank *= 1.5f * float(r.want) / float(max(count, r.want / 8 + 1));
        } else {
          rank *= 0.75f * float(kCandidates) / float(count);
          if (rank < expect) break;
        }
        __syncthreads();  // sh.count has been read
      }
      if (!found) mark_best_of_all(sh, r, t0, map, &turn);
    }
  }
  __syncthreads();
  // The bitmap in order: each thread numbers a run of its words.
  int* out = reinterpret_cast<int*>(cand_v);  // candidates are no longer needed
  const int words = (r.count + 31) / 32, each = (words + kThreads - 1) / kThreads;
  const int w0 = min(words, tid * each), w1 = min(words, w0 + each);
  int mine = 0;
  for (int w = w0; w < w1; ++w) mine += __popc(map[w]);
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) sh.sums[turn][warp][0] = sum;
  __syncthreads();
  int taken = 0, at = sum - mine;
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) at += taken;
    taken += sh.sums[turn][w][0];
  }
  for (int w = w0; w < w1; ++w)
    for (uint32_t bits = map[w]; bits; bits &= bits - 1) out[at++] = 32 * w + __ffs(bits) - 1;
  __syncthreads();
  int* idx = a.idx + (long long)t * a.k;
  for (int i = tid; i < a.k; i += kThreads) {
    int v = i < taken ? out[i] : -1;
    if (kPages && v >= 0) v = a.page_table[(long long)s * a.slots + v];
    idx[i] = v;
  }
  if (tid == 0) {
    const bool ends = taken > 0 && out[taken - 1] == r.count - 1;
    a.len[t] = kPages ? taken * kPageRows - (ends ? r.count * kPageRows - seen : 0) : taken;
  }
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
  const bool pages = s.page_table.rank != 0;
  const int items = pages ? (a.columns + kPageRows - 1) / kPageRows : a.columns;
  a.words = (items + 31) / 32;
  const uint32_t bytes = kCandidates * 8u + uint32_t(a.words) * 4u + (pages ? uint32_t(items) * 4u : 0u);
  auto kernel = pages ? index_select_kernel<true> : index_select_kernel<false>;
  if (bytes > 48 * 1024 - sizeof(Shared) &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)) != cudaSuccess)
    return fail("launch", TQ_ERR_CUDA);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(s.scores.shape[0]), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) return fail("launch", TQ_ERR_CUDA);
  return fail(nullptr, TQ_OK);
}
