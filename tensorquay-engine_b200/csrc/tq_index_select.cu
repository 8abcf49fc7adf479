// Index select (tq_index_select): each token's K best rows or pages, in ascending order.
//
// One block a token. Up to kDirect scores are held in registers, counted into kBins bins of even width
// between the least and the largest, and the few in the bin that the K-th largest falls into are
// ranked against each other. Of a longer row a sample is counted first, for a threshold that a little
// more than K scores reach (how much more: six standard deviations of the sample's count); the row is
// streamed once, what reaches the threshold is kept with its position (1 to 2 K candidates), and these
// are counted and ranked. Where too few or too many reach the threshold it is moved and the row
// streamed again; where that does not help (more equal scores than candidates fit), and where the bins
// do not tell the values apart, the K-th largest is searched by halving. What is taken, ties by
// position, is put into a bitmap of the row, and the bitmap's order is the order of the answer: nothing
// depends on the order in which candidates arrive.
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
constexpr int kDirect = 8192;
constexpr int kCandidates = 3840;  // (4096 and the bitmap of 2^20 columns do not fit)
constexpr int kSample = 8;      // sampled scores of a thread, at a time
constexpr int kMaxSample = 16;
constexpr int kBins = 1024;     // two a thread
constexpr int kRanked = kThreads / 8;  // scores that are ranked against each other, 8 threads each
static_assert(kBins == 2 * kThreads, "two bins a thread");
constexpr int kVectors = 4;     // 16-byte vectors of a lane in a stage of the stream
constexpr int kRing = 2;        // stages on their way
constexpr uint32_t kRingBytes = kThreads * kVectors * kRing * 16;
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
  int hist[kBins];
  float2 ranked[kRanked];  // value and position (as bits)
  int count, bin, above, inside;
  float cut;
  int last;
};

// What is selected: above `t`, and of those equal to it the ones up to position `last`.
struct Cut {
  float t;
  int last;
  __device__ bool takes(float v, int at) const { return v > t || (v == t && at <= last); }
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

// Inclusive sum over the block; `total` gets the whole.
__device__ __forceinline__ int block_scan(Shared& sh, int v, int& turn, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) sh.sums[turn][warp][0] = v;
  __syncthreads();
  const int w = lane < kWarps ? sh.sums[turn][lane][0] : 0;
  turn ^= 1;
  *total = __reduce_add_sync(0xFFFFFFFFu, w);
  return v + __reduce_add_sync(0xFFFFFFFFu, lane < warp ? w : 0);
}

// The bin of a value; larger values never have lower bins. (-inf, which is no candidate, has none.)
struct Bins {
  float least, scale;
  bool apart;  // the bins can tell values apart
  __device__ int of(float v) const { return min(int((v - least) * scale), kBins - 1); }
};

// Counts the values (-inf: none) into bins and finds the one that the `want`-th largest is in: sh.bin,
// with sh.above values in higher bins and sh.inside in it. Returns how many values there are; with
// fewer than `want` there is no bin. sh.hist is zero before and after.
template <int N>
__device__ __forceinline__ int count_bins(Shared& sh, const float* v, int want, Bins* bins, int& turn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float low = INFINITY, high = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    low = fminf(low, v[i] > -INFINITY ? v[i] : INFINITY);
    high = fmaxf(high, v[i]);
  }
  // (Without values: more than any key, and the key of -inf.)
  uint32_t least = high > -INFINITY ? key_of(low) : 0xFFFFFFFFu, most = key_of(high);
  least = __reduce_min_sync(0xFFFFFFFFu, least);
  most = __reduce_max_sync(0xFFFFFFFFu, most);
  if (lane == 0) *reinterpret_cast<int2*>(sh.sums[turn][warp]) = make_int2(int(least), int(most));
  __syncthreads();
  const int2 m = *reinterpret_cast<const int2*>(sh.sums[turn][lane & (kWarps - 1)]);
  turn ^= 1;
  least = __reduce_min_sync(0xFFFFFFFFu, uint32_t(m.x));
  most = __reduce_max_sync(0xFFFFFFFFu, uint32_t(m.y));
  bins->least = value_of(least);
  const float range = value_of(most) - bins->least;
  bins->scale = float(kBins) / range;
  bins->apart = least < most && range > 0.f && bins->scale > 0.f && bins->scale < INFINITY;
  if (bins->apart) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (v[i] > -INFINITY) atomicAdd(&sh.hist[bins->of(v[i])], 1);
  } else {
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += v[i] > -INFINITY;
    if (n) atomicAdd(&sh.hist[0], n);
  }
  __syncthreads();
  // From the highest bin down, two a thread.
  int2& mine = reinterpret_cast<int2*>(sh.hist)[kThreads - 1 - threadIdx.x];
  const int2 n = mine;
  mine = make_int2(0, 0);
  int total;
  const int sum = block_scan(sh, n.x + n.y, turn, &total), before = sum - n.x - n.y;
  if (before < want && want <= sum) {
    const int top = kBins - 1 - 2 * int(threadIdx.x);
    const bool upper = before + n.y >= want;
    sh.bin = upper ? top : top - 1;
    sh.above = upper ? before : before + n.y;
    sh.inside = upper ? n.y : n.x;
  }
  __syncthreads();
  return total;
}

// By halving: the `want`-th largest of the values, more of which are above -inf, and of those equal to
// it the last position that is still wanted. at(i) is value i's position, below `end`.
template <int N, typename At>
__device__ __forceinline__ Cut cut_by_halving(Shared& sh, const float* v, At at, int want, int end,
                                              int& turn) {
  uint32_t lo = kNever + 1, hi = 0xFF800001u;  // `want` reach lo, fewer reach hi
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    const float t = value_of(mid);
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += v[i] >= t;
    if (block_sum(sh, n, 0, turn).x >= want) lo = mid; else hi = mid;
  }
  const float t = value_of(lo);
  int n = 0, m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    n += v[i] > t;
    m += v[i] == t;
  }
  const int2 both = block_sum(sh, n, m, turn);
  const int need = want - both.x;
  if (need >= both.y) return {t, INT_MAX};
  int a = -1, b = end;  // positions <= a hold fewer than `need` of the equal ones, <= b enough
  while (b - a > 1) {
    const int mid = a + (b - a) / 2;
    int c = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) c += v[i] == t && at(i) <= mid;
    if (block_sum(sh, c, 0, turn).x >= need) b = mid; else a = mid;
  }
  return {t, b};
}

// The cut that takes the `want` largest of the values (-inf: none), or all if they are no more.
template <int N, typename At>
__device__ __forceinline__ Cut best_cut(Shared& sh, const float* v, At at, int want, int end, int& turn) {
  Bins bins;
  if (count_bins<N>(sh, v, want, &bins, turn) <= want) return {-INFINITY, -1};
  const int bin = sh.bin, inside = sh.inside, need = want - sh.above;
  if (!bins.apart || inside > kRanked) return cut_by_halving<N>(sh, v, at, want, end, turn);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (v[i] > -INFINITY && bins.of(v[i]) == bin)
      sh.ranked[atomicAdd(&sh.count, 1)] = make_float2(v[i], __int_as_float(at(i)));
  __syncthreads();
  // Rank `need` of them, counted from the largest; equal ones from the lowest position. Eight
  // threads compare one with an eighth of them each.
  const int c = threadIdx.x >> 3;
  const float2 mine = sh.ranked[c];
  int rank = 0;
  if (c < inside)
    for (int j = threadIdx.x & 7; j < inside; j += 8) {
      const float2 x = sh.ranked[j];
      rank += x.x > mine.x || (x.x == mine.x && __float_as_int(x.y) < __float_as_int(mine.y));
    }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) rank += __shfl_xor_sync(0xFFFFFFFFu, rank, o);
  if (c < inside && (threadIdx.x & 7) == 0 && rank == need - 1) {
    sh.cut = mine.x;
    sh.last = __float_as_int(mine.y);
    sh.count = 0;
  }
  __syncthreads();
  return {sh.cut, sh.last};
}

// A threshold that about `rank` of the sampled values reach.
template <int N>
__device__ __forceinline__ float sample_threshold(Shared& sh, const float* v, int rank, int& turn) {
  Bins bins;
  if (count_bins<N>(sh, v, rank, &bins, turn) <= rank) return -3.402823466e38f;
  if (bins.apart && sh.inside <= rank / 8 + 1) return bins.least + float(sh.bin) / bins.scale;
  return cut_by_halving<N>(sh, v, [](int) { return 0; }, rank, 0, turn).t;
}

__device__ __forceinline__ void mark(uint32_t* map, int i) { atomicOr(&map[i >> 5], 1u << (i & 31)); }

// 16-byte vectors of global memory, each read by the lane that asked for it: kRing stages of kVectors a
// lane are on their way while one is worked on, without a register for them and without a barrier.
struct Stream {
  const float4* x;
  int vectors;
  uint32_t ring;  // this thread's first vector of the ring
  __device__ Stream(const float* from, int n, float4* buffer)
      : x(reinterpret_cast<const float4*>(reinterpret_cast<uintptr_t>(from) & ~uintptr_t(15))),
        vectors(n),
        ring(ptx::smem_addr(buffer + threadIdx.x)) {}
  // Vector j of stage k; a warp's are neighbours.
  __device__ int index(int k, int j) const {
    return (k * kWarps + int(threadIdx.x >> 5)) * 32 * kVectors + 32 * j + int(threadIdx.x & 31);
  }
  __device__ void ask(int k) {
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      const int i = index(k, j);
      const uint32_t to = ring + uint32_t(((k % kRing) * kVectors + j) * kThreads * 16);
      ptx::cp_async_16(to, i < vectors ? x + i : x, i < vectors ? 16 : 0);
    }
    ptx::cp_async_commit();
  }
  __device__ void start() {
#pragma unroll
    for (int k = 0; k < kRing; ++k) ask(k);
  }
  // fn(values, index) for each of the warp's vectors in stages, lanes together; those past the end are
  // -inf.
  template <typename Fn>
  __device__ void run(Fn fn) {
    const int stages = (vectors + kThreads * kVectors - 1) / (kThreads * kVectors);
#pragma unroll 1
    for (int k = 0; k < stages; ++k) {
      ptx::cp_async_wait_group<kRing - 1>();
      float4 v[kVectors];
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        const uint32_t from = ring + uint32_t(((k % kRing) * kVectors + j) * kThreads * 16);
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[j].x), "=f"(v[j].y), "=f"(v[j].z), "=f"(v[j].w) : "r"(from) : "memory");
        if (index(k, j) >= vectors) v[j] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      }
      fn(v, k);
      ask(k + kRing);
    }
    ptx::cp_async_wait_all();
  }
};

// Keeps the scores of a row that reach `t`; returns how many do (kCandidates of them are kept).
// `stream` has been started on the row's aligned part.
__device__ __forceinline__ int collect(Shared& sh, const Row& r, float t, float2* cand, Stream& stream,
                                       int first) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // One run of places in the list for a warp's; their order does not matter.
  auto keep = [&](const float4* v, auto position) {
    auto part = [&](int i) {
      const float4& f = v[i / 4];
      return i % 4 == 0 ? f.x : i % 4 == 1 ? f.y : i % 4 == 2 ? f.z : f.w;
    };
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4 * kVectors; ++i) n += part(i) >= t;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, sum, o);
      if (lane >= o) sum += u;
    }
    int to = 0;
    if (lane == 31 && sum) to = atomicAdd(&sh.count, sum);
    to = __shfl_sync(0xFFFFFFFFu, to, 31) + sum - n;
    if (n == 0 || to + n > kCandidates) return;  // (too many: they are counted only)
#pragma unroll
    for (int i = 0; i < 4 * kVectors; ++i)
      if (part(i) >= t) cand[to++] = make_float2(part(i), __int_as_float(position(i / 4) + i % 4));
  };
  stream.run([&](const float4* v, int k) {
    keep(v, [&](int j) { return first + 4 * stream.index(k, j); });
  });
  if (warp == 0) {  // up to three values before the aligned ones, up to three behind them
    const int head = first - r.lo, behind = first + 4 * stream.vectors, tail = r.hi - behind;
    const int i = lane < head ? r.lo + lane : behind + lane - head;
    const float4 none = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    float4 v[kVectors];
#pragma unroll
    for (int j = 0; j < kVectors; ++j) v[j] = none;
    if (lane < head + tail) v[0].x = r.x[i];
    keep(v, [&](int) { return i; });
  }
  __syncthreads();
  const int count = sh.count;
  __syncthreads();
  if (threadIdx.x == 0) sh.count = 0;
  return count;
}

// The same over the whole row, for what the candidates do not hold.
__device__ __forceinline__ void mark_best_of_all(Shared& sh, const Row& r, float guess, uint32_t* map,
                                                 int& turn) {
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
    const int2 both = block_sum(sh, n, m, turn);
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
    if (lane == 0) sh.sums[turn][threadIdx.x >> 5][0] = __popc(ties);
    __syncthreads();
    int before = __popc(ties & ((1u << lane) - 1)), all = 0;
    for (int w = 0; w < kWarps; ++w) {
      const int c = sh.sums[turn][w][0];
      if (w < int(threadIdx.x >> 5)) before += c;
      all += c;
    }
    turn ^= 1;
    if (v > t || (tie && before < need)) mark(map, i);
    need -= min(need, all);
  }
}

// Marks the best of a row of at most N * kThreads scores, held in registers.
template <int N>
__device__ __forceinline__ void mark_direct(Shared& sh, const Row& r, uint32_t* map, int& turn) {
  // Value i of a thread is at r.lo + i * kThreads + threadIdx.x: 32 neighbours a warp, so a ballot is 32
  // bits of the answer (of the row from r.lo on, which need not begin a word).
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = r.hi - r.lo;
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int j = i * kThreads + int(threadIdx.x);
    v[i] = j < n ? r.x[r.lo + j] : -INFINITY;
    if (!(v[i] > -INFINITY)) v[i] = -INFINITY;  // no NaN
  }
  auto at = [&](int i) { return r.lo + i * kThreads + int(threadIdx.x); };
  const Cut cut = best_cut<N>(sh, v, at, r.want, r.hi, turn);
  unsigned bits = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned taken = __ballot_sync(0xFFFFFFFFu, cut.takes(v[i], at(i)));
    if (lane == i) bits = taken;
  }
  if (bits) {  // lane i's are value i's
    const int j = r.lo + lane * kThreads + 32 * warp, shift = j & 31;
    atomicOr(&map[j >> 5], bits << shift);
    if (shift && bits >> (32 - shift)) atomicOr(&map[(j >> 5) + 1], bits >> (32 - shift));
  }
}

template <bool kPages>
__global__ void __launch_bounds__(kThreads, 2) index_select_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t raw[];
  float2* cand = reinterpret_cast<float2*>(raw);
  float4* ring = reinterpret_cast<float4*>(cand + kCandidates);
  uint32_t* map = reinterpret_cast<uint32_t*>(ring + kRingBytes / 16);
  float* page_best = reinterpret_cast<float*>(map + a.words);
  __shared__ Shared sh;
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int turn = 0;
  for (int i = tid; i < a.words; i += kThreads) map[i] = 0;
  reinterpret_cast<int2*>(sh.hist)[tid] = make_int2(0, 0);
  if (tid == 0) sh.count = 0;
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
    auto largest = [](const float4& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); };
    auto either = [&](float x, float y, int bit) {  // this lane's part of x or y, with its partner's
      const bool b = lane & bit;
      return fmaxf(b ? y : x, __shfl_xor_sync(0xFFFFFFFFu, b ? x : y, bit));
    };
    // Whole pages of an aligned row are streamed, four a half warp: the exchanges leave each lane one
    // of the four. What is left is read as it is.
    static_assert(kVectors == 4, "four pages a half warp");
    const bool aligned = (reinterpret_cast<uintptr_t>(scores) & 15) == 0;
    const int whole = aligned ? seen / kPageRows : 0;
    Stream stream(scores, whole * (kPageRows / 4), ring);
    stream.start();
    stream.run([&](const float4* v, int k) {
      float m = either(either(largest(v[0]), largest(v[2]), 8), either(largest(v[1]), largest(v[3]), 8), 4);
      m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
      m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
      const int p = stream.index(k, 2 * ((lane >> 3) & 1) + ((lane >> 2) & 1)) / (kPageRows / 4);
      if ((lane & 3) == 0 && p < whole) page_best[p] = m;
    });
    for (int p0 = whole + 2 * warp; p0 < r.count; p0 += 2 * kWarps) {
      const int p = p0 + (lane >> 4), at = p * kPageRows + 4 * (lane & 15);
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at + i < seen) m = fmaxf(m, scores[at + i]);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      if ((lane & 15) == 0 && p < r.count) page_best[p] = m;
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
    if (n <= kDirect / 4) {
      mark_direct<kDirect / kThreads / 4>(sh, r, map, turn);
    } else if (n <= kDirect) {
      mark_direct<kDirect / kThreads>(sh, r, map, turn);
    } else if (kPages) {  // more pages than registers hold, already in shared memory
      mark_best_of_all(sh, r, lowest, map, turn);
    } else {
      // The stream is asked for first; it arrives while the sample is read and counted.
      const int head = int((16 - (reinterpret_cast<uintptr_t>(r.x + r.lo) & 15)) & 15) / 4;
      const int first = r.lo + head;
      Stream stream(r.x + first, (r.hi - first) / 4, ring);
      stream.start();
      // Sampled in runs of sixteen neighbours (two a warp's load), evenly over the row.
      float x[kMaxSample];
      const int rounds = n > 65536 ? kMaxSample / kSample : 1;
#pragma unroll
      for (int j = 0; j < kMaxSample; ++j) {
        x[j] = -INFINITY;
        if (j < rounds * kSample) {
          const int run = j * 2 * kWarps + (tid >> 4);
          const int from = int((long long)run * (n - 16) / (rounds * kSample * 2 * kWarps));
          const float v = r.x[r.lo + from + (tid & 15)];
          x[j] = v >= lowest ? v : -INFINITY;
        }
      }
      const float sampled = float(rounds * kThreads * kSample), share = sampled / float(n);
      const float expect = float(r.want) * share;
      float rank = expect + 6.f * sqrtf(expect) + 16.f, t0 = lowest;
      rank = fmaxf(fminf(rank, 0.8f * float(kCandidates) * share), expect + 1.f);
      bool found = false;
      for (int attempt = 0; attempt < 3 && !found; ++attempt) {
        t0 = rank >= sampled ? lowest
             : rounds > 1    ? sample_threshold<kMaxSample>(sh, x, int(rank), turn)
                             : sample_threshold<kSample>(sh, x, int(rank), turn);
        if (attempt) stream.start();
        const int count = collect(sh, r, t0, cand, stream, first);
        if (count <= kCandidates && (count >= r.want || t0 == lowest)) {
          found = true;
          constexpr int kHeld = (kCandidates + kThreads - 1) / kThreads;
          float v[kHeld];
          int place[kHeld];
#pragma unroll
          for (int i = 0; i < kHeld; ++i) {
            const int j = i * kThreads + tid;
            const float2 c = j < count ? cand[j] : make_float2(-INFINITY, 0.f);
            v[i] = c.x;
            place[i] = __float_as_int(c.y);
          }
          const Cut cut = best_cut<kHeld>(sh, v, [&](int i) { return place[i]; }, r.want, r.hi, turn);
#pragma unroll
          for (int i = 0; i < kHeld; ++i)
            if (cut.takes(v[i], place[i])) mark(map, place[i]);
        } else if (count < r.want) {
          rank *= 1.5f * float(r.want) / float(max(count, r.want / 8 + 1));
        } else {
          rank *= 0.75f * float(kCandidates) / float(count);
          if (rank < expect) break;
        }
      }
      if (!found) mark_best_of_all(sh, r, t0, map, turn);
    }
  }
  __syncthreads();
  // The bitmap in order: each thread numbers a run of its words.
  int* out = reinterpret_cast<int*>(cand);  // candidates are no longer needed
  const int words = (r.count + 31) / 32, each = (words + kThreads - 1) / kThreads;
  const int w0 = min(words, tid * each), w1 = min(words, w0 + each);
  int mine = 0, taken;
  for (int w = w0; w < w1; ++w) mine += __popc(map[w]);
  int at = block_scan(sh, mine, turn, &taken) - mine;
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
  static_assert(kCandidates * 8 + kRingBytes + (1u << 15) * 4 + sizeof(Shared) <= 227 * 1024 &&
                    kCandidates * 8 + kRingBytes + (1u << 9) * 4 + (1u << 14) * 4 + sizeof(Shared) <= 227 * 1024,
                "shared memory of 2^20 columns");
  const uint32_t bytes = kCandidates * 8u + kRingBytes + uint32_t(a.words) * 4u + (pages ? uint32_t(items) * 4u : 0u);
  auto kernel = pages ? index_select_kernel<true> : index_select_kernel<false>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)) != cudaSuccess)
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
