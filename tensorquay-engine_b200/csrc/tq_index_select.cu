// Index select (tq_index_select): each token's K best rows or pages, in ascending order.
//
// The K-th largest of a row's scores is found by counting: into kBins bins of even width between the
// least and the largest; the scores in the one bin that it falls into, a few dozen as a rule, are ranked
// against each other, equal ones by position. Where more than kRanked are in it, they are counted
// again into bins of their own, now by their bits as whole numbers, 10 of 32 a time, so that no
// distribution takes more than five counts. What is taken goes into a bitmap, whose order is the order
// of the answer; nothing depends on timing. Two kernels:
//   hold_kernel    few rows: a cluster of one to eight blocks a token, each with a run of the row in
//                  registers, their bins added up through distributed shared memory. The page form
//                  reduces its scores to a value a page first, and does the same with those
//   stream_kernel  more rows, or longer ones, than clusters hold at once: a block a token. A sample of
//                  the row gives a threshold that a little more than K scores reach (how much more: six
//                  standard deviations of the sample's count, or as many as the list has room for); the
//                  row is read once and what reaches the threshold is listed; these are counted and
//                  ranked. Where too few or too many reach it, it is moved and the row read again; where
//                  that does not help (more equal scores than the list holds) the whole row is counted.
//                  The blocks are small, five on an SM, where there are many, since each has a chain of
//                  barriers that the others fill (of half the size: 90 us instead of 74 for 2048 rows of
//                  16384, then with four on an SM). Their sample is 1024 scores: of 2048 the chain
//                  was longer (74 us, now 67; with the fifth block 64) and a threshold missed more
//                  seldom than one in a thousand. They are large where a row has an SM to itself (64 rows
//                  of 131072, K 2048: 26 us instead of 84), and for long rows (600 of 65536: 69 us; one
//                  small block in thirty missed its threshold, 87).
//
// What bounds it (captured calls back to back, scores in L2 where they fit): few rows are a chain of loads
// and barriers. 1 x 8192: 5.7 us. 64 rows of 16384 to 32768, K 2048, two blocks each: 12.9 us for 1.1 us of
// reading; of a block's 19300 cycles the token and its scores take 2800, their range 2500, the count 1900,
// the sum of both blocks' counts and the bin 2200, the bitmap 3250, the rank 1900, the list 2800, the answer
// 700, the end 1050, and of these five barriers of the cluster about a quarter. Many rows are bound by the
// latency of the same chain, five rows an SM at a time, and by instructions: 2048 x 16384, K 2048: 64 us, a
// third of it the sample and its threshold, a fifth the row's one reading, the rest the 2700 candidates.
// Pages of 64 rows of 65536 to 131072: 11.8 us, 33% of the copy bandwidth (12.5 us and 41% where all are
// full): one wave of maxima, 8000 cycles, then the chain, 12400.

#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "tq_contracts.h"
#include "tq_ptx.cuh"

namespace tq {
namespace index_select {

constexpr int kThreads = 512;          // of hold_kernel
constexpr int kHold = 32 * kThreads;   // scores that a block of it holds, in registers
constexpr int kMaxCluster = 8;
constexpr int kStreamThreads = 256;    // of stream_kernel where there are many rows,
constexpr int kLongThreads = 512;      // and where a row has an SM to itself, or is long
constexpr int kPageRows = 64;
constexpr int kLongRow = 32768;        // longer rows want a larger sample than a small block's
constexpr int kBins = 1024;
constexpr int kRanked = 64;            // scores that are ranked against each other
constexpr float kLowest = -3.402823466e38f;

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
  int blocks;  // of a cluster
  int words;   // of the bitmaps
};

// Scores as they are compared: -0 is 0, NaN is -inf, which is never selected.
__device__ __forceinline__ float score_of(float v) { return v > -INFINITY ? v + 0.f : -INFINITY; }
// In their order as whole numbers.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

struct Shared {
  int2 sums[2][32];             // of the warps, two buffers taken in turn
  int2 total[2];                // of the block, for the cluster's others, in turn
  uint2 range[2];               // least and largest key of the block, in turn
  int hist[2][kBins];           // in turn; zero when they are not in use
  float2 own[kRanked];          // the block's scores in the one bin, and their positions (as bits)
  float2 ranked[kRanked];       // the cluster's
  int owned, bin, above, inside;
};

// The T threads of a block, and the others of its cluster.
template <int T>
struct Team {
  static constexpr int kWarps = T / 32;
  Shared& sh;
  int blocks, rank;
  int turn = 0, turn2 = 0;

  // (The cluster's barrier is one of whole warps.)
  __device__ static void cluster_sync() {
    __syncwarp();
    ptx::cluster_sync();
  }
  __device__ void sync() const {
    if (blocks > 1) cluster_sync();
    else __syncthreads();
  }
  // Eight bytes of another block's shared memory, at the place of `p` in this one's.
  __device__ long long peer(const void* p, int block) const {
    return ptx::ld_cluster_s64(ptx::map_peer(ptx::smem_addr(p), uint32_t(block)));
  }
  __device__ static int2 halves(long long v) { return make_int2(int(v), int(v >> 32)); }

  // The sum over the cluster's blocks of a number that each has, and over the ones before this.
  __device__ int sum(int mine, int* before) {
    *before = 0;
    if (blocks == 1) return mine;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) sh.total[turn2] = make_int2(mine, 0);
    cluster_sync();
    const int v = lane < blocks ? halves(peer(&sh.total[turn2], lane)).x : 0;
    turn2 ^= 1;
    *before = __reduce_add_sync(0xFFFFFFFFu, lane < rank ? v : 0);
    return __reduce_add_sync(0xFFFFFFFFu, v);
  }
  // Inclusive sum over the block's threads, and the whole; one barrier.
  __device__ int block_scan(int v, int* all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) sh.sums[turn][warp] = make_int2(v, 0);
    __syncthreads();
    const int w = lane < kWarps ? sh.sums[turn][lane].x : 0;
    turn ^= 1;
    *all = __reduce_add_sync(0xFFFFFFFFu, w);
    return v + __reduce_add_sync(0xFFFFFFFFu, lane < warp ? w : 0);
  }
  // Least and largest key over the team.
  __device__ uint2 range(uint32_t least, uint32_t most) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    least = __reduce_min_sync(0xFFFFFFFFu, least);
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    if (lane == 0) sh.sums[turn][warp] = make_int2(int(least), int(most));
    __syncthreads();
    int2 m = sh.sums[turn][lane & (kWarps - 1)];
    turn ^= 1;
    least = __reduce_min_sync(0xFFFFFFFFu, uint32_t(m.x));
    most = __reduce_max_sync(0xFFFFFFFFu, uint32_t(m.y));
    if (blocks > 1) {
      if (threadIdx.x == 0) sh.range[turn2] = make_uint2(least, most);
      cluster_sync();
      m = halves(peer(&sh.range[turn2], lane < blocks ? lane : 0));
      turn2 ^= 1;
      least = __reduce_min_sync(0xFFFFFFFFu, uint32_t(m.x));
      most = __reduce_max_sync(0xFFFFFFFFu, uint32_t(m.y));
    }
    return make_uint2(least, most);
  }
};

// The block's run of the scores that are searched: those at [begin, end) of a row.
// In registers, score i of a thread at begin + i * T + threadIdx.x.
template <int T, int N>
struct Held {
  static constexpr bool kFew = true;  // N <= 32
  int begin, end;
  const float* x;
  const int* place;  // null: score i is x[at(i)]; else x[place[at(i)]]
  float v[N];
  __device__ float value(int i) const { return score_of(place ? x[place[at(i)]] : x[at(i)]); }
  __device__ int at(int i) const { return begin + i * T + int(threadIdx.x); }
  __device__ void load(const float* from) {
    x = from;
    place = nullptr;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = at(i) < end ? x[at(i)] : -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = score_of(v[i]);
  }
  __device__ void gather(const float* from, const int* at_place) {
    x = from;
    place = at_place;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = at(i) < end ? x[place[at(i)]] : -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = score_of(v[i]);
  }
  // fn(value, its number) for all of the thread's scores, lanes together.
  template <typename Fn>
  __device__ __forceinline__ void each(Fn fn) const {
#pragma unroll
    for (int i = 0; i < N; ++i) fn(v[i], i);
  }
  // A bitmap of the scores that take(value, number): a ballot is a word, 32 neighbours a warp. Lane i
  // keeps the i-th.
  template <typename Fn>
  __device__ __forceinline__ void mark(uint32_t* map, Fn take) const {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    static_assert(N <= 32, "a word a lane");
    unsigned mine = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned word = __ballot_sync(0xFFFFFFFFu, take(v[i], i));
      if (lane == i) mine = word;
    }
    if (mine) map[lane * (T / 32) + warp] |= mine;
  }
};
// In memory, read in each pass.
template <int T>
struct Read {
  static constexpr bool kFew = false;
  int begin, end;
  const float* x;
  __device__ float value(int i) const { return read(at(i)); }
  __device__ int at(int i) const { return begin + i * T + int(threadIdx.x); }
  __device__ float read(int j) const { return score_of(j < end ? x[j] : -INFINITY); }
  template <typename Fn>
  __device__ __forceinline__ void each(Fn fn) const {
    const int n = (end - begin + T - 1) / T;
    int i = 0;
#pragma unroll 1
    for (; i + 4 <= n; i += 4) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = read(at(i + j));
#pragma unroll
      for (int j = 0; j < 4; ++j) fn(f[j], i + j);
    }
#pragma unroll 1
    for (; i < n; ++i) fn(read(at(i)), i);
  }
  template <typename Fn>
  __device__ __forceinline__ void mark(uint32_t* map, Fn take) const {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    each([&](float v, int i) {
      const unsigned word = __ballot_sync(0xFFFFFFFFu, take(v, i));
      if (lane == 0 && word) map[i * (T / 32) + warp] |= word;
    });
  }
};

// Bins between the least and the largest of some values. Larger values never have lower bins.
struct Bins {
  uint32_t least, most;  // keys
  float low, scale;      // by value: even widths
  int shift;             // by key
  __device__ explicit Bins(uint2 range) : least(range.x), most(range.y) {
    low = value_of(least);
    const float wide = least < most ? value_of(most) - low : 0.f;
    scale = float(kBins) / wide;
    if (!(wide > 0.f && scale > 0.f && scale < INFINITY)) scale = 0.f;
    shift = max(0, 22 - __clz(int((most - least) | 1u)));
  }
  __device__ bool has(float v) const { return key_of(v) >= least && key_of(v) <= most; }
  // The sum with 2^23 leaves the bin in the low bits, at the rate of an addition (a conversion has an
  // eighth of it).
  static constexpr int kZero = 0x4B000000;
  __device__ int sum(float v) const { return __float_as_int(fmaf(v - low, scale, 8388608.f)); }
  __device__ int by_value(float v) const { return min(sum(v), kZero + kBins - 1) - kZero; }
  __device__ int by_key(float v) const { return int((key_of(v) - least) >> shift); }
};

// The bin that the `want`-th largest is in, from counts that the team has put into hist[which]: sh.bin,
// with sh.above values in higher bins and sh.inside in it. Returns how many values there are; with
// fewer than `want` there is no bin. Leaves the other hist zero, and ends with a barrier.
template <int T>
__device__ __forceinline__ int find_bin(Team<T>& team, int which, int want) {
  constexpr int kEach = kBins / T < 2 ? 2 : kBins / T;
  const bool active = kBins / kEach == T || threadIdx.x < kBins / kEach;
  Shared& sh = team.sh;
  team.sync();
  // From the highest bin down, kEach a thread.
  const int first = kBins - kEach * (1 + int(threadIdx.x));
  int n[kEach] = {}, mine = 0;
#pragma unroll
  for (int i = 0; i < kEach; i += 2) {
    if (!active) break;
    const int* at = &sh.hist[which][first + i];
    int2 two = *reinterpret_cast<const int2*>(at);
    if (team.blocks > 1) {
      long long both = 0;  // (counts do not carry: 2^20 at most)
      for (int b = 0; b < team.blocks; ++b) both += team.peer(at, b);
      two = Team<T>::halves(both);
    }
    n[i] = two.x;
    n[i + 1] = two.y;
    mine += two.x + two.y;
    *reinterpret_cast<int2*>(&sh.hist[which ^ 1][first + i]) = make_int2(0, 0);
  }
  int total;
  int before = team.block_scan(mine, &total) - mine;
  if (before < want && want <= before + mine) {
#pragma unroll
    for (int i = kEach - 1; i >= 0; --i) {
      if (before < want && want <= before + n[i]) {
        sh.bin = first + i;
        sh.above = before;
        sh.inside = n[i];
      }
      before += n[i];
    }
  }
  __syncthreads();
  return total;
}

// Puts the block's share of the team's `want` best into its bitmap, bits from run.begin on. hist[0],
// owned and the bitmap are zero.
template <int T, typename R>
__device__ __forceinline__ void mark_best(Team<T>& team, const R& run, int want, uint32_t* map) {
  Shared& sh = team.sh;
  // The range of all values; -inf is none.
  float low = INFINITY, high = -INFINITY;
  run.each([&](float v, int) {
    low = fminf(low, v > -INFINITY ? v : INFINITY);
    high = fmaxf(high, v);
  });
  Bins bins(team.range(high > -INFINITY ? key_of(low) : 0xFFFFFFFFu, key_of(high)));
  int which = 0;
  bool by_value = bins.scale > 0.f;
  if (by_value) {
    run.each([&](float v, int) {
      if (v > -INFINITY) atomicAdd(&sh.hist[0][bins.by_value(v)], 1);
    });
  } else {
    run.each([&](float v, int) {
      if (v > -INFINITY) atomicAdd(&sh.hist[0][bins.by_key(v)], 1);
    });
  }
  if (find_bin(team, 0, want) <= want) {  // all of them
    run.mark(map, [](float v, int) { return v > -INFINITY; });
    return;
  }
  int need = want;
  for (;;) {
    need -= sh.above;
    if (sh.inside <= kRanked || bins.least == bins.most) break;
    // Too many to rank: their own range and bins.
    const int bin = sh.bin;
    uint32_t least = 0xFFFFFFFFu, most = 0;
    run.each([&](float v, int) {
      if (v > -INFINITY && bins.has(v) && (by_value ? bins.by_value(v) : bins.by_key(v)) == bin) {
        least = min(least, key_of(v));
        most = max(most, key_of(v));
      }
    });
    bins = Bins(team.range(least, most));
    by_value = false;
    which ^= 1;
    run.each([&](float v, int) {
      if (bins.has(v)) atomicAdd(&sh.hist[which][bins.by_key(v)], 1);
    });
    find_bin(team, which, need);
  }
  const int bin = sh.bin, inside = sh.inside;
  if (inside > kRanked) {
    // All equal: of these the first `need`, and then what is above them.
    run.mark(map, [&](float v, int) { return bins.has(v); });
    __syncthreads();
    const int words = (run.end - run.begin + 31) / 32, per = (words + T - 1) / T;
    const int w0 = min(words, int(threadIdx.x) * per), w1 = min(words, w0 + per);
    int mine = 0, block, lower;
    for (int w = w0; w < w1; ++w) mine += __popc(map[w]);
    int place = team.block_scan(mine, &block) - mine;
    team.sum(block, &lower);
    place += lower;
    for (int w = w0; w < w1; ++w) {
      uint32_t take = 0;
      for (uint32_t left = map[w]; left && place < need; left &= left - 1, ++place) take |= left & -left;
      map[w] = take;
    }
    __syncthreads();
    run.mark(map, [&](float v, int) { return v > -INFINITY && key_of(v) > bins.most; });
    return;
  }
  // All above the bin, and those in it by rank: eight threads compare one with an eighth of them each.
  auto own = [&](float v, int i) {
    sh.own[atomicAdd(&sh.owned, 1)] = make_float2(v, __int_as_float(run.at(i)));
  };
  if (by_value) {
    // (-inf has a negative sum; what rounds up past the last bin is in it.)
    const int in = Bins::kZero + bin, top = bin == kBins - 1 ? INT_MAX : in;
    if constexpr (R::kFew) {
      // Which of a thread's are in the bin is a bit each: a branch a score would take longer than all
      // the rest, and few threads have any.
      unsigned mine = 0;
      run.mark(map, [&](float v, int i) {
        const int sum = bins.sum(v);
        mine |= unsigned(unsigned(sum - in) <= unsigned(top - in)) << i;
        return sum > top;
      });
      for (; mine; mine &= mine - 1) own(run.value(__ffs(mine) - 1), __ffs(mine) - 1);
    } else {
      run.mark(map, [&](float v, int i) {
        const int sum = bins.sum(v);
        if (sum >= in && sum <= top) own(v, i);
        return sum > top;
      });
    }
  } else {
    run.mark(map, [&](float v, int i) {
      if (bins.has(v) && bins.by_key(v) == bin) own(v, i);
      return v > -INFINITY && (key_of(v) > bins.most || (bins.has(v) && bins.by_key(v) > bin));
    });
  }
  team.sync();
  for (int c0 = 0; c0 < inside; c0 += T / 8) {
    const int c = c0 + (threadIdx.x >> 3);
    float2 it = make_float2(-INFINITY, 0.f);
    const float2* all = sh.own;
    if (team.blocks > 1) {  // (T / 8 is kRanked: once)
      if (c < inside) {
        int left = c, b = 0;
        for (; b < team.blocks - 1; ++b) {
          const int count = int(ptx::ld_cluster_u32(ptx::map_peer(ptx::smem_addr(&sh.owned), uint32_t(b))));
          if (left < count) break;
          left -= count;
        }
        const int2 two = Team<T>::halves(team.peer(&sh.own[left], b));
        it = make_float2(__int_as_float(two.x), __int_as_float(two.y));
        if ((threadIdx.x & 7) == 0) sh.ranked[c] = it;
      }
      all = sh.ranked;
      __syncthreads();
    } else if (c < inside) {
      it = sh.own[c];
    }
    int rank = 0;
    if (c < inside)
      for (int j = threadIdx.x & 7; j < inside; j += 8) {
        const float2 x = all[j];
        rank += x.x > it.x || (x.x == it.x && __float_as_int(x.y) < __float_as_int(it.y));
      }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) rank += __shfl_xor_sync(0xFFFFFFFFu, rank, o);
    // A block marks what is its own.
    const int at = __float_as_int(it.y) - run.begin;
    if (c < inside && (threadIdx.x & 7) == 0 && rank < need && at >= 0 && at < run.end - run.begin)
      atomicOr(&map[at >> 5], 1u << (at & 31));
  }
}

// Calls put(i, bit) for the i-th of a bitmap's bits, in order: each thread numbers a run of its units.
// Returns how many bits there are; what `put` writes is there after the next barrier.
template <typename Unit, int T, typename Fn>
__device__ __forceinline__ int list_units(Team<T>& team, const Unit* map, int bits, Fn put) {
  constexpr int kBits = 8 * sizeof(Unit);
  const int units = (bits + kBits - 1) / kBits, per = (units + T - 1) / T;
  const int u0 = min(units, int(threadIdx.x) * per), u1 = min(units, u0 + per);
  int mine = 0, total;
  for (int u = u0; u < u1; ++u) mine += __popc(uint32_t(map[u]));
  int at = team.block_scan(mine, &total) - mine;
#pragma unroll 1
  for (int u = u0; u < u1; ++u)
#pragma unroll 1
    for (uint32_t b = map[u]; b; b &= b - 1) put(at++, kBits * u + __ffs(b) - 1);
  return total;
}

// The largest score of each of the pages [p0, p1) of a row, 16 lanes a page; NaN does not count.
__device__ __forceinline__ void page_maxima(const float* scores, int seen, int p0, int p1, float* best) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto largest = [](const float4& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); };
  auto either = [&](float x, float y, int bit) {  // this lane's part of x or y, with its partner's
    const bool b = lane & bit;
    return fmaxf(b ? y : x, __shfl_xor_sync(0xFFFFFFFFu, b ? x : y, bit));
  };
  const bool aligned = (reinterpret_cast<uintptr_t>(scores) & 15) == 0;
  // Eight pages a half warp, all on their way at once: the exchanges leave each lane two of the eight.
  constexpr int kBatch = 8;
  for (int p = p0 + 2 * kBatch * warp; p < p1; p += 2 * kBatch * kWarps) {
    float4 v[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int at = (p + 2 * j + (lane >> 4)) * kPageRows + 4 * (lane & 15);
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
    float m[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) m[j] = largest(v[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = either(m[j], m[j + 4], 8);
#pragma unroll
    for (int j = 0; j < 2; ++j) m[j] = either(m[j], m[j + 2], 4);
    m[0] = either(m[0], m[1], 2);
    m[0] = fmaxf(m[0], __shfl_xor_sync(0xFFFFFFFFu, m[0], 1));
    const int j = ((lane & 8) >> 1) | ((lane & 4) >> 1) | ((lane & 2) >> 1);
    const int page = p + 2 * j + (lane >> 4);
    if ((lane & 1) == 0 && page < p1) best[page - p0] = m[0];
  }
}

// The rows that token t sees, and where its scores are.
struct Token {
  const float* scores;
  int seq, seen;
  template <bool kPages>
  __device__ static Token of(const Args& a, int t, bool tell) {
    Token k;
    k.scores = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.scores) + t * a.stride);
    k.seq = a.seq_id[t];
    k.seen = 0;
    const int pos = a.q_pos[t];
    int bad = 0;
    if (k.seq < 0 || k.seq >= a.sequences) {
      bad = TQ_DEV_SEQ_RANGE;
    } else {
      long long n = min((long long)a.kv_len[k.seq], (long long)pos + 1);
      if (kPages) {
        if (n > (long long)a.slots * kPageRows) bad |= TQ_DEV_TABLE_SHORT;
        n = min(n, (long long)a.slots * kPageRows);
      }
      if (n > a.columns) bad |= TQ_DEV_WORK_OVERFLOW;
      k.seen = int(max(0ll, min(n, (long long)a.columns)));
    }
    if (bad && tell && a.flags) atomicOr(a.flags, bad);
    return k;
  }
};

// What a token keeps anyway, [0, lo) and [hi, count), and how many of those between it may have.
struct Kept {
  int count, lo, hi, want;
  __device__ Kept(const Args& a, int n) : count(n) {
    lo = min(a.keep_first, count);
    hi = max(lo, count - a.keep_last);
    want = a.k - lo - (count - hi);
  }
};

// N: scores (pages) of a thread. Short rows need few registers, and three blocks are on an SM (2000 rows
// of 64 pages: 26 us, with N = 16 and one block 62).
template <bool kPages, int N>
__global__ void __launch_bounds__(kThreads, N <= 4 ? 3 : 1) hold_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t raw[];
  int* list = reinterpret_cast<int*>(raw);
  uint32_t* map = reinterpret_cast<uint32_t*>(list + (a.k + 3) / 4 * 4);
  float* best = reinterpret_cast<float*>(map + a.words);
  __shared__ Shared sh;
  const int tid = threadIdx.x, t = int(blockIdx.x) / a.blocks;
  Team<kThreads> team{sh, a.blocks, int(blockIdx.x) % a.blocks};
  for (int i = tid; i < a.words; i += kThreads) map[i] = 0;
  for (int i = tid; i < kBins; i += kThreads) sh.hist[0][i] = 0;
  if (tid == 0) sh.owned = 0;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const Token token = Token::of<kPages>(a, t, tid == 0 && team.rank == 0);
  const Kept kept(a, kPages ? (token.seen + kPageRows - 1) / kPageRows : token.seen);
  // An even run of what is searched for each block.
  const int n = kept.want > 0 ? kept.hi - kept.lo : 0, each = (n + a.blocks - 1) / a.blocks;
  Held<kThreads, N> run;
  run.begin = kept.lo + min(n, team.rank * each);
  run.end = kept.lo + min(n, (team.rank + 1) * each);
  if (n > 0) {
    const float* x = token.scores;
    if (kPages) {
      page_maxima(token.scores, token.seen, run.begin, run.end, best);
      x = best - run.begin;
    }
    __syncthreads();
    run.load(x);
    mark_best(team, run, kept.want, map);
  }
  __syncthreads();
  int before;
  const int block = list_units(team, reinterpret_cast<const uint16_t*>(map), run.end - run.begin,
                              [&](int i, int bit) { list[i] = run.begin + bit; });
  const int taken = team.sum(block, &before);
  __syncthreads();
  const int* table = kPages ? a.page_table + (long long)max(token.seq, 0) * a.slots : nullptr;
  int* idx = a.idx + (long long)t * a.k;
  auto answer = [&](int i, int v) { idx[i] = kPages ? table[v] : v; };
  for (int i = tid; i < block; i += kThreads) answer(kept.lo + before + i, list[i]);
  // What is kept, and -1 behind the last.
  const int behind = kept.count - kept.hi, all = kept.lo + taken + behind;
  const int first = team.rank * kThreads + tid, step = a.blocks * kThreads;
  for (int i = first; i < kept.lo; i += step) answer(i, i);
  for (int i = first; i < behind; i += step) answer(kept.lo + taken + i, kept.hi + i);
  for (int i = all + first; i < a.k; i += step) idx[i] = -1;
  // The block that has the last page of those searched knows whether it is taken.
  const bool last_kept = behind > 0 || kept.count == kept.lo;
  const bool mine = n == 0 || last_kept ? team.rank == 0 : run.end == kept.hi && run.begin < run.end;
  if (tid == 0 && mine) {
    const int bit = kept.hi - 1 - run.begin;
    const bool ends = last_kept || (n > 0 && (map[bit >> 5] >> (bit & 31) & 1));
    a.len[t] = !kPages ? all : all * kPageRows - (ends ? kept.count * kPageRows - token.seen : 0);
  }
  if (a.blocks > 1) Team<kThreads>::cluster_sync();  // nobody reads this block's memory any more
}

// ------------------------------------------------------------------------------ stream

// Bits 4 i of the result are bits i of the low byte.
__device__ __forceinline__ uint32_t spread(uint32_t x) {
  x &= 0xFFu;
  x = (x | x << 12) & 0x000F000Fu;
  x = (x | x << 6) & 0x03030303u;
  return (x | x << 3) & 0x11111111u;
}

// A bitmap of the scores x[lo, hi) that reach `t` > -inf, from position `base` on (a multiple of 16 bytes
// at or before lo), and how many they are.
template <int T>
__device__ __forceinline__ int map_reach(Team<T>& team, const float* x, int base, int lo, int hi,
                                         float t, uint32_t* map) {
  constexpr int kWarps = T / 32, kBatch = 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // Four ballots a group of 128 scores: word c has lane l's score c. Lanes 0 to 3 write one each.
  auto reach = [&](const float4& v, int g) {
    const unsigned b0 = __ballot_sync(0xFFFFFFFFu, v.x >= t), b1 = __ballot_sync(0xFFFFFFFFu, v.y >= t);
    const unsigned b2 = __ballot_sync(0xFFFFFFFFu, v.z >= t), b3 = __ballot_sync(0xFFFFFFFFu, v.w >= t);
    if (lane < 4) map[4 * g + lane] = lane == 0 ? b0 : lane == 1 ? b1 : lane == 2 ? b2 : b3;
  };
  // Those within [lo, hi), a batch's loads first; a warp's last group again where a batch reaches past.
  const int whole0 = lo > base, whole1 = (hi - base) >> 7;
  const float4* from = reinterpret_cast<const float4*>(x + base) + lane;
#pragma unroll 1
  for (int g0 = whole0 + warp * kBatch; g0 < whole1; g0 += kWarps * kBatch) {
    float4 v[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) v[j] = from[32 * min(g0 + j, whole1 - 1)];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) reach(v[j], min(g0 + j, whole1 - 1));
  }
  // Those at the ends, if any.
  const int groups = (hi - base + 127) >> 7;
  if (warp < 2 && (warp == 0 ? whole0 : groups > max(whole0, whole1))) {
    const int g = warp == 0 ? 0 : groups - 1, at = base + 128 * g + 4 * lane;
    auto one = [&](int i) { return i >= lo && i < hi ? x[i] : -INFINITY; };
    reach(make_float4(one(at), one(at + 1), one(at + 2), one(at + 3)), g);
  }
  __syncthreads();
  // Each group of four words into the order of positions.
  int n = 0;
  for (int g = threadIdx.x; g < groups; g += T) {
    uint4& w = reinterpret_cast<uint4*>(map)[g];
    const uint4 b = w;
    n += __popc(b.x) + __popc(b.y) + __popc(b.z) + __popc(b.w);
    auto part = [&](int s) {
      return spread(b.x >> s) | spread(b.y >> s) << 1 | spread(b.z >> s) << 2 | spread(b.w >> s) << 3;
    };
    w = make_uint4(part(0), part(8), part(16), part(24));
  }
  int total;
  team.block_scan(n, &total);  // (its barrier: the words are there)
  return total;
}

// Marks the best of a whole row, read again in each pass: for what the list does not hold.
template <int T>
__device__ __noinline__ void mark_row(Shared& sh, const float* x, int lo, int hi, int want, uint32_t* map) {
  Team<T> team{sh, 1, 0};
  const Read<T> run = {lo, hi, x};
  mark_best(team, run, want, map);
}

// Scores that it lists: a small block 13 a thread, which leaves it registers, and room beside the most
// that can be asked for.
template <int T>
constexpr int kCandidates = T == kStreamThreads ? 13 * T : 8 * T;

template <int T>
__global__ void __launch_bounds__(T, T == kStreamThreads ? 5 : 2) stream_kernel(const Args a) {
  constexpr int kWarps = T / 32, kCandidates = index_select::kCandidates<T>;
  constexpr int kSample = T == kStreamThreads ? 4 : 16;  // scores of a thread
  extern __shared__ __align__(16) uint8_t raw[];
  int* place = reinterpret_cast<int*>(raw);                        // candidates: positions
  int* order = place + kCandidates;                                // those selected
  uint32_t* map = reinterpret_cast<uint32_t*>(order + (a.k + 3) / 4 * 4);
  __shared__ Shared sh;
  __shared__ __align__(16) uint32_t chosen[kCandidates / 32];    // bitmap of the candidates
  const int tid = threadIdx.x, t = blockIdx.x;
  Team<T> team{sh, 1, 0};
  for (int i = tid; i < kBins; i += T) sh.hist[0][i] = 0;
  for (int i = tid; i < kCandidates / 32; i += T) chosen[i] = 0;
  if (tid == 0) sh.owned = 0;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const Token token = Token::of<false>(a, t, tid == 0);
  const Kept kept(a, token.seen);
  const float* x = token.scores;
  int* idx = a.idx + (long long)t * a.k;
  const int n = kept.want > 0 ? kept.hi - kept.lo : 0;
  int count = 0;         // candidates
  bool listed = false;   // they are all that is needed
  if (n > 0) {
    const int base = kept.lo - int(reinterpret_cast<uintptr_t>(x + kept.lo) & 15) / 4;
    float t0 = kLowest, sampled = float(kSample * T), share = sampled / float(n);
    const float expect = float(kept.want) * share;
    float rank = fminf(expect + 6.f * sqrtf(expect) + 16.f, 0.8f * float(kCandidates) * share);
    rank = fmaxf(rank, expect + 1.f);
    for (int attempt = 0; attempt < 3; ++attempt) {
      if (n > kCandidates && rank < sampled) {
        // Sampled in runs of sixteen neighbours (two a warp's load), evenly over the row.
        float s[kSample];
#pragma unroll
        for (int j = 0; j < kSample; ++j) {
          const int r = j * 2 * kWarps + (tid >> 4);
          s[j] = x[kept.lo + int(uint32_t(r * (n - 16)) / (kSample * 2 * kWarps)) + (tid & 15)];
        }
        if (attempt == 0 && tid == 0)  // the whole row is on its way to L2 meanwhile
          ptx::bulk_prefetch_l2(x + base + (kept.lo > base ? 4 : 0),
                                uint32_t(((kept.hi - base) / 4 - (kept.lo > base)) * 16));
#pragma unroll
        for (int j = 0; j < kSample; ++j) s[j] = score_of(s[j]);
        // About `rank` of the sample reach the low edge of the bin that the rank-th largest is in.
        float low = INFINITY, high = -INFINITY;
#pragma unroll
        for (int j = 0; j < kSample; ++j) {
          low = fminf(low, s[j] > -INFINITY ? s[j] : INFINITY);
          high = fmaxf(high, s[j]);
        }
        const Bins bins(team.range(high > -INFINITY ? key_of(low) : 0xFFFFFFFFu, key_of(high)));
        const int which = attempt & 1;
#pragma unroll
        for (int j = 0; j < kSample; ++j)
          if (s[j] > -INFINITY)
            atomicAdd(&sh.hist[which][bins.scale > 0.f ? bins.by_value(s[j]) : bins.by_key(s[j])], 1);
        t0 = kLowest;
        if (find_bin(team, which, int(rank)) > int(rank))
          t0 = bins.scale > 0.f ? bins.low + (float(sh.bin) - 0.5f) / bins.scale
                                : value_of(bins.least + (uint32_t(sh.bin) << bins.shift));
        if (!(t0 >= kLowest)) t0 = kLowest;
      } else {
        t0 = kLowest;
      }
      __syncthreads();
      for (int i = tid; i < kBins; i += T) sh.hist[0][i] = sh.hist[1][i] = 0;
      count = map_reach(team, x, base, kept.lo, kept.hi, t0, map);
      if (count <= kCandidates && (count >= kept.want || t0 == kLowest)) {
        listed = true;
        break;
      }
      // Half way between too few and too many, by what this threshold gave. (Many equal ones: no use.)
      rank *= 0.5f * float(kept.want + kCandidates) / float(max(count, kept.want / 8 + 1));
      if (rank < 0.5f * expect) break;
      rank = fmaxf(rank, 1.f);
    }
    if (listed) {
      list_units(team, map, kept.hi - base, [&](int i, int bit) { place[i] = base + bit; });
      __syncthreads();
      if (count > kept.want) {
        Held<T, kCandidates / T> run;
        run.begin = 0;
        run.end = count;
        run.gather(x, place);
        mark_best(team, run, kept.want, chosen);
      }
    } else {
      // The whole row, with a bitmap of it.
      for (int i = tid; i < a.words; i += T) map[i] = 0;
      __syncthreads();
      mark_row<T>(sh, x, kept.lo, kept.hi, kept.want, map);
    }
    __syncthreads();
  }
  int taken = 0;
  if (listed && count <= kept.want) {
    taken = count;
    for (int i = tid; i < taken; i += T) idx[kept.lo + i] = place[i];
  } else if (listed) {
    taken = list_units(team, reinterpret_cast<const uint16_t*>(chosen), count,
                       [&](int i, int bit) { order[i] = place[bit]; });
    __syncthreads();
    for (int i = tid; i < taken; i += T) idx[kept.lo + i] = order[i];
  } else if (n > 0) {
    taken = list_units(team, map, n, [&](int i, int bit) { place[i] = kept.lo + bit; });
    __syncthreads();
    for (int i = tid; i < taken; i += T) idx[kept.lo + i] = place[i];
  }
  const int behind = kept.count - kept.hi, all = kept.lo + taken + behind;
  for (int i = tid; i < kept.lo; i += T) idx[i] = i;
  for (int i = tid; i < behind; i += T) idx[kept.lo + taken + i] = kept.hi + i;
  for (int i = all + tid; i < a.k; i += T) idx[i] = -1;
  if (tid == 0) a.len[t] = all;
}

// SMs of the current device, once the kernels have their shared memory granted on it; 0 on failure.
int sms_on(int device) {
  static std::mutex mu;
  static int cached[128] = {0};
  if (device < 0 || device >= 128) return 0;
  std::lock_guard<std::mutex> lock(mu);
  int n = 0;
  const cudaFuncAttribute most = cudaFuncAttributeMaxDynamicSharedMemorySize;
  const int room = 200 * 1024;
  if (!cached[device] &&
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) == cudaSuccess &&
      cudaFuncSetAttribute(hold_kernel<false, 4>, most, room) == cudaSuccess &&
      cudaFuncSetAttribute(hold_kernel<true, 4>, most, room) == cudaSuccess &&
      cudaFuncSetAttribute(hold_kernel<false, 16>, most, room) == cudaSuccess &&
      cudaFuncSetAttribute(hold_kernel<false, 32>, most, room) == cudaSuccess &&
      cudaFuncSetAttribute(hold_kernel<true, 16>, most, room) == cudaSuccess &&
      cudaFuncSetAttribute(hold_kernel<true, 32>, most, room) == cudaSuccess &&
      cudaFuncSetAttribute(stream_kernel<kLongThreads>, most, room) == cudaSuccess &&
      cudaFuncSetAttribute(stream_kernel<kStreamThreads>, most, room) == cudaSuccess)
    cached[device] = n;
  return cached[device];
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
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return fail("device", TQ_ERR_CUDA);
  const int sms = sms_on(device);
  if (sms <= 0) return fail("device", TQ_ERR_CUDA);
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
  const long long rows = (long long)s.scores.shape[0];
  const int items = pages ? (a.columns + kPageRows - 1) / kPageRows : a.columns;
  // A cluster's blocks: as many as it takes to hold a row, and more while the card has room for one on
  // each SM and a block would still have kFew scores (the five barriers of a cluster, about 1000 cycles
  // each, take as long as a block takes for that many: with 14800 scores its range, count and bitmap take
  // 3500 cycles more than with 8192, beside a barrier).
  constexpr int kFew = 8192;
  a.blocks = 1;
  while (a.blocks < kMaxCluster && (items > a.blocks * kHold || (rows * a.blocks * 2 <= sms &&
                                                                 a.columns > 2 * kFew * a.blocks)))
    a.blocks *= 2;
  // The row form streams its rows instead where clusters would not all run at once, or cannot hold a row,
  // unless they are short: then there is nothing to sample, and a block that holds its row reads it once
  // (2000 x 2048, K 512: 29 us, streamed 46).
  const bool stream_rows =
      !pages && items > kHold / 8 && (rows * a.blocks > sms || items > a.blocks * kHold);
  const bool large = stream_rows && (rows <= sms || items > kLongRow);
  const int list = (a.k + 3) / 4 * 16;
  uint32_t bytes;
  if (stream_rows) {
    a.blocks = 1;
    a.words = ((items + 127) / 128 + 1) * 4;
    bytes = uint32_t((large ? kCandidates<kLongThreads> : kCandidates<kStreamThreads>) * 4 + list + a.words * 4);
  } else {
    const int each = (items + a.blocks - 1) / a.blocks;
    a.words = (each + 31) / 32;
    bytes = uint32_t(list + a.words * 4 + (pages ? each * 4 : 0));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows * a.blocks), 1, 1);
  cfg.blockDim = dim3(large ? kLongThreads : stream_rows ? kStreamThreads : kThreads, 1, 1);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  // Not both: clusters that were launched early took the places of the ones before them.
  if (a.blocks == 1) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
  } else {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(a.blocks);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int n = (items + a.blocks - 1) / a.blocks;
  const auto kernel = large            ? stream_kernel<kLongThreads>
                      : stream_rows    ? stream_kernel<kStreamThreads>
                      : n <= kHold / 8 ? pages ? hold_kernel<true, 4> : hold_kernel<false, 4>
                      : n <= kHold / 2 ? pages ? hold_kernel<true, 16> : hold_kernel<false, 16>
                      : pages          ? hold_kernel<true, 32>
                                       : hold_kernel<false, 32>;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) return fail("launch", TQ_ERR_CUDA);
  return fail(nullptr, TQ_OK);
}
