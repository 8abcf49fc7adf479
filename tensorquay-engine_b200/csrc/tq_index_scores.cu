// Index scores (tq_index_scores): a cheap score of every cached row for every query token,
//   scores[t, n] = key_scale[n] * sum_h w[t, h] * max(0, q[t, h] . k[n]),  n < sees(t).
//
// The dots are E4M3 products on tcgen05 (kind::f8f6f4, f32 sums): 128 keys are the M of a tile, the
// heads of up to 256 columns of query tokens its N, K = 128 in four steps. A key is then one lane of
// TMEM. What reads its columns, cuts them at zero and adds them up with the tokens' weights takes one of
// two forms, and either way a warp writes 32 consecutive scores:
//   heads a multiple of 16   a thread has a part of the columns of four keys and its weights in registers;
//                            the sums of four lanes are joined by three exchanges
//   other multiples of 8     a thread has all columns of one key; weights from shared memory, no packing of
//                            several tiles into a step
//
// Work: G consecutive tokens are a group (512 columns, 32 tokens at most); a run is a part of a group
// with one sequence, and a unit of work a run over 128 keys. Every CTA sums the costs of all groups,
// takes its even share of the sum and walks it; a run's keys are loaded once for all its tokens.
// Warps of the one CTA on an SM:
//   0     walks the runs: describes each (tokens, what they see), loads its codes and weights, and
//         its keys and their scales two pages at a time (TMA through the page table, the codes with
//         128-byte swizzle). A scale arrives as the first of four floats, the least that TMA moves;
//         4-byte copies by the warp's lanes took 1100 cycles a tile
//   1     one lane issues the MMAs, a step into one of two halves of TMEM: a tile by half of a group's
//         tokens, or up to kPack tiles by a run of few
//   2-17  four groups of warps, two for each half of TMEM: the sums over heads. In the first form a warp
//         has the tokens' weights in registers for a whole run; what a thread adds for a key and a head
//         is 1.5 instructions (a maximum, half of a packed multiply-add)
//
// What bounds it (times back to back): many tokens, the hand-overs between the MMAs and the sums. 2048
// tokens of 64 heads over 8192 rows take 164 us (151 captured), where the products alone would take 72; without the
// arithmetic of the sums it is 126, without their reads of TMEM 131: a step's MMAs, its commit, its sums
// and their arrival follow one another in each half of TMEM, and two halves hide half of that. (Sixteen
// warps a step instead of eight: the same time. MMAs issued by a converged warp cost half as much,
// 145 cycles for four, and the call took 171 us.) Few tokens, the loads: 64 requests of 16384 to 32768 rows
// 56 us (53 captured) at 60% of the copy bandwidth, 50 without the scales' loads and the sums. TMA takes about 7 cycles
// for a row of 128 bytes at a pitch of 144; seven stages instead of four, or pages brought to L2 ahead (the
// same engine: 76 us), do not help. One token of 8192 rows 7 us, launch and one chain of loads, products
// and sums.
// Waits are bounded (about 2 s); one that gives up sets TQ_DEV_WAIT_TIMEOUT and ends its warp's work.

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>

#include "tq_contracts.h"
#include "tq_ptx.cuh"
#include "tq_tensor_map.h"

namespace tq {
namespace index_scores {

constexpr int kDim = TQ_INDEX_DIM;
constexpr int kPageRows = 64;
constexpr int kKeys = 128;  // keys of a tile, two pages
constexpr int kThreads = 576;
constexpr int kWarps = kThreads / 32;
constexpr int kSumWarp = 2;  // first of sixteen
constexpr int kColumns = 256;     // of a step
constexpr int kSubTokens = 16;    // tokens of a step at most
constexpr int kStages = 4;        // key tiles in flight
constexpr int kPack = 4;          // key tiles of a step at most
constexpr int kScaleSlots = 12;   // see the producer
constexpr int kCached = 512;      // tokens that are looked up once
constexpr uint32_t kKeyBytes = kKeys * kDim;
constexpr uint32_t kQueryBytes = 2 * kColumns * kDim;
constexpr uint32_t kTries = 1u << 21;

struct Unit {
  int t0, tokens;          // run of tokens; 0 tokens: no more work
  int tile0, tiles;        // its key tiles
  int pack;                // of them in one step
  int sees[2 * kSubTokens];
};

struct Shared {  // behind 1024-byte alignment
  uint8_t query[2][kQueryBytes];
  uint8_t key[kStages][kKeyBytes];
  float weight[2][2 * kColumns];
  float4 scale[kScaleSlots][kKeys];  // the first of four; TMA moves 16 bytes at least
  Unit unit[2];
  int2 token[kCached];     // sequence, rows seen
  __align__(8) int row[32];  // first rows of the pages of sixteen tiles
  uint64_t bar_key_full[kStages], bar_key_empty[kStages];
  uint64_t bar_scale[kScaleSlots];
  uint64_t bar_unit_full[2], bar_unit_empty[2];
  uint64_t bar_acc_full[2], bar_acc_empty[2];
  uint64_t bar_drain;
  long long part[kWarps];
  long long start_cost;
  int start_group;
  uint32_t tmem;
};
constexpr uint32_t kSharedBytes = sizeof(Shared) + 1024;
static_assert(kScaleSlots >= 2 * kPack + kStages, "scale slots");
static_assert(kSharedBytes <= 227 * 1024, "shared memory per CTA");

struct Args {
  const float* w;
  const int* page_table;
  const int* seq_id;
  const int* q_pos;
  const int* kv_len;
  uint8_t* scores;
  int* flags;
  long long score_stride;  // bytes
  int tokens, heads, sequences, slots, pages, columns;
  int sub;      // tokens of a step
  int pack;     // several tiles of a short run may share a step
  int nowhere;  // a row past the key map's end: reads as zeros
};

// A bounded wait: kTries suspensions of at most a microsecond. No more instructions than it needs: it
// stands in a dozen places and competes for the instruction caches with the loops around it (with a
// timer in its loop, a wait that had long been satisfied took 200 to 400 cycles).
struct Wait {
  int* flags;
  __device__ __forceinline__ bool on(uint64_t& barrier, uint32_t parity) {
    const uint32_t bar = ptx::smem_addr(&barrier);
#pragma unroll 1
    for (uint32_t i = 0; i < kTries; ++i)
      if (ptx::mbar_try(bar, parity, 1000)) return true;
    if (flags) atomicOr(flags, TQ_DEV_WAIT_TIMEOUT);
    return false;
  }
  // For a converged warp: all lanes go on, or none.
  __device__ __forceinline__ bool warp_on(uint64_t& barrier, uint32_t parity) {
    return __all_sync(0xFFFFFFFFu, on(barrier, parity));
  }
};

// Rows that token t sees, 0 without a sequence; `bad` gets the flags of what is cut.
__device__ __forceinline__ int sees(const Args& a, int s, int pos, int* bad) {
  if (s < 0 || s >= a.sequences) { *bad |= TQ_DEV_SEQ_RANGE; return 0; }
  const long long n = min((long long)a.kv_len[s], (long long)pos + 1);
  const long long held = (long long)a.slots * kPageRows;
  if (n > held) *bad |= TQ_DEV_TABLE_SHORT;
  if (min(n, held) > a.columns) *bad |= TQ_DEV_WORK_OVERFLOW;
  return int(max(0ll, min(min(n, held), (long long)a.columns)));
}

// Cost of a key tile for a run: its load, and 64 columns at a time the products and sums. (A tile
// of one token with 64 heads takes about 0.4 of the time of one with 512 columns.)
__device__ __forceinline__ int tile_cost(const Args& a, int tokens) {
  return 4 + (tokens * a.heads + 63) / 64;
}
// (No sum with `most`: it may be 2^31 - 1.)
__device__ __forceinline__ int tiles_of(int most) { return most / kKeys + (most % kKeys != 0); }

// Sequence and rows seen of four tokens from t on, up to `end`: from the cache, or with their loads in
// flight together.
__device__ __forceinline__ void look_up(const Args& a, const Shared& sh, int t, int end, int2 (&to)[4],
                                        int* bad) {
  if (a.tokens <= kCached) {
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = sh.token[min(t + i, end - 1)];
    return;
  }
  int p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    to[i].x = a.seq_id[min(t + i, end - 1)];
    p[i] = a.q_pos[min(t + i, end - 1)];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) to[i].y = sees(a, to[i].x, p[i], bad);
}

// Cost of group g: its tokens in order, run by run.
__device__ __forceinline__ long long group_cost(const Args& a, const Shared& sh, int g, int* bad) {
  const int size = 2 * a.sub, t0 = g * size, end = min(a.tokens, t0 + size);
  long long cost = 0;
  int seq = 0, run = 0, most = 0;
  for (int t = t0; t < end; t += 4) {
    int2 token[4];
    look_up(a, sh, t, end, token, bad);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (t + i >= end) break;
      if (run && token[i].x != seq) {
        cost += (long long)tiles_of(most) * tile_cost(a, run);
        run = most = 0;
      }
      seq = token[i].x;
      ++run;
      most = max(most, token[i].y);
    }
  }
  return cost + (long long)tiles_of(most) * tile_cost(a, run);
}

// The CTA's share [lo, hi) of all costs, and the group that lo falls in.
__device__ __forceinline__ void find_share(const Args& a, Shared& sh, long long* lo, long long* hi) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int groups = (a.tokens + 2 * a.sub - 1) / (2 * a.sub);
  const int each = (groups + kThreads - 1) / kThreads;
  const int g0 = min(groups, tid * each), g1 = min(groups, g0 + each);
  int bad = 0;
  if (a.tokens <= kCached) {
    if (tid < a.tokens) {
      const int s = a.seq_id[tid];
      sh.token[tid] = make_int2(s, sees(a, s, a.q_pos[tid], &bad));
    }
    __syncthreads();
  }
  long long mine = 0;
  for (int g = g0; g < g1; ++g) mine += group_cost(a, sh, g, &bad);
  if (blockIdx.x == 0 && bad && a.flags) atomicOr(a.flags, bad);
  long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) sh.part[warp] = sum;
  __syncthreads();
  long long total = 0;
  for (int i = 0; i < kWarps; ++i) {
    if (i == warp) sum += total;
    total += sh.part[i];
  }
  *lo = total * blockIdx.x / gridDim.x;
  *hi = total * (blockIdx.x + 1) / gridDim.x;
  long long at = sum - mine;
  if (*lo < *hi && at <= *lo && *lo < sum) {
    int unused = 0, g = g0;
    for (; g < g1; ++g) {
      const long long cost = group_cost(a, sh, g, &unused);
      if (*lo < at + cost) break;
      at += cost;
    }
    sh.start_group = g;
    sh.start_cost = at;
  }
  __syncthreads();
}

// Warp 0. A unit's slot is free once the MMAs that read its codes and the sixteen that read its
// weights are done. A key stage is free once its MMAs are. By then the sums of the step two before theirs
// are done (each half of TMEM is taken in turn), and with them those of the tile 2 kPack before it: a
// scale slot that comes back after 2 kPack + kStages tiles is free too.
__device__ __forceinline__ void produce(const Args& a, Shared& sh, const CUtensorMap* tm_q,
                                        const CUtensorMap* tm_k, const CUtensorMap* tm_s, long long lo,
                                        long long hi) {
  const int lane = threadIdx.x & 31;
  Wait wait{a.flags};
  const int size = 2 * a.sub;
  int tile = 0, s = 0, slot = 0, units = 0;  // (the first three are the issuing lane's)
  uint32_t parity = 0;                       // of the uses of stage s
  bool ok = true;
  long long at = sh.start_cost;
  for (int g = sh.start_group; ok && at < hi && (long long)g * size < a.tokens; ++g) {
    const int end = min(a.tokens, (g + 1) * size);
    for (int t = g * size; ok && at < hi && t < end;) {
      // One token a lane: the run that starts at t.
      int seq = 0, n = 0, unused = 0;
      if (t + lane < end) {
        if (a.tokens <= kCached) {
          seq = sh.token[t + lane].x;
          n = sh.token[t + lane].y;
        } else {
          seq = a.seq_id[t + lane];
          n = sees(a, seq, a.q_pos[t + lane], &unused);
        }
      }
      const int first = __shfl_sync(0xFFFFFFFFu, seq, 0);
      const unsigned same = __ballot_sync(0xFFFFFFFFu, t + lane < end && seq == first);
      const int run = same == 0xFFFFFFFFu ? 32 : __ffs(~same) - 1;
      if (lane >= run) n = 0;
      const int most = __reduce_max_sync(0xFFFFFFFFu, n), tiles = tiles_of(most);
      const int cost = tile_cost(a, run);
      // Tiles that start within the share.
      const int j0 = int(min((long long)tiles, max(0ll, (lo - at + cost - 1) / cost)));
      const int j1 = int(min((long long)tiles, (hi - at + cost - 1) / cost));
      at += (long long)tiles * cost;
      if (j0 < j1) {
        const int u = units & 1;
        ok = units < 2 || wait.warp_on(sh.bar_unit_empty[u], uint32_t((units >> 1) - 1) & 1u);
        if (!ok) break;
        Unit& unit = sh.unit[u];
        unit.sees[lane] = n;
        if (lane == 0) {
          unit.t0 = t;
          unit.tokens = run;
          unit.tile0 = j0;
          unit.tiles = j1 - j0;
          unit.pack = a.pack ? max(1, min(kPack, a.sub / run)) : 1;
        }
        __syncwarp();
        if (lane == 0) {
          const uint32_t bar = ptx::smem_addr(&sh.bar_unit_full[u]);
          const uint32_t rows = uint32_t(run * a.heads);
          ptx::mbar_expect_tx(bar, rows * (kDim + 4));
          for (int i = 0; i < run; ++i)
            ptx::tma_load_2d(ptx::smem_addr(sh.query[u]) + uint32_t(i * a.heads * kDim), tm_q, bar, 0,
                             (t + i) * a.heads);
          ptx::bulk_load(ptx::smem_addr(sh.weight[u]), a.w + (long long)t * a.heads, rows * 4, bar);
        }
        __syncwarp();
        ++units;
        const int* table = a.page_table + (long long)first * a.slots;
        const int seen_pages = most / kPageRows + (most % kPageRows != 0);
        // Page entries 32 at a time, the next ones on their way; behind the last row that the run sees
        // there are none.
        auto entries = [&](int base) {
          const bool seen = base + lane < min(a.slots, seen_pages);
          const int page = seen ? table[base + lane] : -1;
          if (page >= 0 && page < a.pages) return page * kPageRows;
          if (seen && a.flags) atomicOr(a.flags, TQ_DEV_PAGE_RANGE);
          return a.nowhere;
        };
        // Sixteen tiles at a time, by one lane: with the lanes together an iteration took twice as long.
        int rows = entries(2 * j0);
        for (int j = j0; ok && j < j1; j += 16) {
          sh.row[lane] = rows;
          __syncwarp();
          rows = entries(2 * j + 32);
          if (lane == 0) {
            const int2* at_page = reinterpret_cast<const int2*>(sh.row);
#pragma unroll 1
            for (int left = min(16, j1 - j); left; --left, ++tile) {
              ok = tile < kStages || wait.on(sh.bar_key_empty[s], parity ^ 1u);
              if (!ok) break;
              const int2 r = *at_page++;
              const uint32_t bar = ptx::smem_addr(&sh.bar_key_full[s]), dst = ptx::smem_addr(sh.key[s]);
              const uint32_t bar2 = ptx::smem_addr(&sh.bar_scale[slot]), dst2 = ptx::smem_addr(sh.scale[slot]);
              ptx::mbar_expect_tx(bar, kKeyBytes);
              ptx::tma_load_2d(dst, tm_k, bar, 0, r.x);
              ptx::tma_load_2d(dst + kKeyBytes / 2, tm_k, bar, 0, r.y);
              ptx::mbar_expect_tx(bar2, kKeys * 16);
              ptx::tma_load_2d(dst2, tm_s, bar2, 0, r.x);
              ptx::tma_load_2d(dst2 + kKeys * 8, tm_s, bar2, 0, r.y);
              if (++s == kStages) {
                s = 0;
                parity ^= 1u;
              }
              if (++slot == kScaleSlots) slot = 0;
            }
          }
          ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
        }
      }
      t += run;
    }
  }
  // No more work.
  const int u = units & 1;
  if (ok) ok = units < 2 || wait.warp_on(sh.bar_unit_empty[u], uint32_t((units >> 1) - 1) & 1u);
  if (ok && lane == 0) {
    sh.unit[u].tokens = 0;
    ptx::mbar_arrive(ptx::smem_addr(&sh.bar_unit_full[u]));
  }
  __syncwarp();
  if (!ok) {
    // What is on its way lands before the CTA ends.
    Wait last{a.flags};
    tile = __shfl_sync(0xFFFFFFFFu, tile, 0);
    for (int i = max(0, tile - kStages); i < tile; ++i) {
      last.on(sh.bar_key_full[i % kStages], uint32_t(i / kStages) & 1u);
      last.on(sh.bar_scale[i % kScaleSlots], uint32_t(i / kScaleSlots) & 1u);
    }
    for (int i = max(0, units - 2); i < units; ++i)
      last.on(sh.bar_unit_full[i & 1], uint32_t(i >> 1) & 1u);
  }
}

// Warp 1, one lane of it. False when a wait has given up.
__device__ __forceinline__ bool multiply(const Args& a, Shared& sh) {
  Wait wait{a.flags};
  const uint32_t tmem = sh.tmem;
  // Rows of 128 bytes, K-major, 128-byte swizzle: 8-row groups 1 KB apart.
  const uint64_t keys0 = ptx::smem_desc(ptx::smem_addr(sh.key[0]), 16, 1024, 2);
  const uint64_t queries0 = ptx::smem_desc(ptx::smem_addr(sh.query[0]), 16, 1024, 2);
  int s = 0, tile = 0;  // tiles of all units before this
  uint32_t key_parity = 0, steps = 0;
  // The arrivals that nobody else waits for, of the last key stages and the last unit, must not find a CTA
  // that has ended, and its shared memory another's. They are there before the last sums are.
  auto settled = [&](int units) {
    for (int i = max(0, tile - kStages); i < tile; ++i)
      if (!wait.on(sh.bar_key_empty[i % kStages], uint32_t(i / kStages) & 1u)) return false;
    return units == 0 || wait.on(sh.bar_unit_empty[(units - 1) & 1], uint32_t((units - 1) >> 1) & 1u);
  };
  for (int units = 0;; ++units) {
    const int u = units & 1;
    if (!wait.on(sh.bar_unit_full[u], uint32_t(units >> 1) & 1u)) return false;
    const int tokens = sh.unit[u].tokens, tiles = sh.unit[u].tiles;
    if (tokens == 0) return settled(units);
    const uint64_t queries = queries0 + uint64_t(u) * (kQueryBytes >> 4);
    // Columns in whole sixteens: the last ones may be of no token, and nobody reads them.
    auto idesc = [&](int n) { return ptx::idesc_e4m3(kKeys, uint32_t(n * a.heads + 15) & ~15u); };
    const bool two = tokens > a.sub;
    const uint32_t id0 = idesc(two ? a.sub : tokens), id1 = idesc(tokens - a.sub);
    const uint64_t second = queries + uint64_t(a.sub * a.heads * kDim >> 4);
    const int pack = sh.unit[u].pack;
    // A step fills half of TMEM: with a tile by the first or second half of the tokens, or with `pack` tiles.
    auto begin = [&] {
      if (steps >= 2 && !wait.on(sh.bar_acc_empty[steps & 1], (steps >> 1 & 1u) ^ 1u)) return false;
      ptx::tc_fence_after();
      return true;
    };
    for (int j = 0; j < tiles;) {
      if (!begin()) return false;
#pragma unroll 1
      for (int p = 0; p < pack && j < tiles; ++p, ++j) {
        const uint64_t keys = keys0 + uint64_t(s) * (kKeyBytes >> 4);
        if (!wait.on(sh.bar_key_full[s], key_parity)) return false;
        const uint32_t half = steps & 1;
        ptx::mma_f8_ss_x4(tmem + half * kColumns + uint32_t(p * tokens * a.heads), keys, queries, id0);
        if (two) {
          ptx::mma_commit(ptx::smem_addr(&sh.bar_acc_full[half]));
          ++steps;
          if (!begin()) return false;
          ptx::mma_f8_ss_x4(tmem + (half ^ 1) * kColumns, keys, second, id1);
        }
        ptx::mma_commit(ptx::smem_addr(&sh.bar_key_empty[s]));
        if (++s == kStages) {
          s = 0;
          key_parity ^= 1;
        }
      }
      ptx::mma_commit(ptx::smem_addr(&sh.bar_acc_full[steps & 1]));
      ++steps;
    }
    ptx::mma_commit(ptx::smem_addr(&sh.bar_unit_empty[u]));
    tile += tiles;
  }
}

// After a wait that gave up: what the tensor core still does ends before the CTA does.
__device__ __forceinline__ void drain(const Args& a, Shared& sh) {
  Wait last{a.flags};
  ptx::mma_commit(ptx::smem_addr(&sh.bar_drain));
  last.on(sh.bar_drain, 0);
}

// Waits for the loads; what reads `r` stays behind it.
template <int C>
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[C]) {
  ptx::tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < C; ++i) asm volatile("" : "+r"(r[i]));
}

// max(0, x), NaN stays NaN.
__device__ __forceinline__ float cut(uint32_t bits) {
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(__uint_as_float(bits)));
  return r;
}

// Two sums at once (one instruction for two products and additions).
__device__ __forceinline__ void fma2(float2& acc, float2 x, float2 w) { acc = __ffma2_rn(x, w, acc); }
__device__ __forceinline__ float both(float2 acc) { return acc.x + acc.y; }

__device__ __forceinline__ void add_up(const uint32_t (&r)[8], const float* w, float2 (&acc)[4]) {
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(w + i);
    fma2(acc[(i / 2) & 3], make_float2(cut(r[i]), cut(r[i + 1])), make_float2(v.x, v.y));
    fma2(acc[(i / 2 + 1) & 3], make_float2(cut(r[i + 2]), cut(r[i + 3])), make_float2(v.z, v.w));
  }
}

// A token's sum over kH heads for 128 keys: columns from `from` on, weights w. A thread has two columns
// of each eight and four keys, so a weight serves four sums. (One key a thread needs a weight from
// shared memory for each product: 4 cycles a warp for 128 of them.) The four sums end spread over four
// lanes: three exchanges leave one key's in each. `last` is called once all columns are read.
// What bounds it: the instructions, 1.5 for each head of a key and token (its cut at zero, half of a
// product and addition), a cut at half their rate. So the last of the four keys adds |x| to x
// instead, twice the same, and halves its sum. (So that sum leaves f32 at half the size of the others.)
template <int kH, typename Fn>
__device__ __forceinline__ float sum_heads_of(uint32_t from, const float2* w, int lane, Fn last) {
  constexpr int kStep = kH % 32 ? 16 : 32, kChunks = kH / kStep;  // columns read at a time
  float2 acc[4] = {};
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    uint32_t x[kStep];
    if constexpr (kStep == 32) {
      ptx::tmem_ld_16x128b_x8(from + uint32_t(kStep * c), x);
      ptx::tmem_ld_16x128b_x8(from + uint32_t(kStep * c) + (16u << 16), x + kStep / 2);
    } else {
      ptx::tmem_ld_16x128b_x4(from + uint32_t(kStep * c), x);
      ptx::tmem_ld_16x128b_x4(from + uint32_t(kStep * c) + (16u << 16), x + kStep / 2);
    }
    tmem_wait(x);
    if (c + 1 == kChunks) last();
#pragma unroll
    for (int g = 0; g < kStep / 8; ++g) {
      const float2 wg = w[c * (kStep / 8) + g];
      const uint32_t* y = x + 4 * g;
      fma2(acc[0], make_float2(cut(y[0]), cut(y[2])), wg);
      fma2(acc[1], make_float2(cut(y[1]), cut(y[3])), wg);
      y += kStep / 2;
      fma2(acc[2], make_float2(cut(y[0]), cut(y[2])), wg);
      const float z0 = __uint_as_float(y[1]), z1 = __uint_as_float(y[3]);
      fma2(acc[3], make_float2(z0 + fabsf(z0), z1 + fabsf(z1)), wg);
    }
  }
  const float s0 = both(acc[0]), s1 = both(acc[1]), s2 = both(acc[2]), s3 = 0.5f * both(acc[3]);
  const bool b0 = lane & 1, b1 = lane & 2;
  const float p = (b0 ? s2 : s0) + __shfl_xor_sync(0xFFFFFFFFu, b0 ? s0 : s2, 1);
  const float q = (b0 ? s3 : s1) + __shfl_xor_sync(0xFFFFFFFFu, b0 ? s1 : s3, 1);
  return (b1 ? q : p) + __shfl_xor_sync(0xFFFFFFFFu, b1 ? p : q, 2);
}

// The sum warps, heads a multiple of 16 (kH): the first or second part of a step's columns in half `half` of
// TMEM, lanes 32 (warp % 4) on. The weights of its part, about 32 a thread, stay in registers for all tiles
// of a unit.
template <int kH>
__device__ __forceinline__ void sum_heads_in_registers(const Args& a, Shared& sh, int half, int part) {
  constexpr int kSub = kColumns / kH < kSubTokens ? kColumns / kH : kSubTokens;  // tokens of a step
  constexpr int kSlots = (kSub + 1) / 2;                                         // slots of a warp
  const int lane = threadIdx.x & 31, quad = (threadIdx.x >> 5) & 3;
  const uint32_t tmem = sh.tmem + uint32_t(half * kColumns) + (uint32_t(32 * quad) << 16);
  // After the exchanges: lanes with bit 0 hold keys 16 on, with bit 1 the odd eights.
  const int key = 32 * quad + 16 * (lane & 1) + 4 * (lane & 2) + (lane >> 2);
  Wait wait{a.flags};
  auto done = [&] {
    ptx::tc_fence_before();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&sh.bar_acc_empty[half]));
  };
  int tile = 0, steps = 0;
  for (int units = 0;; ++units) {
    const int u = units & 1;
    if (!wait.warp_on(sh.bar_unit_full[u], uint32_t(units >> 1) & 1u)) return;
    const Unit& unit = sh.unit[u];
    const int tokens = unit.tokens, tiles = unit.tiles;
    if (tokens == 0) return;
    float2 w[kSlots * kH / 8];
    auto weights = [&](int i, int t) {
#pragma unroll
      for (int g = 0; g < kH / 8; ++g) {
        const float* from = &sh.weight[u][(t * kH + 8 * g + (lane & 3)) & (2 * kColumns - 1)];
        w[i * (kH / 8) + g] = make_float2(from[0], from[4]);
      }
    };
    if (tokens > kSub) {
      // A tile is two steps, of which this half of TMEM always has the same one.
      const int t0 = (steps & 1) != half ? kSub : 0, all = min(kSub, tokens - t0);
      const int mine = part ? all / 2 : (all + 1) / 2, place = part ? (all + 1) / 2 : 0;
#pragma unroll
      for (int i = 0; i < kSlots; ++i) weights(i, t0 + place + i);
      const int* seen = unit.sees + t0 + place;
      uint8_t* out = a.scores + (long long)(unit.t0 + t0 + place) * a.score_stride +
                     4ll * (unit.tile0 * kKeys + key);
      uint32_t n = uint32_t(unit.tile0 * kKeys + key);  // (one tile on from the last it may pass 2^31)
      int step = steps + (t0 != 0);
      for (int j = 0; j < tiles; ++j, step += 2, n += kKeys, out += 4 * kKeys) {
        const int slot = (tile + j) % kScaleSlots;
        if (!wait.warp_on(sh.bar_acc_full[half], uint32_t(step >> 1) & 1u)) return;
        ptx::tc_fence_after();
        if (mine == 0) {
          done();
          continue;
        }
        if (!wait.warp_on(sh.bar_scale[slot], uint32_t((tile + j) / kScaleSlots) & 1u)) return;
        const float scale = sh.scale[slot][key].x;
        uint8_t* to = out;
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
          if (i >= mine) break;
          const float sum = sum_heads_of<kH>(tmem + uint32_t((place + i) * kH), w + i * (kH / 8), lane, [&] {
            if (i + 1 >= mine) done();
          });
          if (n < uint32_t(seen[i])) *reinterpret_cast<float*>(to) = sum * scale;
          to += a.score_stride;
        }
      }
      steps += 2 * tiles;
      tile += tiles;
    } else {
      // A step has `pack` tiles, and this half every other step. Its columns are slots of kH, a tile and
      // a token each; this warp has `most` of them from `place` on.
      const int pack = unit.pack, all = pack * tokens;
      const int most = part ? all / 2 : (all + 1) / 2, place = part ? (all + 1) / 2 : 0;
#pragma unroll
      for (int i = 0; i < kSlots; ++i) weights(i, (place + i) % tokens);
      for (int j = 0; j < tiles; j += pack, ++steps) {
        const int tile_now = tile, held = min(pack, tiles - j);
        tile += held;
        if ((steps & 1) != half) continue;
        if (!wait.warp_on(sh.bar_acc_full[half], uint32_t(steps >> 1) & 1u)) return;
        ptx::tc_fence_after();
        const int mine = min(most, held * tokens - place);
        if (mine <= 0) {
          done();
          continue;
        }
        int p = place / tokens, t = place % tokens;
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
          if (i >= mine) break;
          const int slot = (tile_now + p) % kScaleSlots;
          if (!wait.warp_on(sh.bar_scale[slot], uint32_t((tile_now + p) / kScaleSlots) & 1u)) return;
          const float scale = sh.scale[slot][key].x;  // before the half is given back
          const float sum = sum_heads_of<kH>(tmem + uint32_t((place + i) * kH), w + i * (kH / 8), lane, [&] {
            if (i + 1 >= mine) done();
          });
          const int n = (unit.tile0 + j + p) * kKeys + key;
          if (n < unit.sees[t])
            reinterpret_cast<float*>(a.scores + (long long)(unit.t0 + t) * a.score_stride)[n] = sum * scale;
          if (++t == tokens) {
            t = 0;
            ++p;
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&sh.bar_unit_empty[u]));
  }
}

// The same for other multiples of 8 heads, one key a thread: a token's columns are read eight at a time,
// the next ones while the last are added up. A weight is read from shared memory for each product, which
// costs up to twice the time (captured, 2048 tokens over 8192 rows: 72 heads 355 us, 80 heads 206; 64 tokens
// over 16384 to 32768 rows: 77 and 53), so that a caller gains by filling its heads up to a multiple of 16.
__device__ __forceinline__ void sum_heads(const Args& a, Shared& sh, int half, int part) {
  const int lane = threadIdx.x & 31, quad = (threadIdx.x >> 5) & 3, key = 32 * quad + lane;
  const uint32_t tmem = sh.tmem + uint32_t(half * kColumns) + (uint32_t(32 * quad) << 16);
  constexpr int C = 8;
  const int chunks = a.heads / C;
  Wait wait{a.flags};
  int tile = 0, subs = 0;
  for (int units = 0;; ++units) {
    const int u = units & 1;
    if (!wait.warp_on(sh.bar_unit_full[u], uint32_t(units >> 1) & 1u)) return;
    const Unit& unit = sh.unit[u];
    const int tokens = unit.tokens, tiles = unit.tiles, tile0 = unit.tile0, t0 = unit.t0;
    if (tokens == 0) return;
    for (int j = 0; j < tiles; ++j, ++tile) {
      for (int t = 0; t < tokens; t += a.sub, ++subs) {
        if ((subs & 1) != half) continue;
        if (!wait.warp_on(sh.bar_scale[tile % kScaleSlots], uint32_t(tile / kScaleSlots) & 1u)) return;
        if (!wait.warp_on(sh.bar_acc_full[half], uint32_t(subs >> 1) & 1u)) return;
        ptx::tc_fence_after();
        const float scale = sh.scale[tile % kScaleSlots][key].x;
        const int n = (tile0 + j) * kKeys + key;
        const int all = min(a.sub, tokens - t), place = part ? (all + 1) / 2 : 0;
        const int steps = (part ? all / 2 : (all + 1) / 2) * chunks;
        if (steps == 0) {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&sh.bar_acc_empty[half]));
          continue;
        }
        const uint32_t from = tmem + uint32_t(place * a.heads);
        const float* w = sh.weight[u] + (t + place) * a.heads;
        const int* seen = unit.sees + t + place;
        uint8_t* out = a.scores + (long long)(t0 + t + place) * a.score_stride + 4ll * n;
        uint32_t r[2][C];
        float2 acc[4] = {};
        int left = chunks;
        ptx::tmem_ld8(from, r[0]);
#pragma unroll 1
        for (int i = 0; i < steps; i += 2) {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            if (i + b < steps) {
              tmem_wait(r[b]);
              if (i + b + 1 < steps) {
                ptx::tmem_ld8(from + uint32_t((i + b + 1) * C), r[b ^ 1]);
              } else {
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&sh.bar_acc_empty[half]));
              }
              add_up(r[b], w, acc);
              w += C;
              if (--left == 0) {
                const float sum = (both(acc[0]) + both(acc[1])) + (both(acc[2]) + both(acc[3]));
                if (n < *seen) *reinterpret_cast<float*>(out) = sum * scale;
                ++seen;
                out += a.score_stride;
                left = chunks;
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] = make_float2(0.f, 0.f);
              }
            }
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&sh.bar_unit_empty[u]));
  }
}

// kH: the heads if they are a multiple of 16; else 0.
template <int kH>
__global__ void __launch_bounds__(kThreads, 1)
    index_scores_kernel(const __grid_constant__ CUtensorMap tm_q,
                        const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_s, const Args a) {
  extern __shared__ uint8_t raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw + ((1024u - (ptx::smem_addr(raw) & 1023u)) & 1023u));
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    auto init = [](uint64_t& bar, uint32_t count) { ptx::mbar_init(ptx::smem_addr(&bar), count); };
    for (int s = 0; s < kStages; ++s) {
      init(sh.bar_key_full[s], 1);
      init(sh.bar_key_empty[s], 1);
    }
    for (int s = 0; s < kScaleSlots; ++s) init(sh.bar_scale[s], 1);
    for (int b = 0; b < 2; ++b) {
      init(sh.bar_unit_full[b], 1);
      init(sh.bar_unit_empty[b], 17);
      init(sh.bar_acc_full[b], 1);
      init(sh.bar_acc_empty[b], 8);
    }
    init(sh.bar_drain, 1);
    ptx::fence_mbar_init_cluster();
    ptx::tma_prefetch_desc(&tm_q);
    ptx::tma_prefetch_desc(&tm_k);
    ptx::tma_prefetch_desc(&tm_s);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_addr(&sh.tmem), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  long long lo, hi;
  find_share(a, sh, &lo, &hi);
  if (lo < hi) {
    if (warp == 0) {
      produce(a, sh, &tm_q, &tm_k, &tm_s, lo, hi);
    } else if (warp == 1) {
      if ((threadIdx.x & 31) == 0 && !multiply(a, sh)) drain(a, sh);
      __syncwarp();
      __syncwarp();
    } else {
      const int group = (warp - kSumWarp) >> 2;
      if constexpr (kH) sum_heads_in_registers<kH>(a, sh, group & 1, group >> 1);
      else sum_heads(a, sh, group & 1, group >> 1);
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(sh.tmem, 512);
  }
}

// Rows of 128 codes as a 2D map with boxes of `box` rows and 128-byte swizzle.
bool encode_rows(CUtensorMap* map, const void* addr, uint64_t rows, uint64_t stride, uint32_t box) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {kDim, rows};
  const cuuint64_t strides[1] = {stride};
  const cuuint32_t boxes[2] = {kDim, box};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(addr), dims, strides, boxes,
            elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A page's scales, one f32 a row, in boxes of 16 bytes a row: the three columns past the map's only one
// read as zeros.
bool encode_scales(CUtensorMap* map, const void* addr, uint64_t rows, uint64_t stride) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {1, rows};
  const cuuint64_t strides[1] = {stride};
  const cuuint32_t boxes[2] = {4, kPageRows};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(addr), dims, strides, boxes,
            elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
            CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

typedef void (*Kernel)(CUtensorMap, CUtensorMap, CUtensorMap, Args);

Kernel kernel_for(int heads) {
  switch (heads) {
    case 16: return index_scores_kernel<16>;
    case 32: return index_scores_kernel<32>;
    case 48: return index_scores_kernel<48>;
    case 64: return index_scores_kernel<64>;
    case 80: return index_scores_kernel<80>;
    case 96: return index_scores_kernel<96>;
    case 112: return index_scores_kernel<112>;
    case 128: return index_scores_kernel<128>;
  }
  return index_scores_kernel<0>;
}

// SMs of the current device, once the kernels have their shared memory granted on it; 0 on failure.
int sms_on(int device) {
  static std::mutex mu;
  static int cached[128] = {0};
  if (device < 0 || device >= 128) return 0;
  std::lock_guard<std::mutex> lock(mu);
  if (cached[device]) return cached[device];
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
  for (int heads : {8, 16, 32, 48, 64, 80, 96, 112, 128})
    if (cudaFuncSetAttribute(kernel_for(heads), cudaFuncAttributeMaxDynamicSharedMemorySize,
                             int(kSharedBytes)) != cudaSuccess)
      return 0;
  cached[device] = n;
  return n;
}

}  // namespace index_scores
}  // namespace tq

extern "C" int32_t tq_index_scores(const TqIndexScoresSpec* spec, int32_t* device_flags,
                                   void* stream, TqContractError* err) {
  using namespace tq::index_scores;
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  const int32_t st = tq::index_scores_validate(spec, err);
  if (st != TQ_OK) return st;
  const TqIndexScoresSpec& s = *spec;
  if (s.q.shape[0] == 0) return fail(nullptr, TQ_OK);
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return fail("device", TQ_ERR_CUDA);
  const int sms = sms_on(device);
  if (sms <= 0) return fail("device", TQ_ERR_CUDA);
  auto ints = [](const TqTensorSpec& t) { return reinterpret_cast<const int*>(t.device_address); };
  Args a = {};
  a.w = reinterpret_cast<const float*>(s.w.device_address);
  a.page_table = ints(s.page_table);
  a.seq_id = ints(s.seq_id);
  a.q_pos = ints(s.q_pos);
  a.kv_len = ints(s.kv_len);
  a.scores = reinterpret_cast<uint8_t*>(s.scores.device_address);
  a.flags = device_flags;
  a.score_stride = (long long)s.scores.strides_bytes[0];
  a.tokens = int(s.q.shape[0]);
  a.heads = int(s.q.shape[1]);
  a.sequences = int(s.page_table.shape[0]);
  a.slots = int(s.page_table.shape[1]);
  a.pages = int(s.kv.shape[0]);
  a.columns = int(s.scores.shape[1]);
  a.pack = a.heads % 16 == 0;
  a.sub = kColumns / a.heads < kSubTokens ? kColumns / a.heads : kSubTokens;
  CUtensorMap tm_q, tm_k, tm_s;
  const void* codes = reinterpret_cast<const void*>(s.q.device_address);
  // A pool without pages has no memory to describe: every page reads past the end of one row of q.
  const uint64_t rows = a.pages ? uint64_t(a.pages) * kPageRows : 1;
  const uint64_t stride = a.pages ? s.kv.strides_bytes[1] : kDim;
  const uint8_t* keys = reinterpret_cast<const uint8_t*>(a.pages ? s.kv.device_address : s.q.device_address);
  a.nowhere = int(rows);
  if (!encode_rows(&tm_q, codes, s.q.shape[0] * s.q.shape[1], kDim, uint32_t(a.heads)) ||
      !encode_rows(&tm_k, keys, rows, stride, kPageRows) ||
      !encode_scales(&tm_s, a.pages ? keys + kDim : keys, rows, stride))
    return fail("tensor map", TQ_ERR_CUDA);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(sms), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = kSharedBytes;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel_for(a.heads), tm_q, tm_k, tm_s, a);
  if (e != cudaSuccess) return fail("launch", TQ_ERR_CUDA);
  return fail(nullptr, TQ_OK);
}
