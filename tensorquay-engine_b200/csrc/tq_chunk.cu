// Chunk attention (tq_mla_chunk): each sequence's chunk of new tokens over its paged latent rows,
// with per-head keys and values expanded from them once per call:
//   k[n, h] = bf16(latent[n] . w_uk[h]^T) | rope[n]      v[n, h] = bf16(latent[n] . w_uv[h]^T)
//   out[t, h] = softmax_n(scale * q[t, h] . k[n, h]) v[n, h],  n < min(kv_len, q_pos[t] + 1)
//
// Launches, in order on the caller's stream:
//   1. plan_kernel    one block: each sequence's cached rows laid end to end in a compact row space
//                     (every sequence padded to kRowTile rows) and its query blocks of kQueryTile
//                     tokens.
//   2. gather_kernel  the cached rows through the page table into that space, as bf16 (FP8 rows
//                     dequantized and rounded once, as this library's other attention takes them:
//                     a scale belongs to 128 values of a row, so it does not come out of the
//                     expansion's sum over all 512): zeros past kv_len and for a row that is not
//                     finite, so that neither stale rows nor such a row can reach an output that
//                     does not see it through 0 * NaN. The first such row of a sequence is kept:
//                     the outputs of the tokens that see it become NaN at the end. One block of
//                     its grid cuts the query blocks into pieces of the row tiles that they see.
//   3. expand_kernel  k and v of every head from the compact rows.
//   4. attend_kernel  attention of every (query block, head); where those are few, each is split
//                     into pieces of its row tiles, and
//   5. join_kernel    merges the pieces by their log sums.
// Heads are taken in passes that bound the scratch of step 3 (kScratchBytes).

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <mutex>

#include "tq_contracts.h"
#include "tq_ptx.cuh"
#include "tq_tensor_map.h"

namespace tq {
namespace chunk {

constexpr int kPage = 64;
constexpr int kLatent = 512;
constexpr int kRopeDim = 64;
constexpr int kRowTile = 128;    // keys per attention step; sequences are padded to it
constexpr int kQueryTile = 256;  // query tokens of one attention unit
// Keys and values of one pass over the heads. It bounds the workspace on a GPU that also holds the
// cache and keeps the serving sizes in one pass; smaller passes, whose keys and values would stay in
// L2, are not measured.
constexpr uint64_t kScratchBytes = 8ull << 30;
// Splitting: at most this many units once split, about four per CTA pair (their partial outputs are
// kept in the workspace), and what a piece costs beside its tiles (query load, pipeline fill,
// output), in tiles.
constexpr int kSplitUnits = 320;
constexpr int kPieceCost = 4;

enum Header : int {
  kHdrError = 0,
  kHdrRows = 1,    // compact rows in use (padded)
  kHdrBlocks = 2,  // query blocks
  kHdrPieces = 3,  // pieces of all blocks: units of one head
  kHdrSplit = 4,   // 1 if some block has more than one piece
  kHdrNext = 8,    // [128] next unit of each pass over the heads
  kHdrWords = 136
};

// One query block of one sequence.
struct Block {
  int row0, rows;       // query tokens
  int key0, tiles;      // first compact row, row tiles seen
  int seq;
  int piece0, pieces;   // its pieces
};

// Row tiles tile0 .. tile0 + tiles - 1 of a block.
struct __align__(16) Piece {
  int row0, rows, key0, tile0;
  int tiles, seq, whole, index;  // whole: the block's only piece; index: in block order
};

struct Work {
  int* header;
  int* seq_key0;   // [S + 1] first compact row of each sequence
  int* seq_keys;   // [S] cached rows in use
  int* seq_block;  // [S + 1] first query block of each sequence
  int* seq_spoilt; // [S] first cached row that is not finite (INT_MAX: none)
  Block* blocks;
  Piece* pieces;    // in block order
  Piece* order;     // in the order in which they run
  float* part_out;  // f32 [units, kQueryTile, Dv] of split blocks, each normalised
  float* part_lse;  // f32 [units, kQueryTile] base-2 log sums
  uint16_t* rows;   // bf16 [cap, 512]
  uint16_t* rope;   // bf16 [cap, 64]
  uint16_t* k;      // bf16 [heads of a pass, cap, Dn]
  uint16_t* v;      // bf16 [heads of a pass, cap, Dv]
};

struct Args {
  Work w;
  const uint8_t* q;
  const uint8_t* kv;
  const uint16_t* w_uk;
  const uint16_t* w_uv;
  const int* page_table;
  const int* q_start;
  const int* q_pos;
  const int* kv_len;
  uint8_t* out;
  float* lse;  // may be null
  long long out_st, out_sh, row_stride;           // bytes
  int tokens, heads, seqs, slots, pages, cap, max_blocks;
  int head0, pass_heads, pass;
  int split_units;  // most units of a pass after splitting; 0: blocks are not split
  int pairs;
  int dn, dr, dv, fp8, out_f32;
  float scale_log2;
};

// ------------------------------------------------------------------------------ plan
__device__ __forceinline__ int warp_inclusive(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Inclusive sum over the kWarps warps of a block.
template <int kWarps>
__device__ __forceinline__ int block_inclusive(int v, int* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int inc = warp_inclusive(v);
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  if (warp == 0) part[lane] = warp_inclusive(lane < kWarps ? part[lane] : 0);
  __syncthreads();
  const int out = inc + (warp ? part[warp - 1] : 0);
  __syncthreads();
  return out;
}

__device__ __forceinline__ int last_at_or_below(const int* start, int n, int x) {
  int b = 0, e = n;
  while (e - b > 1) {
    const int m = (b + e) >> 1;
    if (start[m] <= x) b = m; else e = m;
  }
  return b;
}

__global__ void __launch_bounds__(1024) plan_kernel(const Args a) {
  __shared__ int part[32];
  __shared__ int s_rows, s_blocks, s_over;
  const Work& w = a.w;
  const int tid = threadIdx.x;
  ptx::grid_dependency_wait();
  if (tid < kHdrWords) w.header[tid] = 0;
  if (tid == 0) { s_rows = 0; s_blocks = 0; s_over = 0; }
  __syncthreads();
  int bad = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += 1024) {
    const int s = s0 + tid;
    int keys = 0, blocks = 0;
    if (s < a.seqs) {
      const int b = a.q_start[s], e = a.q_start[s + 1], len = a.kv_len[s];
      int n = e - b;
      if (b < 0 || e < b || e > a.tokens) {
        // Sequences that overlap would write each other's outputs: the whole call is left out.
        bad |= TQ_DEV_SEQ_RANGE;
        s_over = 1;
        n = 0;
      }
      if (n > 0) {
        const long long room = (long long)kPage * a.slots;
        keys = max(len, 0);
        if (keys > room) {
          keys = int(room);
          bad |= TQ_DEV_TABLE_SHORT;
        }
        // A sequence past the bound alone; keeps the sums below in range.
        if (keys > a.cap) { s_over = 1; keys = 0; }
      }
      blocks = (n + kQueryTile - 1) / kQueryTile;
    }
    const int padded = (keys + kRowTile - 1) / kRowTile * kRowTile;
    const int rows_end = block_inclusive<32>(padded, part);
    const int blocks_end = block_inclusive<32>(blocks, part);
    const int rows0 = s_rows, blocks0 = s_blocks;
    __syncthreads();
    // 1024 sequences of at most cap <= 2^25 rows may pass 2^31: a warp's 32 are summed in 64 bits
    // below, and 32 warps within cap stay below 2^30.
    if (s < a.seqs) {
      w.seq_key0[s] = rows0 + rows_end - padded;
      w.seq_keys[s] = keys;
      w.seq_spoilt[s] = INT_MAX;
      w.seq_block[s] = blocks0 + blocks_end - blocks;
    }
    long long sum = padded;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if ((tid & 31) == 0 && sum > a.cap) s_over = 1;
    if (rows_end < 0 || rows_end > a.cap - rows0 || blocks0 + blocks_end > a.max_blocks)
      s_over = 1;
    if (tid == 1023) {
      s_rows = rows0 + rows_end;
      s_blocks = blocks0 + blocks_end;
    }
    __syncthreads();
    const int over = s_over;
    __syncthreads();  // before the next round may set it
    if (over) break;
  }
  if (bad) atomicOr(w.header + kHdrError, bad);
  if (s_over) {
    const int range = __syncthreads_or(bad & TQ_DEV_SEQ_RANGE);
    if (tid == 0) {
      if (!range) atomicOr(w.header + kHdrError, TQ_DEV_WORK_OVERFLOW);
      w.header[kHdrRows] = 0;
      w.header[kHdrBlocks] = 0;
    }
    return;
  }
  if (tid == 0) {
    w.seq_key0[a.seqs] = s_rows;
    w.seq_block[a.seqs] = s_blocks;
    w.header[kHdrRows] = s_rows;
    w.header[kHdrBlocks] = s_blocks;
  }
}

// The query blocks and their pieces, by one block of the gather's grid: only the attention reads
// them, so they run beside the gathering of rows (24 tokens over 124 rows, replayed from a graph:
// 27 us with this in plan_kernel, 22 here and with the attention's first fetch ahead of its wait).
constexpr int kGatherThreads = 256, kGatherWarps = kGatherThreads / 32;

struct PlanShared {
  // The first sequences, blocks and pieces again, near: the steps read each other's results.
  static constexpr int kSeqs = 256, kBlocks = 1024;
  int part[32], at, split;
  int q0[kSeqs + 1], block[kSeqs + 1], key0[kSeqs], keys[kSeqs];
  int tiles[kBlocks], length[kBlocks];  // of blocks; of pieces
  int cost[32], len[32];
};

__device__ void plan_pieces(const Args& a, PlanShared& sh) {
  const Work& w = a.w;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int blocks = w.header[kHdrBlocks];
  const bool near = a.seqs <= PlanShared::kSeqs;
  if (near) {
#pragma unroll 1
    for (int s = tid; s <= a.seqs; s += kGatherThreads) {
      sh.q0[s] = a.q_start[s];
      sh.block[s] = w.seq_block[s];
      if (s < a.seqs) {
        sh.key0[s] = w.seq_key0[s];
        sh.keys[s] = w.seq_keys[s];
      }
    }
  }
  if (tid == 0) { sh.at = 0; sh.split = 0; }
  __syncthreads();
  const int* seq_block = near ? sh.block : w.seq_block;
  const int* q_start = near ? sh.q0 : a.q_start;
  const int* seq_keys = near ? sh.keys : w.seq_keys;
  const int* seq_key0 = near ? sh.key0 : w.seq_key0;
  // Query blocks, one warp each: the tiles that its furthest-seeing token sees.
#pragma unroll 1
  for (int b = warp; b < blocks; b += kGatherWarps) {
    const int s = last_at_or_below(seq_block, a.seqs, b);
    const int row0 = q_start[s] + (b - seq_block[s]) * kQueryTile;
    const int rows = min(kQueryTile, q_start[s + 1] - row0);
    int far = -1;
#pragma unroll
    for (int i = 0; i < kQueryTile; i += 32)
      if (i + lane < rows) far = max(far, a.q_pos[row0 + i + lane]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) far = max(far, __shfl_xor_sync(0xFFFFFFFFu, far, o));
    const int keys = seq_keys[s];
    const int tiles = ((far >= keys ? keys : far + 1) + kRowTile - 1) / kRowTile;
    if (lane == 0) {
      if (b < PlanShared::kBlocks) sh.tiles[b] = tiles;
      else w.blocks[b].tiles = tiles;
    }
  }
  __syncthreads();
  auto tiles_of = [&](int b) { return b < PlanShared::kBlocks ? sh.tiles[b] : w.blocks[b].tiles; };
  // The most tiles that a piece gets. Each k below 32 weighs cutting the longest block into k + 1:
  // the rounds that the CTA pairs need for all units, each as long as such a piece.
  int len = 1 << 30;  // whole blocks
  if (a.split_units) {
    int longest = 1;
#pragma unroll 1
    for (int b = lane; b < blocks; b += 32) longest = max(longest, tiles_of(b));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      longest = max(longest, __shfl_xor_sync(0xFFFFFFFFu, longest, o));
#pragma unroll 1
    for (int k = warp; k < 32; k += kGatherWarps) {
      const int cut = (longest + k) / (k + 1);
      int count = 0;
#pragma unroll 1
      for (int b = lane; b < blocks; b += 32) count += max(1, (tiles_of(b) + cut - 1) / cut);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) count += __shfl_xor_sync(0xFFFFFFFFu, count, o);
      if (lane == 0) {
        const int units = count <= a.split_units ? count * a.pass_heads : INT_MAX;
        sh.len[k] = cut;
        sh.cost[k] = units <= a.split_units ? (units + a.pairs - 1) / a.pairs * (cut + kPieceCost) +
                                                  (k ? 2 * kPieceCost : 0)
                                            : INT_MAX;
      }
    }
    __syncthreads();
    int cost = sh.cost[lane], best = lane;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const int c = __shfl_xor_sync(0xFFFFFFFFu, cost, o);
      const int k = __shfl_xor_sync(0xFFFFFFFFu, best, o);
      if (c < cost || (c == cost && k < best)) {
        cost = c;
        best = k;
      }
    }
    if (best) len = sh.len[best];
  }
  // Number the pieces.
#pragma unroll 1
  for (int b0 = 0; b0 < blocks; b0 += kGatherThreads) {
    const int b = b0 + tid;
    int n = 0, tiles = 0;
    if (b < blocks) {
      tiles = tiles_of(b);
      n = max(1, (tiles + len - 1) / len);
    }
    const int end = block_inclusive<kGatherWarps>(n, sh.part), at = sh.at + end - n;
    if (b < blocks) {
      const int s = last_at_or_below(seq_block, a.seqs, b);
      const int row0 = q_start[s] + (b - seq_block[s]) * kQueryTile;
      const int rows = min(kQueryTile, q_start[s + 1] - row0), key0 = seq_key0[s];
      w.blocks[b] = {row0, rows, key0, tiles, s, at, n};
      // Pieces of one length, the last ones shorter.
      const int each = max(1, (tiles + n - 1) / n);
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int length = max(0, min(each, tiles - i * each));
        w.pieces[at + i] = {row0, rows, key0, i * each, length, s, n == 1, at + i};
        if (at + i < PlanShared::kBlocks) sh.length[at + i] = length;
      }
      if (n > 1) sh.split = 1;
    }
    __syncthreads();
    if (tid == kGatherThreads - 1) sh.at = at + n;
    __syncthreads();
  }
  // The order in which a head's pieces run: the longest first, so that the last ones to run are
  // short (up to kBlocks pieces; more are left in their order).
  const int pieces = sh.at;
#pragma unroll 1
  for (int i = tid; i < pieces; i += kGatherThreads) {
    int rank = i;
    if (pieces <= PlanShared::kBlocks) {
      const int mine = sh.length[i];
      rank = 0;
#pragma unroll 4
      for (int k = 0; k < pieces; ++k) {
        const int other = sh.length[k];
        rank += other > mine || (other == mine && k < i);
      }
    }
    w.order[rank] = w.pieces[i];
  }
  if (tid == 0) {
    w.header[kHdrPieces] = pieces;
    w.header[kHdrSplit] = sh.split;
  }
}

// ------------------------------------------------------------------------------ gather
__device__ __forceinline__ bool finite_bf16x2(uint32_t u) {
  return (u & 0x7F80u) != 0x7F80u && (u & 0x7F800000u) != 0x7F800000u;
}

// Block 0 plans the pieces. The others take kGatherRows compact rows each, four rows a warp with
// all their loads in flight: lane i takes the 16 latent values from 16 i on, and two of the 64 RoPE
// values. What bounds it: the chain of dependent loads (sequence, page, row) for small calls, so
// rows are spread over many blocks; HBM for large ones (a row read and written once).
constexpr int kGatherRows = 4 * kGatherWarps;
static_assert(kRowTile % kGatherRows == 0, "a block's rows lie in one sequence");

__global__ void __launch_bounds__(kGatherThreads) gather_kernel(const Args a) {
  __shared__ PlanShared sh;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const Work& w = a.w;
  if (blockIdx.x == 0) {
    plan_pieces(a, sh);
    return;
  }
  const int r0 = int(blockIdx.x - 1) * kGatherRows;
  if (r0 >= w.header[kHdrRows]) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int s = last_at_or_below(w.seq_key0, a.seqs, r0);
  const int p0 = r0 - w.seq_key0[s] + warp * 4, keys = w.seq_keys[s];
  int page[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    page[i] = p0 + i < keys ? a.page_table[(long long)s * a.slots + (p0 + i) / kPage] : 0;
  uint4 v0[4], v1[4];
  uint32_t rp[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v0[i] = v1[i] = make_uint4(0, 0, 0, 0);
    rp[i] = 0;
    const bool live = p0 + i < keys, known = page[i] >= 0 && page[i] < a.pages;
    if (live && known) {
      const uint8_t* src = a.kv + ((long long)page[i] * kPage + (p0 + i) % kPage) * a.row_stride;
      if (a.fp8) {
        v0[i] = *reinterpret_cast<const uint4*>(src + 16 * lane);
        rp[i] = *reinterpret_cast<const uint32_t*>(src + kLatent + 4 * (lane >> 3));  // scale
      } else {
        v0[i] = *reinterpret_cast<const uint4*>(src + 32 * lane);
        v1[i] = *reinterpret_cast<const uint4*>(src + 32 * lane + 16);
        if (a.dr) rp[i] = *reinterpret_cast<const uint32_t*>(src + 2 * kLatent + 4 * lane);
      }
    }
    if (live && !known && lane == 0) atomicOr(w.header + kHdrError, TQ_DEV_PAGE_RANGE);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (a.fp8) {
      const uint4 c = v0[i];
      const float sc = __uint_as_float(rp[i]);
      rp[i] = 0;
      v0[i] = make_uint4(
          ptx::e4m3x2_scaled_bf16x2(c.x & 0xFFFF, sc), ptx::e4m3x2_scaled_bf16x2(c.x >> 16, sc),
          ptx::e4m3x2_scaled_bf16x2(c.y & 0xFFFF, sc), ptx::e4m3x2_scaled_bf16x2(c.y >> 16, sc));
      v1[i] = make_uint4(
          ptx::e4m3x2_scaled_bf16x2(c.z & 0xFFFF, sc), ptx::e4m3x2_scaled_bf16x2(c.z >> 16, sc),
          ptx::e4m3x2_scaled_bf16x2(c.w & 0xFFFF, sc), ptx::e4m3x2_scaled_bf16x2(c.w >> 16, sc));
    }
    const bool ok = finite_bf16x2(v0[i].x) && finite_bf16x2(v0[i].y) && finite_bf16x2(v0[i].z) &&
                    finite_bf16x2(v0[i].w) && finite_bf16x2(v1[i].x) && finite_bf16x2(v1[i].y) &&
                    finite_bf16x2(v1[i].z) && finite_bf16x2(v1[i].w) && finite_bf16x2(rp[i]);
    if (!__all_sync(0xFFFFFFFFu, ok)) {
      v0[i] = v1[i] = make_uint4(0, 0, 0, 0);
      rp[i] = 0;
      if (lane == 0) atomicMin(w.seq_spoilt + s, p0 + i);
    }
    const long long r = r0 + warp * 4 + i;
    uint16_t* dst = w.rows + r * kLatent + 16 * lane;
    *reinterpret_cast<uint4*>(dst) = v0[i];
    *reinterpret_cast<uint4*>(dst + 8) = v1[i];
    if (a.dr) *reinterpret_cast<uint32_t*>(w.rope + r * kRopeDim + 2 * lane) = rp[i];
  }
}

// ------------------------------------------------------------------------------ waits
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr uint32_t kWaitPolls = 1u << 26;

// Bounded waits of one role of a CTA pair. What they wait for lies in TMEM or is written and read
// by the asynchronous proxies (TMA, MMA), ordered by the barriers and tcgen05 fences themselves: no
// wait or arrival here needs the cluster-scope release or acquire of generic memory, which cost a
// memory barrier per tile (2.0 of 9.8 warps stalled in it). The first wait that runs out writes its
// barrier into both CTAs' abort words, and every later wait of the pair returns false soon; the
// error flag is set at the end, in one place: a wait is inlined at two dozen places, and every
// instruction of it competes for the instruction caches with the loops that it stands in.
struct Waiter {
  uint32_t abort;  // shared address of this CTA's abort word
  bool failed;

  // Polls: a suspended wait (mbarrier.try_wait) can resume long after its phase completed, or not
  // within its bound.
  __device__ bool on(uint32_t bar, uint32_t parity) {
    if (failed) return false;
    uint64_t t0 = 0;  // reading the timer is slow: only a wait of many polls does
    for (uint32_t i = 1;; ++i) {
      if (ptx::mbar_test(bar, parity)) return true;
      if ((i & 1023) == 0) {
        if (ptx::ld_shared_u32(abort)) {
          failed = true;
          return false;
        }
        const uint64_t now = ptx::global_timer_ns();
        if (t0 == 0) t0 = now;
        if (i >= kWaitPolls || now - t0 > kWaitNs) {
          ptx::st_cluster_u32(ptx::map_peer(abort, 0), bar);
          ptx::st_cluster_u32(ptx::map_peer(abort, 1), bar);
          failed = true;
          return false;
        }
      }
    }
  }
  // For a converged warp: all lanes agree.
  __device__ bool all(uint32_t bar, uint32_t parity) {
    const bool ok = on(bar, parity);
    if (__all_sync(0xFFFFFFFFu, ok)) return true;
    failed = true;
    return false;
  }
  // The end of an aborted CTA: the error flag, and a millisecond in which the pair's copies and
  // MMAs in flight land.
  __device__ void settle(int* header) {
    if (!ptx::ld_shared_u32(abort)) return;
    if (threadIdx.x == 0) atomicOr(header + kHdrError, TQ_DEV_WAIT_TIMEOUT);
    const uint64_t t0 = ptx::global_timer_ns();
    for (uint32_t i = 0; i < (1u << 20) && ptx::global_timer_ns() - t0 < 1000000ull; ++i) {
    }
  }
};

// ------------------------------------------------------------------------------ expand
// [k | v] = rows . weights^T on CTA pairs: an item is 256 compact rows by 256 output columns (one
// head's k and v where both are 128 wide, one head's k or v where they are 256 wide), K = 512.
//
// What bounds it: the tensor cores, 2 x 256 x 512 FLOP a row and column block against 1 KB read and
// 512 B written a row. The weights of a column block (256 x 512, half of them in each CTA of the
// pair) therefore stay in shared memory while the pair walks over row tiles; only the rows
// stream (16 KB boxes through a ring), half as many bytes per FLOP as with both operands streamed.
// Two TMEM accumulators: the epilogue of one item runs under the MMAs of the next. The f32 sums are
// rounded to bf16, the type of the attention's operands and of a model's own keys and values (each
// such rounding adds 0.0017 in the relative 2-norm, as much as the output's own). Sums past bf16's
// range become its largest value: an infinite value would reach the tile's other query rows as
// 0 * infinity. NaN does not arise from finite operands: a single product does not overflow inside
// the tensor core and an infinite partial sum stays infinite (rows of 3e38 against weights of both
// signs and magnitudes up to 3e38).
namespace expand {

constexpr int kThreads = 256;  // warp 0 loads, warp 1 MMA, warps 4-7 epilogue
constexpr int kChunks = kLatent / 64;
constexpr uint32_t kBox = 128 * 128;  // 128 rows x 64 values
constexpr int kStages = 6;  // what shared memory holds (5: 65492 rows, 32 heads 440 us, now 427)
constexpr uint32_t kSmW = 0;                              // [kChunks] boxes of weights
constexpr uint32_t kSmA = kChunks * kBox;                 // [kStages] boxes of rows
constexpr uint32_t kSmBars = kSmA + kStages * kBox;
constexpr int kBarAFull = 0, kBarAEmpty = kStages, kBarWFull = 2 * kStages;
constexpr int kBarWEmpty = kBarWFull + kChunks, kBarAccFull = kBarWEmpty + kChunks;
constexpr int kBarAccEmpty = kBarAccFull + 2, kBarDrain = kBarAccEmpty + 2, kBars = kBarDrain + 1;
constexpr uint32_t kSmMisc = kSmBars + 8 * kBars;  // TMEM address, abort word
constexpr uint32_t kSmBytes = kSmMisc + 16 + 1024;
static_assert(kSmBytes <= 232448, "shared memory per CTA");

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    expand_kernel(const __grid_constant__ CUtensorMap tm_rows,
                  const __grid_constant__ CUtensorMap tm_uk,
                  const __grid_constant__ CUtensorMap tm_uv, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(ptx::cluster_rank());
  const int pair = int(blockIdx.x) >> 1, pairs = int(gridDim.x) >> 1;
  auto bar = [&](int i) { return base + kSmBars + 8u * uint32_t(i); };
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(sm + kSmMisc);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kBars; ++i) ptx::mbar_init(bar(i), 1);
    for (int b = 0; b < 2; ++b) ptx::mbar_init(bar(kBarAccEmpty + b), 8);  // 4 warps of each CTA
    tmem_holder[1] = 0;  // the abort word
    ptx::fence_mbar_init_cluster();
    ptx::tma_prefetch_desc(&tm_rows);
    ptx::tma_prefetch_desc(&tm_uk);
    ptx::tma_prefetch_desc(&tm_uv);
  }
  // The allocation is one operation of both CTAs: neither may ask for it before the other runs.
  __syncwarp();
  ptx::cluster_sync_relaxed();
  if (warp == 1) {
    ptx::tmem_alloc_pair(ptx::smem_addr(tmem_holder), 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  ptx::cluster_sync();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  Waiter wt{base + kSmMisc + 4, false};

  // Column blocks (a head, or a head's k or v) by row tiles, one contiguous range per pair. The
  // first one's column block, floor(floor(tiles * blocks * pair / pairs) / tiles), does not depend
  // on the number of row tiles, so its weights load while the rows are still being gathered.
  const int per_head = (a.dn + a.dv) / 256, columns = per_head * a.pass_heads;
  auto load_weights = [&](int g, int c) {
    const bool from_v = per_head == 2 ? (g & 1) != 0 : rank != 0;
    if (rank == 0) ptx::mbar_expect_tx(bar(kBarWFull + c), 2 * kBox);
    ptx::tma_load_3d_pair(base + kSmW + c * kBox, from_v ? &tm_uv : &tm_uk,
                          ptx::map_peer(bar(kBarWFull + c), 0), c * 64,
                          per_head == 2 ? rank * 128 : 0,
                          a.head0 + (per_head == 2 ? g >> 1 : g));
  };
  if (threadIdx.x == 0)
    for (int c = 0; c < kChunks; ++c) load_weights(columns * pair / pairs, c);
  // The number of rows is in place ahead of the wait for the gather: its blocks let this grid start
  // after their own wait for the plan.
  const int rows_used = __ldcg(a.w.header + kHdrRows);
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  // At most kScratchBytes of 128 KB items, or the 2^17 row tiles of one head: 32 bits hold the
  // products with the pairs.
  const uint32_t tiles = uint32_t(rows_used + 255) / 256;
  const uint32_t items = tiles * uint32_t(columns);
  const uint32_t first = items * uint32_t(pair) / uint32_t(pairs);
  const uint32_t last = items * uint32_t(pair + 1) / uint32_t(pairs);
  const uint32_t g0 = tiles ? first / tiles : 0u, tile0 = first - g0 * tiles;
  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, blocks = 0;
      uint32_t g = g0, tile = tile0;
      for (uint32_t i = first; i < last && !wt.failed; ++i) {
        const bool fresh = i == first || tile == 0;
        for (int c = 0; c < kChunks; ++c) {
          if (fresh && blocks > 0) {
            if (!wt.on(bar(kBarWEmpty + c), (blocks - 1) & 1u)) break;
            load_weights(int(g), c);
          }
          if (!wt.on(bar(kBarAEmpty + stage), phase ^ 1u)) break;
          if (rank == 0) ptx::mbar_expect_tx(bar(kBarAFull + stage), 2 * kBox);
          ptx::tma_load_2d_pair(base + kSmA + stage * kBox, &tm_rows,
                                ptx::map_peer(bar(kBarAFull + stage), 0), c * 64,
                                int(tile) * 256 + rank * 128);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (fresh) ++blocks;
        if (++tile == tiles) {
          tile = 0;
          ++g;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = ptx::idesc_bf16(256, 256, 0);
      const uint32_t elected = ptx::elect_one();
      uint32_t stage = 0, phase = 0, blocks = 0, n = 0, tile = tile0;
      for (uint32_t i = first; i < last && !wt.failed; ++i, ++n) {
        const bool fresh = i == first || tile == 0, done = i + 1 == last || tile == tiles - 1;
        const uint32_t buf = n & 1u;
        if (n >= 2 && !wt.all(bar(kBarAccEmpty + buf), ((n >> 1) - 1) & 1u)) break;
        ptx::tc_fence_after();
        const uint32_t d = tmem + buf * 256;
        for (int c = 0; c < kChunks; ++c) {
          if (fresh && !wt.all(bar(kBarWFull + c), blocks & 1u)) break;
          if (!wt.all(bar(kBarAFull + stage), phase)) break;
          ptx::tc_fence_after();
          const uint64_t ad = ptx::smem_desc(base + kSmA + stage * kBox, 16, 1024, 2);
          const uint64_t bd = ptx::smem_desc(base + kSmW + c * kBox, 16, 1024, 2);
          ptx::mma_ss_pair_x4(elected, d, ad, bd, idesc, c > 0 ? 1u : 0u);
          ptx::mma_commit_pair(bar(kBarAEmpty + stage));
          if (done) ptx::mma_commit_pair(bar(kBarWEmpty + c));
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        ptx::mma_commit_pair(bar(kBarAccFull + buf));
        if (fresh) ++blocks;
        if (++tile == tiles) tile = 0;
      }
      // A pair without items has its weights in flight all the same.
      if (first >= last)
        for (int c = 0; c < kChunks; ++c) wt.all(bar(kBarWFull + c), 0);
      ptx::mma_commit_pair(bar(kBarDrain));
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int quad = warp & 3, row = quad * 32 + lane;
    uint32_t n = 0, g = g0, tile = tile0;
    for (uint32_t i = first; i < last; ++i, ++n) {
      const uint32_t buf = n & 1u;
      if (!wt.all(bar(kBarAccFull + buf), (n >> 1) & 1u)) break;
      ptx::tc_fence_after();
      const long long r = (long long)tile * 256 + rank * 128 + row;
      const uint32_t h = per_head == 2 ? g >> 1 : g;  // of this pass
      uint16_t* kd = a.w.k + ((long long)h * a.cap + r) * a.dn;
      uint16_t* vd = a.w.v + ((long long)h * a.cap + r) * a.dv;
      uint16_t* lo = per_head == 2 ? ((g & 1) ? vd : kd) : kd;
      uint16_t* hi = per_head == 2 ? lo + 128 : vd;
      const uint32_t src = tmem + buf * 256 + (uint32_t(quad * 32) << 16);
#pragma unroll 2
      for (int c = 0; c < 256; c += 32) {
        uint32_t x[32], y[16];
        ptx::tmem_ld32(src + c, x);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j)
          y[j] = ptx::pack_bf16x2_finite(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1]));
        uint16_t* dst = c < 128 ? lo + c : hi + (c - 128);
        ptx::st_global_v8(dst, y);
        ptx::st_global_v8(dst + 16, y + 8);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster_relaxed(ptx::map_peer(bar(kBarAccEmpty + buf), 0));
      if (++tile == tiles) {
        tile = 0;
        ++g;
      }
    }
  }
  // Every commit of the leader has arrived in both CTAs before either leaves. One warp polls for
  // it; the others go on to the cluster barrier, which costs no issue slots.
  if (warp == 0) wt.on(bar(kBarDrain), 0);
  wt.settle(a.w.header);
  __syncwarp();
  ptx::tc_fence_before();
  ptx::cluster_sync();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem, 512);
    __syncwarp();
  }
  ptx::cluster_sync_relaxed();  // both CTAs run until both have given their columns back
}

}  // namespace expand

// ------------------------------------------------------------------------------ attend
// Attention of one unit (a block of kQueryTile query tokens, one head) on a CTA pair, row tiles of
// kRowTile keys one after the other with the running maximum and sum of a softmax:
//   S_j = Q K_j^T (M = 256 over the pair, N = 128)  ->  P_j = exp2(c S_j - c m)  ->  O += P_j V_j
// Each CTA holds its 128 query rows of S, P and O in TMEM and Q in shared memory; of B operands
// it loads half: 64 of a tile's keys for QK^T, half the value columns for PV. So a pair moves
// K_j and V_j once for 256 queries, and the shared memory left holds several tiles ahead.
//   warps 0, 2  TMA loads of this CTA's halves of Q and K, and of V; their bytes complete on the
//               leader's barriers (one warp for all waited for V's stages before K's next one)
//   warp 3      fetches the next unit's rows for the softmax warps
//   warp 1      (leader) all MMAs. S_j has kS buffers in TMEM: S_{j+kS} is issued right after
//               PV_j, whose P_j lies in the same columns; MMAs run in issue order. PV_j starts
//               on the first 64 keys while the other half's exponentials run. A softmax warp may
//               be several tiles ahead of PV, so the completion of PV_j has a barrier per buffer:
//               a waiter has seen S_j, which lies behind PV_{j-kS}, and its phase is the next.
//   warps 4-11  softmax, a thread a row, in two groups of four warps. With three score buffers (192
//               columns) the groups take the tiles in turn, so that one group's exponentials run
//               under the other's loads, maxima and waits, and the row's reference maximum passes
//               from group to group through shared memory; with two (256 columns) both work on
//               every tile, half of its keys each, and exchange their maxima (Shape::kHalves). P
//               goes to TMEM as bf16 over the scores. The reference moves only when it would grow
//               by more than 2^8 (kSlack): then O is rescaled, after the last PV; otherwise p
//               stays below 2^8 and the final division makes it exact. Each thread sums its own
//               keys' weights; the two sums of a row meet at the unit's end.
//
// What bounds it: per 128 x 128 tile and CTA the tensor cores need (2 (Dqk + Dv) 128 128) / 8192
// cycles (1280 at 192 + 128, 2048 at 256 + 256), the exponentials 128 128 / 16 = 1024. Measured:
// 64 heads of 192 + 128, 2048 tokens over 4096 cached rows 376 us, the tensor pipe active in 65% of
// the cycles and the exponentials' unit in 52%; 64 heads of 256 + 256, 4096 tokens 403 us, 80% and
// 40%. What is lost lies in the handoffs between a tile's scores, weights and product, and in
// instruction fetch: the roles are seven different loops that share the caches, so that code added
// to any of them (unrolled loops, weights by a polynomial, a second MMA warp) cost more than it
// gained. In long calls the power limit holds the clock at 1.4 GHz of 1.97.
namespace attend {

constexpr int kThreads = 384;
constexpr float kSlack = 8.f;  // log2 units
// A pair takes its next unit when the load warp comes to this many tiles before the end of the one
// at work, itself up to three tiles ahead: late enough that units go to the pairs that are free
// (taken a whole unit ahead, pairs ended 357 to 432 us into the attention of 4096 tokens, now 398
// to 408), early enough that the unit's rows are there in time (1, 2 and 4 measure alike).
constexpr int kClaimAhead = 2;

// A unit as the warps of a CTA take it, fetched ahead by warp 3. tiles < 0: there are no more.
struct Info {
  int seen[128];  // keys that each of this CTA's query rows sees; kSpoilt: one is not finite
  int row0, rows, key0, tile0;
  int tiles, whole, head, slot;  // head of this pass; slot of a piece's partial output
};
constexpr int kSpoilt = 1 << 30;
// A warp's 32 output rows of 64 bytes, 80 bytes apart (16-byte accesses without bank conflicts).
constexpr uint32_t kTurnBytes = 32 * 80;

template <int kDq, int kDv>
struct Shape {
  static constexpr int kQChunks = kDq / 64;
  static constexpr int kVChunks = kDv / 128;              // of this CTA's half
  static constexpr int kS = (512 - kDv) / 128 < 3 ? (512 - kDv) / 128 : 3;  // score buffers
  static constexpr int kKv = kS;                         // K and V stages each
  static constexpr uint32_t kQBytes = kQChunks * 128 * 128;
  static constexpr uint32_t kKBytes = kQChunks * 64 * 128;
  static constexpr uint32_t kVBytes = kVChunks * 128 * 128;
  static constexpr uint32_t kSmK = kQBytes;
  static constexpr uint32_t kSmV = kSmK + kKv * kKBytes;
  static constexpr uint32_t kSmExch = kSmV + kKv * kVBytes;  // f32 [6][128], int [4], mail
  static constexpr uint32_t kSmInfo = kSmExch + 3104;         // 2 x Info
  static constexpr uint32_t kSmTurn = kSmInfo + 2 * sizeof(Info);  // output rows, kTurnBytes a warp
  static constexpr uint32_t kSmBars = kSmTurn + 8 * kTurnBytes;
  static constexpr int kQFull = 0, kQEmpty = 1, kKFull = 2, kKEmpty = kKFull + kKv;
  static constexpr int kVFull = kKEmpty + kKv, kVEmpty = kVFull + kKv;
  static constexpr int kSFull = kVEmpty + kKv, kPFull = kSFull + kS;
  static constexpr int kPvDone = kPFull + 2 * kS, kOFree = kPvDone + kS, kDrain = kOFree + 1;
  static constexpr int kInfoFull = kDrain + 1, kInfoEmpty = kInfoFull + 2;
  static constexpr int kMailFull = kInfoEmpty + 2, kMailEmpty = kMailFull + 1;
  static constexpr int kClaim = kMailEmpty + 1;
  static constexpr int kBars = kClaim + 1;
  static constexpr uint32_t kSmMisc = kSmBars + 8 * kBars;
  static constexpr uint32_t kSmBytes = kSmMisc + 16 + 1024;
  static constexpr uint32_t kTmemO = kS * 128;
  // With two score buffers a tile's own chain (scores, softmax, PV, the next scores in the buffer)
  // is the limit, and both softmax groups work on every tile, half of its keys each (4096 tokens,
  // 64 heads of 256: 622 us a call where in turn took 645); with three the groups take the tiles in
  // turn (2 x 2048 tokens, 128 heads of 192: 2030 us, by halves 2117).
  static constexpr bool kHalves = kS == 2;
  // In turn: the quarter of a tile's exponentials after which the turn passes. The earlier, the
  // more the two groups' exponentials overlap and slow each other; the later, the longer a tile
  // takes (after the first quarter 1553 us of attention for 2 x 2048 tokens of 128 heads, after the
  // second 1545).
  static constexpr int kTurn = 1;
  static_assert(kSmBytes <= 232448, "shared memory per CTA");
  static_assert(kTmemO + kDv <= 512, "TMEM columns");
};

// Parities of the N barriers of a ring that every unit enters at its first stage (so that a tile's
// stage is its number within the unit mod N): bit i is the parity of stage i's next use.
template <int N>
struct Phases {
  uint32_t bits = 0;
  // The parity of stage i's next use, which is now taken.
  __device__ uint32_t take(uint32_t i) {
    const uint32_t b = (bits >> i) & 1u;
    bits ^= 1u << i;
    return b;
  }
  // The parity of stage i's use number k from here on.
  __device__ uint32_t at(uint32_t i, int k) const { return ((bits >> i) ^ uint32_t(k)) & 1u; }
  // A unit of `tiles` tiles is over.
  __device__ void pass(int tiles) {
#pragma unroll
    for (int i = 0; i < N; ++i) bits ^= uint32_t(((tiles - i + N - 1) / N) & 1) << i;
  }
};

struct Unit {
  Piece p;
  int head;  // of this pass
};

// Units in the order in which they are taken: head by head, so that the pairs at work at one time
// share the keys and values of few heads in L2, and within a head the longest piece first. The last
// two rounds' worth of heads go piece by piece instead, so that the call ends on short units.
__device__ __forceinline__ Unit unit_at(const Args& a, int u, int pieces, int pairs) {
  const int last = min(a.pass_heads, (2 * pairs + pieces - 1) / pieces);
  const int first = (a.pass_heads - last) * pieces;  // units of the heads before those
  Unit x;
  int piece;
  if (u < first) {
    x.head = u / pieces;
    piece = u - x.head * pieces;
  } else {
    piece = (u - first) / last;
    x.head = a.pass_heads - last + (u - first) - piece * last;
  }
  const int4* src = reinterpret_cast<const int4*>(a.w.order + piece);
  const int4 lo = __ldcg(src), hi = __ldcg(src + 1);
  x.p = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  return x;
}

template <int kDq, int kDv>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    attend_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_rope,
                  const __grid_constant__ CUtensorMap tm_v, const Args a) {
  using C = Shape<kDq, kDv>;
  constexpr bool kRope = kDq == 192;
  constexpr int kNopeChunks = kRope ? 2 : C::kQChunks;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(ptx::cluster_rank());
  const int pairs = int(gridDim.x) >> 1;
  auto bar = [&](int i) { return base + C::kSmBars + 8u * uint32_t(i); };
  auto lead = [&](int i) { return ptx::map_peer(bar(i), 0); };
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(sm + C::kSmMisc);
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kBars; ++i) {
      // P of half a tile: its group's four warps in either CTA; the release of O: all softmax
      // warps.
      const bool joint = i >= C::kPFull && i < C::kPFull + 2 * C::kS;
      // A unit's info: every warp but the one that fetches it and a follower's idle warp 1.
      const bool read = i >= C::kInfoEmpty && i < C::kInfoEmpty + 2;
      ptx::mbar_init(bar(i), joint ? 8 : read ? 11 - rank : i == C::kOFree ? 16 : 1);
    }
    tmem_holder[1] = 0;  // the abort word
    for (int i = 0; i < 4; ++i) reinterpret_cast<int*>(sm + C::kSmExch + 6 * 128 * 4)[i] = 0;
    ptx::fence_mbar_init_cluster();
    ptx::tma_prefetch_desc(&tm_q);
    ptx::tma_prefetch_desc(&tm_k);
    ptx::tma_prefetch_desc(&tm_v);
    if (kRope) ptx::tma_prefetch_desc(&tm_rope);
  }
  // The allocation is one operation of both CTAs: neither may ask for it before the other runs.
  __syncwarp();
  ptx::cluster_sync_relaxed();
  if (warp == 1) {
    ptx::tmem_alloc_pair(ptx::smem_addr(tmem_holder), 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  ptx::cluster_sync();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  Waiter wt{base + C::kSmMisc + 4, false};
  // The expansion lets this grid start after its own wait for the gather, so the plan and the
  // pieces are in place ahead of the wait for the keys and values: warps 0 and 3 fetch the first
  // unit's rows and queries before it (from L2: lines of an earlier call may lie in L1), then they
  // wait like the others. All 512 columns are this CTA's, so they start at 0.
  if (warp != 0 && warp != 3) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
  }
  const int pieces = __ldcg(a.w.header + kHdrPieces), units = pieces * a.pass_heads;
  // The n-th unit, for one lane of a load warp; the MMA warp takes it as a whole.
  struct UnitRef {
    int row0, key0, tiles, head;
  };
  auto next_unit = [&](uint32_t n) -> UnitRef {
    const int slot = int(n & 1u);
    if (!wt.on(bar(C::kInfoFull + slot), (n >> 1) & 1u)) return {0, 0, -1, 0};
    const Info* info = reinterpret_cast<const Info*>(sm + C::kSmInfo) + slot;
    const UnitRef x = {info->row0, info->key0, info->tiles, info->head};
    ptx::mbar_arrive(bar(C::kInfoEmpty + slot));
    return x;
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t useq = 0;
      Phases<C::kKv> free;
      for (uint32_t n = 0;; ++n) {
        const UnitRef x = next_unit(n);
        if (x.tiles < 0) break;
        if (x.tiles) {
          if (!wt.on(bar(C::kQEmpty), (useq & 1u) ^ 1u)) break;
          if (rank == 0) ptx::mbar_expect_tx(bar(C::kQFull), 2 * C::kQBytes);
#pragma unroll
          for (int c = 0; c < C::kQChunks; ++c)
            ptx::tma_load_3d_pair(base + c * 16384, &tm_q, lead(C::kQFull), c * 64,
                                  a.head0 + x.head, x.row0 + rank * 128);
          ++useq;
        }
        if (n == 0) ptx::grid_dependency_wait();
        if (!x.tiles && rank == 0) ptx::mbar_arrive(bar(C::kClaim));
        for (int j = 0; j < x.tiles; ++j) {
          if (j == max(0, x.tiles - kClaimAhead) && rank == 0) ptx::mbar_arrive(bar(C::kClaim));
          const uint32_t st = uint32_t(j % C::kKv), ph = free.take(st) ^ 1u;
          const int key = x.key0 + j * kRowTile;
          if (!wt.on(bar(C::kKEmpty + st), ph)) break;
          if (rank == 0) ptx::mbar_expect_tx(bar(C::kKFull + st), 2 * C::kKBytes);
          const uint32_t kd = base + C::kSmK + st * C::kKBytes;
#pragma unroll
          for (int c = 0; c < kNopeChunks; ++c)
            ptx::tma_load_3d_pair(kd + c * 8192, &tm_k, lead(C::kKFull + st), c * 64,
                                  key + rank * 64, x.head);
          if (kRope)
            ptx::tma_load_2d_pair(kd + 2 * 8192, &tm_rope, lead(C::kKFull + st), 0,
                                  key + rank * 64);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t idesc_qk = ptx::idesc_bf16(256, 128, 0);
      constexpr uint32_t idesc_pv = ptx::idesc_bf16(256, kDv, 1);
      const uint32_t elected = ptx::elect_one();
      uint32_t useq = 0;  // units with tiles so far
      Phases<C::kS> k_full, v_full, p_full;
      auto issue_qk = [&](uint32_t st) -> bool {
        if (!wt.all(bar(C::kKFull + st), k_full.take(st))) return false;
        ptx::tc_fence_after();
        const uint64_t qd = ptx::smem_desc(base, 16, 1024, 2);
        const uint64_t kd = ptx::smem_desc(base + C::kSmK + st * C::kKBytes, 16, 1024, 2);
        if constexpr (kDq == 192)
          ptx::mma_ss_pair_x12(elected, st * 128, qd, kd, idesc_qk, 0u);
        else
          ptx::mma_ss_pair_x16(elected, st * 128, qd, kd, idesc_qk, 0u);
        ptx::mma_commit_pair(bar(C::kSFull + st));
        ptx::mma_commit_pair(bar(C::kKEmpty + st));
        return true;
      };
      for (uint32_t n = 0;; ++n) {
        const int slot = int(n & 1u);
        if (!wt.all(bar(C::kInfoFull + slot), (n >> 1) & 1u)) break;
        const int tiles = __shfl_sync(
            0xFFFFFFFFu, (reinterpret_cast<const Info*>(sm + C::kSmInfo) + slot)->tiles, 0);
        if (lane == 0) ptx::mbar_arrive(bar(C::kInfoEmpty + slot));
        if (tiles < 0) break;
        if (!tiles) continue;
        if (!wt.all(bar(C::kQFull), useq & 1u)) break;
        // Tile j's PV and, in its place, tile j + kS's QK^T; the first kS tiles' QK^T lead.
        for (int j0 = -C::kS; j0 < tiles && !wt.failed; j0 += C::kS) {
#pragma unroll 1
          for (int st = 0; st < C::kS; ++st) {
            const int j = j0 + st;
            if (j >= tiles || wt.failed) break;
            if (j >= 0) {
              // The unit before must have read its output before this one's first PV replaces it.
              if (j == 0 && useq > 0 && !wt.all(bar(C::kOFree), (useq - 1) & 1u)) break;
              if (!wt.all(bar(C::kVFull + st), v_full.take(st))) break;
              // V as B, MN-major: 64 value columns are a chunk of [128 keys][128 B], 8-key groups
              // 1 KB apart; a step of 16 keys is 2 KB. The first 64 keys go ahead of the rest.
              const uint64_t vd =
                  ptx::smem_desc(base + C::kSmV + st * C::kVBytes, 16384, 1024, 2);
              const uint32_t phase = p_full.take(st);
              if (!wt.all(bar(C::kPFull + 2 * st), phase)) break;
              ptx::tc_fence_after();
              ptx::mma_ts_pair_x4(elected, C::kTmemO, st * 128, vd, idesc_pv, j > 0 ? 1u : 0u);
              if (!wt.all(bar(C::kPFull + 2 * st + 1), phase)) break;
              ptx::tc_fence_after();
              ptx::mma_ts_pair_x4(elected, C::kTmemO, st * 128 + 32, vd + 512, idesc_pv, 1u);
              ptx::mma_commit_pair(bar(C::kVEmpty + st));
              ptx::mma_commit_pair(bar(C::kPvDone + st));
            }
            if (j + C::kS < tiles) {
              if (!issue_qk(st)) break;
              if (j + C::kS + 1 == tiles) ptx::mma_commit_pair(bar(C::kQEmpty));
            }
          }
        }
      ++useq;
      }
      ptx::mma_commit_pair(bar(C::kDrain));
    }
    __syncwarp();
  } else if (warp == 2) {
    if (lane == 0) {
      Phases<C::kKv> free;
      for (uint32_t n = 0;; ++n) {
        const UnitRef x = next_unit(n);
        if (x.tiles < 0) break;
        for (int j = 0; j < x.tiles; ++j) {
          const uint32_t st = uint32_t(j % C::kKv), ph = free.take(st) ^ 1u;
          const int key = x.key0 + j * kRowTile;
          if (!wt.on(bar(C::kVEmpty + st), ph)) break;
          if (rank == 0) ptx::mbar_expect_tx(bar(C::kVFull + st), 2 * C::kVBytes);
          const uint32_t vd = base + C::kSmV + st * C::kVBytes;
#pragma unroll
          for (int c = 0; c < C::kVChunks; ++c)
            ptx::tma_load_3d_pair(vd + c * 16384, &tm_v, lead(C::kVFull + st),
                                  rank * (kDv / 2) + c * 64, key, x.head);
        }
      }
    }
    __syncwarp();
  } else if (warp == 3) {
    // The first unit is the pair's own; then, near the end of each, the leader takes the next one
    // from the pass's counter and tells the other CTA.
    const uint32_t mail = base + C::kSmExch + 3088;
    for (uint32_t n = 0;; ++n) {
      if (n == 1) ptx::grid_dependency_wait();
      int u = int(blockIdx.x) >> 1;
      if (n == 0) {
      } else if (rank == 0) {
        if (!wt.all(bar(C::kClaim), (n & 1u) ^ 1u)) break;
        if (!wt.all(bar(C::kMailEmpty), n & 1u)) break;
        if (lane == 0) {
          u = pairs + atomicAdd(a.w.header + kHdrNext + a.pass, 1);
          ptx::st_cluster_u32(ptx::map_peer(mail, 1), uint32_t(u));
          ptx::mbar_arrive_cluster(ptx::map_peer(bar(C::kMailFull), 1));
        }
        u = __shfl_sync(0xFFFFFFFFu, u, 0);
      } else {
        if (!wt.all(bar(C::kMailFull), (n & 1u) ^ 1u)) break;
        ptx::mbar_test_cluster(bar(C::kMailFull), (n & 1u) ^ 1u);  // acquires the leader's store
        u = __shfl_sync(0xFFFFFFFFu, int(ptx::ld_shared_u32(mail)), 0);
        if (lane == 0) ptx::mbar_arrive_cluster_relaxed(ptx::map_peer(bar(C::kMailEmpty), 0));
      }
      const bool end = u >= units;
      Unit x = {};
      int keys = 0, spoilt = INT_MAX;
      if (!end) {
        x = unit_at(a, u, pieces, pairs);
        keys = __ldcg(a.w.seq_keys + x.p.seq);
        spoilt = __ldcg(a.w.seq_spoilt + x.p.seq);
      }
      if (!wt.all(bar(C::kInfoEmpty + int(n & 1u)), ((n >> 1) & 1u) ^ 1u)) break;
      Info* info = reinterpret_cast<Info*>(sm + C::kSmInfo) + (n & 1u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 32 + lane, at = rank * 128 + r;
        int seen = 0;
        if (at < x.p.rows) {
          const int pos = __ldcg(a.q_pos + x.p.row0 + at);
          seen = pos >= keys ? keys : max(pos + 1, 0);
          if (seen > spoilt) seen |= kSpoilt;
        }
        info->seen[r] = seen;
      }
      if (lane == 0) {
        info->row0 = x.p.row0;
        info->rows = x.p.rows;
        info->key0 = x.p.key0 + x.p.tile0 * kRowTile;
        info->tile0 = x.p.tile0;
        info->tiles = end ? -1 : x.p.tiles;
        info->whole = x.p.whole;
        info->head = x.head;
        info->slot = x.head * pieces + x.p.index;
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(C::kInfoFull + int(n & 1u)));
      if (end) break;
    }
    __syncwarp();
  } else {
    const int group = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lanes = uint32_t(quad * 32) << 16;
    float* shared_m = reinterpret_cast<float*>(sm + C::kSmExch);  // [128], or [2][2][128] in halves
    float* shared_sum = shared_m + 512;                           // [2][128]
    volatile int* gone = reinterpret_cast<volatile int*>(shared_m + 768);  // [4]
    const float c = a.scale_log2, slack = kSlack / c;
    uint32_t it0 = 0;  // tiles of earlier units
    Phases<C::kS> s_full, pv_done;
    for (uint32_t nth = 0;; ++nth) {
      const Info* info = reinterpret_cast<const Info*>(sm + C::kSmInfo) + (nth & 1u);
      wt.all(bar(C::kInfoFull + int(nth & 1u)), (nth >> 1) & 1u);
      // A wait that ran out ends the loop here for both warps of a row, and only here: inside a
      // unit they go through the same barriers to its end, over whatever TMEM holds.
      if (wt.failed && lane == 0) gone[quad] = 1;
      ptx::named_barrier(9 + quad, 64);
      if (gone[quad]) break;
      const int n = info->seen[row] & (kSpoilt - 1);  // keys that this row sees
      const int tiles = info->tiles, tile0 = info->tile0;
      if (tiles < 0) break;
      float m = -INFINITY;   // what this thread's sum is taken against
      float sum[2][2] = {};  // partial sums over this thread's keys
      // Where a row's maximum grew by more than the slack: columns `first` on of its part of O are
      // rescaled, after the PV of the tile before tile j.
      auto rescale = [&](int j, float keep, int first, int columns) {
        const int b = j - 1;
        wt.all(bar(C::kPvDone + b % C::kS), pv_done.at(b % C::kS, b / C::kS));
        ptx::tc_fence_after();
        const uint32_t o = tmem + C::kTmemO + first + lanes;
#pragma unroll 1
        for (int i = 0; i < columns; i += 16) {
          uint32_t v[16];
          ptx::tmem_ld16(o + i, v);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * keep);
          ptx::tmem_st16(o + i, v);
        }
      };
      // Of 32 scores, those behind the first `see` become -inf.
      auto hide = [&](uint32_t (&r)[32], int see) {
        const uint32_t bits = see >= 32 ? 0xFFFFFFFFu : see <= 0 ? 0u : (1u << see) - 1u;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (!(bits & (1u << i))) r[i] = 0xFF800000u;
      };
      float top[4];
      auto raise = [&](const uint32_t (&r)[32]) {
#pragma unroll
        for (int i = 0; i < 32; i += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            top[k] = fmaxf(fmaxf(top[k], __uint_as_float(r[i + k])), __uint_as_float(r[i + 4 + k]));
      };
      // 32 softmax weights, against mc = -c * reference, to TMEM as 16 columns of bf16 pairs (PV's
      // operands have one type, V's); their sum takes them unrounded.
      auto weigh = [&](const uint32_t (&r)[32], float mc, uint32_t dst) {
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float p0 = ptx::ex2(fmaf(__uint_as_float(r[i]), c, mc));
          const float p1 = ptx::ex2(fmaf(__uint_as_float(r[i + 1]), c, mc));
          sum[(i >> 1) & 1][0] += p0;
          sum[(i >> 1) & 1][1] += p1;
          p[i / 2] = ptx::pack_bf16x2(p0, p1);
        }
        ptx::tmem_st16(dst, p);
      };
      auto weighed = [&](int half, uint32_t sb) {
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster_relaxed(lead(C::kPFull + 2 * int(sb) + half));
      };
      const int odd = C::kHalves ? 0 : int((it0 ^ uint32_t(group)) & 1u);
      for (int j = odd; j < tiles; j += C::kHalves ? 1 : 2) {
        const uint32_t it = it0 + uint32_t(j), sb = uint32_t(j % C::kS);
        wt.all(bar(C::kSFull + sb), s_full.at(sb, j / C::kS));
        ptx::tc_fence_after();
        const uint32_t src = tmem + sb * 128 + lanes;
        const int key = (tile0 + j) * kRowTile;
        top[0] = top[1] = top[2] = top[3] = -INFINITY;
        if constexpr (C::kHalves) {
          // This group's 64 keys of every tile.
          uint32_t r0[32], r1[32];
          ptx::tmem_ld32(src + group * 64, r0);
          ptx::tmem_ld32(src + group * 64 + 32, r1);
          ptx::tmem_wait_ld();
          const int see = n - key - group * 64;
          if (!__all_sync(0xFFFFFFFFu, see >= 64)) {
            hide(r0, see);
            hide(r1, see - 32);
          }
          raise(r0);
          raise(r1);
          float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
          // The two threads of a row exchange their maxima, and keep the same reference. Past the
          // barrier both have read their scores, which P may now replace.
          float* ex = shared_m + (it & 1u) * 256;
          ex[group * 128 + row] = high;
          ptx::named_barrier(1 + quad, 64);
          high = fmaxf(high, ex[(group ^ 1) * 128 + row]);
          if (j == 0) {
            m = high;
          } else {
            const bool grow = high > m + slack;
            if (__any_sync(0xFFFFFFFFu, grow)) {
              const float keep =
                  !grow ? 1.f : m == -INFINITY ? 0.f : ptx::ex2((m - high) * c);
              if (grow) m = high;
              rescale(j, keep, group * (kDv / 2), kDv / 2);
              // The first half of PV_j starts on group 0's weights alone and adds to all columns of
              // O, so group 1's are rescaled before group 0 goes on. Both warps of these rows are
              // here: their maxima and references are the same.
              ptx::tmem_wait_st();
              ptx::tc_fence_before();
              ptx::named_barrier(5 + quad, 64);
              ptx::tc_fence_after();
              sum[0][0] *= keep;
              sum[0][1] *= keep;
              sum[1][0] *= keep;
              sum[1][1] *= keep;
            }
          }
          const float mc = m == -INFINITY ? 0.f : -m * c;
          weigh(r0, mc, src + group * 32);
          weigh(r1, mc, src + group * 32 + 16);
          weighed(group, sb);
        } else {
          // Every other tile, all of its keys; its scores are read twice, a quarter at a time.
          // (Holding them from the maximum to the exponentials, or unrolling the quarters, makes
          // code that crowds the instruction caches which all roles share: 1690 to 1780 us of
          // attention for 2 x 2048 tokens of 128 heads instead of 1545.)
          const bool whole = __all_sync(0xFFFFFFFFu, n >= key + kRowTile);
#pragma unroll 1
          for (int g = 0; g < 4; ++g) {
            uint32_t r[32];
            ptx::tmem_ld32(src + 32 * g, r);
            ptx::tmem_wait_ld();
            if (!whole) hide(r, n - key - 32 * g);
            raise(r);
          }
          const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
          // The turn passes from tile to tile, and so from group to group, with the row's reference
          // maximum.
          if (it > 0) ptx::named_barrier(1 + quad + 4 * int(it & 1u), 64);
          float ref = j == 0 ? high : shared_m[row];
          if (j > 0) {
            const bool grow = high > ref + slack;
            if (__any_sync(0xFFFFFFFFu, grow)) {
              const float keep =
                  !grow ? 1.f : ref == -INFINITY ? 0.f : ptx::ex2((ref - high) * c);
              if (grow) ref = high;
              rescale(j, keep, 0, kDv);
            }
          }
          shared_m[row] = ref;
          if (__any_sync(0xFFFFFFFFu, ref != m)) {
            const float keep = m == ref ? 1.f : m == -INFINITY ? 0.f : ptx::ex2((m - ref) * c);
            sum[0][0] *= keep;
            sum[0][1] *= keep;
            sum[1][0] *= keep;
            sum[1][1] *= keep;
            m = ref;
          }
          const float mc = ref == -INFINITY ? 0.f : -ref * c;
#pragma unroll 1
          for (int g = 0; g < 4; ++g) {
            uint32_t r[32];
            ptx::tmem_ld32(src + 32 * g, r);
            ptx::tmem_wait_ld();
            if (!whole) hide(r, n - key - 32 * g);
            weigh(r, mc, src + 16 * g);  // over scores that are read
            if (g == C::kTurn)
              ptx::named_barrier_arrive(1 + quad + 4 * int((it + 1) & 1u), 64);
            if (g & 1) weighed(g >> 1, sb);
          }
        }
      }
      it0 += uint32_t(tiles);
      const int last = tiles - 1;
      const uint32_t last_phase = last >= 0 ? pv_done.at(last % C::kS, last / C::kS) : 0u;
      s_full.pass(tiles);
      pv_done.pass(tiles);
      // The row's last reference maximum and its whole sum, then O / sum to the output: this
      // thread's half of the columns.
      ptx::named_barrier(9 + quad, 64);
      const float ref = C::kHalves ? m : tiles ? shared_m[row] : -INFINITY;
      float total = (sum[0][0] + sum[0][1]) + (sum[1][0] + sum[1][1]);
      if (m != ref) total = m == -INFINITY ? 0.f : total * ptx::ex2((m - ref) * c);
      shared_sum[group * 128 + row] = total;
      ptx::named_barrier(9 + quad, 64);
      total = shared_sum[row] + shared_sum[128 + row];
      if (info->seen[row] & kSpoilt) total = NAN;
      const bool sees = n > tile0 * kRowTile;  // in this piece
      const float inv = sees ? 1.f / total : 0.f;
      if (tiles) {
        wt.all(bar(C::kPvDone + last % C::kS), last_phase);
        ptx::tc_fence_after();
      }
      // The rest of the unit's info, and the info buffer is free.
      const int head = a.head0 + info->head, rows = info->rows - rank * 128;
      const int t0 = info->row0 + rank * 128;
      const bool whole = info->whole != 0;
      const long long part = (long long)info->slot * kQueryTile + rank * 128;
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(C::kInfoEmpty + int(nth & 1u)));
      // Rows of this warp: through shared memory 64 bytes a row at a time, so that four lanes store
      // 64 consecutive bytes (a lane a row stored 16 bytes each to 32 lines at once: 7500 cycles a
      // unit at 256 columns).
      const bool f32 = a.out_f32 || !whole;
      uint8_t* out0 = whole ? a.out + (long long)t0 * a.out_st + (long long)head * a.out_sh
                            : reinterpret_cast<uint8_t*>(a.w.part_out + part * kDv);
      const long long out_row = whole ? a.out_st : (long long)kDv * 4;
      uint8_t* turn = sm + C::kSmTurn + (warp - 4) * kTurnBytes;
      auto emit = [&](const uint32_t (&v)[16], int byte) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<uint4*>(turn + lane * 80 + k * 16) =
              make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = k * 8 + (lane >> 2), at = quad * 32 + r;
          const uint4 w = *reinterpret_cast<const uint4*>(turn + r * 80 + (lane & 3) * 16);
          if (at < rows)
            *reinterpret_cast<uint4*>(out0 + at * out_row + byte + (lane & 3) * 16) = w;
        }
        __syncwarp();
      };
      const uint32_t o = tmem + C::kTmemO + group * (kDv / 2) + lanes;
#pragma unroll 1
      for (int i = 0; i < kDv / 2; i += 32) {
        const int col = group * (kDv / 2) + i;
        uint32_t v[32], y[16];
        if (tiles) {
          ptx::tmem_ld32(o + i, v);
          ptx::tmem_wait_ld();
        }
#pragma unroll
        for (int k = 0; k < 32; ++k)
          v[k] = sees ? __float_as_uint(__uint_as_float(v[k]) * inv) : 0u;
#pragma unroll 1
        for (int g = 0; g <= int(f32); ++g) {
#pragma unroll
          for (int k = 0; k < 16; ++k)
            y[k] = !f32 ? ptx::pack_bf16x2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1]))
                   : g  ? v[16 + k]
                        : v[k];
          emit(y, f32 ? 4 * col + 64 * g : 2 * col);
        }
      }
      if (tiles) {
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster_relaxed(lead(C::kOFree));
      }
      if (row < rows && group == 0) {
        const float l2 = sees ? ref * c + log2f(total) : -INFINITY;
        if (!whole)
          a.w.part_lse[part + row] = l2;
        else if (a.lse)
          a.lse[(long long)(t0 + row) * a.heads + head] = l2 * 0.69314718055994531f;
      }
    }
  }
  if (warp == 0) wt.on(bar(C::kDrain), 0);
  wt.settle(a.w.header);
  __syncwarp();
  ptx::tc_fence_before();
  ptx::cluster_sync();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem, 512);
    __syncwarp();
  }
  ptx::cluster_sync_relaxed();  // both CTAs run until both have given their columns back
}

}  // namespace attend

// ------------------------------------------------------------------------------ join
// Merges the pieces of split blocks: out = sum_i 2^(l_i - l) out_i, l = log2 sum_i 2^l_i, in piece
// order. One thread takes 8 columns of one row and head, all pieces' loads ahead of their use.
// Reads the partial outputs once from L2, where the attention left them.
__global__ void __launch_bounds__(256) join_kernel(const Args a) {
  ptx::grid_dependency_wait();
  const Work& w = a.w;
  if (!w.header[kHdrSplit]) return;
  const int pieces = w.header[kHdrPieces], groups = a.dv / 8;
  const long long all = (long long)w.header[kHdrBlocks] * a.pass_heads * kQueryTile * groups;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all;
       i += (long long)gridDim.x * 256) {
    const int g = int(i % groups);
    long long r = i / groups;
    const int row = int(r % kQueryTile);
    r /= kQueryTile;
    const int head = int(r % a.pass_heads);
    const Block blk = w.blocks[r / a.pass_heads];
    if (blk.pieces == 1 || row >= blk.rows) continue;
    const long long p0 = ((long long)head * pieces + blk.piece0) * kQueryTile + row;
    float top = -INFINITY;
    for (int k = 0; k < blk.pieces; ++k)
      top = fmaxf(top, w.part_lse[p0 + (long long)k * kQueryTile]);
    const float use = top == -INFINITY ? 0.f : top;
    float o[8] = {}, sum = 0.f;
#pragma unroll 4
    for (int k = 0; k < blk.pieces; ++k) {
      const long long p = p0 + (long long)k * kQueryTile;
      const float f = ptx::ex2(w.part_lse[p] - use);
      const float4* src = reinterpret_cast<const float4*>(w.part_out + p * a.dv + 8 * g);
      const float4 x = src[0], y = src[1];
      sum += f;
      o[0] = fmaf(f, x.x, o[0]); o[1] = fmaf(f, x.y, o[1]);
      o[2] = fmaf(f, x.z, o[2]); o[3] = fmaf(f, x.w, o[3]);
      o[4] = fmaf(f, y.x, o[4]); o[5] = fmaf(f, y.y, o[5]);
      o[6] = fmaf(f, y.z, o[6]); o[7] = fmaf(f, y.w, o[7]);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] *= inv;
    const long long t = blk.row0 + row;
    uint8_t* out = a.out + t * a.out_st + (long long)(a.head0 + head) * a.out_sh;
    if (a.out_f32) {
      reinterpret_cast<float4*>(out + 32 * g)[0] = make_float4(o[0], o[1], o[2], o[3]);
      reinterpret_cast<float4*>(out + 32 * g)[1] = make_float4(o[4], o[5], o[6], o[7]);
    } else {
      *reinterpret_cast<uint4*>(out + 16 * g) =
          make_uint4(ptx::pack_bf16x2(o[0], o[1]), ptx::pack_bf16x2(o[2], o[3]),
                     ptx::pack_bf16x2(o[4], o[5]), ptx::pack_bf16x2(o[6], o[7]));
    }
    if (a.lse && g == 0)
      a.lse[t * a.heads + a.head0 + head] =
          sum == 0.f ? -INFINITY : 0.69314718055994531f * (use + log2f(sum));
  }
}

// ------------------------------------------------------------------------------ host
struct Layout {
  uint64_t header, seq_key0, seq_keys, seq_block, seq_spoilt, blocks, pieces, order;
  uint64_t part_out, part_lse, rows, rope, k, v, total;
  uint64_t cap, max_blocks, pass_heads, split_units;
};

uint64_t round256(uint64_t v) { return (v + 255) & ~uint64_t(255); }

Layout layout_of(const TqMlaChunkSpec& s) {
  const uint64_t T = s.q.shape[0], H = s.q.shape[1], S = s.page_table.shape[0];
  const uint64_t dn = s.w_uk.shape[1], dv = s.w_uv.shape[1];
  const uint64_t busy = S < T ? S : T;  // sequences that can have tokens
  Layout l;
  // Every busy sequence may end inside a row tile; whole pairs of tiles for the expansion.
  l.cap = (s.max_keys + busy * (kRowTile - 1) + 255) / 256 * 256;
  if (l.cap == 0) l.cap = 256;
  l.max_blocks = T / kQueryTile + busy;
  const uint64_t per_head = l.cap * (dn + dv) * 2;
  l.pass_heads = kScratchBytes / per_head;
  if (l.pass_heads < 1) l.pass_heads = 1;
  if (l.pass_heads > H) l.pass_heads = H;
  // Blocks are split only where even full query blocks would be fewer than the units allowed.
  const uint64_t full = (T + kQueryTile - 1) / kQueryTile * l.pass_heads;
  l.split_units = full <= kSplitUnits ? kSplitUnits : 0;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += round256(bytes);
    return here;
  };
  l.header = take(kHdrWords * 4);
  l.seq_key0 = take((S + 1) * 4);
  l.seq_keys = take((S + 1) * 4);
  l.seq_block = take((S + 1) * 4);
  l.seq_spoilt = take((S + 1) * 4);
  l.blocks = take(l.max_blocks * sizeof(Block));
  l.pieces = take((l.max_blocks + l.split_units) * sizeof(Piece));
  l.order = take((l.max_blocks + l.split_units) * sizeof(Piece));
  l.part_out = take(l.split_units * kQueryTile * dv * 4);
  l.part_lse = take(l.split_units * kQueryTile * 4);
  l.rows = take(l.cap * kLatent * 2);
  l.rope = take(l.cap * kRopeDim * 2);
  l.k = take(l.pass_heads * l.cap * dn * 2);
  l.v = take(l.pass_heads * l.cap * dv * 2);
  l.total = at;
  return l;
}

// bf16 boxes of 64 values by `box` rows (and one of the third axis) with 128-byte swizzle.
bool encode(CUtensorMap* map, const void* addr, uint64_t width, uint64_t rows, uint64_t planes,
            uint64_t row_bytes, uint64_t plane_bytes, uint32_t box, uint32_t box_planes = 1) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {width, rows, planes};
  const cuuint64_t strides[2] = {row_bytes, plane_bytes};
  const cuuint32_t boxes[3] = {64, box, box_planes};
  const cuuint32_t elem[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, planes ? 3 : 2, const_cast<void*>(addr), dims,
            strides, boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// CTA pairs (two SMs each) of the current device, once the kernels have their shared memory granted
// on it; 0 on failure.
int pairs_on(int device) {
  static std::mutex mu;
  static int cached[128] = {0};
  if (device < 0 || device >= 128) return 0;
  std::lock_guard<std::mutex> lock(mu);
  if (cached[device]) return cached[device];
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
      cudaFuncSetAttribute(expand::expand_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           int(expand::kSmBytes)) != cudaSuccess ||
      cudaFuncSetAttribute(attend::attend_kernel<192, 128>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                           int(attend::Shape<192, 128>::kSmBytes)) != cudaSuccess ||
      cudaFuncSetAttribute(attend::attend_kernel<256, 256>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                           int(attend::Shape<256, 256>::kSmBytes)) != cudaSuccess)
    return 0;
  cached[device] = sms / 2;
  return cached[device];
}

}  // namespace chunk
}  // namespace tq

extern "C" int32_t tq_mla_chunk_workspace_bytes(const TqMlaChunkSpec* spec, int32_t device,
                                                uint64_t* bytes) {
  TqContractError e{nullptr, TQ_OK};
  const int32_t st = tq::chunk_validate(spec, &e);
  if (st != TQ_OK) return st;
  if (!bytes || device < 0) return TQ_ERR_INVALID_ARGUMENT;
  *bytes = tq::chunk::layout_of(*spec).total;
  return TQ_OK;
}

extern "C" int32_t tq_mla_chunk(const TqMlaChunkSpec* spec, void* workspace,
                                uint64_t workspace_bytes, void* stream, TqContractError* err) {
  using namespace tq::chunk;
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  const int32_t st = tq::chunk_validate(spec, err);
  if (st != TQ_OK) return st;
  const TqMlaChunkSpec& s = *spec;
  const uint64_t T = s.q.shape[0], S = s.page_table.shape[0];
  if (T == 0 || S == 0) {
    // Nothing to launch; what the workspace holds is not this call's error word.
    if (workspace && workspace_bytes >= sizeof(int) &&
        cudaMemsetAsync(workspace, 0, sizeof(int), static_cast<cudaStream_t>(stream)) !=
            cudaSuccess)
      return fail("workspace", TQ_ERR_CUDA);
    return fail(nullptr, TQ_OK);
  }
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return fail("device", TQ_ERR_CUDA);
  const int pairs = pairs_on(device);
  if (pairs <= 0) return fail("device", TQ_ERR_CUDA);
  const Layout l = layout_of(s);
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 || workspace_bytes < l.total)
    return fail("workspace", TQ_ERR_WORKSPACE);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Args a = {};
  a.w.header = reinterpret_cast<int*>(ws + l.header);
  a.w.seq_key0 = reinterpret_cast<int*>(ws + l.seq_key0);
  a.w.seq_keys = reinterpret_cast<int*>(ws + l.seq_keys);
  a.w.seq_block = reinterpret_cast<int*>(ws + l.seq_block);
  a.w.seq_spoilt = reinterpret_cast<int*>(ws + l.seq_spoilt);
  a.w.blocks = reinterpret_cast<Block*>(ws + l.blocks);
  a.w.pieces = reinterpret_cast<Piece*>(ws + l.pieces);
  a.w.order = reinterpret_cast<Piece*>(ws + l.order);
  a.w.part_out = reinterpret_cast<float*>(ws + l.part_out);
  a.w.part_lse = reinterpret_cast<float*>(ws + l.part_lse);
  a.w.rows = reinterpret_cast<uint16_t*>(ws + l.rows);
  a.w.rope = reinterpret_cast<uint16_t*>(ws + l.rope);
  a.w.k = reinterpret_cast<uint16_t*>(ws + l.k);
  a.w.v = reinterpret_cast<uint16_t*>(ws + l.v);
  auto ints = [](const TqTensorSpec& t) { return reinterpret_cast<const int*>(t.device_address); };
  a.q = reinterpret_cast<const uint8_t*>(s.q.device_address);
  a.kv = reinterpret_cast<const uint8_t*>(s.kv.device_address);
  a.w_uk = reinterpret_cast<const uint16_t*>(s.w_uk.device_address);
  a.w_uv = reinterpret_cast<const uint16_t*>(s.w_uv.device_address);
  a.page_table = ints(s.page_table);
  a.q_start = ints(s.q_start);
  a.q_pos = ints(s.q_pos);
  a.kv_len = ints(s.kv_len);
  a.out = reinterpret_cast<uint8_t*>(s.out.device_address);
  a.lse = s.lse.rank ? reinterpret_cast<float*>(s.lse.device_address) : nullptr;
  a.out_st = (long long)s.out.strides_bytes[0];
  a.out_sh = (long long)s.out.strides_bytes[1];
  a.row_stride = (long long)s.kv.strides_bytes[1];
  a.tokens = int(T);
  a.heads = int(s.q.shape[1]);
  a.seqs = int(S);
  a.slots = int(s.page_table.shape[1]);
  a.pages = int(s.kv.shape[0]);
  a.cap = int(l.cap);
  a.max_blocks = int(l.max_blocks);
  a.split_units = int(l.split_units);
  a.pairs = pairs;
  a.pass_heads = int(l.pass_heads);
  a.dn = int(s.w_uk.shape[1]);
  a.dv = int(s.w_uv.shape[1]);
  a.dr = int(s.q.shape[2]) - a.dn;
  a.fp8 = s.kv_format == TQ_KV_FP8_E4M3;
  a.out_f32 = s.out.dtype == TQ_DTYPE_F32;
  a.scale_log2 = s.softmax_scale * 1.4426950408889634f;
  CUtensorMap tm_rows, tm_uk, tm_uv, tm_q, tm_k, tm_rope, tm_v;
  // q: 64 values by one head by 128 tokens, tokens past T as zeros.
  if (!encode(&tm_q, a.q, uint64_t(a.dn + a.dr), s.q.shape[1], T, s.q.strides_bytes[1],
              s.q.strides_bytes[0], 1, 128) ||
      !encode(&tm_k, a.w.k, uint64_t(a.dn), l.cap, l.pass_heads, uint64_t(a.dn) * 2,
              l.cap * uint64_t(a.dn) * 2, 64) ||
      !encode(&tm_v, a.w.v, uint64_t(a.dv), l.cap, l.pass_heads, uint64_t(a.dv) * 2,
              l.cap * uint64_t(a.dv) * 2, 128) ||
      !encode(&tm_rope, a.w.rope, kRopeDim, l.cap, 0, kRopeDim * 2, 0, 64) ||
      !encode(&tm_rows, a.w.rows, kLatent, l.cap, 0, kLatent * 2, 0, 128) ||
      !encode(&tm_uk, a.w_uk, kLatent, uint64_t(a.dn), s.w_uk.shape[0], s.w_uk.strides_bytes[1],
              s.w_uk.strides_bytes[0], 128) ||
      !encode(&tm_uv, a.w_uv, kLatent, uint64_t(a.dv), s.w_uv.shape[0], s.w_uv.strides_bytes[1],
              s.w_uv.strides_bytes[0], 128))
    return fail("tensor_map", TQ_ERR_CUDA);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  // Each kernel starts while the one before it ends, and waits inside for its results
  // (griddepcontrol.wait): the setup and the loads that need none run meanwhile.
  auto launch = [&](auto kernel, int grid, int threads, uint32_t smem, auto... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(grid), 1, 1);
    cfg.blockDim = dim3(unsigned(threads), 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = cs;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess;
  };
  if (!launch(plan_kernel, 1, 1024, 0, a) ||
      !launch(gather_kernel, 1 + a.cap / kGatherRows, kGatherThreads, 0, a))
    return fail("launch", TQ_ERR_CUDA);
  for (a.head0 = 0; a.head0 < a.heads; a.head0 += int(l.pass_heads), ++a.pass) {
    a.pass_heads = a.heads - a.head0 < int(l.pass_heads) ? a.heads - a.head0 : int(l.pass_heads);
    using Rope = attend::Shape<192, 128>;
    using Wide = attend::Shape<256, 256>;
    if (!launch(expand::expand_kernel, 2 * pairs, expand::kThreads, expand::kSmBytes, tm_rows,
                tm_uk, tm_uv, a) ||
        !(a.dr ? launch(attend::attend_kernel<192, 128>, 2 * pairs, attend::kThreads,
                        Rope::kSmBytes, tm_q, tm_k, tm_rope, tm_v, a)
               : launch(attend::attend_kernel<256, 256>, 2 * pairs, attend::kThreads,
                        Wide::kSmBytes, tm_q, tm_k, tm_rope, tm_v, a)) ||
        (a.split_units && !launch(join_kernel, 4 * pairs, 256, 0, a)))
      return fail("launch", TQ_ERR_CUDA);
  }
  return fail(nullptr, TQ_OK);
}
