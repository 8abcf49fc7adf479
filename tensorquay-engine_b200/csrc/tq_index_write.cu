// Index write (tq_index_write): index queries and keys of a step, rotated, quantized to E4M3, the
// keys written to their paged cache. A row of 128 values (one head of a query, or a key):
//   k only: k / sqrt(mean(k^2) + eps) * w, or (k - mean(k)) / sqrt(var(k) + eps) * w + b
//   pair (a, b) of the rotary part -> (a c - b s, a s + b c), c and s the cosine and sine of
//   pos * freq[i], times rope_mscale
//   scale = amax / 448, code = E4M3(x * (448 / amax)); w_out = w * scale_c * scale
// All f32 from the read to the code. The angle is a product of f64 and loses its whole turns before
// it is rounded to f32: at position 2^20 an f32 angle would be off by 2^-5, this one is by 2^-26 of a turn
// at most, which moves a value by 1.6 * 2^-24 of its pair's length: as much as a rounding of the cosine.
//
// What bounds it: HBM and instructions for many tokens (256 bytes read and 128 written a head), one launch's
// chain of loads (position, angles, row) for few. Half a warp holds a row, 8 values a lane, loaded while
// the rows before are worked on. A lane's values are four whole pairs, whichever way they are paired, so
// that a turn takes packed arithmetic and no exchange; two rows a half warp share the exchanges of their
// largest values and the divisions. A warp has one token's heads: its lanes make the angles once, and no
// warp waits for another. Keys, one a token, have blocks of eight tokens of their own.
// 8192 tokens of 64 heads take 43 us, 73% of the copy bandwidth (58 with a block a token, pairs
// exchanged between lanes and addresses made anew for every row: half as many instructions again). In a
// captured run of calls they take 41.4 us, one token of 64 heads 2.4, 64 tokens of 32 heads 1.9, 1021
// tokens of 48 heads with a rotary part 6.9 (3 us of traffic).

#include <cuda_runtime.h>

#include <cstdint>

#include "tq_contracts.h"
#include "tq_ptx.cuh"

namespace tq {
namespace index_write {

constexpr int kThreads = 128;
constexpr int kHalves = kThreads / 16;  // rows of a block at a time
constexpr int kMostHeads = 32;  // of a warp
constexpr int kPageRows = 64;
enum Form { kNone, kNeighbours, kHalf };  // of the rotary part

struct Args {
  const uint8_t* q;
  const uint8_t* k;
  const uint8_t* w;
  const uint8_t* norm_weight;  // null: k as it is
  const uint8_t* norm_bias;    // null: RMS
  const float* freq;
  uint8_t* kv;
  uint8_t* q_out;
  float* w_out;
  const int* page_table;
  const int* seq_id;
  const int* pos;
  int* flags;
  long long q_token, k_token, row_stride;  // bytes
  uint32_t q_head;                         // 16 bytes
  int tokens, heads, sequences, slots, pages, w_f32;
  int key_blocks;     // the first blocks; then `parts` warps for each token
  int parts, each;    // warps of a token's heads, and the heads of one
  int start, pairs;   // rotary part: first value, angles
  float mscale, eps, scale;
};

// A lane's eight values, four pairs (f, g): of the rotary part its four turns.
struct Row {
  float2 f[2], g[2];
};

// Which values of a head a lane has: those at [first, first + 4) and [second, second + 4). The eight that
// stand together, but in a rotary part of halves four of each half, so that no pair lies in two lanes.
template <Form F>
struct Place {
  int first, second;
  int turn;     // of the first of four pairs
  bool inside;  // the rotary part
  __device__ __forceinline__ Place(const Args& a, int lane) {
    const int at = 8 * lane - a.start;
    inside = F != kNone && at >= 0 && at < 2 * a.pairs;
    turn = at / 2;
    first = F == kHalf && inside ? a.start + turn : 8 * lane;
    second = F == kHalf && inside ? first + a.pairs : first + 4;
  }
  // From the lane's first value; `apart` is second - first.
  __device__ __forceinline__ uint4 load(const uint8_t* at, int apart) const {
    if (F != kHalf) return *reinterpret_cast<const uint4*>(at);
    const uint2 u = *reinterpret_cast<const uint2*>(at);
    const uint2 v = *reinterpret_cast<const uint2*>(at + 2 * apart);
    return make_uint4(u.x, u.y, v.x, v.y);
  }
  __device__ __forceinline__ uint4 load(const uint8_t* row) const { return load(row + 2 * first, second - first); }
  __device__ __forceinline__ void store(uint8_t* at, int apart, uint2 codes) const {
    if (F != kHalf) {
      *reinterpret_cast<uint2*>(at) = codes;
    } else {
      *reinterpret_cast<uint32_t*>(at) = codes.x;
      *reinterpret_cast<uint32_t*>(at + apart) = codes.y;
    }
  }
};

template <Form F>
__device__ __forceinline__ Row unpack(const uint4& u) {
  using ptx::bf16_hi;
  using ptx::bf16_lo;
  Row r;
  if (F == kHalf) {
    r.f[0] = make_float2(bf16_lo(u.x), bf16_hi(u.x));
    r.f[1] = make_float2(bf16_lo(u.y), bf16_hi(u.y));
    r.g[0] = make_float2(bf16_lo(u.z), bf16_hi(u.z));
    r.g[1] = make_float2(bf16_lo(u.w), bf16_hi(u.w));
  } else {
    r.f[0] = make_float2(bf16_lo(u.x), bf16_lo(u.y));
    r.f[1] = make_float2(bf16_lo(u.z), bf16_lo(u.w));
    r.g[0] = make_float2(bf16_hi(u.x), bf16_hi(u.y));
    r.g[1] = make_float2(bf16_hi(u.z), bf16_hi(u.w));
  }
  return r;
}

__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
template <typename Fn>
__device__ __forceinline__ void each(Row& r, const Row& w, Fn fn) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    r.f[i] = make_float2(fn(r.f[i].x, w.f[i].x), fn(r.f[i].y, w.f[i].y));
    r.g[i] = make_float2(fn(r.g[i].x, w.g[i].x), fn(r.g[i].y, w.g[i].y));
  }
}

// The key's norm.
template <Form F>
__device__ __forceinline__ void normalise(const Args& a, const Place<F>& place, Row& x) {
  const Row w = unpack<F>(place.load(a.norm_weight));
  float s = 0.f;
  if (a.norm_bias) {
    each(x, x, [&](float v, float) { s += v; return v; });
    const float mean = sum16(s) * (1.f / TQ_INDEX_DIM);
    each(x, x, [&](float v, float) { return v - mean; });
  }
  s = 0.f;
  each(x, x, [&](float v, float) { s = fmaf(v, v, s); return v; });
  const float r = 1.f / sqrtf(sum16(s) * (1.f / TQ_INDEX_DIM) + a.eps);
  // (In this order: r times a large weight may overflow where the value times r is small or 0.)
  each(x, w, [&](float v, float by) { return v * r * by; });
  if (a.norm_bias) each(x, unpack<F>(place.load(a.norm_bias)), [](float v, float b) { return v + b; });
}

// Cosine and sine of angle i at position p, times mscale.
__device__ __forceinline__ float2 angle(const Args& a, int p, int i) {
  double turns = double(p) * double(a.freq[i]) * 0.15915494309189533577;
  turns -= rint(turns);
  float s, c;
  sincospif(2.f * float(turns), &s, &c);
  return make_float2(c * a.mscale, s * a.mscale);
}

// What a lane's pairs are turned by: f c - g s and f s + g c.
template <Form F>
struct Turn {
  bool inside;
  float2 c[2], s[2], minus[2];

  __device__ __forceinline__ Turn(const Place<F>& place, const float2* angles) : inside(place.inside) {
    if (!inside) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 t = angles[place.turn + 2 * i], u = angles[place.turn + 2 * i + 1];
      c[i] = make_float2(t.x, u.x);
      s[i] = make_float2(t.y, u.y);
      minus[i] = make_float2(-t.y, -u.y);
    }
  }
  __device__ __forceinline__ void apply(Row& x) const {
    if (!inside) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = x.f[i], g = x.g[i];
      x.f[i] = __ffma2_rn(g, minus[i], __fmul2_rn(f, c[i]));
      x.g[i] = __ffma2_rn(f, s[i], __fmul2_rn(g, c[i]));
    }
  }
};

// The largest magnitude, as the bits of its value; NaN is above all.
__device__ __forceinline__ float largest3(float a, float b, float c) {
  float m;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
__device__ __forceinline__ uint32_t largest(const Row& x) {  // the lane's
  float m = largest3(x.f[0].x, x.f[0].y, x.f[1].x);
  m = largest3(m, x.f[1].y, x.g[0].x);
  m = largest3(m, x.g[0].y, x.g[1].x);
  m = largest3(m, x.g[1].y, x.g[1].y);
  return __float_as_uint(m) & 0x7FFFFFFFu;
}
// The half warp's, of two rows: lanes below 8 get a's, the others b's.
__device__ __forceinline__ uint32_t largest_of_two(uint32_t a, uint32_t b, int lane) {
  const uint32_t give = lane & 8 ? a : b;
  uint32_t m = max(lane & 8 ? b : a, __shfl_xor_sync(0xFFFFFFFFu, give, 8));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  return m;
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Codes of a lane's eight values. `mine` is, in the half warp's lane `at`, the scale amax / 448 and in the
// next 448 / amax, which is multiplied with. (A NaN makes it and all codes NaN, an infinity makes it 0.)
template <Form F>
__device__ __forceinline__ uint2 codes_of(Row x, float mine, int at) {
  float inv = __shfl_sync(0xFFFFFFFFu, mine, at + 1, 16);
  if (inv == __uint_as_float(0x7F800000u)) {
    // It overflows (amax below about 1.3e-36), or is 448 / 0. The scale has few bits then, so it is
    // what the values are divided by, both times 2^64 (which is exact).
    const float scale = __shfl_sync(0xFFFFu << (threadIdx.x & 16), mine, at, 16);
    if (scale == 0.f) return make_uint2(0u, 0u);
    inv = __fdiv_rn(1.f, scale * 0x1p64f);
    each(x, x, [&](float v, float) { return v * 0x1p64f; });
  }
  each(x, x, [&](float v, float) { return __fmul_rn(v, inv); });
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (F == kHalf) {
      c[i] = e4m3x2(x.f[i].x, x.f[i].y);
      c[2 + i] = e4m3x2(x.g[i].x, x.g[i].y);
    } else {
      c[2 * i] = e4m3x2(x.f[i].x, x.g[i].x);
      c[2 * i + 1] = e4m3x2(x.f[i].y, x.g[i].y);
    }
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

// Where token t's key goes, or null with the flag that says why not.
__device__ __forceinline__ uint8_t* slot_of(const Args& a, int s, int p, int* bad) {
  if (s < 0 || s >= a.sequences) { *bad = TQ_DEV_SEQ_RANGE; return nullptr; }
  if (p < 0 || p / kPageRows >= a.slots) { *bad = TQ_DEV_TABLE_SHORT; return nullptr; }
  const int page = a.page_table[(long long)s * a.slots + p / kPageRows];
  if (page < 0 || page >= a.pages) { *bad = TQ_DEV_PAGE_RANGE; return nullptr; }
  return a.kv + ((long long)page * kPageRows + p % kPageRows) * a.row_stride;
}

// Keys of kHalves tokens, a half warp each.
template <Form F>
__device__ __forceinline__ void write_keys(const Args& a, int t0) {
  __shared__ float2 angles[kHalves][TQ_INDEX_DIM / 2];
  const int lane = threadIdx.x & 15, half = threadIdx.x >> 4;
  const int t = min(t0 + half, a.tokens - 1);  // (half warps without a token go along)
  const Place<F> place(a, lane);
  const uint4 row = place.load(a.k + t * a.k_token);
  const int p = a.pos[t], s = a.seq_id[t];
  if constexpr (F != kNone) {
    for (int i = lane; i < a.pairs; i += 16) angles[half][i] = angle(a, p, i);
    __syncwarp();
  }
  Row x = unpack<F>(row);
  if (a.norm_weight) normalise(a, place, x);
  Turn<F>(place, angles[half]).apply(x);
  const uint32_t all = largest(x);
  const float amax = __uint_as_float(largest_of_two(all, all, lane));
  const float mine = __fdiv_rn(lane & 1 ? 448.f : amax, lane & 1 ? amax : 448.f);
  const uint2 codes = codes_of<F>(x, mine, 0);
  if (t0 + half >= a.tokens) return;
  int bad = 0;
  uint8_t* dst = slot_of(a, s, p, &bad);
  if (dst) {
    place.store(dst + place.first, place.second - place.first, codes);
    if (lane == 0) *reinterpret_cast<float*>(dst + TQ_INDEX_DIM) = mine;
  } else if (lane == 0 && a.flags) {
    atomicOr(a.flags, bad);
  }
}

// Heads [h0, h1) of token t by one warp, four at a time.
template <Form F>
__device__ __forceinline__ void write_queries(const Args& a, int t, int h0, int h1) {
  __shared__ __align__(16) float2 angles[kThreads / 32][TQ_INDEX_DIM / 2];
  __shared__ float scales[kThreads / 32][kMostHeads];
  const int lane = threadIdx.x & 15, half = threadIdx.x >> 4 & 1, warp = threadIdx.x >> 5;
  const int in_warp = threadIdx.x & 31;
  const Place<F> place(a, lane);
  const uint8_t* q = a.q + t * a.q_token + 2 * place.first;
  uint8_t* out = a.q_out + (long long)t * a.heads * TQ_INDEX_DIM + place.first;
  const int apart = place.second - place.first;
  // Heads h and h + 2, or the last one again: then two half warps write the same.
  auto head = [&](int h, int i) { return uint32_t(min(h + 2 * i, h1 - 1)); };
  auto load = [&](uint32_t h) { return place.load(q + uint64_t(h * 16u) * a.q_head, apart); };
  uint4 row[2] = {load(head(h0 + half, 0)), load(head(h0 + half, 1))};
  if constexpr (F != kNone) {
    const int p = a.pos[t];
    for (int i = in_warp; i < a.pairs; i += 32) angles[warp][i] = angle(a, p, i);
    __syncwarp();
  }
  const Turn<F> turn(place, angles[warp]);
#pragma unroll 1
  for (int h = h0 + half; h - half < h1; h += 4) {
    Row x[2] = {unpack<F>(row[0]), unpack<F>(row[1])};
    row[0] = load(head(h + 4, 0));
    row[1] = load(head(h + 4, 1));
    turn.apply(x[0]);
    turn.apply(x[1]);
    // Half of the lanes go on with one row's largest, half with the other's; of those one half has the
    // scale, one its inverse.
    const uint32_t m = largest_of_two(largest(x[0]), largest(x[1]), lane);
    const float amax = __uint_as_float(m);
    const float mine = __fdiv_rn(lane & 1 ? 448.f : amax, lane & 1 ? amax : 448.f);
    const uint2 c0 = codes_of<F>(x[0], mine, 0);
    const uint2 c1 = codes_of<F>(x[1], mine, 8);
    place.store(out + head(h, 0) * TQ_INDEX_DIM, apart, c0);
    place.store(out + head(h, 1) * TQ_INDEX_DIM, apart, c1);
    if ((lane & 7) == 0) scales[warp][h - h0 + lane / 4] = mine;  // (at most kMostHeads)
  }
  __syncwarp();
  const int h = h0 + in_warp;
  if (h < h1) {
    const long long at = (long long)t * a.heads + h;
    const float w = a.w_f32 ? reinterpret_cast<const float*>(a.w)[at]
                            : __uint_as_float(uint32_t(reinterpret_cast<const uint16_t*>(a.w)[at]) << 16);
    a.w_out[at] = w * a.scale * scales[warp][h - h0];
  }
}

template <Form F>
__global__ void __launch_bounds__(kThreads, 8) index_write_kernel(const Args a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int block = int(blockIdx.x) - a.key_blocks;
  if (block < 0) {
    write_keys<F>(a, int(blockIdx.x) * kHalves);
  } else {
    const int item = block * (kThreads / 32) + int(threadIdx.x >> 5), t = item / a.parts;
    const int h0 = item % a.parts * a.each;
    if (t < a.tokens) write_queries<F>(a, t, h0, min(a.heads, h0 + a.each));
  }
}

}  // namespace index_write
}  // namespace tq

extern "C" int32_t tq_index_write(const TqIndexWriteSpec* spec, int32_t* device_flags, void* stream,
                                  TqContractError* err) {
  using namespace tq::index_write;
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  const int32_t st = tq::index_write_validate(spec, err);
  if (st != TQ_OK) return st;
  const TqIndexWriteSpec& s = *spec;
  const uint64_t tokens = s.k.shape[0];
  if (tokens == 0) return fail(nullptr, TQ_OK);
  auto at = [](const TqTensorSpec& t) {
    return t.rank ? reinterpret_cast<uint8_t*>(t.device_address) : nullptr;
  };
  Args a = {};
  a.q = at(s.q);
  a.k = at(s.k);
  a.w = at(s.w);
  a.norm_weight = at(s.norm_weight);
  a.norm_bias = at(s.norm_bias);
  a.freq = reinterpret_cast<const float*>(at(s.freq));
  a.kv = at(s.kv);
  a.q_out = at(s.q_out);
  a.w_out = reinterpret_cast<float*>(at(s.w_out));
  a.page_table = reinterpret_cast<const int*>(at(s.page_table));
  a.seq_id = reinterpret_cast<const int*>(at(s.seq_id));
  a.pos = reinterpret_cast<const int*>(at(s.pos));
  a.flags = device_flags;
  if (s.q.rank) {
    a.q_token = (long long)s.q.strides_bytes[0];
    a.q_head = uint32_t(s.q.strides_bytes[1] / 16);
    a.heads = int(s.q.shape[1]);
    a.w_f32 = s.w.dtype == TQ_DTYPE_F32;
  }
  a.k_token = (long long)s.k.strides_bytes[0];
  a.row_stride = (long long)s.kv.strides_bytes[1];
  a.sequences = int(s.page_table.shape[0]);
  a.slots = int(s.page_table.shape[1]);
  a.pages = int(s.kv.shape[0]);
  a.pairs = s.freq.rank ? int(s.freq.shape[0]) : 0;
  a.start = s.rope_start;
  a.mscale = s.rope_mscale;
  a.eps = s.norm_eps;
  a.scale = s.scale;
  a.tokens = int(tokens);
  a.key_blocks = (a.tokens + kHalves - 1) / kHalves;
  // Few tokens: a warp for every four heads, so that they are read at once. More heads of a token share
  // their angles where that leaves enough warps (8192 tokens of 64 heads, captured: 32 a warp 41.4 us, 16
  // 43.5).
  a.each = 4;
  while (a.each < kMostHeads && (long long)a.tokens * a.heads >= 16384ll * a.each) a.each *= 2;
  a.parts = (a.heads + a.each - 1) / a.each;
  const auto kernel = a.pairs == 0 ? index_write_kernel<kNone>
                      : s.rope_half ? index_write_kernel<kHalf>
                                    : index_write_kernel<kNeighbours>;
  cudaLaunchConfig_t cfg = {};
  constexpr int kWarps = kThreads / 32;
  cfg.gridDim = dim3(unsigned(a.key_blocks + ((long long)a.tokens * a.parts + kWarps - 1) / kWarps), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess)
    return fail("launch", TQ_ERR_CUDA);
  return fail(nullptr, TQ_OK);
}
