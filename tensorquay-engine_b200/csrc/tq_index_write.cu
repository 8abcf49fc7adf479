// Index write (tq_index_write): index queries and keys of a step, rotated, quantized to E4M3, the
// keys written to their paged cache. A row of 128 values (one head of a query, or a key):
//   k only: k / sqrt(mean(k^2) + eps) * w, or (k - mean(k)) / sqrt(var(k) + eps) * w + b
//   pair (a, b) of the rotary part -> (a c - b s, a s + b c), c and s the cosine and sine of
//   pos * freq[i], times rope_mscale
//   scale = amax / 448, code = E4M3(x * (448 / amax)); w_out = w * scale_c * scale
// All f32 from the read to the code. The angle is a product of f64 and loses its whole turns before
// it is rounded to f32: at position 2^20 an f32 angle would be off by 2^-5.
//
// What bounds it: instructions and HBM alike for many tokens (256 bytes read and 128 written a head), one
// launch's chain of loads (position, angles, row) for few. Half a warp holds a row, 8 values a lane: one
// 16-byte load, the other value of a pair in the lane or one shuffle away, the row's largest by one
// reduction. A block has one token's heads, 16 at a time, two of them a half warp: a lane's cosines
// and sines stay in registers for all heads, and four lanes share the divisions of two. Keys, one a
// token, have blocks of eight tokens of their own. Blocks are small so that many are at work on an SM:
// their first steps are a chain of loads and the angles. 8192 tokens of 64 heads take 58 us, 55% of
// the copy bandwidth (99 with one block a token's 64 heads and the angles in shared memory); 64 tokens 8 us with
// the launch.

#include <cuda_runtime.h>

#include <cstdint>

#include "tq_contracts.h"
#include "tq_ptx.cuh"

namespace tq {
namespace index_write {

constexpr int kThreads = 128;
constexpr int kHalves = kThreads / 16;  // rows of a block at a time
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
  long long q_token, q_head, k_token, row_stride;  // bytes
  int tokens, heads, sequences, slots, pages, w_f32;
  int key_blocks;     // the first blocks; then `parts` for each token
  int parts, each;    // blocks of a token's heads, and the heads of one
  int start, pairs;   // rotary part: first value, angles
  float mscale, eps, scale;
};

__device__ __forceinline__ void unpack(const uint4& p, float (&v)[8]) {
  const uint32_t u[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = ptx::bf16_lo(u[i]);
    v[2 * i + 1] = ptx::bf16_hi(u[i]);
  }
}

__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// The key's norm.
__device__ __forceinline__ void normalise(const Args& a, float (&x)[8], int lane) {
  float w[8];
  unpack(reinterpret_cast<const uint4*>(a.norm_weight)[lane], w);
  float s = 0.f;
  if (a.norm_bias) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[i];
    const float mean = sum16(s) * (1.f / TQ_INDEX_DIM);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] -= mean;
  }
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(x[i], x[i], s);
  const float r = 1.f / sqrtf(sum16(s) * (1.f / TQ_INDEX_DIM) + a.eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= r * w[i];
  if (a.norm_bias) {
    unpack(reinterpret_cast<const uint4*>(a.norm_bias)[lane], w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] += w[i];
  }
}

// Cosine and sine of angle i at position p, times mscale.
__device__ __forceinline__ float2 angle(const Args& a, int p, int i) {
  double turns = double(p) * double(a.freq[i]) * 0.15915494309189533577;
  turns -= rint(turns);
  float s, c;
  sincospif(2.f * float(turns), &s, &c);
  return make_float2(c * a.mscale, s * a.mscale);
}

// What a lane's eight values are turned by: x -> x c + y s, y the other value of the pair. The sine has
// the sign of the value's place in its pair.
template <Form F>
struct Turn {
  bool inside;  // the lane's values are in the rotary part
  int other;    // the lane of the other values (kHalf)
  float c[8], s[8];

  __device__ __forceinline__ Turn(const Args& a, int lane, const float2* angles) {
    if constexpr (F != kNone) {
      const int at = 8 * lane - a.start;
      inside = at >= 0 && at < 2 * a.pairs;
      const bool first = at < a.pairs;
      other = inside ? (first ? lane + a.pairs / 8 : lane - a.pairs / 8) : lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pair = F == kHalf ? (first ? at : at - a.pairs) + i : (at + i) / 2;
        const float2 t = inside ? angles[pair] : make_float2(1.f, 0.f);
        c[i] = t.x;
        s[i] = (F == kHalf ? first : i % 2 == 0) ? -t.y : t.y;
      }
    }
  }
  __device__ __forceinline__ void apply(float (&x)[8]) const {
    if constexpr (F == kHalf) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = __shfl_sync(0xFFFFFFFFu, x[i], other, 16);
        if (inside) x[i] = fmaf(y, s[i], x[i] * c[i]);
      }
    } else if constexpr (F == kNeighbours) {
      if (inside) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float p = x[i], q = x[i + 1];
          x[i] = fmaf(q, s[i], p * c[i]);
          x[i + 1] = fmaf(p, s[i + 1], q * c[i + 1]);
        }
      }
    }
  }
};

// The largest magnitude of the half warp's row, as the bits of its value; NaN is above all.
__device__ __forceinline__ uint32_t largest(const float (&x)[8]) {
  float m = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(x[i])));
  return __reduce_max_sync(0xFFFFu << (threadIdx.x & 16), __float_as_uint(m) & 0x7FFFFFFFu);
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Codes of a lane's eight values: x * inv, inv = 448 / amax. (A NaN makes inv and all codes NaN, an
// infinity makes inv 0.) `m` is amax's bits.
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], uint32_t m, float inv) {
  uint32_t c[4];
  if (inv == __uint_as_float(0x7F800000u)) {  // 448 / amax overflows (amax below about 1.3e-36), or is 448 / 0
    if (m == 0) return make_uint2(0u, 0u);
    const float scale = __fdiv_rn(__uint_as_float(m), 448.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = e4m3x2(__fdiv_rn(x[2 * i], scale), __fdiv_rn(x[2 * i + 1], scale));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = e4m3x2(__fmul_rn(x[2 * i], inv), __fmul_rn(x[2 * i + 1], inv));
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
  const uint4 row = reinterpret_cast<const uint4*>(a.k + t * a.k_token)[lane];
  const int p = a.pos[t], s = a.seq_id[t];
  if constexpr (F != kNone) {
    for (int i = lane; i < a.pairs; i += 16) angles[half][i] = angle(a, p, i);
    __syncwarp();
  }
  float x[8];
  unpack(row, x);
  if (a.norm_weight) normalise(a, x, lane);
  Turn<F>(a, lane, angles[half]).apply(x);
  const uint32_t m = largest(x);
  const float amax = __uint_as_float(m);
  const uint2 codes = codes_of(x, m, __fdiv_rn(448.f, amax));
  if (t0 + half >= a.tokens) return;
  int bad = 0;
  uint8_t* dst = slot_of(a, s, p, &bad);
  if (dst) {
    reinterpret_cast<uint2*>(dst)[lane] = codes;
    if (lane == 0) *reinterpret_cast<float*>(dst + TQ_INDEX_DIM) = __fdiv_rn(amax, 448.f);
  } else if (lane == 0 && a.flags) {
    atomicOr(a.flags, bad);
  }
}

// Heads [h0, h1) of token t, 2 * kHalves at a time.
template <Form F>
__device__ __forceinline__ void write_queries(const Args& a, int t, int h0, int h1) {
  __shared__ float2 angles[TQ_INDEX_DIM / 2];
  __shared__ float scales[128];
  const int tid = threadIdx.x, lane = tid & 15, half = tid >> 4;
  const uint8_t* q = a.q + t * a.q_token;
  auto load = [&](int h) {
    return h < h1 ? reinterpret_cast<const uint4*>(q + h * a.q_head)[lane] : make_uint4(0, 0, 0, 0);
  };
  uint4 row[2] = {load(h0 + half), load(h0 + half + kHalves)};
  if constexpr (F != kNone) {
    if (tid < a.pairs) angles[tid] = angle(a, a.pos[t], tid);
    __syncthreads();
  }
  const Turn<F> turn(a, lane, angles);
  uint8_t* out = a.q_out + (long long)t * a.heads * TQ_INDEX_DIM + 8 * lane;
#pragma unroll 1
  for (int h = h0 + half; h - half < h1; h += 2 * kHalves) {
    float x[2][8];
    unpack(row[0], x[0]);
    unpack(row[1], x[1]);
    if (h - half + 2 * kHalves < h1) {
      row[0] = load(h + 2 * kHalves);
      row[1] = load(h + 3 * kHalves);
    }
    turn.apply(x[0]);
    turn.apply(x[1]);
    const uint32_t m0 = largest(x[0]), m1 = largest(x[1]);
    // Lanes 0 to 3 of four: scale and inverse of the first row, of the second.
    const float amax = __uint_as_float(lane & 2 ? m1 : m0);
    const float mine = __fdiv_rn(lane & 1 ? 448.f : amax, lane & 1 ? amax : 448.f);
    const float inv0 = __shfl_sync(0xFFFFFFFFu, mine, (lane & ~3) | 1, 16);
    const float inv1 = __shfl_sync(0xFFFFFFFFu, mine, lane | 3, 16);
    const uint2 c0 = codes_of(x[0], m0, inv0), c1 = codes_of(x[1], m1, inv1);
    if (h < h1) *reinterpret_cast<uint2*>(out + h * TQ_INDEX_DIM) = c0;
    if (h + kHalves < h1) *reinterpret_cast<uint2*>(out + (h + kHalves) * TQ_INDEX_DIM) = c1;
    const int of = h + (lane & 2 ? kHalves : 0);
    if ((lane & 13) == 0 && of < h1) scales[of - h0] = mine;
  }
  __syncthreads();
  for (int h = h0 + tid; h < h1; h += kThreads) {
    const long long at = (long long)t * a.heads + h;
    const float w = a.w_f32 ? reinterpret_cast<const float*>(a.w)[at]
                            : __uint_as_float(uint32_t(reinterpret_cast<const uint16_t*>(a.w)[at]) << 16);
    a.w_out[at] = w * a.scale * scales[h - h0];
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
    const int t = block / a.parts, h0 = block % a.parts * a.each;
    write_queries<F>(a, t, h0, min(a.heads, h0 + a.each));
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
    a.q_head = (long long)s.q.strides_bytes[1];
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
  // Few tokens: a block for every 16 heads, so that they are read at once. Many: one for a token's.
  a.parts = a.tokens < 256 ? (a.heads + 2 * kHalves - 1) / (2 * kHalves) : a.heads ? 1 : 0;
  a.each = a.parts ? (a.heads + a.parts - 1) / a.parts : 0;
  const auto kernel = a.pairs == 0 ? index_write_kernel<kNone>
                      : s.rope_half ? index_write_kernel<kHalf>
                                    : index_write_kernel<kNeighbours>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.key_blocks + (long long)a.tokens * a.parts), 1, 1);
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
