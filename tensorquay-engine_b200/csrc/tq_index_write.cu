// Index write (tq_index_write): index queries and keys of a step, rotated, quantized to E4M3, the
// keys written to their paged cache. A row of 128 values (one head of a query, or a key):
//   k only: k / sqrt(mean(k^2) + eps) * w, or (k - mean(k)) / sqrt(var(k) + eps) * w + b
//   pair (a, b) of the rotary part -> (a c - b s, a s + b c), c and s the cosine and sine of
//   pos * freq[i], times rope_mscale
//   scale = amax / 448, code = E4M3(x * (448 / amax)); w_out = w * scale_c * scale
// All f32 from the read to the code. The angle is a product of f64 and loses its whole turns before
// it is rounded to f32: at position 2^20 an f32 angle would be off by 2^-5.
//
// What bounds it: HBM for many tokens (256 bytes read and 128 written a head), one launch's chain of
// loads (position, angles, row) for few. Half a warp holds a row, 8 values a lane, so one 16-byte
// load, no value of a pair more than a shuffle away, and four shuffles for the row's largest. A
// block has one token and 16 rows at a time: its angles are computed once for all heads, while
// the first rows are on their way.

#include <cuda_runtime.h>

#include <cstdint>

#include "tq_contracts.h"
#include "tq_ptx.cuh"

namespace tq {
namespace index_write {

constexpr int kThreads = 256;
constexpr int kRows = kThreads / 16;  // rows of a block at a time
constexpr int kPageRows = 64;

struct Args {
  const uint8_t* q;  // null: keys only
  const uint8_t* k;
  const uint8_t* w;
  const uint8_t* norm_weight;  // null: k as it is
  const uint8_t* norm_bias;    // null: RMS
  const float* freq;           // null: no rotary part
  uint8_t* kv;
  uint8_t* q_out;
  float* w_out;
  const int* page_table;
  const int* seq_id;
  const int* pos;
  int* flags;
  long long q_token, q_head, k_token, row_stride;  // bytes
  int heads, sequences, slots, pages, w_f32;
  int start, half, pairs;  // rotary part: first value, halves or neighbours, angles
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

__device__ __forceinline__ float sum16(float v, unsigned mask) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
  return v;
}

// The key's norm; `mask` names the half warp that holds it.
__device__ __forceinline__ void normalise(const Args& a, float (&x)[8], int lane, unsigned mask) {
  float w[8];
  unpack(reinterpret_cast<const uint4*>(a.norm_weight)[lane], w);
  float s = 0.f;
  if (a.norm_bias) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[i];
    const float mean = sum16(s, mask) * (1.f / TQ_INDEX_DIM);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] -= mean;
  }
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(x[i], x[i], s);
  const float r = 1.f / sqrtf(sum16(s, mask) * (1.f / TQ_INDEX_DIM) + a.eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= r * w[i];
  if (a.norm_bias) {
    unpack(reinterpret_cast<const uint4*>(a.norm_bias)[lane], w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] += w[i];
  }
}

// The rotary part of a row; all lanes of the warp take part. `turn` holds (cosine, sine) by pair.
__device__ __forceinline__ void rotate(const Args& a, float (&x)[8], int lane, const float2* turn) {
  const int at = 8 * lane - a.start;
  const bool inside = at >= 0 && at < 2 * a.pairs;
  if (a.half) {
    // The partner of a value is `pairs` values away: the same place in another lane's eight.
    const bool first = at < a.pairs;
    const int other = inside ? (first ? lane + a.pairs / 8 : lane - a.pairs / 8) : lane;
    const int i0 = inside ? (first ? at : at - a.pairs) : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = __shfl_sync(0xFFFFFFFFu, x[i], other, 16);
      const float2 t = turn[i0 + i];
      if (inside) x[i] = first ? x[i] * t.x - y * t.y : y * t.y + x[i] * t.x;
    }
  } else if (inside) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = turn[at / 2 + i];
      const float p = x[2 * i], q = x[2 * i + 1];
      x[2 * i] = p * t.x - q * t.y;
      x[2 * i + 1] = p * t.y + q * t.x;
    }
  }
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// The codes of a row's eight values in this lane, and the row's scale. All lanes take part.
__device__ __forceinline__ uint2 quantize(const float (&x)[8], int lane, float* scale) {
  // As whole numbers |x| orders like the values, and every NaN is above infinity.
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  const float amax = __uint_as_float(m);
  // One division a lane: even lanes make the scale, odd lanes its inverse.
  const bool odd = lane & 1;
  const float mine = __fdiv_rn(odd ? 448.f : amax, odd ? amax : 448.f);
  const float theirs = __shfl_xor_sync(0xFFFFFFFFu, mine, 1);
  *scale = odd ? theirs : mine;
  const float inv = odd ? mine : theirs;
  if (m > 0x7F800000u) return make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);  // scale is NaN
  if (m == 0) return make_uint2(0u, 0u);
  uint32_t c[4];
  if (inv < __uint_as_float(0x7F800000u)) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c[i] = e4m3x2(__fmul_rn(x[2 * i], inv), __fmul_rn(x[2 * i + 1], inv));
  } else {  // 448 / amax overflows (amax below about 1.3e-36)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c[i] = e4m3x2(__fdiv_rn(x[2 * i], *scale), __fdiv_rn(x[2 * i + 1], *scale));
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

// Where token t's key goes, or null with the flag that says why not.
__device__ __forceinline__ uint8_t* slot_of(const Args& a, int t, int p, int* bad) {
  const int s = a.seq_id[t];
  if (s < 0 || s >= a.sequences) { *bad = TQ_DEV_SEQ_RANGE; return nullptr; }
  if (p < 0 || p / kPageRows >= a.slots) { *bad = TQ_DEV_TABLE_SHORT; return nullptr; }
  const int page = a.page_table[(long long)s * a.slots + p / kPageRows];
  if (page < 0 || page >= a.pages) { *bad = TQ_DEV_PAGE_RANGE; return nullptr; }
  return a.kv + ((long long)page * kPageRows + p % kPageRows) * a.row_stride;
}

__global__ void __launch_bounds__(kThreads) index_write_kernel(const Args a) {
  __shared__ float2 turn[TQ_INDEX_DIM / 2];
  const int lane = threadIdx.x & 15, sub = threadIdx.x >> 4;
  const unsigned mine = 0xFFFFu << (threadIdx.x & 16);
  const int t = blockIdx.x;
  // Row 0 is the key, row 1 + h the query of head h. A warp's two rows go through the loop together.
  const int rows = 1 + a.heads;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  auto load = [&](int r) {
    const uint8_t* src = r == 0 ? a.k + t * a.k_token : a.q + t * a.q_token + (r - 1) * a.q_head;
    return r < rows ? reinterpret_cast<const uint4*>(src)[lane] : make_uint4(0, 0, 0, 0);
  };
  int r = int(blockIdx.y) * kRows + sub;
  const int step = int(gridDim.y) * kRows;
  uint4 next = load(r);
  const int p = a.pos[t];
  if (a.freq) {
    if (threadIdx.x < a.pairs) {
      double turns = double(p) * double(a.freq[threadIdx.x]) * 0.15915494309189533577;
      turns -= rint(turns);
      float s, c;
      sincospif(2.f * float(turns), &s, &c);
      turn[threadIdx.x] = make_float2(c * a.mscale, s * a.mscale);
    }
    __syncthreads();
  }
  for (; (r & ~1) < rows; r += step) {
    float x[8];
    unpack(next, x);
    next = load(r + step);
    if (r == 0 && a.norm_weight) normalise(a, x, lane, mine);
    if (a.freq) rotate(a, x, lane, turn);
    float scale;
    const uint2 codes = quantize(x, lane, &scale);
    if (r == 0) {
      int bad = 0;
      uint8_t* dst = slot_of(a, t, p, &bad);
      if (dst) {
        reinterpret_cast<uint2*>(dst)[lane] = codes;
        if (lane == 0) *reinterpret_cast<float*>(dst + TQ_INDEX_DIM) = scale;
      } else if (lane == 0 && a.flags) {
        atomicOr(a.flags, bad);
      }
    } else if (r < rows) {
      const long long at = (long long)t * a.heads + r - 1;
      reinterpret_cast<uint2*>(a.q_out + at * TQ_INDEX_DIM)[lane] = codes;
      if (lane == 0) {
        const float w = a.w_f32 ? reinterpret_cast<const float*>(a.w)[at]
                                : __uint_as_float(uint32_t(reinterpret_cast<const uint16_t*>(a.w)[at]) << 16);
        a.w_out[at] = w * a.scale * scale;
      }
    }
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
  a.half = s.rope_half != 0;
  a.mscale = s.rope_mscale;
  a.eps = s.norm_eps;
  a.scale = s.scale;
  // Few tokens: a block for every 16 rows, so that they are read at once. Many: one for a token.
  const unsigned blocks = unsigned(1 + a.heads + kRows - 1) / kRows;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(tokens), tokens < 256 ? blocks : 1u, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, index_write_kernel, a) != cudaSuccess)
    return fail("launch", TQ_ERR_CUDA);
  return fail(nullptr, TQ_OK);
}
