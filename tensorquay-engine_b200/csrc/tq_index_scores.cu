// Index scores (tq_index_scores): a cheap score of every cached row for every query token,
//   scores[t, n] = key_scale[n] * sum_h w[t, h] * max(0, q[t, h] . k[n]),  n < sees(t).

#include <cuda_runtime.h>

#include <cstdint>

#include "tq_contracts.h"
#include "tq_ptx.cuh"

namespace tq {
namespace index_scores {

constexpr int kDim = TQ_INDEX_DIM;
constexpr int kPageRows = 64;
constexpr int kKeys = 128;   // keys of a block, one a thread
constexpr int kHeads = 16;   // heads staged at a time

struct Args {
  const uint8_t* q;
  const float* w;
  const uint8_t* kv;
  const int* page_table;
  const int* seq_id;
  const int* q_pos;
  const int* kv_len;
  float* scores;
  int* flags;
  long long row_stride;    // bytes
  long long score_stride;  // bytes
  int tokens, heads, sequences, slots, pages, columns;
};

// Rows that token t sees, 0 without a sequence; `bad` gets the flags of what is cut.
__device__ __forceinline__ int sees(const Args& a, int t, int* bad) {
  const int s = a.seq_id[t];
  if (s < 0 || s >= a.sequences) { *bad |= TQ_DEV_SEQ_RANGE; return 0; }
  const long long n = min((long long)a.kv_len[s], (long long)a.q_pos[t] + 1);
  const long long held = (long long)a.slots * kPageRows;
  if (n > held) *bad |= TQ_DEV_TABLE_SHORT;
  if (min(n, held) > a.columns) *bad |= TQ_DEV_WORK_OVERFLOW;
  return int(max(0ll, min(min(n, held), (long long)a.columns)));
}

__device__ __forceinline__ float2 e4m3_pair(uint32_t codes) {
  uint32_t h2;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}"
      : "=r"(h2) : "r"(codes));
  float lo, hi;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
      : "=f"(lo), "=f"(hi) : "r"(h2));
  return make_float2(lo, hi);
}

__global__ void __launch_bounds__(kKeys) index_scores_kernel(const Args a) {
  __shared__ float4 q[kHeads][kDim / 4];
  const int n = blockIdx.x * kKeys + threadIdx.x;
  for (int t = blockIdx.y; t < a.tokens; t += gridDim.y) {
    int bad = 0;
    const int count = sees(a, t, &bad);
    if (n == 0 && bad && a.flags) atomicOr(a.flags, bad);
    if (int(blockIdx.x) * kKeys >= count) continue;
    float k[kDim], scale = 0.f;
    for (int i = 0; i < kDim; ++i) k[i] = 0.f;
    if (n < count) {
      const int page = a.page_table[(long long)a.seq_id[t] * a.slots + n / kPageRows];
      if (page >= 0 && page < a.pages) {
        const uint8_t* row = a.kv + ((long long)page * kPageRows + n % kPageRows) * a.row_stride;
        scale = *reinterpret_cast<const float*>(row + kDim);
        for (int i = 0; i < kDim / 16; ++i) {
          const uint4 c = reinterpret_cast<const uint4*>(row)[i];
          const uint32_t u[4] = {c.x, c.y, c.z, c.w};
          for (int j = 0; j < 8; ++j) {
            const float2 v = e4m3_pair(u[j / 2] >> (16 * (j & 1)));
            k[16 * i + 2 * j] = v.x;
            k[16 * i + 2 * j + 1] = v.y;
          }
        }
      } else if (a.flags) {
        atomicOr(a.flags, TQ_DEV_PAGE_RANGE);
      }
    }
    float sum = 0.f;
    for (int h0 = 0; h0 < a.heads; h0 += kHeads) {
      const int heads = min(kHeads, a.heads - h0);
      __syncthreads();
      for (int i = threadIdx.x; i < heads * (kDim / 4); i += kKeys) {
        const uint32_t c = reinterpret_cast<const uint32_t*>(
            a.q + ((long long)t * a.heads + h0) * kDim)[i];
        const float2 lo = e4m3_pair(c), hi = e4m3_pair(c >> 16);
        q[i / (kDim / 4)][i % (kDim / 4)] = make_float4(lo.x, lo.y, hi.x, hi.y);
      }
      __syncthreads();
      for (int h = 0; h < heads; ++h) {
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < kDim / 4; ++i) {
          const float4 v = q[h][i];
          dot = fmaf(v.x, k[4 * i], dot);
          dot = fmaf(v.y, k[4 * i + 1], dot);
          dot = fmaf(v.z, k[4 * i + 2], dot);
          dot = fmaf(v.w, k[4 * i + 3], dot);
        }
        const float r = dot < 0.f ? 0.f : dot;  // NaN stays NaN
        sum = fmaf(a.w[(long long)t * a.heads + h0 + h], r, sum);
      }
    }
    if (n < count)
      reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a.scores) + t * a.score_stride)[n] =
          sum * scale;
  }
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
  if (s.q.shape[0] == 0 || s.scores.shape[1] == 0) return fail(nullptr, TQ_OK);
  auto ints = [](const TqTensorSpec& t) { return reinterpret_cast<const int*>(t.device_address); };
  Args a = {};
  a.q = reinterpret_cast<const uint8_t*>(s.q.device_address);
  a.w = reinterpret_cast<const float*>(s.w.device_address);
  a.kv = reinterpret_cast<const uint8_t*>(s.kv.device_address);
  a.page_table = ints(s.page_table);
  a.seq_id = ints(s.seq_id);
  a.q_pos = ints(s.q_pos);
  a.kv_len = ints(s.kv_len);
  a.scores = reinterpret_cast<float*>(s.scores.device_address);
  a.flags = device_flags;
  a.row_stride = (long long)s.kv.strides_bytes[1];
  a.score_stride = (long long)s.scores.strides_bytes[0];
  a.tokens = int(s.q.shape[0]);
  a.heads = int(s.q.shape[1]);
  a.sequences = int(s.page_table.shape[0]);
  a.slots = int(s.page_table.shape[1]);
  a.pages = int(s.kv.shape[0]);
  a.columns = int(s.scores.shape[1]);
  const unsigned blocks = unsigned((a.columns + kKeys - 1) / kKeys);
  const unsigned rows = unsigned(a.tokens < 65535 ? a.tokens : 65535);
  index_scores_kernel<<<dim3(blocks, rows), kKeys, 0, static_cast<cudaStream_t>(stream)>>>(a);
  if (cudaGetLastError() != cudaSuccess) return fail("launch", TQ_ERR_CUDA);
  return fail(nullptr, TQ_OK);
}
