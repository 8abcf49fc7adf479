// Block norm (tq_block_norm): the step between two blocks of a layer, one pass over the rows:
//   b  = post_weight ? rms(y) * post_weight : y
//   h' = residual + scale * gate * b          (written in the residual's type)
//   x  = rms(h') * pre_weight                 (written in bf16)
// with rms(v) = v / sqrt(mean(v^2) + eps). A row stays in registers in f32 from its one read to
// its writes: h' enters the second norm before it is rounded, and each output is rounded once.
//
// What bounds it: HBM for many rows (y and residual read once, h' and x written once, 8 bytes an
// element with a bf16 residual, 12 with f32), the launch and two block sums for few rows. One
// block per row, 8 consecutive elements a thread and step (16-byte loads); all of a row's loads
// are issued before the first sum. The block is sized so that a thread has at most kSteps steps:
// threads cost little, and a wider block shortens a lone row. Measured: 8192 rows of 7168 with an f32
// residual and a gate 136 us, 6.05 TB/s (0.93 of the measured copy rate; 256 threads of 4 steps 142
// us, 1024 of one 162); 64 rows of 4096 and one row of 7168 4.0 us a call where calls follow each
// other, of them 2 to 3 us on the device.

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "tq_contracts.h"
#include "tq_ptx.cuh"

namespace tq {
namespace norm {

struct Args {
  const uint8_t* y;
  const uint8_t* res;
  uint8_t* out;
  uint8_t* x;            // null: no second norm
  const uint8_t* post;   // null: y as it is
  const uint8_t* gate;   // null: 1
  const uint8_t* pre;
  long long y_stride, res_stride, out_stride, x_stride, gate_stride;  // bytes; gate 0: per channel
  int rows, width;
  float scale, post_eps, pre_eps;
};

__device__ __forceinline__ void unpack(const uint4& p, float (&v)[8]) {
  const uint32_t u[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = ptx::bf16_lo(u[k]);
    v[2 * k + 1] = ptx::bf16_hi(u[k]);
  }
}

__device__ __forceinline__ uint4 pack(const float (&v)[8]) {
  return make_uint4(ptx::pack_bf16x2(v[0], v[1]), ptx::pack_bf16x2(v[2], v[3]),
                    ptx::pack_bf16x2(v[4], v[5]), ptx::pack_bf16x2(v[6], v[7]));
}

template <int kThreads>
__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < kThreads / 32; ++k) s += part[k];
  return s;
}

template <int kThreads, int kSteps, bool kF32>
__global__ void __launch_bounds__(kThreads) block_norm_kernel(const Args a) {
  __shared__ float part[2][kThreads / 32];
  // Launched while the kernel before it ends; its results are waited for here.
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long row = blockIdx.x;
  const uint8_t* y = a.y + row * a.y_stride;
  const uint8_t* res = a.res + row * a.res_stride;
  const uint8_t* gate = a.gate ? a.gate + row * a.gate_stride : nullptr;
  uint4 yv[kSteps];
  float h[kSteps][8];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int i = (k * kThreads + int(threadIdx.x)) * 8;
    yv[k] = make_uint4(0, 0, 0, 0);
    if (i < a.width) {
      yv[k] = *reinterpret_cast<const uint4*>(y + 2ll * i);
      if (kF32) {
        const float4 p = *reinterpret_cast<const float4*>(res + 4ll * i);
        const float4 q = *reinterpret_cast<const float4*>(res + 4ll * i + 16);
        h[k][0] = p.x; h[k][1] = p.y; h[k][2] = p.z; h[k][3] = p.w;
        h[k][4] = q.x; h[k][5] = q.y; h[k][6] = q.z; h[k][7] = q.w;
      } else {
        unpack(*reinterpret_cast<const uint4*>(res + 2ll * i), h[k]);
      }
    }
  }
  float r = 1.f;
  if (a.post) {
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      float v[8];
      unpack(yv[k], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(v[j], v[j], sq);
    }
    r = 1.f / sqrtf(block_sum<kThreads>(sq, part[0]) / float(a.width) + a.post_eps);
  }
  float sq = 0.f;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int i = (k * kThreads + int(threadIdx.x)) * 8;
    if (i < a.width) {
      float v[8], w[8];
      unpack(yv[k], v);
      if (a.post) {
        unpack(*reinterpret_cast<const uint4*>(a.post + 2ll * i), w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * r * w[j];
      }
      if (gate) {
        unpack(*reinterpret_cast<const uint4*>(gate + 2ll * i), w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= w[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[k][j] = fmaf(a.scale, v[j], h[k][j]);
        sq = fmaf(h[k][j], h[k][j], sq);
      }
      uint8_t* out = a.out + row * a.out_stride;
      if (kF32) {
        *reinterpret_cast<float4*>(out + 4ll * i) = make_float4(h[k][0], h[k][1], h[k][2], h[k][3]);
        *reinterpret_cast<float4*>(out + 4ll * i + 16) =
            make_float4(h[k][4], h[k][5], h[k][6], h[k][7]);
      } else {
        *reinterpret_cast<uint4*>(out + 2ll * i) = pack(h[k]);
      }
    }
  }
  if (!a.x) return;
  r = 1.f / sqrtf(block_sum<kThreads>(sq, part[1]) / float(a.width) + a.pre_eps);
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int i = (k * kThreads + int(threadIdx.x)) * 8;
    if (i < a.width) {
      float w[8];
      unpack(*reinterpret_cast<const uint4*>(a.pre + 2ll * i), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] *= h[k][j] * r;
      *reinterpret_cast<uint4*>(a.x + row * a.x_stride + 2ll * i) = pack(w);
    }
  }
}

template <int kThreads, int kSteps>
cudaError_t launch(const Args& a, bool f32, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.rows), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return f32 ? cudaLaunchKernelEx(&cfg, block_norm_kernel<kThreads, kSteps, true>, a)
             : cudaLaunchKernelEx(&cfg, block_norm_kernel<kThreads, kSteps, false>, a);
}

}  // namespace norm
}  // namespace tq

extern "C" int32_t tq_block_norm(const TqBlockNormSpec* spec, void* stream, TqContractError* err) {
  using namespace tq::norm;
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  const int32_t st = tq::block_norm_validate(spec, err);
  if (st != TQ_OK) return st;
  const TqBlockNormSpec& s = *spec;
  if (s.y.shape[0] == 0) return fail(nullptr, TQ_OK);
  auto at = [](const TqTensorSpec& t) {
    return t.rank ? reinterpret_cast<uint8_t*>(t.device_address) : nullptr;
  };
  Args a;
  a.y = at(s.y);
  a.res = at(s.residual);
  a.out = at(s.out);
  a.x = at(s.x);
  a.post = at(s.post_weight);
  a.gate = at(s.gate);
  a.pre = at(s.pre_weight);
  a.y_stride = (long long)s.y.strides_bytes[0];
  a.res_stride = (long long)s.residual.strides_bytes[0];
  a.out_stride = (long long)s.out.strides_bytes[0];
  a.x_stride = s.x.rank ? (long long)s.x.strides_bytes[0] : 0;
  a.gate_stride = s.gate.rank == 2 ? (long long)s.gate.strides_bytes[0] : 0;
  a.rows = int(s.y.shape[0]);
  a.width = int(s.y.shape[1]);
  a.scale = s.scale;
  a.post_eps = s.post_eps;
  a.pre_eps = s.pre_eps;
  const bool f32 = s.residual.dtype == TQ_DTYPE_F32;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const int vecs = (a.width + 7) / 8;
  cudaError_t e;
  if (vecs <= 128) e = launch<128, 1>(a, f32, cs);
  else if (vecs <= 256) e = launch<256, 1>(a, f32, cs);
  else if (vecs <= 512) e = launch<256, 2>(a, f32, cs);
  else if (vecs <= 1024) e = launch<512, 2>(a, f32, cs);
  else if (vecs <= 2048) e = launch<512, 4>(a, f32, cs);
  else e = launch<1024, 4>(a, f32, cs);
  if (e != cudaSuccess) return fail("launch", TQ_ERR_CUDA);
  return fail(nullptr, TQ_OK);
}
