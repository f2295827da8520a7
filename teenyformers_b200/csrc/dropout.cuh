// dropout.cuh -- y = dropout(x) (+ residual), its mask drawn from a
// counter-based generator (philox.cuh) and never stored.  The map is
// self-adjoint, so the backward pass is the same call on the gradient.
//
// HBM-bound: each element is read and written once (bf16: 4 bytes, 6 with a
// residual), and one generator call (20 wide multiplies) covers the 8 elements
// that a thread handles at a time, two 16-byte vectors in fp32, one in bf16.
#pragma once

#include "norm_act.cuh"
#include "philox.cuh"

namespace tfb {

__device__ __forceinline__ void dropout_load8(const __nv_bfloat16* p, float (&v)[8]) {
  bf16x8_to_f32(*reinterpret_cast<const uint4*>(p), v);
}
__device__ __forceinline__ void dropout_load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void dropout_store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = f32_to_bf16x8(v);
}
__device__ __forceinline__ void dropout_store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ float dropout_to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float dropout_to_f32(float v) { return v; }
__device__ __forceinline__ void dropout_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void dropout_put(float* p, float v) { *p = v; }

// x, residual and y may be the same buffer (each element is read before it is
// written, by the same thread), so none of them is __restrict__.
template <typename T>
__global__ void __launch_bounds__(256)
    dropout_kernel(const T* x, const T* residual, T* y, long long n, DropoutParams d) {
  PhiloxState s = {};
  if (d.rng) s = philox_state(d);  // null: nothing is dropped
  const long long groups = n / 8;
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long g = (long long)blockIdx.x * blockDim.x + threadIdx.x; g < groups; g += step) {
    float v[8];
    dropout_load8(x + g * 8, v);
    if (d.rng) dropout8(d, s, (uint32_t)g, v);
    if (residual) {
      float r[8];
      dropout_load8(residual + g * 8, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += r[e];
    }
    dropout_store8(y + g * 8, v);
  }
  // the last group, when n is no multiple of 8
  if (blockIdx.x == 0 && threadIdx.x == 0 && (n & 7)) {
    float v[8];
    const int left = (int)(n & 7);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? dropout_to_f32(x[groups * 8 + e]) : 0.0f;
    if (d.rng) dropout8(d, s, (uint32_t)groups, v);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) {
        const float r = residual ? dropout_to_f32(residual[groups * 8 + e]) : 0.0f;
        dropout_put(y + groups * 8 + e, v[e] + r);
      }
  }
}

}  // namespace tfb
