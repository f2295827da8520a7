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
#include "sm100.cuh"

namespace tfb {

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

// x, residual and y may be the same buffer (an element is read before it is
// written, by the CTA that writes it), so none of them is __restrict__.
//
// Persistent CTAs take chunks of 8 KB of x (and of the residual) in turn,
// through a ring of shared-memory stages filled by bulk copies, so that loads
// run on under the generator's arithmetic.  With plain loads, 16384 x 4096
// bf16 with a residual took 89 us (18 stalled cycles an instruction waiting
// for loads), and 126 us with four groups' loads in flight a thread; so 71-74 us.
constexpr int kDropStages = 4;
constexpr int kDropChunkBytes = 8192;
constexpr int kDropSmem = kDropStages * 2 * kDropChunkBytes;
constexpr int kDropCtas = 148 * 3;

__device__ __forceinline__ void dropout_lds8(uint32_t addr, float (&v)[8], __nv_bfloat16) {
  uint4 a;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w)
               : "r"(addr)
               : "memory");
  bf16x8_to_f32(a, v);
}
__device__ __forceinline__ void dropout_lds8(uint32_t addr, float (&v)[8], float) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v[4 * h]), "=f"(v[4 * h + 1]), "=f"(v[4 * h + 2]), "=f"(v[4 * h + 3])
                 : "r"(addr + 16 * h)
                 : "memory");
}

template <typename T>
__global__ void __launch_bounds__(256)
    dropout_kernel(const T* x, const T* residual, T* y, long long n, DropoutParams d) {
  constexpr int GROUP = 8 * (int)sizeof(T);              // bytes of a group
  constexpr int CHUNK = kDropChunkBytes / GROUP;         // groups of a chunk
  extern __shared__ uint4 drop_stages[];
  __shared__ uint64_t bars[kDropStages];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kDropStages; ++i) mbar_init(smem_u32(bars + i), 1);
    abort_word = 0;
    fence_mbar_init();
  }
  __syncthreads();
  PhiloxState s = {};
  if (d.rng) s = philox_state(d);  // null: nothing is dropped
  const long long groups = n / 8;
  const uint32_t data = smem_u32(drop_stages);
  const int per_stage = residual ? 2 : 1;
  auto first = [&](int k) { return ((long long)k * gridDim.x + blockIdx.x) * CHUNK; };
  auto issue = [&](int k) {
    const long long g = first(k);
    if (g >= groups) return;
    const uint32_t bytes = (uint32_t)min((long long)CHUNK, groups - g) * GROUP;
    const uint32_t bar = smem_u32(bars + k % kDropStages);
    const uint32_t dst = data + (k % kDropStages) * 2 * kDropChunkBytes;
    mbar_arrive_expect_tx(bar, bytes * per_stage);
    bulk_load(dst, x + g * 8, bytes, bar);
    if (residual) bulk_load(dst + kDropChunkBytes, residual + g * 8, bytes, bar);
  };
  if (threadIdx.x == 0)
    for (int k = 0; k < kDropStages; ++k) issue(k);
  int k = 0;
  for (; first(k) < groups; ++k) {
    (void)mbar_wait(smem_u32(bars + k % kDropStages), (k / kDropStages) & 1, abort_flag, 951);
    const long long g0 = first(k);
    const uint32_t src = data + (k % kDropStages) * 2 * kDropChunkBytes;
#pragma unroll
    for (int i = threadIdx.x; i < CHUNK; i += 256) {
      if (g0 + i >= groups) break;
      float v[8];
      dropout_lds8(src + i * GROUP, v, T());
      if (d.rng) dropout8(d, s, (uint32_t)(g0 + i), v);
      if (residual) {
        float r[8];
        dropout_lds8(src + kDropChunkBytes + i * GROUP, r, T());
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
      }
      dropout_store8(y + (g0 + i) * 8, v);
    }
    __syncthreads();  // every thread has read the stage
    if (threadIdx.x == 0) issue(k + kDropStages);
  }
  if (*abort_flag && threadIdx.x == 0)  // copies in flight land before the shared memory goes away
    for (int u = max(0, k - kDropStages); u < k; ++u)
      (void)mbar_wait(smem_u32(bars + u % kDropStages), (u / kDropStages) & 1, nullptr, 952);
  // the last group, when n is no multiple of 8
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0 && (n & 7)) {
    float t[8];
    const int left = (int)(n & 7);
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = e < left ? dropout_to_f32(x[groups * 8 + e]) : 0.0f;
    if (d.rng) dropout8(d, s, (uint32_t)groups, t);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) {
        const float b = residual ? dropout_to_f32(residual[groups * 8 + e]) : 0.0f;
        dropout_put(y + groups * 8 + e, t[e] + b);
      }
  }
}

}  // namespace tfb
