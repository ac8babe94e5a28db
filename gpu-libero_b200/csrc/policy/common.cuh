// Element types, conversions and reductions shared by the policy operators.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "b200policy.h"

namespace b200policy {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

inline size_t element_bytes(int dtype) { return dtype == B200_FP32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype >= B200_FP32 && dtype <= B200_BF16; }

// Calls f with a value of the element type that `dtype` names.
template <class F> int by_dtype(int dtype, F f) {
  switch (dtype) {
    case B200_FP32: return f(float());
    case B200_FP16: return f(__half());
    case B200_BF16: return f(__nv_bfloat16());
  }
  return (int)cudaErrorInvalidValue;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
  return x;
}
__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
  return x;
}

// Sum over the block (a multiple of 32 threads, at most 1024), on every
// thread; the order is fixed by the block's size.  `part` holds 32 values and
// may be used again after the call.
template <class V> __device__ __forceinline__ V block_sum(V x, V *part) {
  x = warp_sum(x);
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) part[threadIdx.x >> 5] = x;
  __syncthreads();
  x = warp_sum(lane < warps ? part[lane] : V(0));
  __syncthreads();
  return x;
}

// What one chunk after another leaves of a memory: w = exp(log_left) each time.  w rounded
// to 32 bits would be off by the same amount every time (some decays of 1e-6 to 2e-6 a token by
// 1.7e-4 after 131072 tokens), so the two values around it, 2^-24 apart, take turns as often as
// w lies near them.  Below 1/2 a memory is gone before that counts.
struct Decay {
  float low;
  uint32_t share;  // of the chunks that take the upper value, times 2^32
  __device__ __forceinline__ explicit Decay(float log_left) : low(expf(log_left)), share(0) {
    if (!(low > 0.5f && low <= 1.f)) return;
    const float rest = (expm1f(log_left) - (low - 1.f)) * 0x1p24f, units = floorf(rest);
    low += units * 0x1p-24f;
    share = __float2uint_rz((rest - units) * 0x1p32f);
  }
  // the turn comes where the chunks' shares so far pass a whole one
  __device__ __forceinline__ float at(int chunk) const { return share * (chunk + 1u) < share ? low + 0x1p-24f : low; }
};

// Two values and the instructions that take both at once.
struct F2 {
  unsigned long long v;
  __device__ __forceinline__ F2() : v(0) {}
  __device__ __forceinline__ F2(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
  __device__ __forceinline__ explicit F2(float x) : F2(x, x) {}
  __device__ __forceinline__ float2 get() const {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
  }
  __device__ __forceinline__ float sum() const { return get().x + get().y; }
};
__device__ __forceinline__ F2 add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

}  // namespace b200policy
