// What the attention translation units share: the arguments as the kernels take them, and the
// rule on which keys a query sees.
#pragma once

#include <cuda_fp16.h>

#include "runtime.cuh"

namespace lsr {

struct AttnStride {
  long long b, s, h;  // batch, position, head (elements; the head's entries are contiguous)
};

struct AttnParams {
  int batch, q_len, kv_len, heads, kv_heads, head_dim, causal;
  int group;      // query heads per key head
  float scale;
  const void *q, *k, *v, *dout;
  void *out, *dq, *dk, *dv;
  AttnStride sq, sk, sv, so, sdo, sdq, sdk, sdv;
  const unsigned char* mask;  // [batch][kv_len], nonzero = seen; nullptr: every key is
  long long mask_stride;
  float* lse;    // [batch][heads][q_len], natural logarithm
  float* delta;  // [batch][heads][q_len]: sum over the head's entries of dout * out (backward)
  int* status;
};

template <typename T>
__device__ __forceinline__ const T* attn_at(const void* p, const AttnStride& s, int b, int h) {
  return static_cast<const T*>(p) + (long long)b * s.b + (long long)h * s.h;
}
template <typename T>
__device__ __forceinline__ T* attn_at(void* p, const AttnStride& s, int b, int h) {
  return static_cast<T*>(p) + (long long)b * s.b + (long long)h * s.h;
}

__device__ __forceinline__ float attn_to_f(float x) { return x; }
__device__ __forceinline__ float attn_to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float attn_to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T attn_from_f(float x);
template <>
__device__ __forceinline__ float attn_from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 attn_from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half attn_from_f<__half>(float x) { return __float2half_rn(x); }

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Programmatic dependent launch: the next kernel of the stream may start; wait for the kernel
// before to have finished and its writes to be seen.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_dependency() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// attention_general.cu: 32-bit arithmetic on the CUDA cores, any type, stride and alignment.
int attention_forward_general(const AttnParams& p, int dtype, cudaStream_t st);
int attention_backward_general(const AttnParams& p, int dtype, cudaStream_t st);

}  // namespace lsr
