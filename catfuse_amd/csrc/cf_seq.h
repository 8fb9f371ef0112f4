// Device helpers shared by the sequence operators (decay_attention.hip,
// decay_step.hip, delta_attention.hip, delta_step.hip, rotary.hip) and the dense
// products (linear.hip): element types and their conversions.  These files take
// their argument blocks and limits from the C-ABI header itself (cf_common.h
// restates its constants as enumerators, so they do not include it).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "catfuse_amd.h"

#define CF_API extern "C" __attribute__((visibility("default")))

namespace {

// Element types of the sequence operators (the `dtype` field of their
// argument blocks).
enum { SEQ_F32 = 0, SEQ_F16 = 1, SEQ_BF16 = 2 };

typedef __bf16 bf16_t;

template <typename T>
__device__ __forceinline__ float to_f(T x) { return (float)x; }
template <typename T>
__device__ __forceinline__ T from_f(float x) { return (T)x; }   // to nearest even

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec { T v[N]; };

// Offset i of packed sequences, int32 or int64 (wide) in device memory, where
// nothing has checked it: clamped to the tensors' rows 0 .. tokens.  (That one
// below its predecessor counts as that is left to the caller.)
__device__ __forceinline__ int64_t seq_offset(const void* cu, int wide, int64_t i, int64_t tokens) {
  const int64_t o = wide ? reinterpret_cast<const int64_t*>(cu)[i]
                         : (int64_t)reinterpret_cast<const int32_t*>(cu)[i];
  return o < 0 ? 0 : (o > tokens ? tokens : o);
}

// Number i of a tensor that is fp32 (f32) or of the operator's type.
template <typename T>
__device__ __forceinline__ double load_double(const void* p, int64_t i, int f32) {
  return f32 ? (double)reinterpret_cast<const float*>(p)[i]
             : (double)to_f(reinterpret_cast<const T*>(p)[i]);
}

typedef int i32x4 __attribute__((ext_vector_type(4)));

// One copy of 16 bytes a lane from a buffer straight to LDS: byte `at` of the
// buffer (zeros beyond its range), `add` bytes on, to lds + 16 lane.  In
// assembly, so that the compiler does not wait for it before every read of LDS;
// the kernel waits before the barrier that lets the copies be read.
__device__ __forceinline__ void copy16(i32x4 rsrc, uint32_t at, uint32_t add, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %0, %1, %2 offen lds"
      :
      : "v"(at), "s"(rsrc), "s"(add), "s"(lds)
      : "memory");
}
__device__ __forceinline__ i32x4 buffer_of(const void* base, uint32_t bytes) {
  const uint64_t p = (uint64_t)(uintptr_t)base;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)p);
  r[1] = __builtin_amdgcn_readfirstlane((int)((uint32_t)(p >> 32) & 0xffffu));
  r[2] = __builtin_amdgcn_readfirstlane((int)bytes);
  r[3] = 0x00020000;
  return r;
}

// Head h of the delta rule's states reads head h / (heads / n) of the n of each
// input.
static inline bool delta_heads_fit(int64_t heads, int64_t q, int64_t k, int64_t v) {
  return heads >= 1 && heads <= CF_SEQ_MAX_HEADS && q >= 1 && k >= 1 && v >= 1 && heads % q == 0 &&
         heads % k == 0 && heads % v == 0;
}

}  // namespace
