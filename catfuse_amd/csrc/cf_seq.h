// Device helpers shared by the sequence operators (decay_attention.hip,
// decay_step.hip, rotary.hip): element types and their conversions.  These
// files take their argument blocks and limits from the C-ABI header itself
// (cf_common.h restates its constants as enumerators, so they do not include
// it).
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

}  // namespace
