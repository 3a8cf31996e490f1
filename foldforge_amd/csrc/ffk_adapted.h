// Shared by the kernels of the projections with low-rank adapters (adapted.hip, adapted_rows.hip).
#pragma once

#include "ffk_device.h"

namespace ffk {

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Which adapter a row has: the requests of a call.
struct Requests {
  const int32_t *offsets, *adapter;  // [count + 1], [count]
  const float* scale;                // [adapters], or null (1)
  int count, adapters;
  int64_t rows;
};

// (read from some address in any case: a branch would wait for the value)
__device__ __forceinline__ float scale_of(const Requests& q, int a) {
  const float v = *(q.scale ? q.scale + a : reinterpret_cast<const float*>(q.offsets));
  return q.scale ? v : 1.f;
}

}  // namespace ffk
