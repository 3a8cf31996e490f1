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

// The offsets from `from` on, 256 at most, among which the first behind `row` is (`to` where none of them is): those before
// are at or before the row. By 64 probes of a wave a round; offsets out of order give some place among them.
// 100000 one-row requests, 64 -> 64: 0.11 ms forward and 0.25 backward (3.2 and 6.5 with each workgroup passing over them all).
struct OffsetRange {
  int64_t from, to;
};
__device__ __forceinline__ OffsetRange offsets_near(const Requests& q, int64_t row, int lane) {
  OffsetRange r{0, (int64_t)q.count + 1};
  while (r.to - r.from > 256) {
    const int64_t step = (r.to - r.from + 63) / 64, at = r.from + (lane + 1) * step - 1;
    r.from += __popcll(__ballot(at < r.to && q.offsets[at < r.to ? at : r.to - 1] <= row)) * step;
    if (r.from + step - 1 < r.to) r.to = r.from + step - 1;
  }
  return r;
}

// A sum of products one of whose operands is kept as bf16 parts: `first` is that of the first parts, `rest` that of the
// others. What an infinity leaves for its other parts is NaN, and so is an infinite other operand's product with parts of both
// signs or of zero: where the first parts' sum is not finite it is the value by itself.
__device__ __forceinline__ float parts_sum(float first, float rest) {
  return __builtin_isfinite(first) ? first + rest : first;
}
__device__ __forceinline__ f32x4 parts_sum(const f32x4& first, const f32x4& rest) {
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = parts_sum(first[e], rest[e]);
  return v;
}

}  // namespace ffk
