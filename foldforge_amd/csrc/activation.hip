// 8-bit activations on their own (ffk_activation.h): x -> codes and scales, and back. HBM-bound: x once,
// 33 / 32 bytes a value.
#include <algorithm>

#include "ffk_activation.h"
#include "ffk_device.h"
#include "ffk_kernels.h"

namespace ffk {

namespace {

constexpr int kActUnroll = 4;  // pieces a thread has in flight

// Widths that are whole blocks: the tensor is one run of 16-byte pieces, 32 / VE of them a block; x 16-byte,
// codes VE-byte aligned. A workgroup takes runs of 256 kActUnroll pieces. pieces: a multiple of 32 / VE.
// 196608 x 64 bf16: 8.4 us, and 8.3 back (4.5 TB/s: of each about 4 are the launch's own); 262144 x 128: 20 us, 5.1 TB/s.
template <typename T, int VE>
__global__ __launch_bounds__(256) void quantize_pieces(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                       uint8_t* __restrict__ scales, int64_t pieces) {
  using V = KeptPiece<T, false, VE>;
  const int64_t step = (int64_t)gridDim.x * 256 * kActUnroll;
  for (int64_t i0 = (int64_t)blockIdx.x * 256 * kActUnroll + threadIdx.x; i0 - threadIdx.x < pieces; i0 += step) {
    V v[kActUnroll];
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u)
      if (i0 + 256 * u < pieces) v[u].load(x, nullptr, i0 + 256 * u, 0, VE, 1);
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int64_t i = i0 + 256 * u;
      float f[VE];
      v[u].values(f);
      act_store<VE>(f, i < pieces, i % (kActBlock / VE) == 0, codes + i * VE, scales + i / (kActBlock / VE));
    }
  }
}

template <typename T, int VE>
__global__ __launch_bounds__(256) void restore_pieces(const uint8_t* __restrict__ codes,
                                                      const uint8_t* __restrict__ scales, T* __restrict__ x,
                                                      int64_t pieces) {
  using V = KeptPiece<T, true, VE>;
  typedef T vec __attribute__((__vector_size__(VE * sizeof(T))));
  const int64_t step = (int64_t)gridDim.x * 256 * kActUnroll;
  for (int64_t i0 = (int64_t)blockIdx.x * 256 * kActUnroll + threadIdx.x; i0 < pieces; i0 += step) {
    V v[kActUnroll];
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int64_t i = i0 + 256 * u;
      if (i < pieces) v[u].load(codes + i * VE, scales + i / (kActBlock / VE), 0, 0, VE, 1);
    }
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int64_t i = i0 + 256 * u;
      float f[VE];
      v[u].values(f);
      vec o;
#pragma unroll
      for (int e = 0; e < VE; ++e) o[e] = (T)f[e];
      if (i < pieces) __builtin_nontemporal_store(o, reinterpret_cast<vec*>(x + i * VE));
    }
  }
}

// Any width up to 64 K and any alignment: a wave a row, K values a lane (channels lane + 64 k: a block is half a wave).
// grid-strided; block 256. 10007 x 333 fp32: 7.9 us, and 7.2 back, half of it the launch's own.
template <typename T, int K>
__global__ __launch_bounds__(256) void quantize_rows(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                     uint8_t* __restrict__ scales, int64_t rows, int cols) {
  const int blocks = (cols + kActBlock - 1) / kActBlock, lane = threadIdx.x & 63;
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
    float v[K];
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lane + 64 * k < cols ? (float)x[row * cols + lane + 64 * k] : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = lane + 64 * k;
      act_store<1>(&v[k], c < cols, c % kActBlock == 0, codes + row * cols + c, scales + row * blocks + c / kActBlock);
    }
  }
}
template <typename T, int K>
__global__ __launch_bounds__(256) void restore_rows(const uint8_t* __restrict__ codes,
                                                    const uint8_t* __restrict__ scales, T* __restrict__ x, int64_t rows,
                                                    int cols) {
  const int blocks = (cols + kActBlock - 1) / kActBlock, lane = threadIdx.x & 63;
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
    KeptPiece<T, true, 1> v[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (lane + 64 * k < cols) v[k].load(codes, scales, row, lane + 64 * k, cols, blocks);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float f;
      v[k].values(&f);
      if (lane + 64 * k < cols) x[row * cols + lane + 64 * k] = (T)f;
    }
  }
}

// Wider rows: a wave takes 64 channels at a time.
template <typename T>
__global__ __launch_bounds__(256) void quantize_wide(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                     uint8_t* __restrict__ scales, int64_t rows, int cols) {
  const int blocks = (cols + kActBlock - 1) / kActBlock, lane = threadIdx.x & 63;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    for (int c0 = 64 * (threadIdx.x >> 6); c0 < cols; c0 += 256) {  // (uniform in a wave)
      const int c = c0 + lane;
      const float v = c < cols ? (float)x[row * cols + c] : 0.f;
      act_store<1>(&v, c < cols, c % kActBlock == 0, codes + row * cols + c, scales + row * blocks + c / kActBlock);
    }
  }
}
template <typename T>
__global__ __launch_bounds__(256) void restore_wide(const uint8_t* __restrict__ codes,
                                                    const uint8_t* __restrict__ scales, T* __restrict__ x, int64_t rows,
                                                    int cols) {
  const int blocks = (cols + kActBlock - 1) / kActBlock;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    for (int c = threadIdx.x; c < cols; c += 256) {
      KeptPiece<T, true, 1> k;
      float v;
      k.load(codes, scales, row, c, cols, blocks);
      k.values(&v);
      x[row * cols + c] = (T)v;
    }
  }
}

bool piecewise(const void* x, const void* codes, int cols) {
  return cols % kActBlock == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 8 == 0;
}

template <typename T>
void quantize_typed(const T* x, uint8_t* codes, uint8_t* scales, int64_t rows, int cols, hipStream_t st) {
  constexpr int VE = 16 / sizeof(T);
  if (piecewise(x, codes, cols)) {
    const int64_t pieces = rows * (cols / VE), per = 256 * kActUnroll;
    const dim3 grid((unsigned)std::min<int64_t>((pieces + per - 1) / per, (int64_t)cu_count() * 16));
    quantize_pieces<T, VE><<<grid, 256, 0, st>>>(x, codes, scales, pieces);
    return;
  }
  const dim3 grid((unsigned)std::min<int64_t>((rows + 3) / 4, (int64_t)cu_count() * 32));
  if (cols <= 64) quantize_rows<T, 1><<<grid, 256, 0, st>>>(x, codes, scales, rows, cols);
  else if (cols <= 128) quantize_rows<T, 2><<<grid, 256, 0, st>>>(x, codes, scales, rows, cols);
  else if (cols <= 256) quantize_rows<T, 4><<<grid, 256, 0, st>>>(x, codes, scales, rows, cols);
  else if (cols <= 512) quantize_rows<T, 8><<<grid, 256, 0, st>>>(x, codes, scales, rows, cols);
  else if (cols <= 1024) quantize_rows<T, 16><<<grid, 256, 0, st>>>(x, codes, scales, rows, cols);
  else quantize_wide<T><<<dim3((unsigned)std::min<int64_t>(rows, (int64_t)cu_count() * 8)), 256, 0, st>>>(x, codes, scales, rows, cols);
}

template <typename T>
void restore_typed(const uint8_t* codes, const uint8_t* scales, T* x, int64_t rows, int cols, hipStream_t st) {
  constexpr int VE = 16 / sizeof(T);
  if (piecewise(x, codes, cols)) {
    const int64_t pieces = rows * (cols / VE), per = 256 * kActUnroll;
    const dim3 grid((unsigned)std::min<int64_t>((pieces + per - 1) / per, (int64_t)cu_count() * 16));
    restore_pieces<T, VE><<<grid, 256, 0, st>>>(codes, scales, x, pieces);
    return;
  }
  const dim3 grid((unsigned)std::min<int64_t>((rows + 3) / 4, (int64_t)cu_count() * 32));
  if (cols <= 64) restore_rows<T, 1><<<grid, 256, 0, st>>>(codes, scales, x, rows, cols);
  else if (cols <= 128) restore_rows<T, 2><<<grid, 256, 0, st>>>(codes, scales, x, rows, cols);
  else if (cols <= 256) restore_rows<T, 4><<<grid, 256, 0, st>>>(codes, scales, x, rows, cols);
  else if (cols <= 512) restore_rows<T, 8><<<grid, 256, 0, st>>>(codes, scales, x, rows, cols);
  else if (cols <= 1024) restore_rows<T, 16><<<grid, 256, 0, st>>>(codes, scales, x, rows, cols);
  else restore_wide<T><<<dim3((unsigned)std::min<int64_t>(rows, (int64_t)cu_count() * 8)), 256, 0, st>>>(codes, scales, x, rows, cols);
}

}  // namespace

void launch_quantize(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int cols, int dtype,
                     hipStream_t stream) {
  if (dtype == 0)
    quantize_typed(static_cast<const bf16*>(x), codes, scales, rows, cols, stream);
  else
    quantize_typed(static_cast<const float*>(x), codes, scales, rows, cols, stream);
}

void launch_restore(const uint8_t* codes, const uint8_t* scales, void* x, int64_t rows, int cols, int dtype,
                    hipStream_t stream) {
  if (dtype == 0)
    restore_typed(codes, scales, static_cast<bf16*>(x), rows, cols, stream);
  else
    restore_typed(codes, scales, static_cast<float*>(x), rows, cols, stream);
}

}  // namespace ffk
