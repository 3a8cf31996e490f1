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

// Any width and alignment: a half wave a block. grid-strided over blocks (row, block of the row), walked by
// adding the stride's two digits; block 256 (8 blocks at once).
struct BlockAt {
  int64_t row;
  int blk;
};
__device__ __forceinline__ BlockAt block_at(int64_t i, int blocks) {
  return {i / blocks, (int)(i % blocks)};
}
__device__ __forceinline__ BlockAt block_add(BlockAt t, const BlockAt& step, int blocks) {
  t.blk += step.blk;
  const int carry = t.blk >= blocks ? 1 : 0;
  t.blk -= carry * blocks;
  t.row += step.row + carry;
  return t;
}

template <typename T>
__global__ __launch_bounds__(256) void quantize_blocks(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                       uint8_t* __restrict__ scales, int64_t rows, int cols) {
  const int blocks = (cols + kActBlock - 1) / kActBlock, sub = threadIdx.x & 31, lead = threadIdx.x >> 5;
  const BlockAt step = block_at((int64_t)gridDim.x * 8, blocks);
  BlockAt at[kActUnroll];
  at[0] = block_at((int64_t)blockIdx.x * 8 * kActUnroll + lead, blocks);
  const BlockAt eight = block_at(8, blocks);
#pragma unroll
  for (int u = 1; u < kActUnroll; ++u) at[u] = block_add(at[u - 1], eight, blocks);
  // at[0] of the wave's first half is its least block: the loop ends for the whole wave when that is past
  // the last row (the halves differ by one block, so both are asked)
  while (__ballot(at[0].row < rows) != 0) {
    float v[kActUnroll];
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int c = at[u].blk * kActBlock + sub;
      v[u] = at[u].row < rows && c < cols ? (float)x[at[u].row * cols + c] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int c = at[u].blk * kActBlock + sub;
      act_store<1>(&v[u], at[u].row < rows && c < cols, sub == 0, codes + at[u].row * cols + c,
                   scales + at[u].row * blocks + at[u].blk);
#pragma unroll
      for (int k = 0; k < kActUnroll; ++k) at[u] = block_add(at[u], step, blocks);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void restore_blocks(const uint8_t* __restrict__ codes,
                                                      const uint8_t* __restrict__ scales, T* __restrict__ x,
                                                      int64_t rows, int cols) {
  const int blocks = (cols + kActBlock - 1) / kActBlock, sub = threadIdx.x & 31, lead = threadIdx.x >> 5;
  const BlockAt step = block_at((int64_t)gridDim.x * 8, blocks);
  for (BlockAt at = block_at((int64_t)blockIdx.x * 8 + lead, blocks); at.row < rows; at = block_add(at, step, blocks)) {
    const int c = at.blk * kActBlock + sub;
    if (c < cols) {
      KeptPiece<T, true, 1> k;
      float v;
      k.load(codes, scales, at.row, c, cols, blocks);
      k.values(&v);
      x[at.row * cols + c] = (T)v;
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
  const int64_t all = rows * ((cols + kActBlock - 1) / kActBlock), per = 8 * kActUnroll;
  const dim3 grid((unsigned)std::min<int64_t>((all + per - 1) / per, (int64_t)cu_count() * 32));
  quantize_blocks<T><<<grid, 256, 0, st>>>(x, codes, scales, rows, cols);
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
  const int64_t all = rows * ((cols + kActBlock - 1) / kActBlock);
  const dim3 grid((unsigned)std::min<int64_t>((all + 7) / 8, (int64_t)cu_count() * 32));
  restore_blocks<T><<<grid, 256, 0, st>>>(codes, scales, x, rows, cols);
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
