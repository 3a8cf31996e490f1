// Dropout whose mask is drawn where it is needed, with the residual add:
//   y = residual + (kept ? update / (1 - p) : 0)
// The mask of a tensor [outer][shared][inner] is [outer][inner], the same for all `shared` (AF3's row-wise and column-wise
// dropout of a pair tensor; shared = 1: every value its own). Its number m is a 16-bit draw of Philox4x32-10 (Salmon et al.,
// "Parallel random numbers: as easy as 1, 2, 3", 2011): block m / 8 is the counter's low 64 bits, the call's offset the high
// ones, the seed the key; of the block's four words each gives two numbers, the low half first. Number m is dropped where
// it is below t = 65536 p (whole), and the kept values are scaled by 65536 / (65536 - t), so the expectation is exact at
// the rate t / 65536 that is drawn. 16 bits a value rather than 32: ten rounds are 20 quarter-rate multiplications, which at
// four values a block cost as much time as the six bytes a bf16 value moves. Nothing is stored, the backward pass draws
// again. A dropped value is not read into the result: infinities and NaN behind the mask stay there.
// Bound by bytes: 512 x 512 x 128 bf16 with the residual and one mask for all rows 42.8 us (4.7 TB/s), 40009 x 451 fp32 forward and
// backward 69 us (5.2 TB/s).
#include <algorithm>

#include "ffk_device.h"
#include "ffk_kernels.h"

namespace ffk {

namespace {

struct Draw {
  uint32_t k0, k1, c2, c3, threshold;
};

// The call's draw, with the seed and the offset's base from device memory where they are kept there (a captured call then
// draws anew at each replay).
__device__ __forceinline__ Draw draw_of(const DropoutArgs& a) {
  uint64_t seed = a.seed, offset = a.offset;
  if (a.state) {
    seed = (uint64_t)a.state[0];
    offset += (uint64_t)a.state[1];
  }
  return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset, (uint32_t)(offset >> 32), (uint32_t)a.threshold};
}

// Bit e: whether number 8 block + e is kept.
__device__ __forceinline__ uint32_t keep8(const Draw& d, uint64_t block) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = d.c2, c3 = d.c3, k0 = d.k0, k1 = d.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(q >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)q;
    c2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const uint32_t w[4] = {c0, c1, c2, c3};
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bits |= ((w[i] & 0xffffu) >= d.threshold ? 1u : 0u) << (2 * i);
    bits |= ((w[i] >> 16) >= d.threshold ? 1u : 0u) << (2 * i + 1);
  }
  return bits;
}

// Eight values of a row; WIDE: 16-byte aligned. (Global memory takes wide accesses at any alignment of the type's own.)
template <typename T, bool WIDE>
struct Eight {
  typedef T vec __attribute__((__vector_size__(8 * sizeof(T)), aligned(WIDE ? 16 : sizeof(T))));
  T v[8];
  __device__ __forceinline__ void load(const T* p, int n) {
    if (WIDE || n == 8) {
      const vec t = *reinterpret_cast<const vec*>(p);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = t[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : (T)0.f;
    }
  }
  __device__ __forceinline__ void store(T* p, int n) const {
    if (WIDE || n == 8) {
      vec t;
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = v[e];
      *reinterpret_cast<vec*>(p) = t;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) p[e] = v[e];
    }
  }
};

template <typename T, bool RES, bool WIDE>
__device__ __forceinline__ void drop8(Eight<T, WIDE>& x, const Eight<T, WIDE>& r, uint32_t bits, float scale) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float kept = (bits >> e) & 1u ? (float)x.v[e] * scale : 0.f;
    x.v[e] = (T)(RES ? (float)r.v[e] + kept : kept);
  }
}

// shared = 1: the tensor is one run of n values, a thread takes a block of the generator (8 values) at a time. block 256.
// WIDE: n a multiple of 8, pointers 16-byte aligned.
template <typename T, bool RES, bool WIDE>
__global__ __launch_bounds__(256) void dropout_each(const DropoutArgs a) {
  const Draw d = draw_of(a);
  const int64_t n = a.inner, blocks = (n + 7) / 8;
  for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < blocks; b += (int64_t)gridDim.x * 256) {
    const int count = n - 8 * b < 8 ? (int)(n - 8 * b) : 8;
    Eight<T, WIDE> x, r;
    x.load(static_cast<const T*>(a.x) + 8 * b, count);
    if constexpr (RES) r.load(static_cast<const T*>(a.residual) + 8 * b, count);
    drop8<T, RES, WIDE>(x, r, keep8(d, (uint64_t)b), a.scale);
    x.store(static_cast<T*>(a.y) + 8 * b, count);
  }
}

constexpr int kDropRows = 4;  // rows a thread has in flight

// shared > 1: a thread draws its eight numbers once and takes them down `rows` rows. A workgroup: `lanes` threads along the
// inner axis, 256 / lanes beside each other along the shared one. It walks over the outer x ceil(pieces / lanes) x
// ceil(shared / rows) pieces of work.
template <typename T, bool RES, bool WIDE>
__global__ __launch_bounds__(256) void dropout_shared(const DropoutArgs a, int lanes, int64_t tiles, int64_t chunks,
                                                      int64_t rows) {
  const Draw d = draw_of(a);
  const int step = 256 / lanes;
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  for (int64_t w = blockIdx.x; w < a.outer * tiles * chunks; w += gridDim.x) {
    // (neighbours beside each other in memory)
    const int64_t tile = w % tiles, chunk = w / tiles % chunks, o = w / tiles / chunks;
    const int64_t i = 8 * (tile * lanes + (threadIdx.x & (lanes - 1)));
    if (i >= a.inner) continue;
    const int count = a.inner - i < 8 ? (int)(a.inner - i) : 8;
    // eight numbers from o * inner + i on: of one block, or of two
    const uint64_t m = (uint64_t)(o * a.inner + i);
    uint32_t bits = keep8(d, m >> 3);
    if (!WIDE && (m & 7u)) bits = (bits | keep8(d, (m >> 3) + 1) << 8) >> (m & 7u);
    const int64_t end = (chunk + 1) * rows < a.shared ? (chunk + 1) * rows : a.shared;
    for (int64_t s = chunk * rows + threadIdx.x / lanes; s < end; s += kDropRows * step) {
      Eight<T, WIDE> v[kDropRows], r[kDropRows];
#pragma unroll
      for (int u = 0; u < kDropRows; ++u)
        if (s + u * step < end) {
          const int64_t at = (o * a.shared + s + u * step) * a.inner + i;
          v[u].load(x + at, count);
          if constexpr (RES) r[u].load(res + at, count);
        }
#pragma unroll
      for (int u = 0; u < kDropRows; ++u)
        if (s + u * step < end) {
          drop8<T, RES, WIDE>(v[u], r[u], bits, a.scale);
          v[u].store(static_cast<T*>(a.y) + (o * a.shared + s + u * step) * a.inner + i, count);
        }
    }
  }
}

template <typename T, bool RES, bool WIDE>
void launch(const DropoutArgs& a, hipStream_t stream) {
  const int64_t pieces = (a.inner + 7) / 8;
  if (a.shared == 1) {  // (one run: outer is 1)
    dropout_each<T, RES, WIDE><<<dim3((unsigned)std::min<int64_t>((pieces + 255) / 256, 256 * 16)), 256, 0, stream>>>(a);
    return;
  }
  int lanes = 1;
  while (lanes < 256 && lanes < pieces) lanes *= 2;
  const int64_t step = 256 / lanes, tiles = (pieces + lanes - 1) / lanes, passes = (a.shared + step - 1) / step;
  // eight workgroups a CU where there is that much work, the shared axis cut no finer than that needs
  const int64_t want = std::max<int64_t>(1, 256 * 8 / (a.outer * tiles));
  const int64_t rows = step * ((passes + std::min(want, passes) - 1) / std::min(want, passes));
  const int64_t chunks = (a.shared + rows - 1) / rows;
  dropout_shared<T, RES, WIDE>
      <<<dim3((unsigned)std::min<int64_t>(a.outer * tiles * chunks, 1 << 20)), 256, 0, stream>>>(a, lanes, tiles, chunks, rows);
}

template <typename T>
void launch_type(const DropoutArgs& a, hipStream_t stream) {
  const bool wide = a.inner % 8 == 0 && ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) |
                                          reinterpret_cast<uintptr_t>(a.residual)) & 15u) == 0;
  if (a.residual)
    wide ? launch<T, true, true>(a, stream) : launch<T, true, false>(a, stream);
  else
    wide ? launch<T, false, true>(a, stream) : launch<T, false, false>(a, stream);
}

}  // namespace

void launch_dropout(const DropoutArgs& a, hipStream_t stream) {
  if (a.dtype == 0)
    launch_type<bf16>(a, stream);
  else
    launch_type<float>(a, stream);
}

}  // namespace ffk
