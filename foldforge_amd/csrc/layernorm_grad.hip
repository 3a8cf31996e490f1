// LayerNorm for training on gfx950: the backward pass with the affine's gradients, and the forward pass
// that keeps its input as an 8-bit activation.
//
//   xh = (x - mean) rstd,  g = dy w,
//   dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy,
// at the kept x: the input itself or what its 8-bit activation stands for; the statistics are taken from
// it again (two passes over registers), so nothing else is kept between the passes. HBM-bound: x (or its
// 33 / 32 bytes a value), dy and dx once each.
//
// A row is held by L lanes, P pieces each, as in the forward kernel: 16-byte pieces where the width is
// one of the stacks' (64 to 768 channels, and 1536 in bf16) and the tensors are aligned, single values (L = 64) for
// any other width up to 1024. A workgroup walks over rows and fetches the next ones while it works on the current
// ones; every lane keeps the sums of dw and db of its channels in registers over all its rows, the
// workgroup joins them in LDS at the end and writes one row of partial sums, and a second kernel adds those
// in a fixed order (the same result on every run). One workgroup writes the gradients itself. Wider rows
// take one workgroup a row, then columns.
#include <algorithm>

#include "ffk_activation.h"
#include "ffk_device.h"
#include "ffk_kernels.h"

namespace ffk {

namespace {

template <typename T>
__device__ __forceinline__ void store_grad(void* p, int64_t i, int dtype, T v) {
  if (dtype == 0)
    static_cast<bf16*>(p)[i] = (bf16)v;
  else
    static_cast<float*>(p)[i] = (float)v;
}

constexpr int rows_per_lane(int VE, int P) { return (VE > 1 && P == 1) || P <= 2 ? 2 : 1; }

// grid: persistent workgroups, each of 256 / L * R rows a step; block 256. cols == L P VE where VE > 1,
// cols <= L P where VE == 1. dw / db null: not wanted (both then). part: [gridDim.x][2][cols].
// 262144 rows of 128 bf16: 35 us from the input (5.7 TB/s), 32 from 8 bits (5.3); 40009 fp32 rows of 451: 38 (5.6).
template <typename T, bool CODES, int VE, int L, int P>
__global__ __launch_bounds__(256) void layer_norm_grad(const LayerNormGradArgs a) {
  using Kept = KeptPiece<T, CODES, VE>;
  using Grad = KeptPiece<T, false, VE>;
  constexpr int N = P * VE, G = 256 / L, R = rows_per_lane(VE, P);
  constexpr bool FULL = VE > 1;
  __shared__ float red[G * L * N];
  const int sub = threadIdx.x % L, lead = threadIdx.x / L;
  const int cols = FULL ? L * N : a.cols, blocks = (cols + kActBlock - 1) / kActBlock;
  const float inv = 1.f / (float)cols;
  struct Rows {
    Kept x[R][P];
    Grad dy[R][P];
  };
  auto channel = [&](int p) __attribute__((always_inline)) { return VE * (sub + L * p); };
  auto load = [&](Rows& v, int64_t row0) __attribute__((always_inline)) {
#pragma unroll
    for (int it = 0; it < R; ++it) {
      const int64_t row = row0 + G * it;
      if (row < a.rows) {
#pragma unroll
        for (int p = 0; p < P; ++p)
          if (FULL || channel(p) < cols) {
            v.x[it][p].load(a.x, a.scales, row, channel(p), cols, blocks);
            v.dy[it][p].load(a.dy, nullptr, row, channel(p), cols, blocks);
          }
      }
    }
  };
  float wv[N], dw[N], db[N];
#pragma unroll
  for (int i = 0; i < N; ++i) dw[i] = db[i] = 0.f;
  auto compute = [&](const Rows& v, int64_t row0) __attribute__((always_inline)) {
#pragma unroll
    for (int it = 0; it < R; ++it) {
      const int64_t row = row0 + G * it;
      const bool real = row < a.rows;
      float x[N], dy[N];
      float s = 0.f, sg = 0.f;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        v.x[it][p].values(x + VE * p);
        v.dy[it][p].values(dy + VE * p);
#pragma unroll
        for (int e = VE * p; e < VE * p + VE; ++e) {
          const bool in = real && (FULL || channel(p) < cols);
          x[e] = in ? x[e] : 0.f;
          dy[e] = in ? dy[e] : 0.f;
          s += x[e];
          sg += dy[e] * wv[e];
        }
      }
      const float mean = lanes_sum<L>(s) * inv;
      const float c1 = lanes_sum<L>(sg) * inv;
      float q = 0.f, sx = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x[i] = FULL || channel(i / VE) < cols ? x[i] - mean : 0.f;
        q += x[i] * x[i];
        // the mean of g is taken out first: what is left pairs with x - mean exactly, and large means of
        // either lose nothing
        sx += (dy[i] * wv[i] - c1) * x[i];
      }
      const float var = lanes_sum<L>(q) * inv + a.eps;
      // one hardware reciprocal square root (1 ulp) where dx is rounded to bf16
      // (0 for a row past the end: with eps = 0 its deviation would be 0, and 0 / 0 would reach the sums)
      const float rstd = !real ? 0.f : sizeof(T) == 2 ? __builtin_amdgcn_rsqf(var) : 1.f / sqrtf(var);
      const float c2 = lanes_sum<L>(sx) * inv * rstd * rstd;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        Grad o;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const int i = VE * p + e;
          const float d = rstd * (dy[i] * wv[i] - c1 - x[i] * c2);
          dw[i] += dy[i] * (x[i] * rstd);
          db[i] += dy[i];
          if constexpr (VE > 1)
            o.v[e] = (T)d;
          else
            o.v = (T)d;
        }
        if (real && (FULL || channel(p) < cols)) {
          T* to = static_cast<T*>(a.dx) + row * cols + channel(p);
          if constexpr (VE > 1)
            __builtin_nontemporal_store(o.v, reinterpret_cast<decltype(o.v)*>(to));
          else
            *to = o.v;
        }
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * G * R;
  int64_t row0 = (int64_t)blockIdx.x * G * R + lead;
  Rows va, vb;
  load(va, row0);
#pragma unroll
  for (int i = 0; i < N; ++i) wv[i] = 1.f;
  if (a.w != nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i) wv[i] = FULL || channel(i / VE) < cols ? a.w[channel(i / VE) + i % VE] : 0.f;
  }
  // row0 - lead is the workgroup's first row: the loop condition is uniform
  while (row0 - lead < a.rows) {
    load(vb, row0 + step);
    compute(va, row0);
    row0 += step;
    if (row0 - lead >= a.rows) break;
    load(va, row0 + step);
    compute(vb, row0);
    row0 += step;
  }
  // the workgroup's sums: lane group by lane group through LDS
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (which) __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) red[lead * (L * N) + channel(i / VE) + i % VE] = which ? db[i] : dw[i];
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += 256) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < G; ++k) t += red[k * (L * N) + c];
      if (gridDim.x > 1)
        a.part[((int64_t)blockIdx.x * 2 + which) * cols + c] = t;
      else if (void* to = which ? a.db : a.dw)
        store_grad(to, c, a.grad_dtype, t);
    }
  }
}

// Wide rows. One workgroup a row (grid-strided): dx and the row's mean and rstd. block 256.
template <typename T, bool CODES>
__global__ __launch_bounds__(256) void layer_norm_grad_wide(const LayerNormGradArgs a, float* stats) {
  __shared__ float red[2][4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int blocks = (a.cols + kActBlock - 1) / kActBlock;
  const float inv = 1.f / (float)a.cols;
  auto total = [&](float& u, float& v) __attribute__((always_inline)) {
    u = wave_sum(u);
    v = wave_sum(v);
    __syncthreads();  // the last sums have been read
    if (lane == 0) {
      red[0][wave] = u;
      red[1][wave] = v;
    }
    __syncthreads();
    u = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
    v = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  };
  const T* dy = static_cast<const T*>(a.dy);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    auto x_at = [&](int c) __attribute__((always_inline)) {
      KeptPiece<T, CODES, 1> k;
      float v;
      k.load(a.x, a.scales, row, c, a.cols, blocks);
      k.values(&v);
      return v;
    };
    auto g_at = [&](int c) __attribute__((always_inline)) {
      return (float)dy[row * a.cols + c] * (a.w ? a.w[c] : 1.f);
    };
    float s = 0.f, sg = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
      s += x_at(c);
      sg += g_at(c);
    }
    total(s, sg);
    const float mean = s * inv, c1 = sg * inv;
    float q = 0.f, sx = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
      const float d = x_at(c) - mean;
      q += d * d;
      sx += (g_at(c) - c1) * d;
    }
    total(q, sx);
    const float rstd = 1.f / sqrtf(q * inv + a.eps), c2 = sx * inv * rstd * rstd;
    for (int c = threadIdx.x; c < a.cols; c += 256)
      static_cast<T*>(a.dx)[row * a.cols + c] = (T)(rstd * (g_at(c) - c1 - (x_at(c) - mean) * c2));
    if (threadIdx.x == 0) {
      stats[2 * row] = mean;
      stats[2 * row + 1] = rstd;
    }
  }
}

// The affine's partial sums from the wide rows' statistics: 64 channels and a share of the rows a workgroup.
// grid (ceil(cols / 64), shares); block 256 (64 channels x 4 rows). part: [shares][2][cols].
template <typename T, bool CODES>
__global__ __launch_bounds__(256) void layer_norm_grad_columns(const LayerNormGradArgs a, const float* stats) {
  __shared__ float red[2][256];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), blocks = (a.cols + kActBlock - 1) / kActBlock;
  float dw = 0.f, db = 0.f;
  if (c < a.cols) {
    for (int64_t row = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6); row < a.rows; row += (int64_t)gridDim.y * 4) {
      KeptPiece<T, CODES, 1> k;
      float x;
      k.load(a.x, a.scales, row, c, a.cols, blocks);
      k.values(&x);
      const float dy = (float)static_cast<const T*>(a.dy)[row * a.cols + c];
      dw += dy * ((x - stats[2 * row]) * stats[2 * row + 1]);
      db += dy;
    }
  }
  red[0][threadIdx.x] = dw;
  red[1][threadIdx.x] = db;
  __syncthreads();
  if (threadIdx.x < 64 && c < a.cols) {
    for (int which = 0; which < 2; ++which) {
      const float* r = red[which] + threadIdx.x;
      a.part[((int64_t)blockIdx.y * 2 + which) * a.cols + c] = (r[0] + r[64]) + (r[128] + r[192]);
    }
  }
}

// out[c] = sum over k < count of part[k][c], c < width: 32 columns x 32 rows a workgroup, each thread's rows
// in order, then the 32 row sums in order. The first `split` columns go to out0, the rest to out1 (either may
// be null). grid ceil(width / 32); block 1024.
__global__ __launch_bounds__(1024) void sum_partials(const float* __restrict__ part, int count, int width, int split,
                                                     void* out0, void* out1, int dtype) {
  __shared__ float red[32][33];
  const int tc = threadIdx.x & 31, tr = threadIdx.x >> 5, c = blockIdx.x * 32 + tc;
  float s = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int k = tr; k < count; k += 32) s += part[(int64_t)k * width + c];
  }
  red[tr][tc] = s;
  __syncthreads();
  if (threadIdx.x < 32 && c < width) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += red[k][tc];
    void* out = c < split ? out0 : out1;
    if (out) store_grad(out, c < split ? c : c - split, dtype, t);
  }
}

// LayerNorm and the 8-bit activation of its input in one pass. As layer_norm_vec (VE > 1: cols = L P VE) or
// any width up to L P (VE = 1). block 256. 262144 rows of 128 bf16: 25 us, 6.6 TB/s (the norm and the activation on
// their own 20 each).
template <typename T, int VE, int L, int P>
__global__ __launch_bounds__(256) void layer_norm_keep(const T* __restrict__ x, const float* __restrict__ w,
                                                       const float* __restrict__ b, T* __restrict__ y,
                                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                       int64_t rows, int cols_, float eps) {
  using V = KeptPiece<T, false, VE>;
  constexpr int N = P * VE, G = 256 / L, R = rows_per_lane(VE, P);
  constexpr bool FULL = VE > 1;
  const int sub = threadIdx.x % L, lead = threadIdx.x / L;
  const int cols = FULL ? L * N : cols_, blocks = (cols + kActBlock - 1) / kActBlock;
  const float inv = 1.f / (float)cols;
  auto channel = [&](int p) __attribute__((always_inline)) { return VE * (sub + L * p); };
  auto load = [&](V (&v)[R][P], int64_t row0) __attribute__((always_inline)) {
#pragma unroll
    for (int it = 0; it < R; ++it) {
      const int64_t row = row0 + G * it;
      if (row < rows) {
#pragma unroll
        for (int p = 0; p < P; ++p)
          if (FULL || channel(p) < cols) v[it][p].load(x, nullptr, row, channel(p), cols, blocks);
      }
    }
  };
  float wv[N], bv[N];
  auto compute = [&](const V (&v)[R][P], int64_t row0) __attribute__((always_inline)) {
#pragma unroll
    for (int it = 0; it < R; ++it) {
      const int64_t row = row0 + G * it;
      float xv[N];
      float s = 0.f;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const bool in = row < rows && (FULL || channel(p) < cols);
        v[it][p].values(xv + VE * p);
#pragma unroll
        for (int e = VE * p; e < VE * p + VE; ++e) {
          xv[e] = in ? xv[e] : 0.f;
          s += xv[e];
        }
        const int64_t at = row * cols + channel(p);
        act_store<VE>(xv + VE * p, in, channel(p) % kActBlock == 0, codes + at,
                      scales + row * blocks + channel(p) / kActBlock);
      }
      const float mean = lanes_sum<L>(s) * inv;
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        xv[i] = FULL || channel(i / VE) < cols ? xv[i] - mean : 0.f;
        q += xv[i] * xv[i];
      }
      const float var = lanes_sum<L>(q) * inv + eps;
      const float rstd = sizeof(T) == 2 ? __builtin_amdgcn_rsqf(var) : 1.f / sqrtf(var);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (row < rows && (FULL || channel(p) < cols)) {
          V o;
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const T r = (T)(xv[VE * p + e] * rstd * wv[VE * p + e] + bv[VE * p + e]);
            if constexpr (VE > 1)
              o.v[e] = r;
            else
              o.v = r;
          }
          T* to = y + row * cols + channel(p);
          if constexpr (VE > 1)
            __builtin_nontemporal_store(o.v, reinterpret_cast<decltype(o.v)*>(to));
          else
            *to = o.v;
        }
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * G * R;
  int64_t row0 = (int64_t)blockIdx.x * G * R + lead;
  V va[R][P], vb[R][P];
  load(va, row0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    wv[i] = 1.f;
    bv[i] = 0.f;
  }
  if (w != nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i) wv[i] = FULL || channel(i / VE) < cols ? w[channel(i / VE) + i % VE] : 0.f;
  }
  if (b != nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i) bv[i] = FULL || channel(i / VE) < cols ? b[channel(i / VE) + i % VE] : 0.f;
  }
  while (row0 - lead < rows) {
    load(vb, row0 + step);
    compute(va, row0);
    row0 += step;
    if (row0 - lead >= rows) break;
    load(va, row0 + step);
    compute(vb, row0);
    row0 += step;
  }
}

// How a call's rows are laid over lanes: 16-byte pieces where the width splits evenly and every tensor is
// aligned, else single values of up to 1024 channels; other rows lie in no wave's registers.
enum RowForm { kFormWide, kForm8x1, kForm16x1, kForm32x1, kForm16x3, kForm64x1, kForm32x3, kForm64x3,
               kFormOne1, kFormOne2, kFormOne4, kFormOne8, kFormOne16 };

RowForm row_form(int cols, int pieces_of, bool aligned) {
  if (aligned && cols % pieces_of == 0) {
    switch (cols / pieces_of) {
      case 8: return kForm8x1;
      case 16: return kForm16x1;
      case 32: return kForm32x1;
      case 48: return kForm16x3;
      case 64: return kForm64x1;
      case 96: return kForm32x3;
      case 192: return kForm64x3;
      default: break;
    }
  }
  return cols <= 64 ? kFormOne1 : cols <= 128 ? kFormOne2 : cols <= 256 ? kFormOne4 : cols <= 512 ? kFormOne8
         : cols <= 1024 ? kFormOne16 : kFormWide;
}

// Rows a workgroup takes at once, per form.
int form_rows(RowForm f) {
  switch (f) {
    case kForm8x1: return 64;
    case kForm16x1: return 32;
    case kForm32x1: return 16;
    case kForm64x1: return 8;
    case kForm16x3: return 16;
    case kForm32x3: return 8;
    case kForm64x3: return 4;
    case kFormOne1: case kFormOne2: return 8;
    default: return 4;
  }
}

constexpr int kGradBlocksPerCu = 4;  // 256-thread workgroups of the backward kernel a CU is given

// Rows of partial sums a call needs.
int64_t grad_blocks(int64_t rows, RowForm f) {
  if (f == kFormWide) return std::min<int64_t>((rows + 3) / 4, 64);
  return std::min<int64_t>((rows + form_rows(f) - 1) / form_rows(f), (int64_t)cu_count() * kGradBlocksPerCu);
}

template <typename T, bool CODES>
void grad_typed(const LayerNormGradArgs& a, RowForm f, int64_t blocks, float* stats, hipStream_t st) {
  constexpr int VE = 16 / sizeof(T);
  const dim3 grid((unsigned)blocks);
  switch (f) {
    case kForm8x1: layer_norm_grad<T, CODES, VE, 8, 1><<<grid, 256, 0, st>>>(a); break;
    case kForm16x1: layer_norm_grad<T, CODES, VE, 16, 1><<<grid, 256, 0, st>>>(a); break;
    case kForm32x1: layer_norm_grad<T, CODES, VE, 32, 1><<<grid, 256, 0, st>>>(a); break;
    case kForm64x1: layer_norm_grad<T, CODES, VE, 64, 1><<<grid, 256, 0, st>>>(a); break;
    case kForm16x3: layer_norm_grad<T, CODES, VE, 16, 3><<<grid, 256, 0, st>>>(a); break;
    case kForm32x3: layer_norm_grad<T, CODES, VE, 32, 3><<<grid, 256, 0, st>>>(a); break;
    case kForm64x3: layer_norm_grad<T, CODES, VE, 64, 3><<<grid, 256, 0, st>>>(a); break;
    case kFormOne1: layer_norm_grad<T, CODES, 1, 64, 1><<<grid, 256, 0, st>>>(a); break;
    case kFormOne2: layer_norm_grad<T, CODES, 1, 64, 2><<<grid, 256, 0, st>>>(a); break;
    case kFormOne4: layer_norm_grad<T, CODES, 1, 64, 4><<<grid, 256, 0, st>>>(a); break;
    case kFormOne8: layer_norm_grad<T, CODES, 1, 64, 8><<<grid, 256, 0, st>>>(a); break;
    case kFormOne16: layer_norm_grad<T, CODES, 1, 64, 16><<<grid, 256, 0, st>>>(a); break;
    case kFormWide: {
      const unsigned rows_grid = (unsigned)std::min<int64_t>(a.rows, (int64_t)cu_count() * 8);
      layer_norm_grad_wide<T, CODES><<<rows_grid, 256, 0, st>>>(a, stats);
      layer_norm_grad_columns<T, CODES><<<dim3((unsigned)((a.cols + 63) / 64), (unsigned)blocks), 256, 0, st>>>(a, stats);
      break;
    }
  }
}

bool aligned_to(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T>
void keep_typed(const T* x, const float* w, const float* b, T* y, uint8_t* codes, uint8_t* scales, int64_t rows,
                int cols, float eps, RowForm f, hipStream_t st) {
  constexpr int VE = 16 / sizeof(T);
  const dim3 grid((unsigned)std::min<int64_t>((rows + form_rows(f) - 1) / form_rows(f), (int64_t)cu_count() * 32));
#define FFK_KEEP(VE_, L_, P_) \
  layer_norm_keep<T, VE_, L_, P_><<<grid, 256, 0, st>>>(x, w, b, y, codes, scales, rows, cols, eps)
  switch (f) {
    case kForm8x1: FFK_KEEP(VE, 8, 1); break;
    case kForm16x1: FFK_KEEP(VE, 16, 1); break;
    case kForm32x1: FFK_KEEP(VE, 32, 1); break;
    case kForm64x1: FFK_KEEP(VE, 64, 1); break;
    case kForm16x3: FFK_KEEP(VE, 16, 3); break;
    case kForm32x3: FFK_KEEP(VE, 32, 3); break;
    case kForm64x3: FFK_KEEP(VE, 64, 3); break;
    case kFormOne1: FFK_KEEP(1, 64, 1); break;
    case kFormOne2: FFK_KEEP(1, 64, 2); break;
    case kFormOne4: FFK_KEEP(1, 64, 4); break;
    case kFormOne8: FFK_KEEP(1, 64, 8); break;
    case kFormOne16: FFK_KEEP(1, 64, 16); break;
    case kFormWide: break;  // launch_layer_norm_keep runs the two parts
  }
#undef FFK_KEEP
}

// x: the kept tensor or its codes; row_form's answer depends on the tensors' alignment as well.
RowForm grad_form(const LayerNormGradArgs& a) {
  const bool aligned = aligned_to(a.x, a.scales ? 8 : 16) && aligned_to(a.dy, 16) && aligned_to(a.dx, 16);
  return row_form(a.cols, a.dtype == 0 ? 8 : 4, aligned);
}

}  // namespace

// The workspace holds the partial sums of whichever form the call takes (types and alignment are not known here): rows in
// registers make at most a workgroup for every 4 rows (form_rows), one alone needs none, and the wide rows' statistics come
// behind their sums. Beyond 1024 channels a width may still be one of the 16-byte pieces' (bf16 rows of 1536).
size_t layer_norm_grad_floats(int64_t rows, int cols) {
  const int64_t parts = std::min<int64_t>((rows + 3) / 4, (int64_t)cu_count() * kGradBlocksPerCu);
  const size_t held = parts <= 1 ? 0 : (size_t)parts * 2 * cols;
  if (cols <= 1024) return held;
  const size_t wide = (size_t)64 * 2 * cols + 2 * (size_t)rows;
  const bool pieces = row_form(cols, 8, true) != kFormWide || row_form(cols, 4, true) != kFormWide;
  return pieces ? std::max(held, wide) : wide;
}

void launch_sum_partials(const float* part, int count, int width, int split, void* out0, void* out1, int dtype,
                         hipStream_t stream) {
  sum_partials<<<dim3((unsigned)((width + 31) / 32)), 1024, 0, stream>>>(part, count, width, split, out0, out1, dtype);
}

void launch_layer_norm_grad(const LayerNormGradArgs& a, hipStream_t stream) {
  const RowForm f = grad_form(a);
  const int64_t blocks = grad_blocks(a.rows, f);
  float* stats = a.part + (size_t)64 * 2 * a.cols;
  if (a.dtype == 0 && a.scales) grad_typed<bf16, true>(a, f, blocks, stats, stream);
  else if (a.dtype == 0) grad_typed<bf16, false>(a, f, blocks, stats, stream);
  else if (a.scales) grad_typed<float, true>(a, f, blocks, stats, stream);
  else grad_typed<float, false>(a, f, blocks, stats, stream);
  if ((blocks > 1 || f == kFormWide) && (a.dw || a.db))
    launch_sum_partials(a.part, (int)blocks, 2 * a.cols, a.cols, a.dw, a.db, a.grad_dtype, stream);
}

void launch_layer_norm_keep(const void* x, const float* w, const float* b, void* y, uint8_t* codes, uint8_t* scales,
                            int64_t rows, int cols, float eps, int dtype, hipStream_t stream) {
  const bool aligned = aligned_to(x, 16) && aligned_to(y, 16) && aligned_to(codes, 8);
  const RowForm f = row_form(cols, dtype == 0 ? 8 : 4, aligned);
  if (f == kFormWide) {
    // (x is read twice; y may not be x: the activation is taken after the norm)
    launch_layer_norm(x, w, b, y, rows, cols, eps, dtype, stream);
    launch_quantize(x, codes, scales, rows, cols, dtype, stream);
  } else if (dtype == 0) {
    keep_typed(static_cast<const bf16*>(x), w, b, static_cast<bf16*>(y), codes, scales, rows, cols, eps, f, stream);
  } else {
    keep_typed(static_cast<const float*>(x), w, b, static_cast<float*>(y), codes, scales, rows, cols, eps, f, stream);
  }
}

}  // namespace ffk
