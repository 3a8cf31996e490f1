// Backward pass of the SwiGLU transition on gfx950.
//
//   n = LN(x), a = n A^T, b = n B^T, u = silu(a) b, y = x + u S^T          (A, B [H][d], S [d][H])
//   du = dy S,  da = du b s(a) (1 + a (1 - s(a))),  db = du silu(a)        (s: the logistic function)
//   dA = da^T n,  dB = db^T n,  dS = dy^T u,  dn = da A + db B,  dx = dy + LN'(dn)
// at the kept x (the input or its 8-bit activation): the hidden rows are computed again, nothing but x is
// kept between the passes. 16 M d H flops for M rows, on bf16 operands with fp32 sums.
//
// The form for every width (d and H multiples of 64), in chunks of rows:
//   norm_rows        n in bf16
//   hidden_grad      a, b and du tile by tile, their elementwise part in registers -> E = [da | db | u]
//   gemm64<false>    dn = [da | db] [A; B], split over the hidden channels where the rows are few
//   norm_grad_rows   dx, and the sums of the affine's gradients
//   gemm64<true>     E^T [n or dy], split over the rows: dA, dB and dS^T
// and at the end the partial sums are added in a fixed order.
#include <algorithm>

#include "ffk_activation.h"
#include "ffk_device.h"
#include "ffk_kernels.h"

namespace ffk {

namespace {

// A tile of 64-channel bf16 rows in LDS (128 bytes a row, 8 pieces of 16): piece p of row r lies at piece
// p ^ swz64(r). Sixteen lanes that read one piece of sixteen consecutive rows (an operand fetch) fall on all
// 64 banks, and eight rows' 64-byte halves (a transposing fetch) on each bank twice, the least for 512 bytes.
__device__ __forceinline__ int swz64(int r) { return ((r >> 1) & 1) << 2 | ((r >> 2) & 1) << 1 | ((r >> 3) & 1); }
__device__ __forceinline__ int off64(int r, int p) { return r * 64 + 8 * (p ^ swz64(r)); }

// This wave's share of a 64 x 64 tile (rows row0 .. row0 + 63 of src, clamped to `last`, channels c0 .. c0 + 63)
// into LDS at byte address dst: 8 rows an instruction. 4 waves.
__device__ __forceinline__ void tile_dma(const bf16* src, int64_t ld, int64_t row0, int64_t last, int c0, uint32_t dst,
                                         int wave, int lane) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r0 = 8 * (2 * wave + u), r = r0 + (lane >> 3);
    const int64_t row = row0 + r < last ? row0 + r : last;
    dma16_at(src + row * ld + c0 + 8 * ((lane & 7) ^ swz64(r)), dst + 128 * r0);
  }
}

typedef short s16x4 __attribute__((__vector_size__(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// MFMA operand of a tile whose rows are k: 32 channels from c0 (a multiple of 32), k0 .. k0 + 15. One
// transposing read gives a lane one channel at four k: sixteen lanes take 4 rows x 16 channels (the lane's
// address: row j / 4, channels 4 (j % 4) ..), lane j of them gets channel j. Lanes of half g hold k0 + 4 g + 0..3
// and k0 + 8 + 4 g + 0..3: every operand read this way pairs the same k.
__device__ __forceinline__ bf16x8 ld_turned(const bf16* tile, int c0, int k0, int lane) {
  const int j = lane & 15, q = lane >> 4;
  const int r = k0 + 4 * (q >> 1) + (j >> 2), c = c0 + 16 * (q & 1) + 4 * (j & 3);
  const bf16* p0 = &tile[off64(r, c >> 3) + (c & 7)];
  const bf16* p1 = &tile[off64(r + 8, c >> 3) + (c & 7)];
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p0));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p1));
  union {
    s16x4 s[2];
    bf16x8 v;
  } o;
  o.s[0] = lo;
  o.s[1] = hi;
  return o.v;
}

// fp32 parameters -> bf16, each in the orders the products read: ab [2 H][d] (A, then B), st [H][d] (S^T),
// abt [d][2 H]. A 32 x 32 tile a workgroup: grid (H / 32, d / 32, 3); block 256.
__global__ __launch_bounds__(256) void pack_grad_weights(const float* __restrict__ wa, const float* __restrict__ wb,
                                                         const float* __restrict__ ws, bf16* __restrict__ ab,
                                                         bf16* __restrict__ st, bf16* __restrict__ abt, int d, int H) {
  __shared__ bf16 tile[32][33];
  const int h0 = blockIdx.x * 32, c0 = blockIdx.y * 32, which = blockIdx.z;
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  if (which < 2) {
    const float* src = which ? wb : wa;
    for (int r = row; r < 32; r += 8) {
      const bf16 v = (bf16)src[(int64_t)(h0 + r) * d + c0 + col];
      ab[(int64_t)(which * H + h0 + r) * d + c0 + col] = v;
      tile[r][col] = v;
    }
    __syncthreads();
    for (int r = row; r < 32; r += 8) abt[(int64_t)(c0 + r) * 2 * H + which * H + h0 + col] = tile[col][r];
  } else {
    for (int r = row; r < 32; r += 8) tile[r][col] = (bf16)ws[(int64_t)(c0 + r) * H + h0 + col];
    __syncthreads();
    for (int r = row; r < 32; r += 8) st[(int64_t)(h0 + r) * d + c0 + col] = tile[col][r];
  }
}

// n = LN(x) in bf16, one wave a row, K = d / 64 channels a lane. grid-strided; block 256.
template <bool CODES, int K>
__global__ __launch_bounds__(256) void norm_rows(const void* x, const uint8_t* scales, const float* __restrict__ w,
                                                 const float* __restrict__ b, bf16* __restrict__ n, int64_t rows,
                                                 float eps) {
  constexpr int d = 64 * K, blocks = d / kActBlock;
  const int lane = threadIdx.x & 63;
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
    float v[K];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      KeptPiece<bf16, CODES, 1> p;
      p.load(x, scales, row, lane + 64 * k, d, blocks);
      p.values(&v[k]);
      s += v[k];
    }
    const float mean = lanes_sum<64>(s) * (1.f / d);
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] -= mean;
      q += v[k] * v[k];
    }
    const float rstd = __builtin_amdgcn_rsqf(lanes_sum<64>(q) * (1.f / d) + eps);
#pragma unroll
    for (int k = 0; k < K; ++k) n[row * d + lane + 64 * k] = (bf16)(v[k] * rstd * w[lane + 64 * k] + b[lane + 64 * k]);
  }
}

// da, db and u of an element from a, b and du.
struct SwigluGrad {
  float da, db, u;
};
__device__ __forceinline__ SwigluGrad swiglu_grad(float a, float b, float du) {
  const float s = sigmoidf_(a), sa = a * s;
  return {du * b * (s + sa * (1.f - s)), du * sa, sa * b};
}

// E [rows][3 H] = [da | db | u]. A workgroup: 64 rows x 64 hidden channels, a wave 32 x 32 of each of a, b and du
// (D = weight rows x token rows: a lane holds a token and 16 channels). k in steps of 64, double-buffered by
// LDS DMA. grid (ceil(rows / 64), H / 64); block 256.
__global__ __launch_bounds__(256) void hidden_grad(const bf16* __restrict__ n, const bf16* __restrict__ dy,
                                                   const bf16* __restrict__ ab, const bf16* __restrict__ st,
                                                   bf16* __restrict__ E, int64_t rows, int d, int H) {
  __shared__ bf16 buf[2][5][64 * 64];  // n, dy, A, B, S^T
  const int lane = threadIdx.x & 63, g = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row0 = (int64_t)blockIdx.x * 64;
  const int h0 = blockIdx.y * 64;
  const uint32_t lds = lds_addr(buf);
  auto fetch = [&](int c0, int which) __attribute__((always_inline)) {
    const uint32_t at = lds + which * 5 * 8192;
    tile_dma(n, d, row0, rows - 1, c0, at, wave, lane);
    tile_dma(dy, d, row0, rows - 1, c0, at + 8192, wave, lane);
    tile_dma(ab, d, h0, 2 * H - 1, c0, at + 2 * 8192, wave, lane);
    tile_dma(ab, d, H + h0, 2 * H - 1, c0, at + 3 * 8192, wave, lane);
    tile_dma(st, d, h0, H - 1, c0, at + 4 * 8192, wave, lane);
  };
  f32x16 a = zero16(), b = zero16(), du = zero16();
  const int rt = 32 * (wave & 1) + li, rh = 32 * (wave >> 1) + li;
  fetch(0, 0);
  int which = 0;
  for (int c0 = 0; c0 < d; c0 += 64, which ^= 1) {
    if (c0 + 64 < d) {
      fetch(c0 + 64, which ^ 1);
      wait_vm_lds<10>();
    } else {
      wait_vm_lds<0>();
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const bf16x8 nt = ld8(&buf[which][0][off64(rt, 2 * kk + g)]);
      const bf16x8 dt = ld8(&buf[which][1][off64(rt, 2 * kk + g)]);
      a = mfma32(ld8(&buf[which][2][off64(rh, 2 * kk + g)]), nt, a);
      b = mfma32(ld8(&buf[which][3][off64(rh, 2 * kk + g)]), nt, b);
      du = mfma32(ld8(&buf[which][4][off64(rh, 2 * kk + g)]), dt, du);
    }
    __syncthreads();
  }
  f32x16 u;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const SwigluGrad e = swiglu_grad(a[r], b[r], du[r]);
    a[r] = e.da;
    b[r] = e.db;
    u[r] = e.u;
  }
  const int64_t row = row0 + rt;
  auto put = [&](const f32x16& acc, int part) __attribute__((always_inline)) {
    float y[2][8];
    acc_pieces(acc, y);
    if (row < rows) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        bf16x8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (bf16)y[k][e];
        *reinterpret_cast<bf16x8*>(E + row * 3 * H + part * H + h0 + 32 * (wave >> 1) + 8 * (2 * k + g)) = o;
      }
    }
  };
  put(a, 0);
  put(b, 1);
  put(u, 2);
}

// A 64 x 64 tile of C (fp32) a workgroup, its four waves taking turns of 16 k in each step of 64 and joining
// their sums in LDS at the end: a wave's 2 x 2 MFMA tiles then read one operand a product, which is what LDS
// can deliver beside the matrix cores (a quarter of the tile each would read two).
//   TURN false: C[m][n] = sum over k of A[m][k] B[n][k]    (m clamped to m_rows, n in range)
//   TURN true:  C[m][n] = sum over k of A[k][m] B[k][n]    (k rows past k_rows count as zero)
// Split s of the k axis: k from s * k_share, to C + s * split_stride; add: C is added to. B2 takes the place
// of B from m tile m_two on. grid (m tiles, n tiles, splits); block 256.
struct Gemm64Args {
  const bf16 *A, *B, *B2;
  float* C;
  int64_t lda, ldb, m_rows, k_rows, k_share, split_stride;
  int ldc, m_two, add;
};
template <bool TURN>
__global__ __launch_bounds__(256) void gemm64(const Gemm64Args p) {
  constexpr int NB = 4;
  __shared__ __attribute__((aligned(16))) bf16 buf[NB][2][64 * 64];
  const int lane = threadIdx.x & 63, g = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m0 = (int64_t)blockIdx.x * 64;
  const int n0 = blockIdx.y * 64;
  const int64_t kb = (int64_t)blockIdx.z * p.k_share;
  const int64_t ke = kb + p.k_share < p.k_rows ? kb + p.k_share : p.k_rows;
  const bf16* B = (int)blockIdx.x >= p.m_two ? p.B2 : p.B;
  const int steps = ke > kb ? (int)((ke - kb + 63) / 64) : 0;
  const uint32_t lds = lds_addr(buf);
  auto fetch = [&](int step) __attribute__((always_inline)) {
    const uint32_t at = lds + (step % NB) * 2 * 8192;
    const int64_t k = kb + 64 * (int64_t)step;
    if (TURN) {
      tile_dma(p.A, p.lda, k, p.k_rows - 1, (int)m0, at, wave, lane);
      tile_dma(B, p.ldb, k, p.k_rows - 1, n0, at + 8192, wave, lane);
    } else {
      tile_dma(p.A + k, p.lda, m0, p.m_rows - 1, 0, at, wave, lane);
      tile_dma(B + k, p.ldb, n0, n0 + 63, 0, at + 8192, wave, lane);
    }
  };
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = zero16();
#pragma unroll
  for (int s = 0; s < NB - 1; ++s)
    if (s < steps) fetch(s);
  for (int s = 0; s < steps; ++s) {
    // steps s + 1 .. s + NB - 2 stay in flight (4 transfers of this wave each), fewer at the end
    if (s + 2 < steps)
      wait_vm_lds<8>();
    else if (s + 1 < steps)
      wait_vm_lds<4>();
    else
      wait_vm_lds<0>();
    __syncthreads();
    if (s + NB - 1 < steps) fetch(s + NB - 1);  // into the buffer that step s - 1 read
    bf16* tA = buf[s % NB][0];
    bf16* tB = buf[s % NB][1];
    if (TURN) {
      const int64_t left = ke - (kb + 64 * (int64_t)s);  // rows of this step that count
      if (left < 64) {
        for (int i = threadIdx.x; i < 2 * 64 * 8; i += 256) {
          const int r = (i >> 3) & 63;
          if (r >= left) {
            bf16x8 z;
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = (bf16)0.f;
            *reinterpret_cast<bf16x8*>((i >> 9 ? tB : tA) + r * 64 + 8 * (i & 7)) = z;
          }
        }
        __syncthreads();
      }
    }
    bf16x8 fa[2], fb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (TURN) {
        fa[i] = ld_turned(tA, 32 * i, 16 * wave, lane);
        fb[i] = ld_turned(tB, 32 * i, 16 * wave, lane);
      } else {
        fa[i] = ld8(&tA[off64(32 * i + li, 2 * wave + g)]);
        fb[i] = ld8(&tB[off64(32 * i + li, 2 * wave + g)]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = mfma32(fa[i >> 1], fb[i & 1], acc[i >> 1][i & 1]);
  }
  __syncthreads();
  // the waves' sums: [wave][tile][register][lane] fp32 in the buffers' place (64 KB)
  float* red = reinterpret_cast<float*>(buf);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) red[((wave * 4 + t) * 16 + r) * 64 + lane] = acc[t >> 1][t & 1][r];
  __syncthreads();
  // wave t stores tile t
  float* C = p.C + blockIdx.z * p.split_stride;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) v += red[((w * 4 + wave) * 16 + r) * 64 + lane];
    const int64_t m = m0 + 32 * (wave >> 1) + acc_row(r, g);
    if (m < p.m_rows) {
      float* to = C + m * p.ldc + n0 + 32 * (wave & 1) + li;
      *to = p.add ? *to + v : v;
    }
  }
}
static_assert(4 * 2 * 64 * 64 * sizeof(bf16) >= 4 * 4 * 16 * 64 * sizeof(float), "the waves' sums fit the buffers");

// dx = (residual ? dy : 0) + LN'(dn) of the rows, dn the sum of `splits` fp32 parts, and this workgroup's sums
// of dn xh and dn (part [gridDim.x][2][d], added to where add). One wave a row, K = d / 64; block 256.
template <bool CODES, int K>
__global__ __launch_bounds__(256) void norm_grad_rows(const void* x, const uint8_t* scales, const bf16* __restrict__ dy,
                                                      const float* __restrict__ dn, int splits, int64_t split_stride,
                                                      const float* __restrict__ w, bf16* __restrict__ dx,
                                                      float* __restrict__ part, int64_t rows, int residual, int add,
                                                      float eps) {
  constexpr int d = 64 * K, blocks = d / kActBlock;
  __shared__ float red[2][4][d];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float sw[K], sb[K], wv[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    sw[k] = sb[k] = 0.f;
    wv[k] = w[lane + 64 * k];
  }
  for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < rows; row += (int64_t)gridDim.x * 4) {
    float v[K], t[K];
    float s = 0.f, sg = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = lane + 64 * k;
      KeptPiece<bf16, CODES, 1> p;
      p.load(x, scales, row, c, d, blocks);
      p.values(&v[k]);
      t[k] = 0.f;
      for (int i = 0; i < splits; ++i) t[k] += dn[i * split_stride + row * d + c];
      s += v[k];
      sg += t[k] * wv[k];
    }
    const float mean = lanes_sum<64>(s) * (1.f / d), c1 = lanes_sum<64>(sg) * (1.f / d);
    float q = 0.f, sx = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] -= mean;
      q += v[k] * v[k];
      sx += (t[k] * wv[k] - c1) * v[k];
    }
    const float rstd = __builtin_amdgcn_rsqf(lanes_sum<64>(q) * (1.f / d) + eps);
    const float c2 = lanes_sum<64>(sx) * (1.f / d) * rstd * rstd;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t at = row * d + lane + 64 * k;
      sw[k] += t[k] * (v[k] * rstd);
      sb[k] += t[k];
      dx[at] = (bf16)((residual ? (float)dy[at] : 0.f) + rstd * (t[k] * wv[k] - c1 - v[k] * c2));
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    red[0][wave][lane + 64 * k] = sw[k];
    red[1][wave][lane + 64 * k] = sb[k];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * d; i += 256) {
    const float* r = &red[0][0][0] + (i / d) * 4 * d + i % d;
    float* to = part + (int64_t)blockIdx.x * 2 * d + i;
    const float v = (r[0] + r[d]) + (r[2 * d] + r[3 * d]);
    *to = add ? *to + v : v;
  }
}

// The weights' gradients from `count` parts [3 H][d] (dA, dB, dS^T): dA and dB in order, dS turned. A 32 x 32
// tile a workgroup: grid (d / 32, 3 H / 32); block 256.
__global__ __launch_bounds__(256) void join_weight_grads(const float* __restrict__ part, int count, int d, int H,
                                                         void* da, void* db, void* ds, int dtype) {
  __shared__ float tile[32][33];
  const int c0 = blockIdx.x * 32, h0 = blockIdx.y * 32;
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int64_t size = (int64_t)3 * H * d;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row + 8 * i;
    const float* p = part + (int64_t)(h0 + r) * d + c0 + col;
    float v = 0.f;
    for (int k = 0; k < count; ++k) v += p[k * size];
    if (h0 < 2 * H) {
      void* to = h0 < H ? da : db;
      const int64_t at = (int64_t)(h0 + r - (h0 < H ? 0 : H)) * d + c0 + col;
      if (dtype == 0)
        static_cast<bf16*>(to)[at] = (bf16)v;
      else
        static_cast<float*>(to)[at] = v;
    } else {
      tile[r][col] = v;
    }
  }
  if (h0 < 2 * H) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row + 8 * i;
    const int64_t at = (int64_t)(c0 + r) * H + h0 - 2 * H + col;
    if (dtype == 0)
      static_cast<bf16*>(ds)[at] = (bf16)tile[col][r];
    else
      static_cast<float*>(ds)[at] = tile[col][r];
  }
}

template <bool CODES>
void run_norm_rows(const void* x, const uint8_t* scales, const float* w, const float* b, bf16* n, int64_t rows, int d,
                   float eps, hipStream_t st) {
  const dim3 grid((unsigned)std::min<int64_t>((rows + 3) / 4, (int64_t)cu_count() * 8));
  switch (d / 64) {
#define FFK_K(K_) case K_: norm_rows<CODES, K_><<<grid, 256, 0, st>>>(x, scales, w, b, n, rows, eps); break;
    FFK_K(1) FFK_K(2) FFK_K(3) FFK_K(4) FFK_K(5) FFK_K(6) FFK_K(7) FFK_K(8) FFK_K(9) FFK_K(10) FFK_K(11) FFK_K(12)
#undef FFK_K
  }
}

template <bool CODES>
void run_norm_grad_rows(const void* x, const uint8_t* scales, const bf16* dy, const float* dn, int splits,
                        int64_t split_stride, const float* w, bf16* dx, float* part, int blocks, int64_t rows, int d,
                        int residual, int add, float eps, hipStream_t st) {
  switch (d / 64) {
#define FFK_K(K_)                                                                                                 \
  case K_:                                                                                                        \
    norm_grad_rows<CODES, K_><<<blocks, 256, 0, st>>>(x, scales, dy, dn, splits, split_stride, w, dx, part, rows, \
                                                      residual, add, eps);                                        \
    break;
    FFK_K(1) FFK_K(2) FFK_K(3) FFK_K(4) FFK_K(5) FFK_K(6) FFK_K(7) FFK_K(8) FFK_K(9) FFK_K(10) FFK_K(11) FFK_K(12)
#undef FFK_K
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

TransitionGradPlan transition_grad_plan(int64_t rows, int d, int H) {
  TransitionGradPlan p{};
  // E of a chunk within 96 MB, so that it is still in the 256 MB last-level cache when the products read it
  const int64_t fit = std::max<int64_t>((int64_t)(96 << 20) / (6 * H) / 64 * 64, 64);
  p.chunk = std::min<int64_t>(ceil_div(rows, 64) * 64, fit);
  const int64_t cus = cu_count();
  // both products want a workgroup a CU at least, and four steps of 64 in each
  p.dn_splits = (int)std::max<int64_t>(1, std::min<int64_t>(cus / std::max<int64_t>(1, p.chunk / 64 * (d / 64)), 2 * H / 256));
  p.dw_splits = (int)std::max<int64_t>(1, std::min<int64_t>(2 * cus / std::max<int64_t>(1, 3 * H / 64 * (d / 64)), p.chunk / 256));
  p.norm_blocks = (int)std::min<int64_t>(ceil_div(std::min(rows, p.chunk), 4), cus * 4);
  return p;
}

void launch_transition_grad(const TransitionGradArgs& a, const TransitionGradPlan& p, hipStream_t st) {
  const int d = a.d, H = a.hidden;
  pack_grad_weights<<<dim3(H / 32, d / 32, 3), 256, 0, st>>>(a.wa, a.wb, a.ws, a.ab, a.st, a.abt, d, H);
  const char* x = static_cast<const char*>(a.x);
  for (int64_t r0 = 0; r0 < a.rows; r0 += p.chunk) {
    const int64_t rows = std::min(p.chunk, a.rows - r0);
    const void* xc = x + r0 * d * (a.scales ? 1 : 2);
    const uint8_t* sc = a.scales ? a.scales + r0 * (d / kActBlock) : nullptr;
    const bf16* dy = a.dy + r0 * d;
    const int add = r0 > 0;
    if (sc)
      run_norm_rows<true>(xc, sc, a.ln_w, a.ln_b, a.n, rows, d, a.eps, st);
    else
      run_norm_rows<false>(xc, sc, a.ln_w, a.ln_b, a.n, rows, d, a.eps, st);
    hidden_grad<<<dim3((unsigned)ceil_div(rows, 64), H / 64), 256, 0, st>>>(a.n, dy, a.ab, a.st, a.E, rows, d, H);
    Gemm64Args g{};
    g.A = a.E;
    g.lda = 3 * H;
    g.m_rows = rows;
    g.B = g.B2 = a.abt;
    g.ldb = 2 * H;
    g.k_rows = 2 * H;
    g.k_share = ceil_div(ceil_div(2 * H, p.dn_splits), 64) * 64;
    g.C = a.dn;
    g.ldc = d;
    g.split_stride = p.chunk * d;
    g.m_two = 0x7fffffff;
    gemm64<false><<<dim3((unsigned)ceil_div(rows, 64), d / 64, p.dn_splits), 256, 0, st>>>(g);
    if (sc)
      run_norm_grad_rows<true>(xc, sc, dy, a.dn, p.dn_splits, g.split_stride, a.ln_w, a.dx + r0 * d, a.norm_part,
                               p.norm_blocks, rows, d, a.residual, add, a.eps, st);
    else
      run_norm_grad_rows<false>(xc, sc, dy, a.dn, p.dn_splits, g.split_stride, a.ln_w, a.dx + r0 * d, a.norm_part,
                                p.norm_blocks, rows, d, a.residual, add, a.eps, st);
    Gemm64Args t{};
    t.A = a.E;
    t.lda = 3 * H;
    t.m_rows = 3 * H;
    t.B = a.n;
    t.B2 = dy;
    t.m_two = 2 * H / 64;
    t.ldb = d;
    t.k_rows = rows;
    t.k_share = ceil_div(ceil_div(p.chunk, p.dw_splits), 64) * 64;
    t.C = a.dw_part;
    t.ldc = d;
    t.split_stride = (int64_t)3 * H * d;
    t.add = add;
    gemm64<true><<<dim3(3 * H / 64, d / 64, p.dw_splits), 256, 0, st>>>(t);
  }
  // (no rows: sums over nothing)
  launch_sum_partials(a.norm_part, a.rows > 0 ? p.norm_blocks : 0, 2 * d, d, a.dln_w, a.dln_b, a.grad_dtype, st);
  join_weight_grads<<<dim3(d / 32, 3 * H / 32), 256, 0, st>>>(a.dw_part, a.rows > 0 ? p.dw_splits : 0, d, H, a.dwa, a.dwb, a.dws,
                                                              a.grad_dtype);
}

}  // namespace ffk
