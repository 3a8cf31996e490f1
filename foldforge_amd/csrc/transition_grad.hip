// Backward pass of the SwiGLU transition on gfx950.
//
//   n = LN(x) = xh w + v, a = n A^T, b = n B^T, u = silu(a) b, y = x + u S^T     (A, B [H][d], S [d][H])
//   du = dy S,  da = du b s(a) (1 + a (1 - s(a))),  db = du silu(a)              (s: the logistic function)
//   dA = da^T n,  dB = db^T n,  dS = dy^T u,  dn = da A + db B,  dx = dy + LN'(dn)
// at the kept x (the input or its 8-bit activation): the hidden rows are computed again, nothing but x is
// kept between the passes. 16 M d H flops for M rows, fp32 sums.
//
// The norm's affine is taken out of the rows' way: with Aw = A diag(w) and Bw = B diag(w),
//   a = xh Aw^T + A v,   dxh = da Aw + db Bw,   dx = dy + rstd (dxh - mean(dxh) - xh mean(dxh xh))
//   dA = (da^T xh) diag(w) + (sum da) v^T,   dw = sum over h of A (da^T xh) + B (db^T xh),
//   dv = A^T (sum da) + B^T (sum db)
// so dw and dv come out of the weights' gradients, and the products see xh alone, whose values are at most
// sqrt(d): a and b are products of fp16 operands (Aw and Bw times a power of two that puts the largest of their
// entries and offsets A v, B v, of a hidden channel or (fused kernels) of 32 of them, at 2^14 .. 2^15: entries down to
// 2^-28 of that peak keep fp16's 11 bits, smaller ones lose them, and below 2^-40 of it are 0), which leaves their errors
// at an eighth of bf16's. The gradients' operands are bf16, whose range they need: three bf16 roundings lie between dy
// and a gradient, and one of the result (relative error 3.3e-3 rather than the 4.6e-3 of bf16 throughout).
// The powers of two 2^ka, 2^kb ride along: a' = 2^ka a, b' = 2^kb b, so silu' = 2^ka silu, da' = 2^kb da,
// db' = 2^ka db, u' = 2^(ka+kb) u; the transposed weights carry their inverses, the join takes the rest out.
#include <algorithm>

#include "ffk_activation.h"
#include "ffk_device.h"
#include "ffk_kernels.h"

namespace ffk {

namespace {

typedef f16 f16x8 __attribute__((__vector_size__(8 * sizeof(f16))));

__device__ __forceinline__ f32x16 mfma32h(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16x8 ld8h(const f16* p) { return *reinterpret_cast<const f16x8*>(p); }

// k with peak 2^k in [2^14, 2^15); 0 for a peak of 0, at most 110 (2^-k and peak 2^k stay normal numbers).
__device__ __forceinline__ int peak_power(float peak) {
  if (peak == 0.f) return 0;
  const int k = 14 + 127 - (int)(__float_as_uint(peak) >> 23);
  return k > 110 ? 110 : k;
}
__device__ __forceinline__ float two_to(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }

// What a call makes of its parameters.
struct WeightArgs {
  const float *wa, *wb, *ws, *w, *v;  // A, B [H][d], S [d][H]; the norm's weight and bias
  f16* aw;
  bf16 *st, *abt, *split;
  float *shift, *scale;
  int d, H;
};

// hidden channels of a packing workgroup
template <bool FUSED>
constexpr int kPackGroup = FUSED ? 32 : 8;

// A 32 x 32 tile of S^T [H][d] in bf16. block 256.
__device__ __forceinline__ void turn_squeeze(const WeightArgs& q, int h0, int c0, float (&tile)[32][33]) {
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  for (int r = row; r < 32; r += 8) tile[r][col] = q.ws[(int64_t)(c0 + r) * q.H + h0 + col];
  __syncthreads();
  for (int r = row; r < 32; r += 8) q.st[(int64_t)(h0 + r) * q.d + c0 + col] = (bf16)tile[col][r];
}

// The parameters in the orders the products read, each hidden channel (FUSED: each 32 of them, the rows kernel's chunk)
// with powers ka, kb of its own, so that one pass over them does it all: aw [2 H][d] fp16 (Aw 2^ka, then Bw 2^kb), shift
// [2][H] (the offsets A v, B v so scaled), scale [2][H] = {2^-ka, 2^-kb}, abt [d][2 H] bf16 (Aw^T 2^-kb, Bw^T 2^-ka), st
// [H][d] bf16 (S^T). FUSED: abt within each 16 hidden channels in accumulator order 0-3, 8-11, 4-7, 12-15, and split
// [2][H][8] bf16 = {the scaled offset in three parts, 2^-ka, 0, ..}. The peaks count the offsets, so a', b' <= 2^15 (1 + d)
// whatever w, v and the weights are, and no product of theirs leaves fp32. H / G workgroups of G hidden channels, a
// quarter of them in a wave's registers, then H / 32 x d / 32 of a tile of S^T. block 256. (In one launch with the rows 8.0 us
// at 384 x 4, in a launch after it 4.1 + 7.1; with abt in pieces of 4 hidden channels 11.)
template <int K, bool FUSED>
__device__ __forceinline__ void pack_rows(int block, const WeightArgs& q) {
  constexpr int d = 64 * K, N = FUSED ? 8 : 2, G = kPackGroup<FUSED>;
  static_assert(G == 4 * N, "a quarter a wave");
  __shared__ __attribute__((aligned(16))) bf16 turned[2][d][FUSED ? G + 8 : G];
  const int H = q.H;
  if (block >= H / G) {
    const int t = block - H / G;
    __shared__ float tile[32][33];
    turn_squeeze(q, t % (H / 32) * 32, t / (H / 32) * 32, tile);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h0 = G * block + N * wave;
  float t[2][N][K], dot[2][N], w[K], v[K];
  int power[2][N];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < N; ++r)
#pragma unroll
      for (int k = 0; k < K; ++k) t[m][r][k] = (m ? q.wb : q.wa)[(int64_t)(h0 + r) * d + lane + 64 * k];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    w[k] = q.w[lane + 64 * k];
    v[k] = q.v[lane + 64 * k];
  }
  float peak[2] = {0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < N; ++r) {
      float top = 0.f, sum = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        sum += t[m][r][k] * v[k];
        t[m][r][k] *= w[k];
        top = fmaxf(top, finite_abs(t[m][r][k]));
      }
      dot[m][r] = lanes_sum<64>(sum);
      top = fmaxf(top, finite_abs(dot[m][r]));
      if constexpr (FUSED) {
        peak[m] = fmaxf(peak[m], top);
      } else {
#pragma unroll
        for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
        power[m][r] = peak_power(top);
      }
    }
  if constexpr (FUSED) {
    __shared__ float red[2][4];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int x = 32; x >= 1; x >>= 1) peak[m] = fmaxf(peak[m], __shfl_xor(peak[m], x, 64));
      if (lane == 0) red[m][wave] = peak[m];
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int r = 0; r < N; ++r)
        power[m][r] = peak_power(fmaxf(fmaxf(red[m][0], red[m][1]), fmaxf(red[m][2], red[m][3])));
  }
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < N; ++r) {
      const int h = m * H + h0 + r, place = N * wave + r;
      const float up = two_to(power[m][r]), down = two_to(-power[1 - m][r]);
      if (lane == 0) {
        float o = dot[m][r] * up;
        q.shift[h] = o;
        q.scale[h] = two_to(-power[m][r]);
        if constexpr (FUSED) {
          bf16x8 parts;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            parts[e] = (bf16)(e < 3 ? o : 0.f);
            o -= (float)parts[e];
          }
          if (m == 0) parts[3] = (bf16)two_to(-power[m][r]);
          *reinterpret_cast<bf16x8*>(q.split + 8 * (int64_t)h) = parts;
        }
      }
      const int at = FUSED ? (place & ~12) | ((place & 4) << 1) | ((place & 8) >> 1) : place;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        q.aw[(int64_t)h * d + lane + 64 * k] = (f16)(t[m][r][k] * up);
        turned[m][lane + 64 * k][at] = (bf16)(t[m][r][k] * down);
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * d * (G / 8); i += 256) {
    const int piece = i % (G / 8), c = i / (G / 8) % d, m = i / (G / 8) / d;
    *reinterpret_cast<bf16x8*>(q.abt + (int64_t)c * 2 * H + m * H + G * block + 8 * piece) =
        *reinterpret_cast<const bf16x8*>(&turned[m][c][8 * piece]);
  }
}

// What a call makes of its inputs first, in one launch: the weights (the first `weight_blocks` workgroups: pack_rows),
// and xh in fp16 and bf16 and rstd of the kept rows: 8 lanes a row, K = d / 64 pieces of 8 channels each,
// the other workgroups grid-strided over rows. block 256 (32 rows). 262144 8-bit rows of 128: 31 us, 5.4 TB/s.
template <bool CODES, int K, bool FUSED>
__global__ __launch_bounds__(256) void norm_rows(const void* x, const uint8_t* scales, f16* __restrict__ xh,
                                                 bf16* __restrict__ xhb, float* __restrict__ rstd_out, int64_t rows,
                                                 float eps, int weight_blocks, const WeightArgs q) {
  constexpr int d = 64 * K, blocks = d / kActBlock;
  if ((int)blockIdx.x < weight_blocks) {
    pack_rows<K, FUSED>(blockIdx.x, q);
    return;
  }
  const int sub = threadIdx.x & 7;
  for (int64_t row = (int64_t)(blockIdx.x - weight_blocks) * 32 + (threadIdx.x >> 3); row - (threadIdx.x >> 3) < rows;
       row += (int64_t)(gridDim.x - weight_blocks) * 32) {
    const bool real = row < rows;
    float v[8 * K];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      KeptPiece<bf16, CODES, 8> p;
      p.load(x, scales, real ? row : rows - 1, 8 * sub + 64 * k, d, blocks);
      p.values(v + 8 * k);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[8 * k + e];
    }
    const float mean = lanes_sum<8>(s) * (1.f / d);
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < 8 * K; ++i) {
      v[i] -= mean;
      q += v[i] * v[i];
    }
    const float rstd = __builtin_amdgcn_rsqf(lanes_sum<8>(q) * (1.f / d) + eps);
    if (!real) continue;
    if (sub == 0) rstd_out[row] = rstd;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      f16x8 h;
      bf16x8 b;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[e] = (f16)(v[8 * k + e] * rstd);
        b[e] = (bf16)(v[8 * k + e] * rstd);
      }
      *reinterpret_cast<f16x8*>(xh + row * d + 8 * sub + 64 * k) = h;
      *reinterpret_cast<bf16x8*>(xhb + row * d + 8 * sub + 64 * k) = b;
    }
  }
}

// da' = 2^kb da, db' = 2^ka db and u' = 2^(ka + kb) u of an element from a' = 2^ka a, b' = 2^kb b and du; slow = -log2(e) 2^-ka,
// ia = 2^-ka.
struct SwigluGrad {
  float da, db, u;
};
__device__ __forceinline__ SwigluGrad swiglu_grad(float a, float b, float du, float slow, float ia) {
  const float s = __builtin_amdgcn_rcpf(1.f + fast_exp2(a * slow)), sa = a * s;
  const float slope = fmaf(fmaf(-sa, s, sa), ia, s);  // s + silu(a) (1 - s)
  return {du * b * slope, du * sa, sa * b};
}

// E [rows][3 H] = [da' | db' | u']. A workgroup: 64 rows x 64 hidden channels, a wave 32 x 32 of each of a, b and du
// (D = weight rows x token rows: a lane holds a token and 16 channels). k in steps of 64, double-buffered by
// LDS DMA. grid (ceil(rows / 64), H / 64); block 256. 100 rows x 384 x 1536: 9 us, a chain of six steps' latencies in 48
// workgroups (a third buffer: the same; 32 x 32 a wave straight from memory: 8, but 18 against 12 at 500 rows).
__global__ __launch_bounds__(256) void hidden_grad(const f16* __restrict__ xh, const bf16* __restrict__ dy,
                                                   const f16* __restrict__ aw, const bf16* __restrict__ st,
                                                   const float* __restrict__ offset, const float* __restrict__ scale,
                                                   bf16* __restrict__ E, int64_t rows, int d, int H) {
  __shared__ __attribute__((aligned(16))) bf16 buf[2][5][64 * 64];  // xh, dy, Aw, Bw, S^T
  const int lane = threadIdx.x & 63, g = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row0 = (int64_t)blockIdx.x * 64;
  const int h0 = blockIdx.y * 64;
  const uint32_t lds = lds_addr(buf);
  auto fetch = [&](int c0, int which) __attribute__((always_inline)) {
    const uint32_t at = lds + which * 5 * 8192;
    tile_dma(xh, d, row0, rows - 1, c0, at, wave, lane);
    tile_dma(dy, d, row0, rows - 1, c0, at + 8192, wave, lane);
    tile_dma(aw, d, h0, 2 * H - 1, c0, at + 2 * 8192, wave, lane);
    tile_dma(aw, d, H + h0, 2 * H - 1, c0, at + 3 * 8192, wave, lane);
    tile_dma(st, d, h0, H - 1, c0, at + 4 * 8192, wave, lane);
  };
  f32x16 a, b, du = zero16(), ia;
  const int hw = h0 + 32 * (wave >> 1);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    a[r] = offset[hw + acc_row(r, g)];
    b[r] = offset[H + hw + acc_row(r, g)];
    ia[r] = scale[hw + acc_row(r, g)];
  }
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
      const auto half = [&](int k, int r) __attribute__((always_inline)) {
        return ld8h(reinterpret_cast<const f16*>(&buf[which][k][off64(r, 2 * kk + g)]));
      };
      const f16x8 nt = half(0, rt);
      const bf16x8 dt = ld8(&buf[which][1][off64(rt, 2 * kk + g)]);
      a = mfma32h(half(2, rh), nt, a);
      b = mfma32h(half(3, rh), nt, b);
      du = mfma32(ld8(&buf[which][4][off64(rh, 2 * kk + g)]), dt, du);
    }
    __syncthreads();
  }
  f32x16 u;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const SwigluGrad e = swiglu_grad(a[r], b[r], du[r], -kLog2e * ia[r], ia[r]);
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
// of B from m tile m_two on. TURN: sums[s][m] = sum over k of A[k][m] for the m tiles before m_two (by a product
// with ones, in the workgroups of the first n tile). grid (m tiles, n tiles, splits); block 256. 2000 rows x 128 x 512: 9 us
// (TURN) and 6.5: latency, three steps in flight.
struct Gemm64Args {
  const bf16 *A, *B, *B2;
  float *C, *sums;
  int64_t lda, ldb, m_rows, k_rows, k_share, split_stride, sums_stride;
  int ldc, m_two, add, m_tiles, n_tiles;
};
struct Gemm64Lds {
  bf16 buf[4][2][64 * 64];
  float total[4][64], affine[2][2][64];  // (of a call whose products are the gradients)
};
// What the weights' gradients take where one workgroup has all of a tile's sum: see store_weight_grads.
struct WeightGradArgs {
  const float *wa, *wb, *w, *v, *scale;
  float* part;
  void *da, *db, *ds;
  int d, H, dtype;
};
__device__ __forceinline__ void store_weight_grads(const WeightGradArgs& q, float (&t)[16], Gemm64Lds& lds, int m0, int n0);

template <bool TURN, bool GRADS>
__device__ __forceinline__ void gemm64_tile(const Gemm64Args& p, const WeightGradArgs& q, Gemm64Lds& sh, int bx, int by,
                                            int bz) {
  constexpr int NB = 4;
  auto& buf = sh.buf;
  const int lane = threadIdx.x & 63, g = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m0 = (int64_t)bx * 64;
  const int n0 = by * 64;
  const int64_t kb = (int64_t)bz * p.k_share;
  const int64_t ke = kb + p.k_share < p.k_rows ? kb + p.k_share : p.k_rows;
  const bf16* B = bx >= p.m_two ? p.B2 : p.B;
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
  const bool summed = TURN && (GRADS || by == 0) && bx < p.m_two;
  f32x16 acc[2][2], total[2];
  total[0] = total[1] = zero16();
  bf16x8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (bf16)1.f;
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
    if (TURN && summed) {
      total[0] = mfma32(fa[0], ones, total[0]);
      total[1] = mfma32(fa[1], ones, total[1]);
    }
  }
  __syncthreads();
  // the waves' sums: [wave][tile][register][lane] fp32 in the buffers' place (64 KB)
  float* red = reinterpret_cast<float*>(buf);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) red[((wave * 4 + t) * 16 + r) * 64 + lane] = acc[t >> 1][t & 1][r];
  if (TURN && summed && li == 0) {  // (every column of a total is the same)
#pragma unroll
    for (int r = 0; r < 32; ++r) sh.total[wave][32 * (r >> 4) + acc_row(r & 15, g)] = total[r >> 4][r & 15];
  }
  __syncthreads();
  // wave t has tile t
  float v[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    v[r] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) v[r] += red[((w * 4 + wave) * 16 + r) * 64 + lane];
  }
  if constexpr (GRADS) {
    store_weight_grads(q, v, sh, (int)m0, n0);
    return;
  }
  float* C = p.C + bz * p.split_stride;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int64_t m = m0 + 32 * (wave >> 1) + acc_row(r, g);
    if (m < p.m_rows) {
      float* to = C + m * p.ldc + n0 + 32 * (wave & 1) + li;
      *to = p.add ? *to + v[r] : v[r];
    }
  }
  if (TURN && summed && threadIdx.x < 64) {
    const int i = threadIdx.x;
    float* to = p.sums + bz * p.sums_stride + m0 + i;
    const float t = (sh.total[0][i] + sh.total[1][i]) + (sh.total[2][i] + sh.total[3][i]);
    *to = p.add ? *to + t : t;
  }
}
static_assert(4 * 2 * 64 * 64 * sizeof(bf16) >= 4 * 4 * 16 * 64 * sizeof(float), "the waves' sums fit the buffers");

template <bool TURN>
__global__ __launch_bounds__(256) void gemm64(const Gemm64Args p) {
  __shared__ __attribute__((aligned(16))) Gemm64Lds sh;
  gemm64_tile<TURN, false>(p, {}, sh, blockIdx.x, blockIdx.y, blockIdx.z);
}

// gradient `at` of an output in bf16 (dtype 0) or fp32
__device__ __forceinline__ void put_grad(void* to, int64_t at, float t, int dtype) {
  if (dtype == 0)
    static_cast<bf16*>(to)[at] = (bf16)t;
  else
    static_cast<float*>(to)[at] = t;
}
// 2^-ka 2^-kb t (the product of the two may leave fp32 where the gradient does not)
__device__ __forceinline__ float unscale_both(float t, float ia, float ib) {
  return __builtin_ldexpf(t, __builtin_amdgcn_frexp_expf(ia) + __builtin_amdgcn_frexp_expf(ib) - 2);
}

// As join_weight_grads, from a 64 x 64 tile of G in registers (a wave 32 x 32 of it): part [2 H / 64][2][d].
__device__ __forceinline__ void store_weight_grads(const WeightGradArgs& q, float (&t)[16], Gemm64Lds& sh, int m0, int n0) {
  const int lane = threadIdx.x & 63, g = lane >> 5, li = lane & 31, wave = threadIdx.x >> 6;
  const int mw = 32 * (wave >> 1), c = 32 * (wave & 1) + li;
  if (m0 >= 2 * q.H) {  // dS [d][H]: 4 hidden channels of a row together
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int h = m0 - 2 * q.H + mw + acc_row(4 * k, g);
      const int64_t at = (int64_t)(n0 + c) * q.H + h;
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = unscale_both(t[4 * k + e], q.scale[h + e], q.scale[q.H + h + e]);
      if (q.dtype == 0) {
        const bf16x4 b = {(bf16)o[0], (bf16)o[1], (bf16)o[2], (bf16)o[3]};
        *reinterpret_cast<bf16x4*>(static_cast<bf16*>(q.ds) + at) = b;
      } else {
        *reinterpret_cast<f32x4*>(static_cast<float*>(q.ds) + at) = f32x4{o[0], o[1], o[2], o[3]};
      }
    }
    return;
  }
  const bool first = m0 < q.H;
  const float w = q.w[n0 + c], v = q.v[n0 + c];
  float aw = 0.f, av = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int i = mw + acc_row(r, g);
    const int h = m0 + i - (first ? 0 : q.H);
    const float back = q.scale[first ? q.H + h : h];
    const float total = ((sh.total[0][i] + sh.total[1][i]) + (sh.total[2][i] + sh.total[3][i])) * back;
    const int64_t at = (int64_t)h * q.d + n0 + c;
    t[r] *= back;
    const float own = (first ? q.wa : q.wb)[at];
    put_grad(first ? q.da : q.db, at, t[r] * w + total * v, q.dtype);
    aw += own * t[r];
    av += own * total;
  }
  aw += __shfl_xor(aw, 32, 64);
  av += __shfl_xor(av, 32, 64);
  if (g == 0) {
    sh.affine[wave >> 1][0][c] = aw;
    sh.affine[wave >> 1][1][c] = av;
  }
  __syncthreads();
  if (threadIdx.x < 128) {
    const int which = threadIdx.x >> 6, i = threadIdx.x & 63;
    q.part[((int64_t)(m0 / 64) * 2 + which) * q.d + n0 + i] = sh.affine[0][which][i] + sh.affine[1][which][i];
  }
}

// Few rows: both products of E in one launch, the weights' gradients finished where they are summed. The first
// `tiles` workgroups are those of t (m_tiles = 3 H / 64 by n_tiles = d / 64), the others those of g (m_tiles by n_tiles
// by the splits of k). block 256. 100 rows x 384 x 1536: 11 us, where the two products and the join took 6, 7 and 9
// (g's workgroups first: the call 3 us longer).
__global__ __launch_bounds__(256) void grad_products(const Gemm64Args t, const WeightGradArgs q, const Gemm64Args g,
                                                     int tiles) {
  __shared__ __attribute__((aligned(16))) Gemm64Lds sh;
  const int i = blockIdx.x;
  if (i < tiles) {
    gemm64_tile<true, true>(t, q, sh, i % t.m_tiles, i / t.m_tiles, 0);
  } else {
    const int j = i - tiles, mn = g.m_tiles * g.n_tiles;
    gemm64_tile<false, false>(g, {}, sh, j % g.m_tiles, j % mn / g.m_tiles, j / mn);
  }
}

// The same products in 128 x 128 tiles, a wave 64 x 64 of it over all k, where the matrix is made of such tiles and they
// are enough for every CU: sixteen products a wave between two barriers, and half the reads from memory.
// grid m tiles x n tiles x splits; block 256. 40000 rows x 256 x 512: 57 us (TURN; 75 before neighbours shared an XCD) and 40,
// 0.55 and 0.52 PFLOP/s at 2.6 and 3.1 TB/s (E of 123 MB from the last-level cache, the fp32 result): the waits at the two
// buffers' barriers, 38 and 52% of the waves' time (eight waves that split k: 81).
template <bool TURN>
__global__ __launch_bounds__(256, 2) void gemm128(const Gemm64Args p) {
  __shared__ __attribute__((aligned(16))) bf16 buf[2][4][64 * 64];  // A's two tiles, B's two
  const int lane = threadIdx.x & 63, g = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  // neighbours on an XCD share its L2: TURN, the tiles of one share of k (A by the n tiles, B by all m tiles); else the n
  // tiles of an m tile (A), then the next m tile (B)
  const uint32_t id = xcd_remap(blockIdx.x, gridDim.x);
  const int mt = p.m_tiles, nt = p.n_tiles;
  const int bx = TURN ? id % mt : id / nt % mt, by = TURN ? id / mt % nt : id % nt, bz = id / (mt * nt);
  const int64_t m0 = (int64_t)bx * 128;
  const int n0 = by * 128;
  const int64_t kb = (int64_t)bz * p.k_share;
  const int64_t ke = kb + p.k_share < p.k_rows ? kb + p.k_share : p.k_rows;
  const bf16* B = bx * 2 >= p.m_two ? p.B2 : p.B;
  const int steps = ke > kb ? (int)((ke - kb + 63) / 64) : 0;
  const uint32_t lds = lds_addr(buf);
  auto fetch = [&](int step) __attribute__((always_inline)) {
    const uint32_t at = lds + (step & 1) * 4 * 8192;
    const int64_t k = kb + 64 * (int64_t)step;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (TURN) {
        tile_dma(p.A, p.lda, k, p.k_rows - 1, (int)m0 + 64 * i, at + 8192 * i, wave, lane);
        tile_dma(B, p.ldb, k, p.k_rows - 1, n0 + 64 * i, at + 8192 * (2 + i), wave, lane);
      } else {
        tile_dma(p.A + k, p.lda, m0 + 64 * i, p.m_rows - 1, 0, at + 8192 * i, wave, lane);
        tile_dma(B + k, p.ldb, n0 + 64 * i, n0 + 127, 0, at + 8192 * (2 + i), wave, lane);
      }
    }
  };
  const bool summed = TURN && by == 0 && wn == 0 && bx * 2 < p.m_two;
  f32x16 acc[2][2], total[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = zero16();
  total[0] = total[1] = zero16();
  bf16x8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (bf16)1.f;
  if (steps > 0) fetch(0);
  for (int s = 0; s < steps; ++s) {
    wait_vm_lds<0>();
    __syncthreads();  // the step has landed; the other buffer has been read
    if (s + 1 < steps) fetch(s + 1);
    bf16(*t)[64 * 64] = buf[s & 1];
    if (TURN) {
      const int64_t left = ke - (kb + 64 * (int64_t)s);  // rows of this step that count
      if (left < 64) {
        for (int i = threadIdx.x; i < 4 * 64 * 8; i += 256) {
          const int r = (i >> 3) & 63;
          if (r >= left) {
            bf16x8 z;
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = (bf16)0.f;
            *reinterpret_cast<bf16x8*>(t[i >> 9] + r * 64 + 8 * (i & 7)) = z;
          }
        }
        __syncthreads();
      }
    }
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      bf16x8 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (TURN) {
          fa[i] = ld_turned(t[wm], 32 * i, 16 * kk, lane);
          fb[i] = ld_turned(t[2 + wn], 32 * i, 16 * kk, lane);
        } else {
          fa[i] = ld8(&t[wm][off64(32 * i + li, 2 * kk + g)]);
          fb[i] = ld8(&t[2 + wn][off64(32 * i + li, 2 * kk + g)]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = mfma32(fa[i >> 1], fb[i & 1], acc[i >> 1][i & 1]);
      if (TURN && summed) {
        total[0] = mfma32(fa[0], ones, total[0]);
        total[1] = mfma32(fa[1], ones, total[1]);
      }
    }
  }
  float* C = p.C + bz * p.split_stride;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t m = m0 + 64 * wm + 32 * i + acc_row(r, g);
      if (m < p.m_rows) {
        float* to = C + m * p.ldc + n0 + 64 * wn + li;
        to[0] = p.add ? to[0] + acc[i][0][r] : acc[i][0][r];
        to[32] = p.add ? to[32] + acc[i][1][r] : acc[i][1][r];
      }
    }
  if (summed && li == 0) {  // (every column of a total is the same)
    float* to = p.sums + bz * p.sums_stride + m0 + 64 * wm;
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      float* q = to + 32 * (r >> 4) + acc_row(r & 15, g);
      *q = p.add ? *q + total[r >> 4][r & 15] : total[r >> 4][r & 15];
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// The fused form (d = 64 or 128): two kernels, the hidden rows stay in registers.

// Nothing is scheduled across: left alone the compiler fetches each operand right before its product and waits out the
// LDS latency every time, so the products' loops fetch a step or two ahead in the order they are written.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// One wave's 16 x 16 tile over 32 k: a lane holds row / column lane % 16 of its operands at 8 k, and rows 4 (lane / 16)
// + 0..3 of column lane % 16 of the result.
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16h(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A workgroup's group of hidden channels and share of the rows, in a grid of (groups, splits): the groups of one share, which
// read the same rows, are neighbours on one XCD and share its L2.
struct RowsAt {
  int group, split, splits;
};
__device__ __forceinline__ RowsAt rows_at_of() {
  const uint32_t id = xcd_remap(blockIdx.x + gridDim.x * blockIdx.y, gridDim.x * gridDim.y);
  return {(int)(id % gridDim.x), (int)(id / gridDim.x), (int)gridDim.y};
}

// The weights' gradients G = [da'^T xh; db'^T xh; u'^T dy] and the sums of da', db'.
//
// A wave owns 16 hidden channels: its operands of Aw, Bw and S^T (D k of 16 channels each) and its sums (3 x 16 x D
// fp32) stay in registers while the rows stream by; a workgroup's eight waves share the rows in LDS. Per 32 rows:
// a', b', du as D = rows x hidden (a lane holds a hidden channel at 8 rows), their elementwise part in place, and the
// rounded results are directly the operand [hidden x rows] of the gradients' products, whose other operand (channels
// x rows) comes out of the same rows by transposing LDS reads, in the same order of k. No hidden value leaves the
// registers, nothing is turned through LDS. (32 hidden channels a wave, one wave per SIMD, read half as much LDS, but
// products and elementwise part then waited for each other: 430 us at 262144 rows x 128 x 512, here 248: 0.83 PFLOP/s, the
// matrix cores busy in 52% of the cycles, no LDS conflicts. A SIMD's two waves hide half of each other's elementwise part.)
// grid (ceil(H / 128), splits): split s takes the stages s, s + splits, .. of 64 rows. block 512.
constexpr int kStageRows = 64;
template <int D>
__global__ __launch_bounds__(512, 2) void transition_grad_weights(
    const f16* __restrict__ xh, const bf16* __restrict__ xhb, const bf16* __restrict__ dy, const f16* __restrict__ aw,
    const bf16* __restrict__ st, const float* __restrict__ offset, const float* __restrict__ scale,
    float* __restrict__ G, float* __restrict__ sums, int64_t rows, int H, int add) {
  constexpr int NB = 3, NW = 8, KK = D / 32, CT = D / 16;
  constexpr int kTile = kStageRows * D;              // elements of a tile
  constexpr int kLoads = 3 * (kTile / 512) / NW;     // transfers of a wave a stage
  __shared__ __attribute__((aligned(256))) bf16 buf[NB][3][kTile];  // xh fp16, xh bf16, dy
  const RowsAt at_ = rows_at_of();
  const int lane = threadIdx.x & 63, q = lane >> 4, li = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h0 = at_.group * 128 + 16 * wave;
  const bool own = h0 < H;  // H a multiple of 64: the last workgroup's upper waves may own nothing
  const int hr = own ? h0 + li : li;
  const uint32_t lds = lds_addr(buf);
  const int64_t stages = (rows + kStageRows - 1) / kStageRows;
  const uint32_t rows_at = 2 * off_row<D>(li, q), turned = turned_at<D>(lane);  // a lane's places in a tile
  // transfer u = 0 .. kLoads - 1 of a wave; rows past the end: the last one again
  constexpr int kKb = kLoads / 3;  // its KBs of each array
  const uint32_t lane_row = 2 * D * (lane / (D / 8)), lane_piece = kb_offset<D>(0, lane) - lane_row;
  auto fetch = [&](int64_t stage, int b, int u) __attribute__((always_inline)) {
    const int t = u / kKb, kb = kKb * wave + u % kKb, r0 = kb * (512 / D);
    const int64_t row = stage * kStageRows + r0, from = row < rows ? row : rows - 1;
    const uint32_t most = rows - 1 - from < 512 / D ? 2 * D * (uint32_t)(rows - 1 - from) : 1024u;
    const void* src = t == 0 ? (const void*)xh : t == 1 ? (const void*)xhb : (const void*)dy;
    // (the swizzle of row r0 + i is that of i, turned over by that of r0: their bits are apart)
    dma16(static_cast<const bf16*>(src) + from * D,
          (lane_row < most ? lane_row : most) + (lane_piece ^ (16 * swz<D>(r0))),
          lds + (uint32_t)((b * 3 + t) * kTile * sizeof(bf16)) + 1024 * kb);
  };
  f16x8 wa[KK], wb[KK];
  bf16x8 ws[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    wa[kk] = ld8h(aw + (int64_t)hr * D + 32 * kk + 8 * q);
    wb[kk] = ld8h(aw + (int64_t)(H + hr) * D + 32 * kk + 8 * q);
    ws[kk] = ld8(st + (int64_t)hr * D + 32 * kk + 8 * q);
  }
  const float oa = offset[hr], ob = offset[H + hr], ia = scale[hr], slow = -kLog2e * ia;
  // the parameters have landed: without this the compiler waits for them again in every stage
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) asm volatile("" ::"v"(wa[kk]), "v"(wb[kk]), "v"(ws[kk]));
  asm volatile("" ::"v"(oa), "v"(ob), "v"(ia));
  const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f}, oa4 = {oa, oa, oa, oa}, ob4 = {ob, ob, ob, ob};
  f32x4 ga[CT], gb[CT], gs[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) ga[c] = gb[c] = gs[c] = zero4;
  f32x4 ta = zero4, tb = zero4;  // sums of da', db': products with ones (every column the same)
  bf16x8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (bf16)1.f;
#pragma unroll
  for (int b = 0; b < NB - 1; ++b) {
    const int64_t stage = at_.split + (int64_t)b * at_.splits;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) fetch(stage < stages ? stage : stages - 1, b, u);
  }
  int b = 0;
#pragma unroll 1
  for (int64_t stage = at_.split; stage < stages; stage += at_.splits) {
    wait_vm_lds<(NB - 2) * kLoads>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // the next stage's transfers are spread over this one (past the end: the last rows again, which nothing reads)
    int64_t ahead = stage + (int64_t)(NB - 1) * at_.splits;
    ahead = ahead < stages ? ahead : stages - 1;
    const int into = b == 0 ? NB - 1 : b - 1;
    bf16* td = buf[b][2];
    const int64_t left = rows - stage * kStageRows;
    if (left < kStageRows) {  // rows past the end: dy = 0 makes their gradients 0
      for (int i = threadIdx.x; i < kTile / 8; i += 64 * NW)
        if (i / (D / 8) >= left) {
          bf16x8 z;
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = (bf16)0.f;
          *reinterpret_cast<bf16x8*>(td + 8 * i) = z;
        }
      __syncthreads();
    }
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      const uint32_t tile = lds + (uint32_t)((b * 3 * kTile + half * 32 * D) * sizeof(bf16));
      const uint32_t rows_a = tile + rows_at, turned_a = tile + turned;
      constexpr uint32_t kArray = kTile * sizeof(bf16);
      f32x4 a[2], bb[2], du[2];
      f16x8 lx[2][2];
      bf16x8 ly[2][2];
      auto take = [&](int kk) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          lx[kk & 1][t] = lds_at<f16x8>((rows_a ^ (kk << 6)) + 32 * D * t);
          ly[kk & 1][t] = lds_at<bf16x8>((rows_a ^ (kk << 6)) + 32 * D * t + 2 * kArray);
        }
        in_order();
      };
      bf16x8 tx8[2], ty8[2];
      auto take2 = [&](int c) __attribute__((always_inline)) {
        tx8[c & 1] = ld_turned16<D>((turned_a ^ (c << 5)) + kArray);
        ty8[c & 1] = ld_turned16<D>((turned_a ^ (c << 5)) + 2 * kArray);
        in_order();
      };
      take(0);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if (kk + 1 < KK) take(kk + 1);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          a[t] = mfma16h(lx[kk & 1][t], wa[kk], kk ? a[t] : oa4);
          bb[t] = mfma16h(lx[kk & 1][t], wb[kk], kk ? bb[t] : ob4);
          du[t] = mfma16(ly[kk & 1][t], ws[kk], kk ? du[t] : zero4);
        }
        in_order();
      }
      if (half == 0) {
#pragma unroll
        for (int u = 0; u < kLoads / 2; ++u) fetch(ahead, into, u);
      } else {
#pragma unroll
        for (int u = kLoads / 2; u < kLoads; ++u) fetch(ahead, into, u);
      }
      take2(0);
      bf16x8 fa, fb, fu;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const SwigluGrad e = swiglu_grad(a[r >> 2][r & 3], bb[r >> 2][r & 3], du[r >> 2][r & 3], slow, ia);
        fa[r] = (bf16)e.da;
        fb[r] = (bf16)e.db;
        fu[r] = (bf16)e.u;
      }
      in_order();
      take2(1);
      ta = mfma16(fa, ones, ta);
      tb = mfma16(fb, ones, tb);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        ga[c] = mfma16(fa, tx8[c & 1], ga[c]);
        gb[c] = mfma16(fb, tx8[c & 1], gb[c]);
        gs[c] = mfma16(fu, ty8[c & 1], gs[c]);
        in_order();
        if (c + 2 < CT) take2(c + 2);
      }
    }
    b = b + 1 == NB ? 0 : b + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the transfers past the end
  if (!own) return;
  float* to = G + (int64_t)at_.split * 3 * H * D + (int64_t)h0 * D;
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int at = (4 * q + r) * D + 16 * c + li;
#pragma unroll
      for (int m = 0; m < 3; ++m) {
        float* p = to + (int64_t)m * H * D + at;
        const float v = m == 0 ? ga[c][r] : m == 1 ? gb[c][r] : gs[c][r];
        *p = add ? *p + v : v;
      }
    }
  if (li == 0) {
    float* p = sums + (int64_t)at_.split * 2 * H + h0 + 4 * q;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      p[r] = add ? p[r] + ta[r] : ta[r];
      p[H + r] = add ? p[H + r] + tb[r] : tb[r];
    }
  }
}

// E as hidden_grad makes it, for 256 channels and many rows (40000 rows x 512: 58 us, 0.54 PFLOP/s, 123 MB of E at 2.1 TB/s:
// the matrix cores are busy 27% of the cycles, the elementwise part and the stores take turns with them, and the wait for a
// block's rows, which counts the stores, leaves half a block of rows on its way; 20000 rows: hidden_grad 74, here 49): as
// above a wave keeps its operands of Aw, Bw and S^T of 16 hidden channels in registers (12 D / 32 of them) and the rows
// stream by through LDS, D = hidden x rows (a lane holds a row at 4 hidden channels). grid (ceil(H / 128), splits); block
// 512.
template <int D>
__global__ __launch_bounds__(512, 2) void hidden_stream(const f16* __restrict__ xh, const bf16* __restrict__ dy,
                                                        const f16* __restrict__ aw, const bf16* __restrict__ st,
                                                        const float* __restrict__ shift, const float* __restrict__ scale,
                                                        bf16* __restrict__ E, int64_t rows, int H) {
  constexpr int KK = D / 32, NB = 4, U = D / 128;  // U: a wave's KBs of its 4 rows of an array
  constexpr uint32_t kTile = 32 * D * sizeof(bf16);
  __shared__ __attribute__((aligned(256))) bf16 buf[NB][2][32 * D];  // xh fp16, dy
  const RowsAt at_ = rows_at_of();
  const int lane = threadIdx.x & 63, q = lane >> 4, li = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h0 = at_.group * 128 + 16 * wave;
  const bool own = h0 < H;
  const int hr = own ? h0 + li : li;
  const uint32_t lds = lds_addr(buf), rows_at = 2 * off_row<D>(li, q);
  const int64_t blocks = (rows + 31) / 32;
  // piece u of the wave's 4 rows: its row's and its own place, in bytes (rows past the end: the last one again)
  uint32_t lane_row[U], lane_piece[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = 64 * u + lane, r = i / (D / 8);
    lane_row[u] = 2 * D * r;
    lane_piece[u] = 16 * ((i % (D / 8)) ^ swz<D>(4 * wave + r));
  }
  auto fetch = [&](int64_t block, int b) __attribute__((always_inline)) {
    const int64_t row = (block < blocks ? block : blocks - 1) * 32 + 4 * wave, from = row < rows ? row : rows - 1;
    const uint32_t most = rows - 1 - from < 4 ? 2 * D * (uint32_t)(rows - 1 - from) : 8u * D;
    const uint32_t at = lds + 2 * kTile * b + 8 * D * wave;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t off = (lane_row[u] < most ? lane_row[u] : most) + lane_piece[u];
      dma16(xh + from * D, off, at + 1024 * u);
      dma16(dy + from * D, off, at + kTile + 1024 * u);
    }
  };
  f16x8 wa[KK], wb[KK];
  bf16x8 ws[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    wa[kk] = ld8h(aw + (int64_t)hr * D + 32 * kk + 8 * q);
    wb[kk] = ld8h(aw + (int64_t)(H + hr) * D + 32 * kk + 8 * q);
    ws[kk] = ld8(st + (int64_t)hr * D + 32 * kk + 8 * q);
  }
  const int hq = own ? h0 + 4 * q : 4 * q;
  const f32x4 oa = *reinterpret_cast<const f32x4*>(shift + hq), ob = *reinterpret_cast<const f32x4*>(shift + H + hq);
  const f32x4 ia = *reinterpret_cast<const f32x4*>(scale + hq);
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) asm volatile("" ::"v"(wa[kk]), "v"(wb[kk]), "v"(ws[kk]));
  asm volatile("" ::"v"(oa), "v"(ob), "v"(ia));
  const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int b = 0; b < NB - 1; ++b) fetch(at_.split + (int64_t)b * at_.splits, b);
  int b = 0;
#pragma unroll 1
  for (int64_t block = at_.split; block < blocks; block += at_.splits) {
    // This block has landed. The count takes the stores in too: from the second block on, what stays on its way in a wave
    // that owns channels is the last block's 6 stores and 2 of the transfers issued in it (a wave that owns none, and the
    // first block, leave two blocks of 2 U transfers).
    wait_vm_lds<(NB - 2) * 2 * U>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const uint32_t tile = lds + 2 * kTile * b + rows_at;
    f32x4 a[2], bb[2], du[2];
    f16x8 lx[2][2];
    bf16x8 ly[2][2];
    auto take = [&](int kk) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t p = (tile ^ ((kk & 3) << 6)) + 256 * (kk >> 2) + 32 * D * t;
        lx[kk & 1][t] = lds_at<f16x8>(p);
        ly[kk & 1][t] = lds_at<bf16x8>(p + kTile);
      }
      in_order();
    };
    take(0);
    fetch(block + (int64_t)(NB - 1) * at_.splits, b == 0 ? NB - 1 : b - 1);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      if (kk + 1 < KK) take(kk + 1);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        a[t] = mfma16h(wa[kk], lx[kk & 1][t], kk ? a[t] : oa);
        bb[t] = mfma16h(wb[kk], lx[kk & 1][t], kk ? bb[t] : ob);
        du[t] = mfma16(ws[kk], ly[kk & 1][t], kk ? du[t] : zero4);
      }
      in_order();
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      bf16x4 o[3];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const SwigluGrad e = swiglu_grad(a[t][r], bb[t][r], du[t][r], -kLog2e * ia[r], ia[r]);
        o[0][r] = (bf16)e.da;
        o[1][r] = (bf16)e.db;
        o[2][r] = (bf16)e.u;
      }
      const int64_t row = block * 32 + 16 * t + li;
      if (own && row < rows) {
        bf16* to = E + row * 3 * H + h0 + 4 * q;
#pragma unroll
        for (int m = 0; m < 3; ++m) *reinterpret_cast<bf16x4*>(to + m * H) = o[m];
      }
    }
    b = b + 1 == NB ? 0 : b + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the transfers past the end
}

// dx. A wave owns 32 rows: its operands xh and dy and the sums dxh^T (D x 32 fp32) stay in registers while the weights
// stream by in chunks of 32 hidden channels, double-buffered by LDS DMA and shared by the workgroup's D / 16
// waves. Per chunk: a', b', du as D = hidden x rows (a lane holds a row at 16 hidden channels), and da', db'
// rounded are directly the operand [hidden x rows] of dxh^T = Aw^T da' + Bw^T db' (abt packed in that order of k).
// The offset comes in by one more product step: three bf16 parts of it (24 bits) times ones. At the end the sums over
// channels of the norm's backward pass are a lane's own registers and its partner's (lane ^ 32). 262144 rows x 128 x 512:
// 210 us, 0.82 PFLOP/s, the matrix cores busy in 52% of the cycles; without the elementwise part it would take 180, without
// the transfers too 150: the products, fed by one LDS read each, and the two waves of a SIMD that share it.
// grid: persistent; block 64 NW, NW = D / 16.
template <int D>
struct GradChunk {
  f16 wa[32 * D], wb[32 * D];   // rows h0 .. h0 + 31 (swizzled)
  bf16 ws[32 * D];
  bf16 at[D * 32], bt[D * 32];  // channel rows, the chunk's 32 hidden channels (pieces swizzled)
};
// piece p (of 4) of row r of a 32-wide tile
__device__ __forceinline__ int off_narrow(int r, int p) { return r * 32 + 8 * (p ^ ((r >> 2) & 3)); }

template <int D>
__global__ __launch_bounds__(4 * D, 2) void transition_grad_rows(
    const f16* __restrict__ xh, const bf16* __restrict__ dy, const float* __restrict__ rstd_in,
    const f16* __restrict__ aw, const bf16* __restrict__ st, const bf16* __restrict__ abt,
    const bf16* __restrict__ split, bf16* __restrict__ dx, int64_t rows, int H, int residual) {
  constexpr int NW = D / 16, KK = D / 16, CT = D / 32, P = D / 8;
  __shared__ __attribute__((aligned(256))) GradChunk<D> W[2];
  extern __shared__ __attribute__((aligned(16))) bf16 off_lds[];  // [2][H][8]: the offsets' parts and 2^-ka
  const int lane = threadIdx.x & 63, g = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t lds = lds_addr(W);
  const int chunks = H / 32;
  const uint32_t rows_at = 2 * off_row<D>(li, g), narrow_at = 2 * off_narrow(li, g);  // a lane's places in a chunk
  for (int i = threadIdx.x; i < 2 * H; i += 64 * NW)
    *reinterpret_cast<bf16x8*>(off_lds + 8 * i) = ld8(split + 8 * (int64_t)i);
  // a wave's transfers of a chunk, one KB of each of its five arrays (u = 0 .. 4)
  const int r0 = wave * (512 / D), cr = lane >> 2;
  const uint32_t w_off = kb_offset<D>(r0, lane);
  const uint32_t t_off = 4 * H * cr + 16 * ((lane & 3) ^ ((cr >> 2) & 3));  // 16 channel rows of 2 H values
  auto fetch = [&](int c, int b, int u) __attribute__((always_inline)) {
    const uint32_t at = lds + b * sizeof(GradChunk<D>) + u * 64 * D + 1024 * wave;
    const int64_t row = 32 * c + r0;
    if (u == 0) dma16(aw + row * D, w_off, at);
    if (u == 1) dma16(aw + (H + row) * D, w_off, at);
    if (u == 2) dma16(st + row * D, w_off, at);
    if (u >= 3) dma16(abt + (int64_t)16 * wave * 2 * H + (u == 4 ? H : 0) + 32 * c, t_off, at);
  };
  bf16x8 ones;  // the offsets' operand: 1 at the first three k
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (bf16)(g == 0 && e < 3 ? 1.f : 0.f);
  const int64_t tiles = (rows + 32 * NW - 1) / (32 * NW);
#pragma unroll
  for (int u = 0; u < 5; ++u) fetch(0, 0, u);
  int b = 0;
#pragma unroll 1
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t row = tile * 32 * NW + 32 * wave + li;
    const int64_t rc = row < rows ? row : rows - 1;  // rows past the end: the last one again, never stored
    f16x8 xb[KK];
    bf16x8 yb[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      xb[kk] = ld8h(xh + rc * D + 16 * kk + 8 * g);
      yb[kk] = ld8(dy + rc * D + 16 * kk + 8 * g);
    }
    const float rstd = rstd_in[rc];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) asm volatile("" ::"v"(xb[kk]), "v"(yb[kk]));
    asm volatile("" ::"v"(rstd));
    f32x16 acc[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c] = zero16();
    uint32_t touched[2] = {0, 0};
#pragma unroll 1
    for (int c = 0; c < chunks; ++c, b ^= 1) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();  // the chunk is whole; the other buffer has been read
      asm volatile("" ::: "memory");
      // the next chunk's transfers are spread over this one (all at once, the waves waited for the queue they fill)
      const int ahead = c + 1 == chunks ? 0 : c + 1;  // (wraps into the next tile)
      const uint32_t at = lds + b * sizeof(GradChunk<D>);
      const uint32_t rows_a = at + rows_at, narrow_a = at + 192 * D + narrow_at;
      f32x16 a = zero16(), bb = zero16(), du = zero16();
      a = mfma32(ld8(off_lds + 8 * (32 * c + li)), ones, a);
      bb = mfma32(ld8(off_lds + 8 * (H + 32 * c + li)), ones, bb);
      const float ia = (float)off_lds[8 * 32 * c + 3], slow = -kLog2e * ia;
      f16x8 la[2], lb[2];
      bf16x8 ls[2], lt[2][2];
      auto take = [&](int kk) __attribute__((always_inline)) {
        const uint32_t p = rows_a ^ (kk << 5);
        la[kk & 1] = lds_at<f16x8>(p);
        lb[kk & 1] = lds_at<f16x8>(p + 64 * D);
        ls[kk & 1] = lds_at<bf16x8>(p + 128 * D);
        in_order();
      };
      // i = 0 .. 2 CT - 1: half s of the hidden channels, Aw^T or Bw^T, two channel tiles
      auto take2 = [&](int i) __attribute__((always_inline)) {
        const uint32_t p = (narrow_a ^ (32 * (i / CT))) + 64 * D * (i / (CT / 2) % 2) + 2048 * (2 * i % CT);
        lt[i & 1][0] = lds_at<bf16x8>(p);
        lt[i & 1][1] = lds_at<bf16x8>(p + 2048);
        in_order();
      };
      take(0);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if (kk % (KK / 4) == 0) fetch(ahead, b ^ 1, kk / (KK / 4));
        if (kk + 1 < KK)
          take(kk + 1);
        else
          take2(0);
        a = mfma32h(la[kk & 1], xb[kk], a);
        bb = mfma32h(lb[kk & 1], xb[kk], bb);
        du = mfma32(ls[kk & 1], yb[kk], du);
        in_order();
      }
      fetch(ahead, b ^ 1, 4);
      if (c == chunks / 2) {
        // a value of each line of the next tile's rows: they come into the cache under this tile's products (all tiles
        // start at once, and waiting for their rows took 40 of 230 us)
        constexpr int L = D / 64;  // 128-byte lines of a row
        const int64_t r = (tile + gridDim.x) * 32 * NW + 32 * wave + lane / L % 32;
        const int64_t at = (r < rows ? r : rows - 1) * D + 64 * (lane % L);
        touched[0] = *reinterpret_cast<const uint32_t*>(xh + at);
        touched[1] = *reinterpret_cast<const uint32_t*>(dy + at);
      }
      bf16x8 fa[2], fb[2];
      auto elements = [&](int s) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const SwigluGrad e = swiglu_grad(a[8 * s + r], bb[8 * s + r], du[8 * s + r], slow, ia);
          fa[s][r] = (bf16)e.da;
          fb[s][r] = (bf16)e.db;
        }
      };
      auto second = [&](int i) __attribute__((always_inline)) {
        const int s = i / CT, m = i / (CT / 2) % 2, ct = 2 * i % CT;
        acc[ct] = mfma32(lt[i & 1][0], m ? fb[s] : fa[s], acc[ct]);
        acc[ct + 1] = mfma32(lt[i & 1][1], m ? fb[s] : fa[s], acc[ct + 1]);
      };
      elements(0);
      elements(1);
      in_order();
#pragma unroll
      for (int i = 0; i < 2 * CT; ++i) {
        if (i + 1 < 2 * CT) take2(i + 1);
        second(i);
        in_order();
      }
    }
    asm volatile("" ::"v"(touched[0]), "v"(touched[1]));
    // dxh^T: acc[ct] register 4 v + e holds channel 32 ct + 8 v + 4 g + e. xh and dy in the same places: a lane holds
    // 8 channels 16 kk + 8 g .. of them; its halves and its partner's are exchanged.
    float sg = 0.f, sx = 0.f;
    float xv[KK][8];  // channels 16 kk + 4 g + 0..3, 16 kk + 8 + 4 g + 0..3
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      union {
        f16x8 h;
        uint32_t u[4];
      } q;
      q.h = xb[kk];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const auto sw = __builtin_amdgcn_permlane32_swap(q.u[t], q.u[2 + t], false, false);
        q.u[t] = sw[0];
        q.u[2 + t] = sw[1];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xv[kk][e] = (float)q.h[e];
        const float t = acc[kk >> 1][8 * (kk & 1) + e];
        sg += t;
        sx += t * xv[kk][e];
      }
    }
    const float c1 = pair_sum(sg) * (1.f / D), c2 = pair_sum(sx) * (1.f / D);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      union {
        bf16x8 v;
        uint32_t u[4];
      } q;
      q.v = yb[kk];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const auto sw = __builtin_amdgcn_permlane32_swap(q.u[t], q.u[2 + t], false, false);
        q.u[t] = sw[0];
        q.u[2 + t] = sw[1];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        q.v[e] = (bf16)((residual ? (float)q.v[e] : 0.f) + rstd * (acc[kk >> 1][8 * (kk & 1) + e] - c1 - xv[kk][e] * c2));
      // back to whole pieces (the exchange is its own inverse)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const auto sw = __builtin_amdgcn_permlane32_swap(q.u[t], q.u[2 + t], false, false);
        q.u[t] = sw[0];
        q.u[2 + t] = sw[1];
      }
      if (row < rows) *reinterpret_cast<bf16x8*>(dx + row * D + 16 * kk + 8 * g) = q.v;
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the transfers past the last chunk
}

// dx = (residual ? dy : 0) + rstd (g - mean(g) - xh mean(g xh)), g the sum of `splits` fp32 parts [rows][d]: a wave a row
// (from row `first` in steps), K = d / 64 channels a lane. 40000 rows of 256: 18 us, 5.6 TB/s.
template <int K>
__device__ __forceinline__ void norm_grad(int64_t first, int64_t step, const f16* __restrict__ xh,
                                          const float* __restrict__ rstd_in, const bf16* __restrict__ dy,
                                          const float* __restrict__ dxh, int splits, int64_t split_stride,
                                          bf16* __restrict__ dx, int64_t rows, int residual) {
  constexpr int d = 64 * K;
  for (int64_t row = first; row < rows; row += step) {
    const int64_t at = row * d + (threadIdx.x & 63);
    float t[K], h[K], y[K];
    float sg = 0.f, sx = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      h[k] = (float)xh[at + 64 * k];
      y[k] = residual ? (float)dy[at + 64 * k] : 0.f;
      t[k] = 0.f;
    }
    const float rstd = rstd_in[row];
    // (some parts' values are on their way together; the parts' order is fixed)
#pragma unroll 4
    for (int i = 0; i < splits; ++i) {
#pragma unroll
      for (int k = 0; k < K; ++k) t[k] += dxh[i * split_stride + at + 64 * k];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      sg += t[k];
      sx += t[k] * h[k];
    }
    const float c1 = lanes_sum<64>(sg) * (1.f / d), c2 = lanes_sum<64>(sx) * (1.f / d);
#pragma unroll
    for (int k = 0; k < K; ++k) dx[at + 64 * k] = (bf16)(y[k] + rstd * (t[k] - c1 - h[k] * c2));
  }
}
template <int K>
__global__ __launch_bounds__(64) void norm_grad_rows(const f16* __restrict__ xh, const float* __restrict__ rstd,
                                                     const bf16* __restrict__ dy, const float* __restrict__ dxh,
                                                     int splits, int64_t split_stride, bf16* __restrict__ dx,
                                                     int64_t rows, int residual) {
  norm_grad<K>(blockIdx.x, gridDim.x, xh, rstd, dy, dxh, splits, split_stride, dx, rows, residual);
}
// Few rows: dx, and the affine's gradients from grad_products' parts [count][2 d], in one launch: the first d / 8
// workgroups sum 16 columns each (a thread every 16th part in order, then the 16 sums in order), the others take 4 rows.
// block 256. 100 rows of 384, 48 parts: 5 us, where two launches took 5 and 4.
template <int K>
__global__ __launch_bounds__(256) void finish_rows(const f16* __restrict__ xh, const float* __restrict__ rstd,
                                                   const bf16* __restrict__ dy, const float* __restrict__ dxh, int splits,
                                                   int64_t split_stride, bf16* __restrict__ dx, int64_t rows, int residual,
                                                   const float* __restrict__ part, int count, void* dln_w, void* dln_b,
                                                   int dtype) {
  constexpr int d = 64 * K, sums = d / 8;
  __shared__ float red[16][17];
  const int block = blockIdx.x;
  if (block >= sums) {
    norm_grad<K>(4 * (int64_t)(block - sums) + (threadIdx.x >> 6), 4 * (int64_t)(gridDim.x - sums), xh, rstd, dy, dxh,
                 splits, split_stride, dx, rows, residual);
    return;
  }
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4, c = 16 * block + col;
  float s = 0.f;
#pragma unroll 8
  for (int k = row; k < count; k += 16) s += part[(int64_t)k * 2 * d + c];
  red[row][col] = s;
  __syncthreads();
  if (threadIdx.x < 16) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += red[k][col];
    put_grad(c < d ? dln_w : dln_b, c < d ? c : c - d, s, dtype);
  }
}

// The weights' gradients from `count` parts G [3 H][d] (da'^T xh, db'^T xh, u'^T dy) and sums [2 H] (of da', db'), and
// eight hidden channels' shares of the affine's: part [2 H / 8][2][d]. A workgroup: 32 channels x 8 hidden channels, in Q
// shares of the parts (0, Q, 2 Q, ..; joined in LDS in that order). grid (d / 32, 3 H / 8); block 256 Q. 64 parts of
// 1536 x 128: 12 us, 50 MB at 4.3 TB/s.
template <int Q>
__global__ __launch_bounds__(256 * Q) void join_weight_grads(const float* __restrict__ G, const float* __restrict__ sums,
                                                          int count, const float* __restrict__ wa,
                                                          const float* __restrict__ wb, const float* __restrict__ w,
                                                          const float* __restrict__ v, const float* __restrict__ scale,
                                                          float* __restrict__ part, int d, int H, void* da, void* db,
                                                          void* ds, int dtype) {
  __shared__ float share[2][Q][8][33], tile[2][8][33];
  const int c0 = blockIdx.x * 32, h0 = blockIdx.y * 8;
  const int col = threadIdx.x & 31, row = (threadIdx.x >> 5) & 7, quarter = threadIdx.x >> 8;
  const int64_t size = (int64_t)3 * H * d;
  const bool summed = h0 < 2 * H;
  const float* p = G + (int64_t)(h0 + row) * d + c0 + col;
  float t = 0.f, total = 0.f;
#pragma unroll 8
  for (int k = quarter; k < count; k += Q) t += p[k * size];
  if (summed && col < 4) {  // (the sums' parts: a share over four lanes)
#pragma unroll 4
    for (int k = quarter + Q * col; k < count; k += 4 * Q) total += sums[(int64_t)k * 2 * H + h0 + row];
  }
  share[0][quarter][row][col] = t;
  share[1][quarter][row][col] = total;
  __syncthreads();
  if (quarter) return;
  t = 0.f;
#pragma unroll
  for (int i = 0; i < Q; ++i) t += share[0][i][row][col];
  if (!summed) {
    // 8 hidden channels of a row of dS: 16 or 32 bytes
    const int h = h0 - 2 * H + row;
    put_grad(ds, (int64_t)(c0 + col) * H + h, count ? unscale_both(t, scale[h], scale[H + h]) : 0.f, dtype);
    return;
  }
  total = 0.f;
#pragma unroll
  for (int i = 0; i < 4 * Q; ++i) total += share[1][i >> 2][row][i & 3];
  const bool first = h0 < H;
  const int h = h0 + row - (first ? 0 : H);
  const float back = count ? scale[first ? H + h : h] : 0.f;
  t *= back;
  total *= back;
  const int64_t at = (int64_t)h * d + c0 + col;
  put_grad(first ? da : db, at, t * w[c0 + col] + total * v[c0 + col], dtype);
  const float own = (first ? wa : wb)[at];
  tile[0][row][col] = own * t;
  tile[1][row][col] = own * total;
  __syncthreads();
  if (threadIdx.x < 64) {
    const int which = threadIdx.x >> 5;
    float r = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) r += tile[which][k][col];
    part[((int64_t)blockIdx.y * 2 + which) * d + c0 + col] = r;
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// weights: with the weights (a call's first chunk).
template <bool CODES>
void run_norm_rows(const TransitionGradArgs& a, const void* x, const uint8_t* scales, int64_t rows, bool weights,
                   bool fused, const WeightArgs& q, hipStream_t st) {
  const int extra = !weights ? 0 : q.H / (fused ? kPackGroup<true> : kPackGroup<false>) + q.H / 32 * (q.d / 32);
  const dim3 grid((unsigned)(extra + std::min<int64_t>(ceil_div(rows, 32), (int64_t)cu_count() * 16)));
  const auto run = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(x, scales, a.xh, a.xhb, a.rstd, rows, a.eps, extra, q); };
  if (fused) return a.d == 64 ? run(norm_rows<CODES, 1, true>) : run(norm_rows<CODES, 2, true>);
  switch (a.d / 64) {
#define FFK_K(K_) \
  case K_:        \
    return run(norm_rows<CODES, K_, false>);
    FFK_K(1) FFK_K(2) FFK_K(3) FFK_K(4) FFK_K(5) FFK_K(6) FFK_K(7) FFK_K(8) FFK_K(9) FFK_K(10) FFK_K(11) FFK_K(12)
#undef FFK_K
  }
}

void run_norm_grad_rows(const TransitionGradArgs& a, const bf16* dy, int splits, int64_t split_stride, bf16* dx,
                        int64_t rows, hipStream_t st) {
  const dim3 grid((unsigned)std::min<int64_t>(rows, (int64_t)cu_count() * 64));
  switch (a.d / 64) {
#define FFK_K(K_)                                                                                                 \
  case K_:                                                                                                        \
    norm_grad_rows<K_><<<grid, 64, 0, st>>>(a.xh, a.rstd, dy, a.dxh, splits, split_stride, dx, rows, a.residual); \
    break;
    FFK_K(1) FFK_K(2) FFK_K(3) FFK_K(4) FFK_K(5) FFK_K(6) FFK_K(7) FFK_K(8) FFK_K(9) FFK_K(10) FFK_K(11) FFK_K(12)
#undef FFK_K
  }
}

void run_finish_rows(const TransitionGradArgs& a, int splits, int64_t split_stride, int64_t rows, hipStream_t st) {
  const dim3 grid((unsigned)(a.d / 8 + std::min<int64_t>(ceil_div(rows, 4), (int64_t)cu_count() * 16)));
  switch (a.d / 64) {
#define FFK_K(K_)                                                                                                     \
  case K_:                                                                                                            \
    finish_rows<K_><<<grid, 256, 0, st>>>(a.xh, a.rstd, a.dy, a.dxh, splits, split_stride, a.dx, rows, a.residual,    \
                                          a.norm_part, 2 * a.hidden / 64, a.dln_w, a.dln_b, a.grad_dtype);            \
    break;
    FFK_K(1) FFK_K(2) FFK_K(3) FFK_K(4) FFK_K(5) FFK_K(6) FFK_K(7) FFK_K(8) FFK_K(9) FFK_K(10) FFK_K(11) FFK_K(12)
#undef FFK_K
  }
}

// Widths the fused kernels take: their offsets and two weight chunks within the 160 KB of LDS.
bool fused_shape(int d, int H) { return (d == 64 || d == 128) && H <= 2048; }

template <int D>
size_t grad_rows_lds(int H) { return (size_t)2 * H * 8 * sizeof(bf16); }

template <int D>
void launch_fused(const TransitionGradArgs& a, const TransitionGradPlan& p, const bf16* dy, bf16* dx, int64_t rows,
                  int add, hipStream_t st) {
  constexpr int NW = D / 16;
  const int H = a.hidden;
  const auto rows_kernel = transition_grad_rows<D>;
  const int held = resident_blocks(reinterpret_cast<const void*>(rows_kernel), 64 * NW, grad_rows_lds<D>(H));
  const int64_t tiles = ceil_div(rows, 32 * NW);
  rows_kernel<<<dim3((unsigned)std::min<int64_t>(tiles, (int64_t)cu_count() * held)), 64 * NW, grad_rows_lds<D>(H), st>>>(
      a.xh, dy, a.rstd, a.aw, a.st, a.abt, a.split, dx, rows, H, a.residual);
  transition_grad_weights<D><<<dim3((unsigned)ceil_div(H, 128), (unsigned)p.dw_splits), 512, 0, st>>>(
      a.xh, a.xhb, dy, a.aw, a.st, a.shift, a.scale, a.dw_part, a.sums, rows, H, add);
}

}  // namespace

TransitionGradPlan transition_grad_plan(int64_t rows, int d, int H) {
  TransitionGradPlan p{};
  const int64_t cus = cu_count();
  // Rows from which the fused kernels win (a workgroup walks all chunks of weights however few its rows; the separate ones
  // step up where their 64-row tiles come to one a CU). Separate kernels against fused ones, us, on both sides of the rule:
  // 128 x 128 channels 16384 rows 47 / 48, 16448 rows 53 / 49; 128 x 512 81 / 84 and 91 / 83; 128 x 1024 116 / 123 and (18432
  // rows) 131 / 126; 64 x 256 4096 rows 32.6 / 33.0, 4160 rows 34.2 / 32.9; 64 x 512 6144 rows 46.4 / 46.0, 8192 rows 50.4 /
  // 46.5, 4096 rows 39 / 45; 64 x 1024 8192 rows 62 / 65, 12288 rows 77 / 68; 64 x 64, 4096 rows 27 / 24, 2048 rows 25 / 23.
  p.fused = fused_shape(d, H) && (d == 128 ? rows > 16384 : rows >= (H <= 256 ? 4096 : 8192));
  if (p.fused) {
    p.chunk = std::min<int64_t>(ceil_div(rows, 64) * 64, 1 << 18);
    const int64_t groups = ceil_div(H, 128);
    // a workgroup a CU (its registers let no second one run beside it: 49152 rows x 64 x 256 in twice as many parts 60.5 us,
    // so 52.6), two stages each at least (4096 rows: one 35.5, two 33.6)
    p.dw_splits = (int)std::max<int64_t>(1, std::min<int64_t>(cus / groups, p.chunk / (2 * kStageRows)));
    return p;
  }
  // E of a chunk within 192 MB, so that much of it is still in the 256 MB last-level cache when the products read it, in
  // few chunks (40000 x 256 x 2: 222 us in one, 344 in two of 96 MB)
  const int64_t fit = std::max<int64_t>((int64_t)(192 << 20) / (6 * H) / 64 * 64, 64);
  p.chunk = std::min<int64_t>(ceil_div(rows, 64) * 64, fit);
  // both products want a workgroup a CU at least, and four steps of 64 in each; 128 x 128 tiles where they make so many
  p.dxh_wide = d % 128 == 0 && ceil_div(p.chunk, 128) * (d / 128) >= cus;
  const int64_t dxh_tiles = p.dxh_wide ? ceil_div(p.chunk, 128) * (d / 128) : p.chunk / 64 * (d / 64);
  p.dxh_splits = (int)std::max<int64_t>(1, std::min<int64_t>(cus / std::max<int64_t>(1, dxh_tiles), 2 * H / 256));
  // (64 x 64 against 128 x 128 tiles, us a call: 256 x 1024 channels 4096 rows 71 / 72, 8192 rows 104 / 97; 768 x 1536 180 / 178
  // and 319 / 292; 256 x 512, 2048 rows 42.5 / 44.6, 4096 rows 53.9 / 53.6. Where the small tiles need no join they hold out
  // to some 7000 rows: 384 x 1536 4096 rows 106 / 111, 8192 rows 180 / 177; 512 x 1024 91 / 100 and 176 / 157)
  p.dw_wide = d % 128 == 0 && H % 128 == 0 && p.chunk >= 4096;
  // (hidden_grad against hidden_stream, us a call, below the rule and above: 256 x 256 channels 16384 rows 77.0 / 77.7, 20000
  // rows 90 / 86; 256 x 512 8192 rows 71 / 72, 10240 rows 84.5 / 82.9; 256 x 1024 4096 rows 70 / 72, 6144 rows 86.3 / 85.9)
  p.stream = d == 256 && p.chunk >= 4096 && p.chunk * H >= 5000000;
  const int64_t dw_tiles = p.dw_wide ? 3 * H / 128 * (d / 128) : 3 * H / 64 * (d / 64);
  p.dw_splits = (int)std::max<int64_t>(1, std::min<int64_t>(2 * cus / std::max<int64_t>(1, dw_tiles), p.chunk / 256));
  // both products and the gradients' ends in two launches instead of five (100 rows x 384 x 4: 47 -> 34 us)
  p.few = rows > 0 && rows <= p.chunk && p.dw_splits == 1 && !p.dw_wide && !p.dxh_wide && !p.stream;
  return p;
}

void launch_transition_grad(const TransitionGradArgs& a, const TransitionGradPlan& p, hipStream_t st) {
  const int d = a.d, H = a.hidden;
  const char* x = static_cast<const char*>(a.x);
  for (int64_t r0 = 0; r0 < a.rows; r0 += p.chunk) {
    const int64_t rows = std::min(p.chunk, a.rows - r0);
    const void* xc = x + r0 * d * (a.scales ? 1 : 2);
    const bf16* dy = a.dy + r0 * d;
    const int add = r0 > 0;
    const WeightArgs w{a.wa, a.wb, a.ws, a.ln_w, a.ln_b, a.aw, a.st, a.abt, a.split, a.shift, a.scale, d, H};
    if (a.scales)
      run_norm_rows<true>(a, xc, a.scales + r0 * (d / kActBlock), rows, r0 == 0, p.fused, w, st);
    else
      run_norm_rows<false>(a, xc, nullptr, rows, r0 == 0, p.fused, w, st);
    if (p.fused) {
      if (d == 64)
        launch_fused<64>(a, p, dy, a.dx + r0 * d, rows, add, st);
      else
        launch_fused<128>(a, p, dy, a.dx + r0 * d, rows, add, st);
      continue;
    }
    if (p.stream) {
      const int64_t groups = ceil_div(H, 128);
      const dim3 grid((unsigned)groups, (unsigned)std::max<int64_t>(1, std::min(cu_count() / groups, ceil_div(rows, 32))));
      hidden_stream<256><<<grid, 512, 0, st>>>(a.xh, dy, a.aw, a.st, a.shift, a.scale, a.E, rows, H);
    } else {
      hidden_grad<<<dim3((unsigned)ceil_div(rows, 64), H / 64), 256, 0, st>>>(a.xh, dy, a.aw, a.st, a.shift, a.scale, a.E,
                                                                            rows, d, H);
    }
    Gemm64Args g{};
    g.A = a.E;
    g.lda = 3 * H;
    g.m_rows = rows;
    g.B = g.B2 = a.abt;
    g.ldb = 2 * H;
    g.k_rows = 2 * H;
    g.k_share = ceil_div(ceil_div(2 * H, p.dxh_splits), 64) * 64;
    g.C = a.dxh;
    g.ldc = d;
    g.split_stride = p.chunk * d;
    g.m_two = 0x7fffffff;
    g.m_tiles = (int)ceil_div(rows, 128);
    g.n_tiles = d / 128;
    Gemm64Args t{};
    t.A = a.E;
    t.lda = 3 * H;
    t.m_rows = 3 * H;
    t.B = a.xhb;
    t.B2 = dy;
    t.m_two = 2 * H / 64;
    t.ldb = d;
    t.k_rows = rows;
    t.k_share = ceil_div(ceil_div(p.chunk, p.dw_splits), 64) * 64;
    t.C = a.dw_part;
    t.ldc = d;
    t.split_stride = (int64_t)3 * H * d;
    t.sums = a.sums;
    t.sums_stride = 2 * H;
    t.add = add;
    t.m_tiles = 3 * H / 128;
    t.n_tiles = d / 128;
    if (p.few) {
      g.m_tiles = (int)ceil_div(rows, 64);
      g.n_tiles = d / 64;
      t.m_tiles = 3 * H / 64;
      t.n_tiles = d / 64;
      const WeightGradArgs q{a.wa, a.wb, a.ln_w, a.ln_b, a.scale, a.norm_part, a.dwa, a.dwb, a.dws, d, H, a.grad_dtype};
      const int tiles = t.m_tiles * t.n_tiles;
      grad_products<<<dim3((unsigned)(tiles + g.m_tiles * g.n_tiles * p.dxh_splits)), 256, 0, st>>>(t, q, g, tiles);
      run_finish_rows(a, p.dxh_splits, g.split_stride, rows, st);
      return;
    }
    if (p.dxh_wide)
      gemm128<false><<<dim3((unsigned)(g.m_tiles * g.n_tiles * p.dxh_splits)), 256, 0, st>>>(g);
    else
      gemm64<false><<<dim3((unsigned)ceil_div(rows, 64), d / 64, p.dxh_splits), 256, 0, st>>>(g);
    run_norm_grad_rows(a, dy, p.dxh_splits, g.split_stride, a.dx + r0 * d, rows, st);
    if (p.dw_wide)
      gemm128<true><<<dim3((unsigned)(t.m_tiles * t.n_tiles * p.dw_splits)), 256, 0, st>>>(t);
    else
      gemm64<true><<<dim3(3 * H / 64, d / 64, p.dw_splits), 256, 0, st>>>(t);
  }
  // (no rows: sums over nothing)
  const int parts = a.rows > 0 ? p.dw_splits : 0;
  const auto join = [&](auto kernel, int q) {
    kernel<<<dim3(d / 32, 3 * H / 8), 256 * q, 0, st>>>(a.dw_part, a.sums, parts, a.wa, a.wb, a.ln_w, a.ln_b, a.scale,
                                                       a.norm_part, d, H, a.dwa, a.dwb, a.dws, a.grad_dtype);
  };
  if (parts >= 32)  // (21 parts of 1536 x 256: 13.7 us in four shares, 9 in one)
    join(join_weight_grads<4>, 4);
  else
    join(join_weight_grads<1>, 1);
  launch_sum_partials(a.norm_part, a.rows > 0 ? 2 * H / 8 : 0, 2 * d, d, a.dln_w, a.dln_b, a.grad_dtype, st);
}

}  // namespace ffk
