// A projection with the low-rank adapters of many requests beside it, forward and backward:
//   y_t  = W x_t + b + s_a B_a (A_a x_t)          W [d_out][d_in], A_a [rank][d_in], B_a [d_out][rank]
//   dx_t = W^T dy_t + A_a^T v_t,  v_t = s_a B_a^T dy_t,  u_t = s_a A_a x_t
//   dA_a = sum over its rows of v_t x_t^T,  dB_a = sum over its rows of dy_t u_t^T
// a: the adapter of the request that row t belongs to (request r has the rows offsets[r] .. offsets[r + 1] - 1; rows of no
// request, and requests whose adapter is none of them, have W and b alone). W is frozen: no gradient.
//
// The thin products (u, v: d x rank) go first, into rows of rank numbers; the wide product then takes them as rank more
// channels of the same sum, so its rows are read and written once. Operands of the products are bf16, sums fp32. The
// adapters' gradients are fp32: u and v are kept as three bf16 that add up to the fp32 value, and fp32 adapters enter as
// three (the products of a bf16 pair are exact in fp32, three of them cost little beside the rows' way from memory). The
// outputs, bf16 themselves, take the rounded u and v and rounded weights.
// Rows of other adapters are left out by selection, not by factors of zero: infinities and NaN of one request (or of one
// adapter's weights) reach no other's rows or gradients.
#include <algorithm>
#include <type_traits>

#include "ffk_adapted.h"
#include "ffk_device.h"
#include "ffk_kernels.h"

namespace ffk {

namespace {

// ---------------------------------------------------------------------------------------------------------
// which adapter a row has

// id[i], i < 64: the adapter of row row0 + i, -1 for none (and behind the last row). All threads of the workgroup; start is
// scratch. The first wave passes over the offsets near the tile's rows: how many begin at or before the first row, and which
// begin at each of the others; then the latest request that begins at or before each row. Offsets out of order give some
// adapter or none, never an access out of range.
__device__ __forceinline__ void tile_ids(const Requests& q, int64_t row0, int* id, int* start) {
  const int tid = threadIdx.x;
  if (tid < 64) {
    start[tid] = -1;
    __builtin_amdgcn_wave_barrier();  // (the wave's own: LDS operations complete in order)
    int before = (int)offsets_near(q, row0, tid).from;
    for (int i0 = before + tid; i0 - tid <= q.count; i0 += 256) {
      int offset[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) offset[u] = q.offsets[i0 + 64 * u < q.count ? i0 + 64 * u : q.count];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 64 * u;
        const int64_t at = offset[u] - row0;
        before += __popcll(__ballot(i <= q.count && at <= 0));
        if (i <= q.count && at > 0 && at < 64) atomicMax(&start[at], i);
      }
      if (__ballot(offset[3] - row0 >= 64)) break;  // (the others begin behind the tile)
    }
    __builtin_amdgcn_wave_barrier();
    int r = tid == 0 ? before - 1 : start[tid];
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const int o = __shfl_up(r, m, 64);
      if (tid >= m && o > r) r = o;
    }
    int a = -1;
    if (r >= 0 && r < q.count && row0 + tid < q.rows) a = q.adapter[r];
    id[tid] = a >= 0 && a < q.adapters ? a : -1;
  }
  __syncthreads();
}

// Eight values at p[k ..], those from n on read as zeros. EVEN: n a multiple of 8 (the values lie in one 16- or 32-byte
// piece or none do): no branch, so that loads can run ahead of each other.
template <typename T, bool EVEN>
struct Raw8 {
  typedef T vec __attribute__((__vector_size__(8 * sizeof(T)), aligned(sizeof(T))));
  vec v;
  bool in;
  __device__ __forceinline__ void load(const T* p, int k, int n) {
    in = k < n;
    if constexpr (EVEN) {
      v = *reinterpret_cast<const vec*>(p + (in ? k : 0));
    } else if (k + 8 <= n) {
      v = *reinterpret_cast<const vec*>(p + k);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k + e < n ? p[k + e] : (T)0.f;
    }
  }
  // the same from a column: p[(k ..) * stride]
  __device__ __forceinline__ void load_column(const T* p, int k, int n, int stride) {
    in = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const T t = p[(int64_t)(k + e < n ? k + e : n - 1) * stride];
      v[e] = k + e < n ? t : (T)0.f;
    }
  }
  __device__ __forceinline__ float operator[](int e) const { return in ? (float)v[e] : 0.f; }
  __device__ __forceinline__ bf16x8 operand() const {
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = in ? (bf16)(float)v[e] : (bf16)0.f;
    return o;
  }
  // in so many bf16 that add up to it
  template <int PARTS>
  __device__ __forceinline__ void parts(bf16x8 (&o)[PARTS]) const {
    if constexpr (PARTS == 1) {
      o[0] = operand();
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float t = in ? (float)v[e] : 0.f;
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
          o[q][e] = (bf16)t;
          t -= (float)o[q][e];
        }
      }
    }
  }
};

// ---------------------------------------------------------------------------------------------------------
// operands in the products' orders

// dst [batch][out_rows][out_cols] bf16 from src [batch][rows][cols] (turn: transposed), zeros outside.
struct PackJob {
  const void* src;
  bf16* dst;
  int64_t rows, cols, out_rows, out_cols, tiles;  // tiles: of 32 x 32, all batches
  int f32, turn;
};
constexpr int kPackJobs = 5;
struct PackArgs {
  PackJob job[kPackJobs];
  int jobs;
  int64_t tiles;
};

// The 32 x 32 tiles of the destinations, the jobs' one after the other, from tile `first` on in steps.
__device__ __forceinline__ void pack_tiles(const PackArgs& p, int64_t first, int64_t step, float (&t)[32][33]) {
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  for (int64_t at = first; at < p.tiles; at += step) {
    int64_t tile = at;
    int which = 0;
    while (which + 1 < p.jobs && tile >= p.job[which].tiles) tile -= p.job[which++].tiles;
    const PackJob& j = p.job[which];
    const int64_t across = (j.out_cols + 31) / 32, down = (j.out_rows + 31) / 32;
    const int64_t c0 = tile % across * 32, r0 = tile / across % down * 32, batch = tile / across / down;
    const int64_t sr = j.turn ? c0 : r0, sc = j.turn ? r0 : c0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = sr + row + 8 * i, c = sc + col;
      float v = 0.f;
      if (r < j.rows && c < j.cols) {
        const int64_t from = (batch * j.rows + r) * j.cols + c;
        v = j.f32 ? static_cast<const float*>(j.src)[from] : (float)static_cast<const bf16*>(j.src)[from];
      }
      t[row + 8 * i][col] = v;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = r0 + row + 8 * i, c = c0 + col;
      if (r >= j.out_rows || c >= j.out_cols) continue;
      const float v = j.turn ? t[col][row + 8 * i] : t[row + 8 * i][col];
      const int64_t to = (batch * j.out_rows + r) * j.out_cols + c;
      j.dst[to] = (bf16)v;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------
// the thin products

// Channels of a row of u or v that keeps its parts: RP each of the high, middle and low ones (RP = 16: and of zeros), then none.
constexpr int parts_ld(int rp) { return rp == 16 ? 64 : rp == 32 ? 128 : 3 * rp; }

struct ThinJob {
  const bf16* x;    // [rows][K]
  const void* mat;  // the adapters' [adapters][rank][K], or (turned) [adapters][K][rank]
  bf16* u;          // [rows][ld]: s_a (matrix x) in RP channels, zeros from `rank` on
  int K, turned;
};
struct ThinArgs {
  ThinJob job[2];
  Requests q;
  int32_t* ids;  // [rows], written with the first job
  int rank;
  int64_t row_blocks;
  int share, jobs;  // workgroups: row_blocks x share x jobs
};

struct ThinLds {
  int id[64], start[64];
};

// 16 rows a workgroup of 4 waves, a quarter of K a wave (16 rows a wave over all of K leave the chip half empty with few rows
// and are no faster with many: 768 -> 768 of rank 48 in tiles 43 us against 30 at 4000 rows, 142 against 132 at 40000; the
// backward pass 407 against 311). Each adapter of the rows in turn, `share` workgroups share them; a lane holds a token and 4
// channels. Operands straight from the call's tensors. EVEN: K a multiple of 8. KEEP: u in three parts (rows of parts_ld; fp32
// adapters in three parts as well), else rounded (rows of RP).
template <typename TA, int RP, bool KEEP, bool EVEN>
__device__ __forceinline__ void thin_rows(const ThinArgs& p, int64_t block, ThinLds& lds, f32x4 (*red)[RP / 16][64]) {
  constexpr int PARTS = KEEP && sizeof(TA) == 4 ? 3 : 1;
  constexpr int N = RP / 16, TM = 16, U = N * PARTS <= 3 ? 6 : N * PARTS <= 6 ? 2 : 1;  // steps of k in flight
  constexpr int ld = KEEP ? parts_ld(RP) : RP;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row0 = block % p.row_blocks * TM;
  const int shared = (int)(block / p.row_blocks % p.share), which = (int)(block / p.row_blocks / p.share);
  const ThinJob& j = p.job[which];
  tile_ids(p.q, row0, lds.id, lds.start);
  if (shared == 0 && which == 0 && threadIdx.x < TM && row0 + threadIdx.x < p.q.rows)
    p.ids[row0 + threadIdx.x] = lds.id[threadIdx.x];
  const int64_t row = row0 + i;
  const int mine = lds.id[i];
  const bf16* x = j.x + (row < p.q.rows ? row : p.q.rows - 1) * j.K;
  auto store = [&](int n, const f32x4& v) __attribute__((always_inline)) {
    bf16x4 part[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float t = 16 * n + 4 * g + e < p.rank ? v[e] : 0.f;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        part[k][e] = (bf16)t;
        t -= (float)part[k][e];
      }
    }
    bf16* to = j.u + row * ld + 16 * n + 4 * g;
    *reinterpret_cast<bf16x4*>(to) = part[0];
    if constexpr (KEEP) {
      *reinterpret_cast<bf16x4*>(to + RP) = part[1];
      *reinterpret_cast<bf16x4*>(to + 2 * RP) = part[2];
      if constexpr (RP == 16) {
        const bf16x4 z = {(bf16)0.f, (bf16)0.f, (bf16)0.f, (bf16)0.f};
        *reinterpret_cast<bf16x4*>(to + 3 * RP) = z;
      }
    }
  };
  const f32x4 none = {0.f, 0.f, 0.f, 0.f};
  if (shared == 0 && mine < 0 && row < p.q.rows && wave == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) store(n, none);
  }
  uint64_t todo = __ballot(mine >= 0) & 0xffffu;
  for (int turn = 0; todo != 0; ++turn) {
    const int a = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    const bool is = mine == a;
    todo &= ~__ballot(is);
    if (turn % p.share != shared) continue;
    f32x4 acc[N], rest[N];
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] = rest[n] = none;
    const TA* m[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = 16 * n + i < p.rank ? 16 * n + i : p.rank - 1;
      m[n] = static_cast<const TA*>(j.mat) + (int64_t)a * p.rank * j.K + (j.turned ? r : (int64_t)r * j.K);
    }
    const float s = scale_of(p.q, a);
    // so many steps of k, all their operands asked for before the first product
    const auto steps = [&](int k, auto count) __attribute__((always_inline)) {
      constexpr int C = decltype(count)::value;
      Raw8<bf16, EVEN> xf[C];
      Raw8<TA, EVEN> mf[C][N];
#pragma unroll
      for (int c = 0; c < C; ++c) xf[c].load(x, k + 32 * c + 8 * g, j.K);
      if (j.turned) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int n = 0; n < N; ++n) mf[c][n].load_column(m[n], k + 32 * c + 8 * g, j.K, p.rank);
      } else {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int n = 0; n < N; ++n) mf[c][n].load(m[n], k + 32 * c + 8 * g, j.K);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const bf16x8 xv = xf[c].operand();
#pragma unroll
        for (int n = 0; n < N; ++n) {
          bf16x8 mv[PARTS];
          mf[c][n].template parts<PARTS>(mv);
#pragma unroll
          for (int q = 0; q < PARTS; ++q) {
            f32x4& to = q ? rest[n] : acc[n];
            to = mfma16(mv[q], xv, to);
          }
        }
      }
    };
    // (a wave's share of k in one piece: its steps share cache lines)
    const int all = (j.K + 31) / 32;
    int k = all * wave / 4;
    const int stop = all * (wave + 1) / 4;
    for (; k + U <= stop; k += U) steps(32 * k, std::integral_constant<int, U>());
    if constexpr (U > 3)
      if (k + 3 <= stop) {
        steps(32 * k, std::integral_constant<int, 3>());
        k += 3;
      }
    if constexpr (U > 1)
      for (; k < stop; ++k) steps(32 * k, std::integral_constant<int, 1>());
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) red[wave][n][lane] = PARTS > 1 ? parts_sum(acc[n], rest[n]) : acc[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (n % 4 == wave && is) store(n, (red[0][n][lane] + red[1][n][lane] + (red[2][n][lane] + red[3][n][lane])) * s);
  }
}

// What a call makes first, in one launch: the thin products, and (the workgroups behind theirs) the operands that the wide
// product reads from copies. block 256. 16 us before the backward pass of 2900 rows, 1536 -> 384 of rank 32; 8 to 9 for 1021 rows of
// 449 -> 384: latencies of few steps.
template <typename TA, int RP, bool KEEP, bool EVEN>
__global__ __launch_bounds__(256) void adapted_prepare(const ThinArgs t, const PackArgs p) {
  __shared__ union {
    struct {
      ThinLds lds;
      f32x4 red[4][RP / 16][64];
    } thin;
    float tile[32][33];
  } s;
  const int64_t blocks = t.row_blocks * t.share * t.jobs;
  if (blockIdx.x < blocks)
    thin_rows<TA, RP, KEEP, EVEN>(t, blockIdx.x, s.thin.lds, s.thin.red);
  else
    pack_tiles(p, blockIdx.x - blocks, gridDim.x - blocks, s.tile);
}

// ---------------------------------------------------------------------------------------------------------
// the wide product

struct ProductArgs {
  const bf16 *x, *w;  // [rows][K], [N][K], K a multiple of 64
  const bf16 *u, *b;  // [rows][ld], the adapters' [adapters][N][RP]
  const int32_t* ids;
  const float* bias;  // or null
  bf16* out;          // [rows][N]
  int64_t rows;
  int K, N, RP, ld, n_tiles;
};

// out = x W^T + u B_a^T + bias in TM rows x TN channels a workgroup, a quarter of them a wave: weight rows x token rows, so a
// lane holds a token. K in steps of 64 through STAGES buffers by LDS DMA. The adapters of a wave's 32 tokens one after the
// other at the end, each added to the lanes that have it. grid: m tiles x n tiles, the n tiles of an m tile neighbours (they
// share its rows in an XCD's L2).
template <int TM, int TN, int STAGES>
__device__ __forceinline__ void product_tile(const ProductArgs& p, uint32_t block, uint32_t blocks,
                                             bf16 (&buf)[STAGES][TM / 64 + TN / 64][64 * 64]) {
  constexpr int XT = TM / 64, WT = TN / 64, PER = 2 * (XT + WT);  // 64 x 64 tiles a step, transfers of a wave
  const int lane = threadIdx.x & 63, g = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  const uint32_t id = xcd_remap(block, blocks);
  const int64_t m0 = (int64_t)(id / p.n_tiles) * TM;
  const int n0 = (int)(id % p.n_tiles) * TN;
  const int steps = p.K / 64;
  const uint32_t lds = lds_addr(buf);
  auto fetch = [&](int step) __attribute__((always_inline)) {
    const uint32_t at = lds + step % STAGES * (XT + WT) * 8192;
#pragma unroll
    for (int t = 0; t < XT; ++t) tile_dma(p.x + 64 * step, p.K, m0 + 64 * t, p.rows - 1, 0, at + 8192 * t, wave, lane);
#pragma unroll
    for (int t = 0; t < WT; ++t)
      tile_dma(p.w + 64 * step, p.K, n0 + 64 * t, p.N - 1, 0, at + 8192 * (XT + t), wave, lane);
  };
  f32x16 acc[WT][XT];
#pragma unroll
  for (int c = 0; c < WT; ++c)
#pragma unroll
    for (int t = 0; t < XT; ++t) acc[c][t] = zero16();
  int ids[XT];  // (asked for ahead of the transfers)
#pragma unroll
  for (int x = 0; x < XT; ++x) {
    const int64_t row = m0 + wm * (TM / 2) + 32 * x + li;
    ids[x] = p.ids[row < p.rows ? row : p.rows - 1];
  }
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < steps) fetch(s);
  for (int s = 0; s < steps; ++s) {
    if (s + STAGES - 1 <= steps)
      wait_vm_lds<(STAGES - 2) * PER>();
    else
      wait_vm_lds<0>();
    __syncthreads();  // the step has landed; the buffer of the one before has been read
    if (s + STAGES - 1 < steps) fetch(s + STAGES - 1);
    const bf16(*t)[64 * 64] = buf[s % STAGES];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      bf16x8 fw[WT], fx[XT];
#pragma unroll
      for (int c = 0; c < WT; ++c) {
        const int r = wn * (TN / 2) + 32 * c + li;
        fw[c] = ld8(&t[XT + (r >> 6)][off64(r & 63, 2 * kk + g)]);
      }
#pragma unroll
      for (int c = 0; c < XT; ++c) {
        const int r = wm * (TM / 2) + 32 * c + li;
        fx[c] = ld8(&t[r >> 6][off64(r & 63, 2 * kk + g)]);
      }
#pragma unroll
      for (int c = 0; c < WT; ++c)
#pragma unroll
        for (int x = 0; x < XT; ++x) acc[c][x] = mfma32(fw[c], fx[x], acc[c][x]);
    }
  }
  const int nw = n0 + wn * (TN / 2);
#pragma unroll
  for (int x = 0; x < XT; ++x) {
    const int64_t row = m0 + wm * (TM / 2) + 32 * x + li;
    const bool real = row < p.rows;
    const int mine = real ? ids[x] : -1;
    const bf16* u = p.u + (real ? row : p.rows - 1) * p.ld + 8 * g;
    uint64_t todo = __ballot(mine >= 0) & 0xffffffffu;
    while (todo != 0) {
      const int a = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
      todo &= ~__ballot(mine == a);
      f32x16 add[WT];
      const bf16* b[WT];
#pragma unroll
      for (int c = 0; c < WT; ++c) {
        add[c] = zero16();
        const int n = nw + 32 * c + li;
        b[c] = p.b + ((int64_t)a * p.N + (n < p.N ? n : p.N - 1)) * p.RP + 8 * g;
      }
      for (int j = 0; j < p.RP; j += 16) {
        const bf16x8 uf = ld8(u + j);
#pragma unroll
        for (int c = 0; c < WT; ++c) add[c] = mfma32(ld8(b[c] + j), uf, add[c]);
      }
#pragma unroll
      for (int c = 0; c < WT; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[c][x][r] += mine == a ? add[c][r] : 0.f;
    }
#pragma unroll
    for (int c = 0; c < WT; ++c) {
      float y[2][8];
      acc_pieces(acc[c][x], y);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int n = nw + 32 * c + 8 * (2 * k + g);
        if (!real || n >= p.N) continue;
        if (p.bias) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[k][e] += n + e < p.N ? p.bias[n + e] : 0.f;
        }
        bf16* to = p.out + row * p.N + n;
        if (p.N % 8 == 0) {
          bf16x8 v;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = (bf16)y[k][e];
          *reinterpret_cast<bf16x8*>(to) = v;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + e < p.N) to[e] = (bf16)y[k][e];
        }
      }
    }
  }
}

template <int TM, int TN, int STAGES>
__global__ __launch_bounds__(256, 2) void adapted_product(const ProductArgs p) {
  __shared__ __attribute__((aligned(16))) bf16 buf[STAGES][TM / 64 + TN / 64][64 * 64];
  product_tile<TM, TN, STAGES>(p, blockIdx.x, gridDim.x, buf);
}

// ---------------------------------------------------------------------------------------------------------
// the adapters' gradients

struct GradJob {
  const bf16 *x, *v;       // [rows][ld_x] (ld_x a multiple of 64), [rows][parts_ld]
  void* to;                // element (chunk, a, channel j, column c) at chunk * chunk_stride + (a * rank) * cols + j * sj + c * sc
  int64_t sj, sc;
  int cols, ld_x, tiles;   // tiles = ld_x / 64
};
struct GradArgs {
  GradJob job[2];
  const int32_t* ids;
  int64_t rows, chunk, chunk_stride[2];  // rows of a chunk: a multiple of 64, at most 64 * kMostGradTiles
  int rank, to_bf16, adapters;
};
constexpr int kMostGradTiles = 256;

// sum over a chunk's rows of adapter blockIdx.y of v x^T: RP channels x 64 columns a workgroup. Tiles of 64 rows that have a
// row of the adapter's, in order, through three buffers by LDS DMA; the rows of others in them are zeroed there. A wave takes
// 16 of a tile's rows (k of the product; both operands turned as they are read), the waves' sums meet at the end in a fixed
// order. The parts are products of their own, the high ones' sum apart from that of the others (RP = 16: high and middle ones
// the 32 rows of one product, low ones and zeros of another). Workgroups: both jobs' tiles x adapters x chunks.
template <int RP>
struct GradLds {
  static constexpr int VT = parts_ld(RP) / 64, STAGES = RP == 128 ? 2 : 3;
  __attribute__((aligned(16))) bf16 buf[STAGES][1 + VT][64 * 64];
  uint64_t has[kMostGradTiles];  // which rows of a tile are the adapter's
  int list[kMostGradTiles], listed;
};
template <int RP>
__device__ __forceinline__ void grad_tile(const GradArgs& p, int64_t block, GradLds<RP>& s_) {
  constexpr int ld = parts_ld(RP), VT = ld / 64, JB = RP <= 32 ? 1 : RP / 32, BLOCKS = RP == 16 ? 2 : 3 * RP / 32;
  constexpr int STAGES = GradLds<RP>::STAGES, PER = 2 * (1 + VT);
  auto& buf = s_.buf;
  auto& has = s_.has;
  auto& list = s_.list;
  int& listed = s_.listed;
  const int across = p.job[0].tiles + p.job[1].tiles, tile = (int)(block % across);
  const int a = (int)(block / across % p.adapters);
  const int64_t chunk = block / across / p.adapters;
  const int lane = threadIdx.x & 63, g = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int which = tile >= p.job[0].tiles ? 1 : 0;
  const GradJob& j = p.job[which];
  const int c0 = 64 * (tile - (which ? p.job[0].tiles : 0));
  const int64_t begin = chunk * p.chunk, end = begin + p.chunk < p.rows ? begin + p.chunk : p.rows;
  const int tiles = (int)((end - begin + 63) / 64);
  for (int t0 = wave; t0 < tiles; t0 += 4 * 8) {  // eight tiles' ids in flight
    int id[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t row = begin + 64 * (t0 + 4 * u) + lane;
      id[u] = p.ids[row < end ? row : end - 1];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int t = t0 + 4 * u;
      const uint64_t m = __ballot(begin + 64 * t + lane < end && id[u] == a);
      if (lane == 0 && t < tiles) has[t] = m;
    }
  }
  __syncthreads();
  if (wave == 0) {
    int n = 0;
    for (int t0 = 0; t0 < tiles; t0 += 64) {
      const bool some = t0 + lane < tiles && has[t0 + lane] != 0;
      const uint64_t m = __ballot(some);
      if (some) list[n + __popcll(m & ((1ull << lane) - 1))] = t0 + lane;
      n += __popcll(m);
    }
    if (lane == 0) listed = n;
  }
  __syncthreads();
  const int steps = listed;
  const uint32_t lds = lds_addr(buf);
  auto fetch = [&](int step) __attribute__((always_inline)) {
    const uint32_t at = lds + step % STAGES * (1 + VT) * 8192;
    const int64_t row0 = begin + 64 * list[step];
    tile_dma(j.x, j.ld_x, row0, p.rows - 1, c0, at, wave, lane);
#pragma unroll
    for (int t = 0; t < VT; ++t) tile_dma(j.v, ld, row0, p.rows - 1, 64 * t, at + 8192 * (1 + t), wave, lane);
  };
  f32x16 acc[2][JB][2];
#pragma unroll
  for (int b = 0; b < JB; ++b) acc[0][b][0] = acc[0][b][1] = acc[1][b][0] = acc[1][b][1] = zero16();
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < steps) fetch(s);
  for (int s = 0; s < steps; ++s) {
    if (s + STAGES - 1 <= steps)
      wait_vm_lds<(STAGES - 2) * PER>();
    else
      wait_vm_lds<0>();
    __syncthreads();  // the tile has landed; the buffer of the one before has been read
    if (s + STAGES - 1 < steps) fetch(s + STAGES - 1);
    bf16(*t)[64 * 64] = buf[s % STAGES];
    const uint64_t rows = has[list[s]];
    if (~rows != 0) {
      bf16x8 z;
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = (bf16)0.f;
      for (int i = threadIdx.x; i < (1 + VT) * 64 * 8; i += 256)
        if (!(rows >> ((i >> 3) & 63) & 1u)) *reinterpret_cast<bf16x8*>(t[i >> 9] + 8 * (i & 511)) = z;
      __syncthreads();
    }
    bf16x8 x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) x[h] = ld_turned(t[0], 32 * h, 16 * wave, lane);
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {  // 32 channels each: the high parts, the middle, the low ones
      const bf16x8 v = ld_turned(t[1 + b / 2], 32 * (b & 1), 16 * wave, lane);
#pragma unroll
      for (int h = 0; h < 2; ++h) acc[b >= JB][b % JB][h] = mfma32(v, x[h], acc[b >= JB][b % JB][h]);
    }
  }
  constexpr int ROWS = RP == 16 ? 16 : 32;
  float* sum = reinterpret_cast<float*>(buf);  // [wave][ROWS][64]
#pragma unroll
  for (int b = 0; b < JB; ++b) {
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < ROWS / 2; ++r) {
        // (RP = 16: the middle parts' rows are 16 behind the high ones', eight registers on)
        const float rest = RP == 16 ? acc[0][b][h][(r + 8) & 15] + acc[1][b][h][r] : acc[1][b][h][r];
        sum[(wave * ROWS + acc_row(r, g)) * 64 + 32 * h + li] = parts_sum(acc[0][b][h][r], rest);
      }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * 64; i += 256) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) v += sum[w * ROWS * 64 + i];
      const int row = 32 * b + (i >> 6), c = c0 + (i & 63);
      if (row >= p.rank || c >= j.cols) continue;
      const int64_t at =
          chunk * p.chunk_stride[which] + (int64_t)a * p.rank * j.cols + row * j.sj + c * j.sc;
      if (p.to_bf16)
        static_cast<bf16*>(j.to)[at] = (bf16)v;
      else
        static_cast<float*>(j.to)[at] = v;
    }
  }
}

// The gradients, and (the first workgroups) dx where it is wanted: both go by the thin products alone. block 256.
template <int RP, int TM, int TN, int STAGES>
__global__ __launch_bounds__(256) void adapted_finish(const ProductArgs t, const GradArgs g, uint32_t product_blocks) {
  __shared__ union U {
    __attribute__((aligned(16))) bf16 buf[STAGES][TM / 64 + TN / 64][64 * 64];
    GradLds<RP> grad;
  } s;
  if (blockIdx.x < product_blocks)
    product_tile<TM, TN, STAGES>(t, blockIdx.x, product_blocks, s.buf);
  else
    grad_tile<RP>(g, blockIdx.x - product_blocks, s.grad);
}

struct JoinJob {
  const float* part;  // [chunks][adapters][rank][cols]
  void* to;
  int64_t sj, sc;     // as GradJob's
  int64_t count;      // adapters * rank * cols
  int cols;
};
struct JoinArgs {
  JoinJob job[2];
  int chunks, rank, to_bf16;
};

// The chunks' sums: 64 values a workgroup, four groups of chunks beside each other, joined in order. grid: ceil of both jobs'
// counts / 64; block 256.
__global__ __launch_bounds__(256) void adapted_join(const JoinArgs p) {
  __shared__ float sum[4][64];
  int64_t i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int64_t head = (p.job[0].count + 63) / 64 * 64;
  const int which = (int64_t)blockIdx.x * 64 >= head ? 1 : 0;
  const JoinJob& j = p.job[which];
  if (which) i -= head;
  float v = 0.f;
  if (i < j.count) {
#pragma unroll 8
    for (int k = threadIdx.x >> 6; k < p.chunks; k += 4) v += j.part[k * j.count + i];
  }
  sum[threadIdx.x >> 6][threadIdx.x & 63] = v;
  __syncthreads();
  if (threadIdx.x >= 64 || i >= j.count) return;
  v = (sum[0][threadIdx.x] + sum[1][threadIdx.x]) + (sum[2][threadIdx.x] + sum[3][threadIdx.x]);
  const int64_t c = i % j.cols, row = i / j.cols % p.rank, a = i / j.cols / p.rank;
  const int64_t at = a * p.rank * j.cols + row * j.sj + c * j.sc;
  if (p.to_bf16)
    static_cast<bf16*>(j.to)[at] = (bf16)v;
  else
    static_cast<float*>(j.to)[at] = v;
}

// ---------------------------------------------------------------------------------------------------------
// few rows

struct FewArgs {
  const bf16* x;
  const void *w, *down, *up;
  const float* bias;
  bf16* out;
  Requests q;
  float* u;      // [rows][rank]
  int32_t* ids;  // [rows]
  int K, N, rank;
};

// u of one row a workgroup in fp32, two channels a wave at a time, k across the lanes. grid rows; block 512. 2.7 us for one row
// of 384, 3.7 for 64 of 768 of rank 16: a chain of latencies (the ids, the row, the sum).
template <typename TA, bool EVEN>
__global__ __launch_bounds__(512) void adapted_few_thin(const FewArgs p) {
  __shared__ int id[64], start[64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  tile_ids(p.q, row, id, start);
  const int a = id[0];
  if (threadIdx.x == 0) p.ids[row] = a;
  if (a < 0) return;
  const TA* m = static_cast<const TA*>(p.down) + (int64_t)a * p.rank * p.K;
  const float s = scale_of(p.q, a);
  for (int j0 = 2 * wave; j0 < p.rank; j0 += 16) {
    const TA* mj[2] = {m + (int64_t)j0 * p.K, m + (int64_t)(j0 + 1 < p.rank ? j0 + 1 : j0) * p.K};
    float sum[2] = {0.f, 0.f};
    for (int k = 8 * lane; k < p.K; k += 1024) {
      Raw8<bf16, EVEN> x[2];
      Raw8<TA, EVEN> v[2][2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        x[c].load(p.x + row * p.K, k + 512 * c, p.K);
#pragma unroll
        for (int j = 0; j < 2; ++j) v[c][j].load(mj[j], k + 512 * c, p.K);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[j] += x[c][e] * v[c][j][e];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float v = lanes_sum<64>(sum[j]);
      if (lane == 0 && j0 + j < p.rank) p.u[row * p.rank + j0 + j] = s * v;
    }
  }
}

// 16 channels x 16 RT rows a workgroup, an eighth of k a wave, operands straight from memory; the adapters as dot products of
// rank terms, a thread for each output. grid (ceil(N / 16), ceil(rows / (16 RT))); block 512. 3.3 us for one row 384 -> 1536, 5.2
// for 64 rows 768 -> 768: W's way from memory and the join of the eighths.
template <typename TW, typename TA, int RT, bool EVEN>
__global__ __launch_bounds__(512) void adapted_few(const FewArgs p) {
  __shared__ float red[8][RT][16][20];  // [wave][..][token][channel], rows of 20: 16-byte stores without conflicts
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = 16 * blockIdx.x;
  const int64_t row0 = 16 * RT * (int64_t)blockIdx.y;
  // the output of this thread
  const int part = threadIdx.x >> 8, token = (threadIdx.x >> 4) & 15, c = threadIdx.x & 15, n = n0 + c;
  const int64_t row = row0 + 16 * part + token;
  const bool mine = part < RT && row < p.q.rows && n < p.N;
  const int a = mine ? p.ids[row] : -1;
  f32x4 acc[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const TW* w = static_cast<const TW*>(p.w) + (int64_t)(n0 + i < p.N ? n0 + i : p.N - 1) * p.K;
  const bf16* x[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int64_t r = row0 + 16 * t + i;
    x[t] = p.x + (r < p.q.rows ? r : p.q.rows - 1) * p.K;
  }
  constexpr int U = 3;
  for (int k = 32 * wave; k < p.K; k += 256 * U) {
    Raw8<TW, EVEN> wf[U];
    Raw8<bf16, EVEN> xf[U][RT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      wf[u].load(w, k + 256 * u + 8 * g, p.K);
#pragma unroll
      for (int t = 0; t < RT; ++t) xf[u][t].load(x[t], k + 256 * u + 8 * g, p.K);
    }
    __builtin_amdgcn_sched_barrier(0);  // (all of them asked for before the first product)
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < RT; ++t) acc[t] = mfma16(wf[u].operand(), xf[u][t].operand(), acc[t]);
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) *reinterpret_cast<f32x4*>(&red[wave][t][i][4 * g]) = acc[t];
  float sum = mine && p.bias ? p.bias[n] : 0.f;
  if (a >= 0) {
    const TA* b = static_cast<const TA*>(p.up) + ((int64_t)a * p.N + n) * p.rank;
    const float* u = p.u + row * p.rank;
    for (int j = 0; j < p.rank; j += 8) {
      Raw8<TA, false> v;
      Raw8<float, false> q;
      v.load(b, j, p.rank);
      q.load(u, j, p.rank);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += v[e] * q[e];
    }
  }
  __syncthreads();
  if (!mine) return;
  float y = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) y += red[k][part][token][c];
  p.out[row * p.N + n] = (bf16)(y + sum);
}

// ---------------------------------------------------------------------------------------------------------
// launches

template <typename TW, typename TA, bool EVEN>
void launch_few(const FewArgs& f, hipStream_t st) {
  const int64_t rows = f.q.rows;
  adapted_few_thin<TA, EVEN><<<dim3((unsigned)rows), 512, 0, st>>>(f);
  if (hipPeekAtLastError() != hipSuccess) return;  // (the next launch would index by ids that are not there)
  const unsigned across = (unsigned)((f.N + 15) / 16);
  if (rows <= 16)
    adapted_few<TW, TA, 1, EVEN><<<dim3(across), 512, 0, st>>>(f);
  else
    adapted_few<TW, TA, 2, EVEN><<<dim3(across, (unsigned)((rows + 31) / 32)), 512, 0, st>>>(f);
}
template <typename TW, typename TA>
void launch_few(const FewArgs& f, hipStream_t st) {
  f.K % 8 == 0 ? launch_few<TW, TA, true>(f, st) : launch_few<TW, TA, false>(f, st);
}

constexpr int64_t kMostPackBlocks = 1 << 20;

int64_t tiles32(int64_t batch, int64_t rows, int64_t cols) { return batch * ((rows + 31) / 32) * ((cols + 31) / 32); }

struct Packer {
  PackArgs args{};
  void add(const void* src, int f32, bf16* dst, int64_t batch, int64_t rows, int64_t cols, int64_t out_rows,
           int64_t out_cols, bool turn) {
    PackJob j;
    j.src = src;
    j.dst = dst;
    j.rows = rows;
    j.cols = cols;
    j.out_rows = out_rows;
    j.out_cols = out_cols;
    j.tiles = tiles32(batch, out_rows, out_cols);
    j.f32 = f32;
    j.turn = turn;
    args.job[args.jobs++] = j;
    args.tiles += j.tiles;
  }
};

template <typename TA, int RP, bool KEEP>
void launch_prepare_as(const ThinArgs& t, const PackArgs& p, bool even, hipStream_t st) {
  const dim3 grid((unsigned)(t.row_blocks * t.share * t.jobs + std::min(p.tiles, kMostPackBlocks)));
  even ? adapted_prepare<TA, RP, KEEP, true><<<grid, 256, 0, st>>>(t, p)
       : adapted_prepare<TA, RP, KEEP, false><<<grid, 256, 0, st>>>(t, p);
}
int thin_share(int64_t rows, int requests) { return requests > rows / 16 ? 4 : 1; }  // (16 rows may have many adapters)

template <bool KEEP>
void launch_prepare(ThinArgs t, const PackArgs& p, int rp, int a_f32, hipStream_t st) {
  const int64_t rows = t.q.rows;
  const bool even = t.job[0].K % 8 == 0 && (t.jobs == 1 || t.job[1].K % 8 == 0);
  t.share = thin_share(rows, t.q.count);
  t.row_blocks = (rows + 15) / 16;
#define FFK_PREPARE(RP)                                                           \
  if (rp == RP) {                                                                 \
    a_f32 ? launch_prepare_as<float, RP, KEEP>(t, p, even, st)             \
          : launch_prepare_as<bf16, RP, KEEP>(t, p, even, st);             \
  }
  FFK_PREPARE(16)
  FFK_PREPARE(32)
  FFK_PREPARE(64)
  FFK_PREPARE(128)
#undef FFK_PREPARE
}

// Tiles of 128 x 128 from half a chip's worth on, else of 64 x 64 (us in 128s against 64s): 96 tiles 768 -> 768 26.3 : 21.6,
// 1536 -> 384 34.4 : 30.6; 141 to 144 tiles 26.7 : 28.2 and 40.6 : 42.9. Backward: 48 tiles 30.4 : 29.2, 96 tiles 33.3 : 37.3 and
// (449 channels) 26.3 : 23.7, 192 tiles 28.3 : 31.4.
bool big_tiles(int64_t rows, int N) { return N > 64 && ((rows + 127) / 128) * ((N + 127) / 128) >= 128; }

void launch_product(ProductArgs a, hipStream_t st) {
  const bool big = big_tiles(a.rows, a.N);
  const int t = big ? 128 : 64;
  a.n_tiles = (a.N + t - 1) / t;
  const dim3 grid((unsigned)((a.rows + t - 1) / t * a.n_tiles));
  big ? adapted_product<128, 128, 2><<<grid, 256, 0, st>>>(a) : adapted_product<64, 64, 4><<<grid, 256, 0, st>>>(a);
}

template <int RP>
void launch_finish(ProductArgs a, const GradArgs& g, int chunks, hipStream_t st) {
  const bool big = a.out && big_tiles(a.rows, a.N);
  const int t = big ? 128 : 64;
  a.n_tiles = (a.N + t - 1) / t;
  const uint32_t product = a.out ? (uint32_t)((a.rows + t - 1) / t * a.n_tiles) : 0;
  const dim3 grid(product + (unsigned)((int64_t)(g.job[0].tiles + g.job[1].tiles) * g.adapters * chunks));
  big ? adapted_finish<RP, 128, 128, 2><<<grid, 256, 0, st>>>(a, g, product)
      : adapted_finish<RP, 64, 64, 3><<<grid, 256, 0, st>>>(a, g, product);
}

int64_t up64(int64_t n) { return (n + 63) / 64 * 64; }

Requests requests_of(const AdaptedArgs& a) {
  Requests q;
  q.offsets = a.offsets;
  q.adapter = a.adapter;
  q.scale = a.scale;
  q.count = a.requests;
  q.adapters = a.adapters;
  q.rows = a.rows;
  return q;
}

}  // namespace

AdaptedPlan adapted_plan(int64_t rows, int d_in, int d_out, int adapters, int rank, int requests, int w_f32, int a_f32,
                         int backward) {
  AdaptedPlan p{};
  p.fits = 1;
  p.rp = rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128;
  p.ld = backward ? parts_ld(p.rp) : p.rp;
  p.kp = up64(d_in);
  p.np = up64(d_out);
  p.rows = backward ? adapted_rows_grad_served(rows, d_in, d_out, rank, requests)
                    : adapted_rows_served(rows, d_in, d_out, rank, requests);
  if (p.rows) return p;
  // Few rows straight from the tensors: 768 -> 768 of rank 16 11.4 us at 300 rows (tiles: 13.9), 16.7 at 600 (14.0); 300 -> 900
  // of rank 64 18.9 us at 150, 25.5 at 300 (tiles: 16.8).
  p.few = !backward && rows <= (rank <= 32 ? 384 : 256);
  p.pack_x = d_in % 64 != 0;
  if (backward) {
    p.pack_dy = d_out % 64 != 0;
    const int64_t tiles = (p.kp + p.np) / 64 * adapters;
    // some four workgroups a CU, of 512 of their adapter's rows at least
    const int64_t used = std::max(1, std::min(adapters, requests));
    const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>((1024 + tiles - 1) / tiles, rows / (512 * used)));
    p.chunk = std::min<int64_t>(up64((rows + chunks - 1) / chunks), 64 * kMostGradTiles);
    p.chunks = (int)((rows + p.chunk - 1) / p.chunk);
  } else {
    p.pack_w = w_f32 || d_in % 64 != 0;
    p.pack_up = a_f32 || rank != p.rp;
  }
  if (p.few) return p;
  const int64_t product = (rows + 63) / 64 * (((backward ? d_in : d_out) + 63) / 64);
  int64_t blocks = (rows + 15) / 16 * thin_share(rows, requests) * (backward ? 2 : 1) + kMostPackBlocks;
  blocks = std::max(blocks, product);
  if (backward) {
    const int64_t sums = (p.kp + p.np) / 64 * adapters * p.chunks, values = (int64_t)adapters * rank * (d_in + d_out);
    blocks = std::max(blocks, std::max(product + sums, p.chunks > 1 ? values / 64 + 2 : 0));
  }
  p.fits = blocks < (int64_t(1) << 24);  // (of 256 threads)
  return p;
}

void launch_adapted(const AdaptedArgs& a, const AdaptedPlan& p, hipStream_t st) {
  if (p.rows) return launch_adapted_rows(a, st);
  const Requests q = requests_of(a);
  if (p.few) {
    FewArgs f{};
    f.x = a.x;
    f.w = a.w;
    f.down = a.down;
    f.up = a.up;
    f.bias = a.bias;
    f.out = a.out;
    f.q = q;
    f.u = a.few_u;
    f.ids = a.ids;
    f.K = a.d_in;
    f.N = a.d_out;
    f.rank = a.rank;
    if (a.w_f32)
      a.a_f32 ? launch_few<float, float>(f, st) : launch_few<float, bf16>(f, st);
    else
      a.a_f32 ? launch_few<bf16, float>(f, st) : launch_few<bf16, bf16>(f, st);
    return;
  }
  Packer pack;
  if (p.pack_x) pack.add(a.x, 0, a.xp, 1, a.rows, a.d_in, a.rows, p.kp, false);
  if (p.pack_w) pack.add(a.w, a.w_f32, a.wp, 1, a.d_out, a.d_in, a.d_out, p.kp, false);
  if (p.pack_up) pack.add(a.up, a.a_f32, a.upp, a.adapters, a.d_out, a.rank, a.d_out, p.rp, false);
  ThinArgs t{};
  t.job[0].x = a.x;
  t.job[0].mat = a.down;
  t.job[0].u = a.u;
  t.job[0].K = a.d_in;
  t.q = q;
  t.ids = a.ids;
  t.rank = a.rank;
  t.jobs = 1;
  launch_prepare<false>(t, pack.args, p.rp, a.a_f32, st);
  if (hipPeekAtLastError() != hipSuccess) return;  // (the next launch would index by ids that are not there)
  ProductArgs g{};
  g.x = p.pack_x ? a.xp : a.x;
  g.w = p.pack_w ? a.wp : static_cast<const bf16*>(a.w);
  g.u = a.u;
  g.b = p.pack_up ? a.upp : static_cast<const bf16*>(a.up);
  g.ids = a.ids;
  g.bias = a.bias;
  g.out = a.out;
  g.rows = a.rows;
  g.K = p.kp;
  g.N = a.d_out;
  g.RP = p.rp;
  g.ld = p.ld;
  launch_product(g, st);
}

void launch_adapted_grad(const AdaptedArgs& a, const AdaptedPlan& p, hipStream_t st) {
  if (p.rows) return launch_adapted_rows_grad(a, st);
  Packer pack;
  if (p.pack_x) pack.add(a.x, 0, a.xp, 1, a.rows, a.d_in, a.rows, p.kp, false);
  if (p.pack_dy) pack.add(a.dy, 0, a.dyp, 1, a.rows, a.d_out, a.rows, p.np, false);
  if (a.out) pack.add(a.w, a.w_f32, a.wp, 1, a.d_out, a.d_in, a.d_in, p.np, true);
  if (a.out) pack.add(a.down, a.a_f32, a.down_t, a.adapters, a.rank, a.d_in, a.d_in, p.rp, true);
  ThinArgs t{};
  t.job[0].x = a.x;
  t.job[0].mat = a.down;
  t.job[0].u = a.u;
  t.job[0].K = a.d_in;
  t.job[1].x = a.dy;
  t.job[1].mat = a.up;
  t.job[1].u = a.v;
  t.job[1].K = a.d_out;
  t.job[1].turned = 1;
  t.q = requests_of(a);
  t.ids = a.ids;
  t.rank = a.rank;
  t.jobs = 2;
  launch_prepare<true>(t, pack.args, p.rp, a.a_f32, st);
  if (hipPeekAtLastError() != hipSuccess) return;
  const bf16 *x = p.pack_x ? a.xp : a.x, *dy = p.pack_dy ? a.dyp : a.dy;
  ProductArgs g{};
  g.x = dy;
  g.w = a.wp;
  g.u = a.v;
  g.b = a.down_t;
  g.ids = a.ids;
  g.out = a.out;
  g.rows = a.rows;
  g.K = p.np;
  g.N = a.d_in;
  g.RP = p.rp;
  g.ld = p.ld;
  const bool join = p.chunks > 1;
  GradArgs d{};
  d.job[0].x = x;
  d.job[0].v = a.v;
  d.job[0].cols = a.d_in;
  d.job[0].ld_x = p.kp;
  d.job[1].x = dy;
  d.job[1].v = a.u;
  d.job[1].cols = a.d_out;
  d.job[1].ld_x = p.np;
  void* to[2] = {a.ddown, a.dup};
  const int64_t sj[2] = {a.d_in, 1}, sc[2] = {1, a.rank};
  JoinArgs e{};
  int64_t counts = 0;
  for (int i = 0; i < 2; ++i) {
    GradJob& j = d.job[i];
    const int64_t count = (int64_t)a.adapters * a.rank * j.cols;
    j.tiles = j.ld_x / 64;
    j.to = join ? a.part[i] : to[i];
    j.sj = join ? j.cols : sj[i];
    j.sc = join ? 1 : sc[i];
    d.chunk_stride[i] = join ? count : 0;
    e.job[i].part = a.part[i];
    e.job[i].to = to[i];
    e.job[i].sj = sj[i];
    e.job[i].sc = sc[i];
    e.job[i].count = count;
    e.job[i].cols = j.cols;
    counts += (count + 63) / 64;
  }
  d.ids = a.ids;
  d.rows = a.rows;
  d.chunk = p.chunk;
  d.rank = a.rank;
  d.adapters = a.adapters;
  d.to_bf16 = !join && a.grad_dtype == 0;
  switch (p.rp) {
    case 16: launch_finish<16>(g, d, p.chunks, st); break;
    case 32: launch_finish<32>(g, d, p.chunks, st); break;
    case 64: launch_finish<64>(g, d, p.chunks, st); break;
    default: launch_finish<128>(g, d, p.chunks, st);
  }
  if (join) {
    e.chunks = p.chunks;
    e.rank = a.rank;
    e.to_bf16 = a.grad_dtype == 0;
    adapted_join<<<dim3((unsigned)counts), 256, 0, st>>>(e);
  }
}

}  // namespace ffk
