// Projections with low-rank adapters where rows are many and narrow (the pair stack's): one pass over the rows.
//   y_t = W x_t + b + s_a B_a (A_a x_t)
// The projection stays in registers, a part of its channels a wave; tiles of rows stream through LDS. Every wave takes its rows'
// thin product A x along with its part of the wide one (the rows' operands are there, A's lie in LDS): the 16 x 16
// accumulators, rounded, are as they lie the operand of rank more channels of the wide product, so a row is read once and
// written once, nothing lies between, and the waves meet once a tile. (The thin product split over the waves, its parts
// joined in LDS: 1.8 us for 32 rows of 128 -> 512 without their stores, the chain through three barriers.) A workgroup takes
// consecutive rows, so it meets few requests; a tile that several share is done request by request, each row taking its own's.
#include <algorithm>

#include "ffk_adapted.h"
#include "ffk_device.h"
#include "ffk_kernels.h"

namespace ffk {

namespace {

// The request that a row lies in, walked upwards: rows [.., hi) from the row asked for on have adapter a (-1: none). All
// scalar. Offsets out of order give some request, never an access out of range.
struct RequestAt {
  int r, a;
  int64_t hi;
};
__device__ __forceinline__ int adapter_at(const Requests& q, int r) {
  if (r < 0 || r >= q.count) return -1;
  const int a = q.adapter[r];
  return a >= 0 && a < q.adapters ? a : -1;
}
__device__ __forceinline__ int64_t request_end(const Requests& q, int r) {
  return r < q.count ? (int64_t)q.offsets[r + 1] : q.rows;  // (r = -1: the rows before the first request)
}
__device__ __forceinline__ RequestAt request_first(const Requests& q, int64_t row) {
  int lo = -1, hi = q.count;  // the latest r with offsets[r] <= row
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (q.offsets[mid] <= row)
      lo = mid;
    else
      hi = mid - 1;
  }
  return {lo, adapter_at(q, lo), request_end(q, lo)};
}
__device__ __forceinline__ void request_next(const Requests& q, int64_t row, RequestAt& at) {
  while (at.r < q.count && at.hi <= row) {
    ++at.r;
    at.hi = request_end(q, at.r);
    at.a = adapter_at(q, at.r);
  }
  if (at.r >= q.count) at.hi = q.rows;
}

// Eight values from p on as an operand.
template <typename T>
__device__ __forceinline__ bf16x8 operand8(const T* p) {
  typedef T vec __attribute__((__vector_size__(8 * sizeof(T)), aligned(sizeof(T))));
  const vec v = *reinterpret_cast<const vec*>(p);
  bf16x8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = (bf16)(float)v[e];
  return r;
}

// f(a pointer of the type that p has).
template <typename F>
__device__ __forceinline__ void typed(const void* p, int f32, F f) {
  if (f32)
    f(static_cast<const float*>(p));
  else
    f(static_cast<const bf16*>(p));
}

struct RowsArgs {
  const bf16* x;  // [rows][C]
  const void *w, *down, *up;
  const float* bias;
  bf16* out;      // [rows][N]
  Requests q;
  int rank, w_f32, a_f32;
};

// How a tile of rows of C channels and N outputs are shared among 8 waves.
template <int C, int N>
struct RowsShape {
  static constexpr int TM = C <= 256 && N <= 256 ? 64 : 32;       // rows of a tile
  static constexpr int KS = C / 32;                              // steps of k
  static constexpr int NB = N / 16 / 8 < 2 ? 2 : N / 16 / 8;     // blocks of 16 channels a wave
  static constexpr int NW = N / 16 / NB;                         // waves along the channels
  static constexpr int TT = TM / 16 * NW / 8;                    // blocks of 16 rows a wave
  static constexpr int PER = TM * C / 512 / 8;                   // transfers of a tile a wave
  static constexpr int STORES = NB / 2 * TT;
  static constexpr int STAGES = TM * C <= 4096 ? 6 : TM * C <= 8192 ? 5 : 4;  // tiles in LDS
  static_assert(TT > 0 && PER > 0 && NB % 2 == 0, "");
};

// A tile of rows to LDS (off_row<C>), 1 KB a transfer: a wave's share. Rows behind the last are the last again.
template <int C, int PER>
__device__ __forceinline__ void rows_dma(const bf16* x, int64_t row0, int64_t rows, uint32_t dst, int wave, int lane) {
  constexpr int P = C / 8, R = 512 / C;  // pieces of a row, rows of a transfer
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int t = wave * PER + u, r = R * t + lane / P;
    const int64_t row = row0 + r < rows ? row0 + r : rows - 1;
    dma16_at(x + row * C + 8 * ((lane % P) ^ swz<C>(r)), dst + 1024 * t);
  }
}

// Two neighbouring blocks of 16 channels of 16 rows in 16-byte pieces: lane group g holds channels 4 g .. of each block; after
// v_permlane16_swap (odd rows of 16 lanes of the first against even ones of the second) channels 8 (g / 2) .. of block g % 2.
__device__ __forceinline__ bf16x8 join_blocks(const f32x4& a, const f32x4& b) {
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[e]), __float_as_uint(b[e]), false, false);
    v[e] = (bf16)__uint_as_float(sw[0]);
    v[4 + e] = (bf16)__uint_as_float(sw[1]);
  }
  return v;
}

// out = x W^T + b + u B_a^T, u = s_a x A_a^T rounded to bf16. W and the adapters are read once a workgroup (the adapter's
// again where it changes). The tiles in LDS: one in work, the others on their way. rank <= 16 RB. grid: consecutive tiles each;
// block 512.
template <int C, int N, int RB>
__global__ __launch_bounds__(512, 2) void adapted_rows(const RowsArgs p) {
  using S = RowsShape<C, N>;
  constexpr int PAIRS = (RB + 1) / 2, TM = S::TM, STAGES = C == 512 && RB == 2 ? 3 : S::STAGES;
  __shared__ __attribute__((aligned(16))) bf16 buf[STAGES][TM * C], af[RB * S::KS][64 * 8];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t rows = p.q.rows, tiles = (rows + TM - 1) / TM;
  const int64_t first = tiles * blockIdx.x / gridDim.x, last = tiles * (blockIdx.x + 1) / gridDim.x;
  const uint32_t lds = lds_addr(buf);
  auto fetch = [&](int64_t tile) __attribute__((always_inline)) {
    rows_dma<C, S::PER>(p.x, tile * TM, rows, lds + (uint32_t)((tile - first) % STAGES) * sizeof(buf[0]), wave, lane);
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (first + s < last) fetch(first + s);
  // this wave's channels of W, and its rows of a tile
  const int n0 = 16 * S::NB * (wave % S::NW), r0 = 16 * S::TT * (wave / S::NW);
  bf16x8 w[S::NB][S::KS];
  typed(p.w, p.w_f32, [&](const auto* from) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < S::NB; ++b)
#pragma unroll
      for (int k = 0; k < S::KS; ++k) {
        w[b][k] = operand8(from + (n0 + 16 * b + i) * C + 32 * k + 8 * g);
        if (k % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // (fp32: what is in flight has to fit the registers)
      }
  });
  const f32x4 none = {0.f, 0.f, 0.f, 0.f};
  f32x4 bias[S::NB];
#pragma unroll
  for (int b = 0; b < S::NB; ++b) bias[b] = p.bias ? *reinterpret_cast<const f32x4_a4*>(p.bias + n0 + 16 * b + 4 * g) : none;
  // the adapter: A in LDS as operands, this wave's channels of B in registers
  bf16x8 bf[S::NB][PAIRS];
  float scale = 1.f;
  int loaded = -1;
  auto load = [&](int a) __attribute__((always_inline)) {
    int l = lane;  // (opaque: its addresses are not kept from tile to tile)
    asm volatile("" : "+v"(l));
    const int i = l & 15, g = l >> 4;
    if (loaded >= 0) __syncthreads();  // the last one's has been read
    loaded = a;
    scale = scale_of(p.q, a);
    // (channels behind the rank: those of the last one, loaded without a branch, then zeros)
    typed(p.down, p.a_f32, [&](const auto* from) __attribute__((always_inline)) {
      for (int f = wave; f < RB * S::KS; f += 8) {
        const int j = 16 * (f / S::KS) + i;
        bf16x8 v = operand8(from + ((int64_t)a * p.rank + (j < p.rank ? j : p.rank - 1)) * C + 32 * (f % S::KS) + 8 * g);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = j < p.rank ? v[e] : (bf16)0.f;
        *reinterpret_cast<bf16x8*>(&af[f][8 * l]) = v;
      }
    });
    typed(p.up, p.a_f32, [&](const auto* from) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < S::NB; ++b) {
        const auto* row = from + ((int64_t)a * N + n0 + 16 * b + i) * p.rank;
#pragma unroll
        for (int s = 0; s < PAIRS; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int j = 32 * s + 16 * (e >> 2) + 4 * g + (e & 3);
            const bool is = j < p.rank && (RB > 1 || e < 4);
            const bf16 v = (bf16)(float)row[is ? j : p.rank - 1];
            bf[b][s][e] = is ? v : (bf16)0.f;
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    });
    __syncthreads();
  };
  RequestAt at{p.q.count, -1, rows};
  if (first < last) at = request_first(p.q, first * TM);
  if (first + STAGES - 1 <= last)
    wait_vm_lds<(STAGES - 2) * S::PER>();
  else
    wait_vm_lds<0>();
  __syncthreads();
  for (int64_t tile = first; tile < last; ++tile) {
    if (tile + STAGES - 1 < last) fetch(tile + STAGES - 1);
    const int64_t row0 = tile * TM, end = row0 + TM < rows ? row0 + TM : rows;
    const bf16* t = buf[(tile - first) % STAGES];
    f32x4 acc[S::NB][S::TT];
    for (int64_t row = row0; row < end;) {  // the requests in this tile
      request_next(p.q, row, at);
      if (at.a >= 0 && at.a != loaded) load(at.a);
      f32x4 u[RB][S::TT];
#pragma unroll
      for (int x = 0; x < S::TT; ++x)
#pragma unroll
        for (int b = 0; b < RB; ++b) u[b][x] = none;
      if (row == row0) {
#pragma unroll
        for (int x = 0; x < S::TT; ++x)
#pragma unroll
          for (int b = 0; b < S::NB; ++b) acc[b][x] = bias[b];
#pragma unroll
        for (int k = 0; k < S::KS; ++k) {
          bf16x8 xf[S::TT];
#pragma unroll
          for (int x = 0; x < S::TT; ++x) xf[x] = ld8(&t[off_row<C>(r0 + 16 * x + i, 4 * k + g)]);
#pragma unroll
          for (int x = 0; x < S::TT; ++x) {
#pragma unroll
            for (int b = 0; b < RB; ++b) u[b][x] = mfma16(ld8(&af[b * S::KS + k][8 * lane]), xf[x], u[b][x]);
#pragma unroll
            for (int b = 0; b < S::NB; ++b) acc[b][x] = mfma16(w[b][k], xf[x], acc[b][x]);
          }
        }
      } else if (at.a >= 0) {
#pragma unroll
        for (int k = 0; k < S::KS; ++k)
#pragma unroll
          for (int x = 0; x < S::TT; ++x)
#pragma unroll
            for (int b = 0; b < RB; ++b)
              u[b][x] = mfma16(ld8(&af[b * S::KS + k][8 * lane]), ld8(&t[off_row<C>(r0 + 16 * x + i, 4 * k + g)]), u[b][x]);
      }
      const int64_t stop = at.hi < end ? at.hi : end;
      if (at.a >= 0) {
        const bool whole = row == row0 && stop == end;
#pragma unroll
        for (int x = 0; x < S::TT; ++x) {
          const int64_t mine = row0 + r0 + 16 * x + i;
          bf16x8 uf[PAIRS];
#pragma unroll
          for (int s = 0; s < PAIRS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int b = 2 * s + (e >> 2);
              uf[s][e] = b < RB ? (bf16)(u[b < RB ? b : 0][x][e & 3] * scale) : (bf16)0.f;
            }
          if (whole) {
#pragma unroll
            for (int s = 0; s < PAIRS; ++s)
#pragma unroll
              for (int b = 0; b < S::NB; ++b) acc[b][x] = mfma16(bf[b][s], uf[s], acc[b][x]);
          } else {
#pragma unroll
            for (int b = 0; b < S::NB; ++b) {
              f32x4 add = none;
#pragma unroll
              for (int s = 0; s < PAIRS; ++s) add = mfma16(bf[b][s], uf[s], add);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[b][x][e] += mine >= row && mine < stop ? add[e] : 0.f;
            }
          }
        }
      }
      row = stop;
    }
    // The next tile has landed. Behind its transfers lie those of the tiles after it and the stores of as many tiles before
    // this one (all full: none is short but the last of all): the wave's memory operations complete in order.
    if (tile + STAGES - 1 >= last)
      wait_vm_lds<0>();
    else if (tile - first >= STAGES - 2)
      wait_vm_lds<(STAGES - 2) * (S::PER + S::STORES)>();
    else
      wait_vm_lds<(STAGES - 2) * S::PER>();
    bf16* to = p.out + (row0 + r0 + i) * N + n0 + 16 * (g & 1) + 8 * (g >> 1);
#pragma unroll
    for (int x = 0; x < S::TT; ++x) {
      bf16x8 v[S::NB / 2];
#pragma unroll
      for (int b = 0; b < S::NB / 2; ++b) v[b] = join_blocks(acc[2 * b][x], acc[2 * b + 1][x]);
      if (end - row0 < TM && row0 + r0 + 16 * x + i >= rows) continue;
#pragma unroll
      for (int b = 0; b < S::NB / 2; ++b)
        __builtin_nontemporal_store(v[b], reinterpret_cast<bf16x8*>(to + 16 * x * N + 32 * b));
    }
    __syncthreads();
  }
}

template <int C, int N, int RB>
void launch_rows(const RowsArgs& p, hipStream_t st) {
  const auto kernel = adapted_rows<C, N, RB>;
  constexpr int TM = RowsShape<C, N>::TM;
  const int64_t resident = (int64_t)cu_count() * resident_blocks(reinterpret_cast<const void*>(kernel), 512, 0);
  kernel<<<dim3((unsigned)std::min((p.q.rows + TM - 1) / TM, resident)), 512, 0, st>>>(p);
}

// The widths served: the pair and MSA stacks' projections (d to d, 2 d, 4 d and back, d = 64, 128, 256).
#define FFK_ROWS_WIDTHS(X) \
  X(64, 64) X(64, 128) X(128, 64) X(64, 256) X(256, 64) X(128, 128) X(128, 256) X(256, 128) X(128, 512) X(512, 128) X(256, 256)

template <int C, int N>
void launch_rank(const RowsArgs& p, hipStream_t st) {
  p.rank <= 16 ? launch_rows<C, N, 1>(p, st) : launch_rows<C, N, 2>(p, st);
}

}  // namespace

bool adapted_rows_served(int64_t rows, int d_in, int d_out, int rank, int requests) {
  bool width = false;
#define FFK_ROWS_IS(C, N) width = width || (d_in == C && d_out == N);
  FFK_ROWS_WIDTHS(FFK_ROWS_IS)
#undef FFK_ROWS_IS
  return width && rank <= 32 && rows > 256 && rows >= 64 * (int64_t)requests;
}

void launch_adapted_rows(const AdaptedArgs& a, hipStream_t st) {
  RowsArgs p;
  p.x = a.x;
  p.w = a.w;
  p.down = a.down;
  p.up = a.up;
  p.bias = a.bias;
  p.out = a.out;
  p.q.offsets = a.offsets;
  p.q.adapter = a.adapter;
  p.q.scale = a.scale;
  p.q.count = a.requests;
  p.q.adapters = a.adapters;
  p.q.rows = a.rows;
  p.rank = a.rank;
  p.w_f32 = a.w_f32;
  p.a_f32 = a.a_f32;
#define FFK_ROWS_CASE(C, N) \
  if (a.d_in == C && a.d_out == N) launch_rank<C, N>(p, st);
  FFK_ROWS_WIDTHS(FFK_ROWS_CASE)
#undef FFK_ROWS_CASE
}

}  // namespace ffk
