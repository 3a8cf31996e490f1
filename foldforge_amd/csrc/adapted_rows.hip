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

// The request that a row lies in, walked upwards: rows [.., hi) from the row asked for on have adapter a (-1: none). The same in
// all lanes. The walk reads the offset and the adapter by vector loads (the kernel also stores, so the compiler makes no scalar
// ones) and waits for each with everything else in flight: a boundary between requests drains the tiles on their way, twice, and
// so does each empty request. Offsets out of order give some request, never an access out of range.
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
__device__ __forceinline__ RequestAt request_first(const Requests& q, int64_t row, int lane) {
  const OffsetRange near = offsets_near(q, row, lane);
  int before = (int)near.from;  // the offsets up to `row` (in order: of the first requests), counted by a wave
  int offset[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t i = near.from + lane + 64 * u;
    offset[u] = q.offsets[i < q.count ? i : q.count];
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    before += __popcll(__ballot(near.from + lane + 64 * u < near.to && offset[u] <= row));
  const int r = before - 1;
  return {r, adapter_at(q, r), request_end(q, r)};
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

// A row of `rank` numbers as an operand that goes with the thin product's accumulators as they lie: element e < 4 is number
// 4 g + e, the others 16 on.
template <int RB, typename T>
__device__ __forceinline__ void rank_operand(const T* row, int rank, int g, bf16x8 (&to)[(RB + 1) / 2]) {
  typedef T four __attribute__((__vector_size__(4 * sizeof(T)), aligned(sizeof(T))));
#pragma unroll
  for (int h = 0; h < RB + (RB & 1); ++h) {
    const int j = 16 * h + 4 * g;
    bf16x8& t = to[h >> 1];
    const int e = 4 * (h & 1);
    if (h >= RB) {
#pragma unroll
      for (int c = 0; c < 4; ++c) t[e + c] = (bf16)0.f;
    } else if (rank % 4 == 0) {  // four numbers are all there or none
      const four v = *reinterpret_cast<const four*>(row + (j < rank ? j : 0));
#pragma unroll
      for (int c = 0; c < 4; ++c) t[e + c] = j < rank ? (bf16)(float)v[c] : (bf16)0.f;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bf16 v = (bf16)(float)row[j + c < rank ? j + c : rank - 1];
        t[e + c] = j + c < rank ? v : (bf16)0.f;
      }
    }
  }
}

// f(a pointer of the type that p has).
template <typename F>
__device__ __forceinline__ void typed(const void* p, int f32, F f) {
  if (f32)
    f(static_cast<const float*>(p));
  else
    f(static_cast<const bf16*>(p));
}

// The lane's number, opaque: addresses made of it are not kept in registers from tile to tile.
__device__ __forceinline__ int fresh_lane() {
  int l = threadIdx.x & 63;
  asm volatile("" : "+v"(l));
  return l;
}

// A loaded value is there from here on. Before a loop with transfers in flight: the compiler's own wait for a load that it has
// seen no use of before the loop would stand in the loop, at the first use, and be one for all transfers, each time round.
template <typename T>
__device__ __forceinline__ void landed(T& v) {
  asm volatile("" : "+v"(v));
}

struct RowsArgs {
  const bf16* x;  // [rows][C]
  const void *w, *down, *up;
  const float* bias;
  bf16* out;      // [rows][N]
  Requests q;
  int N, rank, w_f32, a_f32;
};

// How a tile of rows of C channels and N of a workgroup's outputs are shared among 8 waves.
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
  constexpr int P = C / 8;  // pieces of a row
  const int left = rows - row0 < PER * 4096 / C ? (int)(rows - row0) : PER * 4096 / C;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int t = wave * PER + u, piece = 64 * t + lane, r = piece / P, row = r < left ? r : left - 1;
    dma16(x + row0 * C, (uint32_t)(2 * C * row + 16 * ((piece % P) ^ swz<C>(r))), dst + 1024 * t);
  }
}

// Operand of a 16 x 16 product over 32 k from an off_row<C> tile: rows 16 x + i, pieces 4 k + g. at: 2 * off_row<C>(i, g) from
// the tile's LDS address. Bits 0 and 1 of k enter by XOR, the others as an offset (an address for each k would fill the
// registers).
template <int C>
__device__ __forceinline__ bf16x8 row_operand(uint32_t at, int x, int k) {
  return lds_at<bf16x8>((at ^ (uint32_t)((k & 3) << 6)) + (uint32_t)((k >> 2) << 8) + (uint32_t)(x * 32 * C));
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
// again where it changes). The tiles in LDS: one in work, the others on their way. rank <= 16 RB. grid: ranges of consecutive
// tiles, for each the slices of NS outputs (neighbours, so that a range's rows are fetched into one XCD's L2 once); block 512.
// 262144 rows of rank 16: 64 -> 128 23 us (4.5 TB/s), 128 -> 128 30 (4.5), 256 -> 64 33 (5.1), 128 -> 512 79 (4.2), 512 -> 128 74
// to 78 (4.4): bytes, the more so the narrower. 16000 rows, 384 -> 1536: 38 us, chains of tiles behind W's slices. 512 -> 128
// needs 10 registers more than there are: W alone takes half of them, and what is spilled is read again behind a wait for all
// transfers.
template <int C, int NS, int RB>
__global__ __launch_bounds__(512, 2) void adapted_rows(const RowsArgs p, int slices) {
  using S = RowsShape<C, NS>;
  constexpr int PAIRS = (RB + 1) / 2, TM = S::TM, STAGES = C == 512 && RB == 2 ? 3 : S::STAGES;
  __shared__ __attribute__((aligned(16))) bf16 buf[STAGES][TM * C], af[RB * S::KS][64 * 8];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t rows = p.q.rows, tiles = (rows + TM - 1) / TM;
  const int N = p.N, id = (int)xcd_remap(blockIdx.x, gridDim.x), range = id / slices, ranges = gridDim.x / slices;
  const int first = (int)(tiles * range / ranges), last = (int)(tiles * (range + 1) / ranges);
  const uint32_t lds = lds_addr(buf);
  RequestAt at{p.q.count, -1, rows};
  if (first < last) at = request_first(p.q, (int64_t)first * TM, lane);  // (ahead of the transfers, which it would wait for)
  auto fetch = [&](int tile, uint32_t dst) __attribute__((always_inline)) {
    rows_dma<C, S::PER>(p.x, (int64_t)tile * TM, rows, dst, wave, fresh_lane());
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (first + s < last) fetch(first + s, lds + s * sizeof(buf[0]));
  // this wave's channels of W, and its rows of a tile
  const int n0 = NS * (id % slices) + 16 * S::NB * (wave % S::NW), r0 = 16 * S::TT * (wave / S::NW);
  bf16x8 w[S::NB][S::KS];
  typed(p.w, p.w_f32, [&](const auto* from) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < S::NB; ++b)
#pragma unroll
      for (int k = 0; k < S::KS; ++k) {
        w[b][k] = operand8(from + (int64_t)(n0 + 16 * b + i) * C + 32 * k + 8 * g);
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
    const int l = fresh_lane(), i = l & 15, g = l >> 4;
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
        rank_operand<RB>(from + ((int64_t)a * N + n0 + 16 * b + i) * p.rank, p.rank, g, bf[b]);
        if (b % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    });
    landed(scale);
#pragma unroll
    for (int b = 0; b < S::NB; ++b)
#pragma unroll
      for (int s = 0; s < PAIRS; ++s) landed(bf[b][s]);
    __syncthreads();
  };
  if (at.a >= 0) load(at.a);
#pragma unroll
  for (int b = 0; b < S::NB; ++b) {
    landed(bias[b]);
#pragma unroll
    for (int k = 0; k < S::KS; ++k) landed(w[b][k]);
  }
  if (first + STAGES - 1 <= last)
    wait_vm_lds<(STAGES - 2) * S::PER>();
  else
    wait_vm_lds<0>();
  __syncthreads();
  uint32_t xs = lds;  // this tile's buffer
  constexpr uint32_t TOP = (STAGES - 1) * sizeof(buf[0]);
  for (int tile = first; tile < last; ++tile) {
    if (tile + STAGES - 1 < last) fetch(tile + STAGES - 1, xs == lds ? lds + TOP : xs - sizeof(buf[0]));
    const int64_t row0 = (int64_t)tile * TM;
    const int end = rows - row0 < TM ? (int)(rows - row0) : TM;
    const uint32_t t = xs + 2 * off_row<C>(r0 + i, g);
    f32x4 acc[S::NB][S::TT];
    for (int lo = 0; lo < end;) {  // the requests in this tile
      request_next(p.q, row0 + lo, at);
      if (at.a >= 0 && at.a != loaded) load(at.a);
      f32x4 u[RB][S::TT];
#pragma unroll
      for (int x = 0; x < S::TT; ++x)
#pragma unroll
        for (int b = 0; b < RB; ++b) u[b][x] = none;
      if (lo == 0) {
#pragma unroll
        for (int x = 0; x < S::TT; ++x)
#pragma unroll
          for (int b = 0; b < S::NB; ++b) acc[b][x] = bias[b];
#pragma unroll
        for (int k = 0; k < S::KS; ++k) {
          bf16x8 xf[S::TT];
#pragma unroll
          for (int x = 0; x < S::TT; ++x) xf[x] = row_operand<C>(t, x, k);
#pragma unroll
          for (int x = 0; x < S::TT; ++x) {
#pragma unroll
            for (int b = 0; b < RB; ++b) u[b][x] = mfma16(ld8(&af[b * S::KS + k][8 * lane]), xf[x], u[b][x]);
#pragma unroll
            for (int b = 0; b < S::NB; ++b) acc[b][x] = mfma16(w[b][k], xf[x], acc[b][x]);
          }
          // (what is read ahead has to fit the registers)
          if (S::KS * S::TT > 8 && k % (8 / S::TT) == 8 / S::TT - 1) __builtin_amdgcn_sched_barrier(0);
        }
      } else if (at.a >= 0) {
#pragma unroll
        for (int k = 0; k < S::KS; ++k)
#pragma unroll
          for (int x = 0; x < S::TT; ++x)
#pragma unroll
            for (int b = 0; b < RB; ++b)
              u[b][x] = mfma16(ld8(&af[b * S::KS + k][8 * lane]), row_operand<C>(t, x, k), u[b][x]);
      }
      const int hi = __builtin_amdgcn_readfirstlane(at.hi - row0 < end ? (int)(at.hi - row0) : end);
      if (at.a >= 0) {
        const bool whole = lo == 0 && hi == end;
#pragma unroll
        for (int x = 0; x < S::TT; ++x) {
          const int mine = r0 + 16 * x + i;
          bf16x8 uf[PAIRS];
#pragma unroll
          for (int s = 0; s < PAIRS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              // (behind the rank zeros, not the sums of zeros, which an infinite input makes NaN)
              const int b = 2 * s + (e >> 2);
              const bool in = b < RB && 16 * b + 4 * g + (e & 3) < p.rank;
              uf[s][e] = in ? (bf16)(u[b < RB ? b : 0][x][e & 3] * scale) : (bf16)0.f;
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
              for (int e = 0; e < 4; ++e) acc[b][x][e] += mine >= lo && mine < hi ? add[e] : 0.f;
            }
          }
        }
      }
      lo = hi;
    }
    // The next tile has landed. Behind its transfers lie those of the tiles after it and the stores of as many tiles before
    // this one (all full: none is short but the last of all): the wave's memory operations complete in order.
    if (tile + STAGES - 1 >= last)
      wait_vm_lds<0>();
    else if (tile - first >= STAGES - 2)
      wait_vm_lds<(STAGES - 2) * (S::PER + S::STORES)>();
    else
      wait_vm_lds<(STAGES - 2) * S::PER>();
    bf16* to = p.out + row0 * N + ((r0 + i) * N + n0 + 16 * (g & 1) + 8 * (g >> 1));
#pragma unroll
    for (int x = 0; x < S::TT; ++x) {
      bf16x8 v[S::NB / 2];
#pragma unroll
      for (int b = 0; b < S::NB / 2; ++b) v[b] = join_blocks(acc[2 * b][x], acc[2 * b + 1][x]);
      if (end < TM && r0 + 16 * x + i >= end) continue;
#pragma unroll
      for (int b = 0; b < S::NB / 2; ++b)
        __builtin_nontemporal_store(v[b], reinterpret_cast<bf16x8*>(to + 16 * x * N + 32 * b));
    }
    __syncthreads();
    xs = xs == lds + TOP ? lds : xs + sizeof(buf[0]);
  }
}

template <int C, int NS, int RB>
void launch_rows(const RowsArgs& p, hipStream_t st) {
  const auto kernel = adapted_rows<C, NS, RB>;
  constexpr int TM = RowsShape<C, NS>::TM;
  // One workgroup a compute unit, also where registers and LDS hold two: its tiles in flight suffice, and two read W twice
  // (262144 rows, 64 -> 256: 36 us, with two 48; 64 -> 128: 23, with two 27).
  const int64_t slices = p.N / NS, ranges = std::min((p.q.rows + TM - 1) / TM, std::max<int64_t>(1, cu_count() / slices));
  kernel<<<dim3((unsigned)(ranges * slices)), 512, 0, st>>>(p, (int)slices);
}

template <int C, int NS>
void launch_rank(const RowsArgs& p, hipStream_t st) {
  p.rank <= 16 ? launch_rows<C, NS, 1>(p, st) : launch_rows<C, NS, 2>(p, st);
}

// The widest slice of the outputs that divides them and whose weights the registers hold.
template <int C>
void launch_width(const RowsArgs& p, hipStream_t st) {
  if constexpr (C == 128)
    if (p.N % 512 == 0) return launch_rank<C, 512>(p, st);
  if constexpr (C <= 384)
    if (p.N % 256 == 0) return launch_rank<C, 256>(p, st);
  if constexpr (C <= 256)
    if (p.N % 128 != 0) return launch_rank<C, 64>(p, st);
  launch_rank<C, 128>(p, st);
}

// ---------------------------------------------------------------------------------------------------------
// backward

struct RowsGradArgs {
  const bf16 *x, *dy;  // [rows][CI], [rows][CO]
  const void *w, *down, *up;
  bf16* dx;            // or null
  float* part;         // [gridDim.x + requests][16 RB][CI + CO]
  Requests q;
  int rank, w_f32, a_f32;
};

// v as three bf16 that add up to it.
__device__ __forceinline__ void split3(float v, bf16 (&to)[3]) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    to[k] = (bf16)v;
    v -= (float)to[k];
  }
}

template <int CI, int CO, int RB>
struct RowsGradShape {
  static constexpr int KI = CI / 32, KO = CO / 32;                 // steps of k
  static constexpr int NB = CI / 16 < 8 ? 1 : CI / 16 / 8;         // dx: blocks of 16 channels a wave,
  static constexpr int NW = CI / 16 / NB, TT = 2 * NW / 8;         // waves along them, blocks of 16 rows a wave
  // the thin products: parts (shares of k), a wave's steps of k, its blocks of 16 rows (one where k has fewer steps than waves)
  static constexpr int SI = KI < 8 ? KI : 8, SO = KO < 8 ? KO : 8;
  static constexpr int QI = KI / SI, QO = KO / SO, XI = KI < 8 ? 1 : 2, XO = KO < 8 ? 1 : 2;
  static constexpr int GI = (CI / 16 + 7) / 8, GO = (CO / 16 + 7) / 8;  // gradients: blocks of 16 channels a wave
  static constexpr int PER = (CI + CO + 127) / 128;                // transfers of a tile a wave
  static constexpr bool STAGED = NB < 2;                           // dx goes through LDS: 16 channels a wave are 32 bytes a row
  static constexpr int STORES = STAGED ? CI / 128 : NB / 2 * TT;   // stores of a tile a wave (some more with 64 channels)
};

// 16 x 16 x 16: lane group g holds k from 4 g on.
__device__ __forceinline__ f32x4 mfma16_16(bf16x4 a, bf16x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}

// A wave's part of a thin product of 32 rows: steps wave % SLOTS + SLOTS q of k, X blocks of 16 rows.
template <int C, int SLOTS, int Q, int X, int RB, int PARTS>
__device__ __forceinline__ void thin_part(uint32_t at, int wave, int lane, const bf16x8 (&m)[Q][RB][PARTS],
                                          f32x4 (*part)[2][RB][64]) {
  const int first = X == 1 ? wave / SLOTS : 0;
  if (first >= 2) return;  // (fewer shares than waves)
#pragma unroll
  for (int x = 0; x < X; ++x) {
    f32x4 t[RB], rest[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) t[b] = rest[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const bf16x8 v = row_operand<C>(at, first + x, SLOTS * q + wave % SLOTS);
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
          f32x4& to = k ? rest[b] : t[b];
          to = mfma16(m[q][b][k], v, to);
        }
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) part[wave % SLOTS][first + x][b][lane] = PARTS > 1 ? parts_sum(t[b], rest[b]) : t[b];
  }
}

// dx = dy W + v A_a, and the sums over this workgroup's rows of v^T x and u^T dy for each request in them (to
// part[blockIdx.x + request]: a walk through the (workgroup, request) pairs in row order takes each such sum once). Tiles of 32
// rows of x and dy stream through LDS. The thin products, u = s x A^T and v = s dy B, are split over the waves by k; half the
// waves join the parts and lay u and v out as operands: v with tokens as columns for dx (rounded to bf16 as dy is), both in
// three bf16 parts with tokens as k for the gradients (their sum is as exact as fp32's), whose other operand is the tile turned
// as it is read. dx of 16 channels a wave goes through LDS to stores of whole rows. PARTS = 3: fp32 adapters, in three parts
// as well. block 512.
// 262144 rows, 128 -> 512, rank 16: 138 us (fp32 adapters 143 to 150), of which the rows' traffic (403 MB at the rate of a copy)
// is 79; a step's own work is about as long, and one workgroup of a compute unit has only its own eight waves to hide it with. Measured and not
// kept: dy W by halves of k with half the reads of dy (143 us, and 3 us more for few rows), three barriers a step (144).
template <int CI, int CO, int RB, int PARTS>
__global__ __launch_bounds__(512, 2) void adapted_rows_grad(const RowsGradArgs p) {
  using S = RowsGradShape<CI, CO, RB>;
  constexpr int TM = 32, TILE = TM * (CI + CO);
  __shared__ __attribute__((aligned(1024))) bf16 buf[3][TILE];
  __shared__ __attribute__((aligned(16))) f32x4 part[S::SI + S::SO][2][RB][64];
  __shared__ __attribute__((aligned(16))) bf16 stage[S::STAGED ? TM * CI : 8];
  __shared__ __attribute__((aligned(16))) bf16x4 vop[2][RB][64];
  __shared__ __attribute__((aligned(16))) bf16 gop[2][3][RB][64][8];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t rows = p.q.rows, tiles = (rows + TM - 1) / TM;
  const int first = (int)(tiles * blockIdx.x / gridDim.x), last = (int)(tiles * (blockIdx.x + 1) / gridDim.x);
  const uint32_t lds = lds_addr(buf);
  RequestAt at{p.q.count, -1, rows};
  if (first < last) at = request_first(p.q, (int64_t)first * TM, lane);  // (ahead of the transfers, which it would wait for)
  auto fetch = [&](int tile, uint32_t dst) __attribute__((always_inline)) {
    const int64_t row0 = (int64_t)tile * TM;
    const int lane = fresh_lane(), left = rows - row0 < TM ? (int)(rows - row0) : TM;
#pragma unroll
    for (int u = 0; u < S::PER; ++u) {
      // (all waves the same number of transfers, the last one again where they do not go round)
      const int t = wave * S::PER + u < (CI + CO) / 16 ? wave * S::PER + u : (CI + CO) / 16 - 1;
      if (t < CI / 16) {
        const int r = 512 / CI * t + lane / (CI / 8), row = r < left ? r : left - 1;
        dma16(p.x + row0 * CI, (uint32_t)(2 * CI * row + 16 * ((lane % (CI / 8)) ^ swz<CI>(r))), dst + 1024 * t);
      } else {
        const int r = 512 / CO * (t - CI / 16) + lane / (CO / 8), row = r < left ? r : left - 1;
        dma16(p.dy + row0 * CO, (uint32_t)(2 * CO * row + 16 * ((lane % (CO / 8)) ^ swz<CO>(r))), dst + 1024 * t);
      }
    }
  };
  if (first < last) fetch(first, lds);
  if (first + 1 < last) fetch(first + 1, lds + sizeof(buf[0]));
  const f32x4 none = {0.f, 0.f, 0.f, 0.f};
  // W^T: this wave's channels of dx
  const int n0 = 16 * S::NB * (wave % S::NW), r0 = 16 * S::TT * (wave / S::NW);
  bf16x8 w[S::NB][S::KO];
  if (p.dx) {
    typed(p.w, p.w_f32, [&](const auto* from) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < S::NB; ++b)
#pragma unroll
        for (int k = 0; k < S::KO; ++k) {
#pragma unroll
          for (int e = 0; e < 8; ++e) w[b][k][e] = (bf16)(float)from[(32 * k + 8 * g + e) * CI + n0 + 16 * b + i];
          if (k % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
    });
  }
  // the adapter: its share of the thin products (steps wave % S + S q of k, row blocks from wave / S on), this wave's channels
  // of A for dx
  bf16x8 am[S::QI][RB][PARTS], bm[S::QO][RB][PARTS];
  bf16x4 at_[S::NB][RB];
  float scale = 1.f;
  int loaded = -1;
  auto load = [&](int a) __attribute__((always_inline)) {
    const int l = fresh_lane(), i = l & 15, g = l >> 4;
    loaded = a;
    scale = scale_of(p.q, a);
    typed(p.down, p.a_f32, [&](const auto* all) __attribute__((always_inline)) {
      const auto* from = all + (int64_t)a * p.rank * CI;
#pragma unroll
      for (int q = 0; q < S::QI; ++q)
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          const int j = 16 * b + i;
          const auto* row = from + (j < p.rank ? j : p.rank - 1) * CI + 32 * (S::SI * q + wave % S::SI) + 8 * g;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            bf16 t[3];
            split3(j < p.rank ? (float)row[e] : 0.f, t);
#pragma unroll
            for (int k = 0; k < PARTS; ++k) am[q][b][k][e] = t[k];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
      for (int b = 0; b < S::NB; ++b)
#pragma unroll
        for (int s = 0; s < RB; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = 16 * s + 4 * g + e;
            const float v = (float)from[(j < p.rank ? j : p.rank - 1) * CI + n0 + 16 * b + i];
            at_[b][s][e] = j < p.rank ? (bf16)v : (bf16)0.f;
          }
    });
    typed(p.up, p.a_f32, [&](const auto* all) __attribute__((always_inline)) {
      const auto* from = all + (int64_t)a * CO * p.rank;
#pragma unroll
      for (int q = 0; q < S::QO; ++q)
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          const int j = 16 * b + i;
          const auto* row = from + (32 * (S::SO * q + wave % S::SO) + 8 * g) * p.rank + (j < p.rank ? j : p.rank - 1);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            bf16 t[3];
            split3(j < p.rank ? (float)row[e * p.rank] : 0.f, t);
#pragma unroll
            for (int k = 0; k < PARTS; ++k) bm[q][b][k][e] = t[k];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
    });
  };
  // the sums of the request in work: of the first parts of v and u, and of the others
  f32x4 gi[2][RB][S::GI], go[2][RB][S::GO];
  int summed = -1;
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int b = 0; b < RB; ++b) {
#pragma unroll
        for (int q = 0; q < S::GI; ++q) gi[k][b][q] = none;
#pragma unroll
        for (int q = 0; q < S::GO; ++q) go[k][b][q] = none;
      }
  };
  auto flush = [&]() __attribute__((always_inline)) {
    const int l = fresh_lane(), i = l & 15, g = l >> 4;
    float* to = p.part + (int64_t)(blockIdx.x + summed) * (16 * RB * (CI + CO)) + i;
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float* row = to + (16 * b + 4 * g + e) * (CI + CO);
#pragma unroll
        for (int q = 0; q < S::GI; ++q)
          if (8 * q + wave < CI / 16) row[16 * (8 * q + wave)] = parts_sum(gi[0][b][q][e], gi[1][b][q][e]);
#pragma unroll
        for (int q = 0; q < S::GO; ++q)
          if (8 * q + wave < CO / 16) row[CI + 16 * (8 * q + wave)] = parts_sum(go[0][b][q][e], go[1][b][q][e]);
      }
  };
  // this wave's rows of the staged dx
  auto put = [&](int64_t row0) __attribute__((always_inline)) {
    if constexpr (!S::STAGED) return;
    const int lane = fresh_lane(), left = rows - row0 < TM ? (int)(rows - row0) : TM;
#pragma unroll
    for (int u = 0; u < (S::STORES > 0 ? S::STORES : 1); ++u) {
      const int t = wave * (S::STORES > 0 ? S::STORES : 1) + u;
      if (CI == 64 && wave >= 4) continue;
      const int r = 512 / CI * t + lane / (CI / 8), piece = lane % (CI / 8);
      if (r < left)
        __builtin_nontemporal_store(ld8(&stage[off_row<CI>(r, piece)]),
                                    reinterpret_cast<bf16x8*>(p.dx + row0 * CI + (r * CI + 8 * piece)));
    }
  };
  clear();
  f32x4 acc[S::NB][S::TT];
  // What is left of rows lo to hi of the tile at xs (request r): their part of dx beyond dy W, and the gradients' sums
  auto finish = [&](uint32_t xs, int lo, int hi, int r) __attribute__((always_inline)) {
    const uint32_t ys = xs + 2 * TM * CI;
    const bool whole = lo == 0 && hi == TM;
    if (summed != r) {
      if (summed >= 0) {
        flush();
        clear();
      }
      summed = r;
    }
    if (p.dx) {
#pragma unroll
      for (int x = 0; x < S::TT; ++x) {
        const int mine = r0 + 16 * x + i;
#pragma unroll
        for (int b = 0; b < S::NB; ++b) {
          // (selected, also where the whole tile is one request's: behind a branch around the selection the compiler has left
          // out the wait for the product's result)
          f32x4 add = none;
#pragma unroll
          for (int s = 0; s < RB; ++s) add = mfma16_16(at_[b][s], vop[r0 / 16 + x][s][lane], add);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[b][x][e] += mine >= lo && mine < hi ? add[e] : 0.f;
        }
      }
    }
    // tokens as k: element e of lane group g is token 4 g + e, or 16 + 4 g + e - 4; those of other requests are left out
    auto turned = [&](bf16x8 v) __attribute__((always_inline)) {
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = 16 * (e >> 2) + 4 * g + (e & 3);
          v[e] = t >= lo && t < hi ? v[e] : (bf16)0.f;
        }
      }
      return v;
    };
    const uint32_t xa = xs + turned_at<CI>(lane), ya = ys + turned_at<CO>(lane);
    bf16x8 gv[RB][3];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int k = 0; k < 3; ++k) gv[b][k] = ld8(&gop[1][k][b][lane][0]);
#pragma unroll
    for (int q = 0; q < S::GI; ++q)
      if (8 * q + wave < CI / 16) {
        const bf16x8 t = turned(ld_turned16<CI>(xa ^ (uint32_t)(8 * q + wave) << 5));
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int k = 0; k < 3; ++k) gi[k > 0][b][q] = mfma16(gv[b][k], t, gi[k > 0][b][q]);
      }
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int k = 0; k < 3; ++k) gv[b][k] = ld8(&gop[0][k][b][lane][0]);
#pragma unroll
    for (int q = 0; q < S::GO; ++q)
      if (8 * q + wave < CO / 16) {
        const bf16x8 t = turned(ld_turned16<CO>(ya ^ (uint32_t)(8 * q + wave) << 5));
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int k = 0; k < 3; ++k) go[k > 0][b][q] = mfma16(gv[b][k], t, go[k > 0][b][q]);
      }
  };
  // dx of the tile at row0: to the stage, or to its rows
  auto emit = [&](int64_t row0) __attribute__((always_inline)) {
    if constexpr (S::STAGED) {
#pragma unroll
      for (int x = 0; x < S::TT; ++x) {
        bf16x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (bf16)acc[0][x][e];
        const int n = n0 + 4 * g;
        *reinterpret_cast<bf16x4*>(&stage[off_row<CI>(r0 + 16 * x + i, n >> 3) + (n & 7)]) = v;
      }
    } else {
      const int left = rows - row0 < TM ? (int)(rows - row0) : TM;
      bf16* to = p.dx + row0 * CI + ((r0 + i) * CI + n0 + 16 * (g & 1) + 8 * (g >> 1));
#pragma unroll
      for (int x = 0; x < S::TT; ++x) {
        bf16x8 v[(S::NB + 1) / 2];
#pragma unroll
        for (int b = 0; b < S::NB / 2; ++b) v[b] = join_blocks(acc[2 * b][x], acc[2 * b + 1][x]);
        if (left < TM && r0 + 16 * x + i >= left) continue;
#pragma unroll
        for (int b = 0; b < S::NB / 2; ++b)
          __builtin_nontemporal_store(v[b], reinterpret_cast<bf16x8*>(to + 16 * x * CI + 32 * b));
      }
    }
  };
  if (first + 1 < last)
    wait_vm_lds<S::PER>();
  else
    wait_vm_lds<0>();
  __syncthreads();
  // A step is the rows of one request in one tile: what is left of the step before, beside this one's products, and behind a
  // barrier the join of the thin ones. So two barriers a step, and in the longer half the matrix instructions of one step hide
  // the latencies of another's. A tile's buffer is free for the tile two on in the second half of the next tile's first step.
  uint32_t xs0 = 0;  // the step before: its tile, rows and request (-1: none, or no adapter)
  int lo0 = 0, hi0 = 0, r0_ = -1;
  uint32_t xs = lds;  // this tile's buffer, of three in turn
  for (int tile = first;; ++tile) {
    int lo = 0, hi;
    const int64_t row0 = (int64_t)tile * TM;
    const int end = rows - row0 < TM ? (int)(rows - row0) : TM;
    const uint32_t ys = xs + 2 * TM * CI;
    do {
      if (r0_ >= 0) finish(xs0, lo0, hi0, r0_);
      if (lo == 0 && p.dx && tile > first) emit(row0 - TM);
      if (tile >= last) goto done;
      request_next(p.q, row0 + lo, at);
      hi = __builtin_amdgcn_readfirstlane(at.hi - row0 < end ? (int)(at.hi - row0) : end);
      if (at.a >= 0) {
        if (at.a != loaded) load(at.a);
        thin_part<CI, S::SI, S::QI, S::XI>(xs + 2 * off_row<CI>(i, g), wave, lane, am, part);
        thin_part<CO, S::SO, S::QO, S::XO>(ys + 2 * off_row<CO>(i, g), wave, lane, bm, part + S::SI);
      }
      if (lo == 0 && p.dx) {
#pragma unroll
        for (int b = 0; b < S::NB; ++b)
#pragma unroll
          for (int x = 0; x < S::TT; ++x) acc[b][x] = none;
#pragma unroll
        for (int k = 0; k < S::KO; ++k)
#pragma unroll
          for (int x = 0; x < S::TT; ++x) {
            const bf16x8 yf = row_operand<CO>(ys + 2 * off_row<CO>(r0 + i, g), x, k);
#pragma unroll
            for (int b = 0; b < S::NB; ++b) acc[b][x] = mfma16(w[b][k], yf, acc[b][x]);
            // (what is read ahead has to fit the registers)
            if (x == S::TT - 1 && k % (8 / S::TT) == 8 / S::TT - 1) __builtin_amdgcn_sched_barrier(0);
          }
      }
      __syncthreads();
      if (lo == 0 && tile + 2 < last) fetch(tile + 2, xs == lds ? lds + 2 * sizeof(buf[0]) : xs - sizeof(buf[0]));
      if (at.a >= 0 && wave < 4 * RB) {
        const int l = lane, b = wave % RB, x = wave / RB & 1;
        const int y = wave / RB >> 1, token = 16 * x + (l & 15);
        const f32x4(*from)[2][RB][64] = part + (y ? S::SI : 0);
        f32x4 v = from[0][x][b][l];
        for (int s = 1; s < (y ? S::SO : S::SI); ++s) v += from[s][x][b][l];
        const bool in = token >= lo && token < hi;
        bf16x4 high;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          bf16 t[3];
          split3(in && 16 * b + 4 * (l >> 4) + e < p.rank ? v[e] * scale : 0.f, t);  // (an infinite input: v times zeros is NaN)
          high[e] = t[0];
#pragma unroll
          for (int k = 0; k < 3; ++k) gop[y][k][b][4 * (l >> 4) + e + 16 * (l >> 2 & 3)][4 * x + (l & 3)] = t[k];
        }
        if (y) vop[x][b][l] = high;
      }
      if (lo == 0) {
        if (p.dx && tile > first) put(row0 - TM);
        // The next tile has landed: behind its transfers lie those of the tile after it and the stores since then (of whole
        // tiles): the wave's memory operations complete in order.
        constexpr int BEHIND = S::PER + (S::STAGED ? 2 : 1) * S::STORES;
        if (tile + 2 >= last)
          wait_vm_lds<0>();
        else if (p.dx && tile - first >= 2)
          wait_vm_lds<BEHIND>();
        else
          wait_vm_lds<S::PER>();
      }
      __syncthreads();
      xs0 = xs;
      lo0 = lo;
      hi0 = hi;
      r0_ = at.a >= 0 ? at.r : -1;
      lo = hi;
    } while (lo < end);
    xs = xs == lds + 2 * sizeof(buf[0]) ? lds : xs + sizeof(buf[0]);
  }
done:
  __syncthreads();
  if (first < last) {
    if (p.dx) put((int64_t)(last - 1) * TM);
    if (summed >= 0) flush();
  }
}

struct RowsJoinArgs {
  const float* part;  // [slots][rp][CI + CO]
  void *ddown, *dup;
  Requests q;
  int rank, rp, d_in, d_out, grid, to_bf16;
};

constexpr int kMostRowsRequests = 512;

// The gradients of an adapter from its requests' sums: request r has one in slot b + r of each workgroup b of the grid that its
// rows touch. The adapter's slots are counted first (requests beside each other, a scan by the first wave) and then shared out
// in turn: walked request by request they are a chain of latencies (32000 rows of 500 requests, 128 -> 512: 171 us the backward
// pass). A workgroup: 64 columns of one channel of one adapter, sixteen threads beside each other along them, sixteen groups
// of slots. grid (ceil((d_in + d_out) / 64), rank, adapters); block 256.
__global__ __launch_bounds__(256) void adapted_rows_join(const RowsJoinArgs p) {
  __shared__ f32x4 sum[16][16];
  __shared__ int first[kMostRowsRequests + 1], base[kMostRowsRequests];
  const int width = p.d_in + p.d_out, group = threadIdx.x >> 4, c = 64 * blockIdx.x + 4 * (threadIdx.x & 15);
  const int j = blockIdx.y, a = blockIdx.z;
  const int64_t tiles = (p.q.rows + 31) / 32, G = p.grid;
  for (int r = threadIdx.x; r < p.q.count; r += 256) {
    const int64_t lo = p.q.offsets[r] > 0 ? p.q.offsets[r] : 0;
    const int64_t hi = p.q.offsets[r + 1] < p.q.rows ? (int64_t)p.q.offsets[r + 1] : p.q.rows;
    // workgroup b has the tiles from tiles b / G on
    const int64_t b0 = ((lo / 32 + 1) * G - 1) / tiles, b1 = (((hi - 1) / 32 + 1) * G - 1) / tiles;
    first[r] = p.q.adapter[r] == a && lo < hi ? (int)(b1 - b0) + 1 : 0;
    base[r] = (int)b0 + r;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int before = 0;
    for (int r0 = 0; r0 < p.q.count; r0 += 64) {
      const int n = r0 + lane < p.q.count ? first[r0 + lane] : 0;
      int upto = n;
#pragma unroll
      for (int m = 1; m < 64; m *= 2) {
        const int o = __shfl_up(upto, m, 64);
        if (lane >= m) upto += o;
      }
      if (r0 + lane < p.q.count) first[r0 + lane] = before + upto - n;
      before += __shfl(upto, 63, 64);
    }
    if (lane == 0) first[p.q.count] = before;
  }
  __syncthreads();
  const int slots = first[p.q.count];
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (c < width) {
    const float* from = p.part + (int64_t)j * width + c;
    int r = 0;
    for (int s0 = group; s0 < slots; s0 += 64) {
      f32x4 t[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = s0 + 16 * u;
        t[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (s < slots) {
          while (first[r + 1] <= s) ++r;
          t[u] = *reinterpret_cast<const f32x4*>(from + (int64_t)(base[r] + s - first[r]) * p.rp * width);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) v += t[u];
    }
  }
  sum[group][threadIdx.x & 15] = v;
  __syncthreads();
  if (threadIdx.x >= 64 || 64 * (int)blockIdx.x + (int)threadIdx.x >= width) return;
  float total = 0.f;
#pragma unroll
  for (int s = 0; s < 16; ++s) total += sum[s][threadIdx.x >> 2][threadIdx.x & 3];
  const int col = 64 * blockIdx.x + threadIdx.x;
  const bool in = col < p.d_in;
  const int64_t at = in ? ((int64_t)a * p.rank + j) * p.d_in + col : ((int64_t)a * p.d_out + col - p.d_in) * p.rank + j;
  void* to = in ? p.ddown : p.dup;
  if (p.to_bf16)
    static_cast<bf16*>(to)[at] = (bf16)total;
  else
    static_cast<float*>(to)[at] = total;
}

// The widths of the backward pass: the pair and MSA stacks' projections (d to d, 2 d, 4 d and back, d = 64, 128, 256).
#define FFK_ROWS_WIDTHS(X) \
  X(64, 64) X(64, 128) X(128, 64) X(64, 256) X(256, 64) X(128, 128) X(128, 256) X(256, 128) X(128, 512) X(512, 128) X(256, 256)

template <int CI, int CO>
void launch_grad(const RowsGradArgs& p, int grid, hipStream_t st) {
  if (p.a_f32)
    adapted_rows_grad<CI, CO, 1, 3><<<dim3(grid), 512, 0, st>>>(p);
  else
    adapted_rows_grad<CI, CO, 1, 1><<<dim3(grid), 512, 0, st>>>(p);
}

}  // namespace

// Against tiles (adapted.hip; us, one pass : tiles, rank 16). Up to 128 channels in it is the faster at every size (128 -> 512:
// 300 rows 9.1 : 10.4, 64000 26 : 44). Wider ones read W into registers first: 256 -> 256 in requests of 500 12.5 : 9.3 at 4000
// rows, 13.0 : 15.2 at 16000; 512 -> 128 14.3 : 11.1 and 16.7 : 17.7; 384 -> 384 13.3 : 11.3 and 21.2 : 21.8. An adapter's turn
// costs it more than tiles, so short requests need many rows: 32 rows each 8.9 : 11.3 (64 -> 256), 8.7 : 9.3 (128 -> 128) and
// 13.7 : 14.3 (256 -> 256) at 16000, 24 : 29, 21 : 25 and 36 : 39 at 64000, but 8.1 : 6.9, 7.9 : 7.2 and 12.7 : 8.3 at 4000; 16 rows
// each 39 : 32 (64 -> 256, 64000 rows). 384 channels, whose waves all take the thin product: 27 : 21 at 32 rows each, 27 : 25 at
// 62, 23 : 23 at 100 (16000 rows).
bool adapted_rows_served(int64_t rows, int d_in, int d_out, int rank, int requests) {
  const bool width = d_in == 64 || d_in == 128 || d_in == 256 ? d_out % 64 == 0 : (d_in == 384 || d_in == 512) && d_out % 128 == 0;
  const int64_t least = d_in <= 128 ? 257 : d_in == 384 ? 6144 : 12288, each = d_in != 384 && rows >= 16000 ? 32 : 64;
  return width && rank <= 32 && rows >= least && rows >= each * requests;
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
  p.N = a.d_out;
  p.rank = a.rank;
  p.w_f32 = a.w_f32;
  p.a_f32 = a.a_f32;
  switch (a.d_in) {
    case 64: return launch_width<64>(p, st);
    case 128: return launch_width<128>(p, st);
    case 256: return launch_width<256>(p, st);
    case 384: return launch_width<384>(p, st);
    default: return launch_width<512>(p, st);
  }
}

int adapted_rows_grid(int64_t rows) { return (int)std::min<int64_t>((rows + 31) / 32, cu_count()); }

// Against tiles (us, one pass : tiles, fp32 adapters of rank 16; requests of 500): 64 -> 64 15.3 : 14.9 at 4000 rows, 16.6 : 23.7
// at 8000, 128 -> 128 16.9 : 15.6 and 18.9 : 25.2; 128 -> 512 24.6 : 17.8 at 4000, 28.4 : 29.3 at 8000, 43 : 69 at 32000. Requests
// of 48 rows: 20 : 26 (64 -> 64, 4000 rows), 28 : 47 (128 -> 128, 8000), 40 : 52 and 60 : 56 (128 -> 512, 8000 and 16000); of 32:
// 25 : 37 (64 -> 64, 8000), but 44 : 39 at 16000 and 59 : 47 (128 -> 512).
bool adapted_rows_grad_served(int64_t rows, int d_in, int d_out, int rank, int requests) {
  bool width = false;
#define FFK_ROWS_IS(C, N) width = width || (d_in == C && d_out == N);
  FFK_ROWS_WIDTHS(FFK_ROWS_IS)
#undef FFK_ROWS_IS
  const int64_t least = d_in + d_out <= 320 ? 4096 : 8192;
  return width && rank <= 16 && rows >= least && requests <= kMostRowsRequests && rows >= 48 * (int64_t)requests;
}

void launch_adapted_rows_grad(const AdaptedArgs& a, hipStream_t st) {
  RowsGradArgs p;
  p.x = a.x;
  p.dy = a.dy;
  p.w = a.w;
  p.down = a.down;
  p.up = a.up;
  p.dx = a.out;
  p.part = a.part[0];
  p.q.offsets = a.offsets;
  p.q.adapter = a.adapter;
  p.q.scale = a.scale;
  p.q.count = a.requests;
  p.q.adapters = a.adapters;
  p.q.rows = a.rows;
  p.rank = a.rank;
  p.w_f32 = a.w_f32;
  p.a_f32 = a.a_f32;
  const int grid = adapted_rows_grid(a.rows);
#define FFK_ROWS_CASE(C, N) \
  if (a.d_in == C && a.d_out == N) launch_grad<C, N>(p, grid, st);
  FFK_ROWS_WIDTHS(FFK_ROWS_CASE)
#undef FFK_ROWS_CASE
  RowsJoinArgs j;
  j.part = p.part;
  j.ddown = a.ddown;
  j.dup = a.dup;
  j.q = p.q;
  j.rank = a.rank;
  j.rp = 16;
  j.d_in = a.d_in;
  j.d_out = a.d_out;
  j.grid = grid;
  j.to_bf16 = a.grad_dtype == 0;
  adapted_rows_join<<<dim3((unsigned)((a.d_in + a.d_out + 63) / 64), (unsigned)a.rank, (unsigned)a.adapters), 256, 0, st>>>(j);
}

}  // namespace ffk
