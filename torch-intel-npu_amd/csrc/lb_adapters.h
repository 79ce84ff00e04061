// gfx950 kernels of lb_adapters (include/lowbit_decode_hip.h): out = y + s (x A^T) B^T, the factors A [rank, K] and
// B [N, rank] those of each row's own adapter.
//
// z = x A^T in fp32 (adapters_down_kernel), then y + s z B^T (adapters_up_kernel, or of many rows adapters_tile_kernel), or both in one
// launch where that is little (adapters_rows_kernel).  Rows are the columns of 16x16x32 products, whose rows are ranks and
// outputs, so that a lane holds one row throughout.  Of few rows, the columns are up to 16 of one adapter, wherever they lie among 64
// (94 rows of 21 adapters in no order, 14336 by 4096, rank 128: 43.6 us, against 66.2 with columns of 16 rows side by side); of many,
// 64 rows side by side, each adapter's in turn.
#pragma once
#include "lb_serve.h"

namespace lb {

constexpr int kRowsWaves = 8;   // of a workgroup of adapters_rows_kernel (16 spill, which makes every launch 5 us longer)

template <class T>
struct AdaptersParams {
  const T *x, *y, *down, *up;
  T *out;
  const float *scales;      // null: 1
  const int64_t *index;
  float *z;                 // [slices][M][rank]
  long long ldx, ldy, ldo;
  int M, N, K, rank, count;
  int slices, groups;       // parts of K, added in the second launch; groups of ranks
  int shares, shares_up;    // workgroups that share a tile of rows, in each launch
  int span, stack;          // adapters_up_kernel: outputs of a wave, tiles of a workgroup (adapters_rows_kernel: outputs of one)
  int wide;                 // rows of y and out are whole 16-byte pieces
};

// The adapter of row `first` + lane, -1 where there is none, -2 where its number is none.
template <class T>
__device__ __forceinline__ int adapter_of(const AdaptersParams<T> &p, int first, int lane, int rows) {
  if (lane >= rows || first + lane >= p.M) return -1;
  const int64_t a = p.index[first + lane];
  return a >= 0 && a < p.count ? (int)a : a == -1 ? -1 : -2;
}

// Calls f(adapter, rows as a mask) for this workgroup's share of the adapters of a tile.
template <class F>
__device__ __forceinline__ void each_adapter(int id, int share, int shares, F &&f) {
  uint64_t left = __ballot(id >= 0);
  for (int n = 0; left; ++n) {
    const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t mine = __ballot(id == a);
    left &= ~mine;
    if (n % shares == share) f(a, mine);
  }
}

// Calls f(adapter, row, rows) for this share of what a tile of 64 rows holds, up to 16 rows of one adapter at a time: `row` that of the lane's
// column (lane % 16, where that is below `rows`).  So an adapter's factors are read once for its rows, wherever in the tile they are.
// (Every lane finds the rows of its adapter at once, by the bits of its number, so that a share has its part without going through those
// before it: adapter by adapter took 4 us of a tile of 64.)
template <class F>
__device__ __forceinline__ void each_sixteen(int id, int lane, int count, int share, int shares, F &&f) {
  uint64_t same = __ballot(id >= 0);
  for (int bits = count - 1, bit = 0; bits >> bit; ++bit) {
    const uint64_t set = __ballot(id >> bit & 1);
    same &= id >> bit & 1 ? set : ~set;
  }
  const int before = __popcll(same & ((1ull << lane) - 1));      // rows of the lane's adapter before its own
  const uint64_t firsts = __ballot(id >= 0 && before % 16 == 0);
  const int index = __builtin_amdgcn_mbcnt_hi((uint32_t)(firsts >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)firsts, 0));
  for (int n = share; n < (int)__popcll(firsts); n += shares) {
    const int at = __builtin_ctzll(__ballot((firsts >> lane & 1) && index == n));
    const int a = __builtin_amdgcn_readlane(id, at), column = before - __builtin_amdgcn_readlane(before, at);
    const bool mine = id == a && column >= 0 && column < 16;
    const int row = __builtin_amdgcn_ds_permute(4 * (mine ? column : 63), lane);   // (nobody asks lane 63)
    f(a, __shfl(row, lane & 15), (int)__popcll(__ballot(mine)));
  }
}

// z of 16 MT rows and 16 RT ranks over one slice of K: waves take every eighth 64 of it and meet in LDS.  The rows' memory bounds it
// (4001 rows of 4096, rank 32: 13.4 us), or with few rows the chain of index, factors and sums (5.0 us for 64 rows of 64 adapters).
// (MT 1: up to 16 rows of one adapter in 64; MT 4: 64 rows of any, each adapter's in turn.)
template <class T, int RT, int MT>
__global__ __launch_bounds__(512) void adapters_down_kernel(AdaptersParams<T> p) {
  typedef typename Of16<T>::x8 x8;
  constexpr int W = 8, TILES = RT * MT, AHEAD = RT + MT > 6 ? 1 : 2;   // pieces of 64 in flight
  __shared__ f4 met[W][TILES][64];
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slice = blockIdx.x % p.slices, rest = blockIdx.x / p.slices, rank0 = rest % p.groups * (16 * RT), first = rest / p.groups * 64;
  const int id = adapter_of(p, first, lane, 64);
  const int all = (p.K + 63) / 64, size = (all + p.slices - 1) / p.slices, from = slice * size, to = min(all, from + size);
  // Rows of an adapter's columns 16 t + c, behind `first`, and whether they are its own.
  auto part = [&](int a, auto row_of, auto lives) {
    f4 acc[RT][MT] = {};
    const T *const down = p.down + (size_t)a * p.rank * p.K;
    const int row = j % 8, at = 32 * (j / 8) + 8 * g;       // (see rows_from_lines)
    const T *dr[RT][2], *xr[MT][2];
    bool live[MT][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int r = 0; r < RT; ++r) dr[r][b] = down + (size_t)min(rank0 + 16 * r + 8 * b + row, p.rank - 1) * p.K + at;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        live[t][b] = lives(t, 8 * b + row);
        xr[t][b] = p.x + (size_t)min(first + row_of(t, 8 * b + row), p.M - 1) * p.ldx + at;
      }
    }
    const u4 none = {0, 0, 0, 0};
    for (int piece = from + wave; piece < to; piece += W * AHEAD) {
      u4 d[AHEAD][2][RT], x[AHEAD][2][MT];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int k = (piece + n * W) * 64;
          const bool there = piece + n * W < to && k + at < p.K;
#pragma unroll
          for (int r = 0; r < RT; ++r) d[n][b][r] = there ? *reinterpret_cast<const u4 *>(dr[r][b] + k) : none;
#pragma unroll
          for (int t = 0; t < MT; ++t) x[n][b][t] = there && live[t][b] ? *reinterpret_cast<const u4 *>(xr[t][b] + k) : none;
        }
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
#pragma unroll
        for (int r = 0; r < RT; ++r) rows_from_lines(d[n][0][r], d[n][1][r]);
#pragma unroll
        for (int t = 0; t < MT; ++t) rows_from_lines(x[n][0][t], x[n][1][t]);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < MT; ++t)
              acc[r][t] = Of16<T>::mma(__builtin_bit_cast(x8, d[n][c][r]), __builtin_bit_cast(x8, x[n][c][t]), acc[r][t]);
      }
    }
    __syncthreads();                      // (what an earlier adapter left is read)
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < MT; ++t) met[wave][r * MT + t][lane] = acc[r][t];
    __syncthreads();
    for (int i = wave; i < TILES; i += W) {
      f4 sum = met[0][i][lane];
#pragma unroll
      for (int w = 1; w < W; ++w) sum += met[w][i][lane];
      const int rank = rank0 + i / MT * 16 + 4 * g, at_row = row_of(i % MT, j);
      if (rank < p.rank && lives(i % MT, j)) *reinterpret_cast<f4 *>(p.z + ((size_t)slice * p.M + first + at_row) * p.rank + rank) = sum;
    }
  };
  if constexpr (MT == 1)
    each_sixteen(id, lane, p.count, blockIdx.y, p.shares, [&](int a, int at_row, int rows) {
      part(a, [&](int, int c) { return __shfl(at_row, c); }, [&](int, int c) { return c < rows; });
    });
  else
    each_adapter(id, blockIdx.y, p.shares, [&](int a, uint64_t mine) {
      part(a, [&](int t, int c) { return 16 * t + c; }, [&](int t, int c) { return (bool)(mine >> (16 * t + c) & 1); });
    });
}

// Rows row0 .. row0 + 15 of a tile without an adapter, and those whose adapter there is not: y's values or NaNs, outputs from .. to
// - 1, by the lanes of a wave, 8 outputs a lane at once.
template <class T>
__device__ __forceinline__ void rows_without(const AdaptersParams<T> &p, int id, int first, int row0, int lane, int from, int to) {
  typedef typename Of16<T>::x8 x8;
  if (!__ballot(lane >= row0 && lane < row0 + 16 && first + lane < p.M && id < 0 && (id == -2 || p.out != p.y))) return;
  const int pieces = (to - from + 7) / 8;
  const int ids = __shfl(id, row0 + (lane & 15));      // (of lanes that take part to the end)
  for (int i = lane; i < 16 * pieces; i += 64) {
    const int row = row0 + i / pieces, n = from + 8 * (i % pieces), whose = __shfl(ids, row - row0);
    if (first + row >= p.M || whose >= 0 || (whose == -1 && p.out == p.y)) continue;
    const T *const y = p.y + (size_t)(first + row) * p.ldy + n;
    T *const out = p.out + (size_t)(first + row) * p.ldo + n;
    if (p.wide && whose == -1) {
      *reinterpret_cast<x8 *>(out) = *reinterpret_cast<const x8 *>(y);
    } else {
      for (int e = 0; e < 8 && n + e < to; ++e) out[e] = whose == -1 ? y[e] : (T)__builtin_nanf("");
    }
  }
}

// z of a row as the sum of two 16-bit numbers (16 bits of bf16 and 22 of fp16, after a power of two has brought the row's
// largest one below 1, so that no z is too large or small for fp16): its rounding stays far below that of the output.
// A lane holds ranks 32 c + 8 g .. of row j; scale takes the power of two back.
template <class T, int RC>
struct Halves {
  typename Of16<T>::x8 high[RC], low[RC];
  // LANES: 0 where the lanes of a row are 16 apart, else as many side by side.
  template <int LANES = 0>
  __device__ __forceinline__ void split(float (&z)[RC][8], float &scale) {
    if constexpr (__is_same(T, f16)) {
      float top = 0.0f;
#pragma unroll
      for (int c = 0; c < RC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(z[c][e]));
      if constexpr (LANES == 0) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
      } else {
#pragma unroll
        for (int d = LANES / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
      }
      const int e2 = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
      for (int c = 0; c < RC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) z[c][e] = __builtin_amdgcn_ldexpf(z[c][e], -e2);
      scale = __builtin_amdgcn_ldexpf(scale, e2);
    }
#pragma unroll
    for (int c = 0; c < RC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const T h = (T)z[c][e];
        high[c][e] = h;
        low[c][e] = (T)(fabsf((float)h) < INFINITY ? z[c][e] - (float)h : 0.0f);
      }
  }
};

// 64 outputs of 16 rows: their factors, and y and what is stored.  Row j of tile s is output 32 (s / 2) + 8 (j / 4) + 4 (s % 2) +
// j % 4, so that a lane has 8 outputs side by side of its row, twice.
template <class T, int RC>
struct Factors {
  typename Of16<T>::x8 up[4][RC];
  __device__ __forceinline__ void fetch(const AdaptersParams<T> &p, const T *factor, int n0, int j, int g) {
    typedef typename Of16<T>::x8 x8;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int n = min(n0 + 32 * (s / 2) + 8 * (j / 4) + 4 * (s & 1) + (j & 3), p.N - 1);
#pragma unroll
      for (int c = 0; c < RC; ++c)
        up[s][c] = 32 * c + 8 * g < p.rank ? *reinterpret_cast<const x8 *>(factor + (size_t)n * p.rank + 32 * c + 8 * g) : x8{};
    }
  }
};

template <class T>
struct Base {
  typedef typename Of16<T>::x8 x8;
  x8 y[2];
  __device__ __forceinline__ void fetch(const AdaptersParams<T> &p, const T *yrow, int n0, int to, bool live, int g) {
    if (p.wide && live)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (n0 + 32 * s + 8 * g < to) y[s] = *reinterpret_cast<const x8 *>(yrow + n0 + 32 * s + 8 * g);
  }
  template <int RC>
  __device__ __forceinline__ void store(const AdaptersParams<T> &p, const Factors<T, RC> &f, const Halves<T, RC> &z, float scale, const T *yrow, T *out,
                                        int n0, int to, bool live, int g) const {
    f4 acc[4] = {};
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int c = 0; c < RC; ++c) {
        acc[s] = Of16<T>::mma(f.up[s][c], z.high[c], acc[s]);
        acc[s] = Of16<T>::mma(f.up[s][c], z.low[c], acc[s]);
      }
    if (!live) return;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int n = n0 + 32 * s + 8 * g;
      if (p.wide) {
        if (n >= to) continue;
        x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T)((float)y[s][e] + scale * acc[2 * s + e / 4][e % 4]);
        *reinterpret_cast<x8 *>(out + n) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < to) out[n + e] = (T)((float)yrow[n + e] + scale * acc[2 * s + e / 4][e % 4]);
      }
    }
  }
};

// Outputs from .. to - 1 of 16 rows, 64 at a time, every `step`, what they read requested one time ahead.
template <class T, int RC>
struct Writer {
  Factors<T, RC> factors;
  Base<T> base;
  __device__ __forceinline__ void begin(const AdaptersParams<T> &p, const T *up, const T *y, int from, int to, bool live, int j, int g) {
    factors.fetch(p, up, from, j, g);
    base.fetch(p, y, from, to, live, g);
  }
  __device__ __forceinline__ void run(const AdaptersParams<T> &p, const T *up, const T *y, T *out, const Halves<T, RC> &z, float scale, int from, int to,
                                      int step, bool live, int j, int g) {
    for (int n0 = from; n0 < to; n0 += step) {
      const Factors<T, RC> f = factors;
      const Base<T> held = base;
      if (n0 + step < to) begin(p, up, y, n0 + step, to, live, j, g);
      held.store(p, f, z, scale, y, out, n0, to, live, g);
    }
  }
};

// z of a row, its slices added in their order.
template <class T, int RC>
__device__ __forceinline__ void gather(const AdaptersParams<T> &p, int row, bool live, int g, float (&z)[RC][8]) {
  // Parts in flight: the registers of four of rank 128 leave room for one wave a SIMD (64 rows of 60 adapters, 4096 outputs: 31.0 us
  // against 27.1).
  constexpr int SLICES = RC == 4 ? 2 : 4;
  for (int s0 = 0; s0 < p.slices; s0 += SLICES) {
    f4 part[SLICES][RC][2] = {};
#pragma unroll
    for (int s = 0; s < SLICES; ++s)
#pragma unroll
      for (int c = 0; c < RC; ++c)
        if (live && s0 + s < p.slices && 32 * c + 8 * g < p.rank) {
          const float *const at = p.z + ((size_t)(s0 + s) * p.M + row) * p.rank + 32 * c + 8 * g;
          part[s][c][0] = *reinterpret_cast<const f4 *>(at);
          part[s][c][1] = *reinterpret_cast<const f4 *>(at + 4);
        }
#pragma unroll
    for (int s = 0; s < SLICES; ++s)
#pragma unroll
      for (int c = 0; c < RC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) z[c][e] += part[s][c][e / 4][e % 4];
  }
}

// out = y + s z B^T.  A wave takes up to 16 rows of one adapter in 64, and `span` outputs; the waves of a workgroup have `stack` of those and
// 4 / stack spans.  (64 rows of 64 adapters, 4096 outputs, rank 16: 5.4 us, of which the launch and the loads of index, z and factors one after
// the other are most.)
template <class T, int RC>
__global__ __launch_bounds__(256) void adapters_up_kernel(AdaptersParams<T> p) {
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int beside = 4 / p.stack, spans = (p.N + p.span * beside - 1) / (p.span * beside);
  const int from = (blockIdx.x % spans * beside + wave / p.stack) * p.span, to = min(p.N, from + p.span);
  const int first = blockIdx.x / spans * 64;
  if (from >= to) return;
  const int id = adapter_of(p, first, lane, 64);
  if (blockIdx.y == p.shares_up) {        // (workgroups of their own, so that no product waits for it)
    for (int i = wave % p.stack; i < 4; i += p.stack) rows_without(p, id, first, 16 * i, lane, from, to);
    return;
  }
  each_sixteen(id, lane, p.count, blockIdx.y * p.stack + wave % p.stack, p.shares_up * p.stack, [&](int a, int at_row, int rows) {
    const bool live = j < rows;
    const int row = first + at_row;
    const T *const up = p.up + (size_t)a * p.N * p.rank;
    const T *const y = p.y + (size_t)row * p.ldy;
    T *const out = p.out + (size_t)row * p.ldo;
    Writer<T, RC> writer;
    writer.begin(p, up, y, from, to, live, j, g);
    float scale = p.scales ? p.scales[a] : 1.0f, z[RC][8] = {};
    gather<T, RC>(p, row, live, g, z);
    Halves<T, RC> halves;
    halves.split(z, scale);
    writer.run(p, up, y, out, halves, scale, from, to, 64, live, j, g);
  });
}

// out = y + s z B^T of 64 rows and `span` outputs, 128 at a time, for many rows (p.wide).  y is read and out written in rows of
// 256 bytes, 1 KB a wave at once, since a transfer whose lanes have 16 rows costs the address unit twice that of whole lines;
// the products come to the lanes of those rows through LDS.  z is added up and split once a workgroup, and kept in LDS; the
// factors of 32 outputs, which a wave holds, serve all rows of the tile.  Memory bounds it: 4001 rows of 14336 outputs, rank 32, 229 MB
// of y and out, take 52 us (4.4 TB/s).  (out is stored past the caches: 5360 rows of 4096, both launches, 44.3 -> 41.0 us.)
template <class T, int RC>
__global__ __launch_bounds__(256) void adapters_tile_kernel(AdaptersParams<T> p) {
  typedef typename Of16<T>::x8 x8;
  constexpr int ROWS = 64, NB = 128, PITCH = NB + 4, ZP = 32 * RC + 8, PER = ROWS * NB / 2048, LANES = 4 * RC;   // LANES: of a row's ranks
  __shared__ __align__(16) float mem[ROWS][PITCH];
  __shared__ __align__(16) T zh[ROWS][ZP], zl[ROWS][ZP];
  __shared__ float scales[ROWS];
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int spans = (p.N + p.span - 1) / p.span;
  const int from = blockIdx.x % spans * p.span, to = min(p.N, from + p.span), first = blockIdx.x / spans * ROWS;
  const int id = adapter_of(p, first, lane, ROWS);
  x8 yn[PER];
  auto piece_at = [&](int i, int n0, int &row, int &n) {
    row = 16 * i + tid / 16;
    n = n0 + tid % 16 * 8;
    return first + row < p.M && n < to;
  };
  auto fetch = [&](int n0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int row, n;
      if (piece_at(i, n0, row, n)) yn[i] = *reinterpret_cast<const x8 *>(p.y + (size_t)(first + row) * p.ldy + n);
    }
  };
  fetch(from);
  // z of a row by LANES lanes, 8 ranks each: all of a thread's rows at once, SLICES of each in flight.
  constexpr int TURNS = ROWS * LANES / 256, SLICES = TURNS == 4 ? 2 : 4;
  const int rank = tid % LANES * 8;
  float z[TURNS][1][8] = {};
  int whose[TURNS];
#pragma unroll
  for (int t = 0; t < TURNS; ++t) whose[t] = __shfl(id, t * (256 / LANES) + tid / LANES);
  for (int s0 = 0; s0 < p.slices; s0 += SLICES) {
    f4 part[TURNS][SLICES][2] = {};
#pragma unroll
    for (int t = 0; t < TURNS; ++t)
#pragma unroll
      for (int s = 0; s < SLICES; ++s)
        if (s0 + s < p.slices && whose[t] >= 0 && rank < p.rank) {
          const float *const at = p.z + ((size_t)(s0 + s) * p.M + first + t * (256 / LANES) + tid / LANES) * p.rank + rank;
          part[t][s][0] = *reinterpret_cast<const f4 *>(at);
          part[t][s][1] = *reinterpret_cast<const f4 *>(at + 4);
        }
#pragma unroll
    for (int t = 0; t < TURNS; ++t)
#pragma unroll
      for (int s = 0; s < SLICES; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) z[t][0][e] += part[t][s][e / 4][e % 4];
  }
#pragma unroll
  for (int t = 0; t < TURNS; ++t) {
    const int row = t * (256 / LANES) + tid / LANES;
    float scale = whose[t] >= 0 && p.scales ? p.scales[whose[t]] : 1.0f;
    Halves<T, 1> halves;
    halves.template split<LANES>(z[t], scale);
    *reinterpret_cast<x8 *>(&zh[row][rank]) = halves.high[0];
    *reinterpret_cast<x8 *>(&zl[row][rank]) = halves.low[0];
    if (rank == 0) scales[row] = scale;
  }
  __syncthreads();
  for (int n0 = from; n0 < to; n0 += NB) {
    each_adapter(id, 0, 1, [&](int a, uint64_t mine) {
      const T *const up = p.up + (size_t)a * p.N * p.rank;
      x8 factors[2][RC];
#pragma unroll
      for (int s = 0; s < 2; ++s) {       // row j of tile s: output 8 (j / 4) + 4 s + j % 4 of the wave's 32
        const int n = min(n0 + 32 * wave + 8 * (j / 4) + 4 * s + (j & 3), p.N - 1);
#pragma unroll
        for (int c = 0; c < RC; ++c)
          factors[s][c] = 32 * c + 8 * g < p.rank ? *reinterpret_cast<const x8 *>(up + (size_t)n * p.rank + 32 * c + 8 * g) : x8{};
      }
#pragma unroll
      for (int t = 0; t < ROWS / 16; ++t) {
        if ((mine >> (16 * t) & 0xFFFF) == 0) continue;
        f4 acc[2] = {};
#pragma unroll
        for (int c = 0; c < RC; ++c) {
          const x8 h = *reinterpret_cast<const x8 *>(&zh[16 * t + j][32 * c + 8 * g]), l = *reinterpret_cast<const x8 *>(&zl[16 * t + j][32 * c + 8 * g]);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            acc[s] = Of16<T>::mma(factors[s][c], h, acc[s]);
            acc[s] = Of16<T>::mma(factors[s][c], l, acc[s]);
          }
        }
        if (mine >> (16 * t + j) & 1) {
          const float scale = scales[16 * t + j];
#pragma unroll
          for (int s = 0; s < 2; ++s) *reinterpret_cast<f4 *>(&mem[16 * t + j][32 * wave + 8 * g + 4 * s]) = acc[s] * scale;
        }
      }
    });
    __syncthreads();
    x8 y[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) y[i] = yn[i];
    if (n0 + NB < to) fetch(n0 + NB);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int row, n;
      const bool there = piece_at(i, n0, row, n);
      const int whose = __shfl(id, row);
      if (!there || (whose == -1 && p.out == p.y)) continue;
      const f4 lo = *reinterpret_cast<const f4 *>(&mem[row][n - n0]), hi = *reinterpret_cast<const f4 *>(&mem[row][n - n0 + 4]);
      x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float sum = (float)y[i][e] + (e < 4 ? lo[e] : hi[e - 4]);
        v[e] = whose >= 0 ? (T)sum : whose == -1 ? y[i][e] : (T)__builtin_nanf("");
      }
      __builtin_nontemporal_store(v, reinterpret_cast<x8 *>(p.out + (size_t)(first + row) * p.ldo + n));
    }
    __syncthreads();                      // (mem is read)
  }
}

// Both products in one launch, for few rows: a workgroup of W waves computes z of up to 16 rows of one adapter in 64 itself (its
// waves take every W-th 64 of K and meet in LDS) and `span` outputs, 64 a wave at a time, whose factors and y are requested
// before z is there.  Every span's workgroup reads the whole of A again, from the caches.  5 rows of 576 by 576, rank 8: 4.3 us, hardly
// more than an empty launch takes.
template <class T, int RT>
__global__ __launch_bounds__(64 * kRowsWaves) void adapters_rows_kernel(AdaptersParams<T> p) {
  typedef typename Of16<T>::x8 x8;
  constexpr int W = kRowsWaves, RC = (RT + 1) / 2, AHEAD = RT == 1 ? 4 : RT == 2 ? 2 : 1;
  __shared__ f4 met[W][RT][64];
  __shared__ __align__(16) float zs[16][32 * RC + 4];
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int spans = (p.N + p.span - 1) / p.span;
  const int from = blockIdx.x % spans * p.span, to = min(p.N, from + p.span), first = blockIdx.x / spans * 64;
  const int id = adapter_of(p, first, lane, 64), all = (p.K + 63) / 64;
  if (blockIdx.y == p.shares) {           // (workgroups of their own, so that no product waits for it)
    for (int i = 0; i < 64; i += 16)
      for (int n0 = from + 64 * wave; n0 < to; n0 += 64 * W) rows_without(p, id, first, i, lane, n0, min(to, n0 + 64));
    return;
  }
  each_sixteen(id, lane, p.count, blockIdx.y, p.shares, [&](int a, int at_row, int rows) {
    const bool live = j < rows;
    const int row = first + at_row;
    const T *const up = p.up + (size_t)a * p.N * p.rank;
    const T *const y = p.y + (size_t)row * p.ldy;
    T *const out = p.out + (size_t)row * p.ldo;
    Writer<T, RC> writer;
    const int mine0 = from + 64 * wave;
    if (mine0 < to) writer.begin(p, up, y, mine0, to, live, j, g);
    float scale = p.scales ? p.scales[a] : 1.0f;
    f4 acc[RT] = {};
    const T *const down = p.down + (size_t)a * p.rank * p.K + 8 * g, *const x = p.x + (size_t)row * p.ldx + 8 * g;
    for (int piece = wave; piece < all; piece += W * AHEAD) {
      x8 d[AHEAD][2][RT], xv[AHEAD][2];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int k = (piece + n * W) * 64 + 32 * c;
          const bool there = k + 8 * g < p.K;
#pragma unroll
          for (int r = 0; r < RT; ++r) d[n][c][r] = there ? *reinterpret_cast<const x8 *>(down + (size_t)min(16 * r + j, p.rank - 1) * p.K + k) : x8{};
          xv[n][c] = there && live ? *reinterpret_cast<const x8 *>(x + k) : x8{};
        }
#pragma unroll
      for (int n = 0; n < AHEAD; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int r = 0; r < RT; ++r) acc[r] = Of16<T>::mma(d[n][c][r], xv[n][c], acc[r]);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) met[wave][r][lane] = acc[r];
    __syncthreads();
    for (int i = tid; i < RT * 256; i += 64 * W) {       // element i % 4 of lane i / 4 of its tile
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += reinterpret_cast<const float *>(&met[w][0][0])[i];
      const int at = i / 4 % 64;
      zs[at & 15][16 * (i / 256) + 4 * (at >> 4) + i % 4] = sum;
    }
    __syncthreads();
    if (mine0 < to) {
      float z[RC][8];
#pragma unroll
      for (int c = 0; c < RC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) z[c][e] = live && 32 * c + 8 * g < p.rank ? zs[j][32 * c + 8 * g + e] : 0.0f;
      Halves<T, RC> halves;
      halves.split(z, scale);
      writer.run(p, up, y, out, halves, scale, mine0, to, 64 * W, live, j, g);
    }
  });
}

}  // namespace lb
