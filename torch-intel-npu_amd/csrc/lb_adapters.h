// gfx950 kernels of lb_adapters (include/lowbit_decode_hip.h): out = y + s (x A^T) B^T, the factors A [rank, K] and
// B [N, rank] those of each row's own adapter.
//
// Two launches: z = x A^T in fp32 (adapters_down_kernel), then y + s z B^T (adapters_up_kernel).  Both take tiles of rows
// as the columns of 16x16x32 products, whose rows are ranks and outputs, so that a lane holds one row throughout and rows
// of other adapters in the tile cost nothing but their share of an instruction: a tile goes once through the factors
// of each adapter that it holds, whatever their order.
#pragma once
#include "lb_serve.h"

namespace lb {

template <class T>
struct AdaptersParams {
  const T *x, *y, *down, *up;
  T *out;
  const float *scales;      // null: 1
  const int64_t *index;
  float *z;                 // [slices][M][rank]
  long long ldx, ldy, ldo;
  int M, N, K, rank, count;
  int slices;               // parts of K, added by adapters_up_kernel
  int shares;               // workgroups that share a tile's adapters
  int span;                 // adapters_up_kernel: outputs of a workgroup
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

// z of 16 MT rows over one slice of K: waves take every fourth 64 of it and meet in LDS.
template <class T, int RT, int MT>
__global__ __launch_bounds__(256) void adapters_down_kernel(AdaptersParams<T> p) {
  typedef typename Of16<T>::x8 x8;
  constexpr int W = 4, TILES = RT * MT, AHEAD = RT + MT > 5 ? 1 : RT + MT > 2 ? 2 : 4;   // pieces of 64 in flight
  __shared__ f4 met[W][TILES][64];
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slice = blockIdx.x % p.slices, first = blockIdx.x / p.slices * (16 * MT);
  const int id = adapter_of(p, first, lane, 16 * MT);
  const int all = (p.K + 63) / 64, size = (all + p.slices - 1) / p.slices, from = slice * size, to = min(all, from + size);
  const x8 none = {};
  each_adapter(id, blockIdx.y, p.shares, [&](int a, uint64_t mine) {
    f4 acc[RT][MT] = {};
    const T *const down = p.down + (size_t)a * p.rank * p.K;
    const T *dr[RT], *xr[MT];
#pragma unroll
    for (int r = 0; r < RT; ++r) dr[r] = down + (size_t)min(16 * r + j, p.rank - 1) * p.K + 8 * g;
#pragma unroll
    for (int t = 0; t < MT; ++t) xr[t] = p.x + (size_t)min(first + 16 * t + j, p.M - 1) * p.ldx + 8 * g;
    for (int piece = from + wave; piece < to; piece += W * AHEAD) {
      x8 d[AHEAD][2][RT], x[AHEAD][2][MT];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int k = (piece + n * W) * 64 + 32 * c;
          const bool there = piece + n * W < to && k + 8 * g < p.K;
#pragma unroll
          for (int r = 0; r < RT; ++r) d[n][c][r] = there ? *reinterpret_cast<const x8 *>(dr[r] + k) : none;
#pragma unroll
          for (int t = 0; t < MT; ++t) x[n][c][t] = there && (mine >> (16 * t + j) & 1) ? *reinterpret_cast<const x8 *>(xr[t] + k) : none;
        }
#pragma unroll
      for (int n = 0; n < AHEAD; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[r][t] = Of16<T>::mma(d[n][c][r], x[n][c][t], acc[r][t]);
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
      const int rank = i / MT * 16 + 4 * g, row = i % MT * 16 + j;
      if (rank < p.rank && (mine >> row & 1))
        *reinterpret_cast<f4 *>(p.z + ((size_t)slice * p.M + first + row) * p.rank + rank) = sum;
    }
  });
}

// out = y + s z B^T of 16 MT rows and `span` outputs, 64 of them a wave at a time.  z enters as the sum of two 16-bit
// numbers (16 bits of bf16 and 22 of fp16, after a power of two has brought the row's largest one below 1, so that no
// z is too large or small for fp16), so its rounding stays far below that of the output.
template <class T, int RC, int MT>
__global__ __launch_bounds__(256) void adapters_up_kernel(AdaptersParams<T> p) {
  typedef typename Of16<T>::x8 x8;
  constexpr int W = 4;
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int spans = (p.N + p.span - 1) / p.span;
  const int from = blockIdx.x % spans * p.span, to = min(p.N, from + p.span), first = blockIdx.x / spans * (16 * MT);
  const int id = adapter_of(p, first, lane, 16 * MT);
  const x8 none = {};
  if (blockIdx.y == 0) {                  // rows without an adapter, and those whose adapter there is not
    uint64_t left = __ballot(lane < 16 * MT && first + lane < p.M && id < 0 && (id == -2 || p.out != p.y));
    while (left) {
      const int row = __builtin_ctzll(left);
      left &= left - 1;
      const bool bad = __builtin_amdgcn_readlane(id, row) == -2;
      const T *const y = p.y + (size_t)(first + row) * p.ldy;
      T *const out = p.out + (size_t)(first + row) * p.ldo;
      for (int n = from + threadIdx.x; n < to; n += 64 * W) out[n] = bad ? (T)__builtin_nanf("") : y[n];
    }
  }
  each_adapter(id, blockIdx.y, p.shares, [&](int a, uint64_t mine) {
    x8 zh[RC][MT], zl[RC][MT];
    float scale[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const bool live = mine >> (16 * t + j) & 1;
      float z[RC][8], top = 0.0f;
#pragma unroll
      for (int c = 0; c < RC; ++c) {
        f4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
        if (live && 32 * c + 8 * g < p.rank)
          for (int s = 0; s < p.slices; ++s) {
            const float *const at = p.z + ((size_t)s * p.M + first + 16 * t + j) * p.rank + 32 * c + 8 * g;
            lo += *reinterpret_cast<const f4 *>(at);
            hi += *reinterpret_cast<const f4 *>(at + 4);
          }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          z[c][e] = e < 4 ? lo[e] : hi[e - 4];
          top = fmaxf(top, fabsf(z[c][e]));
        }
      }
      scale[t] = p.scales ? p.scales[a] : 1.0f;
      if constexpr (__is_same(T, f16)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const int e2 = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
        for (int c = 0; c < RC; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) z[c][e] = __builtin_amdgcn_ldexpf(z[c][e], -e2);
        scale[t] = __builtin_amdgcn_ldexpf(scale[t], e2);
      }
#pragma unroll
      for (int c = 0; c < RC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const T h = (T)z[c][e];
          const float rest = z[c][e] - (float)h;
          zh[c][t][e] = h;
          zl[c][t][e] = (T)(fabsf((float)h) < INFINITY ? rest : 0.0f);
        }
    }
    const T *const up = p.up + (size_t)a * p.N * p.rank;
    for (int n0 = from + 64 * wave; n0 < to; n0 += 64 * W) {
      f4 acc[4][MT] = {};
#pragma unroll
      for (int s = 0; s < 4; ++s) {       // row j of tile s: output 32 (s / 2) + 8 (j / 4) + 4 (s % 2) + j % 4
        const int n = min(n0 + 32 * (s / 2) + 8 * (j / 4) + 4 * (s & 1) + (j & 3), p.N - 1);
#pragma unroll
        for (int c = 0; c < RC; ++c) {
          const x8 u = 32 * c + 8 * g < p.rank ? *reinterpret_cast<const x8 *>(up + (size_t)n * p.rank + 32 * c + 8 * g) : none;
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            acc[s][t] = Of16<T>::mma(u, zh[c][t], acc[s][t]);
            acc[s][t] = Of16<T>::mma(u, zl[c][t], acc[s][t]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (!(mine >> (16 * t + j) & 1)) continue;
        const T *const y = p.y + (size_t)(first + 16 * t + j) * p.ldy;
        T *const out = p.out + (size_t)(first + 16 * t + j) * p.ldo;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int n = n0 + 32 * s + 8 * g;
          if (p.wide) {
            if (n >= to) continue;
            x8 v = *reinterpret_cast<const x8 *>(y + n);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (T)((float)v[e] + scale[t] * acc[2 * s + e / 4][t][e % 4]);
            *reinterpret_cast<x8 *>(out + n) = v;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (n + e < to) out[n + e] = (T)((float)y[n + e] + scale[t] * acc[2 * s + e / 4][t][e % 4]);
          }
        }
      }
    }
  });
}

}  // namespace lb
