// gfx950 kernel of lb_rotary (include/lowbit_decode_hip.h): rows of heads turned by their positions.
//
//   a' = s (a cos - b sin), b' = s (b cos + a sin) for each pair (a, b) of a head's first dims, in fp32, rounded once.
#pragma once
#include "lb_serve.h"

namespace lb {

template <class T>
struct RotaryParams {
  Rows<const T> x[2];       // queries and keys
  Rows<T> out[2];
  const int64_t *position;  // [batch] of first rows, or [batch, seq]
  Turn turn;
  int batch, seq, dim, heads[2], per_row, back;
  int copies;               // pieces of 2 V dims behind the turned ones, to be copied (0 in place)
  int lanes;                // of a wave that share a row's heads
  int rows, shares;         // of a wave; waves that share a row's heads
};

// A wave takes `rows` rows, and where they have many heads one of their `shares`.  It computes the rows' sines and cosines once, a pair or
// two a lane, behind the first loads of what they turn, and hands them round in LDS; then a lane turns V pairs of a row in every
// `lanes` x `shares`-th head.  (Each lane computing its own eight held the vector units for 93% of the time.)  Memory bounds it: 8192 rows
// of 40 heads of 128, bf16, 168 MB in and out, take 31 us (5.4 TB/s), 2048 of them 9.6 (their inputs in the caches); 8 rows of 12
// heads of 64 3.8, which is the launch.  ONCE: the rows are more than the caches hold.
template <class T, int V, bool ONCE>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams<T> p) {
  typedef T Piece __attribute__((ext_vector_type(V)));
  __shared__ __align__(16) float2 held[4][512];      // (64 pieces of 8 pairs at the most, or a row of up to 1024 dims)
  const int tid = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float2 *const angles = held[wave];
  const int half = p.turn.dims / 2, turned = half / V, pieces = turned + p.copies, per = pieces * p.lanes;
  const unsigned share = p.shares == 1 ? 0 : blockIdx.x % p.shares, block = p.shares == 1 ? blockIdx.x : blockIdx.x / p.shares;
  const unsigned row0 = (block * 4 + wave) * (unsigned)p.rows, end = (unsigned)p.batch * p.seq;
  if (row0 >= end) return;
  const unsigned rows = min((unsigned)p.rows, end - row0);
  const int all = p.heads[0] + p.heads[1];
  bool ready = false;
  for (int slot = tid; slot < p.rows * per || !ready; slot += 64) {
    const int r = slot / per, rest = slot % per, lane = rest / pieces + share * p.lanes, piece = rest % pieces;
    const bool there = (unsigned)r < rows;
    const unsigned row = row0 + min((unsigned)r, rows - 1);
    const int b = row / p.seq, i = row % p.seq;
    // A piece's two halves: the dims of its pairs, or 2 V of those that do not turn (the last one's second half may be none).
    const bool turns = piece < turned;
    const int first = !turns ? p.turn.dims + (piece - turned) * 2 * V : p.turn.neighbours ? 2 * V * piece : V * piece;
    const int step = turns && !p.turn.neighbours ? half : V;
    const bool both = first + step < p.dim;
    float c[V], s[V];
    for (int h = lane; h < all || !ready; h += p.shares * p.lanes) {
      const bool live = there && h < all;
      const int side = h >= p.heads[0], hs = side ? h - p.heads[0] : h;
      Piece lo = {}, hi = {};
      if (live) {
        const T *const in = (side ? p.x[1] : p.x[0]).at(b, i, hs) + first;
        lo = ONCE ? read_once<Piece>(in) : *reinterpret_cast<const Piece *>(in);
        if (both) hi = ONCE ? read_once<Piece>(in + step) : *reinterpret_cast<const Piece *>(in + step);
      }
      if (!ready) {                       // (the first time round, for all lanes at once)
        ready = true;
        for (int k = tid; k < (int)rows * half; k += 64) {
          const unsigned at = row0 + k / half;
          angles[k] = turn_of(p.turn, k % half, (double)(p.per_row ? p.position[at] : p.position[at / p.seq] + at % p.seq));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      if (!live) break;
      if (turns) {
        if (h == lane) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float2 cs = angles[r * half + piece * V + e];
            c[e] = cs.x;
            s[e] = p.back ? -cs.y : cs.y;
          }
        }
        if (!p.turn.neighbours || V == 1) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float x = (float)lo[e], y = (float)hi[e];
            lo[e] = (T)(x * c[e] - y * s[e]);
            hi[e] = (T)(y * c[e] + x * s[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {   // pairs of lo, then of hi
            Piece &v = e < V / 2 ? lo : hi;
            constexpr int mask = V - 1;
            const float x = (float)v[2 * e & mask], y = (float)v[(2 * e + 1) & mask];
            v[2 * e & mask] = (T)(x * c[e] - y * s[e]);
            v[(2 * e + 1) & mask] = (T)(y * c[e] + x * s[e]);
          }
        }
      }
      T *const out = (side ? p.out[1] : p.out[0]).at(b, i, hs) + first;
      *reinterpret_cast<Piece *>(out) = lo;
      if (both) *reinterpret_cast<Piece *>(out + step) = hi;
    }
  }
}

}  // namespace lb
