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
  int lanes;                // threads that share a row's heads
};

// A thread holds V pairs of a row, their sines and cosines, and goes through every `lanes`-th head of the row's queries
// and keys: the sines are computed once for those heads.  Memory bounds it: 8192 rows of 40 heads
// of 128, bf16, 168 MB in and out, take 30.6 us (5.5 TB/s); 8 rows of 12 heads of 64 4.1, which is the launch.  ONCE: the rows are
// more than the caches hold.
template <class T, int V, bool ONCE>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams<T> p) {
  typedef T Piece __attribute__((ext_vector_type(V)));
  const int turned = p.turn.dims / (2 * V), pieces = turned + p.copies;
  const unsigned at = blockIdx.x * 256u + threadIdx.x, per = pieces * p.lanes;
  const unsigned row = at / per, rest = at % per;
  if (row >= (unsigned)p.batch * p.seq) return;
  const int lane = rest / pieces, piece = rest % pieces;
  const int b = row / p.seq, i = row % p.seq;
  const int all = p.heads[0] + p.heads[1];
  // A piece's two halves: the dims of its pairs, or 2 V of those that do not turn (the last one's second half may be none).
  const bool turns = piece < turned;
  const int first = !turns ? p.turn.dims + (piece - turned) * 2 * V : p.turn.neighbours ? 2 * V * piece : V * piece;
  const int step = turns && !p.turn.neighbours ? p.turn.dims / 2 : V;
  const bool both = first + step < p.dim;
  float c[V], s[V];
  if (turns) {
    const double position = (double)(p.per_row ? p.position[row] : p.position[b] + i);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float2 cs = turn_of(p.turn, piece * V + e, position);
      c[e] = cs.x;
      s[e] = p.back ? -cs.y : cs.y;
    }
  }
  for (int h = lane; h < all; h += p.lanes) {
    const int side = h >= p.heads[0], hs = side ? h - p.heads[0] : h;
    const T *in = (side ? p.x[1] : p.x[0]).at(b, i, hs) + first;
    T *out = (side ? p.out[1] : p.out[0]).at(b, i, hs) + first;
    Piece lo = ONCE ? read_once<Piece>(in) : *reinterpret_cast<const Piece *>(in), hi = {};
    if (both) hi = ONCE ? read_once<Piece>(in + step) : *reinterpret_cast<const Piece *>(in + step);
    if (turns) {
      if (!p.turn.neighbours || V == 1) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float x = (float)lo[e], y = (float)hi[e];
          lo[e] = (T)(x * c[e] - y * s[e]);
          hi[e] = (T)(y * c[e] + x * s[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {     // pairs of lo, then of hi
          Piece &v = e < V / 2 ? lo : hi;
          constexpr int mask = V - 1;
          const float x = (float)v[2 * e & mask], y = (float)v[(2 * e + 1) & mask];
          v[2 * e & mask] = (T)(x * c[e] - y * s[e]);
          v[(2 * e + 1) & mask] = (T)(y * c[e] + x * s[e]);
        }
      }
    }
    *reinterpret_cast<Piece *>(out) = lo;
    if (both) *reinterpret_cast<Piece *>(out + step) = hi;
  }
}

}  // namespace lb
