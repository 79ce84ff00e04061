// What the kernels of lowbit_decode_hip.h that serve many requests share: 16-bit types and their matrix products, rows with strides, and the
// rotation of heads by their positions.
#pragma once
#include "lb_common.h"

namespace lb {

typedef __bf16 bf16;

// T x 8 and T x 4, and the 16x16x32 product of two operands of 8 (lane (j, g): row or column j, elements 8 g ..).
template <class T> struct Of16;
template <> struct Of16<f16> {
  typedef f16 x8 __attribute__((ext_vector_type(8)));
  typedef f16 x4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f4 mma(x8 a, x8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Of16<bf16> {
  typedef bf16 x8 __attribute__((ext_vector_type(8)));
  typedef bf16 x4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f4 mma(x8 a, x8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// A load of what nobody reads again soon: it leaves the caches to others.
template <class V>
__device__ __forceinline__ V read_once(const void *p) { return __builtin_nontemporal_load(static_cast<const V *>(p)); }

// Rows of contiguous values, strides in elements.
template <class T>
struct Rows {
  T *data;
  long long batch, row, head;
  __device__ __forceinline__ T *at(int b, int i, int h) const { return data + b * batch + i * row + h * head; }
};

// 64 values of 16 rows as two operands of a product (lane (j, g): row j, values 8 g .. and 32 + 8 g ..), from two loads of whole lines:
// a has rows 0 .. 7 and b rows 8 .. 15, values 8 g + 32 (j / 8) .. of row j % 8 of them.  (A load whose lanes have half a line of 16
// rows each takes the address unit twice as long.)
__device__ __forceinline__ void rows_from_lines(u4 &a, u4 &b) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t x = a[e], y = b[e];
    a[e] = __builtin_amdgcn_update_dpp(x, y, 0x128, 0xF, 0xC, false);   // row_ror 8 into lanes 8 .. 15
    b[e] = __builtin_amdgcn_update_dpp(y, x, 0x128, 0xF, 0x3, false);   // into lanes 0 .. 7
  }
}

// The rotation: pair i of the first `dims` dims turns by position * frequencies[i] (64 bits).
struct Turn {
  const double *frequencies;   // null: nothing turns
  int dims, neighbours;        // pairs (i, i + dims / 2), or (2 i, 2 i + 1)
  float scale;
};

// scale cos and scale sin of pair i at a position.  The angle is formed in 64 bits and reduced to a part of a turn there
// (at position 2^20 a product in 32 bits is off by 0.06); the sine and cosine are 32 bits' own, right to an ulp or two, and
// what the part of a turn loses in 32 bits turns them on by itself (so that a small sine is as exact as a large one).
__device__ __forceinline__ float2 turn_of(const Turn &t, int i, double position) {
  const double turns = position * t.frequencies[i] * 0.15915494309189533577, part = 2.0 * (turns - __builtin_rint(turns));
  const float half_turns = (float)part, rest = 3.14159265358979323846f * (float)(part - (double)half_turns);
  float s, c;
  sincospif(half_turns, &s, &c);
  return make_float2(t.scale * (c - s * rest), t.scale * (s + c * rest));
}

// First dim of pair i, and how far from it the second one lies.
__device__ __forceinline__ int pair_first(const Turn &t, int i) { return t.neighbours ? 2 * i : i; }
__device__ __forceinline__ int pair_step(const Turn &t) { return t.neighbours ? 1 : t.dims / 2; }

}  // namespace lb
