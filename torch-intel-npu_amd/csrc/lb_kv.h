// gfx950 kernels of the 8-bit KV cache (include/lowbit_decode_hip.h: lb_kv_append, lb_kv_read, lb_kv_attention).
//
// A block of 64 slots of one sequence and KV head is quantised as a whole when its last row arrives:
// a = max |x|, int8 code rint(127 x / a) or fp8 code e4m3(448 x / a), scale a / 127 or a / 448 in fp32.  The rows of
// the open block and of the one before it stay in fp16 in a ring of two blocks.
//
// Keys lie by slot, values by dim, each value row's slots in the order of kv_place.  Both are then A operands of
// v_mfma_f32_16x16x32_f16 as they lie: a lane's 16 bytes are 16 dims of a key (two K steps of K.Q^T) or, of a value
// dim, the 16 slots whose probabilities the lane holds as the result of K.Q^T, so neither probabilities nor values
// cross lanes, and a wave's load is 1 KB of consecutive memory.
#pragma once
#include <type_traits>

#include "lb_common.h"

namespace lb {

constexpr int kKvBlock = 64;
enum KvFormat { KV_INT8 = 0, KV_FP8 = 1 };

typedef f16 h4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));

struct KvCache {
  uint8_t *kc, *vc;       // codes [batch, kv_heads, capacity, D], [batch, kv_heads, blocks, D, 64]
  float *ks, *vs;         // [batch, kv_heads, blocks]
  f16 *kt, *vt;           // tails [batch, kv_heads, 2, 64, D], [batch, kv_heads, 2, D, 64]
  int kv_heads, capacity, blocks;
};

// fp16 rows of D contiguous values.
struct KvRows {
  f16 *data;
  long long batch, row, head;   // strides in elements
  __device__ __forceinline__ f16 *at(int b, int i, int h) const { return data + b * batch + i * row + h * head; }
};

// Place of a slot in a value row: slot 16 s + 4 g + r at 16 g + 4 s + r.  (Its own inverse: it swaps s and g.)
__host__ __device__ __forceinline__ constexpr int kv_place(int slot) {
  return (slot >> 2 & 3) << 4 | (slot >> 4 & 3) << 2 | (slot & 3);
}

// First slot and number of rows of sequence b; false where they do not lie in the cache.
__device__ __forceinline__ bool kv_span(const int64_t *position, const int64_t *rows, int b, int seq, int capacity, int &first,
                                        int &count) {
  const int64_t at = position[b], n = rows ? rows[b] : seq;
  first = (int)at;
  count = (int)n;
  return at >= 0 && n >= 0 && n <= seq && at <= capacity - n;
}

// fp16(fp16(t cos) + fp16(rotate_half(t) sin)) of 8 dims from `dim` on, `other` the 8 dims half a head away: the
// reference's rounding points (torch_npu_smollm.py:169-173), with no product fused into the sum.
template <int D>
__device__ __forceinline__ h8 kv_rotate(h8 t, h8 other, const f16 *cos, const f16 *sin, int pos, int dim) {
#pragma clang fp contract(off)
  const h8 cs = *reinterpret_cast<const h8 *>(cos + (size_t)pos * D + dim);
  const h8 sn = *reinterpret_cast<const h8 *>(sin + (size_t)pos * D + dim);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const f16 o = dim < D / 2 ? (f16)-other[e] : other[e];
    const f16 t0 = (f16)((float)t[e] * (float)cs[e]), t1 = (f16)((float)o * (float)sn[e]);
    t[e] = (f16)((float)t0 + (float)t1);
  }
  return t;
}

// Largest magnitude of 8 values as fp16 bits (infinities and NaNs are the largest).
__device__ __forceinline__ uint32_t kv_top(h8 v) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t bits = __builtin_bit_cast(uint16_t, (f16)v[e]) & 0x7FFFu;
    top = bits > top ? bits : top;
  }
  return top;
}

template <int FMT> __device__ __forceinline__ constexpr float kv_limit() { return FMT == KV_INT8 ? 127.0f : 448.0f; }

// Codes of four values, x of at most the block's top, r = limit / top.  x and top have 11 bits and the limits 7 and 3, so
// limit x / top is either exactly between two codes or at least 2^-19 of itself away from there.  x r is off by 2^-23 at
// most: rounded to 20 bits it is the former exactly and never crosses to the latter's other side, so that the code is
// that of the exact quotient.
template <int FMT>
__device__ __forceinline__ uint32_t kv_encode4(f16 x0, f16 x1, f16 x2, f16 x3, float r) {
  float t[4] = {(float)x0, (float)x1, (float)x2, (float)x3};
#pragma unroll
  for (int e = 0; e < 4; ++e) t[e] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, t[e] * r) + 8u) & ~15u);
  if constexpr (FMT == KV_INT8) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __builtin_bit_cast(uint32_t, t[e] + 12582912.0f);  // 1.5 * 2^23: the integer in the low bits
    return __builtin_amdgcn_perm(w[1], w[0], 0x0C0C0400u) | __builtin_amdgcn_perm(w[3], w[2], 0x0C0C0400u) << 16;
  } else {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], w, true);
  }
}

// Eight codes (two dwords) as fp16, exact, in the order of kv_order8.
template <int FMT>
__device__ __forceinline__ h8 kv_decode8(uint32_t w0, uint32_t w1) {
  h2 p[4];
  if constexpr (FMT == KV_INT8) {
    int8_pairs(w0, p);
    int8_pairs(w1, p + 2);
  } else {
    p[0] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false));
    p[1] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true));
    p[2] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false));
    p[3] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true));
  }
  return __builtin_shufflevector(__builtin_shufflevector(p[0], p[1], 0, 1, 2, 3),
                                 __builtin_shufflevector(p[2], p[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}
// The order in which kv_decode8 gives its codes, for what they are multiplied with.
template <int FMT>
__device__ __forceinline__ h8 kv_order8(h8 v) {
  if constexpr (FMT == KV_INT8) return __builtin_shufflevector(v, v, 0, 2, 1, 3, 4, 6, 5, 7);
  return v;
}

// ------------------------------------------------------------------------------------------------ append
// What a thread holds of a block while it is quantised: 8 dims of 4 consecutive slots, keys and values.
template <int D>
struct KvQuad {
  static constexpr int CH = D / 8, THREADS = 2 * D;   // chunks of 8 dims; threads of a block
  h8 k[4], v[4];
};
template <int D>
struct KvTurn {                                       // LDS of kv_close
  static constexpr int PITCH = 20;                    // dwords of a value row (16 and padding)
  uint32_t tops[2][KvQuad<D>::THREADS / 64];
  __align__(16) uint32_t rows[D * PITCH];
};

// A key of NaNs where the row's key or value is not finite; D / 8 neighbouring lanes hold the row.
template <int D>
__device__ __forceinline__ void kv_poison(h8 &k, h8 v) {
  uint32_t bad = kv_top(k) >= 0x7C00u || kv_top(v) >= 0x7C00u;
#pragma unroll
  for (int d = KvQuad<D>::CH / 2; d > 0; d >>= 1) bad |= __shfl_xor(bad, d);
  if (bad)
#pragma unroll
    for (int e = 0; e < 8; ++e) k[e] = __builtin_bit_cast(f16, (uint16_t)0x7E00u);
}

// Quantises a full block from the registers of threads 0 .. 2 D - 1 (the others only meet the barriers): tops over the
// workgroup, key codes as they lie, value codes turned into rows by dim through LDS, where a thread's 4 slots are one
// dword.
template <int FMT, int D>
__device__ __forceinline__ void kv_close(const KvCache &c, size_t bh, int block, const KvQuad<D> &x, KvTurn<D> &turn, int tid) {
  constexpr int CH = KvQuad<D>::CH, THREADS = KvQuad<D>::THREADS, PITCH = KvTurn<D>::PITCH;
  const int dim = 8 * (tid % CH), quad = tid / CH;
  const bool mine = tid < THREADS;
  uint32_t top[2] = {0, 0};
  if (mine) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      top[0] = max(top[0], kv_top(x.k[i]));
      top[1] = max(top[1], kv_top(x.v[i]));
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) top[s] = max(top[s], (uint32_t)__shfl_xor((int)top[s], d));
      if ((tid & 63) == 0) turn.tops[s][tid >> 6] = top[s];
    }
  }
  __syncthreads();
  float scale[2], r[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) top[s] = max(top[s], turn.tops[s][w]);
    const float a = (float)__builtin_bit_cast(f16, (uint16_t)top[s]);
    const bool bad = top[s] >= 0x7C00u;
    scale[s] = bad ? __builtin_nanf("") : a / kv_limit<FMT>();
    r[s] = bad || top[s] == 0 ? 0.0f : kv_limit<FMT>() / a;
  }
  const bool kbad = top[0] >= 0x7C00u, vbad = top[1] >= 0x7C00u;
  const size_t base = (bh * c.capacity + (size_t)block * kKvBlock) * D;
  if (tid == 0) {
    c.ks[bh * c.blocks + block] = scale[0];
    c.vs[bh * c.blocks + block] = scale[1];
  }
  if (mine) {
    uint8_t *const kc = c.kc + base + 4 * quad * D + dim;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const h8 k = x.k[i];
      *reinterpret_cast<u2v *>(kc + i * D) = u2v{kbad ? 0u : kv_encode4<FMT>(k[0], k[1], k[2], k[3], r[0]),
                                                 kbad ? 0u : kv_encode4<FMT>(k[4], k[5], k[6], k[7], r[0])};
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      turn.rows[(dim + e) * PITCH + kv_place(4 * quad) / 4] =
          vbad ? 0u : kv_encode4<FMT>(x.v[0][e], x.v[1][e], x.v[2][e], x.v[3][e], r[1]);
  }
  __syncthreads();
  if (mine) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {         // D rows of four 16-byte pieces
      const int piece = tid + i * THREADS;
      *reinterpret_cast<u4 *>(c.vc + base + 16 * piece) = *reinterpret_cast<const u4 *>(&turn.rows[piece / 4 * PITCH + piece % 4 * 4]);
    }
  }
}

// The rows of a block that lie in the tails, but for those in `have`.
template <int D>
__device__ __forceinline__ void kv_from_tails(const KvCache &c, size_t bh, int block, uint32_t have, KvQuad<D> &x, int tid) {
  const int dim = 8 * (tid % KvQuad<D>::CH), quad = tid / KvQuad<D>::CH;
  const size_t half = (2 * bh + (block & 1)) * (kKvBlock * D);
  const f16 *const kd = c.kt + half + 4 * quad * D + dim, *const vd = c.vt + half + dim * kKvBlock + kv_place(4 * quad);
  h4 v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const h4 *>(vd + e * kKvBlock);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (have >> i & 1) continue;
    x.k[i] = *reinterpret_cast<const h8 *>(kd + i * D);
#pragma unroll
    for (int e = 0; e < 8; ++e) x.v[i][e] = v[e][i];
  }
}

// Quantises a block whose 64 rows all lie in the tails, by a workgroup of W waves: codes lie as the tails do, so
// elements are encoded where they are.  A few values a thread at a time: it stands in the middle of kv_attend_kernel, whose
// registers are full, and one step in 64 comes here.  tops: W words of LDS that nobody uses.
template <int FMT, int D, int W>
__device__ __forceinline__ void kv_close_tails(const KvCache &c, size_t bh, int block, uint32_t *tops, int tid) {
  const size_t half = (2 * bh + (block & 1)) * (kKvBlock * D), base = (bh * c.capacity + (size_t)block * kKvBlock) * D;
#pragma unroll 1
  for (int s = 0; s < 2; ++s) {
    const f16 *const tail = (s == 0 ? c.kt : c.vt) + half;
    uint32_t top = 0;
#pragma unroll 1
    for (int i = tid; i < 8 * D; i += 64 * W) top = max(top, kv_top(*reinterpret_cast<const h8 *>(tail + 8 * i)));
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    __syncthreads();
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) top = max(top, tops[w]);
    const float a = (float)__builtin_bit_cast(f16, (uint16_t)top);
    const bool bad = top >= 0x7C00u;
    const float r = bad || top == 0 ? 0.0f : kv_limit<FMT>() / a;
    if (tid == 0) (s == 0 ? c.ks : c.vs)[bh * c.blocks + block] = bad ? __builtin_nanf("") : a / kv_limit<FMT>();
    uint8_t *const codes = (s == 0 ? c.kc : c.vc) + base;
#pragma unroll 1
    for (int i = tid; i < 8 * D; i += 64 * W) {
      const h8 x = *reinterpret_cast<const h8 *>(tail + 8 * i);
      *reinterpret_cast<u2v *>(codes + 8 * i) = u2v{bad ? 0u : kv_encode4<FMT>(x[0], x[1], x[2], x[3], r),
                                                    bad ? 0u : kv_encode4<FMT>(x[4], x[5], x[6], x[7], r)};
    }
  }
}

struct KvAppendParams {
  KvCache c;
  KvRows k, v;
  const int64_t *position, *rows;
  const f16 *cos, *sin;
  int seq;
};

// One workgroup of 2 D threads per block of 64 slots that new rows fall into, KV head and sequence.  A block that
// becomes full takes its older rows from the tails; rows of the last block and of the one before it go to the tails.
// Each thread holds 8 dims of 4 slots, so that a block is read once, in 16-byte pieces, and a value's 4 slots are one
// dword of the turned codes.  Bound by memory for prompts (four prompts of up to 4100 rows, 8 heads of 128, fp8: 69 MB
// in 18.0 us, 3.8 TB/s), by its launch and one chain of loads for single tokens (64 sequences, 3 heads of 64: 4.8 us, 6.0 where
// blocks become full).
template <int FMT, int D>
__global__ __launch_bounds__(2 * D) void kv_append_kernel(KvAppendParams p) {
  __shared__ KvTurn<D> turn;
  const int tid = threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int dim = 8 * (tid % KvQuad<D>::CH), quad = tid / KvQuad<D>::CH;
  int first, count;
  if (!kv_span(p.position, p.rows, b, p.seq, p.c.capacity, first, count)) return;
  const int end = first + count, oldest = first / kKvBlock, block = oldest + blockIdx.x, base = block * kKvBlock;
  if (count == 0 || base >= end) return;
  const int kept = end / kKvBlock - 1;    // rows from this block on go to the tails
  // The block that was open reads its older rows from its half of the tails.  Blocks of the same half that are written
  // there by the same call wait for that: its own workgroup writes their rows, at the end.
  const bool reads = first % kKvBlock != 0, after = reads && block >= oldest + 2;
  const size_t bh = (size_t)b * p.c.kv_heads + h;

  KvQuad<D> x;
  auto load = [&](int base) {             // the new rows of a block; a bit for each that there is
    uint32_t have = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int slot = base + 4 * quad + i, row = slot - first;
      x.k[i] = x.v[i] = h8{0, 0, 0, 0, 0, 0, 0, 0};
      if (row < 0 || slot >= end) continue;
      have |= 1u << i;
      const f16 *at = p.k.at(b, row, h);
      x.k[i] = *reinterpret_cast<const h8 *>(at + dim);
      x.v[i] = *reinterpret_cast<const h8 *>(p.v.at(b, row, h) + dim);
      if (p.cos) x.k[i] = kv_rotate<D>(x.k[i], *reinterpret_cast<const h8 *>(at + (dim ^ D / 2)), p.cos, p.sin, slot, dim);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) kv_poison<D>(x.k[i], x.v[i]);
    return have;
  };
  auto keep = [&](int block, uint32_t have) {   // the new rows of a block to its half of the tails
    const size_t half = (2 * bh + (block & 1)) * (kKvBlock * D);
    f16 *const kd = p.c.kt + half + 4 * quad * D + dim, *const vd = p.c.vt + half + dim * kKvBlock + kv_place(4 * quad);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (have >> i & 1) *reinterpret_cast<h8 *>(kd + i * D) = x.k[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (have == 15u) {
        *reinterpret_cast<h4 *>(vd + e * kKvBlock) = h4{x.v[0][e], x.v[1][e], x.v[2][e], x.v[3][e]};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (have >> i & 1) vd[e * kKvBlock + i] = x.v[i][e];
      }
    }
  };

  const uint32_t have = load(base);
  if (base + kKvBlock <= end) {
    if (block == oldest && reads) kv_from_tails<D>(p.c, bh, block, have, x, tid);
    kv_close<FMT, D>(p.c, bh, block, x, turn, tid);
  }
  if (block >= kept && !after) keep(block, have);
  if (blockIdx.x == 0 && reads) {         // (behind the barriers after its own reads, where there were any)
    for (int later = max(oldest + 2, kept); later * kKvBlock < end; ++later) keep(later, load(later * kKvBlock));
  }
}

// ------------------------------------------------------------------------------------------------ read
struct KvReadParams {
  KvCache c;
  const int64_t *length;
  KvRows keys, values;
  int start, count;
};

// One workgroup of 2 D threads per block, KV head and sequence.  Keys are decoded where they lie, 8 dims of 4 slots a
// thread; value codes are fetched 16 bytes at a time and turned into rows by slot through LDS.  Bound by memory: of
// 3 bytes moved per value, two are written (131000 slots, 8 heads of 128, int8: 805 MB in 140 us, 5.7 TB/s).
template <int FMT, int D>
__global__ __launch_bounds__(2 * D) void kv_read_kernel(KvReadParams p) {
  constexpr int CH = D / 8, PITCH = 20;
  __shared__ __align__(16) uint32_t turn[D * PITCH];
  const int tid = threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int dim = 8 * (tid % CH), quad = tid / CH;
  const int64_t length = p.length[b];
  const bool bad = length < 0 || length > p.c.capacity;
  const int held = bad ? p.c.capacity : (int)length;
  const int block = p.start / kKvBlock + blockIdx.x, base = block * kKvBlock;
  const int last = min(p.start + p.count, held);     // slots start .. last - 1 are written
  if (base >= last) return;
  const size_t bh = (size_t)b * p.c.kv_heads + h;
  const bool full = base + kKvBlock <= held;
  h8 k[4], v[4];
  if (bad) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) k[i][e] = v[i][e] = __builtin_bit_cast(f16, (uint16_t)0x7E00u);
  } else if (full) {
    const uint8_t *const kc = p.c.kc + (bh * p.c.capacity + base) * D + 4 * quad * D + dim;
    const uint8_t *const vc = p.c.vc + (bh * p.c.capacity + base) * D;
    const float ks = p.c.ks[bh * p.c.blocks + block], vs = p.c.vs[bh * p.c.blocks + block];
    u2v w[4];
    u4 piece[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const u2v *>(kc + i * D);
#pragma unroll
    for (int i = 0; i < 2; ++i) piece[i] = *reinterpret_cast<const u4 *>(vc + 16 * (tid + i * 2 * D));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = tid + i * 2 * D;
      *reinterpret_cast<u4 *>(&turn[at / 4 * PITCH + at % 4 * 4]) = piece[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const h8 c = kv_order8<FMT>(kv_decode8<FMT>(w[i][0], w[i][1]));   // (the order is its own inverse)
#pragma unroll
      for (int e = 0; e < 8; ++e) k[i][e] = (f16)((float)c[e] * ks);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const int at = kv_place(4 * quad) / 4;
      const h8 c = kv_order8<FMT>(kv_decode8<FMT>(turn[(dim + e) * PITCH + at], turn[(dim + e + 1) * PITCH + at]));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i][e] = (f16)((float)c[i] * vs);
        v[i][e + 1] = (f16)((float)c[4 + i] * vs);
      }
    }
  } else {
    const f16 *const kd = p.c.kt + bh * (2 * kKvBlock * D) + (block & 1) * (kKvBlock * D) + 4 * quad * D + dim;
    const f16 *const vd = p.c.vt + bh * (2 * kKvBlock * D) + (block & 1) * (kKvBlock * D) + dim * kKvBlock + kv_place(4 * quad);
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = *reinterpret_cast<const h8 *>(kd + i * D);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const h4 t = *reinterpret_cast<const h4 *>(vd + e * kKvBlock);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i][e] = t[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int slot = base + 4 * quad + i;
    if (slot < p.start || slot >= last) continue;
    *reinterpret_cast<h8 *>(p.keys.at(b, slot - p.start, h) + dim) = k[i];
    *reinterpret_cast<h8 *>(p.values.at(b, slot - p.start, h) + dim) = v[i];
  }
}

// ------------------------------------------------------------------------------------------------ attention
struct KvAttendParams {
  KvCache c;
  KvRows q, out, k, v;    // k.data null: the rows are in the cache
  const int64_t *position, *rows;
  const f16 *cos, *sin;
  uint32_t *tickets;      // kKvTickets zero words
  float *partial;         // [parts][R][D] sums, then [parts][R][2] maxima and totals
  int batch, seq, group;  // group: query heads of a KV head
  int tiles, splits;      // kv_prompt_kernel: row tiles of a KV head, parts that a tile's slots are taken in at the most
  float scale;            // score scale * log2(e)
};

constexpr float kKvLowest = -1e30f;   // a running maximum below every score (scores are under 1e17 in magnitude)
// Probabilities are 2^kKvLift above 1 at a row's running maximum, which is raised where a score exceeds it by more than
// kKvSlack (in units of log2): fp16 then has them in [2^-24, 2^14], of which the smallest are 2^-34 of the largest.
constexpr float kKvLift = 10.0f, kKvSlack = 4.0f;
// The lift minus the maximum is one addend of a block's scores, which is off by half a step of the maximum: by 2^-15 here,
// in a probability a twentieth of its rounding to fp16, but by the whole lift from 2^27 on.  So a maximum further from zero
// than this is subtracted from the scores first (0 to 1.5% of a call for asking).
constexpr float kKvFar = 1024.0f;
constexpr int kKvTickets = 1024;      // (LB_ZEROED_WORKSPACE_BYTES)
constexpr int kKvChunk = 8;           // kv_prompt_kernel: blocks of a part at the least
// kv_attend_kernel: parts that the whole work is split into at the most, besides those that sequences and heads are by
// themselves (the CUs); blocks of a part at the least (one a wave); and places for the sums of parts.
constexpr int kKvSplit = 256, kKvLeast = 4, kKvPlaces = 2 * kKvSplit + 2;

// Inclusive prefix sum over the wave's lanes, in data-parallel shifts of rows of 16 and broadcasts of their ends.
__device__ __forceinline__ uint32_t kv_scan(uint32_t x) {
  x += __builtin_amdgcn_update_dpp(0u, x, 0x111, 0xF, 0xF, true);   // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0u, x, 0x112, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0u, x, 0x114, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0u, x, 0x118, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0u, x, 0x142, 0xA, 0xF, false);  // row_bcast 15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0u, x, 0x143, 0xC, 0xF, false);  // row_bcast 31 into rows 2 and 3
  return x;
}

// A value that is the same in every lane, as one.
__device__ __forceinline__ float kv_uniform(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}

// The largest over the four lanes that hold a query.
__device__ __forceinline__ float kv_max_across(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}

// Counts a part of a unit whose sums this workgroup has written; true in the one that counts last, which leaves the
// ticket zero for the next call.
__device__ __forceinline__ bool kv_last_part(uint32_t *ticket, uint32_t parts, uint32_t *word) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wave's sums are written through
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM) == parts - 1;
    if (last) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    *word = last;
  }
  __syncthreads();
  return *word != 0;
}

// Adds the parts of `rows` rows of D sums, part k in place(k) of po [..][R][D] and pm [..][R][2], and stores the
// quotients.  Many rows: a thread has four quads of dims and four parts of each in flight (509 rows over 32768 slots, four
// parts of 128 rows of 128: 330 -> 322 us; 1024 rows of heads of 64 in two parts 23 -> 19).  Few rows: their quads of
// dims times as many runs of parts as there are threads for, which meet in LDS (`met`, 24 bytes a thread).  The order of
// the additions depends on sizes alone.
template <int R, int D, int NT, class Place, class Store>
__device__ __forceinline__ void kv_join(__amdgpu_buffer_rsrc_t po, __amdgpu_buffer_rsrc_t pm, int rows, uint32_t parts, Place &&place,
                                        f4 *met, Store &&store) {
  constexpr int DQ = D / 4, HELD = 8;     // parts in flight
  constexpr int kOutOfRange = (int)0x80000000u;
  const int tid = threadIdx.x, items = rows * DQ, runs = max(1, NT / items);
  if constexpr (R > 32) {                 // many rows: four a thread at once, four parts of each in flight
    constexpr int U = 4, PARTS = 4;
    if (runs == 1) {
      for (int at = tid; at < items; at += U * NT) {
        float most[U], sum[U];
        f4 o[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          most[u] = kKvLowest;
          sum[u] = 0.0f;
          o[u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (uint32_t i = 0; i < parts; i += PARTS) {
          f4 part[U][PARTS];
          u2v ml[U][PARTS];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int item = at + u * NT, r = item / DQ, d = item % DQ * 4;
#pragma unroll
            for (int e = 0; e < PARTS; ++e) {
              const bool there = i + e < parts && item < items;
              const uint32_t s = place(i + e);
              part[u][e] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(po, there ? (int)((s * R + r) * D + d) * 4 : kOutOfRange, 0, kSysCoherent));
              ml[u][e] = __builtin_amdgcn_raw_buffer_load_b64(pm, there ? (int)(s * R + r) * 8 : kOutOfRange, 0, kSysCoherent);
            }
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            float raised = most[u], top[PARTS];
#pragma unroll
            for (int e = 0; e < PARTS; ++e) {
              top[e] = i + e < parts ? __builtin_bit_cast(float, (uint32_t)ml[u][e][0]) : kKvLowest;
              raised = fmaxf(raised, top[e]);
            }
            const float shrink = __builtin_amdgcn_exp2f(most[u] - raised);
            most[u] = raised;
            sum[u] *= shrink;
            o[u] *= shrink;
#pragma unroll
            for (int e = 0; e < PARTS; ++e) {
              const float f = __builtin_amdgcn_exp2f(top[e] - raised);
              sum[u] += f * __builtin_bit_cast(float, (uint32_t)ml[u][e][1]);
              o[u] += f * part[u][e];
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (at + u * NT < items) store((at + u * NT) / DQ, (at + u * NT) % DQ * 4, o[u], sum[u]);
      }
      return;
    }
  }
  for (int at = 0; at < items; at += NT) {
    const int item = at + (runs > 1 ? tid % items : tid), run = runs > 1 ? tid / items : 0;
    const int r = item / DQ, d = item % DQ * 4;
    const bool live = item < items && run < runs;
    float most = kKvLowest, sum = 0.0f;
    f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t i = run; live && i < parts; i += HELD * runs) {
      f4 part[HELD];
      float ml[HELD][2];
#pragma unroll
      for (int e = 0; e < HELD; ++e) {
        const uint32_t k = i + e * runs, s = place(k);
        part[e] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(po, k < parts ? (int)((s * R + r) * D + d) * 4 : kOutOfRange, 0, kSysCoherent));
        const u2v m = __builtin_amdgcn_raw_buffer_load_b64(pm, k < parts ? (int)(s * R + r) * 8 : kOutOfRange, 0, kSysCoherent);
        ml[e][0] = k < parts ? __builtin_bit_cast(float, (uint32_t)m[0]) : kKvLowest;
        ml[e][1] = __builtin_bit_cast(float, (uint32_t)m[1]);
      }
      float raised = most;
#pragma unroll
      for (int e = 0; e < HELD; ++e) raised = fmaxf(raised, ml[e][0]);
      const float shrink = __builtin_amdgcn_exp2f(most - raised);
      most = raised;
      sum *= shrink;
      o *= shrink;
#pragma unroll
      for (int e = 0; e < HELD; ++e) {
        const float f = __builtin_amdgcn_exp2f(ml[e][0] - most);
        sum += f * ml[e][1];
        o += f * part[e];
      }
    }
    if (runs == 1) {
      if (live) store(r, d, o, sum);
      continue;
    }
    float *const stats = reinterpret_cast<float *>(met + NT);
    if (live) {
      met[tid] = o;
      stats[2 * tid] = most;
      stats[2 * tid + 1] = sum;
    }
    __syncthreads();
    if (run == 0) {
      for (int k = 1; k < runs; ++k) {
        const int other = k * items + item;
        const float raised = fmaxf(most, stats[2 * other]);
        const float f0 = __builtin_amdgcn_exp2f(most - raised), f1 = __builtin_amdgcn_exp2f(stats[2 * other] - raised);
        most = raised;
        sum = sum * f0 + stats[2 * other + 1] * f1;
        o = o * f0 + met[other] * f1;
      }
      store(r, d, o, sum);
    }
  }
}

// Attention of few query rows: those of a KV head (row i of the call and query head g of the group: row i group + g) fit
// R = 16 QT.  A workgroup takes a sequence and KV head, its four waves every fourth block each, with a running maximum
// and total of their own, joined in LDS.  Where a sequence and head has more than a 256th of the whole work it is split
// into parts of at most that; a part's sums are left in memory and the workgroup that counts last (kv_last_part) adds
// them.  All of this is found from the positions, on the device.
//   - Splitting pays down to one block a wave: a CU by itself draws only 50 to 85 GB/s (one sequence of 4096 slots, 8 heads
//     of 128: parts of 4, 16 and 64 blocks take 8.5, 12.8 and 27.9 us; eight waves a workgroup 9.3, 13.5 and 26.6).
//   - A workgroup takes one part: going on with another costs a whole chain of waits, 4 us (64 sequences of 1 to 8192
//     slots, 8 heads of 128, equal shares cut across sequences: 128 us).
//   - Longer sequences first, and every other 256 workgroups backwards, so that the two that share a CU have together what
//     others have: the same 64 sequences 100 us (5.4 TB/s) against 118 in the batch's order.  (Up to 64 sequences, by
//     prefix sums in registers; sorting them outright took 50 ns a sequence.)  Larger batches keep their own order, and every
//     workgroup goes through the positions up to its sequence's: 1.2 us for 65 sequences, but as the square of the batch
//     beyond (one block a sequence, 3 heads of 64: 256 sequences 7.1 us, 1024 27.7, 4096 195).
//   - At 5 TB/s and more the loads in flight are what HBM takes; short ones are bound by the chain of position, codes, two
//     products and the join: 4.2 us for one sequence of 150 slots and 3 heads of 64, 12.6 for 32 of 1984 with the append.
//   - Of two query tiles 128 dims take 354 registers, one wave a SIMD: 64 sequences of 8192 slots, 8 KV heads of 128, five
//     rows of four query heads 195 us (5.5 TB/s) against 189 for four rows in one tile; 16 of 4000 slots 39 against 30.
//
// Scores are K.Q^T and outputs V^T.P^T, so that a lane holds one query throughout (column lane % 16): its maximum,
// total and rescaling are the lane's own, and the probabilities that it computes are the B operand of the second product
// as they are, rounded to fp16 (relative 2^-11, as every output is; the total sums the rounded ones).  Codes enter both
// products exactly as fp16 and the block's scales multiply fp32 sums.  The maximum is raised only where a block exceeds
// it by more than kKvSlack: until then nothing has to cross lanes.
//
// With k and v (one row a sequence) the workgroup that has a sequence's last block appends the row and, where that fills
// the block, quantises it, while the other blocks are under way, and takes that block behind a barrier.
template <int FMT, int D, int QT>
__global__ __launch_bounds__(256, (D == 64 && QT == 1 ? 4 : QT * D > 128 ? 1 : 2)) void kv_attend_kernel(KvAttendParams p) {
  constexpr int W = 4, NT = 64 * W, R = 16 * QT, H = D / 64, DT = D / 16, PITCH = D + 4, DQ = D / 4;
  constexpr bool TIGHT = QT * D > 128;  // two tiles of 128 dims leave no registers for an open block's rows all at once
  struct Sums {
    float sums[W][R][PITCH];
    float tops[W][R], totals[W][R];
  };
  __shared__ __align__(16) Sums mem;
  __shared__ uint32_t found[8], tops[W], sum_of[2][W];
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};

  // Blocks of a sequence: those of its slots, none without rows, and one (to write NaNs) where it lies outside the cache.
  auto blocks_of = [&](bool fine, int first, int count) -> uint32_t {
    return !fine ? 1 : count == 0 ? 0 : (first + count + kKvBlock - 1) / kKvBlock;
  };
  auto blocks_at = [&](int b) {
    int first, count;
    const bool fine = kv_span(p.position, p.rows, b, p.seq, p.c.capacity, first, count);
    return blocks_of(fine, first, count);
  };
  // Workgroups in the order of what they take: longer sequences first, their parts and heads side by side; every
  // other 256 of them backwards, since the two that are 256 apart share a CU.
  const uint32_t heads = p.c.kv_heads, turned = blockIdx.x & 256 && (blockIdx.x | 255) < gridDim.x ? blockIdx.x ^ 255 : blockIdx.x;
  const uint32_t h = turned % heads, ticket = turned / heads;
  // This workgroup's sequence b and part, and `ahead`, the blocks of the sequences before it.
  uint32_t b = 0, part = ticket, most, ahead = 0;   // most: blocks of a part
  auto part_of = [&](uint32_t all) { return max((all * heads + kKvSplit - 1) / kKvSplit, (uint32_t)kKvLeast); };
  int first = 0, count = 0;
  bool fine = true;
  if (p.batch == 1) {
    fine = kv_span(p.position, p.rows, 0, p.seq, p.c.capacity, first, count);
    most = part_of(blocks_of(fine, first, count));
  } else if (p.batch <= 64) {             // a lane per sequence, in every wave by itself
    if (lane < p.batch) fine = kv_span(p.position, p.rows, lane, p.seq, p.c.capacity, first, count);
    const uint32_t n = lane < p.batch ? blocks_of(fine, first, count) : 0, upto = kv_scan(n);
    const uint32_t all = __builtin_amdgcn_readlane(upto, 63);
    most = part_of(all);
    const uint32_t parts = (n + most - 1) / most;
    // Nine classes of length, in quarters of the mean; within one the batch's order.  Three classes' sums share a
    // register, ten bits each: the parts of up to 64 sequences are at most 64 + kKvSplit together.
    static_assert(64 + kKvSplit < 1024, "kv_attend: sums of parts in ten bits");
    const uint32_t mine = 8 - min(8u, (uint32_t)((float)n * (4.0f * p.batch) * __builtin_amdgcn_rcpf((float)max(all, 1u))));
    const uint32_t three = mine / 3, at = (mine - 3 * three) * 10;
    uint32_t before = 0, base = 0;
#pragma unroll
    for (uint32_t c = 0; c < 3; ++c) {
      const uint32_t its = three == c ? parts << at : 0, sum = kv_scan(its), ends = __builtin_amdgcn_readlane(sum, 63);
      const uint32_t e0 = ends & 1023, e1 = ends >> 10 & 1023, e2 = ends >> 20;
      if (three == c) before = base + (at == 0 ? 0 : at == 10 ? e0 : e0 + e1) + (sum >> at & 1023) - parts;
      base += e0 + e1 + e2;
    }
    const uint64_t it = __ballot(ticket >= before && ticket - before < parts);
    if (it == 0) return;
    b = __builtin_ctzll(it);
    part = ticket - __builtin_amdgcn_readlane(before, b);
    ahead = __builtin_amdgcn_readlane(upto - n, b);
    first = __builtin_amdgcn_readlane(first, b);
    count = __builtin_amdgcn_readlane(count, b);
    fine = __builtin_amdgcn_readlane((int)fine, b);
  } else {
    // Larger batches in their own order: a sum over all sequences, then NT sequences at a time.
    uint32_t sum = 0;
    for (int i = tid; i < p.batch; i += NT) sum += blocks_at(i);
    sum = kv_scan(sum);
    if (lane == 63) sum_of[0][wave] = sum;
    if (tid == 0) found[0] = ~0u;
    __syncthreads();
    uint32_t all = 0;
    for (int w = 0; w < W; ++w) all += sum_of[0][w];
    most = part_of(all);
    uint32_t parts_before = 0, blocks_before = 0;   // of the chunks before this one
    for (int c = 0; c < p.batch; c += NT) {
      const uint32_t n = c + tid < p.batch ? blocks_at(c + tid) : 0, parts = (n + most - 1) / most;
      const uint32_t upto = kv_scan(n), parts_upto = kv_scan(parts);
      __syncthreads();
      if (lane == 63) {
        sum_of[0][wave] = upto;
        sum_of[1][wave] = parts_upto;
      }
      __syncthreads();
      uint32_t before = parts_before + parts_upto - parts, longer = blocks_before + upto - n;
      for (int w = 0; w < W; ++w) {
        if (w < wave) {
          longer += sum_of[0][w];
          before += sum_of[1][w];
        }
        blocks_before += sum_of[0][w];
        parts_before += sum_of[1][w];
      }
      if (ticket >= before && ticket - before < parts) {
        found[0] = c + tid;
        found[1] = ticket - before;
        found[2] = longer;
      }
      if (ticket < parts_before) break;
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(found[0]);
    if (b == ~0u) return;
    part = __builtin_amdgcn_readfirstlane(found[1]);
    ahead = __builtin_amdgcn_readfirstlane(found[2]);
    fine = kv_span(p.position, p.rows, b, p.seq, p.c.capacity, first, count);
  }
  b = __builtin_amdgcn_readfirstlane(b);  // (one value all, which is not seen through the ways they come by)
  part = __builtin_amdgcn_readfirstlane(part);
  most = __builtin_amdgcn_readfirstlane(most);
  ahead = __builtin_amdgcn_readfirstlane(ahead);
  first = __builtin_amdgcn_readfirstlane(first);
  count = __builtin_amdgcn_readfirstlane(count);
  fine = __builtin_amdgcn_readfirstlane((int)fine);
  const uint32_t n = blocks_of(fine, first, count), parts = (n + most - 1) / most;
  if (part >= parts) return;
  const int rows = (fine ? count : p.seq) * p.group;
  auto out_row = [&](int r) { return p.out.at(b, r / p.group, h * p.group + r % p.group); };
  if (!fine) {
    for (int i = tid; i < rows * DQ; i += NT) *reinterpret_cast<u2v *>(out_row(i / DQ) + i % DQ * 4) = u2v{0x7E007E00u, 0x7E007E00u};
    return;
  }
  const uint32_t size = (n + parts - 1) / parts, from = part * size, to = min(n, from + size);
  const int closed = (first + count) / kKvBlock;
  const size_t bh = (size_t)b * heads + h;
  const uint8_t *const kc = p.c.kc + bh * p.c.capacity * D + j * D + g * 16;
  const uint8_t *const vc = p.c.vc + bh * p.c.capacity * D + j * kKvBlock + g * 16;
  const float *const ks = p.c.ks + bh * p.c.blocks, *const vs = p.c.vs + bh * p.c.blocks;
  const bool appends = p.k.data && to == n;
  int last = min((int)to - (appends ? 1 : 0), closed);   // blocks before this one are there, as codes

  u4 kn[4][H], vn[DT];                  // codes of the wave's next block, requested as soon as the last ones are used
  float ksn = 0.0f, vsn = 0.0f;
  auto fetch_keys = [&](int block) {
    if (block >= last) return;
    const size_t at = (size_t)block * (kKvBlock * D);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int u = 0; u < H; ++u) kn[s][u] = *reinterpret_cast<const u4 *>(kc + at + s * 16 * D + u * 64);
    ksn = ks[block];
  };
  auto fetch_values = [&](int block) {
    if (block >= last) return;
    const size_t at = (size_t)block * (kKvBlock * D);
#pragma unroll
    for (int d = 0; d < DT; ++d) vn[d] = *reinterpret_cast<const u4 *>(vc + at + d * 16 * kKvBlock);
    vsn = vs[block];
  };
  int block = (int)from + wave;
  fetch_keys(block);
  fetch_values(block);

  // Q as a B operand: lane (j, g) holds 16 dims of query j of each 64, in the order of the keys' codes.
  h8 q[QT][H][2];
  int pos[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int row = min(16 * t + j, rows - 1), i = row / p.group;   // rows past the last repeat it and are not stored
    pos[t] = first + i;
    const f16 *const at = p.q.at(b, i, h * p.group + row % p.group);
#pragma unroll
    for (int u = 0; u < H; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int dim = 64 * u + 16 * g + 8 * c;
        h8 v = *reinterpret_cast<const h8 *>(at + dim);
        if (p.cos) v = kv_rotate<D>(v, *reinterpret_cast<const h8 *>(at + (dim ^ D / 2)), p.cos, p.sin, pos[t], dim);
        q[t][u][c] = kv_order8<FMT>(v);
      }
  }
  if (appends) {
    if (tid < KvQuad<D>::CH) {          // the row to its half of the tails
      const int dim = 8 * tid, slot = first % kKvBlock;
      const f16 *const at = p.k.at(b, 0, h);
      h8 k = *reinterpret_cast<const h8 *>(at + dim);
      const h8 v = *reinterpret_cast<const h8 *>(p.v.at(b, 0, h) + dim);
      if (p.cos) k = kv_rotate<D>(k, *reinterpret_cast<const h8 *>(at + (dim ^ D / 2)), p.cos, p.sin, first, dim);
      kv_poison<D>(k, v);
      const size_t half = (2 * bh + (first / kKvBlock & 1)) * (kKvBlock * D);
      *reinterpret_cast<h8 *>(p.c.kt + half + slot * D + dim) = k;
#pragma unroll
      for (int e = 0; e < 8; ++e) p.c.vt[half + (dim + e) * kKvBlock + kv_place(slot)] = v[e];
    }
  }

  f4 acc[QT][DT];
  float top[QT], total[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    top[t] = kKvLowest;
    total[t] = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[t][d] = zero;
  }
  auto step = [&](auto kind, int block) {
    constexpr bool OPEN = decltype(kind)::value;
    const int base = block * kKvBlock;
    f4 s[QT][4];
    h8 vo[OPEN ? DT : 1][2];
    const size_t half = (2 * bh + (block & 1)) * (kKvBlock * D);
    const f16 *const kd = p.c.kt + half + j * D + g * 16, *const vd = p.c.vt + half + j * kKvBlock + g * 16;
    float kscale = p.scale, vscale = 1.0f;
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t][i] = zero;
    if constexpr (OPEN) {
      // Slots past the last are masked below; what lies there as a value is made finite, as are the values of rows
      // that are not (their keys are NaN, so rows that see them are NaN and the others multiply them by zero).
      if constexpr (D == 64) {            // (of 128 dims they do not fit beside the keys)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int c = 0; c < 2; ++c) vo[d][c] = *reinterpret_cast<const h8 *>(vd + d * 16 * kKvBlock + 8 * c);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h8 ko[H][2];
#pragma unroll
        for (int u = 0; u < H; ++u)
#pragma unroll
          for (int c = 0; c < 2; ++c) ko[u][c] = *reinterpret_cast<const h8 *>(kd + i * 16 * D + u * 64 + 8 * c);
#pragma unroll
        for (int u = 0; u < H; ++u)
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int t = 0; t < QT; ++t)
              s[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv_order8<FMT>(ko[u][c]), q[t][u][c], s[t][i], 0, 0, 0);
        if constexpr (TIGHT) __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (D != 64 && !TIGHT) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int c = 0; c < 2; ++c) vo[d][c] = *reinterpret_cast<const h8 *>(vd + d * 16 * kKvBlock + 8 * c);
      }
    } else {
      kscale *= ksn;
      vscale = vsn;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int u = 0; u < H; ++u)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const h8 kf = kv_decode8<FMT>(kn[i][u][2 * c], kn[i][u][2 * c + 1]);
#pragma unroll
            for (int t = 0; t < QT; ++t) s[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[t][u][c], s[t][i], 0, 0, 0);
          }
      fetch_keys(block + W);
    }
    h8 pf[QT][2];
    float vt[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float most = kKvLowest;
      vt[t] = vscale;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][i][e] *= kscale;
      if (base + kKvBlock - 1 > first) {    // some row does not see the whole block
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (base + 16 * i + 4 * g + e > pos[t]) s[t][i][e] = -INFINITY;
        if (base > pos[t]) vt[t] = 0.0f;    // (a scale may be NaN)
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = fmaxf(most, s[t][i][e]);
      if (__any(most - top[t] > kKvSlack)) {   // (a sum with the slack could round to a step of the maximum more)
        const float raised = fmaxf(top[t], kv_max_across(most));
        const float shrink = __builtin_amdgcn_exp2f(top[t] - raised);
        top[t] = raised;
        total[t] *= shrink;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[t][d] *= shrink;
      }
      float bias = kKvLift - top[t];
      if (__any(fabsf(top[t]) > kKvFar)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][i][e] -= top[t];
        bias = kKvLift;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        h8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (f16)__builtin_amdgcn_exp2f(s[t][2 * c + e / 4][e % 4] + bias);
        const h2 one = {(f16)1.0f, (f16)1.0f};
#pragma unroll
        for (int e = 0; e < 8; e += 2) total[t] = __builtin_amdgcn_fdot2(h2{x[e], x[e + 1]}, one, total[t], false);
        pf[t][c] = kv_order8<FMT>(x);
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      h8 vf[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if constexpr (OPEN) {
          const f16 most = (f16)65504.0f;
          const h8 hi = {most, most, most, most, most, most, most, most};
          const h8 x = TIGHT ? *reinterpret_cast<const h8 *>(vd + d * 16 * kKvBlock + 8 * c) : vo[d][c];
          vf[c] = kv_order8<FMT>(__builtin_elementwise_min(__builtin_elementwise_max(x, -hi), hi));
        } else {
          vf[c] = kv_decode8<FMT>(vn[d][2 * c], vn[d][2 * c + 1]);
        }
      }
      if constexpr (OPEN && TIGHT) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        f4 o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[0], pf[t][0], zero, 0, 0, 0);
        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[1], pf[t][1], o, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][d][e] = __builtin_fmaf(o[e], vt[t], acc[t][d][e]);
      }
    }
    if constexpr (!OPEN) fetch_values(block + W);
  };
  for (bool waits = appends;; waits = false) {
    for (; block < last; block += W) step(std::false_type{}, block);
    if (!waits) break;
    __syncthreads();                    // the row is in the cache
    if (closed * kKvBlock == first + 1) {   // it fills the block
      kv_close_tails<FMT, D, W>(p.c, bh, closed - 1, tops, tid);
      __syncthreads();
    }
    last = min((int)to, closed);
    fetch_keys(block);
    fetch_values(block);
  }
  if (block < (int)to) step(std::true_type{}, block);   // the open block

  // The waves' parts: lane (j, g) has dims 16 d + 4 g .. of query j.
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = 16 * t + j;
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f4 *>(&mem.sums[wave][r][16 * d + 4 * g]) = acc[t][d];
    total[t] += __shfl_xor(total[t], 16);
    total[t] += __shfl_xor(total[t], 32);
    if (g == 0) {
      mem.tops[wave][r] = top[t];
      mem.totals[wave][r] = total[t];
    }
  }
  __syncthreads();
  auto store = [&](int r, int d, f4 o, float total) {
    const float inv = 1.0f / total;
    *reinterpret_cast<h4 *>(out_row(r) + d) = h4{(f16)(o[0] * inv), (f16)(o[1] * inv), (f16)(o[2] * inv), (f16)(o[3] * inv)};
  };
  // Where this part's sums go.  Units that are split have more than `most` blocks each, so that ahead / most is another
  // for each, and as many places as parts lie between two of them at twice that.
  const uint32_t unit = (ahead * heads + h * n) / most;
  const __amdgpu_buffer_rsrc_t po = buffer_rsrc(p.partial, (size_t)kKvPlaces * R * D * 4);
  const __amdgpu_buffer_rsrc_t pm = buffer_rsrc(p.partial + kKvPlaces * R * D, (size_t)kKvPlaces * R * 2 * 4);
  const int slot = 2 * unit + part;
  for (int i = tid; i < rows * DQ; i += NT) {
    const int r = i / DQ, d = i % DQ * 4;
    float top = mem.tops[0][r], sum = 0.0f;
#pragma unroll
    for (int w = 1; w < W; ++w) top = fmaxf(top, mem.tops[w][r]);
    f4 o = zero;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(mem.tops[w][r] - top);
      sum += f * mem.totals[w][r];
      o += f * *reinterpret_cast<const f4 *>(&mem.sums[w][r][d]);
    }
    if (parts == 1) {
      store(r, d, o, sum);
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, o), po, ((slot * R + r) * D + d) * 4, 0, kSysCoherent);
      if (d == 0) {
        const float ml[2] = {top, sum};
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2v, ml), pm, (slot * R + r) * 8, 0, kSysCoherent);
      }
    }
  }
  if (parts > 1 && kv_last_part(p.tickets + unit, parts, &found[6]))
    kv_join<R, D, NT>(po, pm, rows, parts, [&](uint32_t k) { return 2 * unit + k; }, reinterpret_cast<f4 *>(&mem.sums), store);
}

// Attention of more query rows: a KV head's rows (row i of the call and query head g of the group: row i group + g) in
// tiles of 128, a workgroup per tile, 32 rows a wave.  The workgroup goes through the slots that its rows see, 64 at a
// time: a block's codes are fetched one iteration ahead into registers, decoded once into one of two LDS buffers as fp16
// (in the order in which the lanes read it, 16-byte pieces swizzled against bank conflicts) while the other buffer is
// multiplied, and serve all 128 rows.  Long slot ranges of few tiles are taken in parts by several workgroups
// (kv_last_part, kv_join).
//
// As in kv_attend_kernel scores are K.Q^T and outputs V^T.P^T, here on v_mfma_f32_32x32x16_f16, so that a lane holds one
// query (column lane % 32) and its probabilities are the B operand as they are.  The block's value scale would cost an
// operation per output and block as a factor of the fp32 sums; instead the sums are kept in units of `unit`, a recent
// block's scale, and the ratio vs / unit enters the exponent of the probabilities, whose total is divided by it once per
// block.  A block whose ratio is past 4 either way sets the unit anew.
//
// What bounds it: of the cycles of a CU the matrix cores are busy 46% and the vector units 53% (per 64 slots and wave
// D / 4 products of 32 cycles and, a lane, 32 exponentials at a quarter of the rate and some 150 other operations), which
// two waves a SIMD overlap little.  8192 rows of 32 query and 8 KV heads of 128, fp8:
// 581 to 611 us by card, 946 to 900 TFLOP/s; 509 rows over 32768 slots 317 to 334 us; 8 x 500 rows, 9 and 3 heads of 64:
// 13.6 us, 4096 rows of them 51 us, 377 TFLOP/s (half the products a block, as many other operations).  Measured on
// the way: bank conflicts on a fifth of the cycles before the pieces' layout (620 us), scales asked for where they are
// used (598 against 588).  Not kept: the next block's scores beside this one's exponentials (721 against 620, for want of
// registers), 256 rows a workgroup (606 against 615, but 64 rows 45 us against 36).
template <int FMT, int D>
__global__ __launch_bounds__(256, 2) void kv_prompt_kernel(KvAttendParams p) {
  constexpr int R = 128, KS = D / 16, DT = D / 32, RAW = D / 64, DQ = D / 4;
  constexpr int KBYTES = kKvBlock * D * 2, BYTES = 2 * KBYTES;    // a buffer: keys, values
  __shared__ __align__(16) uint8_t mem[2 * BYTES];
  __shared__ uint32_t word;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Sequences and KV heads side by side, so that an XCD (blockIdx % 8) sees few of them and their codes stay in its L2;
  // the tiles that see most first.
  const int pairs = p.batch * p.c.kv_heads, split = blockIdx.x / pairs % p.splits, tile = p.tiles - 1 - blockIdx.x / pairs / p.splits;
  const int b = blockIdx.x % pairs / p.c.kv_heads, h = blockIdx.x % pairs % p.c.kv_heads;
  int first, count;
  const bool fine = kv_span(p.position, p.rows, b, p.seq, p.c.capacity, first, count);
  const int rows = min(R, (fine ? count : p.seq) * p.group - tile * R);
  if (rows <= 0) return;
  auto out_row = [&](int r) {
    const int row = tile * R + r;
    return p.out.at(b, row / p.group, h * p.group + row % p.group);
  };
  if (!fine) {
    if (split == 0)
      for (int i = tid; i < rows * DQ; i += 256) *reinterpret_cast<u2v *>(out_row(i / DQ) + i % DQ * 4) = u2v{0x7E007E00u, 0x7E007E00u};
    return;
  }
  const int closed = (first + count) / kKvBlock;
  const int blocks = (first + (tile * R + rows - 1) / p.group) / kKvBlock + 1;   // blocks that the last row sees some of
  const int chunk = max(kKvChunk, (blocks + p.splits - 1) / p.splits), parts = (blocks + chunk - 1) / chunk;
  if (split >= parts) return;
  const int begin = split * chunk, stop = min(blocks, begin + chunk);
  const size_t bh = (size_t)b * p.c.kv_heads + h;
  const uint8_t *const kc = p.c.kc + bh * p.c.capacity * D, *const vc = p.c.vc + bh * p.c.capacity * D;
  const float *const ks = p.c.ks + bh * p.c.blocks, *const vs = p.c.vs + bh * p.c.blocks;

  // A block of codes on its way, in 16-byte pieces.
  u4 raw[2 * RAW];
  auto fetch = [&](int block) {
    if (block >= stop || block >= closed) return;
    const size_t at = (size_t)block * (kKvBlock * D);
#pragma unroll
    for (int u = 0; u < RAW; ++u) {
      raw[u] = *reinterpret_cast<const u4 *>(kc + at + 16 * (tid + 256 * u));
      raw[RAW + u] = *reinterpret_cast<const u4 *>(vc + at + 16 * (tid + 256 * u));
    }
  };
  // Keys: rows of D, 8 dims a piece; row m of the 32 that a product takes is slot 16 (m / 8) + m % 8, and 8 more in the
  // second product: the 8 probabilities that a lane then has for K step s are those of 8 consecutive codes of a value row.
  // Values: rows of 64 slots by dim, piece 2 s + g for lane half g.  LDS moves 16 lanes' pieces a cycle where they lie in
  // 16 different columns of its 256 bytes: pieces are swizzled so that consecutive lanes' are, written and read.
  auto key_at = [&](int slot, int piece) {
    const int turn = D == 64 ? ((slot >> 1 & 3) | (slot >> 2 & 4)) ^ (slot & 1) : piece >> 3 ^ (slot & 7) ^ (slot >> 1 & 8);
    return slot * (2 * D) + (piece ^ turn) * 16;
  };
  auto value_at = [&](int dim, int piece) {
    const int turn = ((dim & 2) | (dim >> 2 & 1) | (dim >> 1 & 4)) ^ (dim & 1) << 1;
    return KBYTES + dim * (2 * kKvBlock) + (piece ^ turn) * 16;
  };
  auto stage = [&](int block) {
    if (block >= stop) return;
    uint8_t *const to = mem + (block & 1) * BYTES;
    if (block < closed) {
#pragma unroll
      for (int u = 0; u < RAW; ++u) {
        const int at = tid + 256 * u, slot = at / (D / 16), piece = at % (D / 16) * 2;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<h8 *>(to + key_at(slot, piece + e)) = kv_decode8<FMT>(raw[u][2 * e], raw[u][2 * e + 1]);
        const int dim = at / 4, f = at % 4;    // places 16 f ..: slots 16 i + 4 f ..
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<h8 *>(to + value_at(dim, 4 * (f >> 1) + 2 * e + (f & 1))) = kv_decode8<FMT>(raw[RAW + u][2 * e], raw[RAW + u][2 * e + 1]);
      }
    } else {                              // fp16 rows (values as in kv_attend_kernel: finite, whatever lies there)
      const size_t half = (2 * bh + (block & 1)) * (kKvBlock * D);
      const f16 most = (f16)65504.0f;
      const h8 hi = {most, most, most, most, most, most, most, most};
#pragma unroll
      for (int u = 0; u < 2 * RAW; ++u) {
        const int at = tid + 256 * u;
        *reinterpret_cast<h8 *>(to + key_at(at / (D / 8), at % (D / 8))) = kv_order8<FMT>(*reinterpret_cast<const h8 *>(p.c.kt + half + 8 * at));
        const int dim = at / 8, f = at / 2 % 4, e = at % 2;
        const h8 x = *reinterpret_cast<const h8 *>(p.c.vt + half + 8 * at);
        *reinterpret_cast<h8 *>(to + value_at(dim, 4 * (f >> 1) + 2 * e + (f & 1))) =
            kv_order8<FMT>(__builtin_elementwise_min(__builtin_elementwise_max(x, -hi), hi));
      }
    }
  };
  fetch(begin);

  const int mine = wave * 32;             // the wave's rows of the tile
  const int low = first + (tile * R + mine) / p.group;                       // positions of its first and last row
  const int high = first + (tile * R + min(rows, mine + 32) - 1) / p.group;
  const int row = tile * R + min(mine + j, rows - 1), pos = first + row / p.group;   // rows past the last repeat it
  h8 q[KS];
  {
    const f16 *const at = p.q.at(b, row / p.group, h * p.group + row % p.group);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int dim = 16 * s + 8 * g;
      h8 v = *reinterpret_cast<const h8 *>(at + dim);
      if (p.cos) v = kv_rotate<D>(v, *reinterpret_cast<const h8 *>(at + (dim ^ D / 2)), p.cos, p.sin, pos, dim);
      q[s] = kv_order8<FMT>(v);
    }
  }
  f16x acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[d][e] = 0.0f;
  float top = kKvLowest, total = 0.0f, unit = 0.0f;

  // A block's scales are requested ahead of the codes of the block behind it: loads come back in order, so that they
  // are there once those codes are (asked for when they are used, they wait for every code on its way).
  float ksn = 1.0f, vsn = 1.0f;
  auto fetch_scales = [&](int block) {
    const int at = min(block, p.c.blocks - 1);
    ksn = ks[at];
    vsn = vs[at];
  };
  stage(begin);
  fetch_scales(begin);
  fetch(begin + 1);
  __syncthreads();
  for (int block = begin; block < stop; ++block) {
    stage(block + 1);
    const float ksb = kv_uniform(ksn), vsb = kv_uniform(vsn);
    fetch_scales(block + 1);
    fetch(block + 2);
    const int base = block * kKvBlock;
    if (base <= high && mine < rows) {
      const uint8_t *const from = mem + (block & 1) * BYTES;
      const bool open = block >= closed;
      const float kscale = open ? p.scale : p.scale * ksb, vscale = open ? 1.0f : vsb;
      // Eight operands of each product are read ahead: a read is 100 cycles and more from its use, a product 32.
      f16x s[2];
#pragma unroll
      for (int e = 0; e < 16; ++e) s[0][e] = s[1][e] = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int a = 0; a < 2; ++a)
          s[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const h8 *>(from + key_at(16 * (j >> 3) + 8 * a + (j & 7), 2 * k + g)), q[k], s[a], 0, 0, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, KS, 0);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, KS, 0);
      // Where the values' operands lie, settled before the block of the second product (in it the compiler puts these
      // operations, and with them the reads, behind the exponentials).
      uint32_t value_from[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        value_from[k] = (block & 1) * BYTES + value_at(j, 2 * k + g);
        asm volatile("" : "+v"(value_from[k]));
      }
      float shift = 0.0f, part = 1.0f;    // log2 of vs / unit, which the probabilities carry, and unit / vs
      if (vscale > 0.0f) {                // (a block of zeros adds nothing in any unit)
        const float ratio = unit > 0.0f ? vscale * __builtin_amdgcn_rcpf(unit) : 0.0f;
        if (ratio > 4.0f || ratio < 0.25f) {
          if (unit > 0.0f) {
            const float turn = unit / vscale;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= turn;
          }
          unit = vscale;
        } else {
          shift = __builtin_amdgcn_logf(ratio);
          part = unit * __builtin_amdgcn_rcpf(vscale);   // (to 2^-23, as the logarithm)
        }
      } else if (!(vscale == 0.0f) && base <= pos) {
        shift = part = vscale;            // NaN, for the rows that see some of the block
      }
      float most = -INFINITY, factor = kscale;
      if (base + kKvBlock - 1 <= low) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int e = 0; e < 16; ++e) most = fmaxf(most, s[a][e]);
        most *= kscale;
      } else {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int slot = base + 16 * (e / 4) + 8 * a + 4 * g + e % 4;
            s[a][e] = slot <= pos ? s[a][e] * kscale : -INFINITY;
            most = fmaxf(most, s[a][e]);
          }
        factor = 1.0f;
      }
      if (__any(most - top > kKvSlack)) {
        const float raised = fmaxf(top, fmaxf(most, __shfl_xor(most, 32)));
        const float shrink = __builtin_amdgcn_exp2f(top - raised);
        top = raised;
        total *= shrink;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= shrink;
      }
      float bias = kKvLift - 1.0f + shift - top;   // (at most 2^15 with the ratio's 2^2)
      if (__any(fabsf(top) > kKvFar)) {
#pragma clang fp contract(off)            // (products rounded as the maximum was)
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[a][e] = s[a][e] * factor - top;
        factor = 1.0f;
        bias = kKvLift - 1.0f + shift;
      }
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        h8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (f16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[k / 2][8 * (k % 2) + e], factor, bias));
        const h2 one = {(f16)1.0f, (f16)1.0f};
#pragma unroll
        for (int e = 0; e < 8; e += 2) sum = __builtin_amdgcn_fdot2(h2{x[e], x[e + 1]}, one, sum, false);
        const h8 pf = kv_order8<FMT>(x);
#pragma unroll
        for (int d = 0; d < DT; ++d)
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const h8 *>(mem + value_from[k] + d * (64 * kKvBlock)), pf, acc[d], 0, 0, 0);
      }
      total = __builtin_fmaf(sum, part, total);
      // The next step's exponentials stand between a step's products.
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * DT, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 24, 0);
#pragma unroll
      for (int i = 0; i < 4 * DT; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i < 3 * DT) __builtin_amdgcn_sched_group_barrier(0x002, 24 / DT, 0);
        if (i < 2 * DT) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
    }
    __syncthreads();
  }
  total += __shfl_xor(total, 32);
  auto store = [&](int r, int d, f4 o, float total) {
    const float inv = 1.0f / total;
    *reinterpret_cast<h4 *>(out_row(r) + d) = h4{(f16)(o[0] * inv), (f16)(o[1] * inv), (f16)(o[2] * inv), (f16)(o[3] * inv)};
  };
  const uint32_t place = ((uint32_t)(bh * p.tiles + tile)) * p.splits;
  const size_t all = (size_t)pairs * p.tiles * p.splits;
  const __amdgpu_buffer_rsrc_t po = buffer_rsrc(p.partial, all * R * D * 4), pm = buffer_rsrc(p.partial + all * R * D, all * R * 2 * 4);
  if (mine + j < rows) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = mine + j, dim = 32 * d + 8 * e + 4 * g;
        const f4 o = {acc[d][4 * e] * unit, acc[d][4 * e + 1] * unit, acc[d][4 * e + 2] * unit, acc[d][4 * e + 3] * unit};
        if (parts == 1) store(r, dim, o, total);
        else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, o), po, (int)(((place + split) * R + r) * D + dim) * 4, 0, kSysCoherent);
      }
    if (parts > 1 && g == 0) {
      const float ml[2] = {top, total};
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2v, ml), pm, (int)((place + split) * R + mine + j) * 8, 0, kSysCoherent);
    }
  }
  if (parts > 1 && kv_last_part(p.tickets + bh * p.tiles + tile, parts, &word))
    kv_join<R, D, 256>(po, pm, rows, parts, [&](uint32_t k) { return place + k; }, reinterpret_cast<f4 *>(mem), store);
}

}  // namespace lb
