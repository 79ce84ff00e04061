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
struct KvAppendParams {
  KvCache c;
  KvRows k, v;
  const int64_t *position, *rows;
  const f16 *cos, *sin;
  int seq;
};

// One workgroup of 2 D threads per block of 64 slots that new rows fall into, KV head and sequence; a thread owns 8
// dims of 4 consecutive slots.  A block that becomes full takes its older rows from the tail, its top over the
// workgroup, and is encoded from registers; value codes are turned into rows by dim through LDS (a thread's 4 slots are
// one dword there).  Rows of the last block and of the one before it go to the tails as well.  Bound by memory for
// prompts, by its launch for single tokens.
template <int FMT, int D>
__global__ __launch_bounds__(2 * D) void kv_append_kernel(KvAppendParams p) {
  constexpr int CH = D / 8, PITCH = 20;   // chunks of 8 dims; dwords of a value row in LDS (16 and padding)
  __shared__ uint32_t tops[2][2 * D / 64];
  __shared__ __align__(16) uint32_t turn[D * PITCH];
  const int tid = threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int chunk = tid % CH, dim = 8 * chunk, quad = tid / CH;
  int first, count;
  if (!kv_span(p.position, p.rows, b, p.seq, p.c.capacity, first, count)) return;
  const int end = first + count, oldest = first / kKvBlock, block = oldest + blockIdx.x, base = block * kKvBlock;
  if (count == 0 || base >= end) return;
  const bool full = base + kKvBlock <= end;
  const int kept = end / kKvBlock - 1;    // rows from this block on go to the tails
  // The block that was open reads its older rows from its half of the tails.  Blocks of the same half that are written
  // there by the same call wait for that: its own workgroup writes their rows, at the end.
  const bool reads = first % kKvBlock != 0, after = reads && block >= oldest + 2;
  const size_t bh = (size_t)b * p.c.kv_heads + h;
  f16 *const kt = p.c.kt + bh * (2 * kKvBlock * D), *const vt = p.c.vt + bh * (2 * kKvBlock * D);

  h8 k[4], v[4];
  auto load = [&](int base) {             // the new rows of a block; false in `have` where there is none
    uint32_t have = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int slot = base + 4 * quad + i, row = slot - first;
      k[i] = v[i] = h8{0, 0, 0, 0, 0, 0, 0, 0};
      if (row < 0 || slot >= end) continue;
      have |= 1u << i;
      const f16 *at = p.k.at(b, row, h);
      k[i] = *reinterpret_cast<const h8 *>(at + dim);
      v[i] = *reinterpret_cast<const h8 *>(p.v.at(b, row, h) + dim);
      if (p.cos) k[i] = kv_rotate<D>(k[i], *reinterpret_cast<const h8 *>(at + (dim ^ D / 2)), p.cos, p.sin, slot, dim);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {         // a row that is not finite gets a key of NaNs
      uint32_t bad = kv_top(k[i]) >= 0x7C00u || kv_top(v[i]) >= 0x7C00u;
#pragma unroll
      for (int d = CH / 2; d > 0; d >>= 1) bad |= __shfl_xor(bad, d);
      if (bad)
#pragma unroll
        for (int e = 0; e < 8; ++e) k[i][e] = __builtin_bit_cast(f16, (uint16_t)0x7E00u);
    }
    return have;
  };
  auto keep = [&](int block, uint32_t have) {   // the new rows of a block to its half of the tails
    f16 *const kd = kt + (block & 1) * (kKvBlock * D) + 4 * quad * D + dim;
    f16 *const vd = vt + (block & 1) * (kKvBlock * D) + dim * kKvBlock + kv_place(4 * quad);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (have >> i & 1) *reinterpret_cast<h8 *>(kd + i * D) = k[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (have == 15u) {
        *reinterpret_cast<h4 *>(vd + e * kKvBlock) = h4{v[0][e], v[1][e], v[2][e], v[3][e]};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (have >> i & 1) vd[e * kKvBlock + i] = v[i][e];
      }
    }
  };

  const uint32_t have = load(base);
  if (full) {
    if (block == oldest && reads) {
      const f16 *const kd = kt + (block & 1) * (kKvBlock * D) + 4 * quad * D + dim;
      const f16 *const vd = vt + (block & 1) * (kKvBlock * D) + dim * kKvBlock + kv_place(4 * quad);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (have >> i & 1) continue;
        k[i] = *reinterpret_cast<const h8 *>(kd + i * D);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = vd[e * kKvBlock + i];
      }
    }
    uint32_t top[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      top[0] = max(top[0], kv_top(k[i]));
      top[1] = max(top[1], kv_top(v[i]));
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) top[s] = max(top[s], (uint32_t)__shfl_xor((int)top[s], d));
      if ((tid & 63) == 0) tops[s][tid >> 6] = top[s];
    }
    __syncthreads();
    float scale[2], r[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int w = 0; w < 2 * D / 64; ++w) top[s] = max(top[s], tops[s][w]);
      const float a = (float)__builtin_bit_cast(f16, (uint16_t)top[s]);
      const bool bad = top[s] >= 0x7C00u;
      scale[s] = bad ? __builtin_nanf("") : a / kv_limit<FMT>();
      r[s] = bad || top[s] == 0 ? 0.0f : kv_limit<FMT>() / a;
    }
    const bool kbad = top[0] >= 0x7C00u, vbad = top[1] >= 0x7C00u;
    if (tid == 0) {
      p.c.ks[bh * p.c.blocks + block] = scale[0];
      p.c.vs[bh * p.c.blocks + block] = scale[1];
    }
    uint8_t *const kc = p.c.kc + (bh * p.c.capacity + base) * D + 4 * quad * D + dim;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u2v w = {kbad ? 0u : kv_encode4<FMT>(k[i][0], k[i][1], k[i][2], k[i][3], r[0]),
                     kbad ? 0u : kv_encode4<FMT>(k[i][4], k[i][5], k[i][6], k[i][7], r[0])};
      *reinterpret_cast<u2v *>(kc + i * D) = w;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      turn[(dim + e) * PITCH + kv_place(4 * quad) / 4] = vbad ? 0u : kv_encode4<FMT>(v[0][e], v[1][e], v[2][e], v[3][e], r[1]);
    __syncthreads();
    uint8_t *const vc = p.c.vc + (bh * p.c.capacity + base) * D;
#pragma unroll
    for (int i = 0; i < 2; ++i) {         // D rows of four 16-byte pieces
      const int piece = tid + i * 2 * D;
      *reinterpret_cast<u4 *>(vc + 16 * piece) = *reinterpret_cast<const u4 *>(&turn[piece / 4 * PITCH + piece % 4 * 4]);
    }
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
// 3 bytes moved per value, two are written.
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
  KvRows q, out;
  const int64_t *position, *rows;
  const f16 *cos, *sin;
  float *partial;         // splits > 1: [batch, kv_heads * tiles, splits][R][D] sums, then [..][R][2] maxima and totals
  int seq, heads, group;  // group: query heads of a KV head
  int tiles, splits, chunk;   // row tiles of a KV head; parts of its slots, of `chunk` blocks each
  float scale;            // score scale * log2(e)
};

constexpr float kKvLowest = -1e30f;   // a running maximum below every score (scores are under 1e14 in magnitude)

// The largest over the four lanes that hold a query.
__device__ __forceinline__ float kv_max_across(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}

// A KV head's query rows (row i of the call and query head g of the group: row i * group + g) in tiles of 16 QT.  A
// workgroup takes a tile and `chunk` blocks of slots, its four waves every fourth block each, with a running maximum and
// total of their own; they are joined in LDS, and the parts of a tile's slots by kv_join_kernel.
//
// Scores are K.Q^T and outputs V^T.P^T, so that a lane holds one query throughout (column lane % 16): its maximum,
// total and rescaling are the lane's own, and the probabilities that it computes are the B operand of the second product
// as they are, rounded to fp16 (relative 2^-11, as every output is; the total sums the rounded ones).  Codes enter both
// products exactly as fp16 and the block's scales multiply fp32 sums.  The maximum is raised only where a block exceeds
// it by more than 2^8: until then probabilities up to 2^8 are as exact, and nothing has to cross lanes.
template <int FMT, int D, int QT>
__global__ __launch_bounds__(256) void kv_attend_kernel(KvAttendParams p) {
  constexpr int R = 16 * QT, H = D / 64, DT = D / 16, PITCH = D + 4;
  __shared__ __align__(16) float sums[4][R][PITCH];
  __shared__ float tops[4][R], totals[4][R];
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.y, unit = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
  const int h = unit / p.tiles, tile = unit % p.tiles;
  int first, count;
  const bool fine = kv_span(p.position, p.rows, b, p.seq, p.c.capacity, first, count);
  const int rows = min(R, (fine ? count : p.seq) * p.group - tile * R);   // rows of this tile
  if (rows <= 0) return;
  auto out_row = [&](int r) {
    const int row = tile * R + r;
    return p.out.at(b, row / p.group, h * p.group + row % p.group);
  };
  if (!fine) {
    if (split == 0)
      for (int i = tid; i < rows * (D / 4); i += 256)
        *reinterpret_cast<u2v *>(out_row(i / (D / 4)) + i % (D / 4) * 4) = u2v{0x7E007E00u, 0x7E007E00u};
    return;
  }
  const int low = first + tile * R / p.group;                    // position of the tile's first row
  const int seen = first + (tile * R + rows - 1) / p.group + 1;  // slots that its last row sees
  const int blocks = (seen + kKvBlock - 1) / kKvBlock, closed = (first + count) / kKvBlock;
  const int parts = min(p.splits, (blocks + p.chunk - 1) / p.chunk);
  if (split >= parts) return;
  const int begin = split * p.chunk, stop = split == p.splits - 1 ? blocks : min(blocks, begin + p.chunk);
  const size_t bh = (size_t)b * p.c.kv_heads + h;
  const uint8_t *const kc = p.c.kc + bh * p.c.capacity * D + j * D + g * 16;
  const uint8_t *const vc = p.c.vc + bh * p.c.capacity * D + j * kKvBlock + g * 16;
  const float *const ks = p.c.ks + bh * p.c.blocks, *const vs = p.c.vs + bh * p.c.blocks;

  // Q as a B operand: lane (j, g) holds 16 dims of query j of each 64, in the order of the keys' codes.
  h8 q[QT][H][2];
  int pos[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = min(16 * t + j, rows - 1), row = tile * R + r;   // rows past the last repeat it and are not stored
    const int i = row / p.group;
    pos[t] = first + i;
    const f16 *const at = p.q.at(b, i, h * p.group + row % p.group);
#pragma unroll
    for (int u = 0; u < H; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int dim = 64 * u + 16 * g + 8 * c;
        h8 x = *reinterpret_cast<const h8 *>(at + dim);
        if (p.cos) x = kv_rotate<D>(x, *reinterpret_cast<const h8 *>(at + (dim ^ D / 2)), p.cos, p.sin, pos[t], dim);
        q[t][u][c] = kv_order8<FMT>(x);
      }
  }

  const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  f4 acc[QT][DT];
  float top[QT], total[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    top[t] = kKvLowest;
    total[t] = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[t][d] = zero;
  }

  u4 kn[4][H], vn[DT];
  float ksn = 0.0f, vsn = 0.0f;
  auto fetch = [&](int block) {
    if (block >= stop || block >= closed) return;
    const size_t at = (size_t)block * (kKvBlock * D);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int u = 0; u < H; ++u) kn[s][u] = *reinterpret_cast<const u4 *>(kc + at + s * 16 * D + u * 64);
#pragma unroll
    for (int d = 0; d < DT; ++d) vn[d] = *reinterpret_cast<const u4 *>(vc + at + d * 16 * kKvBlock);
    ksn = ks[block];
    vsn = vs[block];
  };
  fetch(begin + wave);
  for (int block = begin + wave; block < stop; block += 4) {
    const bool open = block >= closed;
    const int base = block * kKvBlock;
    f4 s[QT][4];
    h8 vf[DT][2];
    float kscale = p.scale, vscale = 1.0f;
    if (!open) {
      kscale *= ksn;
      vscale = vsn;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int t = 0; t < QT; ++t) s[t][i] = zero;
#pragma unroll
        for (int u = 0; u < H; ++u)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const h8 kf = kv_decode8<FMT>(kn[i][u][2 * c], kn[i][u][2 * c + 1]);
#pragma unroll
            for (int t = 0; t < QT; ++t) s[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[t][u][c], s[t][i], 0, 0, 0);
          }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int c = 0; c < 2; ++c) vf[d][c] = kv_decode8<FMT>(vn[d][2 * c], vn[d][2 * c + 1]);
      fetch(block + 4);
    } else {
      // Slots past the last are masked below; what lies there as a value is made finite, as are the values of rows that
      // are not (their keys are NaN, so rows that see them are NaN and the others multiply them by zero).
      const f16 *const kd = p.c.kt + bh * (2 * kKvBlock * D) + (block & 1) * (kKvBlock * D) + j * D + g * 16;
      const f16 *const vd = p.c.vt + bh * (2 * kKvBlock * D) + (block & 1) * (kKvBlock * D) + j * kKvBlock + g * 16;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int t = 0; t < QT; ++t) s[t][i] = zero;
#pragma unroll
        for (int u = 0; u < H; ++u)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const h8 kf = kv_order8<FMT>(*reinterpret_cast<const h8 *>(kd + i * 16 * D + u * 64 + 8 * c));
#pragma unroll
            for (int t = 0; t < QT; ++t) s[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[t][u][c], s[t][i], 0, 0, 0);
          }
      }
      const f16 most = (f16)65504.0f;
      const h8 hi = {most, most, most, most, most, most, most, most};
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const h8 x = *reinterpret_cast<const h8 *>(vd + d * 16 * kKvBlock + 8 * c);
          vf[d][c] = kv_order8<FMT>(__builtin_elementwise_min(__builtin_elementwise_max(x, -hi), hi));
        }
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float most = kKvLowest, vt = vscale;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][i][e] *= kscale;
      if (base + kKvBlock - 1 > low) {    // some row does not see the whole block
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (base + 16 * i + 4 * g + e > pos[t]) s[t][i][e] = -INFINITY;
        if (base > pos[t]) vt = 0.0f;     // (a scale may be NaN)
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = fmaxf(most, s[t][i][e]);
      if (__any(most > top[t] + 8.0f)) {
        const float raised = fmaxf(top[t], kv_max_across(most));
        const float shrink = __builtin_amdgcn_exp2f(top[t] - raised);
        top[t] = raised;
        total[t] *= shrink;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[t][d] *= shrink;
      }
      h8 pf[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        h8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (f16)__builtin_amdgcn_exp2f(s[t][2 * c + e / 4][e % 4] - top[t]);
        const h2 one = {(f16)1.0f, (f16)1.0f};
#pragma unroll
        for (int e = 0; e < 8; e += 2) total[t] = __builtin_amdgcn_fdot2(h2{x[e], x[e + 1]}, one, total[t], false);
        pf[c] = kv_order8<FMT>(x);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        f4 o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[d][0], pf[0], zero, 0, 0, 0);
        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[d][1], pf[1], o, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][d][e] = __builtin_fmaf(o[e], vt, acc[t][d][e]);
      }
    }
  }

  // The waves' parts: lane (j, g) has dims 16 d + 4 g .. of query j.
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = 16 * t + j;
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f4 *>(&sums[wave][r][16 * d + 4 * g]) = acc[t][d];
    total[t] += __shfl_xor(total[t], 16);
    total[t] += __shfl_xor(total[t], 32);
    if (g == 0) {
      tops[wave][r] = top[t];
      totals[wave][r] = total[t];
    }
  }
  __syncthreads();
  const bool alone = parts == 1;
  const size_t part = ((size_t)b * p.c.kv_heads * p.tiles + unit) * p.splits + split;
  float *const po = p.partial + part * (R * D);
  float *const pm = p.partial + (size_t)gridDim.y * gridDim.x * (R * D) + part * (R * 2);
  for (int i = tid; i < R * (D / 4); i += 256) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    if (r >= rows) break;
    float most = tops[0][r], sum = 0.0f;
#pragma unroll
    for (int w = 1; w < 4; ++w) most = fmaxf(most, tops[w][r]);
    f4 o = zero;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(tops[w][r] - most);
      sum += f * totals[w][r];
      o += f * *reinterpret_cast<const f4 *>(&sums[w][r][d]);
    }
    if (alone) {
      const float inv = 1.0f / sum;
      *reinterpret_cast<h4 *>(out_row(r) + d) = h4{(f16)(o[0] * inv), (f16)(o[1] * inv), (f16)(o[2] * inv), (f16)(o[3] * inv)};
    } else {
      *reinterpret_cast<f4 *>(po + r * D + d) = o;
      if (d == 0) {
        pm[2 * r] = most;
        pm[2 * r + 1] = sum;
      }
    }
  }
}

// Joins the parts of a row's slots, a wave per row.
template <int D, int QT>
__global__ __launch_bounds__(256) void kv_join_kernel(KvAttendParams p, size_t sums) {
  constexpr int R = 16 * QT, PER = D / 64;
  const int lane = threadIdx.x & 63, b = blockIdx.y, item = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int unit = item / R, r = item % R, h = unit / p.tiles, tile = unit % p.tiles;
  int first, count;
  if (!kv_span(p.position, p.rows, b, p.seq, p.c.capacity, first, count)) return;
  const int rows = min(R, count * p.group - tile * R);
  if (r >= rows) return;
  const int seen = first + (tile * R + rows - 1) / p.group + 1, blocks = (seen + kKvBlock - 1) / kKvBlock;
  const int parts = min(p.splits, (blocks + p.chunk - 1) / p.chunk);
  if (parts == 1) return;
  const size_t part = ((size_t)b * p.c.kv_heads * p.tiles + unit) * p.splits;
  const float *const po = p.partial + part * (R * D) + r * D + lane * PER;
  const float *const pm = p.partial + sums + part * (R * 2) + 2 * r;
  float most = kKvLowest, total = 0.0f, o[PER] = {};
  for (int i = 0; i < parts; ++i) most = fmaxf(most, pm[(size_t)i * (R * 2)]);
  for (int i = 0; i < parts; ++i) {
    const float f = __builtin_amdgcn_exp2f(pm[(size_t)i * (R * 2)] - most);
    total += f * pm[(size_t)i * (R * 2) + 1];
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] += f * po[(size_t)i * (R * D) + e];
  }
  const int row = tile * R + r;
  f16 *const out = p.out.at(b, row / p.group, h * p.group + row % p.group) + lane * PER;
#pragma unroll
  for (int e = 0; e < PER; ++e) out[e] = (f16)(o[e] / total);
}

}  // namespace lb
