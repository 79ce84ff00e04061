// gfx950 kernels of the KV cache in pages (include/lowbit_decode_hip.h: lb_paged_append, lb_paged_attention).
//
// A page holds `page` slots (a power of two from 16 on) of every KV head: keys [page][D], values by chunks of 16 slots,
// [page / 16][D][16].  A chunk of keys and one of values thus lie at the same offset, and both are A operands of
// 16x16x32 products as they lie: a lane's 16 bytes are 8 dims of a key, and 8 bytes the 4 slots of a value dim whose
// probabilities the lane holds as the result of K.Q^T (with those of the next chunk, the 8 that a product takes).
#pragma once
#include "lb_kv.h"
#include "lb_serve.h"

namespace lb {

constexpr int kChunk = 16;

template <class T>
struct Paged {
  T *keys, *values;         // [pages, kv_heads, page, D], [pages, kv_heads, page / 16, D, 16]
  const int32_t *table;     // [batch, longest]
  long long table_stride;
  int pages, kv_heads, shift, longest;   // page == 16 << shift; entries of a sequence
  // First element of a chunk of a page (shared by keys and values).
  template <int D> __device__ __forceinline__ size_t chunk(int id, int h, int c) const {
    return (((size_t)id * kv_heads + h) << shift | (c & ((1 << shift) - 1))) * (kChunk * D);
  }
  __device__ __forceinline__ long long slots() const { return (long long)longest << (shift + 4); }
};

// ------------------------------------------------------------------------------------------------ append
template <class T>
struct PagedAppendParams {
  Paged<T> c;
  Rows<const T> k, v;
  const int64_t *position, *rows;
  Turn turn;
  int seq;
};

// A workgroup takes one chunk of 16 slots that new rows fall into, for all KV heads of a sequence: the chunk's sines and
// cosines are computed once, into LDS.  A thread holds 8 dims of 4 slots, so that keys are written in 16-byte pieces and
// values in the 8 bytes that 4 slots of a dim are.
template <class T, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendParams<T> p) {
  typedef typename Of16<T>::x8 x8;
  typedef typename Of16<T>::x4 x4;
  constexpr int CH = D / 8, PER = 4 * CH, LANES = 256 / PER;   // threads of a head; heads at once
  __shared__ float2 turns[kChunk][D / 2];
  const int tid = threadIdx.x, b = blockIdx.y;
  const int64_t at = p.position[b], n = p.rows ? p.rows[b] : p.seq;
  if (at < 0 || n < 0 || n > p.seq || at > p.c.slots() - n) return;
  const int first = (int)at, end = first + (int)n, chunk = first / kChunk + blockIdx.x, base = chunk * kChunk;
  if (base >= end) return;
  const int id = p.c.table[b * p.c.table_stride + (chunk >> p.c.shift)];
  if ((unsigned)id >= (unsigned)p.c.pages) return;
  const int half = p.turn.frequencies ? p.turn.dims / 2 : 0;
  if (half) {
    for (int i = tid; i < kChunk * half; i += 256) turns[i / half][i % half] = turn_of(p.turn, i % half, (double)(base + i / half));
    __syncthreads();
  }
  const int dim = 8 * (tid % CH), quad = tid / CH % 4;
  const bool pieces = p.turn.neighbours || half % 8 == 0;     // a pair's second dims are a piece too
  for (int h = tid / PER; h < p.c.kv_heads; h += LANES) {
    x8 k[4], v[4];
    uint32_t have = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int slot = base + 4 * quad + i;
      k[i] = v[i] = x8{};
      if (slot < first || slot >= end) continue;
      have |= 1u << i;
      const T *const row = p.k.at(b, slot - first, h);
      k[i] = *reinterpret_cast<const x8 *>(row + dim);
      v[i] = *reinterpret_cast<const x8 *>(p.v.at(b, slot - first, h) + dim);
      if (dim >= 2 * half) continue;
      const float2 *const cs = turns[4 * quad + i];
      if (p.turn.neighbours) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          if (dim + e >= 2 * half) continue;
          const float2 t = cs[(dim + e) / 2];
          const float x = (float)k[i][e], y = (float)k[i][e + 1];
          k[i][e] = (T)(x * t.x - y * t.y);
          k[i][e + 1] = (T)(y * t.x + x * t.y);
        }
      } else {
        x8 other = {};
        if (pieces) other = *reinterpret_cast<const x8 *>(row + (dim < half ? dim + half : dim - half));
        else
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (dim + e < 2 * half) other[e] = row[dim + e < half ? dim + e + half : dim + e - half];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (dim + e >= 2 * half) continue;
          const bool low = dim + e < half;
          const float2 t = cs[low ? dim + e : dim + e - half];
          const float x = (float)k[i][e], y = (float)other[e];
          k[i][e] = (T)(low ? x * t.x - y * t.y : x * t.x + y * t.y);
        }
      }
    }
    const size_t to = p.c.template chunk<D>(id, h, chunk);
    T *const kd = p.c.keys + to + 4 * quad * D + dim, *const vd = p.c.values + to + dim * kChunk + 4 * quad;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (have >> i & 1) *reinterpret_cast<x8 *>(kd + i * D) = k[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (have == 15u) *reinterpret_cast<x4 *>(vd + e * kChunk) = x4{v[0][e], v[1][e], v[2][e], v[3][e]};
      else
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (have >> i & 1) vd[e * kChunk + i] = v[i][e];
    }
  }
}

// ------------------------------------------------------------------------------------------------ attention
template <class T>
struct PagedAttendParams {
  Paged<T> c;
  Rows<const T> q, k, v;    // (row strides unused); k.data null: the token's row is in its page
  Rows<T> out;
  const int64_t *position;
  Turn turn;
  uint32_t *tickets;        // kPagedParts zero words
  float *partial;           // [places][16][D] sums, then [places][16][2] references and totals
  int batch, group, tiles;  // group: query heads of a KV head; tiles of up to 16 of them
  float scale;              // score scale * log2(e)
};

constexpr int kUnit = 2 * kChunk;     // slots of a wave's step
// Parts that the whole work is split into at the most, besides those that sequences and heads are by themselves, and places
// for the sums of parts.
constexpr int kPagedParts = 1024, kPagedPlaces = 2 * kPagedParts + 2;
constexpr int kPagedLeast = 16;       // units of a part at the least
constexpr float kPagedLowest = -3.402823466e38f;
// Probabilities are taken relative to a reference 2^kPagedLift below a row's running maximum when it was set, and it is
// set anew where a score exceeds it by kPagedLift + kPagedSlack (units of log2): fp16 then has the probabilities in
// [2^-24, 2^14], of which the smallest are 2^-34 of the largest.
constexpr float kPagedLift = 10.0f, kPagedSlack = 4.0f;

// Sum over the wave's lanes.
__device__ __forceinline__ uint32_t lanes_sum(uint32_t x) { return __builtin_amdgcn_readlane(kv_scan(x), 63); }

// One new token a sequence.  A workgroup takes a part of a sequence's slots for a KV head (and up to 16 of its query heads),
// its W waves every W-th unit of 32 slots each with a reference and total of their own, joined in LDS; parts are joined by
// the workgroup that counts last.  Which part it takes is found from the positions, on the device.
//
// TURNED: queries are turned by their position (and the new key).  A turned query enters the product as the sum of two numbers of
// the type, so that its rounding (2^-9 of bf16, which large scores would pass on whole) is not added to the held keys'.
template <class T, int D, int W, bool TURNED>
__global__ __launch_bounds__(64 * W) void paged_attend_kernel(PagedAttendParams<T> p) {
  typedef typename Of16<T>::x8 x8;
  typedef typename Of16<T>::x4 x4;
  constexpr int NT = 64 * W, R = 16, U = D / 32, DT = D / 16, PITCH = D + 4, DQ = D / 4, QP = D + 8;
  __shared__ __align__(16) float sums[W][R][PITCH];
  __shared__ float tops[W][R], totals[W][R];
  __shared__ __align__(16) T rows_[R + 2][QP];      // queries, and the new key and value
  __shared__ __align__(16) T low[TURNED ? R : 1][QP];   // what rounding took from the turned queries
  __shared__ float2 turns[TURNED ? D / 2 : 1];
  __shared__ uint32_t word;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};

  // Units of a sequence: those of its slots, none where there is no token, one where it lies outside (to write NaNs).
  const int64_t slots = p.c.slots();
  auto units_of = [&](int64_t at) -> uint32_t { return at < 0 ? 1 : at >= slots ? 1 : (uint32_t)(at / kUnit) + 1; };
  const uint32_t heads = p.c.kv_heads * p.tiles, hh = blockIdx.x % heads, ticket = blockIdx.x / heads;
  const int h = hh / p.tiles, tile = hh % p.tiles;
  const int64_t at0 = lane < p.batch ? p.position[lane] : 0;
  uint32_t all = lane < p.batch ? units_of(at0) : 0;
  for (int i = lane + 64; i < p.batch; i += 64) all += units_of(p.position[i]);
  all = lanes_sum(all);
  const uint32_t most = max((uint32_t)(((uint64_t)all * heads + kPagedParts - 1) / kPagedParts), (uint32_t)kPagedLeast);
  uint32_t b = ~0u, part = 0, ahead = 0, parts_before = 0, units_before = 0;
  int64_t token = 0;
  for (int c = 0; c < p.batch; c += 64) {
    const int64_t at = c == 0 ? at0 : c + lane < p.batch ? p.position[c + lane] : 0;
    const uint32_t n = c + lane < p.batch ? units_of(at) : 0, parts = (n + most - 1) / most;
    const uint32_t upto = kv_scan(n), parts_upto = kv_scan(parts), before = parts_before + parts_upto - parts;
    const uint64_t it = __ballot(ticket >= before && ticket - before < parts);
    if (it) {
      const int who = __builtin_ctzll(it);
      b = c + who;
      part = ticket - __builtin_amdgcn_readlane(before, who);
      ahead = units_before + __builtin_amdgcn_readlane(upto - n, who);
      token = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(at >> 32), who) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)at, who));
      break;
    }
    parts_before += __builtin_amdgcn_readlane(parts_upto, 63);
    units_before += __builtin_amdgcn_readlane(upto, 63);
  }
  if (b == ~0u) return;
  const int rows = min(p.group - 16 * tile, 16), head0 = h * p.group + 16 * tile;
  if (token < 0 || token >= slots) {      // no token: zeros; one that does not lie in the table: NaNs
    const T fill = token == -1 ? (T)0.0f : (T)__builtin_nanf("");
    for (int i = tid; i < rows * D; i += NT) p.out.at(b, 0, head0 + i / D)[i % D] = fill;
    return;
  }
  const int pos = (int)token;
  const uint32_t n = units_of(token), parts = (n + most - 1) / most;
  const uint32_t size = (n + parts - 1) / parts, from = part * size, to = min(n, from + size);
  const bool appends = p.k.data && to == n;

  // Pages: lane l holds that of the wave's unit number l % 32 (from `held` on), its first chunk or, from lane 32 on, its second.
  const int32_t *const table = p.c.table + b * p.c.table_stride;
  const int last_chunk = pos / kChunk;
  bool bad = false;
  auto pages_from = [&](int unit) {
    const int chunk = 2 * (unit + (lane & 31) * W) + (lane >> 5);
    int id = 0;
    if (chunk <= last_chunk && chunk < (int)(2 * to)) {
      id = table[chunk >> p.c.shift];
      if ((unsigned)id >= (unsigned)p.c.pages) {
        id = 0;
        bad = true;
      }
    }
    return id;
  };
  int unit = (int)from + wave, step = 0;
  int ids = pages_from(unit);
  const T *kc[2], *vc[2];
  x8 kn[2][U];
  x4 vn[2][DT];
  auto find = [&](int unit, int step) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int id = __builtin_amdgcn_readlane(ids, step + 32 * t);
      const size_t at = p.c.template chunk<D>(id, h, 2 * unit + t);
      kc[t] = p.c.keys + at;
      vc[t] = p.c.values + at;
    }
  };
  auto fetch_keys = [&]() {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int u = 0; u < U; ++u) kn[t][u] = *reinterpret_cast<const x8 *>(kc[t] + j * D + 32 * u + 8 * g);
  };
  auto fetch_values = [&]() {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int d = 0; d < DT; ++d) vn[t][d] = *reinterpret_cast<const x4 *>(vc[t] + (16 * d + j) * kChunk + 4 * g);
  };
  if (unit < (int)to) {
    find(unit, 0);
    fetch_keys();
    fetch_values();
  }

  // The queries (and the new row) through LDS, turned there.
  const int lines = rows + (appends ? 2 : 0);
  for (int i = tid; i < lines * (D / 8); i += NT) {
    const int r = i / (D / 8), d = i % (D / 8) * 8;
    const T *const src = r < rows ? p.q.at(b, 0, head0 + r) : r == rows ? p.k.at(b, 0, h) : p.v.at(b, 0, h);
    *reinterpret_cast<x8 *>(&rows_[r < rows ? r : R + r - rows][d]) = *reinterpret_cast<const x8 *>(src + d);
    if (TURNED && r < rows) *reinterpret_cast<x8 *>(&low[r][d]) = x8{};
  }
  if constexpr (TURNED) {
    const int half = p.turn.dims / 2;
    for (int i = tid; i < half; i += NT) turns[i] = turn_of(p.turn, i, (double)pos);
    __syncthreads();
    for (int i = tid; i < (rows + (appends ? 1 : 0)) * half; i += NT) {
      const int r = i / half, a = i % half;
      const int dx = pair_first(p.turn, a), dy = dx + pair_step(p.turn);
      T *const row = rows_[r < rows ? r : R];
      const float2 t = turns[a];
      const float x = (float)row[dx], y = (float)row[dy], xt = x * t.x - y * t.y, yt = y * t.x + x * t.y;
      row[dx] = (T)xt;
      row[dy] = (T)yt;
      if (r < rows) {                     // (an infinite one has nothing left)
        low[r][dx] = (T)(fabsf((float)(T)xt) < INFINITY ? xt - (float)(T)xt : 0.0f);
        low[r][dy] = (T)(fabsf((float)(T)yt) < INFINITY ? yt - (float)(T)yt : 0.0f);
      }
    }
  }
  __syncthreads();
  if (appends && tile == 0) {             // the new row to its page
    const int c = pos / kChunk, id = table[c >> p.c.shift];
    if ((unsigned)id < (unsigned)p.c.pages) {
      const size_t at = p.c.template chunk<D>(id, h, c);
      for (int d = tid; d < D; d += NT) {
        p.c.keys[at + (pos % kChunk) * D + d] = rows_[R][d];
        p.c.values[at + d * kChunk + pos % kChunk] = rows_[R + 1][d];
      }
    }
  }
  x8 q[U], ql[TURNED ? U : 1];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    q[u] = *reinterpret_cast<const x8 *>(&rows_[min(j, rows - 1)][32 * u + 8 * g]);
    if constexpr (TURNED) ql[u] = *reinterpret_cast<const x8 *>(&low[min(j, rows - 1)][32 * u + 8 * g]);
  }

  f4 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = zero;
  float ref = kPagedLowest, total = 0.0f;
  for (; unit < (int)to; unit += W) {
    const int base = unit * kUnit, next = unit + W;
    const bool edge = base + kUnit > pos;
    if (edge && appends) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (base + kChunk * t + j == pos)
#pragma unroll
          for (int u = 0; u < U; ++u) kn[t][u] = *reinterpret_cast<const x8 *>(&rows_[R][32 * u + 8 * g]);
    }
    f4 s[2] = {zero, zero};
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if constexpr (TURNED) s[t] = Of16<T>::mma(kn[t][u], ql[u], s[t]);
        s[t] = Of16<T>::mma(kn[t][u], q[u], s[t]);
      }
      s[t] *= p.scale;                    // (before the mask: the scale may be 0 or negative)
    }
    ++step;
    if (step == 32) {                     // the pages of the next 32 units
      ids = pages_from(next);
      step = 0;
    }
    x4 vf[2][DT];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int d = 0; d < DT; ++d) vf[t][d] = vn[t][d];
    if (next < (int)to) {
      find(next, step);
      fetch_keys();
    }
    if (edge) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int slot = base + kChunk * t + 4 * g + e;
          if (slot > pos) s[t][e] = -INFINITY;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            if (slot > pos) vf[t][d][e] = (T)0.0f;
            if (appends && slot == pos) vf[t][d][e] = rows_[R + 1][16 * d + j];
          }
        }
    }
    float top = kPagedLowest;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, s[t][e]);
    if (__any(top - ref > kPagedLift + kPagedSlack)) {
      const float raised = fmaxf(ref, kv_max_across(top) - kPagedLift);
      const float shrink = __builtin_amdgcn_exp2f(ref - raised);
      ref = raised;
      total *= shrink;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= shrink;
    }
    x8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = (T)__builtin_amdgcn_exp2f(s[e / 4][e % 4] - ref);
      total += (float)x[e];
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
      acc[d] = Of16<T>::mma(__builtin_shufflevector(vf[0][d], vf[1][d], 0, 1, 2, 3, 4, 5, 6, 7), x, acc[d]);
    if (next < (int)to) fetch_values();
  }
  if (__any(bad)) total = __builtin_nanf("");

  // The waves' parts: lane (j, g) has dims 16 d + 4 g .. of query j.
#pragma unroll
  for (int d = 0; d < DT; ++d) *reinterpret_cast<f4 *>(&sums[wave][j][16 * d + 4 * g]) = acc[d];
  total += __shfl_xor(total, 16);
  total += __shfl_xor(total, 32);
  if (g == 0) {
    tops[wave][j] = ref;
    totals[wave][j] = total;
  }
  __syncthreads();
  auto store = [&](int r, int d, f4 o, float total) {
    const float inv = 1.0f / total;
    *reinterpret_cast<x4 *>(p.out.at(b, 0, head0 + r) + d) = x4{(T)(o[0] * inv), (T)(o[1] * inv), (T)(o[2] * inv), (T)(o[3] * inv)};
  };
  // Where this part's sums go.  Units (a sequence and head) that are split have more than `most` units of slots each, so that
  // the slots before them over `most` are another number for each, and twice that leaves as many places as it has parts.
  const uint32_t pair = ((uint64_t)ahead * heads + (uint64_t)hh * n) / most;
  const __amdgpu_buffer_rsrc_t po = buffer_rsrc(p.partial, (size_t)kPagedPlaces * R * D * 4);
  const __amdgpu_buffer_rsrc_t pm = buffer_rsrc(p.partial + kPagedPlaces * R * D, (size_t)kPagedPlaces * R * 2 * 4);
  const uint32_t place = 2 * pair + part;
  for (int i = tid; i < rows * DQ; i += NT) {
    const int r = i / DQ, d = i % DQ * 4;
    float top = tops[0][r], sum = 0.0f;
#pragma unroll
    for (int w = 1; w < W; ++w) top = fmaxf(top, tops[w][r]);
    f4 o = zero;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(tops[w][r] - top);
      sum += f * totals[w][r];
      o += f * *reinterpret_cast<const f4 *>(&sums[w][r][d]);
    }
    if (parts == 1) {
      store(r, d, o, sum);
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, o), po, (int)((place * R + r) * D + d) * 4, 0, kSysCoherent);
      if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2v, float2{top, sum}), pm, (int)(place * R + r) * 8, 0, kSysCoherent);
    }
  }
  if (parts == 1) return;
  if (!kv_last_part(p.tickets + pair, parts, &word)) return;
  // The parts of each row, in their order.  Few rows: runs of parts side by side, which meet in LDS.
  const int items = rows * DQ, runs = max(1, NT / items);
  f4 *const met = reinterpret_cast<f4 *>(&sums[0][0][0]);
  float *const stats = reinterpret_cast<float *>(met + NT);
  static_assert(sizeof(sums) >= NT * 24, "paged_attend: LDS for the join");
  for (int at = 0; at < items; at += NT) {
    const int item = at + (runs > 1 ? tid % items : tid), run = runs > 1 ? tid / items : 0;
    const int r = item / DQ, d = item % DQ * 4;
    const bool live = item < items && run < runs;
    constexpr int HELD = 8;
    float top = kPagedLowest, sum = 0.0f;
    f4 o = zero;
    for (uint32_t i = run; live && i < parts; i += HELD * runs) {
      f4 other[HELD];
      float ml[HELD][2];
#pragma unroll
      for (int e = 0; e < HELD; ++e) {
        const uint32_t k = i + e * runs, s = 2 * pair + k;
        const bool there = k < parts;
        other[e] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(po, there ? (int)((s * R + r) * D + d) * 4 : (int)0x80000000u, 0, kSysCoherent));
        const u2v m = __builtin_amdgcn_raw_buffer_load_b64(pm, there ? (int)(s * R + r) * 8 : (int)0x80000000u, 0, kSysCoherent);
        ml[e][0] = there ? __builtin_bit_cast(float, (uint32_t)m[0]) : kPagedLowest;
        ml[e][1] = __builtin_bit_cast(float, (uint32_t)m[1]);
      }
      float raised = top;
#pragma unroll
      for (int e = 0; e < HELD; ++e) raised = fmaxf(raised, ml[e][0]);
      const float shrink = __builtin_amdgcn_exp2f(top - raised);
      top = raised;
      sum *= shrink;
      o *= shrink;
#pragma unroll
      for (int e = 0; e < HELD; ++e) {
        const float f = __builtin_amdgcn_exp2f(ml[e][0] - top);
        sum += f * ml[e][1];
        o += f * other[e];
      }
    }
    if (runs == 1) {
      if (live) store(r, d, o, sum);
      continue;
    }
    if (live) {
      met[tid] = o;
      stats[2 * tid] = top;
      stats[2 * tid + 1] = sum;
    }
    __syncthreads();
    if (run == 0) {
      for (int k = 1; k < runs; ++k) {
        const int other = k * items + item;
        const float raised = fmaxf(top, stats[2 * other]);
        const float f0 = __builtin_amdgcn_exp2f(top - raised), f1 = __builtin_amdgcn_exp2f(stats[2 * other] - raised);
        top = raised;
        sum = sum * f0 + stats[2 * other + 1] * f1;
        o = o * f0 + met[other] * f1;
      }
      store(r, d, o, sum);
    }
  }
}

}  // namespace lb
