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
  int seq, heads;           // heads: KV heads of a workgroup
};

// A workgroup takes one chunk of 16 slots that new rows fall into, for `heads` KV heads of a sequence.  Values are read in rows and
// turned in LDS into the 16 bytes that 8 slots of a dim are, so that both sides move whole lines; the chunk's sines and cosines are
// computed behind their loads, once for all heads, into LDS; then keys, 8 dims of a row a thread.  (One loop body for every
// key: straight-line code of four rows took a short call as long to fetch as to run.)  Memory bounds it where rows are many: prompts
// of 4100, 3476, 2526 and 951 rows of 8 heads of 128, bf16, 90 MB in and out, take 20.9 us (4.3 TB/s).  500 rows of 3 heads
// of 64 take 4.3: the launch, and the positions, the table and the rows one after the other.
template <class T, int D, int NT>
__global__ __launch_bounds__(NT) void paged_append_kernel(PagedAppendParams<T> p) {
  typedef typename Of16<T>::x8 x8;
  constexpr int CH = D / 8, LANES = NT / (kChunk * CH), PITCH = D + 8;   // pieces of a row; heads at once
  __shared__ float2 turns[kChunk][D / 2];
  __shared__ __align__(16) T tile[LANES][kChunk][PITCH];
  const int tid = threadIdx.x, b = blockIdx.y, head0 = blockIdx.z * p.heads, head1 = min(head0 + p.heads, p.c.kv_heads);
  const int64_t at = p.position[b], n = p.rows ? p.rows[b] : p.seq;
  if (at < 0 || n < 0 || n > p.seq || at > p.c.slots() - n) return;
  const int first = (int)at, end = first + (int)n, chunk = first / kChunk + blockIdx.x, base = chunk * kChunk;
  if (base >= end) return;
  const int id = p.c.table[b * p.c.table_stride + (chunk >> p.c.shift)];
  if ((unsigned)id >= (unsigned)p.c.pages) return;
  const int from = max(first, base), to = min(end, base + kChunk);
  const int half = p.turn.frequencies ? p.turn.dims / 2 : 0;
  const int lane = tid / (kChunk * CH), piece = tid % (kChunk * CH), mine = base + piece / CH;   // this thread's piece of a head, its slot
  auto value = [&](int h) {
    return h < head1 && mine >= from && mine < to ? read_once<x8>(p.v.at(b, mine - first, h) + 8 * (piece % CH)) : x8{};
  };
  x8 next = value(head0 + lane);
#pragma unroll 1
  for (int i = tid; i < kChunk * (D / 2); i += NT)
    if (i % (D / 2) < half) turns[i / (D / 2)][i % (D / 2)] = turn_of(p.turn, i % (D / 2), (double)(base + i / (D / 2)));
  for (int h0 = head0; h0 < head1; h0 += LANES) {
    *reinterpret_cast<x8 *>(&tile[lane][piece / CH][8 * (piece % CH)]) = next;
    __syncthreads();
    next = value(h0 + LANES + lane);
    const int h = h0 + lane, dim = piece / 2, low = 8 * (piece % 2);      // 8 slots of a dim
    if (h < head1) {
      x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = tile[lane][low + e][dim];
      T *const out = p.c.values + p.c.template chunk<D>(id, h, chunk) + dim * kChunk + low;
      if (base + low >= from && base + low + 8 <= to) {
        *reinterpret_cast<x8 *>(out) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (base + low + e >= from && base + low + e < to) out[e] = v[e];
      }
    }
    __syncthreads();
  }
  // Keys.
  const bool pieces = p.turn.neighbours || half % 8 == 0;     // a pair's second dims are a piece too
  const int items = (head1 - head0) * (kChunk * CH);
  for (int i = tid; i < items; i += NT) {
    const int dim = 8 * (i % CH), slot = base + i / CH % kChunk, h = head0 + i / (CH * kChunk);
    if (slot < from || slot >= to) continue;
    const T *const row = p.k.at(b, slot - first, h);
    x8 k = *reinterpret_cast<const x8 *>(row + dim);
    if (dim < 2 * half) {
      const float2 *const cs = turns[slot - base];
      if (p.turn.neighbours) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          if (dim + e >= 2 * half) continue;
          const float2 t = cs[(dim + e) / 2];
          const float x = (float)k[e], y = (float)k[e + 1];
          k[e] = (T)(x * t.x - y * t.y);
          k[e + 1] = (T)(y * t.x + x * t.y);
        }
      } else {
        x8 other = {};
        if (pieces) {
          other = *reinterpret_cast<const x8 *>(row + (dim < half ? dim + half : dim - half));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (dim + e < 2 * half) other[e] = row[dim + e < half ? dim + e + half : dim + e - half];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (dim + e >= 2 * half) continue;
          const bool low = dim + e < half;
          const float2 t = cs[low ? dim + e : dim + e - half];
          const float x = (float)k[e], y = (float)other[e];
          k[e] = (T)(low ? x * t.x - y * t.y : x * t.x + y * t.y);
        }
      }
    }
    *reinterpret_cast<x8 *>(p.c.keys + p.c.template chunk<D>(id, h, chunk) + (slot - base) * D + dim) = k;
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
  int rounds;               // of workgroups that fit on the chip, besides those of sequences and heads: what the grid has
  int batch, group, tiles;  // group: query heads of a KV head; tiles of up to 16 of them
  float scale;              // score scale * log2(e)
};

constexpr int kUnit = 2 * kChunk;     // slots of a wave's step
// Parts that the whole work is split into at the most, besides those that sequences and heads are by themselves, and places
// for the sums of parts.
constexpr int kPagedParts = 1024, kPagedPlaces = 2 * kPagedParts + 2;
// Slots of a sequence up to which it is never split (the host leaves out what only splitting needs).
constexpr int paged_whole(int dim) { return (dim == 64 ? 32 : 16) * kUnit; }
constexpr float kPagedLowest = -3.402823466e38f;
// Probabilities are taken relative to a reference kPagedLift below a row's running maximum when it was set, and it is set anew where
// a score exceeds it by kPagedLift + kPagedSlack (units of log2).  fp16 then has the probabilities in [2^-24, 2^14], of which the
// smallest are 2^-34 of the largest.  bf16 has exponents enough, and takes them up to 2^-20: the values of 2^20 slots, whatever their
// size, stay in the range of a sum.
template <class T> constexpr float kPagedLift = 10.0f;
template <> inline constexpr float kPagedLift<bf16> = -24.0f;
constexpr float kPagedSlack = 4.0f;

// Sum over the wave's lanes.
__device__ __forceinline__ uint32_t lanes_sum(uint32_t x) { return __builtin_amdgcn_readlane(kv_scan(x), 63); }

// The largest of them.
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x111, 0xF, 0xF, true));   // row_shr 1, 2, 4, 8
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x112, 0xF, 0xF, true));
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x114, 0xF, 0xF, true));
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x118, 0xF, 0xF, true));
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x142, 0xA, 0xF, false));  // row_bcast 15, 31
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x143, 0xC, 0xF, false));
  return __builtin_amdgcn_readlane(x, 63);
}

// One new token a sequence.  A workgroup takes a part of a sequence's slots for a KV head (and up to 16 of its query heads),
// its W waves every W-th unit of slots each with a reference and total of their own, joined in LDS; parts are joined by
// the workgroup that counts last.  Which part it takes is found from the positions, on the device.
//
// Memory bounds it where the slots are many, 16-bit keys and values read once: one sequence of 130999 slots, 8 heads of 128, takes
// 86.5 us (6.2 TB/s), 64 of up to 8193 178 us (6.1).  The products take K (as rows of 16 slots) and V (as rows of 16 dims) straight from
// their pages, and P comes out of one as the operand of the other, so LDS holds only what waves exchange.  Few slots cost the
// chain of loads (positions, table, keys and values: 5.8 us for 150), and parts another 4 us (sums out, count, sums in).
//
// Batches of more than 64 keep a simpler plan, parts of a 1024th of the work but never of sequences that are short, and every workgroup
// goes through the positions up to its own: as the square of the batch where sequences are short (3 heads of 64, up to 60 slots: 64, 256,
// 1024 and 4096 sequences 5.2, 11.0, 55.7, 534 us), hardly where they are long (8 heads of 128, up to 2000 slots: 64, 128 and 256
// sequences 53.0, 95.6, 173 us; 64 and 65 with one of 60001 slots, 16 query heads over one of 128, 25.3, 27.0).  Of more than 16 query
// heads a KV head, each tile of 16 reads the slots anew, side by side, the second time mostly from the caches (131000 slots, one
// head of 64: 16 and 24 query heads 20.6, 22.1 us).
//
// TURNED: queries are turned by their position (and the new key).  A turned query enters the product as the sum of two numbers of
// the type, so that its rounding (2^-8 of bf16, which large scores would pass on whole) is not added to the held keys'.
template <class T, int D, int W, bool TURNED>
__global__ __launch_bounds__(64 * W) void paged_attend_kernel(PagedAttendParams<T> p) {
  typedef typename Of16<T>::x8 x8;
  typedef typename Of16<T>::x4 x4;
  constexpr int NT = 64 * W, R = 16, U = D / 32, DT = D / 16, C = 2, UNIT = kUnit, PER = 64 / C, PITCH = D + 4, DQ = D / 4, QP = D + 8;
  __shared__ __align__(16) float sums[W][R][PITCH];
  __shared__ float tops[W][R], totals[W][R];
  __shared__ __align__(16) T rows_[R + 2][QP];      // queries, and the new key and value
  __shared__ __align__(16) T low[TURNED ? R : 1][QP];   // what rounding took from the turned queries
  __shared__ float2 turns[TURNED ? D / 2 : 1];
  __shared__ uint32_t word;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};

  // Units of a sequence: those of its slots, one where there is no token or it lies outside (to write zeros or NaNs).
  const int64_t slots = p.c.slots();
  auto units_of = [&](int64_t at) -> uint32_t { return at < 0 || at >= slots ? 1 : (uint32_t)(at / UNIT) + 1; };
  const uint32_t heads = p.c.kv_heads * p.tiles, hh = blockIdx.x % heads, ticket = blockIdx.x / heads;
  const int h = hh / p.tiles, tile = hh % p.tiles;
  const int64_t at0 = lane < p.batch ? p.position[lane] : 0;
  uint32_t all = lane < p.batch ? units_of(at0) : 0;
  for (int i = lane + 64; i < p.batch; i += 64) all += units_of(p.position[i]);
  all = lanes_sum(all);
  // Units of a part at the most.  As many workgroups of W waves as fit on the chip are a round, which takes `kStart` units' time
  // to start; the memory takes 1.4 times a CU's time for its share of the work.  So as few rounds as cost the least (half a part
  // of a sequence and head lies idle in the mean), and parts no smaller than they must be to fit in them.  (Parts are never
  // more than sequences times heads and the rounds': each sequence has less than one part over what its share of the work is.)
  // Short sequences are not split, for joining parts takes 4 us (one of 500 slots, 3 heads of 64: 6.6 us whole, 8.0 split; of 1200
  // 9.6 and 8.1; two of 803, one head of 128: 11.7 and 9.3).  Where they are, parts may be small: 8 units, one for each wave.  But the
  // workgroup that joins n parts reads n sums of as many rows as it has query heads, a CU by itself, while each part takes 1 / n of the
  // slots, read at that rate too: the two are even where a part has sqrt(units x query heads / 32) units (16 heads of 128 over one KV
  // head, a sequence of 60001 slots: 39.7 -> 25.3 us; 24 of 64, two of up to 26499: 15.0 -> 13.5).
  constexpr int kRound = 256 * 8 / W;
  constexpr uint32_t kWhole = paged_whole(D) / kUnit, kLeast = 8;
  uint32_t most = kWhole;
  if (p.batch > 64) {
    most = max((uint32_t)(((uint64_t)all * heads + kRound * p.rounds - 1) / (kRound * p.rounds)), most);
  } else {
    const uint32_t n = lane < p.batch ? units_of(at0) : 0;
    if (__any(n > most)) {
      constexpr float kStart = D == 128 ? 10.0f : 20.0f;
      const float work = (float)all * heads, pairs = (float)p.batch * heads;
      const float longest = (float)lanes_max(n);
      float least = INFINITY, size = 0.0f;
      uint32_t room = 0;
      for (int k = 1; k <= p.rounds; ++k) {
        const float m = fminf(longest, work * __builtin_amdgcn_rcpf(fmaxf((float)kRound * k - 0.5f * pairs, 1.0f)));
        const float cost = fmaxf(work * (1.4f / 256), k * (8 / W) * (fmaxf(m, (float)kLeast) + kStart));
        if (kRound * k >= pairs && cost < 0.95f * least) {
          least = cost;
          size = m;
          room = kRound * k;
        }
      }
      if (room == 0) {                    // more sequences and heads than that
        room = ~0u;
        size = work / (float)(kRound * p.rounds);
      }
      const uint32_t even = __builtin_amdgcn_sqrtf(longest * min(p.group, 16) * (1.0f / 32));
      most = max(max((uint32_t)size + 1, kLeast), even);
      for (int i = 0; i < 4 && lanes_sum((n + most - 1) / most) * heads > room; ++i) most += most / 8 + 1;
    }
  }
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

  // Pages: lane l holds that of chunk l / PER of the wave's unit number l % PER (from a first one on).
  const int32_t *const table = p.c.table + b * p.c.table_stride;
  const int last_chunk = pos / kChunk;
  bool bad = false;
  auto pages_from = [&](int unit) {
    const int chunk = C * (unit + lane % PER * W) + lane / PER;
    int id = 0;
    if (chunk <= last_chunk && chunk < (int)(C * to)) {
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
  // Every load is 1 KB of whole lines of one chunk (lanes with 64 bytes of 16 rows each take the address unit more than twice as
  // long).  Of the keys of two chunks, 32 slots, product s has 8 rows of each, slots 8 q + 4 s + r (r = 0 .. 3) of the 8 q from
  // row 4 q on: half a line by lanes j < 8, the other by j >= 8, who then swap.  The lanes (., g) thus get the scores of
  // slots 8 g .. 8 g + 7 in the two products.  Of the values, two tiles of 16 dims by halves of the wave, swapped likewise.
  const int kd = (8 * (j / 4 % 2) + j % 4) * D + 32 * (j / 8) + 8 * g, vd = (16 * (g / 2) + j) * kChunk + 8 * (g % 2);
  const T *kc[C], *vc[C];
  u4 kn[C][U], vn[C][DT / 2];             // [chunk][4-slot product s, 64 dims], [chunk][32 dims]
  auto find = [&](int unit, int step) {
#pragma unroll
    for (int t = 0; t < C; ++t) {
      const int id = __builtin_amdgcn_readlane(ids, step + PER * t);
      const size_t at = p.c.template chunk<D>(id, h, C * unit + t);
      kc[t] = p.c.keys + at;
      vc[t] = p.c.values + at;
    }
  };
  auto fetch_keys = [&]() {
#pragma unroll
    for (int t = 0; t < C; ++t)
#pragma unroll
      for (int u = 0; u < U; ++u) kn[t][u] = read_once<u4>(kc[t] + kd + (u & 1) * 4 * D + u / 2 * 64);
  };
  auto fetch_values = [&]() {
#pragma unroll
    for (int t = 0; t < C; ++t)
#pragma unroll
      for (int d = 0; d < DT / 2; ++d) vn[t][d] = read_once<u4>(vc[t] + vd + d * 32 * kChunk);
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
    const int base = unit * UNIT, next = unit + W;
    const bool edge = base + UNIT > pos;
    f4 s[C];                              // s[2 t + i]: slots base + 32 t + 8 g + 4 i ..
#pragma unroll
    for (int t = 0; t < C; t += 2)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool fresh = edge && appends && base + 16 * t + 8 * (j / 4) + 4 * i + j % 4 == pos;
        s[t + i] = zero;
#pragma unroll
        for (int u = 0; u < U; u += 2) {  // 64 dims
          u4 a[2];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a[0][e] = __builtin_amdgcn_update_dpp(kn[t][u + i][e], kn[t + 1][u + i][e], 0x128, 0xF, 0xC, false);   // row_ror 8, lanes 8 .. 15
            a[1][e] = __builtin_amdgcn_update_dpp(kn[t + 1][u + i][e], kn[t][u + i][e], 0x128, 0xF, 0x3, false);   // lanes 0 .. 7
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const x8 k = __builtin_bit_cast(x8, fresh ? *reinterpret_cast<const u4 *>(&rows_[R][32 * (u + c) + 8 * g]) : a[c]);
            if constexpr (TURNED) s[t + i] = Of16<T>::mma(k, ql[u + c], s[t + i]);
            s[t + i] = Of16<T>::mma(k, q[u + c], s[t + i]);
          }
        }
        s[t + i] *= p.scale;              // (before the mask: the scale may be 0 or negative)
      }
    if (++step == PER) {                  // the pages of the next units
      ids = pages_from(next);
      step = 0;
    }
    if (next < (int)to) {
      find(next, step);
      fetch_keys();
    }
    x8 vf[C / 2][DT];                     // 8 slots base + 32 t + 8 g .. of dim 16 d + j
#pragma unroll
    for (int t = 0; t < C; t += 2)
#pragma unroll
      for (int d = 0; d < DT; d += 2) {
        u4 lo, hi;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const auto two = __builtin_amdgcn_permlane32_swap(vn[t][d / 2][e], vn[t + 1][d / 2][e], false, false);
          lo[e] = two[0];
          hi[e] = two[1];
        }
        vf[t / 2][d] = __builtin_bit_cast(x8, lo);
        vf[t / 2][d + 1] = __builtin_bit_cast(x8, hi);
      }
    if (edge) {
#pragma unroll
      for (int t = 0; t < C / 2; ++t) {
        const int there = pos + 1 - (base + 32 * t + 8 * g), held = there - (appends ? 1 : 0);   // slots that there are, and values held
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e >= there) s[2 * t + e / 4][e % 4] = -INFINITY;
        u4 mask, mine;                    // of the values: what is kept, and where the new one goes
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          mask[e] = (2 * e < held ? 0xFFFFu : 0u) | (2 * e + 1 < held ? 0xFFFF0000u : 0u);
          mine[e] = !appends || held < 2 * e || held > 2 * e + 1 ? 0u : held & 1 ? 0xFFFF0000u : 0xFFFFu;
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const uint32_t fresh = __builtin_bit_cast(uint16_t, rows_[R + 1][16 * d + j]) * 0x10001u;
          vf[t][d] = __builtin_bit_cast(x8, (__builtin_bit_cast(u4, vf[t][d]) & mask) | (mine & fresh));
        }
      }
    }
    float top = kPagedLowest;
#pragma unroll
    for (int t = 0; t < C; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, s[t][e]);
    if (__any(top - ref > kPagedLift<T> + kPagedSlack)) {
      // (Where a score's own step is 16, from 2^27 on, the difference rounds to one past what fp16 has room for.)
      const float largest = kv_max_across(top), below = largest - kPagedLift<T>;
      const float raised = fmaxf(ref, largest - below > kPagedLift<T> + kPagedSlack ? largest : below);
      const float shrink = __builtin_amdgcn_exp2f(ref - raised);
      ref = raised;
      total *= shrink;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= shrink;
    }
    // A probability enters the product as the sum of two numbers of the type, for its rounding to one (2^-8 of it in bf16, 2^-11 in fp16)
    // is as large as the output's own, and larger where values cancel (one sequence of 130999 slots, 8 heads of 128, bf16: 86.0 -> 86.4
    // us; 32 of up to 1984, 3 of 64, fp16: 11.35 -> 11.45; 4 of 1000: 10.8 -> 11.1; 64 of up to 8192, 8 of 128: 177.1 -> 178.2).  fp16's first
    // number is cut off rather than rounded, which leaves the second as exact and needs no conversion back (4 of 1000: 11.2 -> 11.1).
    x8 x[C / 2], rest[C / 2];
#pragma unroll
    for (int t = 0; t < C; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float prob = __builtin_amdgcn_exp2f(s[t][e] - ref);
        const float high = __is_same(T, f16) ? __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, prob) & 0xFFFFE000u) : (float)(T)prob;
        x[t / 2][t % 2 * 4 + e] = (T)high;
        rest[t / 2][t % 2 * 4 + e] = (T)(prob - high);
        total += prob;
      }
#pragma unroll
    for (int t = 0; t < C; t += 2)
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        acc[d] = Of16<T>::mma(vf[t / 2][d], x[t / 2], acc[d]);
        acc[d] = Of16<T>::mma(vf[t / 2][d], rest[t / 2], acc[d]);
      }
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
