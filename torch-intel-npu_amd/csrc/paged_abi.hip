// lb_paged_append and lb_paged_attention: the KV cache in pages.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "lb_paged.h"
#include "serve_check.h"

using namespace lb;
using namespace lb::abi;

namespace {

static_assert(kPagedParts * 4 <= LB_ZEROED_WORKSPACE_BYTES, "tickets are the workspace's zeroed bytes");

template <class T>
Paged<T> cache_params(const lb_paged_cache &c, const lb_page_table &t) {
  Paged<T> p{};
  p.keys = static_cast<T *>(c.keys);
  p.values = static_cast<T *>(c.values);
  p.table = t.data;
  p.table_stride = t.stride;
  p.pages = (int)c.pages;
  p.kv_heads = (int)c.kv_heads;
  p.shift = __builtin_ctzll((unsigned long long)c.page / kChunk);
  p.longest = (int)t.longest;
  return p;
}

// The cache's sizes, and the table's.
lb_status check_shape(const char *what, const lb_paged_cache &c, const lb_page_table &t, int64_t batch) {
  if (c.type > LB_TYPE_BF16) return fail(LB_INVALID_ARGUMENT, "%s: the cache's type must be fp16 or bf16", what);
  if (c.head_dim != 64 && c.head_dim != 128) return fail(LB_UNSUPPORTED, "%s: head_dim %u (64 and 128 are supported)", what, c.head_dim);
  if (c.pages < 1 || c.pages > INT32_MAX || c.kv_heads < 1 || c.kv_heads > 65535)
    return fail(LB_INVALID_ARGUMENT, "%s: pages 1 to 2^31 - 1 and kv_heads 1 to 65535 required", what);
  if (c.page < kChunk || c.page > 1024 || (c.page & (c.page - 1)) != 0)
    return fail(LB_INVALID_ARGUMENT, "%s: page must be a power of two, 16 to 1024 slots", what);
  if (batch < 1 || batch > 65535) return fail(LB_INVALID_ARGUMENT, "%s: batch 1 to 65535 required", what);
  if (t.longest < 1 || t.longest > ((int64_t)1 << 30) / c.page) return fail(LB_INVALID_ARGUMENT, "%s: the table's rows must have 1 to 2^30 / page entries", what);
  if (t.stride < 0 || t.stride > kMaxStride) return fail(LB_INVALID_ARGUMENT, "%s: the table's stride must be 0 to 2^40", what);
  return LB_OK;
}

// Its buffers: keys, values, and the table (read).
lb_status check_cache(const char *what, const lb_paged_cache &c, const lb_page_table &t, int64_t batch, Range (&cache)[2], Range &table) {
  if (const lb_status st = check_shape(what, c, t, batch); st != LB_OK) return st;
  const unsigned __int128 bytes = (unsigned __int128)c.pages * c.kv_heads * c.page * c.head_dim * 2;
  if (bytes > kMaxBytes) return fail(LB_INVALID_ARGUMENT, "%s: the cache does not fit the address space", what);
  if (const lb_status st = check_array(what, "keys", c.keys, (size_t)bytes, 16, true, cache[0]); st != LB_OK) return st;
  if (const lb_status st = check_array(what, "values", c.values, (size_t)bytes, 16, true, cache[1]); st != LB_OK) return st;
  if (overlaps(cache[0], cache[1])) return fail(LB_INVALID_ARGUMENT, "%s: keys overlaps values", what);
  return check_array(what, "table", t.data, (size_t)((batch - 1) * t.stride + t.longest) * 4, 4, true, table);
}

template <class F>
void with_kind(const lb_paged_cache &c, F &&f) {
  typedef std::integral_constant<int, 64> D64;
  typedef std::integral_constant<int, 128> D128;
  if (c.type == LB_TYPE_FP16) c.head_dim == 64 ? f(f16{}, D64{}) : f(f16{}, D128{});
  else c.head_dim == 64 ? f(bf16{}, D64{}) : f(bf16{}, D128{});
}

struct AttendPlan {
  int tiles, waves, rounds;
  int64_t grid;
  size_t bytes;
};

AttendPlan attend_plan(const lb_paged_attention_args *a) {
  AttendPlan plan{};
  const lb_paged_cache &c = a->cache;
  plan.tiles = (int)((a->heads / c.kv_heads + 15) / 16);
  const int64_t heads = c.kv_heads * plan.tiles, pairs = heads * a->batch;
  // Eight waves a workgroup; where heads of 128, whose registers leave room for one on a CU, are more than CUs, two of four
  // (54 sequences of up to 22 slots, 8 heads: 11.3 -> 7.9 us; 40 of up to 2001 39.6 -> 38.0; 33 of up to 8192 98.5 -> 98.7.
  // 128 of up to 800, 3 heads of 64: 13.8 with eight, 15.3 with four).
  plan.waves = c.head_dim == 128 && pairs > 256 ? 4 : 8;
  // A workgroup per sequence and head, and where sequences can be long enough the rounds of 256 or 512 that they can be split into:
  // few sequences are split evenly in one, more of them need more to end together.
  const bool split = a->table.longest * c.page > paged_whole((int)c.head_dim);
  plan.rounds = pairs <= 128 ? 1 : kPagedParts / (256 * 8 / plan.waves);
  plan.grid = pairs + (split ? plan.rounds * (256 * 8 / plan.waves) : 0);
  plan.grid = (plan.grid + heads - 1) / heads * heads;   // whole tickets
  plan.bytes = split ? LB_ZEROED_WORKSPACE_BYTES + (size_t)kPagedPlaces * 16 * (c.head_dim + 2) * sizeof(float) : 0;
  return plan;
}

lb_status check_heads(const char *what, const lb_paged_attention_args *a) {
  const lb_paged_cache &c = a->cache;
  if (a->heads < 1 || a->heads > 65535 || a->heads % c.kv_heads != 0)
    return fail(LB_INVALID_ARGUMENT, "%s: heads must be a multiple of kv_heads up to 65535", what);
  if (!std::isfinite(a->scale)) return fail(LB_INVALID_ARGUMENT, "%s: scale must be finite", what);
  const int64_t tiles = (a->heads / c.kv_heads + 15) / 16;
  if (a->batch * c.kv_heads * tiles > (1 << 22)) return fail(LB_UNSUPPORTED, "%s: more than 2^22 sequences times heads", what);
  if (a->batch * ((a->table.longest * c.page + 31) / 32) > (int64_t)1 << 31)
    return fail(LB_UNSUPPORTED, "%s: a batch of more than 2^36 slots", what);
  return LB_OK;
}

}  // namespace

extern "C" {

lb_status lb_paged_append(const lb_paged_append_args *a, void *stream) {
  const char *what = "lb_paged_append";
  if (const lb_status bad = refuse_if_failed(what); bad != LB_OK) return bad;
  if (!a) return fail(LB_INVALID_ARGUMENT, "%s: args is NULL", what);
  if (a->struct_size < sizeof *a) return fail(LB_INVALID_ARGUMENT, "%s: struct_size %u < %zu", what, a->struct_size, sizeof *a);
  const lb_paged_cache &c = a->cache;
  Range cache[2], reads[6];
  if (const lb_status st = check_cache(what, c, a->table, a->batch, cache, reads[0]); st != LB_OK) return st;
  if (a->seq < 1 || a->seq > kMaxSeq) return fail(LB_INVALID_ARGUMENT, "%s: seq 1 to 2^25 required", what);
  if (const lb_status st = check_strided(what, "k", a->k, a->batch, a->seq, c.kv_heads, c.head_dim, 2, true, false, reads[1]); st != LB_OK) return st;
  if (const lb_status st = check_strided(what, "v", a->v, a->batch, a->seq, c.kv_heads, c.head_dim, 2, true, false, reads[2]); st != LB_OK) return st;
  if (const lb_status st = check_array(what, "position", a->position, (size_t)a->batch * 8, 8, true, reads[3]); st != LB_OK) return st;
  if (const lb_status st = check_array(what, "rows", a->rows, (size_t)a->batch * 8, 8, false, reads[4]); st != LB_OK) return st;
  if (const lb_status st = check_rotation(what, a->rotation, c.head_dim, false, reads[5]); st != LB_OK) return st;
  if (const lb_status st = check_apart(what, cache, 2, reads, 6); st != LB_OK) return st;
  // Chunks that seq consecutive slots can fall into, wherever the first lies.
  const int64_t chunks = std::min((a->seq + 2 * kChunk - 2) / kChunk, a->table.longest * c.page / kChunk);
  // Heads of a workgroup: they share its sines and cosines, so as many as leave two workgroups a CU (8 heads of 128: prompts of 4100,
  // 3476, 2526 and 951 rows, 2, 4, 8 heads 23.1, 22.3, 20.5 us; one of 4096 rows 10.2, 9.4, 10.0).  Threads: up to 1024, of which three
  // of four have something to do (the first of these with 8 heads in 256, 512, 1024: 26.8, 24.3, 20.5; 4 x 8000 rows of 5 heads of 64
  // in 256, 512: 17.9, 19.6; 8 x 2000 of 3: 9.3, 8.3).
  const int64_t heads = std::max<int64_t>(1, std::min<int64_t>(c.kv_heads, chunks * a->batch * c.kv_heads / 512));
  int threads = 1024;
  for (; threads > 256; threads /= 2) {
    const int64_t beside = threads / (kChunk * (int64_t)c.head_dim / 8);   // heads at once
    if ((heads + beside - 1) / beside * beside * 3 <= heads * 4) break;
  }
  with_kind(c, [&](auto type, auto dim) {
    typedef decltype(type) T;
    PagedAppendParams<T> p{};
    p.c = cache_params<T>(c, a->table);
    p.k = strided<const T>(a->k);
    p.v = strided<const T>(a->v);
    p.position = a->position;
    p.rows = a->rows;
    p.turn = turn_params(a->rotation);
    p.seq = (int)a->seq;
    p.heads = (int)heads;
    const dim3 grid((unsigned)chunks, (unsigned)a->batch, (unsigned)((c.kv_heads + heads - 1) / heads));
    auto go = [&](auto nt) {
      hipLaunchKernelGGL((paged_append_kernel<T, dim(), decltype(nt)::value>), grid, dim3(threads), 0, static_cast<hipStream_t>(stream), p);
    };
    threads == 1024 ? go(std::integral_constant<int, 1024>{}) : threads == 512 ? go(std::integral_constant<int, 512>{})
                                                                              : go(std::integral_constant<int, 256>{});
  });
  return launch_status(what);
}

lb_status lb_paged_attention_workspace_bytes(const lb_paged_attention_args *a, size_t *bytes) {
  const char *what = "lb_paged_attention_workspace_bytes";
  if (!a || !bytes) return fail(LB_INVALID_ARGUMENT, "%s: args and bytes must be non-NULL", what);
  *bytes = 0;
  if (a->struct_size < sizeof *a) return fail(LB_INVALID_ARGUMENT, "%s: struct_size %u < %zu", what, a->struct_size, sizeof *a);
  if (const lb_status st = check_shape(what, a->cache, a->table, a->batch); st != LB_OK) return st;
  if (const lb_status st = check_heads(what, a); st != LB_OK) return st;
  *bytes = attend_plan(a).bytes;
  return ok();
}

lb_status lb_paged_attention(const lb_paged_attention_args *a, void *stream) {
  const char *what = "lb_paged_attention";
  if (const lb_status bad = refuse_if_failed(what); bad != LB_OK) return bad;
  if (!a) return fail(LB_INVALID_ARGUMENT, "%s: args is NULL", what);
  if (a->struct_size < sizeof *a) return fail(LB_INVALID_ARGUMENT, "%s: struct_size %u < %zu", what, a->struct_size, sizeof *a);
  const lb_paged_cache &c = a->cache;
  const bool appends = a->k.data || a->v.data;
  Range cache[2], reads[6], out;
  if (const lb_status st = check_cache(what, c, a->table, a->batch, cache, reads[0]); st != LB_OK) return st;
  if (const lb_status st = check_heads(what, a); st != LB_OK) return st;
  if (const lb_status st = check_strided(what, "q", a->q, a->batch, 1, a->heads, c.head_dim, 2, true, false, reads[1]); st != LB_OK) return st;
  if (const lb_status st = check_strided(what, "out", a->out, a->batch, 1, a->heads, c.head_dim, 2, true, true, out); st != LB_OK) return st;
  if (const lb_status st = check_array(what, "position", a->position, (size_t)a->batch * 8, 8, true, reads[2]); st != LB_OK) return st;
  if (const lb_status st = check_rotation(what, a->rotation, c.head_dim, false, reads[3]); st != LB_OK) return st;
  if (appends) {
    if (const lb_status st = check_strided(what, "k", a->k, a->batch, 1, c.kv_heads, c.head_dim, 2, true, false, reads[4]); st != LB_OK) return st;
    if (const lb_status st = check_strided(what, "v", a->v, a->batch, 1, c.kv_heads, c.head_dim, 2, true, false, reads[5]); st != LB_OK) return st;
  }
  const AttendPlan plan = attend_plan(a);
  if (plan.bytes && (!a->workspace || !aligned(a->workspace, 256) || a->workspace_bytes < plan.bytes))
    return fail(LB_INVALID_ARGUMENT, "%s: a 256-byte aligned workspace of %zu bytes required (got %zu)", what, plan.bytes, a->workspace_bytes);
  const Range writes[] = {out, plan.bytes ? range_of(a->workspace, plan.bytes, "workspace") : Range{}};
  if (const lb_status st = check_apart(what, writes, 2, reads, 6); st != LB_OK) return st;
  if (const lb_status st = check_apart(what, writes, 2, cache, 2); st != LB_OK) return st;
  if (appends)
    if (const lb_status st = check_apart(what, cache, 2, reads, 6); st != LB_OK) return st;
  with_kind(c, [&](auto type, auto dim) {
    typedef decltype(type) T;
    PagedAttendParams<T> p{};
    p.c = cache_params<T>(c, a->table);
    p.q = strided<const T>(a->q);
    p.out = strided<T>(a->out);
    if (appends) {
      p.k = strided<const T>(a->k);
      p.v = strided<const T>(a->v);
    }
    p.position = a->position;
    p.turn = turn_params(a->rotation);
    p.tickets = static_cast<uint32_t *>(a->workspace);
    p.partial = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + LB_ZEROED_WORKSPACE_BYTES);
    p.rounds = plan.rounds;
    p.batch = (int)a->batch;
    p.group = (int)(a->heads / c.kv_heads);
    p.tiles = plan.tiles;
    p.scale = a->scale * 1.44269504088896340736f;
    auto go = [&](auto waves) {
      constexpr int W = decltype(waves)::value;
      const dim3 grid((unsigned)plan.grid), block(64 * W);
      if (p.turn.frequencies) hipLaunchKernelGGL((paged_attend_kernel<T, dim(), W, true>), grid, block, 0, static_cast<hipStream_t>(stream), p);
      else hipLaunchKernelGGL((paged_attend_kernel<T, dim(), W, false>), grid, block, 0, static_cast<hipStream_t>(stream), p);
    };
    if constexpr (dim() == 128) {
      if (plan.waves == 4) return go(std::integral_constant<int, 4>{});
    }
    go(std::integral_constant<int, 8>{});
  });
  return launch_status(what);
}

}  // extern "C"
