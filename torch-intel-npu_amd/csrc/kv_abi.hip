// lb_kv_append, lb_kv_read and lb_kv_attention: the KV cache in 8 bits.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/lowbit_decode_hip.h"
#include "abi_util.h"
#include "lb_kv.h"

using namespace lb;
using namespace lb::abi;

namespace {

constexpr int64_t kMaxCapacity = (int64_t)1 << 28, kMaxStride = (int64_t)1 << 40, kMaxRows = (int64_t)1 << 28;
constexpr size_t kMaxBytes = (size_t)1 << 60;   // (no buffer is larger; sums of a few stay in 64 bits)
constexpr float kMaxScale = 65536.0f;   // |q| and |k| are below 2^16, so scores stay within 2^56

KvCache cache_params(const lb_kv_cache &c) {
  KvCache p{};
  p.kc = static_cast<uint8_t *>(c.key_codes);
  p.vc = static_cast<uint8_t *>(c.value_codes);
  p.ks = c.key_scales;
  p.vs = c.value_scales;
  p.kt = static_cast<f16 *>(c.key_tail);
  p.vt = static_cast<f16 *>(c.value_tail);
  p.kv_heads = (int)c.kv_heads;
  p.capacity = (int)c.capacity;
  p.blocks = (int)(c.capacity / kKvBlock);
  return p;
}

KvRows rows_params(const lb_kv_rows &r) {
  return {static_cast<f16 *>(const_cast<void *>(r.data)), (long long)r.batch_stride, (long long)r.row_stride, (long long)r.head_stride};
}

// The cache's buffers, and whether they are sound.
lb_status check_cache(const char *what, const lb_kv_cache &c, Range (&r)[6]) {
  if (c.format > LB_KV_FP8) return fail(LB_INVALID_ARGUMENT, "%s: unknown cache format %u", what, c.format);
  if (c.head_dim != 64 && c.head_dim != 128) return fail(LB_UNSUPPORTED, "%s: head_dim %u (64 and 128 are supported)", what, c.head_dim);
  if (c.batch < 1 || c.batch > 65535 || c.kv_heads < 1 || c.kv_heads > 65535 || c.capacity < kKvBlock || c.capacity > kMaxCapacity ||
      c.capacity % kKvBlock != 0)
    return fail(LB_INVALID_ARGUMENT, "%s: batch and kv_heads 1..65535, capacity a multiple of %d up to 2^28 required", what, kKvBlock);
  const size_t heads = (size_t)c.batch * c.kv_heads;
  if (heads > kMaxBytes / ((size_t)c.capacity * c.head_dim))
    return fail(LB_INVALID_ARGUMENT, "%s: the cache's codes do not fit the address space", what);
  const size_t codes = heads * c.capacity * c.head_dim, scales = heads * (c.capacity / kKvBlock) * 4,
               tail = heads * (2 * kKvBlock) * c.head_dim * 2;   // (heads below 2^32, so scales below 2^56, tails 2^47)
  r[0] = range_of(c.key_codes, codes, "key_codes");
  r[1] = range_of(c.value_codes, codes, "value_codes");
  r[2] = range_of(c.key_scales, scales, "key_scales");
  r[3] = range_of(c.value_scales, scales, "value_scales");
  r[4] = range_of(c.key_tail, tail, "key_tail");
  r[5] = range_of(c.value_tail, tail, "value_tail");
  for (int i = 0; i < 6; ++i) {
    if (!r[i].lo || r[i].lo % 16 != 0) return fail(LB_INVALID_ARGUMENT, "%s: %s must be non-NULL with 16-byte alignment", what, r[i].name);
    if (r[i].hi < r[i].lo) return fail(LB_INVALID_ARGUMENT, "%s: %s does not fit the address space", what, r[i].name);
    for (int k = 0; k < i; ++k)
      if (overlaps(r[i], r[k])) return fail(LB_INVALID_ARGUMENT, "%s: %s overlaps %s", what, r[k].name, r[i].name);
  }
  return LB_OK;
}

// fp16 rows [batch, seq, heads] of dim values; written ones may not share memory with one another.
lb_status check_rows(const char *what, const char *name, const lb_kv_rows &v, int64_t batch, int64_t seq, int64_t heads, int64_t dim,
                     bool written, Range &range) {
  if (!v.data || !aligned(v.data, 16)) return fail(LB_INVALID_ARGUMENT, "%s: %s must be non-NULL with 16-byte alignment", what, name);
  struct Axis { int64_t size, stride; } axes[3] = {{batch, v.batch_stride}, {seq, v.row_stride}, {heads, v.head_stride}};
  unsigned __int128 span = dim;
  for (Axis &a : axes) {
    if (a.size == 1) a.stride = 0;
    if (a.stride < 0 || a.stride > kMaxStride || a.stride % 8 != 0)
      return fail(LB_INVALID_ARGUMENT, "%s: strides of %s must be multiples of 8, 0 to 2^40 elements", what, name);
    span += (unsigned __int128)(a.size - 1) * a.stride;   // (up to 2^28 * 2^40 each)
  }
  if (span > kMaxBytes / 2) return fail(LB_INVALID_ARGUMENT, "%s: %s is past the address space", what, name);
  if (written) {
    std::sort(axes, axes + 3, [](const Axis &a, const Axis &b) { return a.stride < b.stride; });
    int64_t extent = dim;
    for (const Axis &a : axes) {
      if (a.size == 1) continue;
      if (a.stride < extent) return fail(LB_INVALID_ARGUMENT, "%s: rows of %s overlap one another", what, name);
      extent += (a.size - 1) * a.stride;
    }
  }
  range = range_of(v.data, (size_t)span * 2, name);
  return range.hi < range.lo ? fail(LB_INVALID_ARGUMENT, "%s: %s does not fit the address space", what, name) : LB_OK;
}

lb_status check_counts(const char *what, const char *name, const int64_t *p, int64_t batch, bool needed, Range &range) {
  if (!p && !needed) {
    range = Range{};
    return LB_OK;
  }
  if (!p || !aligned(p, 8)) return fail(LB_INVALID_ARGUMENT, "%s: %s must be a non-NULL device array of 64-bit integers", what, name);
  range = range_of(p, (size_t)batch * 8, name);
  return LB_OK;
}

lb_status check_tables(const char *what, const void *cos, const void *sin, const lb_kv_cache &c, Range (&r)[2]) {
  r[0] = r[1] = Range{};
  if (!cos && !sin) return LB_OK;
  if (!cos || !sin || !aligned(cos, 16) || !aligned(sin, 16))
    return fail(LB_INVALID_ARGUMENT, "%s: cos and sin go together, with 16-byte alignment", what);
  r[0] = range_of(cos, (size_t)c.capacity * c.head_dim * 2, "cos");
  r[1] = range_of(sin, (size_t)c.capacity * c.head_dim * 2, "sin");
  return LB_OK;
}

lb_status check_apart(const char *what, const Range *written, int nw, const Range *read, int nr) {
  for (int i = 0; i < nw; ++i)
    for (int k = 0; k < nr; ++k)
      if (overlaps(written[i], read[k])) return fail(LB_INVALID_ARGUMENT, "%s: %s overlaps %s", what, written[i].name, read[k].name);
  return LB_OK;
}

// Calls f with the kernels' format and head size as constants.
template <class F>
void with_kind(const lb_kv_cache &c, F &&f) {
  if (c.format == LB_KV_INT8) {
    c.head_dim == 64 ? f(std::integral_constant<int, KV_INT8>{}, std::integral_constant<int, 64>{})
                     : f(std::integral_constant<int, KV_INT8>{}, std::integral_constant<int, 128>{});
  } else {
    c.head_dim == 64 ? f(std::integral_constant<int, KV_FP8>{}, std::integral_constant<int, 64>{})
                     : f(std::integral_constant<int, KV_FP8>{}, std::integral_constant<int, 128>{});
  }
}

lb_status check_append(const char *what, const lb_kv_cache &c, int64_t seq, const lb_kv_rows &k, const lb_kv_rows &v,
                       const int64_t *position, const int64_t *rows, const void *cos, const void *sin, Range (&cache)[6], Range (&ins)[6]) {
  if (const lb_status st = check_cache(what, c, cache); st != LB_OK) return st;
  if (seq < 1 || seq > kMaxRows) return fail(LB_INVALID_ARGUMENT, "%s: seq 1 to 2^28 required", what);
  Range tables[2];
  if (const lb_status st = check_rows(what, "k", k, c.batch, seq, c.kv_heads, c.head_dim, false, ins[0]); st != LB_OK) return st;
  if (const lb_status st = check_rows(what, "v", v, c.batch, seq, c.kv_heads, c.head_dim, false, ins[1]); st != LB_OK) return st;
  if (const lb_status st = check_counts(what, "position", position, c.batch, true, ins[2]); st != LB_OK) return st;
  if (const lb_status st = check_counts(what, "rows", rows, c.batch, false, ins[3]); st != LB_OK) return st;
  if (const lb_status st = check_tables(what, cos, sin, c, tables); st != LB_OK) return st;
  ins[4] = tables[0];
  ins[5] = tables[1];
  return check_apart(what, cache, 6, ins, 6);
}

void launch_append(const lb_kv_cache &c, int64_t seq, const lb_kv_rows &k, const lb_kv_rows &v, const int64_t *position,
                   const int64_t *rows, const void *cos, const void *sin, hipStream_t s) {
  KvAppendParams p{};
  p.c = cache_params(c);
  p.k = rows_params(k);
  p.v = rows_params(v);
  p.position = position;
  p.rows = rows;
  p.cos = static_cast<const f16 *>(cos);
  p.sin = static_cast<const f16 *>(sin);
  p.seq = (int)seq;
  // Blocks that seq consecutive slots can fall into, wherever the first lies.
  const int64_t blocks = std::min((seq + 2 * kKvBlock - 2) / kKvBlock, c.capacity / kKvBlock);
  with_kind(c, [&](auto fmt, auto dim) {
    hipLaunchKernelGGL((kv_append_kernel<fmt(), dim()>), dim3((unsigned)blocks, (unsigned)c.kv_heads, (unsigned)c.batch), dim3(2 * dim()), 0, s, p);
  });
}

// Which kernel, its grid and its workspace: LB_ZEROED_WORKSPACE_BYTES of tickets, then the sums of parts.
struct AttendPlan {
  bool prompt;
  int qt, tiles, splits;
  int64_t grid;
  size_t bytes;
};
static_assert(kKvTickets * 4 == LB_ZEROED_WORKSPACE_BYTES, "tickets are the workspace's zeroed bytes");

constexpr int kCus = 256, kKvAlone = 6;   // the CUs; parts of a tile from which they are held to one a CU

AttendPlan attend_plan(const lb_kv_attention_args *a) {
  AttendPlan plan{};
  const lb_kv_cache &c = a->cache;
  const int64_t rows = a->seq * (a->heads / c.kv_heads), pairs = c.batch * c.kv_heads;
  plan.prompt = rows > 32;
  plan.qt = rows > 16 ? 2 : 1;
  plan.tiles = plan.splits = 1;
  size_t parts, height = 16 * plan.qt;   // parts of `height` rows that are left in the workspace at the most
  if (plan.prompt) {
    height = 128;
    plan.tiles = (int)((rows + 127) / 128);
    // Parts only where there are not tiles enough for the workgroups that fit on the CUs, of kKvChunk blocks at the least
    // (4096 rows, 9 and 3 heads of 64: 52 us for three a CU, 74 for two; 509 rows over 32768 slots, 32 and 8 heads of 128,
    // of which two fit: 327 us, 350 for three).  Where one a CU makes kKvAlone parts of a tile there are no more: a part
    // costs the workgroup that adds them as much as a block or two, and CUs that have two set the pace (64 rows over 30000
    // slots, 32 and 8 heads of 128: 16 parts 82 us, 18 to 21 parts 111, 32 parts 122; 4 x 100 rows over 8000, 9 and 3 heads
    // of 64: 7 parts 33 us, 21 parts 46; but 256 rows over 30000: 4 parts 208 us, 8 parts 182).
    const int64_t units = pairs * plan.tiles, fit = (c.head_dim == 64 ? 3 : 2) * kCus, alone = kCus / units;
    plan.splits = (int)std::max<int64_t>(1, std::min<int64_t>(alone >= kKvAlone ? alone : fit / units, (c.capacity / kKvBlock + kKvChunk - 1) / kKvChunk));
    plan.grid = units * plan.splits;     // (at most 3 * kCus where there are parts: the tickets are enough)
    parts = plan.splits > 1 ? (size_t)plan.grid : 0;
  } else {
    // A workgroup per sequence and KV head, and where they can be long enough as many again as they can be split into.
    const bool split = c.capacity / kKvBlock > kKvLeast;
    plan.grid = pairs + (split ? (kKvSplit + c.kv_heads - 1) / c.kv_heads * c.kv_heads : 0);
    parts = split ? kKvPlaces : 0;
  }
  plan.bytes = parts ? LB_ZEROED_WORKSPACE_BYTES + parts * height * (c.head_dim + 2) * sizeof(float) : 0;
  return plan;
}

lb_status check_shape(const char *what, const lb_kv_attention_args *a) {
  const lb_kv_cache &c = a->cache;
  if (a->seq < 1 || a->seq > kMaxRows || a->heads < 1 || a->heads > 65535 || a->heads % c.kv_heads != 0 ||
      a->seq * (a->heads / c.kv_heads) > kMaxRows)
    return fail(LB_INVALID_ARGUMENT, "%s: heads a multiple of kv_heads up to 65535, and 1 to 2^28 rows of a KV head required", what);
  if (c.batch * c.kv_heads > (1 << 23) || c.batch * c.kv_heads * ((a->seq * (a->heads / c.kv_heads) + 127) / 128) > (1 << 23))   // 2^32 threads a launch
    return fail(LB_UNSUPPORTED, "%s: more than 2^23 tiles of 128 rows of a sequence and KV head", what);
  if (!(a->scale >= 0.0f && a->scale <= kMaxScale)) return fail(LB_INVALID_ARGUMENT, "%s: scale must be 0 to 2^16", what);
  return LB_OK;
}

}  // namespace

extern "C" {

lb_status lb_kv_append(const lb_kv_append_args *a, void *stream) {
  const char *what = "lb_kv_append";
  if (const lb_status bad = refuse_if_failed(what); bad != LB_OK) return bad;
  if (!a) return fail(LB_INVALID_ARGUMENT, "%s: args is NULL", what);
  if (a->struct_size < sizeof *a) return fail(LB_INVALID_ARGUMENT, "%s: struct_size %u < %zu", what, a->struct_size, sizeof *a);
  Range cache[6], ins[6];
  if (const lb_status st = check_append(what, a->cache, a->seq, a->k, a->v, a->position, a->rows, a->cos, a->sin, cache, ins); st != LB_OK)
    return st;
  launch_append(a->cache, a->seq, a->k, a->v, a->position, a->rows, a->cos, a->sin, static_cast<hipStream_t>(stream));
  return launch_status(what);
}

lb_status lb_kv_read(const lb_kv_read_args *a, void *stream) {
  const char *what = "lb_kv_read";
  if (const lb_status bad = refuse_if_failed(what); bad != LB_OK) return bad;
  if (!a) return fail(LB_INVALID_ARGUMENT, "%s: args is NULL", what);
  if (a->struct_size < sizeof *a) return fail(LB_INVALID_ARGUMENT, "%s: struct_size %u < %zu", what, a->struct_size, sizeof *a);
  const lb_kv_cache &c = a->cache;
  Range cache[6], outs[2], length;
  if (const lb_status st = check_cache(what, c, cache); st != LB_OK) return st;
  if (a->start < 0 || a->count < 1 || a->count > c.capacity || a->start > c.capacity - a->count)
    return fail(LB_INVALID_ARGUMENT, "%s: start >= 0, count >= 1 and start + count <= capacity required", what);
  if (const lb_status st = check_counts(what, "length", a->length, c.batch, true, length); st != LB_OK) return st;
  if (const lb_status st = check_rows(what, "keys", a->keys, c.batch, a->count, c.kv_heads, c.head_dim, true, outs[0]); st != LB_OK) return st;
  if (const lb_status st = check_rows(what, "values", a->values, c.batch, a->count, c.kv_heads, c.head_dim, true, outs[1]); st != LB_OK) return st;
  if (const lb_status st = check_apart(what, outs, 2, cache, 6); st != LB_OK) return st;
  if (const lb_status st = check_apart(what, outs, 2, &length, 1); st != LB_OK) return st;
  if (overlaps(outs[0], outs[1])) return fail(LB_INVALID_ARGUMENT, "%s: keys overlaps values", what);
  KvReadParams p{};
  p.c = cache_params(c);
  p.length = a->length;
  p.keys = rows_params(a->keys);
  p.values = rows_params(a->values);
  p.start = (int)a->start;
  p.count = (int)a->count;
  const int64_t blocks = (a->start + a->count - 1) / kKvBlock - a->start / kKvBlock + 1;
  with_kind(c, [&](auto fmt, auto dim) {
    hipLaunchKernelGGL((kv_read_kernel<fmt(), dim()>), dim3((unsigned)blocks, (unsigned)c.kv_heads, (unsigned)c.batch), dim3(2 * dim()), 0,
                       static_cast<hipStream_t>(stream), p);
  });
  return launch_status(what);
}

lb_status lb_kv_attention_workspace_bytes(const lb_kv_attention_args *a, size_t *bytes) {
  const char *what = "lb_kv_attention_workspace_bytes";
  if (!a || !bytes) return fail(LB_INVALID_ARGUMENT, "%s: args and bytes must be non-NULL", what);
  *bytes = 0;
  if (a->struct_size < sizeof *a) return fail(LB_INVALID_ARGUMENT, "%s: struct_size %u < %zu", what, a->struct_size, sizeof *a);
  Range cache[6];
  if (const lb_status st = check_cache(what, a->cache, cache); st != LB_OK) return st;
  if (const lb_status st = check_shape(what, a); st != LB_OK) return st;
  *bytes = attend_plan(a).bytes;
  return ok();
}

lb_status lb_kv_attention(const lb_kv_attention_args *a, void *stream) {
  const char *what = "lb_kv_attention";
  if (const lb_status bad = refuse_if_failed(what); bad != LB_OK) return bad;
  if (!a) return fail(LB_INVALID_ARGUMENT, "%s: args is NULL", what);
  if (a->struct_size < sizeof *a) return fail(LB_INVALID_ARGUMENT, "%s: struct_size %u < %zu", what, a->struct_size, sizeof *a);
  const lb_kv_cache &c = a->cache;
  const bool appends = a->k.data || a->v.data;
  Range cache[6], ins[6], q, out, counts[2], tables[2];
  if (const lb_status st = check_cache(what, c, cache); st != LB_OK) return st;
  if (const lb_status st = check_shape(what, a); st != LB_OK) return st;
  if (appends)
    if (const lb_status st = check_append(what, c, a->seq, a->k, a->v, a->position, a->rows, a->cos, a->sin, cache, ins); st != LB_OK) return st;
  if (const lb_status st = check_rows(what, "q", a->q, c.batch, a->seq, a->heads, c.head_dim, false, q); st != LB_OK) return st;
  if (const lb_status st = check_rows(what, "out", a->out, c.batch, a->seq, a->heads, c.head_dim, true, out); st != LB_OK) return st;
  if (const lb_status st = check_counts(what, "position", a->position, c.batch, true, counts[0]); st != LB_OK) return st;
  if (const lb_status st = check_counts(what, "rows", a->rows, c.batch, false, counts[1]); st != LB_OK) return st;
  if (const lb_status st = check_tables(what, a->cos, a->sin, c, tables); st != LB_OK) return st;
  const AttendPlan plan = attend_plan(a);
  if (plan.bytes && (!a->workspace || !aligned(a->workspace, 256) || a->workspace_bytes < plan.bytes))
    return fail(LB_INVALID_ARGUMENT, "%s: a 256-byte aligned workspace of %zu bytes required (got %zu)", what, plan.bytes, a->workspace_bytes);
  const Range writes[] = {out, plan.bytes ? range_of(a->workspace, plan.bytes, "workspace") : Range{}};
  const Range reads[] = {q, counts[0], counts[1], tables[0], tables[1], appends ? ins[0] : Range{}, appends ? ins[1] : Range{}};
  if (const lb_status st = check_apart(what, writes, 2, reads, 7); st != LB_OK) return st;
  if (const lb_status st = check_apart(what, writes, 2, cache, 6); st != LB_OK) return st;
  if (appends)
    if (const lb_status st = check_apart(what, cache, 6, &q, 1); st != LB_OK) return st;
  if (overlaps(writes[0], writes[1])) return fail(LB_INVALID_ARGUMENT, "%s: out overlaps workspace", what);

  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool fused = appends && a->seq == 1 && !plan.prompt;   // one row a sequence: appended by the attention's launch
  if (appends && !fused) launch_append(c, a->seq, a->k, a->v, a->position, a->rows, a->cos, a->sin, s);
  KvAttendParams p{};
  p.c = cache_params(c);
  p.q = rows_params(a->q);
  p.out = rows_params(a->out);
  if (fused) {
    p.k = rows_params(a->k);
    p.v = rows_params(a->v);
  }
  p.position = a->position;
  p.rows = a->rows;
  p.cos = static_cast<const f16 *>(a->cos);
  p.sin = static_cast<const f16 *>(a->sin);
  p.tickets = static_cast<uint32_t *>(a->workspace);
  p.partial = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + LB_ZEROED_WORKSPACE_BYTES);
  p.batch = (int)c.batch;
  p.seq = (int)a->seq;
  p.group = (int)(a->heads / c.kv_heads);
  p.tiles = plan.tiles;
  p.splits = plan.splits;
  p.scale = a->scale * 1.44269504088896340736f;
  const dim3 grid((unsigned)plan.grid);
  with_kind(c, [&](auto fmt, auto dim) {
    if (plan.prompt) hipLaunchKernelGGL((kv_prompt_kernel<fmt(), dim()>), grid, dim3(256), 0, s, p);
    else if (plan.qt == 1) hipLaunchKernelGGL((kv_attend_kernel<fmt(), dim(), 1>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((kv_attend_kernel<fmt(), dim(), 2>), grid, dim3(256), 0, s, p);
  });
  return launch_status(what);
}

}  // extern "C"
