// lb_adapters: the low-rank adapters of many requests beside a shared projection.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "lb_adapters.h"
#include "serve_check.h"

using namespace lb;
using namespace lb::abi;

namespace {

struct AdaptersPlan {
  bool fused, tile;         // adapters_rows_kernel; adapters_tile_kernel
  int rows, ranks, groups;  // adapters_down_kernel: rows and ranks of a tile / 16, groups of those ranks
  int64_t tiles;
  int slices, shares, shares_up, span, wide_span, stack;   // (wide_span: of adapters_tile_kernel)
  size_t bytes;
};

AdaptersPlan adapters_plan(const lb_adapters_args *a) {
  AdaptersPlan plan{};
  const int64_t tiles16 = (a->M + 15) / 16;
  plan.tiles = (a->M + 63) / 64;
  // What a tile of 64 rows comes to at the most, up to 16 rows of one adapter each.
  const int64_t full = std::min<int64_t>(tiles16, 4), units = std::min<int64_t>({a->M, 64, a->count + full});
  // One launch where every workgroup has little of A to go through, and there are few (fp16, one launch and two: 576x576, rank 64 of 8 rows
  // 7.1, 8.2 us; 576x1536, rank 64 of 2 10.4, 8.3; 4096x4096, rank 8 of 20 rows of 20 adapters 7.5, 8.6, rank 16 of 1 8.1, 8.3;
  // 960x2560, rank 8 of 30 rows of 40 6.4, 8.6, of 96 of 64 11.4, 9.2; 14336x4096, rank 8 of 64 of 64 68, 13).
  plan.span = 256;
  const int64_t all = std::min<int64_t>(a->M, a->count * plan.tiles + tiles16);
  plan.fused = a->M <= 128 && a->rank <= 64 && a->K * a->rank <= 3 << 14 && all * ((a->N + plan.span - 1) / plan.span) <= 320;
  if (plan.fused) {
    plan.shares = (int)units;
    return plan;
  }
  // Tiles of 64 rows and 64 ranks where x is large, so that it is read once (4096x4096 rank 128 of 3000 rows: 16, 32, 64 ranks a
  // workgroup 68.4, 51.7, 47.0 us); sooner where there are more groups of ranks that each read it (64 rows and 16: rank 128, 270 rows of
  // 14336 28.7, 37.8 us, 150 rows 30.5, 23.4; rank 64, 400 rows 23.9, 27.1, 300 rows 22.4, 20.7; rank 32, 2000 rows of 4096 20.2, 23.6,
  // 300 of 14336 17.5, 14.8); elsewhere of 16 rows, and of 16 ranks where those are few, for more workgroups (rank 128
  // of 40 rows 13.2, 14.3, 16.2 us; rank 64 of 827 rows 25.7, 22.9, 24.0).  Parts of K, of 1024 at the least, while there are
  // fewer than 224 workgroups (4096x14336 rank 32 of one row: 4, 8, 14 parts 10.7, 9.8, 9.8 us), but no more than the second launch
  // adds up quickly, four at once: each of its workgroups reads them all (4096x14336, rank 64 of 1500 rows, 8 parts 30.7, 9 37.0;
  // rank 32 of 3000, 4 parts 41.3, 5 54.2; 4096x4096, rank 32 of 5360, 2 parts 37.3, 3 42.4; rank 128 of 30 rows, 4 parts 18.2, 14 22.3).
  plan.rows = a->M * a->K < (a->rank <= 32 ? 7 : a->rank <= 64 ? 5 : 3) << 20 ? 1 : 4;
  const int64_t rank16 = (a->rank + 15) / 16;
  plan.ranks = rank16 <= 1 ? 1 : plan.rows == 1 ? (a->M <= 256 ? 1 : 2) : rank16 <= 2 ? 2 : 4;
  plan.groups = (int)((rank16 + plan.ranks - 1) / plan.ranks);
  const int64_t alone = (plan.rows == 1 ? tiles16 : plan.tiles) * plan.groups;
  plan.slices = (int)std::max<int64_t>(1, std::min<int64_t>({224 / alone, (a->K + 1023) / 1024, plan.rows == 1 ? 512 / a->rank : 16, 16}));
  if (plan.slices > 4) plan.slices -= plan.slices % 4;
  plan.shares = (int)(plan.rows == 1 ? std::min<int64_t>(units, std::max<int64_t>(full, 512 / (plan.tiles * plan.groups * plan.slices)))
                                     : std::max<int64_t>(1, std::min<int64_t>({a->count, 64, 512 / (alone * plan.slices)})));
  plan.tile = a->M >= 256;    // (4096x4096 rank 32: 500 rows 13.5 -> 12.0 us, 763 rows of 14336x4096 24.5 -> 18.7)
  plan.stack = tiles16 >= 4 ? 4 : tiles16 >= 2 ? 2 : 1;
  plan.shares_up = (int)(a->M < 1024 ? (units + plan.stack - 1) / plan.stack : 1);
  plan.span = plan.wide_span = 512;
  while (plan.span > (a->rank > 32 ? 64 : 128) && plan.tiles * plan.shares_up * plan.stack * ((a->N + plan.span - 1) / plan.span) < 2048) plan.span /= 2;
  while (plan.wide_span > 128 && (a->M + 63) / 64 * ((a->N + plan.wide_span - 1) / plan.wide_span) < 512) plan.wide_span /= 2;
  plan.bytes = ((size_t)plan.slices * a->M * a->rank * 4 + 255) / 256 * 256;
  return plan;
}

lb_status check_sizes(const char *what, const lb_adapters_args *a) {
  if (a->type > LB_TYPE_BF16) return fail(LB_INVALID_ARGUMENT, "%s: type must be fp16 or bf16", what);
  if (a->M < 1 || a->M > (1 << 28) || a->N < 1 || a->N > (1 << 28) || a->K < 8 || a->K > (1 << 28) || a->K % 8 != 0)
    return fail(LB_INVALID_ARGUMENT, "%s: M, N and K 1 to 2^28 and K a multiple of 8 required", what);
  if (a->rank < 8 || a->rank > LB_ADAPTERS_MAX_RANK || a->rank % 8 != 0)
    return fail(LB_INVALID_ARGUMENT, "%s: rank must be a multiple of 8 up to %d", what, LB_ADAPTERS_MAX_RANK);
  if (a->count < 1 || a->count > (1 << 24)) return fail(LB_INVALID_ARGUMENT, "%s: 1 to 2^24 adapters required", what);
  const AdaptersPlan plan = adapters_plan(a);
  if ((a->M + 15) / 16 * std::max<int64_t>(plan.slices, (a->N + 63) / 64) > (1 << 23))   // 2^32 threads a launch
    return fail(LB_UNSUPPORTED, "%s: more than 2^23 tiles of outputs", what);
  return LB_OK;
}

lb_status check_matrix(const char *what, const char *name, const void *p, int64_t rows, int64_t columns, int64_t ld, bool pieces, bool written, Range &r) {
  if (rows > 1 && written && ld < columns) return fail(LB_INVALID_ARGUMENT, "%s: rows of %s overlap one another", what, name);
  return check_strided(what, name, lb_rows{const_cast<void *>(p), 0, ld, 0}, 1, rows, 1, columns, 2, pieces, false, r);
}

template <class T>
void launch(const lb_adapters_args *a, const AdaptersPlan &plan, hipStream_t s) {
  AdaptersParams<T> p{};
  p.x = static_cast<const T *>(a->x);
  p.y = static_cast<const T *>(a->y);
  p.out = static_cast<T *>(a->out);
  p.down = static_cast<const T *>(a->down);
  p.up = static_cast<const T *>(a->up);
  p.scales = a->scales;
  p.index = a->index;
  p.z = static_cast<float *>(a->workspace);
  p.ldx = a->ldx;
  p.ldy = a->ldy;
  p.ldo = a->ldo;
  p.M = (int)a->M;
  p.N = (int)a->N;
  p.K = (int)a->K;
  p.rank = (int)a->rank;
  p.count = (int)a->count;
  p.slices = plan.slices;
  p.groups = plan.groups;
  p.span = plan.span;
  p.wide = a->N % 8 == 0 && aligned(a->y, 16) && aligned(a->out, 16) && (a->M == 1 || (a->ldy % 8 == 0 && a->ldo % 8 == 0));
  p.shares = plan.shares;
  p.shares_up = plan.shares_up;
  p.stack = plan.stack;
  typedef std::integral_constant<int, 1> One;
  typedef std::integral_constant<int, 2> Two;
  typedef std::integral_constant<int, 4> Four;
  if (plan.fused) {
    const dim3 grid((unsigned)(plan.tiles * ((a->N + plan.span - 1) / plan.span)), (unsigned)plan.shares + 1);
    auto go = [&](auto rt) { hipLaunchKernelGGL((adapters_rows_kernel<T, decltype(rt)::value>), grid, dim3(64 * kRowsWaves), 0, s, p); };
    a->rank <= 16 ? go(One{}) : a->rank <= 32 ? go(Two{}) : go(Four{});
    return;
  }
  const int64_t wide = plan.span * (4 / plan.stack);   // outputs of a workgroup of adapters_up_kernel
  const dim3 down((unsigned)(plan.tiles * plan.slices * plan.groups), (unsigned)plan.shares);
  const dim3 up((unsigned)(plan.tiles * ((a->N + wide - 1) / wide)), (unsigned)plan.shares_up + 1);
  const dim3 tile((unsigned)((a->M + 63) / 64 * ((a->N + plan.wide_span - 1) / plan.wide_span)));
  auto first = [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
    if constexpr (RT <= 2)
      if (plan.rows == 1) {
        hipLaunchKernelGGL((adapters_down_kernel<T, RT, 1>), down, dim3(512), 0, s, p);
        return;
      }
    hipLaunchKernelGGL((adapters_down_kernel<T, RT, 4>), down, dim3(512), 0, s, p);
  };
  plan.ranks == 1 ? first(One{}) : plan.ranks == 2 ? first(Two{}) : first(Four{});
  auto second = [&](auto rc) {
    constexpr int RC = decltype(rc)::value;
    if (plan.tile && p.wide) {
      p.span = plan.wide_span;
      hipLaunchKernelGGL((adapters_tile_kernel<T, RC>), tile, dim3(256), 0, s, p);
    } else {
      hipLaunchKernelGGL((adapters_up_kernel<T, RC>), up, dim3(256), 0, s, p);
    }
  };
  a->rank <= 32 ? second(One{}) : a->rank <= 64 ? second(Two{}) : second(Four{});
}

}  // namespace

extern "C" {

lb_status lb_adapters_workspace_bytes(const lb_adapters_args *a, size_t *bytes) {
  const char *what = "lb_adapters_workspace_bytes";
  if (!a || !bytes) return fail(LB_INVALID_ARGUMENT, "%s: args and bytes must be non-NULL", what);
  *bytes = 0;
  if (a->struct_size < sizeof *a) return fail(LB_INVALID_ARGUMENT, "%s: struct_size %u < %zu", what, a->struct_size, sizeof *a);
  if (const lb_status st = check_sizes(what, a); st != LB_OK) return st;
  *bytes = adapters_plan(a).bytes;
  return ok();
}

lb_status lb_adapters(const lb_adapters_args *a, void *stream) {
  const char *what = "lb_adapters";
  if (const lb_status bad = refuse_if_failed(what); bad != LB_OK) return bad;
  if (!a) return fail(LB_INVALID_ARGUMENT, "%s: args is NULL", what);
  if (a->struct_size < sizeof *a) return fail(LB_INVALID_ARGUMENT, "%s: struct_size %u < %zu", what, a->struct_size, sizeof *a);
  if (const lb_status st = check_sizes(what, a); st != LB_OK) return st;
  Range reads[6], writes[2];
  const size_t factor = (size_t)a->count * a->rank * 2;   // (below 2^32; K and N below 2^28)
  if (const lb_status st = check_matrix(what, "x", a->x, a->M, a->K, a->ldx, true, false, reads[0]); st != LB_OK) return st;
  if (const lb_status st = check_array(what, "down", a->down, factor * a->K, 16, true, reads[1]); st != LB_OK) return st;
  if (const lb_status st = check_array(what, "up", a->up, factor * a->N, 16, true, reads[2]); st != LB_OK) return st;
  if (const lb_status st = check_array(what, "scales", a->scales, (size_t)a->count * 4, 4, false, reads[3]); st != LB_OK) return st;
  if (const lb_status st = check_array(what, "index", a->index, (size_t)a->M * 8, 8, true, reads[4]); st != LB_OK) return st;
  if (const lb_status st = check_matrix(what, "y", a->y, a->M, a->N, a->ldy, false, false, reads[5]); st != LB_OK) return st;
  if (const lb_status st = check_matrix(what, "out", a->out, a->M, a->N, a->ldo, false, true, writes[0]); st != LB_OK) return st;
  const AdaptersPlan plan = adapters_plan(a);
  if (plan.bytes && (!a->workspace || !aligned(a->workspace, 256) || a->workspace_bytes < plan.bytes))
    return fail(LB_INVALID_ARGUMENT, "%s: a 256-byte aligned workspace of %zu bytes required (got %zu)", what, plan.bytes, a->workspace_bytes);
  if (plan.bytes) writes[1] = range_of(a->workspace, plan.bytes, "workspace");
  const bool in_place = a->out == a->y && (a->M == 1 || a->ldo == a->ldy);
  if (const lb_status st = check_apart(what, writes, 2, reads, 5); st != LB_OK) return st;
  if (const lb_status st = check_apart(what, in_place ? writes + 1 : writes, in_place ? 1 : 2, reads + 5, 1); st != LB_OK) return st;
  hipStream_t s = static_cast<hipStream_t>(stream);
  a->type == LB_TYPE_FP16 ? launch<f16>(a, plan, s) : launch<bf16>(a, plan, s);
  return launch_status(what);
}

}  // extern "C"
