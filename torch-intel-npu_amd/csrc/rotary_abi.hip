// lb_rotary: rows of heads turned by their positions.
#include <hip/hip_runtime.h>

#include "lb_rotary.h"
#include "serve_check.h"

using namespace lb;
using namespace lb::abi;

namespace {

// Whether rows may be read and written in pieces of V values.
bool in_pieces(const lb_rows &r, int64_t batch, int64_t seq, int64_t heads, int V, size_t size) {
  return aligned(r.data, V * size) && (batch == 1 || r.batch_stride % V == 0) && (seq == 1 || r.row_stride % V == 0) &&
         (heads == 1 || r.head_stride % V == 0);
}

template <class T, int V>
void launch(const lb_rotary_args *a, bool in_place, hipStream_t s) {
  RotaryParams<T> p{};
  const lb_rows *x[2] = {&a->q, &a->k}, *out[2] = {&a->out, &a->out_k};
  const int64_t heads[2] = {a->heads, a->k_heads};
  for (int i = 0; i < 2; ++i) {
    p.x[i] = strided<const T>(*x[i]);
    p.out[i] = strided<T>(*out[i]);
    p.heads[i] = (int)heads[i];
  }
  p.position = a->position;
  p.turn = turn_params(a->rotation);
  p.batch = (int)a->batch;
  p.seq = (int)a->seq;
  p.dim = (int)a->head_dim;
  p.per_row = a->per_row != 0;
  p.back = a->back != 0;
  p.copies = in_place ? 0 : (int)((a->head_dim - p.turn.dims + 2 * V - 1) / (2 * V));
  const int64_t rows = a->batch * a->seq, pieces = p.turn.dims / (2 * V) + p.copies, all = a->heads + a->k_heads;
  // A row's heads side by side in a wave, as many as it has lanes for, and where a lane would have more than two of them, more waves (8192
  // rows of 40 heads of 128, bf16: 1, 2, 3, 5 waves a row 33.4, 31.7, 30.5, 36.4 us; 2048 rows 10.0, 9.5, 9.4, 10.0).
  const int64_t lanes = std::min<int64_t>(all, std::max<int64_t>(1, 64 / pieces)), turns = (all + lanes - 1) / lanes;
  p.lanes = (int)((all + turns - 1) / turns);
  p.shares = (int)std::min<int64_t>((turns + 1) / 2, std::max<int64_t>(1, (1 << 20) / rows));
  p.rows = (int)std::max<int64_t>(1, std::min<int64_t>(64 / (pieces * p.lanes), rows / 4096));
  // Rows of 48 MB and more are hardly in the caches, and read past them (rows of 40 heads of 128, bf16, in turn over three inputs: 6000
  // rows 27.2 -> 24.2 us, 4500 20.1 either way, 3000 12.2 -> 15.0).
  const bool once = rows * all * a->head_dim * (int64_t)sizeof(T) >= 48 << 20;
  const dim3 grid((unsigned)((rows + 4 * p.rows - 1) / (4 * p.rows) * p.shares)), block(256);
  if (once) hipLaunchKernelGGL((rotary_kernel<T, V, true>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((rotary_kernel<T, V, false>), grid, block, 0, s, p);
}

}  // namespace

extern "C" lb_status lb_rotary(const lb_rotary_args *a, void *stream) {
  const char *what = "lb_rotary";
  if (const lb_status bad = refuse_if_failed(what); bad != LB_OK) return bad;
  if (!a) return fail(LB_INVALID_ARGUMENT, "%s: args is NULL", what);
  if (a->struct_size < sizeof *a) return fail(LB_INVALID_ARGUMENT, "%s: struct_size %u < %zu", what, a->struct_size, sizeof *a);
  if (a->type > LB_TYPE_FP32) return fail(LB_INVALID_ARGUMENT, "%s: unknown type %u", what, a->type);
  if (a->head_dim < 2 || a->head_dim > LB_ROTARY_MAX_DIMS || a->heads < 1 || a->heads > 65535 || a->k_heads < 0 || a->k_heads > 65535)
    return fail(LB_INVALID_ARGUMENT, "%s: head_dim 2 to %d, heads 1 to 65535 and k_heads 0 to 65535 required", what, LB_ROTARY_MAX_DIMS);
  if (a->batch < 1 || a->seq < 1 || a->batch > kMaxSeq || a->seq > kMaxSeq / a->batch)
    return fail(LB_INVALID_ARGUMENT, "%s: 1 to 2^25 rows required", what);
  const size_t size = a->type == LB_TYPE_FP32 ? 4 : 2;
  Range reads[4], writes[2];
  if (const lb_status st = check_strided(what, "q", a->q, a->batch, a->seq, a->heads, a->head_dim, size, false, false, reads[0]); st != LB_OK) return st;
  if (const lb_status st = check_strided(what, "out", a->out, a->batch, a->seq, a->heads, a->head_dim, size, false, true, writes[0]); st != LB_OK) return st;
  if (a->k_heads) {
    if (const lb_status st = check_strided(what, "k", a->k, a->batch, a->seq, a->k_heads, a->head_dim, size, false, false, reads[1]); st != LB_OK) return st;
    if (const lb_status st = check_strided(what, "out_k", a->out_k, a->batch, a->seq, a->k_heads, a->head_dim, size, false, true, writes[1]); st != LB_OK) return st;
  }
  if (const lb_status st = check_array(what, "position", a->position, (size_t)(a->per_row ? a->batch * a->seq : a->batch) * 8, 8, true, reads[2]); st != LB_OK) return st;
  if (const lb_status st = check_rotation(what, a->rotation, a->head_dim, true, reads[3]); st != LB_OK) return st;
  // In place: out is q's rows and out_k k's.  What is written and read may else be slices of one tensor that lie between one another.
  const bool q_same = same_rows(a->q, a->out, a->batch, a->seq, a->heads);
  const bool k_same = !a->k_heads || same_rows(a->k, a->out_k, a->batch, a->seq, a->k_heads);
  const bool in_place = q_same && k_same;
  if (!in_place && q_same != k_same && a->k_heads) return fail(LB_INVALID_ARGUMENT, "%s: q and k are turned in place both or neither", what);
  if (const lb_status st = check_apart(what, writes, 1, reads + 2, 2); st != LB_OK) return st;
  if (const lb_status st = check_apart(what, writes + 1, 1, reads + 2, 2); st != LB_OK) return st;
  auto apart = [&](const lb_rows &x, int64_t x_heads, const lb_rows &y, int64_t y_heads) {
    return rows_apart(x, x_heads, y, y_heads, a->batch, a->seq, a->head_dim, size);
  };
  if (in_place) {
    if (a->k_heads && !apart(a->q, a->heads, a->k, a->k_heads)) return fail(LB_INVALID_ARGUMENT, "%s: rows of q and k overlap", what);
  } else {
    const struct { const char *name; const lb_rows &rows; int64_t heads; } out[2] = {{"out", a->out, a->heads}, {"out_k", a->out_k, a->k_heads}},
                                                                          in[2] = {{"q", a->q, a->heads}, {"k", a->k, a->k_heads}};
    for (int i = 0; i < (a->k_heads ? 2 : 1); ++i)
      for (int j = 0; j < (a->k_heads ? 2 : 1); ++j)
        if (!apart(out[i].rows, out[i].heads, in[j].rows, in[j].heads)) return fail(LB_INVALID_ARGUMENT, "%s: %s overlaps %s", what, out[i].name, in[j].name);
    if (a->k_heads && !apart(a->out, a->heads, a->out_k, a->k_heads)) return fail(LB_INVALID_ARGUMENT, "%s: out_k overlaps out", what);
  }
  auto fits = [&](int V) {
    return a->rotation.dims % (2 * V) == 0 && a->head_dim % V == 0 && in_pieces(a->q, a->batch, a->seq, a->heads, V, size) &&
           in_pieces(a->out, a->batch, a->seq, a->heads, V, size) &&
           (!a->k_heads || (in_pieces(a->k, a->batch, a->seq, a->k_heads, V, size) && in_pieces(a->out_k, a->batch, a->seq, a->k_heads, V, size)));
  };
  const int V = size == 2 && fits(8) ? 8 : fits(4) ? 4 : 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->type == LB_TYPE_FP32) {
    V == 4 ? launch<float, 4>(a, in_place, s) : launch<float, 1>(a, in_place, s);
  } else if (a->type == LB_TYPE_FP16) {
    V == 8 ? launch<f16, 8>(a, in_place, s) : V == 4 ? launch<f16, 4>(a, in_place, s) : launch<f16, 1>(a, in_place, s);
  } else {
    V == 8 ? launch<bf16, 8>(a, in_place, s) : V == 4 ? launch<bf16, 4>(a, in_place, s) : launch<bf16, 1>(a, in_place, s);
  }
  return launch_status(what);
}
