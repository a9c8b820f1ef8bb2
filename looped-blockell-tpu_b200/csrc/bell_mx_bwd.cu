// bell_mx_bwd.cu — the straight-through backward of the MXFP4 linear and gated
// feed-forward: the bf16 backward at the quantised operands Q(x), Q(W), Q(h),
// whose values are exact in bf16.  Each entry point is the sequence of launches
// on the caller's stream and one workspace:
//
//   W_down^T  gathered and unpacked; [d_gate | d_up] from d_h = dy Q(W_down)
//             and the SiLU backward (one kernel at B = 64, two at B = 128, as
//             the bf16 backward measured faster)
//   [W_gate ; W_up]^T likewise; dx = [d_gate | d_up] Q([W_gate ; W_up]) (+ dy)
//   Q(x), Q(h) unpacked; the three tile gradients, summed in fp32
//
// The unpacked operands live in the workspace only while their product runs:
// they add 2 bytes a value to the traffic and nothing to what training keeps.
#include <algorithm>
#include <string>

#include "bell_mx.cuh"

namespace bell {
namespace mx {

static size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

// Offsets of the workspace.
struct BwdWs {
  size_t tiles, plan, rows, mid, grads, dgu, total;
};

// tiles: the larger of the unpacked transposes; rows: unpacked rows; mid: d_h,
// then Q(h); grads: fp32 sums whose result is bf16; dgu: [d_gate | d_up].
static BwdWs bwd_ws(size_t tiles, size_t plan, size_t rows, size_t mid, size_t grads, size_t dgu) {
  BwdWs w{};
  w.tiles = 0;
  w.plan = up256(tiles);
  w.rows = w.plan + up256(plan);
  w.mid = w.rows + up256(rows);
  w.grads = w.mid + up256(mid);
  w.dgu = w.grads + up256(grads);
  w.total = w.dgu + up256(dgu);
  return w;
}

static BwdWs linear_ws(const BellMxLinearBwdDesc& d) {
  const size_t BB = size_t(d.w.B) * d.w.B;
  return bwd_ws(size_t(d.w.C) * d.K_t * BB * 2, bell_plan_bytes(0, 0, 0, d.w.C, d.K_t),
                size_t(d.T) * d.w.C * d.w.B * 2, 0, d.grad_dtype == BELL_DTYPE_BF16 ? size_t(d.w.R) * d.w.K * BB * 4 : 0, 0);
}

static BwdWs swiglu_ws(const BellMxFFNBwdDesc& d) {
  const BellMxEll &g = d.gate, &u = d.up, &w = d.down;
  const size_t BB = size_t(g.B) * g.B, F = size_t(g.R) * g.B;
  const size_t tiles = std::max(size_t(g.R) * d.K_t_down, size_t(g.C) * d.K_t_gate_up) * BB * 2;
  const size_t plan = std::max(bell_plan_bytes(0, 0, 0, g.R, d.K_t_down), bell_plan_bytes(0, 0, 0, g.C, d.K_t_gate_up));
  size_t most = 0;
  if (d.gate_dtype == BELL_DTYPE_BF16) most = std::max(most, size_t(g.R) * g.K);
  if (d.up_dtype == BELL_DTYPE_BF16) most = std::max(most, size_t(u.R) * u.K);
  if (d.down_dtype == BELL_DTYPE_BF16) most = std::max(most, size_t(w.R) * w.K);
  return bwd_ws(tiles, plan, size_t(d.T) * g.C * g.B * 2, size_t(d.T) * F * 2, most * BB * 4, size_t(d.T) * 2 * F * 2);
}

static int tile_grad(int64_t T, const void* a, const void* b, int64_t ldb, const int32_t* cols, const BellMxEll& w,
                     int32_t layout, void* out, int32_t dtype, void* sums, int32_t* status, void* stream) {
  BellSddmmDesc s{};
  s.T = T;
  s.a = a;
  s.b = b;
  s.lda = int64_t(w.C) * w.B;
  s.ldb = ldb;
  s.col_indices = cols;
  s.R = w.R;
  s.C = w.C;
  s.K = w.K;
  s.B = w.B;
  s.layout = layout;
  s.grad = static_cast<float*>(dtype == BELL_DTYPE_BF16 ? sums : out);
  s.grad_bf16 = dtype == BELL_DTYPE_BF16 ? out : nullptr;
  s.status = status;
  return bell_sddmm_bf16(&s, stream);
}

// Transposed weight in bf16: rows = column blocks of the (stacked) weight.
// Tiles are unpacked [B_out, B_in], which their transpose reads as [B_in, B_out].
static int transposed(const BellMxEll& w0, const BellMxEll* w1, const int32_t* cols_t, const int64_t* index, int32_t K_t,
                      int32_t C_t, void* tiles, BellEll* out, void* stream) {
  *out = BellEll{tiles, cols_t, w0.C, C_t, K_t, w0.B, BELL_TILE_IN_OUT, 0};
  return bell_mx_unpack_tiles(w0.chunks, int64_t(w0.R) * w0.K, w1 ? w1->chunks : nullptr, w1 ? int64_t(w1->R) * w1->K : 0,
                              w0.B, index, int64_t(w0.C) * K_t, tiles, stream);
}

static int product(int64_t T, const void* x, const BellEll& w, const void* residual, void* out, void* plan,
                   int32_t* status, void* stream) {
  BellLinearDesc d{};
  d.T = T;
  d.dtype = d.out_dtype = BELL_DTYPE_BF16;
  d.add_residual = residual != nullptr;
  d.x = x;
  d.residual = residual;
  d.out = out;
  d.plan = plan;
  d.w = w;
  d.status = status;
  return bell_linear_bf16(&d, stream);
}

static int check_weight(const BellMxEll& w, const char* name) {
  if (!w.chunks) return fail(BELL_ERR_ARG, std::string(name) + ": NULL chunks");
  if (w.B != 64 && w.B != 128) return fail(BELL_ERR_SHAPE, std::string(name) + ": tile size B must be 64 or 128");
  if (w.R < 1 || w.C < 1 || w.K < 1) return fail(BELL_ERR_SHAPE, std::string(name) + ": R, C, K must be >= 1");
  return BELL_OK;
}

static bool grad_type(int32_t t) { return t == BELL_DTYPE_BF16 || t == BELL_DTYPE_F32; }

}  // namespace mx
}  // namespace bell

using namespace bell;

extern "C" {

size_t bell_linear_bwd_mx_workspace_bytes(const BellMxLinearBwdDesc* d) {
  return d && !mx::check_weight(d->w, "weight") && d->T >= 0 && d->K_t >= 1 ? mx::linear_ws(*d).total : 0;
}

int bell_linear_bwd_mx(const BellMxLinearBwdDesc* d, void* stream) {
  if (!d) return fail(BELL_ERR_ARG, "descriptor is NULL");
  if (int rc = mx::check_weight(d->w, "weight")) return rc;
  const BellMxEll& w = d->w;
  if (d->T < 0 || d->T > (int64_t(1) << 31) - 256) return fail(BELL_ERR_SHAPE, "T must be in [0, 2^31 - 256)");
  if (d->T > 0 && (!d->grad_out || !d->x)) return fail(BELL_ERR_ARG, "grad_out and x must be non-NULL");
  if (d->dx && (!d->cols_t || !d->index_t || d->K_t < 1)) return fail(BELL_ERR_ARG, "dx needs the transposed topology");
  if (d->dw && (!d->col_indices || !mx::grad_type(d->grad_dtype)))
    return fail(BELL_ERR_ARG, "dw needs col_indices and a bf16 or f32 grad_dtype");
  if (!d->workspace || !aligned16(d->workspace)) return fail(BELL_ERR_ALIGN, "workspace must be non-NULL and aligned");
  if (int rc = require_sm100()) return rc;
  char* ws = static_cast<char*>(d->workspace);
  const mx::BwdWs o = mx::linear_ws(*d);
  if (d->dx && d->T > 0) {
    BellEll wt;
    if (int rc = mx::transposed(w, nullptr, d->cols_t, d->index_t, d->K_t, w.R, ws + o.tiles, &wt, stream)) return rc;
    if (int rc = mx::product(d->T, d->grad_out, wt, nullptr, d->dx, ws + o.plan, d->status, stream)) return rc;
  }
  if (!d->dw) return BELL_OK;
  const int32_t in_f = w.C * w.B;
  if (int rc = bell_mx_dequantize_rows(d->T, in_f, w.B, d->x, BELL_DTYPE_BF16, ws + o.rows, in_f, stream)) return rc;
  return mx::tile_grad(d->T, ws + o.rows, d->grad_out, int64_t(w.R) * w.B, d->col_indices, w, d->layout, d->dw,
                       d->grad_dtype, ws + o.grads, d->status, stream);
}

size_t bell_swiglu_bwd_mx_workspace_bytes(const BellMxFFNBwdDesc* d) {
  if (!d || mx::check_weight(d->gate, "gate") || mx::check_weight(d->up, "up") || mx::check_weight(d->down, "down") ||
      d->T < 0 || d->K_t_down < 1 || d->K_t_gate_up < 1)
    return 0;
  return mx::swiglu_ws(*d).total;
}

int bell_swiglu_bwd_mx(const BellMxFFNBwdDesc* d, void* stream) {
  if (!d) return fail(BELL_ERR_ARG, "descriptor is NULL");
  if (int rc = mx::check_weight(d->gate, "gate")) return rc;
  if (int rc = mx::check_weight(d->up, "up")) return rc;
  if (int rc = mx::check_weight(d->down, "down")) return rc;
  const BellMxEll &g = d->gate, &u = d->up, &w = d->down;
  if (g.R != u.R || g.C != u.C || g.B != u.B || w.B != g.B || w.C != g.R || w.R != g.C)
    return fail(BELL_ERR_SHAPE, "gate, up and down do not fit");
  if (d->T < 0 || d->T > (int64_t(1) << 31) - 256) return fail(BELL_ERR_SHAPE, "T must be in [0, 2^31 - 256)");
  if (d->T > 0 && (!d->grad_out || !d->gate_pre || !d->up_out || !d->x || !d->h))
    return fail(BELL_ERR_ARG, "grad_out, gate_pre, up_out, x and h must be non-NULL");
  if (!d->cols_t_down || !d->index_t_down || d->K_t_down < 1 || !d->cols_t_gate_up || !d->index_t_gate_up ||
      d->K_t_gate_up < 1)
    return fail(BELL_ERR_ARG, "the transposed topologies must be given");
  if ((d->d_gate && (!d->cols_gate || !mx::grad_type(d->gate_dtype))) ||
      (d->d_up && (!d->cols_up || !mx::grad_type(d->up_dtype))) ||
      (d->d_down && (!d->cols_down || !mx::grad_type(d->down_dtype))))
    return fail(BELL_ERR_ARG, "a tile gradient needs its col_indices and a bf16 or f32 type");
  if (!d->workspace || !aligned16(d->workspace)) return fail(BELL_ERR_ALIGN, "workspace must be non-NULL and aligned");
  if (int rc = require_sm100()) return rc;
  char* ws = static_cast<char*>(d->workspace);
  const mx::BwdWs o = mx::swiglu_ws(*d);
  const int32_t F = g.R * g.B, D = g.C * g.B;
  char* dgu = ws + o.dgu;
  BellEll wt;
  if (d->T > 0 && (d->dx || d->d_gate || d->d_up)) {
    if (int rc = mx::transposed(w, nullptr, d->cols_t_down, d->index_t_down, d->K_t_down, w.R, ws + o.tiles, &wt, stream))
      return rc;
    if (g.B == 64) {
      BellDownBwdDesc b{};
      b.T = d->T;
      b.grad_out = d->grad_out;
      b.gate_pre = d->gate_pre;
      b.up_out = d->up_out;
      b.d_gate_up = dgu;
      b.plan = ws + o.plan;
      b.w_t = wt;
      b.status = d->status;
      if (int rc = bell_down_silu_bwd_bf16(&b, stream)) return rc;
    } else {
      if (int rc = mx::product(d->T, d->grad_out, wt, nullptr, ws + o.mid, ws + o.plan, d->status, stream)) return rc;
      if (int rc = bell_silu_mul_bwd_bf16(d->T, F, ws + o.mid, d->gate_pre, d->up_out, dgu, dgu + size_t(F) * 2,
                                          int64_t(F) * 2, stream))
        return rc;
    }
  }
  if (d->T > 0 && d->dx) {
    if (int rc = mx::transposed(g, &u, d->cols_t_gate_up, d->index_t_gate_up, d->K_t_gate_up, 2 * g.R, ws + o.tiles, &wt,
                                stream))
      return rc;
    if (int rc = mx::product(d->T, dgu, wt, d->add_residual ? d->grad_out : nullptr, d->dx, ws + o.plan, d->status, stream))
      return rc;
  }
  if (d->d_gate || d->d_up) {
    if (int rc = bell_mx_dequantize_rows(d->T, D, g.B, d->x, BELL_DTYPE_BF16, ws + o.rows, D, stream)) return rc;
    if (d->d_gate)
      if (int rc = mx::tile_grad(d->T, ws + o.rows, dgu, int64_t(F) * 2, d->cols_gate, g, d->layout, d->d_gate,
                                 d->gate_dtype, ws + o.grads, d->status, stream))
        return rc;
    if (d->d_up)
      if (int rc = mx::tile_grad(d->T, ws + o.rows, dgu + size_t(F) * 2, int64_t(F) * 2, d->cols_up, u, d->layout, d->d_up,
                                 d->up_dtype, ws + o.grads, d->status, stream))
        return rc;
  }
  if (d->d_down) {
    if (int rc = bell_mx_dequantize_rows(d->T, F, g.B, d->h, BELL_DTYPE_BF16, ws + o.mid, F, stream)) return rc;
    if (int rc = mx::tile_grad(d->T, ws + o.mid, d->grad_out, D, d->cols_down, w, d->layout, d->d_down, d->down_dtype,
                               ws + o.grads, d->status, stream))
      return rc;
  }
  return BELL_OK;
}

}  // extern "C"
