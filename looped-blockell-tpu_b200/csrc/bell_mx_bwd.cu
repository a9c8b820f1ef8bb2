// bell_mx_bwd.cu — the straight-through backward of the MXFP4 linear and gated
// feed-forward: the bf16 backward at the quantised operands Q(x), Q(W), Q(h),
// whose values are exact in bf16.  Each entry point is the sequence of launches
// on the caller's stream and one workspace:
//
//   unpack    the gathered tiles of W_down^T and [W_gate ; W_up]^T, and Q(x):
//             one launch
//   d_h = dy Q(W_down), fp32
//   [d_gate | d_up] from d_h and the projections, computed again (bell_mx.cu)
//   dx = [d_gate | d_up] Q([W_gate ; W_up]) (+ dy)
//   the three tile gradients, summed in fp32; one launch completes the sums
//   that CTAs shared, in a fixed order, and rounds them to bf16
//
// d_h stays in fp32: rounded to bf16, its error and that of d_gate and d_up
// together made the tile gradients' 1.7 times that of one rounding.  The
// unpacked operands live in the workspace only during the call; Q(h) takes the
// place of d_h once that has been read.
#include <algorithm>
#include <initializer_list>
#include <string>

#include "bell_mx.cuh"

namespace bell {
namespace mx {

static size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

// Offsets of the workspace: the unpacked transposes (of down, and of gate and
// up or the one weight), a plan, the unpacked rows, d_h then Q(h), fp32 sums
// whose result is bf16, the parts of sums that CTAs share, [d_gate | d_up], and
// the sums of dx where it takes several passes.
struct BwdWs {
  size_t tiles_down, tiles, plan, rows, mid, grads[3], parts[3], dgu, dx[2], total;
};

struct Layout {
  size_t at = 0;
  size_t take(size_t n) {
    const size_t from = at;
    at += up256(n);
    return from;
  }
};

static size_t sums_bytes(const BellMxEll& w, bool wanted, int32_t dtype) {
  return wanted && dtype == BELL_DTYPE_BF16 ? size_t(w.R) * w.K * w.B * w.B * 4 : 0;
}

// Which transposed topologies a call needs: down's for d_gate and d_up, that of
// gate and up for dx.
static bool needs_down_t(const BellMxFFNBwdDesc& d) { return d.dx || d.d_gate || d.d_up || !d.d_down; }
static bool needs_gate_up_t(const BellMxFFNBwdDesc& d) { return d.dx || !(d.d_gate || d.d_up || d.d_down); }

static int32_t passes_of(const BellMxFFNBwdDesc& d) { return d.gate_up_passes ? d.gate_up_passes : 1; }

static size_t parts_bytes(const BellMxEll& w, bool wanted, int64_t T) {
  return wanted ? sddmm_parts_bytes(T, w.R, w.C, w.K, w.B) : 0;
}

static BwdWs linear_ws(const BellMxLinearBwdDesc& d) {
  BwdWs o{};
  Layout l;
  o.tiles = l.take(d.dx ? size_t(d.w.C) * d.K_t * d.w.B * d.w.B * 2 : 0);
  o.plan = l.take(d.dx ? bell_plan_bytes(0, 0, 0, d.w.C, d.K_t) : 0);
  o.rows = l.take(d.dw ? size_t(d.T) * d.w.C * d.w.B * 2 : 0);
  o.grads[0] = l.take(sums_bytes(d.w, d.dw != nullptr, d.grad_dtype));
  o.parts[0] = l.take(parts_bytes(d.w, d.dw != nullptr, d.T));
  o.total = std::max<size_t>(l.at, 256);
  return o;
}

static BwdWs swiglu_ws(const BellMxFFNBwdDesc& d) {
  const BellMxEll& g = d.gate;
  const size_t BB = size_t(g.B) * g.B, F = size_t(g.R) * g.B, T = size_t(d.T);
  BwdWs o{};
  Layout l;
  const int32_t kd = needs_down_t(d) ? d.K_t_down : 0, kg = needs_gate_up_t(d) ? d.K_t_gate_up : 0;
  o.tiles_down = l.take(size_t(g.R) * kd * BB * 2);
  o.tiles = l.take(size_t(g.C) * kg * passes_of(d) * BB * 2);
  o.plan = l.take(std::max(bell_plan_bytes(0, 0, 0, g.R, kd), bell_plan_bytes(0, 0, 0, g.C, kg)));
  o.rows = l.take(T * g.C * g.B * 2);
  o.mid = l.take(T * F * 4);
  o.grads[0] = l.take(sums_bytes(d.gate, d.d_gate != nullptr, d.gate_dtype));
  o.grads[1] = l.take(sums_bytes(d.up, d.d_up != nullptr, d.up_dtype));
  o.grads[2] = l.take(sums_bytes(d.down, d.d_down != nullptr, d.down_dtype));
  o.parts[0] = l.take(parts_bytes(d.gate, d.d_gate != nullptr, d.T));
  o.parts[1] = l.take(parts_bytes(d.up, d.d_up != nullptr, d.T));
  o.parts[2] = l.take(parts_bytes(d.down, d.d_down != nullptr, d.T));
  o.dgu = l.take(T * 2 * F * 2);
  if (d.dx && passes_of(d) > 1) {
    o.dx[0] = l.take(d.dx_dtype == BELL_DTYPE_F32 ? 0 : T * g.C * g.B * 4);
    o.dx[1] = l.take(T * g.C * g.B * 4);
  }
  o.total = l.at;
  return o;
}

// One tile gradient's place: its fp32 sums (the result itself, or workspace),
// the parts of those that CTAs share, and its bf16 result.
static TileGrad grad_of(int64_t T, const BellMxEll& w, const int32_t* cols, void* out, int32_t dtype, char* ws,
                        size_t sums, size_t parts) {
  TileGrad g{};
  if (!out) return g;
  const bool half = dtype == BELL_DTYPE_BF16;
  g.sums = half ? reinterpret_cast<float*>(ws + sums) : static_cast<float*>(out);
  g.rounded = half ? out : nullptr;
  g.cols = cols;
  g.R = w.R, g.C = T > 0 ? w.C : 0, g.K = w.K, g.B = w.B;
  int sms = 0;
  if (!parts_bytes(w, true, T) || device_sm_count(&sms)) return g;
  g.parts = reinterpret_cast<float*>(ws + parts);
  g.cuts = sddmm_cuts(T, w.R, w.C, w.K, w.B, std::min(sms, kMaxParts), true);
  return g;
}

static int tile_grad(int64_t T, const void* a, const void* b, int64_t ldb, const int32_t* cols, const BellMxEll& w,
                     int32_t layout, const TileGrad& g, int32_t* status, void* stream) {
  if (!g.sums || T == 0) return BELL_OK;
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
  s.grad = g.sums;
  s.status = status;
  return sddmm_bf16(&s, true, const_cast<float*>(g.parts), stream);
}

static int product(int64_t T, const void* x, const BellEll& w, const void* residual, void* out, int32_t out_dtype,
                   void* plan, int32_t* status, void* stream) {
  BellLinearDesc d{};
  d.T = T;
  d.dtype = BELL_DTYPE_BF16;
  d.out_dtype = out_dtype;
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
  if (w.R < 1 || w.C < 1 || w.K < 1 || w.R > (1 << 23) || w.C > 65535 || w.K > 65535)
    return fail(BELL_ERR_SHAPE, std::string(name) + ": R, C, K must be >= 1, R <= 2^23 and C, K <= 65535");
  return BELL_OK;
}

// the bf16 products' rows have at most 254 slots
static int check_k_t(int32_t k_t, const char* name) {
  if (k_t > 254)
    return fail(BELL_ERR_SHAPE, std::string(name) + ": a column block is used by " + std::to_string(k_t) +
                                    " block-rows; the backward takes at most 254");
  return BELL_OK;
}

// The kernels' widest accesses: 32 bytes in the gated backward's workspace, 16 in
// rows, chunks and results, and each index's own size.
static bool aligned_to(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
static int check_aligned(std::initializer_list<const void*> by16, std::initializer_list<const void*> by8,
                         std::initializer_list<const void*> by4, const void* workspace, uintptr_t n) {
  if (!workspace || !aligned_to(workspace, n))
    return fail(BELL_ERR_ALIGN, "workspace must be non-NULL and aligned to " + std::to_string(n) + " bytes");
  for (const void* p : by16)
    if (!aligned16(p)) return fail(BELL_ERR_ALIGN, "rows, chunks, plans and results must be 16-byte aligned");
  for (const void* p : by8)
    if (!aligned_to(p, 8)) return fail(BELL_ERR_ALIGN, "index_t must be 8-byte aligned");
  for (const void* p : by4)
    if (!aligned_to(p, 4)) return fail(BELL_ERR_ALIGN, "column indices must be 4-byte aligned");
  return BELL_OK;
}

static int check_layout(int32_t layout) {
  return layout == BELL_TILE_IN_OUT || layout == BELL_TILE_OUT_IN ? BELL_OK : fail(BELL_ERR_ARG, "unknown tile layout");
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
  if (d->dx)
    if (int rc = mx::check_k_t(d->K_t, "weight")) return rc;
  if (d->dx && !mx::grad_type(d->dx_dtype)) return fail(BELL_ERR_DTYPE, "dx_dtype must be bf16 or f32");
  if (d->dw && (!d->col_indices || !mx::grad_type(d->grad_dtype)))
    return fail(BELL_ERR_ARG, "dw needs col_indices and a bf16 or f32 grad_dtype");
  if (int rc = mx::check_layout(d->layout)) return rc;
  if (int rc = mx::check_aligned({d->grad_out, d->x, w.chunks, d->dx, d->dw}, {d->index_t}, {d->col_indices, d->cols_t},
                                 d->workspace, 16))
    return rc;
  if (int rc = require_sm100()) return rc;
  char* ws = static_cast<char*>(d->workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const mx::BwdWs o = mx::linear_ws(*d);
  const bool want_dx = d->dx && d->T > 0;
  const int32_t in_f = w.C * w.B;
  const mx::FinishArgs grads{{mx::grad_of(d->T, w, d->col_indices, d->dw, d->grad_dtype, ws, o.grads[0], o.parts[0]), {}, {}}};
  mx::ExpandArgs e{};
  e.T = d->T;
  e.B = w.B;
  if (want_dx)
    e.gather[0] = {w.chunks, int64_t(w.R) * w.K, nullptr, 0, d->index_t, int64_t(w.C) * d->K_t, ws + o.tiles};
  if (d->dw && d->T > 0) e.rows[0] = {d->x, in_f, ws + o.rows};
  if (int rc = mx::expand(e, s)) return rc;
  if (want_dx) {
    const BellEll wt{ws + o.tiles, d->cols_t, w.C, w.R, d->K_t, w.B, BELL_TILE_IN_OUT, 0};
    if (int rc = mx::product(d->T, d->grad_out, wt, nullptr, d->dx, d->dx_dtype, ws + o.plan, d->status, stream)) return rc;
  }
  if (int rc = mx::tile_grad(d->T, ws + o.rows, d->grad_out, int64_t(w.R) * w.B, d->col_indices, w, d->layout, grads.g[0],
                             d->status, stream))
    return rc;
  return mx::finish_grads(grads, s);
}

size_t bell_swiglu_bwd_mx_workspace_bytes(const BellMxFFNBwdDesc* d) {
  if (!d || mx::check_weight(d->gate, "gate") || mx::check_weight(d->up, "up") || mx::check_weight(d->down, "down") ||
      d->T < 0 || d->gate_up_passes < 0 || (mx::needs_down_t(*d) && d->K_t_down < 1) || (mx::needs_gate_up_t(*d) && d->K_t_gate_up < 1))
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
  if (d->T > 0 && (!d->grad_out || !d->x || !d->h)) return fail(BELL_ERR_ARG, "grad_out, x and h must be non-NULL");
  if (!g.plan || !u.plan) return fail(BELL_ERR_ARG, "gate and up need their plans");
  if ((mx::needs_down_t(*d) && (!d->cols_t_down || !d->index_t_down || d->K_t_down < 1)) ||
      (mx::needs_gate_up_t(*d) && (!d->cols_t_gate_up || !d->index_t_gate_up || d->K_t_gate_up < 1)))
    return fail(BELL_ERR_ARG, "the transposed topologies must be given");
  if (d->dx || d->d_gate || d->d_up)
    if (int rc = mx::check_k_t(d->K_t_down, "down")) return rc;
  if (d->dx)
    if (int rc = mx::check_k_t(d->K_t_gate_up, "gate and up")) return rc;
  if (d->gate_up_passes < 0) return fail(BELL_ERR_SHAPE, "gate_up_passes must be >= 0");
  if (d->dx && !mx::grad_type(d->dx_dtype)) return fail(BELL_ERR_DTYPE, "dx_dtype must be bf16 or f32");
  if ((d->d_gate && (!d->cols_gate || !mx::grad_type(d->gate_dtype))) ||
      (d->d_up && (!d->cols_up || !mx::grad_type(d->up_dtype))) ||
      (d->d_down && (!d->cols_down || !mx::grad_type(d->down_dtype))))
    return fail(BELL_ERR_ARG, "a tile gradient needs its col_indices and a bf16 or f32 type");
  if (int rc = mx::check_layout(d->layout)) return rc;
  if (int rc = mx::check_aligned({d->grad_out, d->x, d->h, g.chunks, u.chunks, w.chunks, g.plan, u.plan, d->dx, d->d_gate,
                                  d->d_up, d->d_down},
                                 {d->index_t_down, d->index_t_gate_up},
                                 {d->cols_gate, d->cols_up, d->cols_down, d->cols_t_down, d->cols_t_gate_up},
                                 d->workspace, 32))
    return rc;
  if (int rc = require_sm100()) return rc;
  char* ws = static_cast<char*>(d->workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const mx::BwdWs o = mx::swiglu_ws(*d);
  const int32_t F = g.R * g.B, D = g.C * g.B;
  const int64_t T = d->T;
  const bool want_dgu = T > 0 && (d->dx || d->d_gate || d->d_up), want_dx = T > 0 && d->dx;
  char *dgu = ws + o.dgu, *mid = ws + o.mid;
  const mx::FinishArgs grads{{mx::grad_of(T, g, d->cols_gate, d->d_gate, d->gate_dtype, ws, o.grads[0], o.parts[0]),
                              mx::grad_of(T, u, d->cols_up, d->d_up, d->up_dtype, ws, o.grads[1], o.parts[1]),
                              mx::grad_of(T, w, d->cols_down, d->d_down, d->down_dtype, ws, o.grads[2], o.parts[2])}};
  mx::ExpandArgs e{};
  e.T = T;
  e.B = g.B;
  if (want_dgu)
    e.gather[0] = {w.chunks, int64_t(w.R) * w.K, nullptr, 0, d->index_t_down, int64_t(g.R) * d->K_t_down,
                   ws + o.tiles_down};
  if (want_dx)
    e.gather[1] = {g.chunks, int64_t(g.R) * g.K, u.chunks, int64_t(u.R) * u.K, d->index_t_gate_up,
                   int64_t(g.C) * d->K_t_gate_up * mx::passes_of(*d), ws + o.tiles};
  if (T > 0 && (d->d_gate || d->d_up)) e.rows[0] = {d->x, D, ws + o.rows};
  if (int rc = mx::expand(e, s)) return rc;
  if (want_dgu) {
    const BellEll wt{ws + o.tiles_down, d->cols_t_down, g.R, w.R, d->K_t_down, g.B, BELL_TILE_IN_OUT, 0};
    if (int rc = mx::product(T, d->grad_out, wt, nullptr, mid, BELL_DTYPE_F32, ws + o.plan, d->status, stream)) return rc;
    if (int rc = mx::gated_backward(T, d->x, g, u, reinterpret_cast<const float*>(mid), dgu, d->status, s)) return rc;
  }
  const int32_t passes = mx::passes_of(*d);
  for (int32_t p = 0; want_dx && p < passes; ++p) {
    const int64_t tiles = int64_t(g.C) * d->K_t_gate_up;
    const BellEll wt{ws + o.tiles + size_t(p * tiles) * g.B * g.B * 2, d->cols_t_gate_up + p * tiles, g.C, 2 * g.R,
                     d->K_t_gate_up, g.B, BELL_TILE_IN_OUT, 0};
    float* sums = d->dx_dtype == BELL_DTYPE_F32 ? static_cast<float*>(d->dx) : reinterpret_cast<float*>(ws + o.dx[0]);
    float* more = reinterpret_cast<float*>(ws + o.dx[1]);
    const bool whole = passes == 1, last = p == passes - 1;
    if (int rc = mx::product(T, dgu, wt, d->add_residual && p == 0 ? d->grad_out : nullptr, whole ? d->dx : p ? more : sums,
                             whole ? int32_t(d->dx_dtype) : BELL_DTYPE_F32, ws + o.plan, d->status, stream))
      return rc;
    if (p)
      if (int rc = mx::add_sums(sums, more, T * D, last ? d->dx : sums, last ? int32_t(d->dx_dtype) : BELL_DTYPE_F32, s)) return rc;
  }
  if (int rc = mx::tile_grad(T, ws + o.rows, dgu, int64_t(F) * 2, d->cols_gate, g, d->layout, grads.g[0], d->status, stream))
    return rc;
  if (int rc = mx::tile_grad(T, ws + o.rows, dgu + size_t(F) * 2, int64_t(F) * 2, d->cols_up, u, d->layout, grads.g[1],
                             d->status, stream))
    return rc;
  if (T > 0 && d->d_down)
    if (int rc = bell_mx_dequantize_rows(T, F, g.B, d->h, BELL_DTYPE_BF16, mid, F, stream)) return rc;
  if (int rc = mx::tile_grad(T, mid, d->grad_out, D, d->cols_down, w, d->layout, grads.g[2], d->status, stream)) return rc;
  return mx::finish_grads(grads, s);
}

}  // extern "C"
