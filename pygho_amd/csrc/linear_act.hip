// Entry points of the linear operators: argument checks, which form runs (linear_stream.h, linear_tile.h), the launches of a backward pass.
#include "linear_ops.h"

namespace pygho {

#define PYGHO_LINEAR_DECL(T)                                                                  \
  template <> int LinearOps<T>::stream_lds(int64_t, int64_t, int, bool, bool);                \
  template <> int LinearOps<T>::out_lds(int64_t, int64_t);                                    \
  template <> bool LinearOps<T>::dw_fits(int64_t, int64_t, int);                              \
  template <> int LinearOps<T>::stream_fwd(const LsArgs&, int, hipStream_t);                  \
  template <> int LinearOps<T>::out_fwd(const LsArgs&, hipStream_t);                          \
  template <> int LinearOps<T>::stream_bwd(const LsArgs&, int, bool, int*, hipStream_t);      \
  template <> int LinearOps<T>::tile_act(const LaArgs&, hipStream_t);                         \
  template <> int LinearOps<T>::transpose(void*, const void*, int64_t, int64_t, int64_t, hipStream_t); \
  template <> int LinearOps<T>::tile_dw(const LaArgs&, hipStream_t);
PYGHO_LINEAR_DECL(float)
PYGHO_LINEAR_DECL(bf16)
PYGHO_LINEAR_DECL(f16)
#undef PYGHO_LINEAR_DECL

// f(LinearOps<T>{}) for the storage type
template <typename F> static auto la_type(int dtype, F&& f) {
  if (dtype == PYGHO_F32) return f(LinearOps<float>{});
  if (dtype == PYGHO_BF16) return f(LinearOps<bf16>{});
  return f(LinearOps<f16>{});
}
static int la_size(int dtype) { return dtype == PYGHO_F32 ? 4 : 2; }

static int la_check(const char* what, int64_t m, int64_t k, int64_t n, double eps, int act, int dtype) {
  if (m < 0 || k <= 0 || n <= 0 || k >= (1 << 26) || n >= (1 << 26)) { set_error("%s: bad size", what); return PYGHO_ERR_INVALID; }
  if (!ro_float(dtype)) { set_error("%s: f32 / bf16 / f16 only", what); return PYGHO_ERR_UNSUPPORTED; }
  if (act < 0 || act > kActElu) { set_error("%s: unknown activation %d", what, act); return PYGHO_ERR_INVALID; }
  if (!(eps >= 0.0)) { set_error("%s: eps must not be negative", what); return PYGHO_ERR_INVALID; }
  return PYGHO_OK;
}
static int la_param_check(const char* what, const void* p, int pdt, int dtype) {
  if (p && pdt != dtype && pdt != PYGHO_F32) { set_error("%s: parameters in the rows' type or in f32", what); return PYGHO_ERR_UNSUPPORTED; }
  return PYGHO_OK;
}
static int la_stride_check(const char* what, int64_t a, int64_t b, int dtype) {        // 32-bit offsets inside a block of 32 rows
  if (a < 0 || b < 0 || std::max(a, b) * la_size(dtype) >= (1 << 27)) { set_error("%s: row strides of 0 .. 2^27 bytes", what); return PYGHO_ERR_UNSUPPORTED; }
  return PYGHO_OK;
}

// The form of a forward over (k, n).  W fits a CU's LDS: linear_stream.h where a norm needs the row, for up to 128 output channels (linear_out.h forms
// 64 at a time) and for k beyond what linear_out.h holds in registers; linear_out.h for the rest.  Otherwise tiles.
// bf16, 1.05 M rows, silu, us of stream / out / tile: 128 -> 16 53 / 70 / 68, -> 32 65 / 75 / 88, -> 64 82 / 85 / 108, -> 128 111 / 121 / 183,
// 256 -> 256 270 / 253 / 436
enum { FORM_TILE = 0, FORM_STREAM = 1, FORM_OUT = 2 };
static int la_form(int64_t k, int64_t n, int norm, int dtype) {
  return la_type(dtype, [&](auto ops) {
    const bool stream = ops.stream_lds(k, n, 0, false, false) <= kLsLds, out = !norm && ops.out_lds(k, n) <= kLsLds;
    return stream && (!out || n <= 128) ? FORM_STREAM : out ? FORM_OUT : FORM_TILE;
  });
}
static int la_forward(const LsArgs& a, int form, int norm, int dtype, hipStream_t st) {
  return la_type(dtype, [&](auto ops) { return form == FORM_OUT ? ops.out_fwd(a, st) : ops.stream_fwd(a, norm, st); });
}
// whether x, the rows of gy and what is stored beside them allow the unmasked accesses of linear_stream.h
static int la_vec(const void* x, int64_t x_ld, const void* r, int64_t r_ld, const void* out, int64_t k, int64_t n, int dtype) {
  const int es = la_size(dtype);
  return (k % (64 / es) == 0 && la_aligned(x, x_ld, es, 16) ? 1 : 0) | (n % 16 == 0 && la_aligned(r, r_ld, es, 16) && la_aligned(out, n, es, 16) ? 2 : 0);
}
static LsArgs la_stream_args(const void* x, int64_t x_ld, const void* w, int64_t w_ld, const void* bias, int bias_dtype, const void* g, const void* h,
                             int norm_dtype, const void* r, int64_t r_ld, void* out, int64_t m, int64_t k, int64_t n, double eps, int act, int dtype) {
  LsArgs a{};
  a.x = x; a.x_ld = x_ld;
  a.w = w; a.w_ld = w_ld;
  a.bias = bias; a.bias_dtype = bias_dtype; a.g = g; a.h = h; a.norm_dtype = norm_dtype;
  a.r = r; a.r_ld = r_ld;
  a.out = out;
  a.vec = la_vec(x, x_ld, r, r_ld, out, k, n, dtype);
  a.m = m; a.k = (int)k; a.n = (int)n; a.eps = (float)eps; a.act = act;
  return a;
}
static int la_tile_act(const void* x, int64_t x_ld, const void* w, int64_t w_ld, const void* bias, int bias_dtype, const void* residual, int64_t residual_ld,
                       void* y, void* z, int z_f32, int64_t m, const int32_t* m_dev, int64_t k, int64_t n, int act, int dtype, hipStream_t st) {
  const int es = la_size(dtype);
  LaArgs a{};
  a.a = {x, x_ld};
  a.b = {w, w_ld};
  a.m = m; a.n = n; a.k = k; a.dev = m_dev;
  a.out = y;
  a.z = z; a.z_f32 = z_f32;
  a.bias = bias; a.bias_dtype = bias_dtype;
  a.res = residual; a.res_ld = residual_ld;
  a.act = act;
  return la_type(dtype, [&](auto ops) { return ops.tile_act(a, st); });
}

// slabs of a weight gradient: enough workgroups for two per CU, at most one per chunk of rows
static int64_t la_dw_slabs(int64_t m, int64_t k, int64_t n) {
  if (m <= 0) return 0;
  const int64_t tiles = (n > 64 && k > 64) ? ceil_div(n, 128) * ceil_div(k, 128) : ceil_div(n, 64) * ceil_div(k, k <= 16 ? 16 : 64);
  return std::min<int64_t>(ceil_div(m, kLaChunk), std::max<int64_t>(1, 512 / tiles));
}
static int64_t la_pad4(int64_t v) { return (v + 3) / 4 * 4; }

// The launches of a backward pass and its workspace, in bytes: [dz] [z] [slabs of the sums over n] [slabs of dW | db] [W^T]
//   fused   dz, dX, dW and every sum from one streaming launch (dW asked for, operands aligned; its slabs are [sums | dW]): 1.05 M rows of 128 -> 64 / 128
//           bf16 151 / 220 us, in separate launches 261 / 357
//   stream  dz with the sums (and dX where W fits as that product needs it) from a streaming launch: 1.05 M rows of 256 -> 256 bf16 770 us,
//           dX in a launch of its own 549 + 273
//   else    dz by the row kernel from the pre-activation: kept by the forward, or (z) formed again in f32 where the forward streams
// dz is in the rows' type everywhere: see linear_stream.h for what that rounding costs (its sums are taken before it).  It reaches memory where a later
// launch reads it
struct LaAsk { bool gx, gw, gb, aligned; };                    // the gradients of a call; aligned: VEC 3 of linear_stream.h
struct LaSpace { int64_t dz, z, sums, dw, wt, total; int nsum; int64_t dw_k; bool fused, stream, own_dz, gx_here; };
static LaSpace la_space(int64_t m, int64_t k, int64_t n, int norm, int act, int dtype, const LaAsk& ask) {
  LaSpace s{};
  s.nsum = norm ? 3 : 1;
  s.fused = ask.gw && ask.aligned && la_type(dtype, [&](auto ops) { return ops.dw_fits(k, n, s.nsum); });
  if (s.fused) {
    s.total = s.dw = std::min<int64_t>(kLsDwGrid, ceil_div(m, 16 * kLsDwWaves)) * la_pad4(s.nsum * n + n * k) * 4;
    return s;
  }
  s.own_dz = norm || act != kActNone;
  s.stream = s.own_dz && n <= ls_bwd_max(norm, la_size(dtype)) && la_type(dtype, [&](auto ops) { return ops.stream_lds(k, n, s.nsum, false, false) <= kLsLds; });
  s.gx_here = ask.gx && s.stream && la_type(dtype, [&](auto ops) { return ops.stream_lds(k, n, s.nsum, true, false) <= kLsLds; });
  const bool gx_later = ask.gx && !s.gx_here, db = ask.gb && !s.own_dz;     // (dz = gy: its column sums come with dW, or with 16 columns of it)
  s.dw_k = ask.gw ? k : db ? std::min<int64_t>(k, 16) : 0;
  s.dz = s.own_dz && (!s.stream || ask.gw || gx_later) ? (m * n * la_size(dtype) + 15) / 16 * 16 : 0;
  s.z = s.own_dz && !s.stream && la_form(k, n, norm, dtype) != FORM_TILE ? (m * n * 4 + 15) / 16 * 16 : 0;
  const int64_t slabs = std::min<int64_t>(kLsGrid, ceil_div(m, 16));      // a streaming launch: at most one workgroup per block of rows
  s.sums = !s.own_dz ? 0 : s.stream ? slabs * la_pad4(s.nsum * n) * 4 : ln_bwd_slab_floats(m, n, s.nsum) * 4;
  s.dw = s.dw_k ? la_dw_slabs(m, s.dw_k, n) * la_pad4(n * s.dw_k + n) * 4 : 0;
  s.wt = gx_later && la_form(n, k, 0, dtype) == FORM_TILE ? (n * k * la_size(dtype) + 15) / 16 * 16 : 0;
  s.total = s.dz + s.z + s.sums + s.dw + s.wt;
  return s;
}
static int la_vec_bwd(const void* gx, const void* x, int64_t x_ld, const void* gy, int64_t gy_ld, int64_t k, int64_t n, int dtype) {
  const int vec = la_vec(x, x_ld, gy, gy_ld, nullptr, k, n, dtype);       // (dz's place in the workspace is aligned; dX is stored in the same launch)
  return gx && !(k % 16 == 0 && la_aligned(gx, k, la_size(dtype), 16)) ? vec & 1 : vec;
}

}  // namespace pygho

using namespace pygho;

// what the forward keeps for the backward besides x: 0 nothing, 1 the pre-activation in the rows' type or in f32 (PYGHO_ROW_Z_F32), 2 the
// pre-activation in f32 (needed by the forward itself as well)
extern "C" int pygho_linear_act_keeps(int64_t k, int64_t n, int norm, int act, int dtype) {
  if (k <= 0 || n <= 0 || !ro_float(dtype) || la_form(k, n, norm, dtype) != FORM_TILE) return 0;
  return norm ? 2 : act != kActNone ? 1 : 0;
}

extern "C" int pygho_linear_act(void* y, void* z, const void* x, int64_t x_ld, const void* w, int64_t w_ld, const void* bias, int bias_dtype, int norm,
                                const void* g, const void* h, int norm_dtype, double eps, const void* residual, int64_t residual_ld, int64_t m,
                                int64_t k, int64_t n, int act, int dtype, void* stream) {
  const int z_f32 = (act & PYGHO_ROW_Z_F32) != 0;
  act &= ~PYGHO_ROW_Z_F32;
  if (int rc = la_check("linear_act", m, k, n, eps, act, dtype)) return rc;
  if (int rc = la_param_check("linear_act", bias, bias_dtype, dtype)) return rc;
  if (g || h) { if (int rc = la_param_check("linear_act", g ? g : h, norm_dtype, dtype)) return rc; }
  if (int rc = la_stride_check("linear_act", x_ld, residual ? residual_ld : 0, dtype)) return rc;
  if (m == 0) return PYGHO_OK;
  if (!y || !x || !w) { set_error("null pointer"); return PYGHO_ERR_INVALID; }
  hipStream_t st = (hipStream_t)stream;
  if (const int form = la_form(k, n, norm, dtype); form != FORM_TILE)
    return la_forward(la_stream_args(x, x_ld, w, w_ld, bias, bias_dtype, g, h, norm_dtype, residual, residual_ld, y, m, k, n, eps, act, dtype), form, norm, dtype, st);
  if (!norm) return la_tile_act(x, x_ld, w, w_ld, bias, bias_dtype, residual, residual_ld, y, z, z_f32, m, nullptr, k, n, act, dtype, st);
  if (!z) { set_error("linear_act: this norm needs the pre-activation's buffer (pygho_linear_act_keeps)"); return PYGHO_ERR_INVALID; }
  if (int rc = la_tile_act(x, x_ld, w, w_ld, bias, bias_dtype, nullptr, 0, nullptr, z, 1, m, nullptr, k, n, kActNone, dtype, st)) return rc;
  return ln_fwd_launch(y, z, n, g, h, norm_dtype, residual, residual_ld, m, n, (float)eps, act, dtype, PYGHO_F32, st);
}

extern "C" size_t pygho_linear_act_bwd_workspace(int64_t m, int64_t k, int64_t n, int norm, int act, int dtype) {
  if (m <= 0 || k <= 0 || n <= 0 || !ro_float(dtype)) return 0;
  return (size_t)std::max(la_space(m, k, n, norm, act, dtype, LaAsk{true, true, true, true}).total, la_space(m, k, n, norm, act, dtype, LaAsk{true, true, true, false}).total);
}

extern "C" size_t pygho_linear_act_bwd_workspace_for(const void* gx, int want_gw, int want_gb, const void* x, int64_t x_ld, const void* gy, int64_t gy_ld,
                                                     int64_t m, int64_t k, int64_t n, int norm, int act, int dtype) {
  if (m <= 0 || k <= 0 || n <= 0 || !ro_float(dtype)) return 0;
  return (size_t)la_space(m, k, n, norm, act, dtype, LaAsk{gx != nullptr, want_gw != 0, want_gb != 0, la_vec_bwd(gx, x, x_ld, gy, gy_ld, k, n, dtype) == 3}).total;
}

extern "C" int pygho_linear_act_bwd(void* gx, void* gw, int gw_dtype, void* gb, int gb_dtype, void* gg, int gg_dtype, void* gh, int gh_dtype,
                                    const void* z, const void* x, int64_t x_ld, const void* w, int64_t w_ld, const void* bias, int bias_dtype,
                                    int norm, const void* g, const void* h, int norm_dtype, double eps, const void* gy, int64_t gy_ld,
                                    int64_t m_cap, const int32_t* m_dev, int64_t k, int64_t n, int act, int dtype, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const bool z_f32 = (act & PYGHO_ROW_Z_F32) != 0;
  act &= ~PYGHO_ROW_Z_F32;
  if (int rc = la_check("linear_act_bwd", m_cap, k, n, eps, act, dtype)) return rc;
  if (int rc = la_param_check("linear_act_bwd", bias, bias_dtype, dtype)) return rc;
  if (g || h) { if (int rc = la_param_check("linear_act_bwd", g ? g : h, norm_dtype, dtype)) return rc; }
  if ((gw && !ro_float(gw_dtype)) || (gb && !ro_float(gb_dtype)) || (gg && !ro_float(gg_dtype)) || (gh && !ro_float(gh_dtype)) || (!norm && (gg || gh))) {
    set_error("linear_act_bwd: gradients in f32 / bf16 / f16; gg and gh with a norm only");
    return PYGHO_ERR_UNSUPPORTED;
  }
  if (int rc = la_stride_check("linear_act_bwd", x_ld, gy_ld, dtype)) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (m_cap == 0) {                                           // no rows: every gradient of a parameter is zero
    if (int rc = fold_launch(FoldOut{{gw, gb, gg, gh}, {gw ? n * k : 0, gb ? n : 0, gg ? n : 0, gh ? n : 0}, {gw_dtype, gb_dtype, gg_dtype, gh_dtype}}, nullptr, 0, 0, st)) return rc;
    return PYGHO_OK;
  }
  if (!x || !w || !gy) { set_error("null pointer"); return PYGHO_ERR_INVALID; }
  const int vec = la_vec_bwd(gx, x, x_ld, gy, gy_ld, k, n, dtype);
  const LaSpace sp = la_space(m_cap, k, n, norm, act, dtype, LaAsk{gx != nullptr, gw != nullptr, gb != nullptr, vec == 3});
  if (sp.total > 0 && !workspace) { set_error("null pointer"); return PYGHO_ERR_INVALID; }
  if (workspace_bytes < (size_t)sp.total || (uintptr_t)workspace % 16 != 0) { set_error("linear_act_bwd: workspace too small or not 16-byte aligned"); return PYGHO_ERR_INVALID; }
  if (pygho_linear_act_keeps(k, n, norm, act, dtype) != 0 && !z) { set_error("linear_act_bwd: the kept pre-activation is missing"); return PYGHO_ERR_INVALID; }
  char* base = reinterpret_cast<char*>(workspace);
  LsArgs fa = la_stream_args(x, x_ld, w, w_ld, bias, bias_dtype, g, h, norm_dtype, gy, gy_ld, base, m_cap, k, n, eps, act, dtype);
  fa.vec = vec;
  fa.m_dev = m_dev;
  if (sp.fused) {
    fa.out = nullptr;
    fa.gx = gx;
    fa.slabs = reinterpret_cast<float*>(base);
    fa.slab_stride = la_pad4(sp.nsum * n + n * k);
    int used = 0;
    if (int rc = la_type(dtype, [&](auto ops) { return ops.stream_bwd(fa, norm, true, &used, st); })) return rc;
    const FoldOut o = norm ? FoldOut{{gg, gh, gb, gw}, {n, n, n, n * k}, {gg_dtype, gh_dtype, gb_dtype, gw_dtype}}
                           : FoldOut{{gb, gw, nullptr, nullptr}, {n, n * k, 0, 0}, {gb_dtype, gw_dtype, 0, 0}};
    return gb || gg || gh || gw ? fold_launch(o, fa.slabs, used, fa.slab_stride, st) : PYGHO_OK;
  }
  const void* dz = gy;
  int64_t dz_ld = gy_ld;
  bool have_gx = gx == nullptr;
  if (sp.own_dz) {
    void* own = base;
    float* slabs = reinterpret_cast<float*>(base + sp.dz + sp.z);
    int64_t stride = la_pad4(sp.nsum * n);
    int used = 0;
    if (sp.stream) {
      fa.slabs = slabs; fa.slab_stride = stride;
      if (!sp.dz) fa.out = nullptr;
      if (sp.gx_here) {
        fa.gx = gx;
        have_gx = true;
      }
      if (int rc = la_type(dtype, [&](auto ops) { return ops.stream_bwd(fa, norm, false, &used, st); })) return rc;
    } else {
      if (sp.z) {
        LsArgs a = la_stream_args(x, x_ld, w, w_ld, bias, bias_dtype, nullptr, nullptr, 0, nullptr, 0, base + sp.dz, m_cap, k, n, 0.0, kActNone, dtype);
        a.out_f32 = 1;
        a.m_dev = m_dev;
        if (int rc = la_forward(a, la_form(k, n, 0, dtype), 0, dtype, st)) return rc;
        z = base + sp.dz;
      }
      if (int rc = ln_bwd_launch(own, slabs, &stride, &used, sp.nsum, z, n, gy, gy_ld, g, h, norm_dtype, m_cap, m_dev, n, (float)eps, act, dtype,
                                 norm || sp.z || z_f32 ? PYGHO_F32 : dtype, st)) return rc;
    }
    dz = own;
    dz_ld = n;
    if (gb || gg || gh) {
      const FoldOut o = norm ? FoldOut{{gg, gh, gb, nullptr}, {n, n, n, 0}, {gg_dtype, gh_dtype, gb_dtype, 0}}
                             : FoldOut{{gb, nullptr, nullptr, nullptr}, {n, 0, 0, 0}, {gb_dtype, 0, 0, 0}};
      if (int rc = fold_launch(o, slabs, used, stride, st)) return rc;
    }
  }
  if (!have_gx) {
    // dX = dz . W: a product over n with k output channels
    if (const int form = la_form(n, k, 0, dtype); form != FORM_TILE) {
      LsArgs a = la_stream_args(dz, dz_ld, w, w_ld, nullptr, 0, nullptr, nullptr, 0, nullptr, 0, gx, m_cap, n, k, 0.0, kActNone, dtype);
      a.w_trans = 1;
      a.m_dev = m_dev;
      if (int rc = la_forward(a, form, 0, dtype, st)) return rc;
    } else {
      void* wt = base + sp.dz + sp.z + sp.sums + sp.dw;
      if (int rc = la_type(dtype, [&](auto ops) { return ops.transpose(wt, w, w_ld, n, k, st); })) return rc;
      if (int rc = la_tile_act(dz, dz_ld, wt, n, nullptr, 0, nullptr, 0, gx, nullptr, 0, m_cap, m_dev, n, k, kActNone, dtype, st)) return rc;
    }
  }
  const bool db_here = gb && !sp.own_dz;                      // dz is gy itself: its column sums come with dW
  if (sp.dw_k) {
    LaArgs a{};
    a.a = {dz, dz_ld};
    a.b = {x, x_ld};
    a.m = n; a.n = sp.dw_k; a.k = m_cap; a.dev = m_dev;
    a.slabs = reinterpret_cast<float*>(base + sp.dz + sp.z + sp.sums);
    a.slab_stride = la_pad4(n * sp.dw_k + n);
    a.splits = (int)la_dw_slabs(m_cap, sp.dw_k, n);
    a.want_sums = db_here;
    if (int rc = la_type(dtype, [&](auto ops) { return ops.tile_dw(a, st); })) return rc;
    const FoldOut o{{gw, db_here ? gb : nullptr, nullptr, nullptr}, {n * sp.dw_k, db_here ? n : 0, 0, 0}, {gw_dtype, gb_dtype, 0, 0}};
    if (int rc = fold_launch(o, a.slabs, a.splits, a.slab_stride, st)) return rc;
  }
  return PYGHO_OK;
}
