// Entry points of the linear operators (kernels and their reasons: linear_tile.h): argument checks, operand alignment, type dispatch.
#include "linear_tile.h"

namespace pygho {

template <> int la_forward<float>(const LaArgs&, int, hipStream_t);
template <> int la_forward<bf16>(const LaArgs&, int, hipStream_t);
template <> int la_forward<f16>(const LaArgs&, int, hipStream_t);
template <> int la_dz<float>(const LaArgs&, int, hipStream_t, int*);
template <> int la_dz<bf16>(const LaArgs&, int, hipStream_t, int*);
template <> int la_dz<f16>(const LaArgs&, int, hipStream_t, int*);
template <> int la_dx<float>(const LaArgs&, hipStream_t);
template <> int la_dx<bf16>(const LaArgs&, hipStream_t);
template <> int la_dx<f16>(const LaArgs&, hipStream_t);
template <> int la_dw<float>(const LaArgs&, hipStream_t);
template <> int la_dw<bf16>(const LaArgs&, hipStream_t);
template <> int la_dw<f16>(const LaArgs&, hipStream_t);

static bool la_float(int d) { return d == PYGHO_F32 || d == PYGHO_BF16 || d == PYGHO_F16; }
static int la_check(const char* what, int64_t m, int64_t k, int64_t n, int act, int dtype) {
  if (m < 0 || k <= 0 || n <= 0 || k > INT32_MAX / 2 || n > INT32_MAX / 2) { set_error("%s: bad size", what); return PYGHO_ERR_INVALID; }
  if (!la_float(dtype)) { set_error("%s: f32 / bf16 / f16 only", what); return PYGHO_ERR_UNSUPPORTED; }
  if (act < 0 || act > kActElu) { set_error("%s: unknown activation %d", what, act); return PYGHO_ERR_INVALID; }
  return PYGHO_OK;
}
static LaOperand la_operand(const void* p, int64_t ld, int dtype) {
  return LaOperand{p, ld, la_aligned(p, ld, dtype == PYGHO_F32 ? 4 : 2, 16) ? 1 : 0};
}

}  // namespace pygho

using namespace pygho;

extern "C" int pygho_linear_norm_max(void) { return kLaNormMax; }

extern "C" int pygho_linear_act(void* y, const void* x, int64_t x_ld, const void* w, int64_t w_ld, const void* bias, int bias_dtype, int norm,
                                const void* g, const void* h, int norm_dtype, double eps, const void* residual, int64_t residual_ld, int64_t m,
                                int64_t k, int64_t n, int act, int dtype, int y_dtype, void* stream) {
  if (int rc = la_check("linear_act", m, k, n, act, dtype)) return rc;
  if (y_dtype != dtype && (y_dtype != PYGHO_F32 || norm || residual)) { set_error("linear_act: an f32 output has no norm and no residual"); return PYGHO_ERR_UNSUPPORTED; }
  if (norm && (n > kLaNormMax || !(eps >= 0.0))) { set_error("linear_act: a norm over at most %d channels, eps >= 0", kLaNormMax); return PYGHO_ERR_UNSUPPORTED; }
  if (m == 0) return PYGHO_OK;
  if (!y || !x || !w) { set_error("null pointer"); return PYGHO_ERR_INVALID; }
  const int es = dtype == PYGHO_F32 ? 4 : 2;
  LaArgs a{};
  a.a = la_operand(x, x_ld, dtype);
  a.b = la_operand(w, w_ld, dtype);
  a.m = m; a.n = n; a.k = k;
  a.out_f32 = y_dtype == PYGHO_F32;
  a.out = y; a.out_ld = n; a.out_vec = la_aligned(y, n, a.out_f32 ? 4 : es, 4 * (a.out_f32 ? 4 : es));
  a.bias = bias; a.bias_dtype = bias_dtype;
  a.res = residual; a.res_ld = residual_ld; a.res_vec = la_aligned(residual, residual_ld, es, 4 * es);
  a.g = g; a.h = h; a.norm_dtype = norm_dtype; a.eps = (float)eps; a.act = act;
  if (dtype == PYGHO_F32) return la_forward<float>(a, norm, (hipStream_t)stream);
  return dtype == PYGHO_BF16 ? la_forward<bf16>(a, norm, (hipStream_t)stream) : la_forward<f16>(a, norm, (hipStream_t)stream);
}

extern "C" int pygho_linear_act_dz_slabs(int64_t m) { return m <= 0 ? 0 : (int)std::min<int64_t>((ceil_div(m, 64) + 7) / 8 * 8, kLaNormGrid); }

extern "C" int pygho_linear_act_dz(void* dz, float* slabs, int64_t slab_stride, int* n_slabs, const void* x, int64_t x_ld, const void* w, int64_t w_ld,
                                   const void* bias, int bias_dtype, int norm, const void* g, const void* h, int norm_dtype, double eps,
                                   const void* gy, int64_t gy_ld, int64_t m_cap, const int32_t* m_dev, int64_t k, int64_t n, int act, int dtype,
                                   void* stream) {
  if (int rc = la_check("linear_act_dz", m_cap, k, n, act, dtype)) return rc;
  if (norm && (n > kLaNormMax || !(eps >= 0.0))) { set_error("linear_act_dz: a norm over at most %d channels, eps >= 0", kLaNormMax); return PYGHO_ERR_UNSUPPORTED; }
  if (!n_slabs || (norm && slab_stride < 2 * n)) { set_error("linear_act_dz: n_slabs, and 2 n floats per slab"); return PYGHO_ERR_INVALID; }
  *n_slabs = 0;
  if (m_cap == 0) return PYGHO_OK;
  if (!dz || !x || !w || !gy || (norm && !slabs)) { set_error("null pointer"); return PYGHO_ERR_INVALID; }
  const int es = dtype == PYGHO_F32 ? 4 : 2;
  LaArgs a{};
  a.a = la_operand(x, x_ld, dtype);
  a.b = la_operand(w, w_ld, dtype);
  a.m = m_cap; a.n = n; a.k = k; a.m_dev = m_dev;
  a.out = dz; a.out_ld = n; a.out_vec = la_aligned(dz, n, es, 4 * es);
  a.bias = bias; a.bias_dtype = bias_dtype;
  a.res = gy; a.res_ld = gy_ld; a.res_vec = la_aligned(gy, gy_ld, es, 4 * es);
  a.g = g; a.h = h; a.norm_dtype = norm_dtype; a.eps = (float)eps; a.act = act;
  a.slabs = slabs; a.slab_stride = slab_stride;
  if (dtype == PYGHO_F32) return la_dz<float>(a, norm, (hipStream_t)stream, norm ? n_slabs : nullptr);
  return dtype == PYGHO_BF16 ? la_dz<bf16>(a, norm, (hipStream_t)stream, norm ? n_slabs : nullptr)
                             : la_dz<f16>(a, norm, (hipStream_t)stream, norm ? n_slabs : nullptr);
}

extern "C" int pygho_linear_dx(void* gx, const void* dz, int64_t dz_ld, const void* w, int64_t w_ld, int64_t m, int64_t k, int64_t n, int dtype,
                               void* stream) {
  if (int rc = la_check("linear_dx", m, k, n, 0, dtype)) return rc;
  if (m == 0) return PYGHO_OK;
  if (!gx || !dz || !w) { set_error("null pointer"); return PYGHO_ERR_INVALID; }
  const int es = dtype == PYGHO_F32 ? 4 : 2;
  LaArgs a{};
  a.a = la_operand(dz, dz_ld, dtype);
  a.b = la_operand(w, w_ld, dtype);                     // W (n, k): stored with the OUTPUT channel k of this product contiguous
  a.m = m; a.n = k; a.k = n;
  a.out = gx; a.out_ld = k; a.out_vec = la_aligned(gx, k, es, 4 * es);
  if (dtype == PYGHO_F32) return la_dx<float>(a, (hipStream_t)stream);
  return dtype == PYGHO_BF16 ? la_dx<bf16>(a, (hipStream_t)stream) : la_dx<f16>(a, (hipStream_t)stream);
}

// slabs of a weight gradient: enough workgroups for two per CU, at most one per chunk of rows
extern "C" int pygho_linear_dw_slabs(int64_t m, int64_t k, int64_t n) {
  if (m <= 0 || k <= 0 || n <= 0) return 0;
  const int64_t tiles = (n > 64 && k > 64) ? ceil_div(n, 128) * ceil_div(k, 128) : ceil_div(n, 64) * ceil_div(k, k <= 16 ? 16 : 64);
  return (int)std::min<int64_t>(ceil_div(m, kLaChunk), std::max<int64_t>(1, 512 / tiles));
}

extern "C" int pygho_linear_dw(float* slabs, int64_t slab_stride, const void* dz, int64_t dz_ld, const void* x, int64_t x_ld, int64_t m_cap,
                               const int32_t* m_dev, int64_t k, int64_t n, int want_colsum, int dtype, void* stream) {
  if (int rc = la_check("linear_dw", m_cap, k, n, 0, dtype)) return rc;
  if (slab_stride < n * k + (want_colsum ? n : 0)) { set_error("linear_dw: slab_stride below n k (+ n)"); return PYGHO_ERR_INVALID; }
  if (m_cap == 0) return PYGHO_OK;
  if (!slabs || !dz || !x) { set_error("null pointer"); return PYGHO_ERR_INVALID; }
  LaArgs a{};
  a.a = la_operand(dz, dz_ld, dtype);
  a.b = la_operand(x, x_ld, dtype);
  a.m = n; a.n = k; a.k = m_cap; a.k_dev = m_dev;
  a.slabs = slabs; a.slab_stride = slab_stride; a.splits = pygho_linear_dw_slabs(m_cap, k, n); a.want_sums = want_colsum;
  if (dtype == PYGHO_F32) return la_dw<float>(a, (hipStream_t)stream);
  return dtype == PYGHO_BF16 ? la_dw<bf16>(a, (hipStream_t)stream) : la_dw<f16>(a, (hipStream_t)stream);
}
