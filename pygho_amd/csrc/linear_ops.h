// What one storage type of the linear operators offers the entry points (linear_act.hip); linear_f32.hip, linear_bf16.hip and linear_f16.hip
// instantiate it, so that the kernels of the types compile side by side.
#pragma once
#include "linear_out.h"

namespace pygho {

template <typename T> struct LinearOps {
  // bytes of LDS: the forms of linear_stream.h (a backward needs `sums` per channel, dX and dW more of it) and of linear_out.h
  static int stream_lds(int64_t k, int64_t n, int sums, bool dx, bool dw);
  static int out_lds(int64_t k, int64_t n);
  static bool dw_fits(int64_t k, int64_t n, int sums);
  static int stream_fwd(const LsArgs& a, int norm, hipStream_t st);
  static int out_fwd(const LsArgs& a, hipStream_t st);
  static int stream_bwd(const LsArgs& a, int norm, bool dw, int* n_slabs, hipStream_t st);
  static int tile_act(const LaArgs& a, hipStream_t st);
  static int transpose(void* wt, const void* w, int64_t w_ld, int64_t n, int64_t k, hipStream_t st);
  static int tile_dw(const LaArgs& a, hipStream_t st);
};

#define PYGHO_LINEAR_TYPE(T)                                                                                                                   \
  template <> int LinearOps<T>::stream_lds(int64_t k, int64_t n, int sums, bool dx, bool dw) { return ls_lds_any<T>(k, n, sums, dx, dw); }     \
  template <> int LinearOps<T>::out_lds(int64_t k, int64_t n) { return lo_lds<T>(k, n); }                                                      \
  template <> bool LinearOps<T>::dw_fits(int64_t k, int64_t n, int sums) { return ls_dw_fits<T>(k, n, sums); }                                 \
  template <> int LinearOps<T>::stream_fwd(const LsArgs& a, int norm, hipStream_t st) {                                                        \
    return norm ? ls_pick<T, LS_NORM, false>(a, nullptr, st) : ls_pick<T, LS_ACT, false>(a, nullptr, st);                                      \
  }                                                                                                                                            \
  template <> int LinearOps<T>::out_fwd(const LsArgs& a, hipStream_t st) { return lo_pick<T>(a, st); }                                         \
  template <> int LinearOps<T>::stream_bwd(const LsArgs& a, int norm, bool dw, int* n_slabs, hipStream_t st) {                                 \
    if (dw) return norm ? ls_pick_dw<T, LS_DNORM>(a, n_slabs, st) : ls_pick_dw<T, LS_DACT>(a, n_slabs, st);                                    \
    if (a.gx) return norm ? ls_pick<T, LS_DNORM, true>(a, n_slabs, st) : ls_pick<T, LS_DACT, true>(a, n_slabs, st);                            \
    return norm ? ls_pick<T, LS_DNORM, false>(a, n_slabs, st) : ls_pick<T, LS_DACT, false>(a, n_slabs, st);                                    \
  }                                                                                                                                            \
  template <> int LinearOps<T>::tile_act(const LaArgs& a, hipStream_t st) { return la_any<T, LA_ROWS, LA_ROWS, LA_ACT>(a, st); }               \
  template <> int LinearOps<T>::transpose(void* wt, const void* w, int64_t w_ld, int64_t n, int64_t k, hipStream_t st) {                       \
    return la_transpose<T>(wt, w, w_ld, n, k, st);                                                                                             \
  }                                                                                                                                            \
  template <> int LinearOps<T>::tile_dw(const LaArgs& a, hipStream_t st) { return la_any<T, LA_COLS, LA_COLS, LA_SLAB>(a, st); }

}  // namespace pygho
