// What one storage type of the linear operators offers the entry points (linear_act.hip); linear_f32.hip, linear_bf16.hip and linear_f16.hip
// instantiate it, so that the kernels of the types compile side by side.
#pragma once
#include "linear_stream.h"

namespace pygho {

template <typename T> struct LinearOps {
  // does a launch of the streaming form fit: the forward / dz, dz with dX, dX alone (k and n swapped, W read transposed)
  static bool stream_fits(int64_t k, int64_t n, int norm);
  static bool stream_dx_fits(int64_t k, int64_t n, int norm);
  static int stream_fwd(const LsArgs& a, int norm, hipStream_t st);
  static int stream_bwd(const LsArgs& a, int norm, int* n_slabs, hipStream_t st);
  static int tile_act(const LaArgs& a, hipStream_t st);
  static int tile_dx(const LaArgs& a, hipStream_t st);
  static int tile_dw(const LaArgs& a, hipStream_t st);
};

#define PYGHO_LINEAR_TYPE(T)                                                                                                                   \
  template <> bool LinearOps<T>::stream_fits(int64_t k, int64_t n, int norm) { return ls_lds_any<T>(k, n, norm ? 3 : 1, false) <= kLsLds; }    \
  template <> bool LinearOps<T>::stream_dx_fits(int64_t k, int64_t n, int norm) { return ls_lds_any<T>(k, n, norm ? 3 : 1, true) <= kLsLds; }  \
  template <> int LinearOps<T>::stream_fwd(const LsArgs& a, int norm, hipStream_t st) {                                                        \
    return norm ? ls_pick<T, LS_NORM, false>(a, nullptr, st) : ls_pick<T, LS_ACT, false>(a, nullptr, st);                                      \
  }                                                                                                                                            \
  template <> int LinearOps<T>::stream_bwd(const LsArgs& a, int norm, int* n_slabs, hipStream_t st) {                                          \
    if (a.gx) return norm ? ls_pick<T, LS_DNORM, true>(a, n_slabs, st) : ls_pick<T, LS_DACT, true>(a, n_slabs, st);                            \
    return norm ? ls_pick<T, LS_DNORM, false>(a, n_slabs, st) : ls_pick<T, LS_DACT, false>(a, n_slabs, st);                                    \
  }                                                                                                                                            \
  template <> int LinearOps<T>::tile_act(const LaArgs& a, hipStream_t st) { return la_any<T, LA_ROWS, LA_ROWS, LA_ACT>(a, st); }               \
  template <> int LinearOps<T>::tile_dx(const LaArgs& a, hipStream_t st) { return la_any<T, LA_ROWS, LA_COLS, LA_ACT>(a, st); }                \
  template <> int LinearOps<T>::tile_dw(const LaArgs& a, hipStream_t st) { return la_any<T, LA_COLS, LA_COLS, LA_SLAB>(a, st); }

}  // namespace pygho
