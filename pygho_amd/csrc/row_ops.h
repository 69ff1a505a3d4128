// Shared pieces of the row-wise block operators (layer_norm.hip, linear_act.hip): activations and their slopes over register arrays,
// vectors of a storage type <-> f32 registers, parameters of either storage type, sums over the lanes that share a row.
#pragma once
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace pygho {

// enum pygho_row_act (pygho_hip.h)
constexpr int kActNone = PYGHO_ACT_NONE, kActRelu = PYGHO_ACT_RELU, kActSilu = PYGHO_ACT_SILU, kActElu = PYGHO_ACT_ELU;

// f32 storage takes the library's expf and expm1f (about one ulp) and the correctly rounded divide; 16-bit storage the hardware exp2 and
// reciprocal (1 ulp of f32 each, 2^-13 of a 16-bit half step)
template <typename T> struct Precise { static constexpr bool value = std::is_same<T, float>::value; };

template <bool P> __device__ __forceinline__ float ro_exp(float z) { return P ? expf(z) : __expf(z); }
template <bool P> __device__ __forceinline__ float ro_sigmoid(float z) {
  if constexpr (P) return 1.f / (1.f + expf(-z));
  return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}
// exp(z) - 1 for z <= 0.  exp(z) - 1 in f32 is off by 2^-25 absolutely: below |z| = 2^-6 the series z + z^2/2 + z^3/6 (+ z^4/24) takes
// over, whose first dropped term is z^5/120 < 2^-30 |z|
template <bool P> __device__ __forceinline__ float ro_expm1(float z) {
  if constexpr (P) return expm1f(z);
  const float series = z * fmaf(z, fmaf(z, fmaf(z, 1.f / 24.f, 1.f / 6.f), 0.5f), 1.f);
  return z > -0.015625f ? series : __expf(z) - 1.f;
}

// v <- act(v).  The switch is on a launch-uniform value and stands outside the loop over the registers
template <bool P, int N> __device__ __forceinline__ void ro_act(float (&v)[N], int act) {
  if (act == kActSilu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] * ro_sigmoid<P>(v[i]);
  } else if (act == kActRelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];        // a NaN stays
  } else if (act == kActElu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] <= 0.f ? ro_expm1<P>(v[i]) : v[i];
  }
}

// g <- g * act'(z)
template <bool P, int N> __device__ __forceinline__ void ro_act_slope(float (&g)[N], const float (&z)[N], int act) {
  if (act == kActSilu) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float s = ro_sigmoid<P>(z[i]);
      g[i] *= fmaf(z[i] * s, 1.f - s, s);                              // s (1 + z (1 - s))
    }
  } else if (act == kActRelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = z[i] <= 0.f ? 0.f : g[i];
  } else if (act == kActElu) {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] *= z[i] <= 0.f ? ro_exp<P>(z[i]) : 1.f;          // (not expm1 + 1: that is 0 below -17)
  }
}

// ---- VE consecutive elements of T <-> f32 registers (p aligned to VE * sizeof(T), to 16 bytes beyond that) --------------------
template <typename T, int VE> __device__ __forceinline__ void ro_load(const T* p, float (&v)[VE]) {
  constexpr int B = VE * (int)sizeof(T);
  if constexpr (VE == 1) {
    v[0] = load_as_acc<T>(p);
  } else if constexpr (B == 16) {
    Vec16<T>::unpack(*reinterpret_cast<const uint4*>(p), v);
  } else {
    static_assert(B == 32 && std::is_same<T, float>::value, "vector width");
    const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 4);
    v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
    v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
  }
}
template <typename T, int VE> __device__ __forceinline__ void ro_store(T* p, const float (&v)[VE]) {
  if constexpr (VE == 1) {
    store_from_acc<T>(p, v[0]);
  } else {
    static_assert(VE * (int)sizeof(T) == 16, "vector width");
    *reinterpret_cast<uint4*>(p) = Vec16<T>::pack(v);
  }
}

// one value of a parameter vector (nullable: `none`) that is stored in f32 or in the 16-bit type `dtype`
__device__ __forceinline__ float ro_param(const void* p, int dtype, int64_t i, float none) {
  if (!p) return none;
  if (dtype == PYGHO_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == PYGHO_BF16) return load_as_acc<bf16>(reinterpret_cast<const bf16*>(p) + i);
  return load_as_acc<f16>(reinterpret_cast<const f16*>(p) + i);
}
__device__ __forceinline__ void ro_store_param(void* p, int dtype, int64_t i, float v) {
  if (dtype == PYGHO_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == PYGHO_BF16) store_from_acc<bf16>(reinterpret_cast<bf16*>(p) + i, v);
  else store_from_acc<f16>(reinterpret_cast<f16*>(p) + i, v);
}

// ---- sum over groups of L consecutive lanes (L = 1 .. 64, a power of two); every lane of a group gets the same bits ----------------
template <int CTRL> __device__ __forceinline__ float ro_dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int L> __device__ __forceinline__ float ro_lane_sum(float v) {
  if constexpr (L >= 2) v += ro_dpp<0xB1>(v);       // quad_perm [1, 0, 3, 2]
  if constexpr (L >= 4) v += ro_dpp<0x4E>(v);       // quad_perm [2, 3, 0, 1]
  if constexpr (L >= 8) v += ro_dpp<0x141>(v);      // row_half_mirror: the other quad of 8 lanes
  if constexpr (L >= 16) v += ro_dpp<0x140>(v);     // row_mirror: the other 8 of 16 lanes
  if constexpr (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
  }
  if constexpr (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
  }
  return v;
}

// ---- shared launches (layer_norm.hip) -------------------------------------------------------------------------------------------------
bool ro_float(int dtype);
// the norm / activation of rows kept in `x_dtype` (dtype or f32), see pygho_layer_norm_act; sums = 3 (gg, gh, column sums of gx), 2 (gg, gh) or
// 1 (no norm: gx = gy act'(x) and its column sums)
int ln_fwd_launch(void* y, const void* x, int64_t x_ld, const void* weight, const void* bias, int param_dtype, const void* residual,
                  int64_t residual_ld, int64_t m, int64_t c, float eps, int act, int dtype, int x_dtype, hipStream_t st);
int64_t ln_bwd_slab_floats(int64_t m, int64_t c, int sums);
int ln_bwd_launch(void* gx, float* slabs, int64_t* stride, int* n_slabs, int sums, const void* x, int64_t x_ld, const void* gy, int64_t gy_ld,
                  const void* weight, const void* bias, int param_dtype, int64_t m, const int32_t* m_dev, int64_t c, float eps, int act, int dtype,
                  int x_dtype, hipStream_t st);
// out.p[0][0 .. len[0]) | out.p[1][..] | .. = the columns of n_slabs slabs (`stride` floats apart, a multiple of 4) added in a fixed order that
// trailing slabs of zeros do not change; null outputs are skipped
struct FoldOut { void* p[4]; int64_t len[4]; int dt[4]; };
int fold_launch(const FoldOut& out, const float* slabs, int64_t n_slabs, int64_t stride, hipStream_t st);

}  // namespace pygho
