// Streaming form of a product whose reduction fits a lane's registers and whose output may be wide: y = act(x W^T + b) + r with K <= 256 16-bit
// (128 f32) values, and dX = dz W (the same product with W read transposed).
// As linear_stream.h: W in LDS for the whole launch, wavefronts walk blocks of rows without barriers.  Here the roles of the registers are the other
// way round: a block's x (32 rows x K) stays in them while the output channels go by, 64 at a time -- no state per output channel, so the width is
// bounded by LDS only, and every fragment of W serves 32 rows (at K = N = 256 with 16 rows per fragment, reading W took 64 of the ~114 cycles that
// HBM takes per row, and the launch 0.73 ms instead of the 0.46 ms of its bytes).  Measured: bf16 2.39 M x 256 -> 256 0.51 ms = 4.8 TB/s.
#pragma once
#include "linear_stream.h"

namespace pygho {

constexpr int kLoThreads = 512;

// 16-row blocks of a wavefront and turn: two, one for the longest f32 rows (their x and the next block's would not fit beside the products, and an f32
// fragment already feeds four MFMAs of 32 cycles)
template <typename T, int KS> constexpr int lo_blocks() { return sizeof(T) == 4 && KS == 8 ? 1 : 2; }

// KS: 64-byte steps of k held in registers
template <typename T, int KS, int VEC>
__global__ __launch_bounds__(kLoThreads) void linear_out_kernel(LsArgs a) {
  constexpr bool P = Precise<T>::value;
  constexpr bool XV = VEC & 1, NV = VEC & 2, PAIR = sizeof(T) == 2 && NV;      // as in linear_stream.h
  constexpr int ES = sizeof(T), E = 16 / ES, MB = lo_blocks<T, KS>(), PITCH = KS * 64 + 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int K = a.k, N = a.n, NP = (N + 15) & ~15;
  char* lds_w = smem;
  float* lds_bias = reinterpret_cast<float*>(smem + NP * PITCH);
  const int lane = threadIdx.x & 63, wave = PYGHO_WAVE_INDEX(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
  const T* wp = reinterpret_cast<const T*>(a.w);
  if (!a.w_trans) {
    for (int c = threadIdx.x; c < NP * KS * 4; c += blockDim.x) {
      const int n = c / (KS * 4), kc = c - n * (KS * 4);
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (n < N) v = ls_load16<T>(wp + (int64_t)n * a.w_ld, kc * E, K);
      *reinterpret_cast<uint4*>(lds_w + n * PITCH + kc * 16) = v;
    }
  } else {
    const int cn = NP / E;
    for (int c = threadIdx.x; c < KS * 64 / ES * cn; c += blockDim.x) {
      const int k = c / cn, nc = c - k * cn;
      union { uint4 u; uint16_t h[8]; uint32_t f[4]; } v;
      v.u = make_uint4(0u, 0u, 0u, 0u);
      if (k < K) v.u = ls_load16<T>(wp + (int64_t)k * a.w_ld, nc * E, N);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if constexpr (ES == 2) *reinterpret_cast<uint16_t*>(lds_w + (nc * E + j) * PITCH + k * 2) = v.h[j];
        else *reinterpret_cast<uint32_t*>(lds_w + (nc * E + j) * PITCH + k * 4) = v.f[j];
      }
    }
  }
  for (int n = threadIdx.x; n < NP; n += blockDim.x) lds_bias[n] = n < N ? ro_param(a.bias, a.bias_dtype, n, 0.f) : 0.f;
  __syncthreads();

  const int waves = blockDim.x >> 6;
  const int64_t m_rows = a.m_dev ? *a.m_dev : a.m, n_blocks = (m_rows + MB * 16 - 1) / (MB * 16), stride = (int64_t)gridDim.x * waves;
  auto load_x = [&](int64_t b, uint4 (&dst)[MB][KS]) {
    const int last = (int)min((int64_t)(MB * 16 - 1), m_rows - 1 - b * (MB * 16));
    const char* base = reinterpret_cast<const char*>(a.x) + b * (MB * 16) * a.x_ld * ES;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const uint32_t off = (uint32_t)min(mb * 16 + r16, last) * (uint32_t)(a.x_ld * ES) + (XV ? q * 16 : 0);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if constexpr (XV) dst[mb][s] = s * (64 / ES) < K ? *reinterpret_cast<const uint4*>(base + off + s * 64) : make_uint4(0u, 0u, 0u, 0u);
        else dst[mb][s] = ls_load16<T>(reinterpret_cast<const T*>(base + off), s * (64 / ES) + q * E, K);
      }
    }
  };
  uint4 xc[MB][KS], xn[MB][KS];
  int64_t blk = (int64_t)blockIdx.x * waves + wave;
  if (blk < n_blocks) load_x(blk, xc);
  for (; blk < n_blocks; blk += stride) {
    asm volatile("" ::: "memory");                             // (see linear_stream.h)
    load_x(min(blk + stride, n_blocks - 1), xn);
    __builtin_amdgcn_sched_barrier(0);                         // (loads first: see linear_tile.h)
    const int last = (int)min((int64_t)(MB * 16 - 1), m_rows - 1 - blk * (MB * 16));
    const char* rbase = reinterpret_cast<const char*>(a.r) + blk * (MB * 16) * a.r_ld * ES;
    char* obase = reinterpret_cast<char*>(a.out) + blk * (MB * 16) * N * (a.out_f32 ? 4 : ES);
    for (int n0 = 0; n0 < NP; n0 += 64) {
      // (16-channel blocks past the end are formed again from the last one and not stored)
      la_f32x4_t o[MB][4];
      typename Raw4<T>::type rv[MB][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int nb = min(n0 + t * 16, NP - 16);
        const la_f32x4_t b4 = *reinterpret_cast<const la_f32x4_t*>(lds_bias + nb + q * 4);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          o[mb][t] = b4;
          rv[mb][t] = typename Raw4<T>::type{};
        }
      }
      auto load_r = [&]() {
        if (!a.r) return;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const uint32_t row = (uint32_t)min(mb * 16 + r16, last) * (uint32_t)(a.r_ld * ES);
#pragma unroll
          for (int t = 0; t < 4; t += 2) {
            if constexpr (PAIR) {
              if (n0 + t * 16 + 32 <= N) {
                const uint4 v = *reinterpret_cast<const uint4*>(rbase + row + (n0 + t * 16 + ls_pair_col(q)) * ES);
                rv[mb][t] = make_uint2(v.x, v.y);
                rv[mb][t + 1] = make_uint2(v.z, v.w);
                continue;
              }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int nb = min(n0 + (t + i) * 16, NP - 16);
              if constexpr (NV) rv[mb][t + i] = *reinterpret_cast<const typename Raw4<T>::type*>(rbase + row + (nb + q * 4) * ES);
              else rv[mb][t + i] = ls_load4<T>(reinterpret_cast<const T*>(rbase + row), nb + q * 4, N);
            }
          }
        }
      };
      if constexpr (KS < 8) load_r();                          // in flight during the products; with 8 steps of x there are no registers for it
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int nb = min(n0 + t * 16, NP - 16);
          const uint4 fa = *reinterpret_cast<const uint4*>(lds_w + (nb + r16) * PITCH + s * 64 + q * 16);
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) o[mb][t] = la_mfma<T>(fa, xc[mb][s], o[mb][t]);
        }
      if constexpr (KS == 8) load_r();
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const int rr = mb * 16 + r16;
        const uint32_t row16 = (uint32_t)rr * (uint32_t)(N * ES), row32 = (uint32_t)rr * (uint32_t)(N * 4);
#pragma unroll
        for (int t = 0; t < 4; t += 2) {
          const bool pair = PAIR && n0 + t * 16 + 32 <= N;     // (uniform)
          if constexpr (PAIR) { if (pair) ls_pair(rv[mb][t], rv[mb][t + 1]); }
          float u[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float r4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) u[i][e] = o[mb][t + i][e];
            ro_act<P, 4>(u[i], a.act);
            ls_unpack4<T>(rv[mb][t + i], r4);
#pragma unroll
            for (int e = 0; e < 4; ++e) u[i][e] += r4[e];
          }
          if constexpr (PAIR) {
            if (pair && !a.out_f32) {
              uint2 lo = ls_pack4<T>(u[0]), hi = ls_pack4<T>(u[1]);
              ls_pair(lo, hi);
              if (rr <= last) *reinterpret_cast<uint4*>(obase + row16 + (n0 + t * 16 + ls_pair_col(q)) * ES) = make_uint4(lo.x, lo.y, hi.x, hi.y);
              continue;
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int n = n0 + (t + i) * 16 + q * 4;
            if (rr <= last && (NV ? n0 + (t + i) * 16 : n) < N) {
              if (a.out_f32) la_store4<float>(reinterpret_cast<float*>(obase + row32 + n * 4), NV ? 4 : N - n, u[i]);
              else la_store4<T>(reinterpret_cast<T*>(obase + row16 + n * ES), NV ? 4 : N - n, u[i]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int s = 0; s < KS; ++s) xc[mb][s] = xn[mb][s];
  }
}

template <typename T> static int lo_steps(int64_t k) {         // instantiated sizes of the register-held x
  const int64_t s = (k * (int64_t)sizeof(T) + 63) / 64;
  return s <= 2 ? 2 : s <= 4 ? 4 : s <= 8 ? 8 : 0;
}
template <typename T> static int lo_lds(int64_t k, int64_t n) {
  const int s = lo_steps<T>(k);
  const int64_t np = (n + 15) / 16 * 16;
  return s == 0 || n > (1 << 14) ? INT32_MAX : (int)std::min<int64_t>(np * (s * 64 + 16) + np * 4, INT32_MAX);
}

template <typename T, int KS, int VEC> static int lo_go(const LsArgs& a, hipStream_t st) {
  static bool attr_set_dev[64] = {};
  bool& attr_set = per_device_flag(attr_set_dev);
  if (!attr_set) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&linear_out_kernel<T, KS, VEC>), hipFuncAttributeMaxDynamicSharedMemorySize, kLsLds);
    if (e != hipSuccess) { set_error("linear_out: cannot reserve %d B of LDS: %s", kLsLds, hipGetErrorString(e)); return PYGHO_ERR_LAUNCH; }
    attr_set = true;
  }
  const int lds = lo_lds<T>(a.k, a.n);
  const int64_t blocks = ceil_div(a.m, 16 * lo_blocks<T, KS>());
  const int threads = blocks < 256 * 8 ? 256 : kLoThreads;
  const int grid = (int)std::min<int64_t>(ceil_div(blocks, threads / kWave), lds <= 80 * 1024 ? 512 : 256);
  hipLaunchKernelGGL((linear_out_kernel<T, KS, VEC>), dim3(grid), dim3(threads), lds, st, a);
  return check_launch("linear_out");
}
template <typename T, int VEC> static int lo_pick_vec(const LsArgs& a, hipStream_t st) {
  switch (lo_steps<T>(a.k)) {
    case 2: return lo_go<T, 2, VEC>(a, st);
    case 4: return lo_go<T, 4, VEC>(a, st);
    case 8: return lo_go<T, 8, VEC>(a, st);
  }
  set_error("linear_out: k = %d", a.k);
  return PYGHO_ERR_UNSUPPORTED;
}
template <typename T> static int lo_pick(const LsArgs& a, hipStream_t st) {
  if (a.vec == 3) return lo_pick_vec<T, 3>(a, st);
  return a.vec & 1 ? lo_pick_vec<T, 1>(a, st) : lo_pick_vec<T, 0>(a, st);
}

}  // namespace pygho
