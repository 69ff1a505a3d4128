// Streaming form of the linear operators: W stays in LDS, every wavefront walks its own blocks of rows without a barrier.
// The tuple-wise maps have K and N of one or two hundred and 10^5 .. 10^6 rows: a row moves 0.5 .. 2 KB and needs 2 K N operations, which
// the matrix cores do in less time than HBM takes for the row.  What has to go well is the stream:
//   * W (N x K, padded rows) is read once per workgroup and serves all its rows; a workgroup lives until the rows are done;
//   * a block is 16 rows of one wavefront.  Its x fragments (lane = row, 16 bytes of k) are global loads straight into registers, the next
//     block's are in flight during this block's products and epilogue; wavefronts never wait for each other;
//   * swapped MFMA (D[n][m]): a lane ends up with 4 consecutive channels of ONE row, a row's channels sit in 4 lanes: bias (the accumulator's
//     start value), norm, activation, residual and the store happen in those registers;
//   * backward: dz leaves the epilogue in exactly the lanes and order in which the product dz . W wants its operand (the order of n inside
//     a reduction is free as long as W is read in the same one), so dX follows in the same launch without moving a value;
//   * channel sums (gg, gh, gb) are taken from the unrounded f32 values, over a block's 16 rows by lane exchanges (ls_row_sums).
// Block b of the rows belongs to wavefront b % (all wavefronts), so sums depend on the true row count only (see layer_norm.hip).
// Measured, bf16 with a norm and a residual, 1.83 M x 128 -> 128: forward 265 us (1.41 GB: 5.3 TB/s, what a copy reaches), whole gradient in one
// launch 475 .. 525 us (1.41 GB; vector issue 63 %, matrix cores 18 % of the cycles: bound by instructions at two wavefronts per SIMD, a quarter
// of them the three row sums; bank conflicts are 47 % of the LDS-active cycles, waits for LDS 11 % of the wavefronts') + fold 16
#pragma once
#include "linear_tile.h"

namespace pygho {

enum { LS_ACT = 0, LS_NORM = 1, LS_DACT = 2, LS_DNORM = 3 };

struct LsArgs {
  const void* x; int64_t x_ld;
  const void* w; int64_t w_ld; int w_trans;                   // w_trans: w is stored [k][n] (the W of dz . W)
  const void* bias; int bias_dtype; const void* g; const void* h; int norm_dtype;
  const void* r; int64_t r_ld;                                // residual (forward) / output gradient (backward)
  void* out; int out_f32;                                     // y / dz (nullable: no later launch reads it); out_f32 (LS_ACT): f32 values as they are
  void* gx;                                                   // backward, nullable: dX (rows of k)
  float* slabs; int64_t slab_stride;                          // backward: LS_DACT [gb], LS_DNORM [gg | gh | gb]
  int64_t m; const int32_t* m_dev; int k; int n; float eps; int act;
  int vec;                                                    // VEC of the kernels
  int red_bytes;                                              // bytes reserved for W and, at the end, for the reduction
};

template <typename T> struct Raw4 { using type = uint2; };
template <> struct Raw4<float> { using type = uint4; };

// 16 bytes of a row from element `off`; zeros from `end` on
template <typename T> __device__ __forceinline__ uint4 ls_load16(const T* row, int off, int end) {
  constexpr int E = 16 / (int)sizeof(T);
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (off + E <= end) return la_ld<uint4>(row + off);
  if (off >= end) return v;
  const int left = end - off;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      w[j] = j < left ? reinterpret_cast<const uint32_t*>(row + off)[j] : 0u;
    } else {
      const uint32_t lo = 2 * j < left ? reinterpret_cast<const uint16_t*>(row + off)[2 * j] : 0u;
      const uint32_t hi = 2 * j + 1 < left ? reinterpret_cast<const uint16_t*>(row + off)[2 * j + 1] : 0u;
      w[j] = lo | (hi << 16);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T> __device__ __forceinline__ typename Raw4<T>::type ls_load4(const T* row, int off, int end) {
  typename Raw4<T>::type v{};
  if (off + 4 <= end) return la_ld<typename Raw4<T>::type>(row + off);
  if (off >= end) return v;
  const int left = end - off;
  if constexpr (sizeof(T) == 4) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(row + off);
    v.x = p[0];
    v.y = left > 1 ? p[1] : 0u;
    v.z = left > 2 ? p[2] : 0u;
    v.w = left > 3 ? p[3] : 0u;
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row + off);
    v.x = (uint32_t)p[0] | (left > 1 ? (uint32_t)p[1] << 16 : 0u);
    v.y = (left > 2 ? (uint32_t)p[2] : 0u) | (left > 3 ? (uint32_t)p[3] << 16 : 0u);
  }
  return v;
}
template <typename T> __device__ __forceinline__ void ls_unpack4(const typename Raw4<T>::type& r, float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  } else {
    float t[8];
    Vec16<T>::unpack(make_uint4(r.x, r.y, 0u, 0u), t);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = t[i];
  }
}

// 16-bit rows of whole 16-channel blocks: two neighbouring blocks' 4 channels per lane become 8 consecutive channels of one of them -- a swap of the odd
// 16-lane groups of the first with the even ones of the second -- so that a load or store moves 64 contiguous bytes per row, not 2 x 32.  The swap
// is its own inverse.  Lane (r16, q) then holds channels ls_pair_col(q) .. + 7 of the two blocks' 32
__device__ __forceinline__ void ls_pair(uint2& a, uint2& b) {
  auto r = __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false);
  a.x = r[0]; b.x = r[1];
  r = __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false);
  a.y = r[0]; b.y = r[1];
}
__device__ __forceinline__ int ls_pair_col(int q) { return (q & 1) * 16 + (q >> 1) * 8; }
template <typename T> __device__ __forceinline__ uint2 ls_pack4(const float (&v)[4]) {
  const float t[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
  const uint4 r = Vec16<T>::pack(t);
  return make_uint2(r.x, r.y);
}

// 8 16-bit values per lane out of a row-major LDS tile, transposed: lane r16 gets column r16 of 4 rows at p's 16 lanes and of 4 rows `dist` bytes on
__device__ __forceinline__ uint4 ls_read_tr(const char* p, int dist) {
  const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) la_s4_t*)p));
  const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) la_s4_t*)(p + dist)));
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

// Sums over the 16 rows of a block (lanes r16 of a group): V values per lane -> their totals dealt out over the lanes.  A step gives half of the values
// to the partner lane and takes the partner's half of the others: V / 2 additions instead of V.  Partners i ^ 15, ^ 7, ^ 3, ^ 1 are single DPP
// moves; `up[s]` says which half a lane keeps (bit 3 - s of its number).  Lane i ends up with values [i * V / 16, + V / 16); below 16 values the
// steps that are left are plain sums.  Held per lane instead, the sums of 128 channels took 96 registers and one wavefront per SIMD less
template <int V, int S> __device__ __forceinline__ void ls_row_sums(float (&v)[V], const bool (&up)[4]) {
  constexpr int ctrl[4] = {0x140, 0x141, 0x1B, 0xB1};
  if constexpr (V == 1) {
    v[0] += ro_dpp<ctrl[S]>(v[0]);
    if constexpr (S < 3) ls_row_sums<1, S + 1>(v, up);
  } else {
    float w[V / 2];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float keep = up[S] ? v[j + V / 2] : v[j], send = up[S] ? v[j] : v[j + V / 2];
      w[j] = keep + ro_dpp<ctrl[S]>(send);
    }
    if constexpr (S < 3) ls_row_sums<V / 2, S + 1>(w, up);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) v[j] = w[j];
  }
}

// wavefronts per SIMD the registers are limited to (512 / this many per lane): latency, not throughput, is what a turn of 16 rows has most of
// (fewer where they do not hold the kernel: the gradient through a norm of 65 .. 128 channels with the next block's rows in flight, and masked accesses
// with an address each)
constexpr int ls_wps(int nb, int epi, int vec, int es) {
  if (vec != 3) return nb <= 2 ? 4 : nb == 4 ? 3 : nb == 8 ? 2 : 1;
  return nb <= 4 ? (nb == 4 && es == 4 && epi == LS_DNORM ? 3 : 4) : nb == 8 && epi != LS_DNORM ? 3 : 2;
}

// geometry that host and device share
template <typename T, int NB> struct LsGeom {
  static constexpr int ES = sizeof(T), NP = NB * 16;
  static constexpr int NS = (NP * ES + 63) / 64;               // 64-byte steps over n (dX)
  static constexpr int ROWS = NS * 64 / ES;                    // rows of W in LDS: whole steps of n (zeros beyond NP)
  static constexpr int PITCH_T = NS * 64 + 16;                 // f32: a row of the copy with n contiguous
  __host__ __device__ static int steps(int k) { return (k * ES + 63) / 64; }
  __host__ __device__ static int pitch_w(int k) { return steps(k) * 64 + 16; }
  __host__ __device__ static int rows_t(int k) { return (k + 15) / 16 * 16; }
  __host__ __device__ static int w_bytes(int k) { return ROWS * pitch_w(k); }
  // 16-bit: dX reads W transposed (ds_read_b64_tr_b16); f32 has no such read and keeps the copy
  __host__ __device__ static int t_bytes(int k) { return ES == 2 ? 0 : rows_t(k) * PITCH_T; }
  static constexpr int param_bytes = 4 * NP * 4;
};
// the fused weight gradient: workgroups of 4 wavefronts, two per CU, each at its own place in the sequence of phases between its barriers
constexpr int kLsDwWaves = 4, kLsDwGrid = 256 * 2;

// VEC & 1: k is a whole number of 64-byte steps and x's rows allow 16-byte accesses.  VEC & 2: n is a whole number of 16 channels and the rows of r, out
// and gx are on 16-byte boundaries (k of 16, with gx).  A block's rows then are one uniform base address, one 32-bit offset per lane and
// constants -- 64-bit addresses per access, or masks per element, take more registers than the sums do.  Otherwise vectors from any element's
// address with the ragged end masked (bf16 1.05 M rows of 100 -> 100: forward 160 us, 341 element by element; 128 -> 128 without a mask 111)
//
// DW (16-bit, k <= 128): the weight gradient in the same launch.  The workgroup's wavefronts go through their blocks in step; each puts its dz
// and its x (16 rows, row-major) into LDS, and after a barrier forms its share of dW += dz^T x over the 64 rows, both operands read back
// transposed by the LDS (ds_read_b64_tr_b16).  dz never reaches memory and x is read once: 3 streams instead of 6
template <typename T, int NB, int EPI, bool DX, int VEC, bool DW = false>
__global__ __launch_bounds__(DW ? kLsDwWaves * kWave : ls_wps(NB, EPI, VEC, sizeof(T)) * 256, DW ? 2 : ls_wps(NB, EPI, VEC, sizeof(T))) void linear_stream_kernel(LsArgs a) {
  using G = LsGeom<T, NB>;
  constexpr bool P = Precise<T>::value, BWD = EPI == LS_DACT || EPI == LS_DNORM, NORM = EPI == LS_NORM || EPI == LS_DNORM;
  constexpr int ES = G::ES, E = 16 / ES, NP = G::NP, KC = 4;
  constexpr bool XV = VEC & 1, NV = VEC & 2;
  static_assert(!DW || (DX && BWD && ES == 2 && VEC == 3 && NB >= 4 && NB <= 8), "fused weight gradient");
  constexpr int NSUM = EPI == LS_DNORM ? 3 : EPI == LS_DACT ? 1 : 0;      // sums per channel
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int K = a.k, N = a.n, KS = G::steps(K), pitch = G::pitch_w(K);
  char* lds_w = smem;
  float* lds_bias = reinterpret_cast<float*>(smem + a.red_bytes);
  float* lds_g = lds_bias + NP;
  float* lds_h = lds_g + NP;
  float* lds_on = lds_h + NP;                                  // 1 for a channel of the row, 0 for padding (comparisons would hold 32 masks)
  char* lds_t = smem + a.red_bytes + G::param_bytes;
  const int lane = threadIdx.x & 63, wave = PYGHO_WAVE_INDEX(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
  const T* wp = reinterpret_cast<const T*>(a.w);

  // ---- W -> LDS (padding: zeros) ----------------------------------------------------------------------------------------------------
  if (!a.w_trans) {
    const int cpr = KS * 4;                                    // 16-byte chunks per row
    for (int c = threadIdx.x; c < G::ROWS * cpr; c += blockDim.x) {
      const int n = c / cpr, kc = c - n * cpr;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (n < N) v = ls_load16<T>(wp + (int64_t)n * a.w_ld, kc * E, K);
      *reinterpret_cast<uint4*>(lds_w + n * pitch + kc * 16) = v;
    }
  } else {
    constexpr int CN = NP / E;
    const int kp = KS * 64 / ES;
    for (int c = threadIdx.x; c < kp * CN; c += blockDim.x) {
      const int k = c / CN, nc = c - k * CN;
      union { uint4 u; uint16_t h[8]; uint32_t f[4]; } v;
      v.u = make_uint4(0u, 0u, 0u, 0u);
      if (k < K) v.u = ls_load16<T>(wp + (int64_t)k * a.w_ld, nc * E, N);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if constexpr (ES == 2) *reinterpret_cast<uint16_t*>(lds_w + (nc * E + j) * pitch + k * 2) = v.h[j];
        else *reinterpret_cast<uint32_t*>(lds_w + (nc * E + j) * pitch + k * 4) = v.f[j];
      }
    }
  }
  if constexpr (DX && ES == 4) {                               // the copy with n contiguous
    const int kr = G::rows_t(K), ck = kr / E;
    for (int c = threadIdx.x; c < G::ROWS * ck; c += blockDim.x) {
      const int n = c / ck, kc = c - n * ck;
      union { uint4 u; uint32_t f[4]; } v;
      v.u = make_uint4(0u, 0u, 0u, 0u);
      if (n < N) v.u = ls_load16<T>(wp + (int64_t)n * a.w_ld, kc * E, K);
#pragma unroll
      for (int j = 0; j < E; ++j) *reinterpret_cast<uint32_t*>(lds_t + (kc * E + j) * G::PITCH_T + n * 4) = v.f[j];
    }
  }
  for (int n = threadIdx.x; n < NP; n += blockDim.x) {
    lds_bias[n] = n < N ? ro_param(a.bias, a.bias_dtype, n, 0.f) : 0.f;
    lds_g[n] = n < N ? ro_param(a.g, a.norm_dtype, n, 1.f) : 0.f;
    lds_h[n] = n < N ? ro_param(a.h, a.norm_dtype, n, 0.f) : 0.f;
    lds_on[n] = n < N ? 1.f : 0.f;
  }
  __syncthreads();

  int64_t m_rows = a.m;
  if (a.m_dev) m_rows = *a.m_dev;
  const int waves = blockDim.x >> 6;
  const int64_t n_blocks = (m_rows + 15) / 16, stride = (int64_t)gridDim.x * waves;
  const int nk = (KS + KC - 1) / KC;
  const bool n_full = N == NP;
  const float inv_n = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, 1.f / (float)N)));

  constexpr int VS = NB * 4 / 16 > 0 ? NB * 4 / 16 : 1;        // channels of a lane's 4 NB whose sums it keeps (ls_row_sums)
  float sums[NSUM ? NSUM : 1][VS];
#pragma unroll
  for (int s = 0; s < (NSUM ? NSUM : 1); ++s)
#pragma unroll
    for (int i = 0; i < VS; ++i) sums[s][i] = 0.f;
  const bool up[4] = {(lane & 8) != 0, (lane & 4) != 0, (lane & 2) != 0, (lane & 1) != 0};
  auto add_rows = [&](int s, float (&t)[NB * 4]) {
    ls_row_sums<NB * 4, 0>(t, up);
#pragma unroll
    for (int i = 0; i < VS; ++i) sums[s][i] += t[i];
  };

  // the block's rows from b0 on: this lane's row (a row past the end repeats the last one and is never stored), as bytes from the block's first row
  auto lane_row = [&](int64_t b) { return min(r16, (int)min((int64_t)15, m_rows - 1 - b * 16)); };
  uint4 xc[KC], xn[KC];
  auto load_x = [&](int64_t b, int kc, uint4 (&dst)[KC]) {
    if (DW) b = min(b, n_blocks - 1);                          // (in step: a wavefront may be past the last block)
    const char* base = reinterpret_cast<const char*>(a.x) + b * 16 * a.x_ld * ES + kc * (KC * 64);
    const uint32_t off = (uint32_t)lane_row(b) * (uint32_t)(a.x_ld * ES) + (XV ? q * 16 : 0);
#pragma unroll
    for (int s = 0; s < KC; ++s) {
      if constexpr (XV) {
        if (kc * KC + s < KS) dst[s] = *reinterpret_cast<const uint4*>(base + off + s * 64);
      } else {
        dst[s] = ls_load16<T>(reinterpret_cast<const T*>(base + off), s * (64 / ES) + q * E, K - kc * (KC * 64 / ES));
      }
    }
  };
  int64_t blk = (int64_t)blockIdx.x * waves + wave;
  // DW: stage rows, this wavefront's NW x KW blocks of dW
  constexpr int SP = 128 * ES + 32, SR = kLsDwWaves * 16, NW = DW ? NB / 2 : 1, KW = DW ? 4 : 1;
  char* stage_z = lds_t;
  char* stage_x = stage_z + SR * SP;
  const int dw_n = (wave & 1) * (NW * 16), dw_k = (wave >> 1) * (KW * 16);
  la_f32x4_t wacc[NW][KW];
#pragma unroll
  for (int i = 0; i < NW; ++i)
#pragma unroll
    for (int j = 0; j < KW; ++j) wacc[i][j] = la_f32x4_t{0.f, 0.f, 0.f, 0.f};
  // the residual's / the output gradient's 4 channels per lane and 16.  They arrive a whole turn ahead: the next block's are asked for as soon as this
  // block's are used (requested at the top of their own turn they held every wavefront up for most of HBM's latency)
  typename Raw4<T>::type rv[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) rv[nb] = typename Raw4<T>::type{};
  constexpr bool PAIR = ES == 2 && NV && NB > 1;
  constexpr bool PAIR_R = PAIR && !DW;                         // (in the fused gradient the swap comes in front of everything: 0.60 against 0.53 ms)
  constexpr bool AHEAD = VEC == 3 && !(ES == 4 && NB == 16);   // (256 f32 channels, or addresses per element: more registers than there are)
  auto load_r = [&](int64_t b) {
    if (!a.r) return;
    b = min(b, n_blocks - 1);
    const char* base = reinterpret_cast<const char*>(a.r) + b * 16 * a.r_ld * ES;
    const uint32_t row = (uint32_t)lane_row(b) * (uint32_t)(a.r_ld * ES), off = row + (NV ? q * 4 * ES : 0);
    int N_here = N;                                            // (compared here, not held as 16 masks for the whole loop)
    asm volatile("" : "+s"(N_here));
#pragma unroll
    for (int p = 0; p < NB; p += 2) {
      if constexpr (PAIR_R) {
        if ((p + 2) * 16 <= N_here) {
          const uint4 v = *reinterpret_cast<const uint4*>(base + row + (p * 16 + ls_pair_col(q)) * ES);
          rv[p] = make_uint2(v.x, v.y);
          rv[p + 1] = make_uint2(v.z, v.w);
          continue;
        }
      }
#pragma unroll
      for (int nb = p; nb < (p + 2 < NB ? p + 2 : NB); ++nb) {
        if constexpr (NV) {
          if (nb * 16 < N_here) rv[nb] = *reinterpret_cast<const typename Raw4<T>::type*>(base + off + nb * 16 * ES);
        } else {
          rv[nb] = ls_load4<T>(reinterpret_cast<const T*>(base + off), nb * 16 + q * 4, N);
        }
      }
    }
  };
  auto use_r = [&](int nb, float (&v)[4]) {                    // (called for nb = 0, 1, ..)
    if constexpr (PAIR_R) { if (nb % 2 == 0 && (nb + 2) * 16 <= N) ls_pair(rv[nb], rv[nb + 1 < NB ? nb + 1 : 0]); }
    ls_unpack4<T>(rv[nb], v);
  };
  if ((DW ? blk - wave : blk) < n_blocks) {
    load_x(blk, 0, xc);
    if constexpr (AHEAD) load_r(blk);
  }
  for (; (DW ? blk - wave : blk) < n_blocks; blk += stride) {
    const bool row_ok = r16 <= (int)min((int64_t)15, m_rows - 1 - blk * 16);
    if constexpr (DW) {
      if ((blk + 1) * 16 > m_rows) {                           // a repeated row's dz is zero; its x has to be as well: 0 * inf would be NaN
#pragma unroll
        for (int s = 0; s < KC; ++s) xc[s] = row_ok ? xc[s] : make_uint4(0u, 0u, 0u, 0u);
      }
      __syncthreads();                                         // the stage is read
#pragma unroll
      for (int s = 0; s < KC; ++s)
        *reinterpret_cast<uint4*>(stage_x + (wave * 16 + r16) * SP + s * 64 + q * 16) = s < KS ? xc[s] : make_uint4(0u, 0u, 0u, 0u);
    }
    // the parameters are read from LDS block after block: hoisted out of the loop they would take up to 96 registers
    asm volatile("" ::: "memory");
    int N_here = N;
    asm volatile("" : "+s"(N_here));
    if constexpr (!AHEAD) load_r(blk);
    if (BWD && (blk + 1) * 16 > m_rows) {                      // a repeated row adds nothing to the sums: its gradient is zero
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        rv[nb].x = row_ok ? rv[nb].x : 0u;
        rv[nb].y = row_ok ? rv[nb].y : 0u;
        if constexpr (ES == 4) { rv[nb].z = row_ok ? rv[nb].z : 0u; rv[nb].w = row_ok ? rv[nb].w : 0u; }
      }
    }
    la_f32x4_t acc[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) acc[nb] = *reinterpret_cast<const la_f32x4_t*>(lds_bias + nb * 16 + q * 4);
    for (int kc = 0; kc < nk; ++kc) {
      if constexpr (!DW) {
        if (kc + 1 < nk) load_x(blk, kc + 1, xn);
        else load_x(min(blk + stride, n_blocks - 1), 0, xn);
      }
      // (dz = gy without an activation: the fused gradient has no use for z)
#pragma unroll
      for (int s = 0; s < KC; ++s) {
        if (kc * KC + s < KS && !(DW && EPI == LS_DACT && a.act == kActNone)) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const uint4 fa = *reinterpret_cast<const uint4*>(lds_w + (nb * 16 + r16) * pitch + (kc * KC + s) * 64 + q * 16);
            acc[nb] = la_mfma<T>(fa, xc[s], acc[nb]);
          }
        }
      }
      if constexpr (DW) {                                      // (k <= 128: one step of the loop, the registers are free for the next block)
        load_x(blk + stride, 0, xc);
      } else {
#pragma unroll
        for (int s = 0; s < KC; ++s) xc[s] = xn[s];
      }
    }
    {
      float v[NB][4], rstd = 0.f;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[nb][e] = acc[nb][e];
      if constexpr (NORM) {                                    // v becomes xh; channels beyond N are zero throughout
        float s = 0.f, ss = 0.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) s += v[nb][e];
        const float mean = la_q_sum(s) * inv_n;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[nb][e] -= mean;
        if (!n_full) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[nb][e] *= lds_on[nb * 16 + q * 4 + e];
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) ss = fmaf(v[nb][e], v[nb][e], ss);
        rstd = 1.f / sqrtf(la_q_sum(ss) * inv_n + a.eps);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[nb][e] *= rstd;
      }
      // where this lane's channels of its row go: byte offset from the block's first row
      auto store_rows = [&](auto* rows, float (&val)[NB][4], int64_t width) {
        using O = std::remove_reference_t<decltype(*rows)>;
        char* base = reinterpret_cast<char*>(rows) + blk * 16 * width * (int64_t)sizeof(O);
        const uint32_t row = (uint32_t)r16 * (uint32_t)(width * sizeof(O));
#pragma unroll
        for (int nb = 0; nb < NB; nb += 2) {
          if constexpr (PAIR && sizeof(O) == 2) {
            if ((nb + 2) * 16 <= N_here) {
              uint2 lo = ls_pack4<T>(val[nb]), hi = ls_pack4<T>(val[nb + 1 < NB ? nb + 1 : nb]);
              ls_pair(lo, hi);                                 // (before the rows past the end drop out: every lane takes part)
              if (row_ok) *reinterpret_cast<uint4*>(base + row + (nb * 16 + ls_pair_col(q)) * 2) = make_uint4(lo.x, lo.y, hi.x, hi.y);
              continue;
            }
          }
#pragma unroll
          for (int i = 0; i < 2 && nb + i < NB; ++i) {
            const int n = (nb + i) * 16 + q * 4;
            if (row_ok && (NV ? (nb + i) * 16 : n) < N_here) la_store4<O>(reinterpret_cast<O*>(base + row + n * sizeof(O)), NV ? 4 : N - n, val[nb + i]);
          }
        }
      };
      // (channel block by channel block: whole-row arrays of intermediates do not fit beside the sums and the next block's x)
      if constexpr (!BWD) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int n = nb * 16 + q * 4;
          if constexpr (NORM) {
            const float4 g4 = *reinterpret_cast<const float4*>(lds_g + n), h4 = *reinterpret_cast<const float4*>(lds_h + n);
            v[nb][0] = fmaf(v[nb][0], g4.x, h4.x); v[nb][1] = fmaf(v[nb][1], g4.y, h4.y);
            v[nb][2] = fmaf(v[nb][2], g4.z, h4.z); v[nb][3] = fmaf(v[nb][3], g4.w, h4.w);
          }
          ro_act<P, 4>(v[nb], a.act);
          float r4[4];
          use_r(nb, r4);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[nb][e] += r4[e];
        }
        if constexpr (AHEAD) load_r(blk + stride);
        if (EPI == LS_ACT && a.out_f32) store_rows(reinterpret_cast<float*>(a.out), v, N);
        else store_rows(reinterpret_cast<T*>(a.out), v, N);
      } else {
        float d[NB][4], k1 = 0.f, k2 = 0.f;
        constexpr int GB = NB >= 8 ? 2 : 1;                    // channel blocks per activation switch
#pragma unroll
        for (int n0 = 0; n0 < NB; n0 += GB) {
#pragma unroll
          for (int i = 0; i < GB; ++i) use_r(n0 + i, d[n0 + i]);
          if (a.act != kActNone) {
            float z[GB][4];
#pragma unroll
            for (int i = 0; i < GB; ++i) {
              if constexpr (NORM) {
                const int n = (n0 + i) * 16 + q * 4;
                const float4 g4 = *reinterpret_cast<const float4*>(lds_g + n), h4 = *reinterpret_cast<const float4*>(lds_h + n);
                z[i][0] = fmaf(v[n0 + i][0], g4.x, h4.x); z[i][1] = fmaf(v[n0 + i][1], g4.y, h4.y);
                z[i][2] = fmaf(v[n0 + i][2], g4.z, h4.z); z[i][3] = fmaf(v[n0 + i][3], g4.w, h4.w);
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) z[i][e] = v[n0 + i][e];
              }
            }
            ro_act_slope<P, GB * 4>(reinterpret_cast<float(&)[GB * 4]>(d[n0]), reinterpret_cast<const float(&)[GB * 4]>(z), a.act);
          }
          if constexpr (NORM) {
#pragma unroll
            for (int i = 0; i < GB; ++i) {
              const float4 g4 = *reinterpret_cast<const float4*>(lds_g + (n0 + i) * 16 + q * 4);
              const float gv[4] = {g4.x, g4.y, g4.z, g4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float ev = d[n0 + i][e] * gv[e];
                k1 += ev;
                k2 = fmaf(ev, v[n0 + i][e], k2);
              }
            }
          }
        }
        if constexpr (NORM) {
          k1 = la_q_sum(k1) * inv_n;
          k2 = la_q_sum(k2) * inv_n;
          // (a repeated row's gy is zero: it adds nothing)
          float t[NB * 4];
#pragma unroll
          for (int i = 0; i < NB * 4; ++i) t[i] = d[i / 4][i % 4] * v[i / 4][i % 4];
          add_rows(0, t);
#pragma unroll
          for (int i = 0; i < NB * 4; ++i) t[i] = d[i / 4][i % 4];
          add_rows(NSUM > 1 ? 1 : 0, t);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int n = nb * 16 + q * 4;
          if constexpr (NORM) {
            const float4 g4 = *reinterpret_cast<const float4*>(lds_g + n);
            const float gv[4] = {g4.x, g4.y, g4.z, g4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) d[nb][e] = rstd * fmaf(-v[nb][e], k2, fmaf(d[nb][e], gv[e], -k1));
            if (!n_full) {
#pragma unroll
              for (int e = 0; e < 4; ++e) d[nb][e] *= lds_on[n + e];
            }
          }
        }
        {                                                      // (gy = 0 gives dz = 0 through the norm too)
          float t[NB * 4];
#pragma unroll
          for (int i = 0; i < NB * 4; ++i) t[i] = d[i / 4][i % 4];
          add_rows(NSUM ? NSUM - 1 : 0, t);
        }
        if constexpr (!DW) { if (a.out) store_rows(reinterpret_cast<T*>(a.out), d, N); }
        if constexpr (!DX && AHEAD) load_r(blk + stride);
        if constexpr (DX) {
          // dz as the operand of dz . W and dz^T x: step s of n = this lane's registers 2 s, 2 s + 1 (16-bit) or s (f32).  16-bit rows: dz is rounded to
          // their type here, the one rounding of these operators that is not an output's -- the matrix cores take 16-bit operands, and a second
          // term (dz - its rounding) would double the products of both gradients.  gx and gw are off by two independent roundings instead of one
          // (bf16, relative to 64 bits: 0.0024 for 0.0017; the plain formula with dz rounded agrees to 0.0002); the sums above are of the f32 values
          uint4 f[G::NS];
#pragma unroll
          for (int s = 0; s < G::NS; ++s) {
            if constexpr (ES == 4) {
              f[s] = make_uint4(__float_as_uint(d[s][0]), __float_as_uint(d[s][1]), __float_as_uint(d[s][2]), __float_as_uint(d[s][3]));
            } else {
              float t[8];
#pragma unroll
              for (int e = 0; e < 4; ++e) { t[e] = d[2 * s][e]; t[4 + e] = 2 * s + 1 < NB ? d[2 * s + 1 < NB ? 2 * s + 1 : 0][e] : 0.f; }
              f[s] = Vec16<T>::pack(t);
            }
          }
          if constexpr (AHEAD) load_r(blk + stride);           // (xh and dz have left their registers)
          if constexpr (DW) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              *reinterpret_cast<uint2*>(stage_z + (wave * 16 + r16) * SP + (nb * 16 + q * 4) * 2) =
                  nb & 1 ? make_uint2(f[nb / 2].z, f[nb / 2].w) : make_uint2(f[nb / 2].x, f[nb / 2].y);
            __syncthreads();                                   // the stage is written
            auto tr = [&](const char* stage, int ms, int col) {
              return ls_read_tr(stage + (ms * 32 + q * 8 + (r16 >> 2)) * SP + col * 2 + (r16 & 3) * 8, 4 * SP);
            };
#pragma unroll
            for (int ms = 0; ms < SR / 32; ++ms) {
              uint4 fz[NW];
#pragma unroll
              for (int i = 0; i < NW; ++i) fz[i] = tr(stage_z, ms, dw_n + i * 16);
#pragma unroll
              for (int j = 0; j < KW; ++j) {
                const uint4 fx = tr(stage_x, ms, dw_k + j * 16);
#pragma unroll
                for (int i = 0; i < NW; ++i) wacc[i][j] = la_mfma<T>(fz[i], fx, wacc[i][j]);
              }
            }
          }
          char* base = reinterpret_cast<char*>(a.gx) + blk * 16 * K * ES;
          const uint32_t row = (uint32_t)r16 * (uint32_t)(K * ES);
          const int kb_end = DW && !a.gx ? 0 : (K + 15) / 16;
          // 16-channel blocks at once: two where the norm's or 128 f32 channels' registers leave room for no more (f32 262144 x 96 -> 112 gradients
          // 261 us, with four 279; 1.05 M x 128 -> 128 1050, 1055)
          constexpr int KG = NORM || (ES == 4 && NB == 8) ? 2 : 4;
          for (int kg = 0; kg < kb_end; kg += KG) {
            la_f32x4_t o[KG];
#pragma unroll
            for (int t = 0; t < KG; ++t) o[t] = la_f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < G::NS; ++s)
#pragma unroll
              for (int t = 0; t < KG; ++t) {
                const int kb = min(kg + t, kb_end - 1);        // (a block past the end is formed again and not stored)
                uint4 fa;                                      // row k, and n in the order of f[s]
                if constexpr (ES == 4) fa = *reinterpret_cast<const uint4*>(lds_t + (kb * 16 + r16) * G::PITCH_T + s * 64 + q * 16);
                else fa = ls_read_tr(lds_w + (s * 32 + q * 4 + (r16 >> 2)) * pitch + kb * 32 + (r16 & 3) * 8, 16 * pitch);
                o[t] = la_mfma<T>(fa, f[s], o[t]);
              }
#pragma unroll
            for (int t = 0; t < KG; t += 2) {
              if constexpr (ES == 2 && NV) {
                if ((kg + t + 2) * 16 <= K) {
                  const float l4[4] = {o[t][0], o[t][1], o[t][2], o[t][3]}, h4[4] = {o[t + 1][0], o[t + 1][1], o[t + 1][2], o[t + 1][3]};
                  uint2 lo = ls_pack4<T>(l4), hi = ls_pack4<T>(h4);
                  ls_pair(lo, hi);
                  if (row_ok) *reinterpret_cast<uint4*>(base + row + ((kg + t) * 16 + ls_pair_col(q)) * 2) = make_uint4(lo.x, lo.y, hi.x, hi.y);
                  continue;
                }
              }
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int k = (kg + t + i) * 16 + q * 4;
                const float o4[4] = {o[t + i][0], o[t + i][1], o[t + i][2], o[t + i][3]};
                if (row_ok && k < K) la_store4<T>(reinterpret_cast<T*>(base + row + k * ES), NV ? 4 : K - k, o4);
              }
            }
          }
        }
      }
    }
  }
  if constexpr (NSUM > 0) {
    // lanes of a channel group -> wavefronts (in wave order) -> this workgroup's slab.  The buffer is W's place
    float* red = reinterpret_cast<float*>(smem);
    __syncthreads();
    constexpr int SAME = NB >= 4 ? 1 : 4 / NB;                 // (fewer than 16 values: so many lanes hold the same one)
    if (r16 % SAME == 0) {
#pragma unroll
      for (int i = 0; i < VS; ++i) {
        const int idx = r16 / SAME * VS + i;
#pragma unroll
        for (int t = 0; t < NSUM; ++t) red[(wave * NSUM + t) * NP + (idx >> 2) * 16 + q * 4 + (idx & 3)] = sums[t][i];
      }
    }
    __syncthreads();
    float* slab = a.slabs + (int64_t)blockIdx.x * a.slab_stride;
    for (int c = threadIdx.x; c < NSUM * NP; c += blockDim.x) {
      const int s = c / NP, n = c - s * NP;
      if (n >= N) continue;
      float t = 0.f;
      for (int w = 0; w < waves; ++w) t += red[(w * NSUM + s) * NP + n];
      slab[(int64_t)s * N + n] = t;
    }
    if constexpr (DW) {                                        // behind the sums: this workgroup's dW (n, k)
      float* dw = slab + (int64_t)NSUM * N;
#pragma unroll
      for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int j = 0; j < KW; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = dw_n + i * 16 + q * 4 + e, k = dw_k + j * 16 + r16;
            if (n < N && k < K) dw[(int64_t)n * K + k] = wacc[i][j][e];
          }
    }
  }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------------
constexpr int kLsLds = 158 * 1024;                             // a workgroup's share of the CU's 160 KB
constexpr int ls_nb(int64_t n) { return n <= 16 ? 1 : n <= 32 ? 2 : n <= 64 ? 4 : n <= 128 ? 8 : n <= 256 ? 16 : 0; }

template <typename T, int NB> static int ls_red(int k, int sums) {      // W, and at the end the wavefronts' sums in its place
  using G = LsGeom<T, NB>;
  return std::max(G::w_bytes(k), ls_wps(NB, LS_ACT, 3, sizeof(T)) * 4 * sums * G::NP * 4);
}
template <typename T, int NB> static int ls_lds(int k, int sums, bool dx, bool dw = false) {
  using G = LsGeom<T, NB>;
  return ls_red<T, NB>(k, sums) + G::param_bytes + (dx ? G::t_bytes(k) : 0) + (dw ? 2 * kLsDwWaves * 16 * (128 * (int)sizeof(T) + 32) : 0);
}
// bytes of LDS a launch over (k, n) needs (beyond kLsLds, or n beyond 256: the tiled product takes over)
template <typename T> static int ls_lds_any(int64_t k, int64_t n, int sums, bool dx, bool dw = false) {
  if (k > 4096) return INT32_MAX;
  switch (ls_nb(n)) {
    case 1: return ls_lds<T, 1>((int)k, sums, dx, dw);
    case 2: return ls_lds<T, 2>((int)k, sums, dx, dw);
    case 4: return ls_lds<T, 4>((int)k, sums, dx, dw);
    case 8: return ls_lds<T, 8>((int)k, sums, dx, dw);
    case 16: return ls_lds<T, 16>((int)k, sums, dx, dw);
  }
  return INT32_MAX;
}
// the fused weight gradient: 16-bit rows of up to 128 values on both sides
template <typename T> static bool ls_dw_fits(int64_t k, int64_t n, int sums) {
  return sizeof(T) == 2 && k <= 128 && (ls_nb(n) == 4 || ls_nb(n) == 8) && ls_lds_any<T>(k, n, sums, true, true) <= kLsLds / 2;
}

// channels of a streaming backward pass: beyond 128, xh, dz and the temporaries of the sums (f32: the rows themselves) do not fit a lane's registers
constexpr int ls_bwd_max(int norm, int elem_size) { return norm || elem_size == 4 ? 128 : 256; }
constexpr int kLsGrid = 1024;                                  // most workgroups of a launch (and slabs)

template <typename T, int NB, int EPI, bool DX, int VEC, bool DW = false> static int ls_go(LsArgs a, int* n_slabs, hipStream_t st) {
  constexpr int NSUM = EPI == LS_DNORM ? 3 : EPI == LS_DACT ? 1 : 0, WPS = ls_wps(NB, EPI, VEC, sizeof(T));
  const int lds = ls_lds<T, NB>(a.k, NSUM, DX, DW);
  a.red_bytes = ls_red<T, NB>(a.k, NSUM);
  static bool attr_set_dev[64] = {};
  bool& attr_set = per_device_flag(attr_set_dev);
  if (!attr_set) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&linear_stream_kernel<T, NB, EPI, DX, VEC, DW>), hipFuncAttributeMaxDynamicSharedMemorySize, kLsLds);
    if (e != hipSuccess) { set_error("linear_stream: cannot reserve %d B of LDS: %s", kLsLds, hipGetErrorString(e)); return PYGHO_ERR_LAUNCH; }
    attr_set = true;
  }
  // workgroups per CU: as many as LDS allows copies of W, the CU's 4 WPS wavefronts divided evenly among them.  With few rows, workgroups of 4
  // wavefronts, so that more CUs take part (not in a backward: its sums must not depend on the row count's upper bound)
  const int64_t blocks = ceil_div(a.m, 16);
  int per_cu = std::min(WPS, std::max(1, 160 * 1024 / lds));
  while (WPS * 4 % per_cu != 0) --per_cu;
  int waves = WPS * 4 / per_cu;
  if (DW) waves = kLsDwWaves;
  else if (NSUM == 0 && blocks < 256 * 4 * WPS) waves = std::min(waves, 4);
  const int grid = (int)std::min<int64_t>(ceil_div(blocks, waves), DW ? kLsDwGrid : 256 * per_cu);
  if (n_slabs) *n_slabs = grid;
  hipLaunchKernelGGL((linear_stream_kernel<T, NB, EPI, DX, VEC, DW>), dim3(grid), dim3(waves * kWave), lds, st, a);
  return check_launch("linear_stream");
}

// One 16-row block per wavefront and turn: the registers go to the epilogue and the prefetch; reading W's fragments costs 16 of the ~85 cycles that HBM
// takes per row at K = N = 128
template <typename T, int EPI, bool DX, int VEC> static int ls_pick_vec(const LsArgs& a, int* n_slabs, hipStream_t st) {
  switch (ls_nb(a.n)) {
    case 1: return ls_go<T, 1, EPI, DX, VEC>(a, n_slabs, st);
    case 2: return ls_go<T, 2, EPI, DX, VEC>(a, n_slabs, st);
    case 4: return ls_go<T, 4, EPI, DX, VEC>(a, n_slabs, st);
    case 8: return ls_go<T, 8, EPI, DX, VEC>(a, n_slabs, st);
    case 16:
      if constexpr (EPI == LS_ACT || EPI == LS_NORM || (EPI == LS_DACT && sizeof(T) == 2)) return ls_go<T, 16, EPI, DX, VEC>(a, n_slabs, st);
      break;                                                   // ls_bwd_max
  }
  set_error("linear_stream: %d channels", a.n);
  return PYGHO_ERR_UNSUPPORTED;
}
template <typename T, int EPI, bool DX> static int ls_pick(const LsArgs& a, int* n_slabs, hipStream_t st) {
  if (a.vec == 3) return ls_pick_vec<T, EPI, DX, 3>(a, n_slabs, st);
  return a.vec & 1 ? ls_pick_vec<T, EPI, DX, 1>(a, n_slabs, st) : ls_pick_vec<T, EPI, DX, 0>(a, n_slabs, st);
}
template <typename T, int EPI> static int ls_pick_dw(const LsArgs& a, int* n_slabs, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (ls_nb(a.n) == 4) return ls_go<T, 4, EPI, true, 3, true>(a, n_slabs, st);
    if (ls_nb(a.n) == 8) return ls_go<T, 8, EPI, true, 3, true>(a, n_slabs, st);
  }
  set_error("linear_stream: no fused weight gradient for %d channels", a.n);
  return PYGHO_ERR_UNSUPPORTED;
}

}  // namespace pygho
