// Layer norm over the channels of row-major (M, C) activations, with the MLP's activation and the layer's residual connection in the same
// pass (reference honn/utils.py:64-73 LayerNorm, :126-138 its place in the MLP; example/zinc.py:287-290 the residual):
//   mu = mean_c x,  v = mean_c (x - mu)^2,  xh = (x - mu) / sqrt(v + eps),  u = xh g + h,  y = act(u) + r
//   du = gy act'(u),  gg = sum_m du xh,  gh = sum_m du,  e = du g,  gx = (e - mean_c e - xh mean_c(e xh)) / sqrt(v + eps)
// ~10 / ~30 operations per element against 2..3 / 3 elements moved: both directions are bound by HBM, so each is ONE pass over its rows.
// A row lives in the registers of LPR lanes (NV vectors of VE elements each): the mean, the centred sum of squares (two passes over
// registers: no cancellation, however far the mean is from zero) and the two sums of the backward are lane-group sums.  The backward
// takes the statistics from x again instead of loading them: the row is in registers anyway.
// gg / gh: a lane keeps its channels' sums over all rows of its workgroup; workgroups write one slab each, a second launch adds the
// slabs in a fixed order.  Chunk k of the rows belongs to workgroup k % grid, so a slab depends on the true rows only: a launch sized for a
// capacity (m_dev: the count is on the device) gives the bits of an exactly sized one.
// Measured: bf16 1.83 M x 128 with residual 287 us forward (1.41 GB: 4.9 TB/s), 327 us backward (1.41 GB: 4.3 TB/s) + fold 6; f16 40531 x 1000
// forward 52 us (0.24 GB: 4.7 TB/s); f32 23719 x 193 (element by element) 14 + 18 + 5 us; f32 128 x 128 forward 4.8 us.
// 16-byte vectors where rows allow them, single elements otherwise: neighbouring lanes then still read neighbouring addresses
#include "row_ops.h"

namespace pygho {

constexpr int kLnFwdGrid = 256 * 8;      // 8 workgroups of 4 wavefronts per CU
constexpr int kLnBwdGrid = 256 * 4;      // every workgroup writes a slab of 2..3 C floats: half of that is enough to hide the loads

// statistics of a row held as U x NV x VE registers per lane (absent channels hold 0; they are masked in the centred sum)
template <int LPR, int NV, int VE>
__device__ __forceinline__ void ln_stats(float (&x)[NV][VE], const bool (&on)[NV], float inv_c, float eps, float& rstd) {
  float s = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int j = 0; j < VE; ++j) s += x[v][j];
  const float mean = ro_lane_sum<LPR>(s) * inv_c;
  float q = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      x[v][j] = on[v] ? x[v][j] - mean : 0.f;
      q = fmaf(x[v][j], x[v][j], q);
    }
  rstd = 1.f / sqrtf(ro_lane_sum<LPR>(q) * inv_c + eps);
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int j = 0; j < VE; ++j) x[v][j] *= rstd;       // x now holds xh
}

template <typename T, typename TX, int VE, int LPR, int NV, int U>
__global__ __launch_bounds__(kBlock) void ln_fwd_kernel(T* __restrict__ y, const TX* __restrict__ x, int64_t x_ld, const void* __restrict__ w,
                                                        const void* __restrict__ b, int pdt, const T* __restrict__ res, int64_t res_ld,
                                                        int64_t m, int c, float eps, int act) {
  constexpr bool P = Precise<T>::value;
  constexpr int GROUPS = kBlock / LPR, ROWS = GROUPS * U;
  const int lr = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const float inv_c = 1.f / (float)c;
  bool on[NV];
  float g[NV][VE], h[NV][VE];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int col = (v * LPR + lr) * VE;
    on[v] = col < c;
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      g[v][j] = on[v] ? ro_param(w, pdt, col + j, 1.f) : 0.f;
      h[v][j] = on[v] ? ro_param(b, pdt, col + j, 0.f) : 0.f;
    }
  }
  const int64_t n_chunks = (m + ROWS - 1) / ROWS;
  for (int64_t chunk = blockIdx.x; chunk < n_chunks; chunk += gridDim.x) {
    float xv[U][NV][VE], rv[U][NV][VE];
    int64_t row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      row[u] = chunk * ROWS + u * GROUPS + grp;
      const int64_t r = row[u] < m ? row[u] : m - 1;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int col = (v * LPR + lr) * VE;
#pragma unroll
        for (int j = 0; j < VE; ++j) { xv[u][v][j] = 0.f; rv[u][v][j] = 0.f; }
        if (on[v]) {
          ro_load<TX, VE>(x + r * x_ld + col, xv[u][v]);
          if (res) ro_load<T, VE>(res + r * res_ld + col, rv[u][v]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float rstd;
      ln_stats<LPR, NV, VE>(xv[u], on, inv_c, eps, rstd);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int j = 0; j < VE; ++j) xv[u][v][j] = fmaf(xv[u][v][j], g[v][j], h[v][j]);
        ro_act<P, VE>(xv[u][v], act);
#pragma unroll
        for (int j = 0; j < VE; ++j) xv[u][v][j] += rv[u][v][j];
        if (on[v] && row[u] < m) ro_store<T, VE>(y + row[u] * c + (v * LPR + lr) * VE, xv[u][v]);
      }
    }
  }
}

// NS = 2: slabs of (gg, gh); 3: (gg, gh, column sums of gx before their rounding: the bias gradient of a Linear in front of the norm);
// 1: no norm, gx = gy act'(x) and the column sums of gx (the gradient of a Linear's kept pre-activation)
template <typename T, typename TX, int VE, int LPR, int NV, int U, int NS>
__global__ __launch_bounds__(kBlock) void ln_bwd_kernel(T* __restrict__ gx, float* __restrict__ slabs, int64_t slab_stride, const TX* __restrict__ x,
                                                        int64_t x_ld, const T* __restrict__ gy, int64_t gy_ld, const void* __restrict__ w,
                                                        const void* __restrict__ b, int pdt, int64_t m, const int32_t* __restrict__ m_dev, int c,
                                                        float eps, int act) {
  constexpr bool P = Precise<T>::value;
  constexpr int GROUPS = kBlock / LPR, ROWS = GROUPS * U;
  __shared__ float red[kBlock * NV * VE];
  if (m_dev) m = *m_dev;
  const int lr = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const float inv_c = 1.f / (float)c;
  bool on[NV];
  float g[NV][VE], h[NV][VE], acc[NS][NV][VE];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int col = (v * LPR + lr) * VE;
    on[v] = col < c;
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      g[v][j] = on[v] ? ro_param(w, pdt, col + j, 1.f) : 0.f;
      h[v][j] = on[v] ? ro_param(b, pdt, col + j, 0.f) : 0.f;
#pragma unroll
      for (int s = 0; s < NS; ++s) acc[s][v][j] = 0.f;
    }
  }
  const int64_t n_chunks = (m + ROWS - 1) / ROWS;
  for (int64_t chunk = blockIdx.x; chunk < n_chunks; chunk += gridDim.x) {
    float xv[U][NV][VE], gv[U][NV][VE];
    int64_t row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      row[u] = chunk * ROWS + u * GROUPS + grp;
      const int64_t r = row[u] < m ? row[u] : m - 1;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int col = (v * LPR + lr) * VE;
#pragma unroll
        for (int j = 0; j < VE; ++j) { xv[u][v][j] = 0.f; gv[u][v][j] = 0.f; }
        if (on[v]) {
          ro_load<TX, VE>(x + r * x_ld + col, xv[u][v]);
          ro_load<T, VE>(gy + r * gy_ld + col, gv[u][v]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool valid = row[u] < m;
      float rstd, s1 = 0.f, s2 = 0.f;
      if constexpr (NS == 1) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          ro_act_slope<P, VE>(gv[u][v], xv[u][v], act);
#pragma unroll
          for (int j = 0; j < VE; ++j) acc[0][v][j] += valid ? gv[u][v][j] : 0.f;
          if (on[v] && valid) ro_store<T, VE>(gx + row[u] * c + (v * LPR + lr) * VE, gv[u][v]);
        }
        continue;
      }
      ln_stats<LPR, NV, VE>(xv[u], on, inv_c, eps, rstd);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (act != kActNone) {
          float z[VE];
#pragma unroll
          for (int j = 0; j < VE; ++j) z[j] = fmaf(xv[u][v][j], g[v][j], h[v][j]);
          ro_act_slope<P, VE>(gv[u][v], z, act);
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          if (valid) {                                     // (a row past the end repeats the last one: it must not count twice)
            acc[0][v][j] = fmaf(gv[u][v][j], xv[u][v][j], acc[0][v][j]);
            acc[NS > 1 ? 1 : 0][v][j] += gv[u][v][j];
          }
          gv[u][v][j] *= g[v][j];
          s1 += gv[u][v][j];
          s2 = fmaf(gv[u][v][j], xv[u][v][j], s2);
        }
      }
      const float k1 = ro_lane_sum<LPR>(s1) * inv_c, k2 = ro_lane_sum<LPR>(s2) * inv_c;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          gv[u][v][j] = rstd * (gv[u][v][j] - k1 - xv[u][v][j] * k2);
          if constexpr (NS == 3) { if (valid) acc[NS - 1][v][j] += gv[u][v][j]; }
        }
        if (on[v] && valid) ro_store<T, VE>(gx + row[u] * c + (v * LPR + lr) * VE, gv[u][v]);
      }
    }
  }
  // the workgroup's lane groups -> one slab row per sum, in group order
  float* slab = slabs + (int64_t)blockIdx.x * slab_stride;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    __syncthreads();
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < VE; ++j) red[grp * (LPR * NV * VE) + (v * LPR + lr) * VE + j] = acc[s][v][j];
    __syncthreads();
    for (int col = threadIdx.x; col < c; col += kBlock) {
      float a = 0.f;
      for (int k = 0; k < GROUPS; ++k) a += red[k * (LPR * NV * VE) + col];
      slab[(int64_t)s * c + col] = a;
    }
  }
}

// ---- rows that do not fit 64 lanes' registers: a workgroup per row, every pass over it from the cache ---------------------------
__device__ __forceinline__ float ln_block_sum(float v, float* lds) {
  v = ro_lane_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

template <typename T, typename TX, int VE>
__device__ __forceinline__ void ln_wide_stats(const TX* xr, int64_t c, float eps, float* lds, float& mean, float& rstd) {
  float s = 0.f, q = 0.f, t[VE];
  for (int64_t col = (int64_t)threadIdx.x * VE; col < c; col += kBlock * VE) {
    ro_load<TX, VE>(xr + col, t);
#pragma unroll
    for (int j = 0; j < VE; ++j) s += t[j];
  }
  mean = ln_block_sum(s, lds) / (float)c;
  for (int64_t col = (int64_t)threadIdx.x * VE; col < c; col += kBlock * VE) {
    ro_load<TX, VE>(xr + col, t);
#pragma unroll
    for (int j = 0; j < VE; ++j) q = fmaf(t[j] - mean, t[j] - mean, q);
  }
  rstd = 1.f / sqrtf(ln_block_sum(q, lds) / (float)c + eps);
}

template <typename T, typename TX, int VE>
__global__ __launch_bounds__(kBlock) void ln_fwd_wide_kernel(T* __restrict__ y, const TX* __restrict__ x, int64_t x_ld, const void* __restrict__ w,
                                                             const void* __restrict__ b, int pdt, const T* __restrict__ res, int64_t res_ld,
                                                             int64_t m, int64_t c, float eps, int act) {
  __shared__ float lds[4];
  for (int64_t row = blockIdx.x; row < m; row += gridDim.x) {
    const TX* xr = x + row * x_ld;
    float mean, rstd, t[VE], r[VE];
    ln_wide_stats<T, TX, VE>(xr, c, eps, lds, mean, rstd);
    for (int64_t col = (int64_t)threadIdx.x * VE; col < c; col += kBlock * VE) {
      ro_load<TX, VE>(xr + col, t);
#pragma unroll
      for (int j = 0; j < VE; ++j) t[j] = fmaf((t[j] - mean) * rstd, ro_param(w, pdt, col + j, 1.f), ro_param(b, pdt, col + j, 0.f));
      ro_act<Precise<T>::value, VE>(t, act);
      if (res) {
        ro_load<T, VE>(res + row * res_ld + col, r);
#pragma unroll
        for (int j = 0; j < VE; ++j) t[j] += r[j];
      }
      ro_store<T, VE>(y + row * c + col, t);
    }
  }
}

// the slab is the workgroup's running sum: every column of it belongs to one thread, the first row writes it, the later ones add
template <typename T, typename TX, int VE, int NS>
__global__ __launch_bounds__(kBlock) void ln_bwd_wide_kernel(T* __restrict__ gx, float* __restrict__ slabs, int64_t slab_stride, const TX* __restrict__ x,
                                                             int64_t x_ld, const T* __restrict__ gy, int64_t gy_ld, const void* __restrict__ w,
                                                             const void* __restrict__ b, int pdt, int64_t m, const int32_t* __restrict__ m_dev,
                                                             int64_t c, float eps, int act) {
  __shared__ float lds[4];
  if (m_dev) m = *m_dev;
  float* slab = slabs + (int64_t)blockIdx.x * slab_stride;
  bool first = true;
  for (int64_t row = blockIdx.x; row < m; row += gridDim.x, first = false) {
    const TX* xr = x + row * x_ld;
    const T* gr = gy + row * gy_ld;
    if constexpr (NS == 1) {
      for (int64_t col = (int64_t)threadIdx.x * VE; col < c; col += kBlock * VE) {
        float z[VE], t[VE];
        ro_load<TX, VE>(xr + col, z);
        ro_load<T, VE>(gr + col, t);
        ro_act_slope<Precise<T>::value, VE>(t, z, act);
#pragma unroll
        for (int j = 0; j < VE; ++j) slab[col + j] = (first ? 0.f : slab[col + j]) + t[j];
        ro_store<T, VE>(gx + row * c + col, t);
      }
      continue;
    }
    float mean, rstd, s1 = 0.f, s2 = 0.f, xh[VE], d[VE];
    ln_wide_stats<T, TX, VE>(xr, c, eps, lds, mean, rstd);
    auto load_du = [&](int64_t col) {
      ro_load<TX, VE>(xr + col, xh);
      ro_load<T, VE>(gr + col, d);
      float z[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        xh[j] = (xh[j] - mean) * rstd;
        z[j] = fmaf(xh[j], ro_param(w, pdt, col + j, 1.f), ro_param(b, pdt, col + j, 0.f));
      }
      ro_act_slope<Precise<T>::value, VE>(d, z, act);
    };
    for (int64_t col = (int64_t)threadIdx.x * VE; col < c; col += kBlock * VE) {
      load_du(col);
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        float* p = slab + col + j;
        const float a = first ? 0.f : p[0], bb = first ? 0.f : p[c];
        p[0] = fmaf(d[j], xh[j], a);
        p[c] = bb + d[j];
        const float e = d[j] * ro_param(w, pdt, col + j, 1.f);
        s1 += e;
        s2 = fmaf(e, xh[j], s2);
      }
    }
    const float k1 = ln_block_sum(s1, lds) / (float)c, k2 = ln_block_sum(s2, lds) / (float)c;
    for (int64_t col = (int64_t)threadIdx.x * VE; col < c; col += kBlock * VE) {
      load_du(col);
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        d[j] = rstd * (d[j] * ro_param(w, pdt, col + j, 1.f) - k1 - xh[j] * k2);
        if constexpr (NS == 3) {
          float* p = slab + 2 * c + col + j;
          p[0] = (first ? 0.f : p[0]) + d[j];
        }
      }
      ro_store<T, VE>(gx + row * c + col, d);
    }
  }
  if (first)                                               // no row of the true count fell to this workgroup
    for (int64_t col = threadIdx.x; col < NS * c; col += kBlock) slab[col] = 0.f;
}

// ---- slabs -> sums in a fixed order: 4 lanes x 4 columns by 64 slab lanes, lane t adds slabs t, t + 64, .., the 64 lanes a tree.  The order
// does not depend on the slab count, so trailing slabs of zeros change nothing.  64 slab lanes: a fold of a few hundred columns is a
// handful of workgroups, and with 16 the serial loads of one lane took longer than everything else --------------------------------
__global__ __launch_bounds__(kBlock) void fold_partials_kernel(FoldOut out, const float* __restrict__ slabs, int64_t n_slabs, int64_t stride,
                                                               int64_t width) {
  __shared__ float4 red[64][4];
  const int cx = threadIdx.x & 3, sx = threadIdx.x >> 2;
  const int64_t col = ((int64_t)blockIdx.x * 4 + cx) * 4;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < width) {
    const float* p = slabs + col;
#pragma unroll 8
    for (int64_t s = sx; s < n_slabs; s += 64) {
      const float4 v = *reinterpret_cast<const float4*>(p + s * stride);     // (stride is a multiple of 4: the tail stays inside the slab)
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
  }
  red[sx][cx] = a;
  for (int half = 32; half > 0; half >>= 1) {
    __syncthreads();
    if (sx < half) {
      const float4 v = red[sx + half][cx];
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
      red[sx][cx] = a;
    }
  }
  if (sx != 0 || col >= width) return;
  const float r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int64_t i = col + j;
    if (i >= width) break;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i < out.len[k]) {
        if (out.p[k]) ro_store_param(out.p[k], out.dt[k], i, r[j]);
        break;
      }
      i -= out.len[k];
    }
  }
}

// ---- launch shapes ------------------------------------------------------------------------------------------------------------------
// Vectors of 16 bytes need every row of every operand on a 16-byte boundary and a width of whole vectors; anything else goes element by
// element (still coalesced).  Lanes per row: the fewest that hold it, so that a narrow row does not idle a wavefront.  Beyond 64 lanes x 32
// (vectors) or x 16 (elements) registers the workgroup-per-row kernels take over.
struct LnShape { int ve; int lpr; int nv; bool wide; };
static LnShape ln_shape(int64_t c, int vec_elems, bool vec) {
  const int ve = vec ? vec_elems : 1;
  const int64_t n = (c + ve - 1) / ve;
  LnShape s{ve, 4, 1, false};
  while (s.lpr < 64 && s.lpr < n) s.lpr *= 2;
  while ((int64_t)s.lpr * s.nv < n) s.nv *= 2;
  const int most = !vec ? 16 : vec_elems == 8 ? 4 : 8;
  s.wide = s.nv > most;
  return s;
}
// rows in flight per lane group: two while a row is at most 16 registers of a lane, one beyond
static constexpr int ln_unroll(int regs) { return regs <= 4 ? 4 : regs <= 16 ? 2 : 1; }

struct LnFwd {
  void* y; const void* x; int64_t x_ld; const void* w; const void* b; int pdt; const void* res; int64_t res_ld; int64_t m; int64_t c;
  float eps; int act; hipStream_t st;
};
struct LnBwd {
  void* gx; float* slabs; int64_t stride; int* n_slabs; const void* x; int64_t x_ld; const void* gy; int64_t gy_ld; const void* w; const void* b;
  int pdt; int64_t m; const int32_t* m_dev; int64_t c; float eps; int act; hipStream_t st;
};

template <typename T, typename TX, int VE, int LPR, int NV> static int ln_go(const LnFwd& a) {
  constexpr int U = ln_unroll(NV * VE);
  const int grid = grid_for(a.m, kBlock / LPR * U, kLnFwdGrid);
  hipLaunchKernelGGL((ln_fwd_kernel<T, TX, VE, LPR, NV, U>), dim3(grid), dim3(kBlock), 0, a.st, (T*)a.y, (const TX*)a.x, a.x_ld, a.w, a.b, a.pdt,
                     (const T*)a.res, a.res_ld, a.m, (int)a.c, a.eps, a.act);
  return check_launch("layer_norm_act");
}
template <typename T, typename TX, int VE, int LPR, int NV, int NS> static int ln_go(const LnBwd& a) {
  constexpr int U = ln_unroll(NV * VE);
  *a.n_slabs = grid_for(a.m, kBlock / LPR * U, kLnBwdGrid);
  hipLaunchKernelGGL((ln_bwd_kernel<T, TX, VE, LPR, NV, U, NS>), dim3(*a.n_slabs), dim3(kBlock), 0, a.st, (T*)a.gx, a.slabs, a.stride, (const TX*)a.x,
                     a.x_ld, (const T*)a.gy, a.gy_ld, a.w, a.b, a.pdt, a.m, a.m_dev, (int)a.c, a.eps, a.act);
  return check_launch("layer_norm_act_bwd");
}

template <typename T, typename TX, int VE, int NS, typename A> static int ln_pick(const LnShape& s, const A& a) {
#define PYGHO_LN(L, N)                                                              \
  if (s.lpr == L && s.nv == N) {                                                    \
    if constexpr (NS == 0) return ln_go<T, TX, VE, L, N>(a);                        \
    else return ln_go<T, TX, VE, L, N, NS>(a);                                      \
  }
  PYGHO_LN(4, 1) PYGHO_LN(8, 1) PYGHO_LN(16, 1) PYGHO_LN(32, 1) PYGHO_LN(64, 1) PYGHO_LN(64, 2) PYGHO_LN(64, 4)
  if constexpr (VE <= 4) { PYGHO_LN(64, 8) }
  if constexpr (VE == 1) { PYGHO_LN(64, 16) }
#undef PYGHO_LN
  set_error("layer_norm_act: no launch shape");
  return PYGHO_ERR_UNSUPPORTED;
}

static bool ln_vec(int64_t c, int es, const void* const* ptrs, const int64_t* lds, const int* esz, int n) {
  if ((c * es) % 16 != 0) return false;
  for (int i = 0; i < n; ++i)
    if (ptrs[i] && (((uintptr_t)ptrs[i] | (uint64_t)(lds[i] * esz[i])) % 16) != 0) return false;
  return true;
}

template <typename T, typename TX> static int ln_fwd_typed(const LnFwd& a) {
  constexpr int VE = Vec16<T>::N;
  const void* ptrs[] = {a.y, a.x, a.res};
  const int64_t lds[] = {a.c, a.x_ld, a.res_ld};
  const int esz[] = {(int)sizeof(T), (int)sizeof(TX), (int)sizeof(T)};
  const bool vec = ln_vec(a.c, sizeof(T), ptrs, lds, esz, 3);
  const LnShape s = ln_shape(a.c, VE, vec);
  if (!s.wide) return vec ? ln_pick<T, TX, VE, 0>(s, a) : ln_pick<T, TX, 1, 0>(s, a);
  const dim3 grid(grid_for(a.m, 1, kLnFwdGrid)), block(kBlock);
  if (vec)
    hipLaunchKernelGGL((ln_fwd_wide_kernel<T, TX, VE>), grid, block, 0, a.st, (T*)a.y, (const TX*)a.x, a.x_ld, a.w, a.b, a.pdt, (const T*)a.res,
                       a.res_ld, a.m, a.c, a.eps, a.act);
  else
    hipLaunchKernelGGL((ln_fwd_wide_kernel<T, TX, 1>), grid, block, 0, a.st, (T*)a.y, (const TX*)a.x, a.x_ld, a.w, a.b, a.pdt, (const T*)a.res,
                       a.res_ld, a.m, a.c, a.eps, a.act);
  return check_launch("layer_norm_act");
}

template <typename T, typename TX, int NS> static int ln_bwd_typed(const LnBwd& a) {
  constexpr int VE = Vec16<T>::N;
  const void* ptrs[] = {a.gx, a.x, a.gy};
  const int64_t lds[] = {a.c, a.x_ld, a.gy_ld};
  const int esz[] = {(int)sizeof(T), (int)sizeof(TX), (int)sizeof(T)};
  const bool vec = ln_vec(a.c, sizeof(T), ptrs, lds, esz, 3);
  const LnShape s = ln_shape(a.c, VE, vec);
  if (!s.wide) return vec ? ln_pick<T, TX, VE, NS>(s, a) : ln_pick<T, TX, 1, NS>(s, a);
  *a.n_slabs = grid_for(a.m, 1, kLnBwdGrid);
  const dim3 grid(*a.n_slabs), block(kBlock);
  if (vec)
    hipLaunchKernelGGL((ln_bwd_wide_kernel<T, TX, VE, NS>), grid, block, 0, a.st, (T*)a.gx, a.slabs, a.stride, (const TX*)a.x, a.x_ld, (const T*)a.gy,
                       a.gy_ld, a.w, a.b, a.pdt, a.m, a.m_dev, a.c, a.eps, a.act);
  else
    hipLaunchKernelGGL((ln_bwd_wide_kernel<T, TX, 1, NS>), grid, block, 0, a.st, (T*)a.gx, a.slabs, a.stride, (const TX*)a.x, a.x_ld, (const T*)a.gy,
                       a.gy_ld, a.w, a.b, a.pdt, a.m, a.m_dev, a.c, a.eps, a.act);
  return check_launch("layer_norm_act_bwd");
}

bool ro_float(int dtype) { return dtype == PYGHO_F32 || dtype == PYGHO_BF16 || dtype == PYGHO_F16; }

}  // namespace pygho

using namespace pygho;

static int ln_check(const char* what, const void* a, const void* b, int64_t m, int64_t c, double eps, int act, int dtype, int x_dtype, int param_dtype) {
  if (m < 0 || c <= 0 || c > INT32_MAX / 2) { set_error("%s: bad size", what); return PYGHO_ERR_INVALID; }
  if (!ro_float(dtype) || !(x_dtype == dtype || x_dtype == PYGHO_F32) || !(param_dtype == dtype || param_dtype == PYGHO_F32)) {
    set_error("%s: f32 / bf16 / f16 rows, input and parameters in the same type or f32", what);
    return PYGHO_ERR_UNSUPPORTED;
  }
  if (act < 0 || act > kActElu) { set_error("%s: unknown activation %d", what, act); return PYGHO_ERR_INVALID; }
  if (!(eps >= 0.0)) { set_error("%s: eps must not be negative", what); return PYGHO_ERR_INVALID; }
  if (m > 0 && (!a || !b)) { set_error("null pointer"); return PYGHO_ERR_INVALID; }
  return PYGHO_OK;
}

extern "C" int pygho_layer_norm_act(void* y, const void* x, int64_t x_ld, const void* weight, const void* bias, int param_dtype, const void* residual,
                                    int64_t residual_ld, int64_t m, int64_t c, double eps, int act, int dtype, void* stream) {
  if (int rc = ln_check("layer_norm_act", y, x, m, c, eps, act, dtype, dtype, param_dtype)) return rc;
  if (m == 0) return PYGHO_OK;
  return ln_fwd_launch(y, x, x_ld, weight, bias, param_dtype, residual, residual_ld, m, c, (float)eps, act, dtype, dtype, (hipStream_t)stream);
}

int pygho::ln_fwd_launch(void* y, const void* x, int64_t x_ld, const void* weight, const void* bias, int param_dtype, const void* residual,
                         int64_t residual_ld, int64_t m, int64_t c, float eps, int act, int dtype, int x_dtype, hipStream_t st) {
  const LnFwd a{y, x, x_ld, weight, bias, param_dtype, residual, residual_ld, m, c, eps, act, st};
  if (dtype == PYGHO_F32) return ln_fwd_typed<float, float>(a);
  if (dtype == PYGHO_BF16) return x_dtype == PYGHO_F32 ? ln_fwd_typed<bf16, float>(a) : ln_fwd_typed<bf16, bf16>(a);
  return x_dtype == PYGHO_F32 ? ln_fwd_typed<f16, float>(a) : ln_fwd_typed<f16, f16>(a);
}

// ---- backward: rows and slabs in one launch, the fold in a second; both on the caller's workspace ------------------------------------
namespace pygho {

int64_t ln_bwd_slab_floats(int64_t m, int64_t c, int sums) {
  return m <= 0 ? 0 : (int64_t)grid_for(m, 1, kLnBwdGrid) * ((sums * c + 3) / 4 * 4);
}

int ln_bwd_launch(void* gx, float* slabs, int64_t* stride, int* n_slabs, int sums, const void* x, int64_t x_ld, const void* gy, int64_t gy_ld,
                  const void* weight, const void* bias, int param_dtype, int64_t m, const int32_t* m_dev, int64_t c, float eps, int act, int dtype,
                  int x_dtype, hipStream_t st) {
  *stride = (sums * c + 3) / 4 * 4;
  const LnBwd a{gx, slabs, *stride, n_slabs, x, x_ld, gy, gy_ld, weight, bias, param_dtype, m, m_dev, c, eps, act, st};
#define PYGHO_LNB(T, TX) (sums == 3 ? ln_bwd_typed<T, TX, 3>(a) : sums == 2 ? ln_bwd_typed<T, TX, 2>(a) : ln_bwd_typed<T, TX, 1>(a))
  if (dtype == PYGHO_F32) return PYGHO_LNB(float, float);
  if (dtype == PYGHO_BF16) return x_dtype == PYGHO_F32 ? PYGHO_LNB(bf16, float) : PYGHO_LNB(bf16, bf16);
  return x_dtype == PYGHO_F32 ? PYGHO_LNB(f16, float) : PYGHO_LNB(f16, f16);
#undef PYGHO_LNB
}

int fold_launch(const FoldOut& o, const float* slabs, int64_t n_slabs, int64_t stride, hipStream_t st) {
  int64_t width = 0;
  for (int k = 0; k < 4; ++k) width += o.len[k];
  if (width == 0) return PYGHO_OK;
  const int64_t grid = ceil_div(width, 16);
  if (grid > INT32_MAX) { set_error("fold_partials: too wide"); return PYGHO_ERR_UNSUPPORTED; }
  hipLaunchKernelGGL(fold_partials_kernel, dim3((unsigned)grid), dim3(kBlock), 0, st, o, slabs, n_slabs, stride, width);
  return check_launch("fold_partials");
}

}  // namespace pygho

extern "C" size_t pygho_layer_norm_act_bwd_workspace(int64_t m, int64_t c) { return m <= 0 || c <= 0 ? 0 : (size_t)ln_bwd_slab_floats(m, c, 2) * 4; }

extern "C" int pygho_layer_norm_act_bwd(void* gx, void* gweight, int gweight_dtype, void* gbias, int gbias_dtype, const void* x, int64_t x_ld,
                                        const void* gy, int64_t gy_ld, const void* weight, const void* bias, int param_dtype, int64_t m_cap,
                                        const int32_t* m_dev, int64_t c, double eps, int act, int dtype, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  if (int rc = ln_check("layer_norm_act_bwd", gx, x, m_cap, c, eps, act, dtype, dtype, param_dtype)) return rc;
  if ((gweight && !ro_float(gweight_dtype)) || (gbias && !ro_float(gbias_dtype))) { set_error("layer_norm_act_bwd: gradient dtype"); return PYGHO_ERR_UNSUPPORTED; }
  if (m_cap > 0 && (!gy || !workspace)) { set_error("null pointer"); return PYGHO_ERR_INVALID; }
  if (workspace_bytes < pygho_layer_norm_act_bwd_workspace(m_cap, c) || (uintptr_t)workspace % 16 != 0) {
    set_error("layer_norm_act_bwd: workspace too small or not 16-byte aligned");
    return PYGHO_ERR_INVALID;
  }
  hipStream_t st = (hipStream_t)stream;
  float* slabs = reinterpret_cast<float*>(workspace);
  int64_t stride = (2 * c + 3) / 4 * 4;
  int n = 0;
  if (m_cap > 0) {
    if (int rc = ln_bwd_launch(gx, slabs, &stride, &n, 2, x, x_ld, gy, gy_ld, weight, bias, param_dtype, m_cap, m_dev, c, (float)eps, act, dtype, dtype, st)) return rc;
  }
  if (!gweight && !gbias) return PYGHO_OK;
  return fold_launch(FoldOut{{gweight, gbias, nullptr, nullptr}, {c, c, 0, 0}, {gweight_dtype, gbias_dtype, 0, 0}}, slabs, n, stride, st);
}
