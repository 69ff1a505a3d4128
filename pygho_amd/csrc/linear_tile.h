// Tiled product behind the linear operators where W does not fit a CU's LDS (linear_stream.h is the other form), and for the weight
// gradient, whose long dimension is the reduction.  Any width, row stride, alignment, f32 / bf16 / f16.
// Output element (m, n) = sum_k P(m, k) Q(n, k); an operand is stored with its k contiguous ("rows": x and W of the forward, dz of dX) or
// with its m / n contiguous ("columns": dz and x of dW; dX takes W's transposed copy, which costs less than reading it transposed tile by tile).  A step of the k loop moves 128 bytes of k per row (64 16-bit or 32 f32
// values) global -> registers -> LDS, one step ahead of the matrix instructions.  The MFMA runs in the swapped form D[n][m]: a lane holds one
// row m and 4 consecutive n, which it stores as one vector.
// Column operands stay in their storage order in LDS; 16-bit fragments are read back transposed by the LDS itself (ds_read_b64_tr_b16),
// f32 ones element by element (conflict-free, and an f32 MFMA takes 32 cycles).
// f32 products run on v_mfma_f32_16x16x4f32: true f32, no reduced-precision path.
// Measured, bf16 65536 x 512 -> 512: forward 66 us with a 16-bit pre-activation stored, 87 with an f32 one (34 GFLOP: 520 / 390 TFLOP/s, bound by the wait for a
// step's loads at one workgroup per CU), weight gradient 85 us (400 TFLOP/s)
#pragma once
#include "row_ops.h"

namespace pygho {

typedef __attribute__((ext_vector_type(8))) __bf16 la_bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 la_f16x8_t;
typedef __attribute__((ext_vector_type(4))) float la_f32x4_t;
typedef __attribute__((ext_vector_type(4))) short la_s4_t;

enum { LA_ROWS = 0, LA_COLS = 1 };
// epilogues: bias, activation, residual, one store (the pre-activation beside it if asked); f32 slab of a split product
enum { LA_ACT = 0, LA_SLAB = 4 };

struct LaOperand { const void* p; int64_t ld; };

struct LaArgs {
  LaOperand a, b;                     // P (m, k), Q (n, k)
  int64_t m; int64_t n; int64_t k;    // LA_SLAB: k may be an upper bound of the reduction, LA_ACT: m one of the rows (dev: the true count)
  const int32_t* dev;
  void* out;                          // nullable: only z
  void* z; int z_f32;                 // nullable: the pre-activation, in the storage type or in f32
  const void* bias; int bias_dtype;
  const void* res; int64_t res_ld;
  int act;
  float* slabs; int64_t slab_stride; int splits;      // LA_SLAB: slab s = [m * n product | m column sums (want_sums)]
  int want_sums;
};

// 16 or 8 bytes at any element's address.  gfx950 loads and stores vectors from there in one instruction (a packed type makes the compiler use it),
// so odd widths and strides need no path of their own: what is left is the ragged end of a row
template <typename V, typename T> struct __attribute__((packed, aligned(sizeof(T)))) LaAny { uint32_t w[sizeof(V) / 4]; };
template <typename V, typename T> __device__ __forceinline__ V la_ld(const T* p) { return __builtin_bit_cast(V, *reinterpret_cast<const LaAny<V, T>*>(p)); }
template <typename V, typename T> __device__ __forceinline__ void la_st(T* p, const V& v) { *reinterpret_cast<LaAny<V, T>*>(p) = __builtin_bit_cast(LaAny<V, T>, v); }

// one step of k (64 bytes per row): bf16 / f16 one 16x16x32 MFMA, f32 four 16x16x4 (element j of every lane's 4 is k = 4 q + j on both sides)
template <typename T> __device__ __forceinline__ la_f32x4_t la_mfma(const uint4& a, const uint4& b, la_f32x4_t c) {
  if constexpr (std::is_same<T, bf16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(la_bf16x8_t, a), __builtin_bit_cast(la_bf16x8_t, b), c, 0, 0, 0);
  } else if constexpr (std::is_same<T, f16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(la_f16x8_t, a), __builtin_bit_cast(la_f16x8_t, b), c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
}
template <typename T> __device__ __forceinline__ uint4 la_ones() {
  if constexpr (std::is_same<T, bf16>::value) return make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  if constexpr (std::is_same<T, f16>::value) return make_uint4(0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u);
  return make_uint4(0x3f800000u, 0x3f800000u, 0x3f800000u, 0x3f800000u);
}
__device__ __forceinline__ float la_q_sum(float v) {     // over the 4 lanes of a row: q = lane / 16
  auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
  r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

// geometry of an operand tile of R rows x 128 bytes of k in LDS
template <typename T, int MODE, int R, int THREADS> struct LaTile {
  static constexpr int ES = sizeof(T);
  static constexpr int KE = 128 / ES;                                            // k values per step of the loop
  // + 16 bytes per row: the 16 rows of a fragment read fall on different banks.  Columns: + 32 (16-bit: the 4 k rows of a transposed read)
  // or + 16 bytes (f32: the 4 k rows of a wavefront's element reads)
  static constexpr int PITCH = MODE == LA_ROWS ? 128 + 16 : R * ES + (ES == 2 ? 32 : 16);
  static constexpr int BYTES = MODE == LA_ROWS ? R * PITCH : KE * PITCH;
  static constexpr int CHUNKS = R * 8;                                           // 16-byte chunks per step
  static constexpr int PER_THREAD = (CHUNKS + THREADS - 1) / THREADS;
  static constexpr int CPR = MODE == LA_ROWS ? 8 : R * ES / 16;                  // chunks per LDS row

  // chunk `i` of this thread: rows [r0, r0 + R) x k [k0, k0 + KE) of the operand; everything outside (n_rows, k_end) is zero
  static __device__ __forceinline__ uint4 load(const LaOperand& op, int64_t r0, int64_t n_rows, int64_t k0, int64_t k_end, int i) {
    constexpr int E = 16 / ES;
    const int c = i * THREADS + (int)threadIdx.x;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (CHUNKS % THREADS != 0 && c >= CHUNKS) return v;
    const int lr = c / CPR, lc = c % CPR;
    const T* base = reinterpret_cast<const T*>(op.p);
    // `outer` runs over LDS rows, `inner` is the contiguous direction
    const int64_t outer = MODE == LA_ROWS ? r0 + lr : k0 + lr, outer_end = MODE == LA_ROWS ? n_rows : k_end;
    const int64_t inner = (MODE == LA_ROWS ? k0 : r0) + lc * E, inner_end = MODE == LA_ROWS ? k_end : n_rows;
    if (outer >= outer_end || inner >= inner_end) return v;
    const T* p = base + outer * op.ld + inner;
    if (inner + E <= inner_end) return la_ld<uint4>(p);
    const int left = (int)min((int64_t)E, inner_end - inner);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (ES == 4) {
        w[j] = j < left ? reinterpret_cast<const uint32_t*>(p)[j] : 0u;
      } else {
        const uint32_t lo = 2 * j < left ? reinterpret_cast<const uint16_t*>(p)[2 * j] : 0u;
        const uint32_t hi = 2 * j + 1 < left ? reinterpret_cast<const uint16_t*>(p)[2 * j + 1] : 0u;
        w[j] = lo | (hi << 16);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // whole steps of k (FULL): one uniform base and 32-bit offsets; a row past the end repeats the last one (its products are not stored)
  static __device__ __forceinline__ uint4 load_full(const LaOperand& op, int64_t r0, int64_t n_rows, int64_t k0, int i) {
    static_assert(MODE == LA_ROWS && CHUNKS % THREADS == 0, "row operands");
    const char* base = reinterpret_cast<const char*>(op.p) + (r0 * op.ld + k0) * ES;
    const int last = (int)min((int64_t)(R - 1), n_rows - 1 - r0);
    return la_ld<uint4>(reinterpret_cast<const T*>(base + (uint32_t)min(i * (THREADS / 8) + (int)threadIdx.x / 8, last) * (uint32_t)(op.ld * ES) +
                                                   ((int)threadIdx.x % 8) * 16));
  }
  static __device__ __forceinline__ void store(char* lds, const uint4& v, int i) {
    const int c = i * THREADS + (int)threadIdx.x;
    if (CHUNKS % THREADS != 0 && c >= CHUNKS) return;
    *reinterpret_cast<uint4*>(lds + (c / CPR) * PITCH + (c % CPR) * 16) = v;
  }
  // the lane's 16 bytes of k of row `row0 + lane % 16` in half-step ks (0, 1)
  static __device__ __forceinline__ uint4 frag(const char* lds, int row0, int ks, int r16, int q) {
    if constexpr (MODE == LA_ROWS) {
      return *reinterpret_cast<const uint4*>(lds + (row0 + r16) * PITCH + ks * 64 + q * 16);
    } else if constexpr (ES == 2) {
      const char* p = lds + (ks * 32 + q * 8 + (r16 >> 2)) * PITCH + row0 * 2 + (r16 & 3) * 8;
      const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) la_s4_t*)p));
      const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) la_s4_t*)(p + 4 * PITCH)));
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    } else {
      const char* p = lds + (ks * 16 + q * 4) * PITCH + (row0 + r16) * 4;
      return make_uint4(*reinterpret_cast<const uint32_t*>(p), *reinterpret_cast<const uint32_t*>(p + PITCH),
                        *reinterpret_cast<const uint32_t*>(p + 2 * PITCH), *reinterpret_cast<const uint32_t*>(p + 3 * PITCH));
    }
  }
};

constexpr int kLaChunk = 128;         // rows of a split product's reduction per chunk: chunk j belongs to split j % splits

// 4 consecutive elements (of row m, from n) <-> registers, `left` of them in the row
template <typename T> __device__ __forceinline__ void la_load4(const T* p, int left, float (&v)[4]) {
  if (left >= 4) {
    if constexpr (sizeof(T) == 4) {
      const uint4 r = la_ld<uint4>(p);
      v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
    } else {
      const uint2 r = la_ld<uint2>(p);
      float t[8];
      Vec16<T>::unpack(make_uint4(r.x, r.y, 0u, 0u), t);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = t[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? load_as_acc<T>(p + i) : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void la_store4(T* p, int left, const float (&v)[4]) {
  if (left >= 4) {
    if constexpr (sizeof(T) == 4) {
      la_st(p, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
    } else {
      const float t[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
      const uint4 r = Vec16<T>::pack(t);
      la_st(p, make_uint2(r.x, r.y));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i < left) store_from_acc<T>(p + i, v[i]);
  }
}

// A pre-activation on its way into 16-bit storage (a caller's choice: rowops.py keeps it in f32).  A finite one beyond the type's range becomes the
// type's largest value: as an infinity it would make silu's slope inf * 0 = NaN, where f32 gives 0 or 1 (f16 reaches 65504).  Infinities and NaN stay
template <typename T> __device__ __forceinline__ float la_in_range(float v) {
  constexpr float most = std::is_same<T, f16>::value ? 65504.f : std::is_same<T, bf16>::value ? 3.38953139e38f : 3.40282347e38f;
  return fabsf(v) <= 3.40282347e38f ? fminf(fmaxf(v, -most), most) : v;
}

// a workgroup of WM x WN wavefronts forms BM x BN output tiles.  Two wavefronts per SIMD at least: left alone, the 128 x 128 tile took 259 registers
// and had one (bf16 forward 65536 x 500 -> 500 163 us, with two 92 .. 103)
template <typename T, int MA, int MB, int BM, int BN, int WM, int WN, int EPI, bool FULL = false>
__global__ __launch_bounds__(WM * WN * 64, 2) void linear_tile_kernel(LaArgs g) {
  using TA = LaTile<T, MA, BM, WM * WN * 64>;
  using TB = LaTile<T, MB, BN, WM * WN * 64>;
  constexpr int KE = TA::KE, TM = BM / WM, TN = BN / WN, NM = TM / 16, NN = TN / 16;
  constexpr bool P = Precise<T>::value;
  static_assert(TM % 16 == 0 && TN % 16 == 0, "tile");
  __shared__ __attribute__((aligned(16))) char lds_a[TA::BYTES];
  __shared__ __attribute__((aligned(16))) char lds_b[TB::BYTES];
  const int lane = threadIdx.x & 63, wave = PYGHO_WAVE_INDEX(threadIdx.x >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  const int wm = (wave / WN) * TM, wn = (wave % WN) * TN;
  const int64_t m_rows = EPI == LA_ACT && g.dev ? *g.dev : g.m;
  const int64_t k_end = EPI == LA_SLAB && g.dev ? *g.dev : g.k;
  const int64_t tiles_n = (g.n + BN - 1) / BN, tiles_m = (m_rows + BM - 1) / BM;
  const int splits = EPI == LA_SLAB ? g.splits : 1;
  const int64_t tiles = tiles_m * tiles_n * splits;
  // consecutive workgroups go to the 8 XCDs in turn: with several column tiles, an XCD takes a contiguous range of tiles (column tile
  // innermost), so that the row tile they share is read from HBM once and from that XCD's L2 after that
  const int64_t per_xcd = (tiles + 7) / 8;

  for (int64_t slot = blockIdx.x; slot < per_xcd * 8; slot += gridDim.x) {
    const int64_t t = tiles_n * splits > 1 ? (slot & 7) * per_xcd + (slot >> 3) : slot;
    if (t >= tiles) continue;
    const int split = (int)(t % splits);                // (splits of one output tile side by side: they write far apart anyway)
    const int64_t tt = t / splits;
    const int64_t m0 = (tt / tiles_n) * BM, n0 = (tt % tiles_n) * BN;
    // the steps of the reduction: k0(it).  A split walks chunks split, split + splits, ...
    constexpr int SUB = kLaChunk / KE;
    int64_t n_it;
    if constexpr (EPI == LA_SLAB) {
      const int64_t chunks = (k_end + kLaChunk - 1) / kLaChunk;
      n_it = chunks > split ? ((chunks - 1 - split) / splits + 1) * SUB : 0;
    } else {
      n_it = (k_end + KE - 1) / KE;
    }
    auto k_of = [&](int64_t it) -> int64_t {
      if constexpr (EPI == LA_SLAB) return (split + (it / SUB) * splits) * kLaChunk + (it % SUB) * KE;
      return it * KE;
    };
    uint4 ra[TA::PER_THREAD], rb[TB::PER_THREAD];
    auto fetch = [&](int64_t k0) __attribute__((always_inline)) {
      if constexpr (FULL) {
#pragma unroll
        for (int i = 0; i < TA::PER_THREAD; ++i) ra[i] = TA::load_full(g.a, m0, m_rows, k0, i);
#pragma unroll
        for (int i = 0; i < TB::PER_THREAD; ++i) rb[i] = TB::load_full(g.b, n0, g.n, k0, i);
      } else {
#pragma unroll
        for (int i = 0; i < TA::PER_THREAD; ++i) ra[i] = TA::load(g.a, m0, m_rows, k0, k_end, i);
#pragma unroll
        for (int i = 0; i < TB::PER_THREAD; ++i) rb[i] = TB::load(g.b, n0, g.n, k0, k_end, i);
      }
    };
    la_f32x4_t acc[NM][NN], ones_acc[EPI == LA_SLAB ? NM : 1];
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
      for (int j = 0; j < NN; ++j) acc[i][j] = la_f32x4_t{0.f, 0.f, 0.f, 0.f};
    if constexpr (EPI == LA_SLAB) {
#pragma unroll
      for (int i = 0; i < NM; ++i) ones_acc[i] = la_f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    const bool sums = EPI == LA_SLAB && g.want_sums && n0 == 0 && wn == 0;
    if (FULL || n_it > 0) fetch(k_of(0));                      // (FULL: k is at least one step)
    for (int64_t it = 0; it < n_it; ++it) {
      __syncthreads();                                   // the previous step's fragments are read
#pragma unroll
      for (int i = 0; i < TA::PER_THREAD; ++i) TA::store(lds_a, ra[i], i);
#pragma unroll
      for (int i = 0; i < TB::PER_THREAD; ++i) TB::store(lds_b, rb[i], i);
      __syncthreads();
      if constexpr (FULL) fetch(k_of(min(it + 1, n_it - 1)));   // (unconditional: the registers stay registers)
      else if (it + 1 < n_it) fetch(k_of(it + 1));
      __builtin_amdgcn_sched_barrier(0);                         // (the scheduler puts the loads behind the products otherwise, and all of their latency in front of the next step)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        uint4 fm[NM];
#pragma unroll
        for (int i = 0; i < NM; ++i) fm[i] = TA::frag(lds_a, wm + i * 16, ks, r16, q);
#pragma unroll
        for (int j = 0; j < NN; ++j) {
          const uint4 fn = TB::frag(lds_b, wn + j * 16, ks, r16, q);
#pragma unroll
          for (int i = 0; i < NM; ++i) acc[i][j] = la_mfma<T>(fn, fm[i], acc[i][j]);
        }
        if (sums) {                                      // column sums of dz: the same fragments against ones
#pragma unroll
          for (int i = 0; i < NM; ++i) ones_acc[i] = la_mfma<T>(la_ones<T>(), fm[i], ones_acc[i]);
        }
      }
    }

    // ---- epilogue: lane (r16, q) holds rows m0 + wm + 16 i + r16, channels n0 + wn + 16 j + 4 q .. + 3 ----------------------------
    if constexpr (EPI == LA_SLAB) {
      float* slab = g.slabs + (int64_t)split * g.slab_stride;
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        const int64_t m = m0 + wm + i * 16 + r16;
        if (m >= g.m) continue;
#pragma unroll
        for (int j = 0; j < NN; ++j) {
          const int64_t n = n0 + wn + j * 16 + q * 4;
#pragma unroll
          for (int e = 0; e < 4; ++e) if (n + e < g.n) slab[m * g.n + n + e] = acc[i][j][e];
        }
        if (sums && q == 0) slab[g.m * g.n + m] = ones_acc[i][0];
      }
    } else {
      const T* res = reinterpret_cast<const T*>(g.res);
      T* out = reinterpret_cast<T*>(g.out);
      // every load in front of the stores it does not depend on: a load's wait also waits for all older stores
      float bias[NN][4];
#pragma unroll
      for (int j = 0; j < NN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t n = n0 + wn + j * 16 + q * 4 + e;
          bias[j][e] = n < g.n ? ro_param(g.bias, g.bias_dtype, n, 0.f) : 0.f;
        }
#pragma unroll
      for (int j = 0; j < NN; ++j) {
        const int64_t n = n0 + wn + j * 16 + q * 4;
        const int left = (int)min((int64_t)4, g.n - n);
#pragma unroll
        for (int i = 0; i < NM; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] += bias[j][e];
        if (g.z) {
#pragma unroll
          for (int i = 0; i < NM; ++i) {
            const int64_t m = m0 + wm + i * 16 + r16;
            const float u[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
            if (m < m_rows && left > 0) {
              if (g.z_f32) {
                la_store4<float>(reinterpret_cast<float*>(g.z) + m * g.n + n, left, u);
              } else {
                const float v[4] = {la_in_range<T>(u[0]), la_in_range<T>(u[1]), la_in_range<T>(u[2]), la_in_range<T>(u[3])};
                la_store4<T>(reinterpret_cast<T*>(g.z) + m * g.n + n, left, v);
              }
            }
          }
        }
        if (!out) continue;
        float r[NM][4];
#pragma unroll
        for (int i = 0; i < NM; ++i) {
          const int64_t m = m0 + wm + i * 16 + r16;
#pragma unroll
          for (int e = 0; e < 4; ++e) r[i][e] = 0.f;
          if (res && m < m_rows && left > 0) la_load4<T>(res + m * g.res_ld + n, left, r[i]);
        }
#pragma unroll
        for (int i = 0; i < NM; ++i) {
          const int64_t m = m0 + wm + i * 16 + r16;
          float u[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
          ro_act<P, 4>(u, g.act);
#pragma unroll
          for (int e = 0; e < 4; ++e) u[e] += r[i][e];
          if (m < m_rows && left > 0) la_store4<T>(out + m * g.n + n, left, u);
        }
      }
    }
  }
}

// wt (k, n) = w (n, k) transposed: 32 x 32 tiles through LDS
template <typename T> __global__ __launch_bounds__(kBlock) void la_transpose_kernel(T* __restrict__ wt, const T* __restrict__ w, int64_t w_ld, int64_t n, int64_t k) {
  __shared__ T tile[32][33];
  const int64_t n0 = (int64_t)blockIdx.y * 32, k0 = (int64_t)blockIdx.x * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = ty; i < 32; i += 8) if (n0 + i < n && k0 + tx < k) tile[i][tx] = w[(n0 + i) * w_ld + k0 + tx];
  __syncthreads();
  for (int i = ty; i < 32; i += 8) if (k0 + i < k && n0 + tx < n) wt[(k0 + i) * n + n0 + tx] = tile[tx][i];
}
template <typename T> static int la_transpose(void* wt, const void* w, int64_t w_ld, int64_t n, int64_t k, hipStream_t st) {
  if (ceil_div(n, 32) > 65535) { set_error("linear: %lld output channels", (long long)n); return PYGHO_ERR_UNSUPPORTED; }
  hipLaunchKernelGGL((la_transpose_kernel<T>), dim3((unsigned)ceil_div(k, 32), (unsigned)ceil_div(n, 32)), dim3(kBlock), 0, st, (T*)wt, (const T*)w, w_ld, n, k);
  return check_launch("linear_transpose");
}

static bool la_aligned(const void* p, int64_t ld, int es, int bytes) { return ((uintptr_t)p % bytes) == 0 && (ld * es) % bytes == 0; }

template <typename T, int MA, int MB, int BM, int BN, int WM, int WN, int EPI, bool FULL = false> static int la_go(const LaArgs& a, int grid_cap, hipStream_t st) {
  const int64_t tiles = ceil_div(a.m, BM) * ceil_div(a.n, BN) * (EPI == LA_SLAB ? a.splits : 1);
  const int grid = (int)std::min<int64_t>((tiles + 7) / 8 * 8, grid_cap);
  hipLaunchKernelGGL((linear_tile_kernel<T, MA, MB, BM, BN, WM, WN, EPI, FULL>), dim3(grid), dim3(WM * WN * 64), 0, st, a);
  return check_launch("linear_tile");
}

constexpr int kLaGrid = 1 << 20;        // workgroups of a launch (a larger product loops)

// Tile of an (m, n) product without a norm: the largest that still gives every CU a workgroup, no wider than the product (128 x 128 against 64 x 64, bf16:
// 65536 x 500 -> 500 forward 92 us, 100, gradients 445, 502; gradients of 1.05 M x 256 -> 256 970, 1276)
template <typename T, int MA, int MB, int EPI> static int la_any(const LaArgs& a, hipStream_t st) {
  const int64_t sp = EPI == LA_SLAB ? a.splits : 1;
  auto count = [&](int bm, int bn) { return ceil_div(a.m, bm) * ceil_div(a.n, bn) * sp; };
  if (a.n <= 16) return la_go<T, MA, MB, 64, 16, 4, 1, EPI>(a, kLaGrid, st);
  // 16-bit products large enough for a 256 x 256 tile per CU: a wavefront's 128 x 64 part reads 12 fragments of LDS per 32 MFMAs, a 64 x 64 part 8 per 16
  if constexpr (sizeof(T) == 2 && EPI == LA_ACT)
    // (bf16 forward 65536 x 512 -> 512 66 us, 80 with 128 x 128 tiles; 262144 x 512 -> 256 151, 168).  Its 32-bit offsets reach over 256 rows.  The weight gradient stays on 128 x 128
    // tiles with a condition per load: unconditional ones took registers and a workgroup per CU with them (84 -> 116 us)
    if (a.n > 128 && count(256, 256) >= 256 && a.k % 64 == 0 && std::max(a.a.ld, a.b.ld) * (int64_t)sizeof(T) < (1 << 24))
      return la_go<T, MA, MB, 256, 256, 2, 4, EPI, true>(a, kLaGrid, st);
  if (a.n > 64 && a.m > 64 && count(128, 128) >= 256) return la_go<T, MA, MB, 128, 128, 2, 2, EPI>(a, kLaGrid, st);
  return la_go<T, MA, MB, 64, 64, 2, 2, EPI>(a, kLaGrid, st);
}

}  // namespace pygho
