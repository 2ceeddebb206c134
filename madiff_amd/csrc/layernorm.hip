// Layer norm over the channels of channels-last rows, forward and backward.
//
//   mu = mean_c x,  v = mean_c (x - mu)^2,  r = (v + eps)^-1/2,  h = (x - mu) r,  y = h w + b
//   g = dy w,  dx = r (g - mean_c g - h mean_c(g h)),  dw = sum_rows dy h,  db = sum_rows dy
//
// Bandwidth-bound: forward reads x and writes y once, backward reads x and dy and writes dx once.  A row lives in the registers of
// a group of lanes, 16 elements (or fewer) each: 8..64 lanes of one wave, or a workgroup of 128..1024; only above 16384 columns a
// lane has 32.  (32 bf16 elements a lane in one wave, or 256 lanes for rows up to 8192 columns with one workgroup a CU: too few
// waves and loads in flight; 65536 x 2048 backward took 460 us, now 173; 16384 x 8192 418, now 178.)  Groups stride over the rows
// with their share of w and b in registers (read from L2 for every row they would cost four times the bf16 row itself) and with
// the next row's loads in flight.  Measured with cold caches, where a 4 GiB copy reaches 4.6 TB/s: bf16 262144 x 1024 forward 230 us
// (4.7 TB/s) and backward 316 (5.1), 32768 x 4096 128 and 168 (4.2, 4.8), 4093 x 16384 74 and 97 (3.7, 4.2); fp32 65536 x 1024 116
// and 157 (4.6, 5.1).  The widest rows, 2000 x 32768 bf16: 92 and 259 (2.9, 1.5; dw and db fill the registers).  The variance
// is the second pass over the registers, not E[x^2] - mu^2.  All arithmetic is fp32; the only rounding to fewer bits is
// that of y and dx to the storage type of x.
// dw / db: every lane sums its own columns over the rows of its group in fp32 registers, a workgroup's groups meet in LDS,
// each workgroup leaves one [2, C] partial, and a second launch adds the partials in index order: no atomics, so the same
// call gives the same bits.
#include "common.h"

// 16 bytes of a row as they lie in memory: four registers whatever the type (as eight bf16 values they took eight)
template <typename T> struct LnVec {
  static constexpr int N = 16 / sizeof(T);
  uint32_t u[4];
  __device__ __forceinline__ float at(int e) const {
    if constexpr (N == 4) return __uint_as_float(u[e]);
    else return __uint_as_float(e & 1 ? u[e >> 1] & 0xffff0000u : u[e >> 1] << 16);
  }
};

// from an address that is only element-aligned (rows of odd widths begin anywhere; the hardware takes it)
template <typename T> __device__ __forceinline__ LnVec<T> ln_load(const T* p) {
  LnVec<T> r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
template <typename T> __device__ __forceinline__ LnVec<T> ln_load_part(const T* p, int n) {   // n elements, zeros behind
  LnVec<T> r;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    r.u[k] = 0;
    if constexpr (sizeof(T) == 4) {
      if (k < n) __builtin_memcpy(&r.u[k], p + k, 4);
    } else {
      uint16_t lo = 0, hi = 0;
      if (2 * k < n) __builtin_memcpy(&lo, p + 2 * k, 2);
      if (2 * k + 1 < n) __builtin_memcpy(&hi, p + 2 * k + 1, 2);
      r.u[k] = lo | (uint32_t)hi << 16;
    }
  }
  return r;
}
// R vectors of a lane from its FROM-th on: columns (l + i LPR) N .. + N
template <typename T, int LPR, int R, int FROM = 0>
__device__ __forceinline__ void ln_row(LnVec<T> (&d)[R], const T* row, int l, int C) {
  constexpr int N = LnVec<T>::N;
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int c = (l + (FROM + i) * LPR) * N;
    if (c + N <= C) d[i] = ln_load(row + c);
    else d[i] = ln_load_part(row + (c < C ? c : 0), c < C ? C - c : 0);
  }
}
// N gains (or shifts) from column c on; `none` where there is no such vector, 0 behind the row's end
template <int N>
__device__ __forceinline__ void ln_gain(float (&d)[N], const float* w, int c, int C, float none) {
  if (w && c + N <= C) {
    __builtin_memcpy(d, w + c, 4 * N);
  } else {
#pragma unroll
    for (int e = 0; e < N; e++) d[e] = c + e < C ? (w ? w[c + e] : none) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void ln_put(T* row, const float (&y)[LnVec<T>::N], int c, int C) {
  constexpr int N = LnVec<T>::N;
  if (c + N <= C) {
    T o[N];
#pragma unroll
    for (int e = 0; e < N; e++) o[e] = from_f32<T>(y[e]);
    __builtin_memcpy(row + c, &o, 16);
  } else if (c < C) {
#pragma unroll
    for (int e = 0; e < N; e++)
      if (c + e < C) row[c + e] = from_f32<T>(y[e]);
  }
}

// Sum over LPR = 2..64 neighbouring lanes, the same bits in each of them: by DPP within rows of 16 lanes, then by swaps of rows
// and halves.  (Through LDS the six dependent shuffles of a row took longer than its arithmetic.)
template <int LPR> __device__ __forceinline__ float ln_lanes(float v) {
#define LN_DPP(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true))
  LN_DPP(0xB1);                            // lane ^ 1
  if constexpr (LPR >= 4) LN_DPP(0x4E);    // lane ^ 2
  if constexpr (LPR >= 8) LN_DPP(0x141);   // 7 - lane: the other four of eight
  if constexpr (LPR >= 16) LN_DPP(0x140);  // 15 - lane: the other eight
#undef LN_DPP
  if constexpr (LPR >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const unsigned lo = r[0], hi = r[1];
    v = __uint_as_float(lo) + __uint_as_float(hi);
  }
  if constexpr (LPR >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const unsigned lo = r[0], hi = r[1];
    v = __uint_as_float(lo) + __uint_as_float(hi);
  }
  return v;
}

// Sum of K values over the LPR lanes of a group: within its waves, then across them through LDS.  `slot`
// alternates from call to call, so that one barrier a call is enough: the values of a call are overwritten two calls later,
// behind the barrier of the call between.
template <int LPR, int K>
__device__ __forceinline__ void ln_sum(float (&v)[K], float* lds, int& slot) {
#pragma unroll
  for (int k = 0; k < K; k++) v[k] = ln_lanes<(LPR < 64 ? LPR : 64)>(v[k]);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    float* s = lds + slot * (K * W);
    slot ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; k++) s[k * W + (threadIdx.x >> 6)] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) v[k] = ln_lanes<W>(s[k * W + (threadIdx.x & (W - 1))]);
  }
}

template <typename T, int LPR, int R>
__global__ __launch_bounds__(LPR > 64 ? LPR : 256) void layer_norm_fwd_kernel(
    const T* __restrict__ x, long ldx, T* __restrict__ y, long ldy, const float* __restrict__ w, const float* __restrict__ b,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, long rows, int C, int Cpad, float eps) {
  constexpr int N = LnVec<T>::N, BLOCK = LPR > 64 ? LPR : 256, GPB = LPR > 64 ? 1 : BLOCK / LPR;
  __shared__ float lds[LPR > 64 ? 2 * (LPR / 64) : 1];
  int l = threadIdx.x % LPR;
  const long g0 = (long)blockIdx.x * GPB + (GPB > 1 ? threadIdx.x / LPR : 0), gs = (long)gridDim.x * GPB;
  int slot = 0;
  constexpr bool LEAN = R * N > 16;      // 128 registers a lane: gains and shifts come from L2 row by row, no row is prefetched
  float wv[LEAN ? 1 : R][N], bv[LEAN ? 1 : R][N];
  if constexpr (!LEAN)
#pragma unroll
    for (int i = 0; i < R; i++) {
      ln_gain<N>(wv[i], w, (l + i * LPR) * N, C, 1.f);
      ln_gain<N>(bv[i], b, (l + i * LPR) * N, C, 0.f);
    }
  LnVec<T> nx[R];
  if (!LEAN && g0 < rows) ln_row<T, LPR, R>(nx, x + g0 * ldx, l, C);
  const float inv = 1.f / (float)C;
  for (long r = g0; r < rows; r += gs) {
    asm("" : "+v"(l));                   // (else every vector's addresses and tail tests stay in registers over all rows)
    const float *wr = w, *br = b;
    if constexpr (LEAN) {
      asm("" : "+s"(wr), "+s"(br));        // (not loop-invariant to the compiler: it would hold them in registers)
      ln_row<T, LPR, R>(nx, x + r * ldx, l, C);
    }
    float v[R][N];
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
      for (int e = 0; e < N; e++) {
        v[i][e] = nx[i].at(e);
        s[0] += v[i][e];
      }
    if (!LEAN && r + gs < rows) ln_row<T, LPR, R>(nx, x + (r + gs) * ldx, l, C);
    ln_sum<LPR, 1>(s, lds, slot);
    const float mean = s[0] / (float)C;      // (divided: the mean of equal values is that value)
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
      for (int e = 0; e < N; e++) {
        v[i][e] -= mean;
        const float d = (l + i * LPR) * N + e < C ? v[i][e] : 0.f;
        s[0] += d * d;
      }
    ln_sum<LPR, 1>(s, lds, slot);
    const float rstd = 1.f / sqrtf(s[0] * inv + eps);
    if (l == 0 && mean_out) { mean_out[r] = mean; rstd_out[r] = rstd; }
#pragma unroll
    for (int i = 0; i < R; i++) {
      if constexpr (LEAN) {
        ln_gain<N>(wv[0], wr, (l + i * LPR) * N, C, 1.f);
        ln_gain<N>(bv[0], br, (l + i * LPR) * N, C, 0.f);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int e = 0; e < N; e++) v[i][e] = v[i][e] * rstd * wv[LEAN ? 0 : i][e] + bv[LEAN ? 0 : i][e];
      ln_put<T>(y + r * ldy, v[i], (l + i * LPR) * N, C);
    }
    for (int c = C + l; c < Cpad; c += LPR) y[r * ldy + c] = from_f32<T>(0.f);   // pad columns of the layout stay zero
  }
}

// part: [gridDim.x, 2, C] column sums (dw then db) of the workgroup's rows; null = no parameter gradient wanted.
template <typename T, int LPR, int R>
// (bf16 up to 128 lanes: 128 registers, four waves a SIMD, for three spilled ones: 262144 x 1024 316 us, with 130 registers and three
// waves 354.  fp32 would spill forty: 6151 x 777 21 us, held to 128 registers 37.)
__global__ __launch_bounds__((LPR > 64 ? LPR : 256), (sizeof(T) == 2 && LPR <= 128 ? 4 : 1)) void layer_norm_bwd_kernel(
    const T* __restrict__ x, long ldx, const T* __restrict__ dy, long lddy, const float* __restrict__ w,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx, long lddx,
    float* __restrict__ part, long rows, int C, int Cpad) {
  constexpr int N = LnVec<T>::N, BLOCK = LPR > 64 ? LPR : 256, GPB = LPR > 64 ? 1 : BLOCK / LPR;
  constexpr int COLS = 64 * R * N;                           // columns a wave covers (LPR <= 64)
  __shared__ float lds[LPR > 64 ? 4 * (LPR / 64) : 3 * COLS];
  int l = threadIdx.x % LPR;
  const long g0 = (long)blockIdx.x * GPB + (GPB > 1 ? threadIdx.x / LPR : 0), gs = (long)gridDim.x * GPB;
  int slot = 0;
  // LEAN: 1024 lanes have 128 registers each.  h and g are formed twice, gains come from L2 row by row, no row is prefetched;
  // KEEP: x waits in LDS, each lane's vectors for itself (no barrier).
  constexpr bool LEAN = R * N > 16 || (LPR == 1024 && N == 4), KEEP = R * N > 16;
  __shared__ LnVec<T> keep[KEEP ? R * LPR : 1];
  float wv[LEAN ? 1 : R][N], aw[R][N], ab[R][N];
#pragma unroll
  for (int i = 0; i < R; i++) {
    if constexpr (!LEAN) ln_gain<N>(wv[i], w, (l + i * LPR) * N, C, 1.f);
#pragma unroll
    for (int e = 0; e < N; e++) aw[i][e] = ab[i][e] = 0.f;
  }
  LnVec<T> nx[KEEP ? R / 2 : R], nd[R];
  if (!LEAN && g0 < rows) {
    ln_row<T, LPR, (KEEP ? R / 2 : R)>(nx, x + g0 * ldx, l, C);
    ln_row<T, LPR, R>(nd, dy + g0 * lddy, l, C);
  }
  const float inv = 1.f / (float)C;
  for (long r = g0; r < rows; r += gs) {
    asm("" : "+v"(l));                   // (else every vector's addresses and tail tests stay in registers over all rows)
    const float mean = mean_in[r], rstd = rstd_in[r];
    const float* wr = w;
    if constexpr (LEAN) {
      asm("" : "+s"(wr));
      if constexpr (KEEP) {
        ln_row<T, LPR, R / 2>(nx, x + r * ldx, l, C);
#pragma unroll
        for (int i = 0; i < R / 2; i++) keep[i * LPR + l] = nx[i];
        __builtin_amdgcn_sched_barrier(0);
        ln_row<T, LPR, R / 2, R / 2>(nx, x + r * ldx, l, C);
#pragma unroll
        for (int i = 0; i < R / 2; i++) keep[(R / 2 + i) * LPR + l] = nx[i];
        asm volatile("" ::: "memory");       // (read back, not held in registers)
      } else {
        ln_row<T, LPR, R>(nx, x + r * ldx, l, C);
      }
      ln_row<T, LPR, R>(nd, dy + r * lddy, l, C);
    }
    const auto xs = [&](int i) { return KEEP ? keep[i * LPR + l] : nx[KEEP ? 0 : i]; };
    float h[LEAN ? 1 : R][N], g[LEAN ? 1 : R][N];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < R; i++) {
      const int k = LEAN ? 0 : i;
      if constexpr (LEAN) {
        ln_gain<N>(wv[0], wr, (l + i * LPR) * N, C, 1.f);
        __builtin_amdgcn_sched_barrier(0);
      }
      const LnVec<T> xi = xs(i);
#pragma unroll
      for (int e = 0; e < N; e++) {
        const float d = nd[i].at(e);                         // 0 behind the row's end, and so is all it multiplies
        h[k][e] = (xi.at(e) - mean) * rstd;
        g[k][e] = d * wv[k][e];
        aw[i][e] += d * h[k][e];
        ab[i][e] += d;
        s[0] += g[k][e];
        s[1] += g[k][e] * h[k][e];
      }
    }
    if (!LEAN && r + gs < rows) {
      ln_row<T, LPR, (KEEP ? R / 2 : R)>(nx, x + (r + gs) * ldx, l, C);
      ln_row<T, LPR, R>(nd, dy + (r + gs) * lddy, l, C);
    }
    if (dx) {
      ln_sum<LPR, 2>(s, lds, slot);
      const float c1 = s[0] * inv, c2 = s[1] * inv;
      if constexpr (LEAN) asm volatile("" : "+s"(wr) : : "memory");
#pragma unroll
      for (int i = 0; i < R; i++) {
        const int k = LEAN ? 0 : i;
        if constexpr (LEAN) {
          ln_gain<N>(wv[0], wr, (l + i * LPR) * N, C, 1.f);
          const LnVec<T> xi = xs(i);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int e = 0; e < N; e++) {
            h[0][e] = (xi.at(e) - mean) * rstd;
            g[0][e] = nd[i].at(e) * wv[0][e];
          }
        }
#pragma unroll
        for (int e = 0; e < N; e++) g[k][e] = rstd * (g[k][e] - c1 - h[k][e] * c2);
        ln_put<T>(dx + r * lddx, g[k], (l + i * LPR) * N, C);
      }
      for (int c = C + l; c < Cpad; c += LPR) dx[r * lddx + c] = from_f32<T>(0.f);
    }
  }
  if (!part) return;
  float* out = part + (size_t)blockIdx.x * 2 * C;
  if constexpr (LPR > 64) {                                  // every lane owns its columns
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
      for (int e = 0; e < N; e++) {
        const int c = (l + i * LPR) * N + e;
        if (c < C) { out[c] = aw[i][e]; out[C + c] = ab[i][e]; }
      }
  } else {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int q = 0; q < 2; q++) {                            // the groups of a wave, then the four waves in order
#pragma unroll
      for (int i = 0; i < R; i++)
#pragma unroll
        for (int e = 0; e < N; e++) {
          float a = q ? ab[i][e] : aw[i][e];
#pragma unroll
          for (int o = LPR; o < 64; o <<= 1) a += __shfl_xor(a, o, 64);
          if (q) ab[i][e] = a; else aw[i][e] = a;
        }
      __syncthreads();
      if (wave > 0 && lane < LPR)
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
          for (int e = 0; e < N; e++) lds[(wave - 1) * COLS + (i * N + e) * LPR + l] = q ? ab[i][e] : aw[i][e];
      __syncthreads();
      if (wave == 0 && lane < LPR)
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
          for (int e = 0; e < N; e++) {
            float a = q ? ab[i][e] : aw[i][e];
#pragma unroll
            for (int o = 0; o < 3; o++) a += lds[o * COLS + (i * N + e) * LPR + l];
            const int c = (l + i * LPR) * N + e;
            if (c < C) out[q * C + c] = a;
          }
    }
  }
}

// dw / db (+)= sum over the partials, in index order: 64 columns a workgroup, 16 lanes a column.
__global__ __launch_bounds__(1024) void layer_norm_param_kernel(const float* __restrict__ part, int n, int C,
                                                               float* __restrict__ dw, float* __restrict__ db, int accumulate) {
  __shared__ float lds[16][64];
  const int cl = threadIdx.x & 63, k = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + cl;                        // column of [2, C]
  float s = 0.f;
  if (c < 2 * C) {
    const int per = (n + 15) / 16, lo = k * per, hi = min(n, lo + per);
    const float* p = part + (size_t)lo * 2 * C + c;
#pragma unroll 8
    for (int i = lo; i < hi; i++, p += 2 * (size_t)C) s += *p;
  }
  lds[k][cl] = s;
  __syncthreads();
  if (k == 0 && c < 2 * C) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) s += lds[i][cl];
    float* o = c < C ? (dw ? dw + c : nullptr) : (db ? db + (c - C) : nullptr);
    if (o) *o = accumulate ? *o + s : s;
  }
}

#define LN_MAX_COLS 32768

// Lanes a row and vectors a lane: calls F(LPR, R) for rows of C elements of T.  8..64 lanes of one wave, four waves to a workgroup,
// while 16 elements a lane hold it, else a workgroup of its own.
#define LN_DISPATCH(F)                                                   \
  do {                                                                   \
    constexpr int N = 16 / sizeof(T), R = 16 / N;                        \
    const int v = (C + N - 1) / N;                                       \
    if (v <= 8) F(8, 1);                                                 \
    else if (v <= 16) F(16, 1);                                          \
    else if (v <= 32) F(32, 1);                                          \
    else if (v <= 64) F(64, 1);                                          \
    else if (R == 4 && v <= 128) F(64, R / 2);                           \
    else if (v <= 64 * R) F(64, R);                                      \
    else if (v <= 128 * R) F(128, R);                                    \
    else if (v <= 256 * R) F(256, R);                                    \
    else if (v <= 512 * R) F(512, R);                                    \
    else if (v <= 1024 * R) F(1024, R);                                  \
    else F(1024, 2 * R);                                                 \
  } while (0)

// The grid, from the same rule.  (By a second one it took fp32 rows of 257..512 columns for 32 lanes where the kernel has 64: half the
// workgroups, 64 x 512 forward and backward 15.3 us, now 11.2, 6151 x 300 26.2, now 20.1.)
template <typename T> static inline long ln_blocks(long rows, int C, int per_group, long lanes) {
  long lpr = 0;
#define LN_LANES(LPR, R) lpr = LPR
  LN_DISPATCH(LN_LANES);
#undef LN_LANES
  const long block = lpr > 64 ? lpr : 256, gpb = block / lpr, most = lanes / block;
  const long b = (rows + gpb * per_group - 1) / (gpb * per_group);
  return b < 1 ? 1 : (b > most ? most : b);
}

template <typename T>
static int ln_fwd(const T* x, long ldx, T* y, long ldy, const float* w, const float* b, float* mean, float* rstd, long rows,
                  int C, int Cpad, float eps, hipStream_t st) {
  const dim3 grid((unsigned)ln_blocks<T>(rows, C, 1, 2048 * 256));
#define LN_F(LPR, R)                                                                                                      \
  hipLaunchKernelGGL((layer_norm_fwd_kernel<T, LPR, R>), grid, dim3(LPR > 64 ? LPR : 256), 0, st, x, ldx, y, ldy, w, b, \
                     mean, rstd, rows, C, Cpad, eps)
  LN_DISPATCH(LN_F);
#undef LN_F
  MADIFF_CHECK_LAUNCH();
  return 0;
}

template <typename T>
static int ln_bwd(const T* x, long ldx, const T* dy, long lddy, const float* w, const float* mean, const float* rstd, T* dx,
                  long lddx, float* part, int groups, long rows, int C, int Cpad, hipStream_t st) {
#define LN_B(LPR, R)                                                                                                      \
  hipLaunchKernelGGL((layer_norm_bwd_kernel<T, LPR, R>), dim3(groups), dim3(LPR > 64 ? LPR : 256), 0, st, x, ldx, dy,   \
                     lddy, w, mean, rstd, dx, lddx, part, rows, C, Cpad)
  LN_DISPATCH(LN_B);
#undef LN_B
  MADIFF_CHECK_LAUNCH();
  return 0;
}

extern "C" int madiff_layer_norm_fwd(int dtype, const void* x, long ldx, void* y, long ldy, const float* w, const float* b,
                                     float* mean, float* rstd, long rows, int C, int Cpad, float eps, hipStream_t stream) {
  if ((dtype != MADIFF_F32 && dtype != MADIFF_BF16) || rows < 0 || C < 1 || C > LN_MAX_COLS || Cpad < C || ldx < C ||
      ldy < Cpad || !(eps >= 0.f) || (mean == nullptr) != (rstd == nullptr))
    return -1;
  if (rows == 0) return 0;
  if (!x || !y) return -1;
  return dtype == MADIFF_BF16
             ? ln_fwd<bf16_t>((const bf16_t*)x, ldx, (bf16_t*)y, ldy, w, b, mean, rstd, rows, C, Cpad, eps, stream)
             : ln_fwd<float>((const float*)x, ldx, (float*)y, ldy, w, b, mean, rstd, rows, C, Cpad, eps, stream);
}

extern "C" int madiff_layer_norm_groups(int dtype, long rows, int C) {
  if ((dtype != MADIFF_F32 && dtype != MADIFF_BF16) || rows < 0 || C < 1 || C > LN_MAX_COLS) return -1;
  return (int)(dtype == MADIFF_BF16 ? ln_blocks<bf16_t>(rows, C, 4, 1024 * 256) : ln_blocks<float>(rows, C, 4, 1024 * 256));
}

extern "C" int madiff_layer_norm_bwd(int dtype, const void* x, long ldx, const void* dy, long lddy, const float* w,
                                     const float* mean, const float* rstd, void* dx, long lddx, float* dw, float* db,
                                     int accumulate, float* ws, long ws_floats, long rows, int C, int Cpad,
                                     hipStream_t stream) {
  const int groups = madiff_layer_norm_groups(dtype, rows, C);
  const bool params = dw || db;
  if (groups < 0 || Cpad < C || ldx < C || lddy < C || (dx && lddx < Cpad) || (params && (!ws || ws_floats < 2L * groups * C)))
    return -1;
  if (rows > 0) {
    if (!x || !dy || !mean || !rstd) return -1;
    if (!dx && !params) return 0;
    float* part = params ? ws : nullptr;
    const int rc = dtype == MADIFF_BF16 ? ln_bwd<bf16_t>((const bf16_t*)x, ldx, (const bf16_t*)dy, lddy, w, mean, rstd,
                                                         (bf16_t*)dx, lddx, part, groups, rows, C, Cpad, stream)
                                        : ln_bwd<float>((const float*)x, ldx, (const float*)dy, lddy, w, mean, rstd,
                                                        (float*)dx, lddx, part, groups, rows, C, Cpad, stream);
    if (rc) return rc;
  }
  if (params) {                          // rows == 0: the sums are zero (no partial is read)
    hipLaunchKernelGGL(layer_norm_param_kernel, dim3((2 * C + 63) / 64), dim3(1024), 0, stream, ws, rows > 0 ? groups : 0, C,
                       dw, db, accumulate);
    MADIFF_CHECK_LAUNCH();
  }
  return 0;
}
