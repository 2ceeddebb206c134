// Newton-Schulz orthogonalisation of many matrices at once, and the Muon optimizer step built on it.
//
// For G [rows, cols], s = min(rows, cols), l = max: X = G (or its transpose: s x l) / max(|G|_F, eps), then `steps` times
//     A = X X^T      R = b A + c A A      X <- a X + R X
// The three products are matrix-core work; everything else rides in their epilogues.
//
// Arithmetic: the iteration multiplies rounding errors by up to a^steps (485 at the usual coefficients), so 8 or 11 bit
// operands lose the small directions of G.  Every operand is therefore kept as TWO fp16 numbers, 2^11 x = hi + 2^-12 lo: hi is
// 2^11 x rounded to fp16, lo what is left, times 2^12, rounded (together 22 bits, 2^-23 of the value at worst).  A product is three
// fp16 matrix instructions, hi hi into one fp32 sum, hi lo + lo hi into another that joins it at the end; the missing lo lo is below
// 2^-22 of the product.  fp16 holds the range because X, A, R and their products are bounded (|X| <= 1.3 or so, |R| <= 5 at the usual
// coefficients; other coefficients are checked on the host).  Values keep their 22 bits down to 2^-25; what is smaller is held to a
// step of 2^-47.  (The second sum is for that: with lo in hi's unit the bits went below 2^-13 already and the step was 2^-35.  Of a 200 x
// 600 matrix whose other half of rows is 1e-6 times the first, small rows came out 2.4e-3 off, now 8e-7, an fp32 iteration's 2.7e-6.
// It costs 128 x 128 tiles 34 registers; 7 x 1024 x 5120 took 1981 us and takes 1999, 5 x 2048 x 256 156 and 161.)  Against 64 bits the
// result is nearer than an fp32 iteration's from 96 rows on (half as far off at 200) and 0.7 to 1.4 times as far off, by length and
// spectrum, between 32 and 96; fewer rows than that go in fp32 (ns_rows_kernel) unless they are very long or in a plan.
//
// Storage: a matrix [R, K] (both padded with zeros to multiples of 32) is a grid of blocks of 16 rows x 16 columns, 1 KB each, a
// row's blocks one after the other.  In a block every row has four 16-byte chunks: hi of columns 0-7, hi of 8-15, lo of 0-7, lo of
// 8-15, in an order that depends on the row and the column block (ns_chunk), so that the straight copy of a block into LDS is free
// of bank conflicts both for the row-wise fragment reads and for the transposing ones.  A K-step of a product is 16: whole
// blocks, each moved by one asynchronous load instruction of a wave.  A and R are symmetric: only their tiles on and above
// the diagonal are computed, the others are written as mirror images.
#include "common.h"
#include <limits.h>
#include <math.h>
#include <string.h>
#include <algorithm>
#include <functional>
#include <queue>
#include <type_traits>
#include <utility>
#include <vector>

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;
typedef s16x4 __attribute__((address_space(3))) * lds_s16x4;

#define NS_PAD 32                  // both axes of a stored matrix
#define NS_SCALE 2048.f            // stored value = 2^11 x
#define NS_LOW 4096.f              // lo is stored 2^12 times as large
#define NS_CHUNK 16384             // elements a workgroup of the norm pass reads
#define NS_MAX_SHORT 16384
#define NS_MAX_LONG (1 << 22)
#define NS_MAX_STEPS 64
#define NS_MAX_GROUPS (1L << 21)   // workgroups of a launch: 2^31 work-items of 1024-lane ones

// One matrix.  Offsets into the user's buffers are in elements, into the workspace in bytes.
struct NsMat {
  long at;                         // first element, row-major [rows, cols]
  int rows, cols;
  int s, l, sp, lp;                // short / long side, padded
  int tall, parts;                 // rows > cols; number of norm partials
  float scale, pad_;
  long x, sq, norm;                // X (two buffers of 4 sp lp bytes), squares (four of 4 sp sp), partials (doubles) and
                                   // behind them e(0) .. e(steps - 1) and a 0, a byte each (ns_shift)
};

// What every kernel here gets: the matrices, the tiles, the workspace.  Lists come with a plan; without
// them every matrix looks like `one` and workgroups are numbered matrix by matrix.
struct NsGroup {
  const NsMat* mats;
  NsMat one;
  long ws_stride, at_stride;       // bytes / elements from one matrix of the batch to the next
  long partials, counters;         // where the workspace's partial sums and their counters begin, in bytes
  int n_counters;
  unsigned char* ws;
};
struct NsTile { int mat, ti, tj; };

// Workgroups reach the 8 XCDs round-robin, each with its own L2.  The tiles of one matrix read the same rows of X (or R) at about
// the same time, so they are given to one XCD: number `id` of `n` becomes a contiguous run per XCD.  (Plans have their lists in
// that order already.)  The tiles of R X go through the matrix in bands of 1024 columns, all rows of a band back to back: a band
// of X and R at one K-step is what an L2 then holds.
__device__ __forceinline__ int ns_xcd_run(int id, int n) {
  const int xcd = id & 7, local = id >> 3, q = n >> 3, r = n & 7;
  return xcd * q + (xcd < r ? xcd : r) + local;
}
// Tile number r of a matrix.  APPLY: the whole [sp, lp]; GRAM and SQUARE: the tiles that reach the diagonal or lie above it.
__host__ __device__ inline int ns_div_up(int a, int b) { return (a + b - 1) / b; }
__host__ __device__ inline int ns_tiles(bool whole, int sp, int lp, int bm, int bn) {
  const int ni = ns_div_up(sp, bm);
  if (whole) return ni * ns_div_up(lp, bn);
  const int nj = ns_div_up(sp, bn);
  int n = 0;
  for (int ti = 0; ti < ni; ti++) n += nj - ti * bm / bn;
  return n;
}
__host__ __device__ inline void ns_tile_at(bool whole, int r, int sp, int lp, int bm, int bn, int& ti, int& tj) {
  if (whole) {
    const int ni = ns_div_up(sp, bm), nj = ns_div_up(lp, bn), wide = 1024 / bn;
    const int band = r / (ni * wide), left = nj - band * wide, w = left < wide ? left : wide;
    r -= band * ni * wide;
    ti = r / w;
    tj = band * wide + r - ti * w;
  } else {
    const int nj = ns_div_up(sp, bn);
    ti = 0;
    while (r >= nj - ti * bm / bn) { r -= nj - ti * bm / bn; ti++; }
    tj = ti * bm / bn + r;
  }
}

// Matrices below eps start as X = G / eps, of any size.  Step k works on Y = 2^e(k) X, e(k) the most that keeps Y and the next step's
// result within 1 (0 where X is near 1 already, so nothing changes for other matrices):
//     Y Y^T = 4^e A        R = b A + c A A = b 4^-e (Y Y^T) + c 16^-e (Y Y^T)^2        Y' = 2^(e(k+1) - e(k)) (a Y + R Y)
// and the last step takes its shift out.  (Without it |G| = 1e-5 eps came out 3e-4 off and 1e-10 eps as zeros; now 1e-7.)
struct NsShift {
  float a, b, c, turn, most;       // the polynomial a + b y + c y^2 of y = x^2, where it turns (or -1), the largest |x| on its orbits
  int cap;                         // the most an e can be for 2^(11 + e) / eps to be an fp32 number
};
// -> e for |X| <= u, and u for the next step
__device__ __forceinline__ int ns_shift(const NsShift& h, double& u) {
  const double y = u * u;
  double grow = fmax(fabs((double)h.a), fabs(h.a + y * (h.b + y * h.c)));
  if (h.turn > 0.f && h.turn < y) grow = fmax(grow, fabs(h.a + 0.5 * h.b * h.turn));
  int x;
  frexp(u * fmax(grow, 1.0), &x);
  u = fmin(u * grow, (double)h.most);
  return min(max(-x, 0), h.cap);
}
// the table e(0) .. e(steps - 1) where it is not 0
__device__ __forceinline__ void ns_shifts(const NsShift& h, double u, int steps, unsigned char* to) {
  for (int k = 0; k < steps; k++) {
    const int e = ns_shift(h, u);
    if (e == 0 && fabsf(h.a) >= 1.f) break;                  // X never gets smaller: only 0s from here on
    to[k] = e;
  }
}
// -> the factor that makes 2^(11 + e(0)) X of an element of G, and u = |X| at the start
__device__ __forceinline__ float ns_start(const NsShift& h, double norm, float eps, double& u) {
  u = norm > 0.0 && norm < (double)eps ? norm / (double)eps : 1.0;
  const double over = norm > (double)eps ? norm : (norm <= (double)eps ? (double)eps : norm);      // (NaN stays)
  double next = u;
  return (float)ldexp((double)NS_SCALE / over, ns_shift(h, next));
}

__device__ __forceinline__ NsMat ns_mat(const NsGroup& g, int mat) {
  if (g.mats) return g.mats[mat];
  NsMat m = g.one;
  m.at += mat * g.at_stride;
  m.x += mat * g.ws_stride;
  m.sq += mat * g.ws_stride;
  m.norm += mat * g.ws_stride;
  return m;
}

typedef __attribute__((ext_vector_type(16))) float f32x16;

// byte of the 16-byte chunk holding `plane` (0 hi, 1 lo) of columns k .. k + 7 (k % 8 == 0) of row r, from the matrix's start
__device__ __forceinline__ size_t ns_chunk(int r, int k, int plane, int kblocks) {
  const int c = (plane * 2 + ((k >> 3) & 1)) ^ ((r >> 2) & 3) ^ ((k >> 3) & 2);
  return ((size_t)(r >> 4) * kblocks + (k >> 4)) * 1024 + (r & 15) * 64 + c * 16;
}

__device__ __forceinline__ void ns_split(float v, _Float16& hi, _Float16& lo) {      // v already scaled
  // v as ONE fp32 number: contracted into the product it came from, hi was formed twice, once rounded from the exact product and
  // once from its fp32 rounding, and where those two differ lo belonged to the other one (an error of 2^-11, one value in thousands)
  asm("" : "+v"(v));
  hi = (_Float16)v;
  lo = (_Float16)((v - (float)hi) * NS_LOW);
}
__device__ __forceinline__ float ns_join(_Float16 hi, _Float16 lo) { return (float)hi + (float)lo * (1.f / NS_LOW); }

template <int N> __device__ __forceinline__ void ns_wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
template <typename F, int... I>
__device__ __forceinline__ void ns_unroll_(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, typename F> __device__ __forceinline__ void ns_unroll(F&& f) {
  ns_unroll_(f, std::make_integer_sequence<int, N>{});
}
// 64 lanes x 16 bytes, per-lane global address -> LDS [addr + 16 lane]; addr is wave-uniform.  In asm so that the compiler's
// waits for the fragment reads stay counted ones; ordered by the explicit vmcnt waits and barriers.
__device__ __forceinline__ void ns_dma(const void* src, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(src)
               : "memory");
}
__device__ __forceinline__ unsigned ns_lds(const void* p) { return (unsigned)(uintptr_t)(lptr_t)p; }

// ------------------------------------------------------------------------------------------------ norm, momentum, split
struct NsSource {
  const void* src;                 // orthogonalize: the matrices, fp32 or bf16
  float *g, *m;                    // Muon: gradient and momentum
  float mu, rest, grad_scale;      // rest = 1 - mu, formed in 64 bits by the caller
  int nesterov, zero_grad, bf16;
  float eps;
  int steps;
  NsShift shift;
};

// Partial sums of squares in 64 bits (no gradient is too small or too large), one per NS_CHUNK elements.  Muon: the momentum
// update M <- mu M + (1 - mu) g on the way, and the squares are those of U = (1 - mu) g + mu M (Nesterov) or M.
// Four (eight) consecutive elements a lane and pass, all of a chunk's passes in flight together.
template <int KIND>                // 0 fp32, 1 bf16, 2 Muon
__global__ __launch_bounds__(1024) void ns_norm_kernel(NsGroup grp, NsSource q, const int* __restrict__ chunks, int per) {
  int mat, chunk;
  if (chunks) { mat = chunks[2 * blockIdx.x]; chunk = chunks[2 * blockIdx.x + 1]; }
  else { mat = blockIdx.x / per; chunk = blockIdx.x - mat * per; }
  const NsMat M = ns_mat(grp, mat);
  const long n = (long)M.rows * M.cols, lo = (long)chunk * NS_CHUNK, hi = min(n, lo + NS_CHUNK);
  constexpr int V = KIND == 1 ? 8 : 4, PASSES = NS_CHUNK / 1024 / V;
  for (int i = blockIdx.x * 1024 + threadIdx.x; i < grp.n_counters; i += gridDim.x * 1024) ((int*)(grp.ws + grp.counters))[i] = 0;
  double sum = 0.0;
  auto take = [&](float v) { sum += (double)v * (double)v; };
  auto step = [&](float g, float m) {                        // -> the new momentum
    const float now = q.mu * m + q.rest * (g * q.grad_scale);
    take(q.nesterov ? q.rest * (g * q.grad_scale) + q.mu * now : now);
    return now;
  };
  if (lo + NS_CHUNK <= n) {
    typedef __attribute__((ext_vector_type(4))) float f4;
    f4 a[PASSES], b[PASSES];
    const long at = M.at + lo + threadIdx.x * V;
#pragma unroll
    for (int p = 0; p < PASSES; p++) {                       // (element-aligned addresses: the hardware takes them)
      if constexpr (KIND == 2) {
        __builtin_memcpy(&a[p], q.g + at + p * 1024 * V, 16);
        __builtin_memcpy(&b[p], q.m + at + p * 1024 * V, 16);
      } else if constexpr (KIND == 1) {
        __builtin_memcpy(&a[p], (const bf16_t*)q.src + at + p * 1024 * V, 16);
      } else {
        __builtin_memcpy(&a[p], (const float*)q.src + at + p * 1024 * V, 16);
      }
    }
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
      if constexpr (KIND == 2) {
#pragma unroll
        for (int e = 0; e < 4; e++) b[p][e] = step(a[p][e], b[p][e]);
        __builtin_memcpy(q.m + at + p * 1024 * V, &b[p], 16);
      } else if constexpr (KIND == 1) {
        bf16_t h[8];
        __builtin_memcpy(h, &a[p], 16);
#pragma unroll
        for (int e = 0; e < 8; e++) take(to_f32(h[e]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) take(a[p][e]);
      }
    }
  } else {
    for (long e = lo + threadIdx.x; e < hi; e += 1024) {
      if constexpr (KIND == 2) q.m[M.at + e] = step(q.g[M.at + e], q.m[M.at + e]);
      else take(KIND == 1 ? to_f32(((const bf16_t*)q.src)[M.at + e]) : ((const float*)q.src)[M.at + e]);
    }
  }
  __shared__ double lds[16];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < 16; w++) sum += lds[w];
    ((double*)(grp.ws + M.norm))[chunk] = sum;
  }
}

// X0 = U / max(|U|, eps) in split form, padding included; a 64 x 64 piece of X a workgroup, through LDS so that the source is
// read along its rows in both orientations.
template <int KIND>
__global__ __launch_bounds__(256) void ns_split_kernel(NsGroup grp, NsSource q, const int* __restrict__ list, int per) {
  NsTile t;
  if (list) { t.mat = list[4 * blockIdx.x]; t.ti = list[4 * blockIdx.x + 1]; t.tj = list[4 * blockIdx.x + 2]; }
  else {
    const int nj = ns_div_up(grp.one.lp, 64);
    t.mat = blockIdx.x / per;
    t.ti = (blockIdx.x - t.mat * per) / nj;
    t.tj = blockIdx.x - t.mat * per - t.ti * nj;
  }
  const NsMat M = ns_mat(grp, t.mat);
  __shared__ float tilebuf[64][65];
  __shared__ double part[4];
  const int i0 = t.ti * 64, j0 = t.tj * 64;                  // X rows (short side), columns
  // four neighbours of a row of the user's a lane, 16 rows a pass; 16 (8) bytes at once from any element-aligned address (one
  // element a lane and load: 57 us for the 17 M elements of a Muon step's gradient and momentum, so 40, at 5 TB/s)
  const int c = 4 * (threadIdx.x & 15), k0 = threadIdx.x >> 4;
  const int col = (M.tall ? i0 : j0) + c, row0 = (M.tall ? j0 : i0) + k0;
  float v[4][4];
#pragma unroll
  for (int u = 0; u < 4; u++) {                              // the piece is on its way while the norm is put together
    const int r = row0 + 16 * u;
    const long e = M.at + (long)r * M.cols + col;
    const int n = r < M.rows ? min(4, M.cols - col) : 0;
    float g[4] = {0.f, 0.f, 0.f, 0.f};
    if constexpr (KIND == 1) {
      const bf16_t* src = (const bf16_t*)q.src;
      bf16_t h[4];
      if (n == 4) __builtin_memcpy(h, src + e, 8);
#pragma unroll
      for (int i = 0; i < 4; i++) v[u][i] = n == 4 ? to_f32(h[i]) : i < n ? to_f32(src[e + i]) : 0.f;
    } else {
      const float* src = KIND == 2 ? q.m : (const float*)q.src;
      if (n == 4) {
        __builtin_memcpy(v[u], src + e, 16);
        if constexpr (KIND == 2) __builtin_memcpy(g, q.g + e, 16);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          v[u][i] = i < n ? src[e + i] : 0.f;
          if constexpr (KIND == 2) g[i] = i < n ? q.g[e + i] : 0.f;
        }
      }
      if constexpr (KIND == 2)
#pragma unroll
        for (int i = 0; i < 4; i++) v[u][i] = q.nesterov ? q.rest * (g[i] * q.grad_scale) + q.mu * v[u][i] : v[u][i];
    }
  }
  double sum = 0.0;
  const double* parts = (const double*)(grp.ws + M.norm);
  for (int i = threadIdx.x; i < M.parts; i += 256) sum += parts[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  double size;
  const float inv = ns_start(q.shift, sqrt(part[0] + part[1] + part[2] + part[3]), q.eps, size);
  if (t.ti == 0 && t.tj == 0 && threadIdx.x == 0) {
    unsigned char* shifts = grp.ws + M.norm + M.parts * 8L;
    for (int k = 0; k <= q.steps; k++) shifts[k] = 0;
    ns_shifts(q.shift, size, q.steps, shifts);
  }
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int k = k0 + 16 * u;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (M.tall) tilebuf[c + i][k] = v[u][i] * inv;
      else tilebuf[k][c + i] = v[u][i] * inv;
    }
    if constexpr (KIND == 2) {
      const int r = row0 + 16 * u;
      if (q.zero_grad && r < M.rows) {
        float* g = q.g + M.at + (long)r * M.cols + col;
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        if (col + 4 <= M.cols) __builtin_memcpy(g, zero, 16);
        else
#pragma unroll
          for (int i = 0; i < 3; i++)
            if (col + i < M.cols) g[i] = 0.f;
      }
    }
  }
  __syncthreads();
  unsigned char* X = grp.ws + M.x;
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int item = threadIdx.x + 256 * u, row = item >> 3, g8 = item & 7;
    f16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      _Float16 h, l;
      ns_split(tilebuf[row][g8 * 8 + e], h, l);
      hi[e] = h;
      lo[e] = l;
    }
    const int col = j0 + g8 * 8;
    if (i0 + row < M.sp && col < M.lp) {
      *(f16x8*)(X + ns_chunk(i0 + row, col, 0, M.lp >> 4)) = hi;
      *(f16x8*)(X + ns_chunk(i0 + row, col, 1, M.lp >> 4)) = lo;
    }
  }
}

// ------------------------------------------------------------------------------------------------ products
enum { NS_GRAM = 0, NS_SQUARE = 1, NS_APPLY = 2 };
enum { NS_OUT_PLANES = 0, NS_OUT_F32 = 1, NS_OUT_BF16 = 2, NS_OUT_MUON = 3 };

struct NsProduct {
  int a, b, e2, out;               // square buffers (SQUARE: A, B^T = B, addend or -1, result) / X buffer read and written (APPLY: b, out)
  float ca, c1, c2;                // result = ca A B + c1 B + c2 E2
  int step, then;                  // APPLY: from step `step`'s shift to step `then`'s; SQUARE: the shift R is formed at, or -1
  void* dst;                       // last APPLY: the user's buffer
  float *p, *ema;                  // Muon
  bf16_t* shadow;
  float decay, lr, ema_beta, ema_rest;   // W <- decay W - lr scale O
  int do_ema;
  const int* state;
};

// The workgroups of one launch: tile (ti, tj) of matrix `mat`, slice `part` of `parts` of its reduction.  A tile in several parts leaves
// fp32 partial sums at `slot` (the first part's slot: part p is at slot + p); whoever comes last to the tile adds them up.
struct NsWork { int mat, ti, tj, part, parts, slot, pad0, pad1; };
struct NsList {
  const NsWork* work;              // null: numbered matrix by matrix, tile by tile, part by part
  int n, tiles, parts;             // (without a list) per matrix, per tile
};

template <bool WHOLE, int BM, int BN>
__device__ __forceinline__ NsWork ns_work(const NsGroup& g, const NsList& l, int id) {
  if (l.work) return l.work[id];
  NsWork w = {};
  const int per = l.tiles * l.parts, r = id % per, tile = r % l.tiles;      // part by part: its tiles read the same columns
  w.mat = id / per;
  w.part = r / l.tiles;
  w.parts = l.parts;
  w.slot = (w.mat * l.tiles + tile) * l.parts;
  ns_tile_at(WHOLE, tile, g.one.sp, g.one.lp, BM, BN, w.ti, w.tj);
  return w;
}

// What becomes of a wave's 32 x 32 blocks of sums.  A lane's accumulators are groups of four columns of its row; swapping halves of
// register pairs with the lane 32 away makes them eight, a 16-byte chunk of each plane: p = 0, 1 has columns 16 p + 8 fh .. + 7.
// (Chunk by chunk the address units keep up; 8-byte pieces took them four times as long, a third of a tile's whole time.)
// What the next block reads is on its way while a block is finished.  Mirror images and the user's rows are turned through a
// piece of LDS of the wave's own.
template <int KIND, int OUT, int BX>
struct NsFinish {
  struct Extra { f16x8 h1[2], l1[2], h2[2], l2[2]; f32x4 p[4], e[4]; };
  const NsProduct& q;
  const NsMat& M;
  uint32_t* turn;                  // 32 x 33 words
  const unsigned char *e1, *e2;
  unsigned char* out;
  int lane, rows, cols, kb, do_ema;
  float ca, c1;

  __device__ __forceinline__ NsFinish(const NsGroup& grp, const NsProduct& q_, const NsMat& M_, uint32_t* turn_, int lane_, int e_now,
                                      int e_then)
      : q(q_), M(M_), turn(turn_), lane(lane_) {
    const size_t sq = (size_t)M.sp * M.sp * 4, xs = (size_t)M.sp * M.lp * 4;
    rows = M.sp;
    cols = KIND == NS_APPLY ? M.lp : M.sp;
    kb = cols >> 4;
    e1 = KIND == NS_APPLY ? grp.ws + M.x + q.b * xs : grp.ws + M.sq + q.b * sq;
    e2 = KIND == NS_SQUARE && q.e2 >= 0 ? grp.ws + M.sq + q.e2 * sq : nullptr;
    out = KIND == NS_APPLY ? grp.ws + M.x + q.out * xs : grp.ws + M.sq + q.out * sq;
    do_ema = 0;
    if constexpr (OUT == NS_OUT_MUON) do_ema = q.state ? q.state[1] : q.do_ema;
    ca = q.ca * (1.f / NS_SCALE);                            // sums are in units of the scale squared
    c1 = q.c1;
    if constexpr (KIND == NS_APPLY) {
      const float f = ldexpf(1.f, e_then - e_now);
      ca *= f;
      c1 *= f;
    } else if (e_now) {
      ca = ldexpf(ca, -4 * e_now);
      c1 = ldexpf(c1, -2 * e_now);
    }
  }
  // The user's side of the block at (m0, n0): 32 rows of 32 columns; lane & 7 picks four columns, pass k the rows 8 k + lane / 8.
  __device__ __forceinline__ long user(int m0, int n0, int k, int& row, int& col) const {
    row = (M.tall ? n0 : m0) + 8 * k + (lane >> 3);
    col = (M.tall ? m0 : n0) + 4 * (lane & 7);
    return M.at + (long)row * M.cols + col;
  }
  __device__ __forceinline__ f32x4 four(const float* from, long e, int row, int col) const {
    f32x4 d = {0.f, 0.f, 0.f, 0.f};
    if (row < M.rows && col + 3 < M.cols) __builtin_memcpy(&d, from + e, 16);
    else if (row < M.rows)
#pragma unroll
      for (int r = 0; r < 3; r++)
        if (col + r < M.cols) d[r] = from[e + r];
    return d;
  }
  template <typename T, typename V> __device__ __forceinline__ void put(T* to, const V& d, long e, int row, int col) const {
    if (row < M.rows && col + 3 < M.cols) __builtin_memcpy(to + e, &d, sizeof d);
    else if (row < M.rows)
#pragma unroll
      for (int r = 0; r < 3; r++)
        if (col + r < M.cols) to[e + r] = d[r];
  }
  __device__ __forceinline__ void fetch(Extra& x, int m0, int n0) const {
    if (m0 >= rows || n0 >= cols) return;                    // (blocks lie inside or outside as a whole)
    if (KIND != NS_GRAM)
#pragma unroll
      for (int p = 0; p < 2; p++) {
        const size_t at = ns_chunk(m0 + (lane & 31), n0 + 8 * (lane >> 5) + 16 * p, 0, kb);
        x.h1[p] = *(const f16x8*)(e1 + at);
        x.l1[p] = *(const f16x8*)(e1 + (at ^ 32));
        if (KIND == NS_SQUARE && e2) {
          x.h2[p] = *(const f16x8*)(e2 + at);
          x.l2[p] = *(const f16x8*)(e2 + (at ^ 32));
        }
      }
    if constexpr (OUT == NS_OUT_MUON)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        int row, col;
        const long e = user(m0, n0, k, row, col);
        x.p[k] = four(q.p, e, row, col);
        if (do_ema == 1) x.e[k] = four(q.ema, e, row, col);
      }
  }
  __device__ __forceinline__ void finish(const Extra& x, const f32x16& sum, int m0, int n0) const {
    if (m0 >= rows || n0 >= cols) return;
    const int fr = lane & 31, nl = 8 * (lane >> 5);          // this lane's row, and its columns + 16 p
    float v[2][8];
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float s0 = sum[8 * p + r], s1 = sum[8 * p + 4 + r];
        const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(s0), __float_as_uint(s1), false, false);
        v[p][r] = ca * __uint_as_float(w[0]);
        v[p][4 + r] = ca * __uint_as_float(w[1]);
      }
    if (KIND != NS_GRAM)
#pragma unroll
      for (int p = 0; p < 2; p++)
#pragma unroll
        for (int r = 0; r < 8; r++) {
          // (said, not left to the compiler, which took one or the other product for the exact one, by tile shape)
          v[p][r] = fmaf(c1, ns_join(x.h1[p][r], x.l1[p][r]), v[p][r]);
          if (KIND == NS_SQUARE && e2) v[p][r] = fmaf(q.c2, ns_join(x.h2[p][r], x.l2[p][r]), v[p][r]);
        }
    if constexpr (OUT == NS_OUT_PLANES) {
      // what no tile computes: the mirror images of tiles to the right of their row of the diagonal
      const bool mirror = KIND != NS_APPLY && m0 / BX < n0 / BX;
#pragma unroll
      for (int p = 0; p < 2; p++) {
        f16x8 h, l;
        uint32_t both[8];                                    // hi | lo << 16
#pragma unroll
        for (int r = 0; r < 8; r++) {
          _Float16 hh, ll;
          ns_split(v[p][r], hh, ll);
          h[r] = hh;
          l[r] = ll;
          both[r] = (uint32_t)__builtin_bit_cast(uint16_t, hh) | (uint32_t)__builtin_bit_cast(uint16_t, ll) << 16;
        }
        const size_t at = ns_chunk(m0 + fr, n0 + nl + 16 * p, 0, kb);
        *(f16x8*)(out + at) = h;
        *(f16x8*)(out + (at ^ 32)) = l;
        if (mirror)
#pragma unroll
          for (int r = 0; r < 8; r++) turn[fr * 33 + nl + 16 * p + r] = both[r];
      }
      if (mirror) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int p = 0; p < 2; p++) {
          typedef __attribute__((ext_vector_type(8))) uint16_t u16x8;
          u16x8 h, l;
#pragma unroll
          for (int r = 0; r < 8; r++) {
            const uint32_t both = turn[(nl + 16 * p + r) * 33 + fr];
            h[r] = (uint16_t)both;
            l[r] = (uint16_t)(both >> 16);
          }
          const size_t at = ns_chunk(n0 + fr, m0 + nl + 16 * p, 0, kb);
          *(u16x8*)(out + at) = h;
          *(u16x8*)(out + (at ^ 32)) = l;
        }
        __builtin_amdgcn_wave_barrier();
      }
    } else {
      float* t = (float*)turn;
#pragma unroll
      for (int p = 0; p < 2; p++)
#pragma unroll
        for (int r = 0; r < 8; r++) {
          const int n = nl + 16 * p + r;
          t[M.tall ? n * 33 + fr : fr * 33 + n] = v[p][r] * (1.f / NS_SCALE);
        }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int k = 0; k < 4; k++) {
        int row, col;
        const long e = user(m0, n0, k, row, col);
        f32x4 o;
#pragma unroll
        for (int r = 0; r < 4; r++) o[r] = t[(8 * k + (lane >> 3)) * 33 + 4 * (lane & 7) + r];
        typedef __attribute__((ext_vector_type(4))) bf16_t b16x4;
        b16x4 w16;
        if constexpr (OUT == NS_OUT_F32) {
          put((float*)q.dst, o, e, row, col);
        } else if constexpr (OUT == NS_OUT_BF16) {
#pragma unroll
          for (int r = 0; r < 4; r++) w16[r] = (bf16_t)o[r];
          put((bf16_t*)q.dst, w16, e, row, col);
        } else {
          f32x4 w, a;
#pragma unroll
          for (int r = 0; r < 4; r++) {
            w[r] = q.decay * x.p[k][r] - q.lr * M.scale * o[r];
            a[r] = do_ema == 1 ? q.ema_beta * x.e[k][r] + q.ema_rest * w[r] : w[r];
            w16[r] = (bf16_t)w[r];
          }
          put(q.p, w, e, row, col);
          if (do_ema) put(q.ema, a, e, row, col);
          if (q.shadow) put(q.shadow, w16, e, row, col);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
};

// Tile BM x BN by WM x WN waves, K-steps of 16.  A stage is BM / 16 blocks of A and BN / 16 of B: for a product with a symmetric or
// transposed right side B's rows are read like A's; for R X the blocks are those of 16 rows of X, and fragments come out of
// the transposing LDS read.  D stages are filled by asynchronous loads.  Step k waits (counted) for stage k + 1, passes one
// barrier, sends stage k + D - 1 on its way into the buffer whose fragments everybody has taken, reads the fragments of step
// k + 1 and multiplies those of step k meanwhile.
template <int KIND, int BM, int BN, int WM, int WN, int D, int OUT>
__global__ __launch_bounds__(64 * WM * WN, 2) void ns_product_kernel(NsGroup grp, NsProduct q, NsList list) {
  constexpr int NW = WM * WN, TI = BM / WM / 32, TJ = BN / WN / 32, BX = BM > BN ? BM : BN;
  constexpr int AB = BM / 16, BB = BN / 16, STAGE = (AB + BB) * 1024, PIECES = (AB + BB) / NW;
  static_assert((AB + BB) % NW == 0 && D >= 3 && D * STAGE >= NW * 32 * 33 * 4, "whole pieces a wave");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[D * STAGE];
  const NsWork t = ns_work<KIND == NS_APPLY, BM, BN>(grp, list, list.work ? (int)blockIdx.x : ns_xcd_run(blockIdx.x, gridDim.x));
  if (t.mat < 0) return;           // a list's filler
  const NsMat M = ns_mat(grp, t.mat);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave - wm * WN;
  const size_t sq = (size_t)M.sp * M.sp * 4, xs = (size_t)M.sp * M.lp * 4;
  const unsigned char* Ap = KIND == NS_GRAM ? grp.ws + M.x + q.b * xs : grp.ws + M.sq + q.a * sq;
  const unsigned char* Bp = KIND == NS_SQUARE ? grp.ws + M.sq + q.b * sq : grp.ws + M.x + q.b * xs;
  const int kblocks = (KIND == NS_GRAM ? M.lp : M.sp) >> 4;  // a multiple of 2
  const int kfirst = kblocks / 2 * t.part / t.parts * 2, nsteps = kblocks / 2 * (t.part + 1) / t.parts * 2 - kfirst;
  const int i0 = t.ti * BM, j0 = t.tj * BN;
  const unsigned char* shifts = grp.ws + M.norm + M.parts * 8L;
  const int e_now = KIND == NS_APPLY || (KIND == NS_SQUARE && q.step >= 0) ? shifts[q.step] : 0, e_then = KIND == NS_APPLY ? shifts[q.then] : 0;
  // this wave's blocks of a stage; blocks of a tile that hangs over the matrix's end repeat its last one
  const unsigned char* src[PIECES];
  size_t hop[PIECES];
#pragma unroll
  for (int j = 0; j < PIECES; j++) {
    const int p = wave * PIECES + j;
    if (p < AB) {
      src[j] = Ap + (size_t)min((i0 >> 4) + p, (M.sp >> 4) - 1) * kblocks * 1024;
      hop[j] = 1024;
    } else if (KIND != NS_APPLY) {
      src[j] = Bp + (size_t)min((j0 >> 4) + p - AB, (M.sp >> 4) - 1) * kblocks * 1024;
      hop[j] = 1024;
    } else {
      src[j] = Bp + (size_t)min((j0 >> 4) + p - AB, (M.lp >> 4) - 1) * 1024;
      hop[j] = (size_t)(M.lp >> 4) * 1024;
    }
    src[j] += kfirst * hop[j];
  }
  auto issue = [&](int step, int buf, int j) {
    ns_dma(src[j] + (size_t)step * hop[j] + lane * 16, ns_lds(&smem[buf * STAGE + (wave * PIECES + j) * 1024]));
  };
  // fragment offsets in a stage.  Rows: lane & 31 is the row, lane >> 5 the half of the 16 columns; the other plane is 32 bytes
  // away (xor), and odd column blocks have the planes swapped.
  const int fr = lane & 31, fh = lane >> 5;
  const int frag = (fr >> 4) * 1024 + (fr & 15) * 64 + ((fh ^ ((fr >> 2) & 3)) << 4);
  const int aoff = wm * (BM / WM / 16) * 1024 + frag;
  int boff, boff2 = 0;
  if constexpr (KIND == NS_APPLY) {          // transposing read: 16 lanes take 4 rows x 16 columns of a block, twice
    const int tq = (lane & 15) >> 2, tp = lane & 3, odd = (lane >> 4) & 1, r = 8 * fh + tq;
    boff = AB * 1024 + (wn * (BN / WN / 16) + odd) * 1024 + r * 64 + (((tp >> 1) ^ (2 * fh) ^ (2 * odd)) << 4) + 8 * (tp & 1);
    boff2 = (boff + 256) ^ 16;               // rows + 4: their chunks are one further (xor)
  } else {
    boff = AB * 1024 + wn * (BN / WN / 16) * 1024 + frag;
  }
  struct Frags { f16x8 ah[TI], al[TI], bh[TJ], bl[TJ]; };
  constexpr int READS = TI + TJ;                              // pairs of fragment reads a step
  auto fragment = [&](Frags& f, int buf, int odd_step, int n) {           // pair n: hi and lo of one operand block
    const unsigned char* S = &smem[buf * STAGE];
    const int swap = odd_step * 32;
    if (n < TI) {
      f.ah[n] = *(const f16x8*)(S + ((aoff ^ swap) + n * 2048));
      f.al[n] = *(const f16x8*)(S + ((aoff ^ swap ^ 32) + n * 2048));
    } else if constexpr (KIND == NS_APPLY) {
      const int j = n - TI;
      const s16x4 h0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(S + boff + j * 2048));
      const s16x4 h1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(S + boff2 + j * 2048));
      const s16x4 l0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(S + (boff ^ 32) + j * 2048));
      const s16x4 l1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(S + (boff2 ^ 32) + j * 2048));
      f.bh[j] = __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7));
      f.bl[j] = __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int j = n - TI;
      f.bh[j] = *(const f16x8*)(S + ((boff ^ swap) + j * 2048));
      f.bl[j] = *(const f16x8*)(S + ((boff ^ swap ^ 32) + j * 2048));
    }
  };
  f32x16 acc[TI][TJ], low[TI][TJ];     // hi hi, and hi lo + lo hi, which are 2^12 times as large
#pragma unroll
  for (int i = 0; i < TI; i++)
#pragma unroll
    for (int j = 0; j < TJ; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = low[i][j][r] = 0.f;
  // stage k lives in buffer k % D; stages up to k + D - 2 are on their way when step k begins
#pragma unroll
  for (int d = 0; d < D - 1; d++)
    if (d < nsteps)
#pragma unroll
      for (int j = 0; j < PIECES; j++) issue(d, d, j);
  Frags f0, f1;
  if (nsteps >= D - 1) ns_wait_vm<(D - 2) * PIECES>();
  else ns_wait_vm<0>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int n = 0; n < READS; n++) fragment(f0, 0, 0, n);
  int buf = 0;                                               // of step k
  // One step.  Operands swapped: a lane then holds groups of four consecutive columns of one row.  The three products of an
  // accumulator are a tile's worth of instructions apart (back to back, each would wait for the one before it), and the
  // next step's fragment reads and the loads of stage k + D - 1 are dealt out between them: issued in one go, they kept every
  // wave from its matrix instructions for a third to a half of a step more.
  auto step = [&](auto steady, int k, Frags& c, Frags& n, int odd_next) {
    constexpr bool STEADY = decltype(steady)::value;
    const int next = buf + 1 == D ? 0 : buf + 1, last = buf == 0 ? D - 1 : buf - 1;
    const bool more = STEADY || k + 1 < nsteps, send = STEADY || k + D - 1 < nsteps;
    if (more) {
      // stages k + 1 .. k + D - 2 may be outstanding: D - 3 of them may stay so
      if (STEADY || k + D - 1 <= nsteps) ns_wait_vm<(D - 3) * PIECES>();
      else ns_wait_vm<0>();
      __builtin_amdgcn_s_barrier();    // every wave has the fragments of step k - 1: stage k + D - 1 takes that step's buffer
    }
    if constexpr (!STEADY) {
      if (send)
#pragma unroll
        for (int j = 0; j < PIECES; j++) issue(k + D - 1, last, j);
      if (more)
#pragma unroll
        for (int e = 0; e < READS; e++) fragment(n, next, odd_next, e);
    }
    constexpr int TOTAL = 3 * TI * TJ;
#pragma unroll
    for (int m = 0; m < TOTAL; m++) {
      const int part = m / (TI * TJ), i = m % (TI * TJ) / TJ, j = m % TJ;
      if constexpr (STEADY) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < READS; e++)
          if (e * TOTAL / READS == m) fragment(n, next, odd_next, e);
#pragma unroll
        for (int e = 0; e < PIECES; e++)
          if ((2 * e + 1) * TOTAL / (2 * PIECES) == m) issue(k + D - 1, last, e);
        __builtin_amdgcn_sched_barrier(0);
      }
      f32x16& sum = part == 2 ? acc[i][j] : low[i][j];
      sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(part == 0 ? c.bl[j] : c.bh[j], part == 1 ? c.al[i] : c.ah[i], sum, 0, 0, 0);
    }
    buf = next;
  };
  int k = 0;
  for (; k + D < nsteps; k += 2) {
    step(std::true_type{}, k, f0, f1, 1);
    step(std::true_type{}, k + 1, f1, f0, 0);
  }
  for (; k < nsteps; k += 2) {
    step(std::false_type{}, k, f0, f1, 1);
    step(std::false_type{}, k + 1, f1, f0, 0);
  }
  ns_unroll<TI * TJ>([&](auto at) __attribute__((always_inline)) {
    constexpr int b = decltype(at)::value;
#pragma unroll
    for (int r = 0; r < 16; r++) acc[b / TJ][b % TJ][r] += low[b / TJ][b % TJ][r] * (1.f / NS_LOW);
  });
  const int m0 = i0 + wm * (BM / WM), n0 = j0 + wn * (BN / WN);
  if (t.parts > 1) {
    // A cut reduction: the parts leave their sums as the lanes hold them, and the workgroup that finds itself the last of its tile
    // adds them up in part order (the same bits whoever it is) and goes on; nobody waits.  Sums and counter go past the XCDs' own
    // L2s (agent-scope accesses; the stores have arrived before the count).  Fences instead write back and drop whole L2s: 1300 us
    // where this takes 734 (2048 x 2048).  The sum as a launch of its own: a Muon step of 75 small matrices 150 us, so 131; 256 x
    // 2048 144, so 124; 1024 x 5120 421, so 416; only squares lose, 2048 x 2048 had 684 (a tile's sums all go to one workgroup).  (All
    // of that while hi and lo products shared a sum; now, in the same order, 743, 126, 130, 434.)
    float* to = (float*)(grp.ws + grp.partials) + (size_t)t.slot * (BM * BN) + (size_t)wave * (TI * TJ * 1024) + lane * 2;
    int* counter = (int*)(grp.ws + grp.counters) + t.slot;
    ns_unroll<TI * TJ>([&](auto at) __attribute__((always_inline)) {
      constexpr int b = decltype(at)::value;
#pragma unroll
      for (int g = 0; g < 8; g++) {
        const float s0 = acc[b / TJ][b % TJ][2 * g], s1 = acc[b / TJ][b % TJ][2 * g + 1];
        __hip_atomic_store((uint64_t*)(to + (size_t)t.part * (BM * BN) + b * 1024 + g * 128),
                           __float_as_uint(s0) | (uint64_t)__float_as_uint(s1) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    });
    __shared__ int before;
    ns_wait_vm<0>();
    __syncthreads();
    if (tid == 0) before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (before != t.parts - 1) return;
    if (tid == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);      // for the next product
    ns_unroll<TI * TJ>([&](auto at) __attribute__((always_inline)) {
#pragma unroll
      for (int r = 0; r < 16; r++) acc[decltype(at)::value / TJ][decltype(at)::value % TJ][r] = 0.f;
    });
#pragma unroll(TI * TJ == 1 ? 4 : 2)
    for (int p = 0; p < t.parts; p++) {
      uint64_t v[TI * TJ][8];
#pragma unroll
      for (int b = 0; b < TI * TJ; b++)
#pragma unroll
        for (int g = 0; g < 8; g++)
          v[b][g] = __hip_atomic_load((const uint64_t*)(to + (size_t)p * (BM * BN) + b * 1024 + g * 128), __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT);
      ns_unroll<TI * TJ>([&](auto at) __attribute__((always_inline)) {
        constexpr int b = decltype(at)::value;
#pragma unroll
        for (int g = 0; g < 8; g++) {
          acc[b / TJ][b % TJ][2 * g] += __uint_as_float((uint32_t)v[b][g]);
          acc[b / TJ][b % TJ][2 * g + 1] += __uint_as_float((uint32_t)(v[b][g] >> 32));
        }
      });
    }
  }
  __syncthreads();                                           // the stages are free from here on
  const NsFinish<KIND, OUT, BX> fin(grp, q, M, (uint32_t*)smem + wave * (32 * 33), lane, e_now, e_then);
  typename NsFinish<KIND, OUT, BX>::Extra x0, x1;
  fin.fetch(x0, m0, n0);
  ns_unroll<TI * TJ>([&](auto at) __attribute__((always_inline)) {      // (acc lives in registers: its indices are constants)
    constexpr int t0 = decltype(at)::value, t1 = t0 + 1;
    auto &now = t0 & 1 ? x1 : x0, &then = t0 & 1 ? x0 : x1;
    if constexpr (t1 < TI * TJ) fin.fetch(then, m0 + t1 / TJ * 32, n0 + t1 % TJ * 32);
    fin.finish(now, acc[t0 / TJ][t0 % TJ], m0 + t0 / TJ * 32, n0 + t0 % TJ * 32);
  });
}

// ------------------------------------------------------------------------------------------------ up to 32 rows, in registers
// At these sizes sums are short and the 22 bits of a split operand would show (1.1 to 1.8 times an fp32 iteration's error): fp32 matrix
// instructions, and no operand leaves the registers.  A wave has blocks of 16 columns of X, each twice for every 16 rows: `down`, lane (q, n)
// with X[4 q + r][n], and `along`, with X[n][4 q + r], r = 0 .. 3.  A 16 x 16 x 4 instruction takes L[n][q] and M[q][n] from lane (q, n) and
// leaves D[4 q + r][n] there, so four of them over r multiply
//     along by along:  the block's part of A = X X^T          A and R, which are symmetric, by themselves:  A A
//     R by down:  R X as `down`                               down by R:  (R X)^T, which is R X as `along`
// (where there are many blocks a wave turns R X in LDS instead of forming it twice).  The waves' parts of A meet in LDS and are added up
// in wave order: by everybody, one barrier a step, or, where that would be more reading, block by block by one wave each.
// The kernel takes 4.4 us for 16 x 16, 7.1 for 16 x 128 (18.7 as split fp16 in LDS), 16 for 32 x 128, 44 for 32 x 512: a step's products
// follow from each other, and from 32 x 256 on the fp32 matrix rate of the one CU counts.
template <bool BF16, int RB, int NW, int U>                  // row blocks, waves, column blocks a wave
__global__ __launch_bounds__(64 * NW) void ns_rows_kernel(const void* __restrict__ src, void* __restrict__ dst, NsMat one, long stride,
                                                      int steps, float a, float b, float c, float eps) {
  constexpr int Q = RB * RB;
  constexpr bool TWICE = NW * Q > 8;
  // TWICE: the parts, then the sums.  Else two sets of parts by turns: who writes a step's has seen everybody behind the last one's.
  __shared__ f32x4 parts[NW > 1 ? (TWICE ? NW + 1 : 2 * NW) * Q * 64 : 1];
  __shared__ double norms[NW];
  constexpr bool TURN = RB > 1 || U > 4;
  __shared__ float turns[TURN ? NW * 16 * 20 : 1];
  const NsMat& M = one;
  const long at0 = (long)blockIdx.x * stride;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, n = lane & 15;
  auto value = [&](int row, int col) __attribute__((always_inline)) {          // of X; 0 outside
    const long e = at0 + (M.tall ? (long)col * M.cols + row : (long)row * M.cols + col);
    if (row >= M.s || col >= M.l) return 0.f;
    return BF16 ? to_f32(((const bf16_t*)src)[e]) : ((const float*)src)[e];
  };
  f32x4 down[U][RB], along[U][RB];
  double sum = 0.0;
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int i = 0; i < RB; i++) {
      const int col = 16 * (wave + NW * u);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        down[u][i][r] = value(16 * i + 4 * q + r, col + n);
        along[u][i][r] = value(16 * i + n, col + 4 * q + r);
      }
#pragma unroll
      for (int r = 0; r < 4; r++) sum += (double)down[u][i][r] * (double)down[u][i][r];
      if constexpr (U > 4) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if constexpr (NW > 1) {
    if (lane == 0) norms[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < NW; w++) sum += norms[w];
  }
  const double norm = sqrt(sum), over = norm > (double)eps ? norm : (norm <= (double)eps ? (double)eps : norm);      // (NaN stays)
  int two;
  const float inv = (float)(1.0 / frexp(over, &two));        // over = 2^two / inv, whatever its size
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        down[u][i][r] = ldexpf(down[u][i][r], -two) * inv;
        along[u][i][r] = ldexpf(along[u][i][r], -two) * inv;
      }
  auto multiply = [](const f32x4& x, const f32x4& y, f32x4& d) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 4; r++) d = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], y[r], d, 0, 0, 0);
  };
  const f32x4 none = {0.f, 0.f, 0.f, 0.f};
  for (int step = 0; step < steps; step++) {
    f32x4 A[RB][RB], R[RB][RB];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
      for (int j = 0; j < RB; j++) {
        A[i][j] = none;
#pragma unroll
        for (int u = 0; u < U; u++)
          if (16 * (wave + NW * u) < M.l) multiply(along[u][i], along[u][j], A[i][j]);
      }
    if constexpr (NW > 1) {
      f32x4* const s = parts + (TWICE ? 0 : (step & 1) * NW * Q * 64) + lane;
#pragma unroll
      for (int k = 0; k < Q; k++) s[(wave * Q + k) * 64] = A[k / RB][k % RB];
      __syncthreads();
      if constexpr (TWICE) {
        static_assert(Q <= NW, "a wave a block");
        if (wave < Q) {
          f32x4 d = s[wave * 64];
#pragma unroll
          for (int w = 1; w < NW; w++) d += s[(w * Q + wave) * 64];
          s[(NW * Q + wave) * 64] = d;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < Q; k++) A[k / RB][k % RB] = s[(NW * Q + k) * 64];
      } else {
#pragma unroll
        for (int k = 0; k < Q; k++) {
          A[k / RB][k % RB] = s[k * 64];
#pragma unroll
          for (int w = 1; w < NW; w++) A[k / RB][k % RB] += s[(w * Q + k) * 64];
        }
      }
    }
    // block (i, j) as lanes hold it is also block (j, i) as an instruction's left side
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
      for (int j = 0; j < RB; j++) {
        R[i][j] = none;
#pragma unroll
        for (int k = 0; k < RB; k++) multiply(A[k][i], A[k][j], R[i][j]);
#pragma unroll
        for (int r = 0; r < 4; r++) R[i][j][r] = fmaf(c, R[i][j][r], b * A[i][j][r]);
      }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (16 * (wave + NW * u) >= M.l) continue;
      f32x4 x[RB], y[RB];
#pragma unroll
      for (int i = 0; i < RB; i++) {
        x[i] = y[i] = none;
#pragma unroll
        for (int k = 0; k < RB; k++) {
          multiply(R[k][i], down[u][k], x[i]);
          if constexpr (!TURN) multiply(down[u][k], R[k][i], y[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < RB; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          down[u][i][r] = fmaf(a, down[u][i][r], x[i][r]);
          if constexpr (!TURN) along[u][i][r] = fmaf(a, along[u][i][r], y[i][r]);
        }
      if constexpr (TURN) {
        float* const t = turns + wave * (16 * 20);
#pragma unroll
        for (int i = 0; i < RB; i++) {
          *(f32x4*)(t + n * 20 + 4 * q) = down[u][i];
#pragma unroll
          for (int r = 0; r < 4; r++) along[u][i][r] = t[(4 * q + r) * 20 + n];
        }
      }
    }
  }
  // four neighbours of a row of G's a lane
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int i = 0; i < RB; i++) {
      const f32x4 v = M.tall ? down[u][i] : along[u][i];
      const int col = 16 * (wave + NW * u), row = M.tall ? col + n : 16 * i + n, at = M.tall ? 16 * i + 4 * q : col + 4 * q;
#pragma unroll
      for (int r = 0; r < 4; r++)
        if (row < M.rows && at + r < M.cols) {
          const long e = at0 + (long)row * M.cols + at + r;
          if constexpr (BF16) ((bf16_t*)dst)[e] = (bf16_t)v[r];
          else ((float*)dst)[e] = v[r];
        }
    }
}

// ------------------------------------------------------------------------------------------------ one workgroup a matrix
// A small matrix whole in LDS (X and one square of it, split and laid out as in memory), one launch for everything: 64 x 512 takes 68 us,
// 128 x 96 52, and by launches 90 to 100, next to none of it work.
// What bounds it is one CU's chain of dependent products, fifteen of them with a barrier or two each.  NW waves deal the
// 32 x 32 blocks of a product among them (no mirror images: the whole squares are computed); a product that overwrites what it
// reads keeps its blocks in registers until everybody has read.
// Eight waves up to 64 rows, sixteen (which spill) above, us a call in a row of calls: a thousand of 64 x 512 305 (with sixteen 383), one
// 128 x 160 69 with sixteen and 75 with eight; a thousand of 128 x 160 the other way round, 398 and 312.
#define NS_SMALL_LDS 163840
#define NS_TINY_LDS 32768

template <int BYTES, bool BF16, int NW>
__global__ __launch_bounds__(64 * NW) void ns_small_kernel(const void* __restrict__ src, void* __restrict__ dst, NsMat one, long stride,
                                                       int steps, float a, float b, float c, float eps, NsShift shift) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[BYTES == NS_SMALL_LDS ? BYTES - 128 : BYTES];
  __shared__ double part[NW];
  // blocks of X (4 sp lp + 4 sp^2 <= BYTES leaves at most 39, or 7) and of a square a wave
  constexpr int NX = ((BYTES == NS_SMALL_LDS ? 39 : 7) + NW - 1) / NW, NQ = ((BYTES == NS_SMALL_LDS ? 16 : 4) + NW - 1) / NW;
  const NsMat& M = one;
  const long at0 = (long)blockIdx.x * stride, n = (long)M.rows * M.cols;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 31, fh = lane >> 5, sb = M.sp >> 5, lb = M.lp >> 5, skb = M.sp >> 4, lkb = M.lp >> 4;
  unsigned char *X = smem, *S = smem + 4 * M.sp * M.lp;
  // X0: eight columns of X an item, read once and kept while the norm is put together
  constexpr int ITEMS = (BYTES / 4 / 8 + 64 * NW - 1) / (64 * NW);
  float v0[ITEMS][8];
  double sum = 0.0;
#pragma unroll
  for (int u = 0; u < ITEMS; u++) {
    const int item = tid + 64 * NW * u, row = item / (M.lp / 8), col = (item - row * (M.lp / 8)) * 8;
    const long e = M.tall ? at0 + (long)col * M.cols + row : at0 + (long)row * M.cols + col;
    const bool in = row < M.s;
    if (!M.tall && in && col + 8 <= M.l) {
      if constexpr (BF16) {
        bf16_t h[8];
        __builtin_memcpy(h, (const bf16_t*)src + e, 16);
#pragma unroll
        for (int k = 0; k < 8; k++) v0[u][k] = to_f32(h[k]);
      } else {
        __builtin_memcpy(v0[u], (const float*)src + e, 32);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const long ek = e + (M.tall ? (long)k * M.cols : k);
        v0[u][k] = !in || col + k >= M.l ? 0.f : BF16 ? to_f32(((const bf16_t*)src)[ek]) : ((const float*)src)[ek];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < ITEMS; u++)
#pragma unroll
    for (int k = 0; k < 8; k++) sum += (double)v0[u][k] * (double)v0[u][k];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int w = 0; w < NW; w++) sum += part[w];
  double size;
  const float inv = ns_start(shift, sqrt(sum), eps, size);
#pragma unroll
  for (int u = 0; u < ITEMS; u++) {
    const int item = tid + 64 * NW * u, row = item / (M.lp / 8), col = (item - row * (M.lp / 8)) * 8;
    if (row >= M.sp) continue;
    f16x8 h, l;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      _Float16 hh, ll;
      ns_split(v0[u][k] * inv, hh, ll);
      h[k] = hh;
      l[k] = ll;
    }
    *(f16x8*)(X + ns_chunk(row, col, 0, lkb)) = h;
    *(f16x8*)(X + ns_chunk(row, col, 1, lkb)) = l;
  }
  __syncthreads();
  // e(0) .. e(63) in the sums' place, read behind the barrier of the first product
  static_assert(sizeof part >= NS_MAX_STEPS, "a byte each");
  unsigned char* const shifts = (unsigned char*)part;
  if (wave == 0) {
    shifts[lane] = 0;
    if (lane == 0) ns_shifts(shift, size, steps, shifts);
  }
  // hi and lo of the rows 32 i .. + 31, columns 16 k .. + 15 of a matrix, as an operand
  auto rows_of = [&](const unsigned char* P, int kb, int i, int k, f16x8& h, f16x8& l) {
    const unsigned char* p = P + ((2 * i + (fr >> 4)) * kb + k) * 1024 + (fr & 15) * 64 + ((fh ^ ((fr >> 2) & 3) ^ ((k & 1) << 1)) << 4);
    h = *(const f16x8*)p;
    l = *(const f16x8*)(smem + ((p - smem) ^ 32));
  };
  // the same of the columns 32 j .. + 31 of X, rows 16 k .. + 15 (transposing read)
  auto columns_of = [&](int j, int k, f16x8& h, f16x8& l) {
    const int tq = (lane & 15) >> 2, tp = lane & 3, odd = (lane >> 4) & 1;
    const int o = (k * lkb + 2 * j + odd) * 1024 + (8 * fh + tq) * 64 + (((tp >> 1) ^ (2 * fh) ^ (2 * odd)) << 4) + 8 * (tp & 1);
    const int o2 = (o + 256) ^ 16;
    const s16x4 h0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(X + o));
    const s16x4 h1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(X + o2));
    const s16x4 l0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(X + (o ^ 32)));
    const s16x4 l1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(X + (o2 ^ 32)));
    h = __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7));
    l = __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  f32x16 acc[NX > NQ ? NX : NQ];
  // kind 0: X X^T, 1: S S, 2: S X, steps k0 to k1; block number first + NW u of the result.  The large and the small
  // products go into sums of their own: one chain would be three latencies long a step.
  struct Pair { f16x8 ah, al, bh, bl; };
  auto product = [&](auto kind, auto most, int blocks, int cols, int first, int k0, int k1) __attribute__((always_inline)) {
    constexpr int KIND = decltype(kind)::value, MOST = decltype(most)::value;
    ns_unroll<MOST>([&](auto uu) __attribute__((always_inline)) {
      constexpr int u = decltype(uu)::value;
      const int id = first + NW * u;
      if (id >= blocks) return;
      const int i = id / cols, j = id - i * cols;
      auto load = [&](Pair& f, int k) __attribute__((always_inline)) {
        rows_of(KIND == 0 ? X : S, KIND == 0 ? lkb : skb, i, k, f.ah, f.al);
        if constexpr (KIND == 2) columns_of(j, k, f.bh, f.bl);
        else rows_of(KIND == 0 ? X : S, KIND == 0 ? lkb : skb, j, k, f.bh, f.bl);
      };
      f32x16 low;
#pragma unroll
      for (int r = 0; r < 16; r++) low[r] = acc[u][r] = 0.f;
      auto multiply = [&](const Pair& f) __attribute__((always_inline)) {
        low = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.bl, f.ah, low, 0, 0, 0);
        acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.bh, f.ah, acc[u], 0, 0, 0);
        low = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.bh, f.al, low, 0, 0, 0);
      };
      Pair f0, f1;
      if (k0 < k1) load(f0, k0);
      for (int k = k0; k < k1; k += 2) {                     // the next step's operands are read under this one's products
        if (k + 1 < k1) load(f1, k + 1);
        multiply(f0);
        if (k + 2 < k1) load(f0, k + 2);
        if (k + 1 < k1) multiply(f1);
      }
#pragma unroll
      for (int r = 0; r < 16; r++) acc[u][r] += low[r] * (1.f / NS_LOW);
    });
  };
  // the lane's values of block u, 16-byte chunk by chunk (columns 32 j + 16 p + 8 fh ..): f(v[8], row, column, number)
  auto each = [&](auto most, int blocks, int cols, int first, auto f) __attribute__((always_inline)) {
    ns_unroll<2 * decltype(most)::value>([&](auto at) __attribute__((always_inline)) {
      constexpr int u = decltype(at)::value / 2, p = decltype(at)::value % 2;
      const int id = first + NW * u;
      if (id >= blocks) return;
      const int i = id / cols, j = id - i * cols;
      float v[8];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float s0 = acc[u][8 * p + r], s1 = acc[u][8 * p + 4 + r];
        const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(s0), __float_as_uint(s1), false, false);
        v[r] = __uint_as_float(w[0]) * (1.f / NS_SCALE);
        v[4 + r] = __uint_as_float(w[1]) * (1.f / NS_SCALE);
      }
      f(v, 32 * i + fr, 32 * j + 16 * p + 8 * fh, at);
    });
  };
  auto store = [&](unsigned char* P, int kb, const float (&v)[8], int row, int col) {
    f16x8 h, l;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      _Float16 hh, ll;
      ns_split(v[e], hh, ll);
      h[e] = hh;
      l[e] = ll;
    }
    *(f16x8*)(P + ns_chunk(row, col, 0, kb)) = h;
    *(f16x8*)(P + ns_chunk(row, col, 1, kb)) = l;
  };
  auto add = [&](float (&v)[8], const unsigned char* P, int kb, int row, int col, float f) {
    const f16x8 h = *(const f16x8*)(P + ns_chunk(row, col, 0, kb)), l = *(const f16x8*)(P + ns_chunk(row, col, 1, kb));
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] += f * ns_join(h[e], l[e]);
  };
  using K0 = std::integral_constant<int, 0>;
  using K1 = std::integral_constant<int, 1>;
  using K2 = std::integral_constant<int, 2>;
  using NQs = std::integral_constant<int, NQ>;
  using NXs = std::integral_constant<int, NX>;
  const int slices = max(1, min(min(8, NW / (sb * sb)), lkb / 4));
  for (int step = 0; step < steps; step++) {
    // A = X X^T has few blocks and a long reduction: `slices` waves share a block, each adding its part to what the one before it
    // left in the block's own place
    const int nb = sb * sb, part_of = wave / nb, block = part_of < slices ? wave - part_of * nb : nb;
    product(K0{}, NQs{}, nb, sb, block, lkb * part_of / slices, lkb * (part_of + 1) / slices);
    for (int t = 0; t + 1 < slices; t++) {
      f32x4* mine = (f32x4*)(S + block * 4096) + lane;
      if (block < nb && part_of == t)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          f32x4 v;
#pragma unroll
          for (int r = 0; r < 4; r++) v[r] = acc[0][4 * g + r];
          mine[64 * g] = v;
        }
      __syncthreads();
      if (block < nb && part_of == t + 1)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const f32x4 v = mine[64 * g];
#pragma unroll
          for (int r = 0; r < 4; r++) acc[0][4 * g + r] += v[r];
        }
      __syncthreads();
    }
    each(NQs{}, part_of == slices - 1 ? nb : 0, sb, block, [&](float (&v)[8], int row, int col, auto) __attribute__((always_inline)) {
      store(S, skb, v, row, col);
    });
    __syncthreads();
    product(K1{}, NQs{}, sb * sb, sb, wave, 0, skb);
    // R = b A + c A A, kept in the accumulators' place until every wave has read A
    const float bs = ldexpf(b, -2 * shifts[step]), cs = ldexpf(c, -4 * shifts[step]);
    float keep[2 * NQ][8];
    each(NQs{}, sb * sb, sb, wave, [&](float (&v)[8], int row, int col, auto at) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] *= cs;
      add(v, S, skb, row, col, bs);
#pragma unroll
      for (int e = 0; e < 8; e++) keep[decltype(at)::value][e] = v[e];
    });
    __syncthreads();
    each(NQs{}, sb * sb, sb, wave, [&](float (&)[8], int row, int col, auto at) __attribute__((always_inline)) {
      store(S, skb, keep[decltype(at)::value], row, col);
    });
    __syncthreads();
    product(K2{}, NXs{}, sb * lb, lb, wave, 0, skb);
    __syncthreads();                                         // X has been read: a X is added from a block's own place
    const float f = ldexpf(1.f, step + 1 < steps ? shifts[step + 1] - shifts[step] : 0), as = a * f;
    each(NXs{}, sb * lb, lb, wave, [&](float (&v)[8], int row, int col, auto) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] *= f;
      add(v, X, lkb, row, col, as);
      store(X, lkb, v, row, col);
    });
    __syncthreads();
  }
  const float unit = ldexpf(1.f / NS_SCALE, -shifts[steps - 1]);
  // out of the split form (22 bits: a last rounding of 2^-23), along the user's rows
  for (long e = tid; e < n; e += 64 * NW) {
    const int r = (int)(e / M.cols), cc = (int)(e - (long)r * M.cols), row = M.tall ? cc : r, col = M.tall ? r : cc;
    const unsigned char* at = X + ns_chunk(row, col & ~7, 0, lkb) + (col & 7) * 2;
    const float v = ns_join(*(const _Float16*)at, *(const _Float16*)(smem + ((at - smem) ^ 32))) * unit;
    if constexpr (BF16) ((bf16_t*)dst)[at0 + e] = (bf16_t)v;
    else ((float*)dst)[at0 + e] = v;
  }
}

// Whatever else fits goes through LDS.  Both ways measured, fp32, single calls from an idle GPU (some 10 us of which are the way there):
// one matrix 64 x 512 78 us (by launches 117), 32 x 1216 79 (116), 128 x 160 77 (108); a thousand 64 x 512 321 (664), 128 x 160 383 (766).
static inline long ns_small_bytes(const NsMat& m) { return 4L * m.sp * m.lp + 4L * m.sp * m.sp; }
// Up to 32 rows in registers, fp32.  Both ways measured, calls in a row, through LDS as split fp16 and here: one 16 x 16 17 us and 11, 16 x
// 128 21 and 12, 16 x 2000 104 (by launches) and 58, 32 x 128 21 and 20, 32 x 512 45 and 46, 32 x 1000 64 and 83; a thousand 16 x 128 47 and 21,
// 32 x 32 37 and 26, 32 x 224 63 and 80, 32 x 256 122 and 82, 32 x 512 177 and 152, 32 x 1000 262 and 360.  From 512 columns on it is the error that decides (1.2 times an
// fp32 iteration's and 0.9), which a bf16 result does not show.
static inline bool ns_rows(const NsMat& m) { return m.s <= 32 && m.l <= (m.s <= 16 ? 2048 : 1024); }
static inline bool ns_rows(const NsMat& m, int dtype) { return ns_rows(m) && (m.s <= 16 || m.l <= 512 || dtype == MADIFF_F32); }
static inline bool ns_small(const NsMat& m) { return ns_rows(m) || (m.sp <= 128 && ns_small_bytes(m) <= NS_SMALL_LDS - 128); }

// ------------------------------------------------------------------------------------------------ host
struct NsPlan {                    // start of a plan; matrices and lists follow
  long magic, bytes, ws_bytes, need, partials;       // need: elements the flat buffers must have
  int mats, chunks, areas, shape[3], works[3], counters, pairs, pad_;
  long at_mats, at_chunks, at_areas, at_works[3];
};
static const long NS_MAGIC = 0x6d7502;

static bool ns_describe(NsMat& m, long at, int rows, int cols, float scale, long& ws) {
  if (rows < 1 || cols < 1 || at < 0 || at > LONG_MAX - (long)rows * cols) return false;
  m.at = at;
  m.rows = rows;
  m.cols = cols;
  m.tall = rows > cols;
  m.s = m.tall ? cols : rows;
  m.l = m.tall ? rows : cols;
  if (m.s > NS_MAX_SHORT || m.l > NS_MAX_LONG) return false;
  m.sp = ns_div_up(m.s, NS_PAD) * NS_PAD;
  m.lp = ns_div_up(m.l, NS_PAD) * NS_PAD;
  const long parts = ((long)rows * cols + NS_CHUNK - 1) / NS_CHUNK;
  m.parts = (int)parts;
  m.scale = scale;
  m.pad_ = 0.f;
  m.x = ws;
  ws += 2L * m.sp * m.lp * 4;
  m.sq = ws;
  ws += 4L * m.sp * m.sp * 4;
  m.norm = ws;
  ws += (parts * 8 + NS_MAX_STEPS + 1 + 255) / 256 * 256;
  return true;
}

// ---- which tile, and how many parts.  Two tile shapes; what one workgroup takes, in microseconds, as measured on an MI355X: a K-step
// with two workgroups on every CU and with one, the rest of a tile (first loads, ending), the same for a part.  64 x 64 gives
// the most workgroups (5 of 256 x 2048: A A 6.2 us where 128 x 128 takes 11.8), 128 x 128 loads half as much for the same work
// (28 of 1024 x 1024: R X 189 us where 64 x 64 takes 275).  256 x 256 with one workgroup a CU reaches four fifths of the matrix rate in
// its loop but loses it again to its ending and to unfilled rounds (200 us there), 128 x 256 likewise: neither is kept.  Parts pay
// where there are few tiles (1024 x 5120 alone: A = X X^T 82 us whole, 28 us in three parts).
struct NsShape { int bm, bn; double full, alone, rest, part; };
static const NsShape ns_shapes[2] = {{64, 64, 0.25, 0.127, 4.0, 3.0}, {128, 128, 0.70, 0.39, 8.0, 5.0}};
static inline int ns_ksteps(int kind, int sp, int lp) { return (kind == NS_GRAM ? lp : sp) / 16; }
static inline int ns_tiles_of(int kind, int shape, int sp, int lp) {
  return ns_tiles(kind == NS_APPLY, sp, lp, ns_shapes[shape].bm, ns_shapes[shape].bn);
}
static inline int ns_parts(int ksteps, int len) {             // parts of about `len` steps, two at least each
  const int most = ksteps / 2, p = (ksteps + len / 2) / len;
  return p < 1 ? 1 : (p > most ? most : (p > 64 ? 64 : p));
}
static inline double ns_tile_time(const NsShape& s, int ksteps, int parts, bool alone) {
  return (double)ksteps / parts * (alone ? s.alone : s.full) + (parts > 1 ? s.part : s.rest);
}
// a tile's last workgroup fetches the sums of all its parts; everything written and read
static inline double ns_join_time(const NsShape& s, int parts, double all) {
  return parts > 1 ? 4.0 + parts * s.bm * s.bn * 4 / 50e3 + all * s.bm * s.bn * 4 / 4.5e6 : 0.0;
}
static const int NS_SLOTS = 512;                              // two workgroups a CU
static const int ns_lens[] = {1 << 30, 512, 320, 256, 192, 160, 128, 112, 96, 80, 64, 56, 48, 40, 32, 24, 16, 12, 8};

// `batch` equal matrices
static void ns_choose(int kind, int batch, int sp, int lp, int& shape, int& parts) {
  const int ks = ns_ksteps(kind, sp, lp);
  double best = -1.0;
  for (int s = 0; s < 2; s++)
    for (int len : ns_lens) {
      const int p = ns_parts(ks, len);
      const double tiles = (double)batch * ns_tiles_of(kind, s, sp, lp), n = tiles * p;
      if (n > (double)NS_MAX_GROUPS) continue;             // (one part a tile of 64 x 64 always fits)
      const double rounds = n <= NS_SLOTS ? 1.0 : n / NS_SLOTS + 0.25;
      const double t = rounds * ns_tile_time(ns_shapes[s], ks, p, n <= 256.0) + ns_join_time(ns_shapes[s], p, n);
      if (best < 0.0 || t < best) { best = t; shape = s; parts = p; }
    }
}

// Two steps in one: one A and one pass over X saved against four square products more.  For equal matrices it goes by their sides alone,
// so that a matrix gets the same form alone, in a batch and in what is left of one.  Step by step and in twos, us: 12 x 333 x 1001 220
// and 205, one of them 130 and 139; 12 x 1024 x 2048 1444 and 1303, one 254 and 255; 7 x 1024 x 5120 1927 and 1450; below twice as long
// 24 x 333 x 500 241 and 244, one 118 and 131, 12 x 1024 x 1500 1183 and 1159, one 233 and 244.  A plan, whose launches hold all
// its matrices, has one form for them all, by the time of its launches.
static inline bool ns_pairs(int sp, int lp) { return lp >= 2 * sp; }
static inline bool ns_pairs(const double (&time)[3]) { return time[NS_GRAM] + time[NS_APPLY] > 4.0 * time[NS_SQUARE]; }

struct NsRun {                     // one call
  NsGroup grp;
  const int *chunks, *areas;       // norm and split passes: (matrix, chunk), (matrix, ti, tj, 0); null: numbered
  int n_chunks, per_chunks, n_areas, per_areas;
  int shape[3];
  bool pairs;                      // two steps in one go are the faster
  NsList work[3];
};

template <int KIND, int OUT, int BM, int BN, int D>
static void ns_go(const NsRun& r, const NsProduct& q, hipStream_t st) {
  hipLaunchKernelGGL((ns_product_kernel<KIND, BM, BN, 2, 2, D, OUT>), dim3(r.work[KIND].n), dim3(256), 0, st, r.grp, q, r.work[KIND]);
}
template <int KIND, int OUT>
static void ns_launch(const NsRun& r, const NsProduct& q, hipStream_t st) {
  if (r.shape[KIND] == 1) ns_go<KIND, OUT, 128, 128, 4>(r, q, st);
  else ns_go<KIND, OUT, 64, 64, 8>(r, q, st);
}
template <int KIND>
static void ns_launch_source(const NsRun& r, const NsSource& q, hipStream_t st) {
  hipLaunchKernelGGL((ns_norm_kernel<KIND>), dim3(r.n_chunks), dim3(1024), 0, st, r.grp, q, r.chunks, r.per_chunks);
  hipLaunchKernelGGL((ns_split_kernel<KIND>), dim3(r.n_areas), dim3(256), 0, st, r.grp, q, r.areas, r.per_areas);
}

// out: NS_OUT_F32 / BF16 / MUON for the last product; `last` holds its destination.
// pairs: two steps share one A = X X^T and one product with X.  With R = b A + c A A and everything a polynomial in A,
//   A' = (a + R)^2 A = a T + R T,  T = a A + R A        R' = b A' + c A' A'        X'' = a^2 X + P X,  P = R' R + a R + a R'
// six square products for two and two passes over X for four.  A' carries the rounding of A rather than that of a new X X^T: the
// result is 1.3 to 1.8 times as far from the 64-bit one as step by step, which is nothing next to a rounding to bf16 or an
// update of fp32 weights, and is not done for an fp32 result.
static int ns_iterate(const NsRun& r, int steps, float a, float b, float c, int out, const NsProduct& last, bool pairs,
                      hipStream_t st) {
  enum { G = 0, R = 1, T = 2, R2 = 3 };
  auto square = [&](int x, int y, float ca, float c1, int e2, float c2, int to, int shift = -1) {   // to = ca x y + c1 y + c2 e2
    NsProduct q = {};
    q.step = shift;
    q.a = x;
    q.b = y;
    q.ca = ca;
    q.c1 = c1;
    q.e2 = e2;
    q.c2 = c2;
    q.out = to;
    ns_launch<NS_SQUARE, NS_OUT_PLANES>(r, q, st);
  };
  int x = 0;
  for (int k = 0; k < steps;) {
    const bool two = pairs && k + 2 <= steps;
    NsProduct q = {};
    q.b = x;
    q.out = G;
    q.ca = 1.f;
    ns_launch<NS_GRAM, NS_OUT_PLANES>(r, q, st);
    square(G, G, c, b, -1, 0.f, R, k);
    if (two) {
      square(R, G, 1.f, a, -1, 0.f, T);
      square(R, T, 1.f, a, -1, 0.f, G);
      square(G, G, c, b, -1, 0.f, R2, k);
      square(R2, R, 1.f, a, R2, a, T);
    }
    const int from = k;
    k += two ? 2 : 1;
    q = k >= steps ? last : NsProduct{};
    q.step = from;
    q.then = k;
    q.a = two ? T : R;
    q.b = x;
    q.out = x ^ 1;
    q.ca = 1.f;
    q.c1 = two ? a * a : a;
    if (k < steps) ns_launch<NS_APPLY, NS_OUT_PLANES>(r, q, st);
    else if (out == NS_OUT_F32) ns_launch<NS_APPLY, NS_OUT_F32>(r, q, st);
    else if (out == NS_OUT_BF16) ns_launch<NS_APPLY, NS_OUT_BF16>(r, q, st);
    else ns_launch<NS_APPLY, NS_OUT_MUON>(r, q, st);
    x ^= 1;
    MADIFF_CHECK_LAUNCH();
  }
  return 0;
}

// The polynomial's orbit from every start in [0, 1]: the largest |x|, |A| and |R| on it, and what pairs of steps store besides,
// have to stay in the stored range.  `most`: the largest |x|.
static bool ns_bounded(int steps, float a, float b, float c, bool pairs, double& most) {
  most = 1.0;
  const double top = 65504.0 / NS_SCALE / 2;
  auto in = [&](double v) { return v < top && v > -top; };
  for (int i = 0; i <= 4096; i++) {
    double x = (double)i / 4096, before = 0.0;
    for (int k = 0; k < steps; k++) {
      const double g = x * x, q = b * g + c * g * g;
      x = x * (a + q);
      most = fmax(most, fabs(x));
      if (!(in(x) && in(g) && in(q))) return false;
      if (pairs && !(in((a + q) * g) && (k % 2 == 0 || in((a + q) * (a + before) - (double)a * a)))) return false;
      before = q;
    }
  }
  return true;
}

// the same, remembered per thread for the last polynomial: walking the orbits takes longer than a small call
struct NsOrbit { int steps; float a, b, c; bool fits; double most; };
static const NsOrbit& ns_orbit(int steps, float a, float b, float c, bool pairs) {
  static thread_local NsOrbit last[2] = {{-1, 0.f, 0.f, 0.f, false, 0.0}, {-1, 0.f, 0.f, 0.f, false, 0.0}};
  NsOrbit& l = last[pairs];
  if (l.steps != steps || l.a != a || l.b != b || l.c != c) {
    l = {steps, a, b, c, false, 0.0};
    l.fits = ns_bounded(steps, a, b, c, pairs, l.most);
  }
  return l;
}
static bool ns_fits(int steps, float a, float b, float c, bool pairs) { return ns_orbit(steps, a, b, c, pairs).fits; }
static NsShift ns_shift_of(int steps, float a, float b, float c, float eps) {
  return {a, b, c, c != 0.f ? -b / (2.f * c) : -1.f, (float)ns_orbit(steps, a, b, c, false).most * 1.01f, 115 + ilogbf(eps)};
}

extern "C" int madiff_ortho_check(int steps, float a, float b, float c, float eps) {
  // (eps: 2^11 over it has to be an fp32 number, or a matrix of zeros would come out as NaN)
  return steps >= 1 && steps <= NS_MAX_STEPS && eps >= 1e-30f && eps < 1e30f && ns_fits(steps, a, b, c, false) ? 0 : -1;
}

// Everything about a call on `batch` equal matrices but its pointers
static int ns_uniform(int batch, int rows, int cols, NsRun& r, long& ws_bytes) {
  NsMat& m = r.grp.one;
  long ws = 0;
  if (batch < 0 || !ns_describe(m, 0, rows, cols, 1.f, ws)) return -1;
  const long areas = (long)ns_div_up(m.sp, 64) * ns_div_up(m.lp, 64);
  if (batch > 0 && (areas > NS_MAX_GROUPS / batch || m.parts > NS_MAX_GROUPS / batch)) return -1;
  r.grp.ws_stride = ws;
  r.grp.at_stride = (long)rows * cols;
  r.grp.partials = ws * batch;
  r.per_chunks = m.parts;
  r.n_chunks = batch * m.parts;
  r.per_areas = (int)areas;
  r.n_areas = batch * (int)areas;
  if (ns_small(m)) {               // everything in LDS
    ws_bytes = 0;
    return 0;
  }
  long slots = 0;
  for (int k = 0; k < 3; k++) {
    int parts = 1;
    ns_choose(k, batch, m.sp, m.lp, r.shape[k], parts);
    const int tiles = ns_tiles_of(k, r.shape[k], m.sp, m.lp);
    r.work[k] = {nullptr, batch * tiles * parts, tiles, parts};
    if (parts > 1 && r.work[k].n > r.grp.n_counters) r.grp.n_counters = r.work[k].n;
    const long bytes = parts > 1 ? (long)r.work[k].n * ns_shapes[r.shape[k]].bm * ns_shapes[r.shape[k]].bn * 4 : 0;
    slots = bytes > slots ? bytes : slots;
  }
  r.pairs = ns_pairs(m.sp, m.lp);
  r.grp.counters = ws * batch + slots;
  ws_bytes = r.grp.counters + ((long)r.grp.n_counters * 4 + 255) / 256 * 256;
  return 0;
}

extern "C" int madiff_ortho_ws(int batch, int rows, int cols, long* ws_bytes) {
  NsRun r = {};
  return ws_bytes ? ns_uniform(batch, rows, cols, r, *ws_bytes) : -1;
}

extern "C" int madiff_orthogonalize(int dtype, const void* src, void* dst, int batch, int rows, int cols, int steps, float a,
                                    float b, float c, float eps, void* ws, long ws_bytes, hipStream_t stream) {
  NsRun r = {};
  long need = 0;
  if ((dtype != MADIFF_F32 && dtype != MADIFF_BF16) || ns_uniform(batch, rows, cols, r, need) ||
      madiff_ortho_check(steps, a, b, c, eps))
    return -1;
  if (batch == 0) return 0;
  if (!src || !dst || (need > 0 && (!ws || ws_bytes < need || ((size_t)ws & 255)))) return -1;
  const NsMat& m = r.grp.one;
  const NsShift shift = ns_shift_of(steps, a, b, c, eps);
  if (ns_small(m)) {
#define NS_GO(BYTES, BF16, NW)                                                                                                    \
  hipLaunchKernelGGL((ns_small_kernel<BYTES, BF16, NW>), dim3(batch), dim3(64 * NW), 0, stream, src, dst, m, r.grp.at_stride, steps, \
                     a, b, c, eps, shift)
#define NS_ANY(BYTES, NW) do { if (dtype == MADIFF_BF16) NS_GO(BYTES, true, NW); else NS_GO(BYTES, false, NW); } while (0)
#define NS_ROWS(BF16, RB, NW, U)                                                                                                      \
  hipLaunchKernelGGL((ns_rows_kernel<BF16, RB, NW, U>), dim3(batch), dim3(64 * NW), 0, stream, src, dst, m, r.grp.at_stride, steps, a, b, c, \
                     eps)
#define NS_ANY_ROWS(RB, NW, U) do { if (dtype == MADIFF_BF16) NS_ROWS(true, RB, NW, U); else NS_ROWS(false, RB, NW, U); } while (0)
    if (ns_rows(m, dtype) && m.s <= 16) {
      if (m.l <= 32) NS_ANY_ROWS(1, 1, 2);
      else if (m.l <= 128) NS_ANY_ROWS(1, 4, 2);
      else if (m.l <= 512) NS_ANY_ROWS(1, 8, 4);
      else NS_ANY_ROWS(1, 16, 8);
    } else if (ns_rows(m, dtype)) {
      if (m.l <= 64) NS_ANY_ROWS(2, 4, 1);
      else if (m.l <= 128) NS_ANY_ROWS(2, 4, 2);
      else if (m.l <= 256) NS_ANY_ROWS(2, 4, 4);
      else if (m.l <= 512) NS_ANY_ROWS(2, 8, 4);
      else NS_ROWS(false, 2, 8, 8);
    } else if (ns_small_bytes(m) <= NS_TINY_LDS) NS_ANY(NS_TINY_LDS, 8);    // several workgroups a CU
    else if (m.sp <= 64) NS_ANY(NS_SMALL_LDS, 8);
    else NS_ANY(NS_SMALL_LDS, 16);
#undef NS_ANY
#undef NS_GO
#undef NS_ANY_ROWS
#undef NS_ROWS
    MADIFF_CHECK_LAUNCH();
    return 0;
  }
  r.grp.ws = (unsigned char*)ws;
  NsSource q = {};
  q.src = src;
  q.eps = eps;
  q.steps = steps;
  q.shift = shift;
  if (dtype == MADIFF_BF16) ns_launch_source<1>(r, q, stream);
  else ns_launch_source<0>(r, q, stream);
  MADIFF_CHECK_LAUNCH();
  NsProduct last = {};
  last.dst = dst;
  const bool pairs = dtype == MADIFF_BF16 && r.pairs && ns_fits(steps, a, b, c, true);
  return ns_iterate(r, steps, a, b, c, dtype == MADIFF_BF16 ? NS_OUT_BF16 : NS_OUT_F32, last, pairs, stream);
}

// ---- Muon plans: a host blob that is copied to the device as it is
namespace {
// What the chip needs for a product over all matrices with a tile shape and a part length: list scheduling, longest first
double ns_plan_time(const std::vector<NsMat>& mats, int kind, int shape, int len) {
  const NsShape& s = ns_shapes[shape];
  std::vector<std::pair<double, long>> runs;                 // duration, how many
  double n = 0.0, joined = 0.0;
  int most = 1;
  for (const NsMat& m : mats) n += (double)ns_tiles_of(kind, shape, m.sp, m.lp) * ns_parts(ns_ksteps(kind, m.sp, m.lp), len);
  double total = 0.0;
  for (const NsMat& m : mats) {
    const int ks = ns_ksteps(kind, m.sp, m.lp), p = ns_parts(ks, len);
    const long c = (long)ns_tiles_of(kind, shape, m.sp, m.lp) * p;
    const double d = ns_tile_time(s, ks, p, n <= 256.0);
    runs.push_back({d, c});
    total += d * c;
    if (p > 1) joined += c;
    most = p > most ? p : most;
  }
  double end = total / NS_SLOTS;
  if (n < 3000.0) {
    std::sort(runs.begin(), runs.end(), [](auto& x, auto& y) { return x.first > y.first; });
    std::priority_queue<double, std::vector<double>, std::greater<double>> free;
    for (int i = 0; i < NS_SLOTS; i++) free.push(0.0);
    end = 0.0;
    for (const auto& r : runs)
      for (long i = 0; i < r.second; i++) {
        const double t = free.top() + r.first;
        free.pop();
        free.push(t);
        end = t > end ? t : end;
      }
  }
  return end + ns_join_time(s, most, joined);
}

// The order of one list: runs of neighbouring tiles of a matrix go to the XCD with the least work so far, the costly runs first;
// the XCDs' queues, long reductions first, are then dealt out in turn (workgroup i starts on XCD i % 8), mat = -1 filling the gaps.
int ns_order(const std::vector<NsMat>& mats, int kind, std::vector<NsWork>& out, int& slots, long& partial_bytes, double& best) {
  int shape = 0, len = 1 << 30;
  best = -1.0;
  for (int s = 0; s < 2; s++)
    for (int l : ns_lens) {
      const double t = ns_plan_time(mats, kind, s, l);
      if (best < 0.0 || t < best) { best = t; shape = s; len = l; }
    }
  const NsShape& sh = ns_shapes[shape];
  struct Run { int mat, lo, hi; double cost; };              // works [lo, hi) of a matrix: part by part, tile by tile
  std::vector<Run> runs;
  std::vector<std::vector<NsWork>> works(mats.size());
  double total = 0.0;
  slots = 0;
  auto cost = [&](const NsWork& w) {
    return ns_tile_time(sh, ns_ksteps(kind, mats[w.mat].sp, mats[w.mat].lp), w.parts, false);
  };
  for (int i = 0; i < (int)mats.size(); i++) {
    const NsMat& m = mats[i];
    const int tiles = ns_tiles_of(kind, shape, m.sp, m.lp), parts = ns_parts(ns_ksteps(kind, m.sp, m.lp), len);
    for (int p = 0; p < parts; p++)
      for (int t = 0; t < tiles; t++) {
        NsWork w = {i, 0, 0, p, parts, parts > 1 ? slots + t * parts : 0, 0, 0};
        ns_tile_at(kind == NS_APPLY, t, m.sp, m.lp, sh.bm, sh.bn, w.ti, w.tj);
        works[i].push_back(w);
        total += cost(w);
      }
    if (parts > 1) slots += tiles * parts;
  }
  partial_bytes = (long)slots * sh.bm * sh.bn * 4;
  for (int i = 0; i < (int)mats.size(); i++) {
    const double c = cost(works[i][0]);
    const int n = (int)works[i].size();
    int most = (int)(total / 32 / c);
    most = most < 1 ? 1 : (most > 64 ? 64 : most);
    for (int lo = 0; lo < n; lo += most) {
      const int hi = lo + most < n ? lo + most : n;
      runs.push_back({i, lo, hi, c * (hi - lo)});
    }
  }
  std::stable_sort(runs.begin(), runs.end(), [](const Run& x, const Run& y) { return x.cost > y.cost; });
  std::vector<NsWork> queue[8];
  double load[8] = {};
  for (const Run& r : runs) {
    int x = 0;
    for (int y = 1; y < 8; y++)
      if (load[y] < load[x]) x = y;
    load[x] += r.cost;
    queue[x].insert(queue[x].end(), works[r.mat].begin() + r.lo, works[r.mat].begin() + r.hi);
  }
  size_t longest = 0;
  for (auto& x : queue) {
    std::stable_sort(x.begin(), x.end(), [&](const NsWork& p, const NsWork& q) { return cost(p) > cost(q); });
    longest = x.size() > longest ? x.size() : longest;
  }
  const NsWork none = {-1, 0, 0, 0, 1, 0, 0, 0};
  for (size_t at = 0; at < longest; at++)
    for (auto& x : queue) out.push_back(at < x.size() ? x[at] : none);
  while (!out.empty() && out.back().mat < 0) out.pop_back();
  return shape;
}

int ns_plan(int n, const long* at, const int* rows, const int* cols, const float* scales, void* plan, long plan_bytes,
            long* need_bytes) {
  std::vector<NsMat> mats(n);
  long ws = 0, chunks = 0, need = 0, areas = 0, partials = 0;
  for (int i = 0; i < n; i++) {
    if (!ns_describe(mats[i], at[i], rows[i], cols[i], scales ? scales[i] : 1.f, ws)) return -1;
    chunks += mats[i].parts;
    areas += (long)ns_div_up(mats[i].sp, 64) * ns_div_up(mats[i].lp, 64);
    const long end = mats[i].at + (long)rows[i] * cols[i];
    need = end > need ? end : need;
    if (chunks > NS_MAX_GROUPS || areas > NS_MAX_GROUPS) return -1;
  }
  std::vector<NsWork> work[3];
  NsPlan h = {};
  double time[3];
  for (int k = 0; k < 3; k++) {
    long bytes = 0;
    int slots = 0;
    h.shape[k] = ns_order(mats, k, work[k], slots, bytes, time[k]);
    h.works[k] = (int)work[k].size();
    h.counters = slots > h.counters ? slots : h.counters;
    partials = bytes > partials ? bytes : partials;
  }
  h.pairs = ns_pairs(time);
  h.magic = NS_MAGIC;
  h.partials = ws;
  h.ws_bytes = ws + partials + ((long)h.counters * 4 + 255) / 256 * 256;
  h.need = need;
  h.mats = n;
  h.chunks = (int)chunks;
  h.areas = (int)areas;
  long end = 256;
  auto take = [&](long bytes) {
    const long from = end;
    end += (bytes + 31) / 32 * 32;
    return from;
  };
  h.at_mats = take((long)n * sizeof(NsMat));
  h.at_chunks = take(chunks * 8);
  h.at_areas = take(areas * 16);
  for (int k = 0; k < 3; k++) h.at_works[k] = take((long)h.works[k] * sizeof(NsWork));
  h.bytes = end;
  *need_bytes = h.bytes;
  if (!plan) return 0;
  if (plan_bytes < h.bytes) return -1;
  unsigned char* out = (unsigned char*)plan;
  memset(out, 0, h.bytes);
  memcpy(out, &h, sizeof h);
  memcpy(out + h.at_mats, mats.data(), (size_t)n * sizeof(NsMat));
  int *ck = (int*)(out + h.at_chunks), *ar = (int*)(out + h.at_areas);
  for (int i = 0; i < n; i++) {
    for (int p = 0; p < mats[i].parts; p++) { *ck++ = i; *ck++ = p; }
    for (int ti = 0; ti < ns_div_up(mats[i].sp, 64); ti++)
      for (int tj = 0; tj < ns_div_up(mats[i].lp, 64); tj++) { *ar++ = i; *ar++ = ti; *ar++ = tj; *ar++ = 0; }
  }
  for (int k = 0; k < 3; k++) memcpy(out + h.at_works[k], work[k].data(), work[k].size() * sizeof(NsWork));
  return 0;
}
}  // namespace

extern "C" int madiff_muon_plan(int n, const long* at, const int* rows, const int* cols, const float* scales, void* plan,
                                long plan_bytes, long* need_bytes) {
  if (n < 1 || !at || !rows || !cols || !need_bytes) return -1;
  try {
    return ns_plan(n, at, rows, cols, scales, plan, plan_bytes, need_bytes);
  } catch (...) {                  // out of host memory: nothing leaves a C entry by an exception
    return -1;
  }
}

extern "C" int madiff_muon_plan_ws(const void* plan, long* ws_bytes, long* need_elements) {
  const NsPlan* h = (const NsPlan*)plan;
  if (!h || !ws_bytes || !need_elements || h->magic != NS_MAGIC) return -1;
  *ws_bytes = h->ws_bytes;
  *need_elements = h->need;
  return 0;
}

extern "C" int madiff_muon_step(const void* plan, const void* plan_device, float* p, float* g, float* m, float* ema,
                                void* shadow_bf16, long n, float lr, float momentum, float momentum_rest, int nesterov, float decay,
                                float grad_scale, int zero_grad, int do_ema, float ema_beta, float ema_rest, const int* state,
                                int steps, float a, float b, float c, float eps, void* ws, long ws_bytes, hipStream_t stream) {
  const NsPlan* h = (const NsPlan*)plan;
  if (!h || h->magic != NS_MAGIC || !plan_device || !p || !g || !m || n < h->need || !ws || ws_bytes < h->ws_bytes ||
      ((size_t)ws & 255) || madiff_ortho_check(steps, a, b, c, eps) || do_ema < 0 || do_ema > 2 || (!ema && do_ema) ||
      !(momentum >= 0.f && momentum < 1.f))
    return -1;
  const unsigned char* dev = (const unsigned char*)plan_device;
  NsRun r = {};
  r.grp.mats = (const NsMat*)(dev + h->at_mats);
  r.grp.ws = (unsigned char*)ws;
  r.grp.partials = h->partials;
  r.grp.n_counters = h->counters;
  r.grp.counters = h->ws_bytes - ((long)h->counters * 4 + 255) / 256 * 256;
  r.chunks = (const int*)(dev + h->at_chunks);
  r.areas = (const int*)(dev + h->at_areas);
  r.n_chunks = h->chunks;
  r.n_areas = h->areas;
  r.per_chunks = r.per_areas = 1;
  for (int k = 0; k < 3; k++) {
    r.shape[k] = h->shape[k];
    r.work[k] = {(const NsWork*)(dev + h->at_works[k]), h->works[k], 1, 1};
  }
  NsSource q = {};
  q.g = g;
  q.m = m;
  q.mu = momentum;
  q.rest = momentum_rest;
  q.grad_scale = grad_scale;
  q.nesterov = nesterov;
  q.zero_grad = zero_grad;
  q.eps = eps;
  q.steps = steps;
  q.shift = ns_shift_of(steps, a, b, c, eps);
  ns_launch_source<2>(r, q, stream);
  MADIFF_CHECK_LAUNCH();
  NsProduct last = {};
  last.p = p;
  last.ema = ema;
  last.shadow = (bf16_t*)shadow_bf16;
  last.decay = decay;
  last.lr = lr;
  last.ema_beta = ema_beta;
  last.ema_rest = ema_rest;
  last.do_ema = do_ema;
  last.state = ema ? state : nullptr;
  return ns_iterate(r, steps, a, b, c, NS_OUT_MUON, last, h->pairs && ns_fits(steps, a, b, c, true), stream);
}
